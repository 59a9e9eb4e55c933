"""Layer norm with its residual sum, mixed types and 8 bit activations.

Forward: ``total = x + residual``, ``y = (total - mean) * rstd * weight +
bias``, in one pass over memory (csrc/norm.hip), with y in the type that the
next linear layer computes in and, on request, total and y in 8 bits.
Backward: the gradients of total, weight and bias in one pass, the
parameters' summed over rows in a fixed order.
"""

from __future__ import annotations

from typing import Any
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from kfac_amd import ops
from kfac_amd.ops import reference as ref
from kfac_amd.ops.activations import check_packed
from kfac_amd.ops.activations import check_rows
from kfac_amd.ops.activations import check_same_shape
from kfac_amd.ops.activations import FLOAT_TYPES
from kfac_amd.ops.activations import Packed8


class Normed(NamedTuple):
    """What :func:`layer_norm_forward` returns.

    Attributes:
        y: the normalised rows.
        total: ``x + residual``, or ``x`` itself without a residual.
        mean, rstd: float32, one for each row, flat.
        packed_input: the 8 bit form of ``total``, if asked for.
        packed_output: the 8 bit form of ``y``, if asked for.
    """

    y: torch.Tensor
    total: torch.Tensor
    mean: torch.Tensor
    rstd: torch.Tensor
    packed_input: Packed8 | None
    packed_output: Packed8 | None


def _check_types(inner: torch.dtype, outer: torch.dtype) -> None:
    if inner not in FLOAT_TYPES or outer not in FLOAT_TYPES or (
        inner != outer and torch.float32 not in (inner, outer)
    ):
        raise TypeError(
            f'no layer norm from {inner} to {outer}: the types must be the '
            'same or one of them float32',
        )


def _check_param(p: torch.Tensor | None, name: str, x: torch.Tensor) -> None:
    if p is None:
        return
    if p.dtype not in FLOAT_TYPES:
        raise TypeError(f'{name} must be a float tensor, got {p.dtype}')
    if p.shape != x.shape[-1:] or p.device != x.device:
        raise ValueError(
            f'{name} must have shape ({x.shape[-1]},) on {x.device}, got '
            f'{tuple(p.shape)} on {p.device}',
        )


def layer_norm_forward(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    *,
    residual: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    packed_input: bool = False,
    packed_output: bool = False,
) -> Normed:
    """Layer norm over the last dimension, without autograd.

    Args:
        x: (..., D), float32, bfloat16 or float16.
        weight: (D,) or None for ones.
        bias: (D,) or None for zeros.
        eps: added to the variance.
        residual: added to ``x`` first; the sum keeps x's type, so the
            residual's may not be wider.
        out_dtype: y's type, by default x's; one of the two is float32 if
            they differ.
        packed_input: return the 8 bit form of the sum, which
            :func:`layer_norm_backward` takes in its place.
        packed_output: return the 8 bit form of y, the same as ``pack8(y)``.
    """
    if x.is_cuda:
        ext = ops._require_ext('layer_norm_forward')
        if ext is not None:
            y, total, mean, rstd, *packed = ext.norm_forward(
                x,
                residual,
                weight,
                bias,
                eps,
                out_dtype,
                packed_input,
                packed_output,
            )
            return Normed(
                y,
                total,
                mean,
                rstd,
                Packed8(*packed[:2]) if packed_input else None,
                Packed8(*packed[-2:]) if packed_output else None,
            )
    check_rows(x, 'x')
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _check_types(x.dtype, out_dtype)
    _check_param(weight, 'weight', x)
    _check_param(bias, 'bias', x)
    if residual is not None:
        check_rows(residual, 'residual')
        check_same_shape(x, residual, 'x and residual')
        if torch.promote_types(x.dtype, residual.dtype) != x.dtype:
            raise TypeError(
                f'a residual of {residual.dtype} does not fit a sum of '
                f'{x.dtype}',
            )
    y, total, mean, rstd = ref.layer_norm_forward(
        x, weight, bias, eps, residual, out_dtype,
    )
    return Normed(
        y,
        total,
        mean,
        rstd,
        Packed8(*ref.pack8(total)) if packed_input else None,
        Packed8(*ref.pack8(y)) if packed_output else None,
    )


def layer_norm_backward(
    dy: torch.Tensor,
    total: torch.Tensor | Packed8,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor | None = None,
    *,
    weight_grad: bool = True,
    bias: bool = True,
    grad_total: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
    bias_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Gradients of :func:`layer_norm_forward`: (dx, dweight, dbias).

    Args:
        dy: gradient of y.
        total: ``Normed.total``, or its 8 bit form ``Normed.packed_input``.
        mean: of the forward pass.
        rstd: of the forward pass.
        weight: of the forward pass; without one dweight is None.
        weight_grad: whether to return the weight's gradient.
        bias: whether to return the bias's gradient.
        grad_total: gradient that reaches the sum past the norm; added.
        dtype: dx's type, total's if that is a tensor, else by default dy's.
        bias_dtype: dbias's type, by default dweight's.

    dx is the gradient of the sum, hence of x and of the residual alike.
    dweight comes in the weight's type (float32 without a weight). The same
    inputs give the same bits each time.
    """
    packed = not isinstance(total, torch.Tensor)
    if dy.is_cuda:
        ext = ops._require_ext('layer_norm_backward')
        if ext is not None:
            return ext.norm_backward(
                dy,
                None if packed else total,
                total[0] if packed else None,
                total[1] if packed else None,
                mean,
                rstd,
                weight,
                weight_grad,
                bias,
                grad_total,
                dtype,
                bias_dtype,
            )
    check_rows(dy, 'dy')
    if packed:
        check_packed(total)
        check_same_shape(dy, total.codes, 'dy and total')
        dtype = dy.dtype if dtype is None else dtype
    else:
        check_rows(total, 'total')
        check_same_shape(dy, total, 'dy and total')
        if dtype not in (None, total.dtype):
            raise TypeError(f'dx has the type of total, {total.dtype}')
        dtype = total.dtype
    _check_types(dtype, dy.dtype)
    _check_param(weight, 'weight', dy)
    rows = dy.numel() // dy.shape[-1]
    for t, name in ((mean, 'mean'), (rstd, 'rstd')):
        if (
            t.dtype != torch.float32
            or t.shape != (rows,)
            or t.device != dy.device
        ):
            raise ValueError(f'{name} must hold a float32 for each row')
    if grad_total is not None:
        check_same_shape(dy, grad_total, 'dy and grad_total')
        if grad_total.dtype != dtype:
            raise TypeError(f'grad_total must be {dtype}, as dx is')
    wtype = torch.float32 if weight is None else weight.dtype
    bias_dtype = wtype if bias_dtype is None else bias_dtype
    if bias_dtype not in FLOAT_TYPES:
        raise TypeError(f'no gradients of type {bias_dtype}')
    if packed:
        total = ref.unpack8(*total)
    dx, dw, db = ref.layer_norm_backward(
        dy, total, mean, rstd, weight, grad_total, dtype,
    )
    return (
        dx,
        dw.to(wtype) if weight is not None and weight_grad else None,
        db.to(bias_dtype) if bias else None,
    )


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
        x: torch.Tensor,
        residual: torch.Tensor | None,
        weight: torch.Tensor | None,
        bias: torch.Tensor | None,
        eps: float,
        out_dtype: torch.dtype | None,
        keep8: bool,
        packed_output: bool,
    ) -> tuple[torch.Tensor, ...]:
        n = layer_norm_forward(
            x,
            weight,
            bias,
            eps,
            residual=residual,
            out_dtype=out_dtype,
            packed_input=keep8,
            packed_output=packed_output,
        )
        kept = n.packed_input if keep8 else (n.total, None)
        ctx.save_for_backward(n.mean, n.rstd, weight, *kept)
        ctx.dtype = x.dtype
        ctx.residual_dtype = None if residual is None else residual.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        out = [n.y]
        if residual is not None:
            out.append(n.total)
        if n.packed_output is not None:
            ctx.mark_non_differentiable(*n.packed_output)
            out.extend(n.packed_output)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: torch.Tensor | None, *more: Any) -> Any:
        mean, rstd, weight, kept, exps = ctx.saved_tensors
        dt = more[0] if ctx.residual_dtype is not None else None
        dx, dw, db = dt, None, None
        if dy is not None:
            want = ctx.needs_input_grad
            dx, dw, db = layer_norm_backward(
                dy,
                kept if exps is None else Packed8(kept, exps),
                mean,
                rstd,
                weight,
                weight_grad=want[2],
                bias=want[3],
                grad_total=dt,
                dtype=ctx.dtype,
                bias_dtype=ctx.bias_dtype,
            )
        dr = None
        if ctx.residual_dtype is not None and dx is not None:
            dr = dx.to(ctx.residual_dtype)
        return dx, dr, dw, db, None, None, None, None


class NormOutput(NamedTuple):
    """What :func:`layer_norm` returns: see :class:`Normed`."""

    y: torch.Tensor
    total: torch.Tensor
    packed_output: Packed8 | None


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    *,
    residual: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    keep8: bool = False,
    packed_output: bool = False,
) -> NormOutput:
    """Differentiable layer norm of ``x + residual``.

    Arguments are those of :func:`layer_norm_forward`; ``keep8`` keeps the
    sum in 8 bits for the backward pass instead of the tensor. ``total`` of
    the result continues the residual stream: its gradient joins the norm's
    in one pass.
    """
    keep8 = keep8 and torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, residual, weight, bias)
    )
    y, *more = _LayerNorm.apply(
        x, residual, weight, bias, eps, out_dtype, keep8, packed_output,
    )
    total = more.pop(0) if residual is not None else x
    return NormOutput(y, total, Packed8(*more) if more else None)
