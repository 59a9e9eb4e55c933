"""Activations kept in 8 bits, and the operators that read them.

A transformer block keeps what its backward pass needs: the input of every
linear layer, of GELU and of layer norm. Here these are kept as 8 bit codes
with a power of two for each 64 consecutive values of a row (1.016 bytes a
value): :func:`pack8` makes the codes, :func:`gelu8`, :func:`linear8` and
:func:`kfac_amd.ops.layer_norm` keep them instead of the tensors, and their
backward passes read the codes directly. Forward values are those of the
exact inputs; only gradients see the rounding, at most 1/254 to 1/127 of the
largest value in the block (half a step of 2^e, 2^e <= max / 63.5).

On the GPU the ops run hand-written HIP kernels (csrc/act8.hip,
csrc/wgrad8.hip), on the CPU :mod:`kfac_amd.ops.reference`.
"""

from __future__ import annotations

from typing import Any
from typing import NamedTuple

import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from kfac_amd import ops
from kfac_amd.ops import reference as ref

FLOAT_TYPES = (torch.float32, torch.bfloat16, torch.float16)


class Packed8(NamedTuple):
    """A tensor's rows in 8 bits.

    Attributes:
        codes: int8, of the tensor's shape.
        exponents: uint8, ceil(n / 64) for each row of n values. A value is
            ``code * 2**(exponent - 127)``; 255 marks a block that held a
            NaN or an infinity, and all of it reads as NaN.
    """

    codes: torch.Tensor
    exponents: torch.Tensor


class Activated8(NamedTuple):
    """What :func:`gelu8_forward` returns."""

    y: torch.Tensor
    packed_input: Packed8 | None
    packed_output: Packed8 | None


# The checks below are those of the CPU; csrc/training.cpp has the same.


def check_rows(x: torch.Tensor, name: str) -> None:
    """Raise unless ``x`` is a tensor of rows of one or more floats."""
    if x.dtype not in FLOAT_TYPES:
        raise TypeError(
            f'{name} must be float32, bfloat16 or float16, got {x.dtype}',
        )
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(
            f'{name} must have rows of one value or more, got shape '
            f'{tuple(x.shape)}',
        )


def check_same_shape(
    a: torch.Tensor,
    b: torch.Tensor,
    names: str,
) -> None:
    """Raise unless both tensors have one shape and device."""
    if a.shape != b.shape or a.device != b.device:
        raise ValueError(
            f'{names} must have the same shape and device, got '
            f'{tuple(a.shape)} on {a.device} and {tuple(b.shape)} on '
            f'{b.device}',
        )


def check_packed(packed: Packed8) -> None:
    """Raise unless ``packed`` is what :func:`pack8` returns."""
    codes, exps = packed
    if codes.dtype != torch.int8 or exps.dtype != torch.uint8:
        raise TypeError(
            'a Packed8 holds int8 codes and uint8 exponents, got '
            f'{codes.dtype} and {exps.dtype}',
        )
    if codes.dim() < 1 or codes.shape[-1] < 1:
        raise ValueError('codes must have rows of one value or more')
    blocks = -(-codes.shape[-1] // ref.BLOCK8)
    if (
        exps.shape != (*codes.shape[:-1], blocks)
        or exps.device != codes.device
    ):
        raise ValueError(
            f'codes of shape {tuple(codes.shape)} do not go with exponents '
            f'of shape {tuple(exps.shape)}',
        )


def check_approximate(approximate: str) -> None:
    """Raise unless ``approximate`` names a form of GELU."""
    if approximate not in ('none', 'tanh'):
        raise ValueError(
            f"approximate must be 'none' or 'tanh', got {approximate!r}",
        )


def pack8(x: torch.Tensor) -> Packed8:
    """The 8 bit form of a tensor's rows (its last dimension).

    Blocks of 64 consecutive values (the last one may be shorter) share the
    least power of two 2^e, -126 <= e <= 121, with max |x| <= 127 * 2^e; a
    code is x / 2^e rounded to the nearest integer, ties to even. Values are
    off by at most 2^(e-1); zero stays zero. ``x`` may be float32, bfloat16
    or float16, of any strides.
    """
    if x.is_cuda:
        ext = ops._require_ext('pack8')
        if ext is not None:
            return Packed8(*ext.pack8(x))
    check_rows(x, 'x')
    return Packed8(*ref.pack8(x))


def unpack8(
    packed: Packed8,
    dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """The values that a :class:`Packed8` stands for.

    Exact in float32 and bfloat16 (a code times a power of two has 7 bits);
    rounded, and beyond 65504 infinite, in float16.
    """
    codes, exps = packed
    if codes.is_cuda:
        ext = ops._require_ext('unpack8')
        if ext is not None:
            return ext.unpack8(codes, exps, dtype)
    check_packed(packed)
    if dtype not in FLOAT_TYPES:
        raise TypeError(f'no values of type {dtype}')
    return ref.unpack8(codes, exps, dtype)


def gelu8_forward(
    x: torch.Tensor,
    *,
    approximate: str = 'none',
    packed_input: bool = True,
    packed_output: bool = False,
) -> Activated8:
    """GELU of ``x`` and, in the same pass, ``x`` in 8 bits.

    ``packed_output`` asks for the 8 bit form of the rounded result too,
    which is what the next linear layer's weight gradient reads: the same
    as ``pack8(y)``, without reading y again. ``packed_input=False`` leaves
    out what only a backward pass needs.
    """
    check_approximate(approximate)
    if x.is_cuda:
        ext = ops._require_ext('gelu8_forward')
        if ext is not None:
            y, *packed = ext.gelu8_forward(
                x, approximate == 'tanh', packed_input, packed_output,
            )
            return Activated8(
                y,
                Packed8(*packed[:2]) if packed_input else None,
                Packed8(*packed[-2:]) if packed_output else None,
            )
    check_rows(x, 'x')
    y = ref.gelu(x, approximate)
    return Activated8(
        y,
        Packed8(*ref.pack8(x)) if packed_input else None,
        Packed8(*ref.pack8(y)) if packed_output else None,
    )


def gelu8_backward(
    dy: torch.Tensor,
    packed_input: Packed8,
    *,
    approximate: str = 'none',
) -> torch.Tensor:
    """Gradient of GELU's input, whose 8 bit form was kept; in dy's type."""
    check_approximate(approximate)
    codes, exps = packed_input
    if dy.is_cuda:
        ext = ops._require_ext('gelu8_backward')
        if ext is not None:
            return ext.gelu8_backward(dy, codes, exps, approximate == 'tanh')
    check_rows(dy, 'dy')
    check_packed(packed_input)
    check_same_shape(dy, codes, 'dy and the packed input')
    return ref.gelu_backward(dy, ref.unpack8(codes, exps), approximate)


def weight_grad8(
    g: torch.Tensor,
    packed_input: Packed8,
    *,
    bias: bool = True,
    dtype: torch.dtype = torch.float32,
    bias_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """A linear layer's weight and bias gradient from its 8 bit input.

    ``dW = g^T a`` and ``db = sum of g`` over all rows: ``g`` is the gradient
    of the layer's output, (..., N); ``packed_input`` holds the layer's
    input, (..., K), with as many rows. Every product is exact and sums are
    kept in float32 for each type of ``g``; the results, (N, K) and (N,),
    are rounded once, to ``dtype`` and ``bias_dtype`` (by default the same).
    Without rows they are zero. The same inputs give the same bits each time.
    N and K are below 2^27.
    """
    codes, exps = packed_input
    if g.is_cuda:
        ext = ops._require_ext('weight_grad8')
        if ext is not None:
            return ext.weight_grad8(g, codes, exps, bias, dtype, bias_dtype)
    check_rows(g, 'g')
    check_packed(packed_input)
    if g.shape[:-1] != codes.shape[:-1] or g.device != codes.device:
        raise ValueError(
            'g and the packed input must have the same rows and device, got '
            f'{tuple(g.shape)} on {g.device} and {tuple(codes.shape)} on '
            f'{codes.device}',
        )
    bias_dtype = dtype if bias_dtype is None else bias_dtype
    for t in (dtype, bias_dtype):
        if t not in FLOAT_TYPES:
            raise TypeError(f'no gradients of type {t}')
    return ref.weight_grad(
        g, ref.unpack8(codes, exps), bias, dtype, bias_dtype,
    )


# -- autograd ----------------------------------------------------------------


class _GELU8(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
        x: torch.Tensor,
        approximate: str,
        packed_output: bool,
    ) -> tuple[torch.Tensor, ...]:
        f = gelu8_forward(
            x,
            approximate=approximate,
            packed_input=ctx.needs_input_grad[0],
            packed_output=packed_output,
        )
        if f.packed_input is not None:
            ctx.save_for_backward(*f.packed_input)
        ctx.save_for_forward(x)  # for jvp only, which runs at once
        ctx.approximate = approximate
        ctx.packed_output = packed_output
        ctx.set_materialize_grads(False)
        if f.packed_output is None:
            return (f.y,)
        ctx.mark_non_differentiable(*f.packed_output)
        return (f.y, *f.packed_output)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: torch.Tensor | None, *_: Any) -> Any:
        if dy is None:
            return None, None, None
        dx = gelu8_backward(
            dy, Packed8(*ctx.saved_tensors), approximate=ctx.approximate,
        )
        return dx, None, None

    @staticmethod
    def jvp(ctx: Any, dx: torch.Tensor, *_: Any) -> Any:
        # the exact input is there: its slope, in elementary operations
        (x,) = ctx.saved_tensors
        dy = ref.gelu_backward(dx, x, ctx.approximate)
        return (dy, None, None) if ctx.packed_output else dy


def gelu8(
    x: torch.Tensor,
    *,
    approximate: str = 'none',
    packed_output: bool = False,
) -> tuple[torch.Tensor, Packed8 | None]:
    """GELU that keeps its input in 8 bits for the backward pass.

    Returns ``(y, packed)``: ``packed`` is y's 8 bit form for the next
    :func:`linear8` if ``packed_output`` asks for it, else None. Forward
    mode's tangents are those of the exact input.
    """
    backward = torch.is_grad_enabled() and x.requires_grad
    # the kernels carry no tangents, the CPU's elementary operations do
    forward = x.is_cuda and fwAD.unpack_dual(x).tangent is not None
    if not backward and not forward:
        f = gelu8_forward(
            x,
            approximate=approximate,
            packed_input=False,
            packed_output=packed_output,
        )
        return f.y, f.packed_output
    y, *packed = _GELU8.apply(x, approximate, packed_output)
    return y, Packed8(*packed) if packed else None


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
        x: torch.Tensor,
        weight: torch.Tensor,
        bias: torch.Tensor | None,
        codes: torch.Tensor | None,
        exps: torch.Tensor | None,
        dtype: torch.dtype,
    ) -> torch.Tensor:
        w = weight.to(dtype)
        b = None if bias is None else bias.to(dtype)
        if ctx.needs_input_grad[1]:
            if codes is None or exps is None:
                codes, exps = pack8(x)
            ctx.save_for_backward(weight, codes, exps)
        else:
            ctx.save_for_backward(weight)
        ctx.dtype = dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        with torch.autocast(x.device.type, enabled=False):
            return F.linear(x, w, b)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, g: torch.Tensor) -> Any:
        weight, *packed = ctx.saved_tensors
        dx = dw = db = None
        with torch.autocast(g.device.type, enabled=False):
            if ctx.needs_input_grad[0]:
                dx = g @ weight.to(ctx.dtype)
        if ctx.needs_input_grad[1]:
            # a bias of another type (float64, say) takes the float32 sum
            own = ctx.bias_dtype in FLOAT_TYPES
            dw, db = weight_grad8(
                g,
                Packed8(*packed),
                bias=ctx.needs_input_grad[2],
                dtype=weight.dtype,
                bias_dtype=ctx.bias_dtype if own else torch.float32,
            )
        elif ctx.needs_input_grad[2]:
            db = g.reshape(-1, g.shape[-1]).sum(0, dtype=torch.float32)
        if db is not None:
            db = db.to(ctx.bias_dtype)
        return dx, dw, db, None, None, None


def linear8(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    packed: Packed8 | None = None,
) -> torch.Tensor:
    """``x @ weight.T + bias`` that keeps ``x`` in 8 bits for its gradients.

    The result is that of ``torch.nn.functional.linear`` (under autocast in
    autocast's type); the weight's gradient comes from the codes.
    The bias may be of another type than ``x`` and ``weight``. ``packed`` is
    the 8 bit form of ``x`` if the op before has made it
    (``packed_output``), which saves the pass that packs it here. Without a
    gradient to compute nothing is packed.
    """
    check_rows(x, 'x')
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(
            f'weight of shape {tuple(weight.shape)} does not fit rows of '
            f'{x.shape[-1]} values',
        )
    if packed is not None:
        check_packed(packed)
        check_same_shape(x, packed.codes, 'x and its packed form')
    dtype = x.dtype
    autocast = torch.is_autocast_enabled(x.device.type)
    if autocast:
        dtype = torch.get_autocast_dtype(x.device.type)
        x = x.to(dtype)
    elif weight.dtype != dtype:
        raise TypeError(
            f'x is {dtype} and weight {weight.dtype}: they must be of one '
            'type outside autocast',
        )
    if not torch.is_grad_enabled() or not (
        weight.requires_grad or x.requires_grad
        or (bias is not None and bias.requires_grad)
    ):
        # autocast casts 16 and 32 bit biases, and keeps the result
        if bias is not None and not (autocast and bias.dtype in FLOAT_TYPES):
            bias = bias.to(dtype)
        return F.linear(x, weight, bias)
    codes, exps = packed if packed is not None else (None, None)
    return _Linear8.apply(x, weight, bias, codes, exps, dtype)
