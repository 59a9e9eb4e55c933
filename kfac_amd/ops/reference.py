"""Pure-torch reference implementations of every K-FAC compute op.

These are the numerics ground truth for the HIP kernels in ``csrc/`` and the
execution path on CPU. Semantics match the reference package
(kfac/layers/utils.py:18-59, kfac/layers/modules.py:123-192) but are fused
differently: the covariance op takes an explicit ``coeff``/``beta`` pair so
the EMA factor update (reference kfac/layers/base.py:375-405) and the
conv spatial scaling fold into a single accumulation epilogue — on MI355X
the HIP kernel does all of this in one pass over HBM.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def append_bias_ones(tensor: torch.Tensor) -> torch.Tensor:
    """Append a column of ones to the last dim (reference utils.py:8-15)."""
    shape = list(tensor.shape[:-1]) + [1]
    return torch.cat([tensor, tensor.new_ones(shape)], dim=-1)


def cov_linear(
    a: torch.Tensor,
    *,
    bias: bool,
    out: torch.Tensor,
    beta: float,
    coeff: float,
) -> torch.Tensor:
    """out = beta * out + coeff * (a'^T @ a'), a' = [a, 1] if bias.

    ``a`` is 2D (rows = batch*seq, cols = in/out features), any float dtype;
    ``out`` is square fp32 and is updated in place. The product is
    symmetrized, matching reference get_cov (utils.py:55-57).
    """
    a = a.reshape(-1, a.shape[-1])
    if bias:
        a = append_bias_ones(a)
    a32 = a.to(out.dtype)
    cov = a32.t() @ a32
    cov = (cov + cov.t()).mul_(0.5 * coeff)
    if beta == 0.0:
        out.copy_(cov)
    else:
        out.mul_(beta).add_(cov)
    return out


def extract_patches(
    x: torch.Tensor,
    kernel_size: tuple[int, int],
    stride: tuple[int, int],
    padding: tuple[int, int],
) -> torch.Tensor:
    """im2col: (N, C, H, W) -> (N, oh, ow, C*kh*kw).

    Matches reference Conv2dModuleHelper._extract_patches
    (kfac/layers/modules.py:210-237).
    """
    if padding[0] + padding[1] > 0:
        x = F.pad(x, (padding[1], padding[1], padding[0], padding[0]))
    x = x.unfold(2, kernel_size[0], stride[0])
    x = x.unfold(3, kernel_size[1], stride[1])
    x = x.permute(0, 2, 3, 1, 4, 5).contiguous()
    return x.view(x.size(0), x.size(1), x.size(2), -1)


def cov_conv_a(
    x: torch.Tensor,
    *,
    kernel_size: tuple[int, int],
    stride: tuple[int, int],
    padding: tuple[int, int],
    bias: bool,
    out: torch.Tensor,
    beta: float,
    coeff_scale: float = 1.0,
) -> torch.Tensor:
    """A-factor contribution of a Conv2d input.

    Equivalent to reference get_a_factor (modules.py:170-178):
    patches / spatial_size, append ones (also divided), cov with
    scale = N*oh*ow. Folded here into a single coefficient
    ``coeff_scale / (M * s^2)`` applied to the raw patch product.
    """
    patches = extract_patches(x, kernel_size, stride, padding)
    s = patches.size(1) * patches.size(2)
    a = patches.view(-1, patches.size(-1))
    m = a.size(0)
    if bias:
        a = append_bias_ones(a)
    coeff = coeff_scale / (m * s * s)
    return cov_linear(a, bias=False, out=out, beta=beta, coeff=coeff)


def cov_conv_g(
    g: torch.Tensor,
    *,
    out: torch.Tensor,
    beta: float,
    coeff_scale: float = 1.0,
) -> torch.Tensor:
    """G-factor contribution of a Conv2d output-gradient (NCHW).

    Reference get_g_factor (modules.py:180-192): NCHW -> rows (N*oh*ow, O),
    divided by spatial size, cov with scale = rows.
    """
    s = g.size(2) * g.size(3)
    rows = g.permute(0, 2, 3, 1).reshape(-1, g.size(1))
    m = rows.size(0)
    coeff = coeff_scale / (m * s * s)
    return cov_linear(rows, bias=False, out=out, beta=beta, coeff=coeff)


def precond_eigen(
    grad: torch.Tensor,
    qa: torch.Tensor,
    qg: torch.Tensor,
    *,
    dgda: torch.Tensor | None = None,
    da: torch.Tensor | None = None,
    dg: torch.Tensor | None = None,
    damping: float = 0.0,
) -> torch.Tensor:
    """Kronecker-eigenbasis preconditioning (reference eigen.py:350-385).

    v1 = QG^T @ grad @ QA; v2 = v1 * dGdA (or v1 / (outer(dG, dA)+damping));
    out = QG @ v2 @ QA^T, cast back to grad dtype.
    """
    g32 = grad.to(qa.dtype)
    v1 = qg.t() @ g32 @ qa
    if dgda is not None:
        v2 = v1 * dgda
    else:
        assert da is not None and dg is not None
        v2 = v1 / (torch.outer(dg, da) + damping)
    return (qg @ v2 @ qa.t()).to(grad.dtype)


def precond_inverse(
    grad: torch.Tensor,
    a_inv: torch.Tensor,
    g_inv: torch.Tensor,
) -> torch.Tensor:
    """Explicit-inverse preconditioning: G^-1 @ grad @ A^-1 (inverse.py:215-234)."""
    g32 = grad.to(g_inv.dtype)
    return (g_inv @ g32 @ a_inv.to(g_inv.dtype)).to(grad.dtype)


def eigh(x: torch.Tensor, *, clamp: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric eigendecomposition in fp32 (reference eigen.py:309-344).

    Returns (d, Q) with eigenvalues ascending; eigenvalues clamped >= 0.
    """
    dt = torch.float64 if x.dtype == torch.float64 else torch.float32
    d, q = torch.linalg.eigh(x.to(dt))
    if clamp:
        d = torch.clamp(d, min=0.0)
    # rocSOLVER can return the eigenvector matrix as a transposed view;
    # downstream kernels and collectives need contiguous storage.
    return d.contiguous(), q.contiguous()


def inv_damped(x: torch.Tensor, damping: float) -> torch.Tensor:
    """(x + damping*I)^-1 via Cholesky in fp32 (reference inverse.py:186-213).

    Falls back to LU inverse if the damped matrix is not positive definite.
    """
    dt = torch.float64 if x.dtype == torch.float64 else torch.float32
    xd = x.to(dt).clone()
    torch.diagonal(xd).add_(damping)
    try:
        chol = torch.linalg.cholesky(xd)
        return torch.cholesky_inverse(chol)
    except Exception:  # singular / not PD: LU fallback
        return torch.linalg.inv(xd)


def triu_pack(x: torch.Tensor) -> torch.Tensor:
    """Pack the upper triangle of a square matrix into a flat vector.

    Wire format for symmetric factors (reference distributed.py:422-446);
    halves bytes on xGMI.
    """
    if x.dim() != 2 or x.size(0) != x.size(1):
        raise ValueError(f'Expected square 2D tensor, got {tuple(x.shape)}')
    n = x.size(0)
    idx = torch.triu_indices(n, n, device=x.device)
    return x[idx[0], idx[1]].contiguous()


def triu_unpack(v: torch.Tensor, n: int) -> torch.Tensor:
    """Inverse of triu_pack: rebuild the full symmetric matrix."""
    out = v.new_empty((n, n))
    idx = torch.triu_indices(n, n, device=v.device)
    out[idx[0], idx[1]] = v
    out.t()[idx[0], idx[1]] = v
    return out


# -- a transformer block's training path, activations kept in 8 bits --------

BLOCK8 = 64  # consecutive values of a row that share a power of two


def pack8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, exponents) of the last dimension's blocks of 64 values.

    value = code * 2^(exponent - 127), with the least power of two that
    keeps the block within +-127; 255 marks a block that holds a NaN or an
    infinity. See :func:`kfac_amd.ops.pack8`.
    """
    *lead, d = x.shape
    blocks = -(-d // BLOCK8)
    v = F.pad(x.to(torch.float32), (0, blocks * BLOCK8 - d))
    v = v.view(*lead, blocks, BLOCK8)
    top = v.abs().amax(-1)
    bad = ~v.isfinite().all(-1)
    part, power = torch.frexp(torch.where(bad, 0.0, top))  # part in [0.5, 1)
    # 127 = 127/128 * 2^7
    e = power.to(torch.int32) - 7 + (part > 127 / 128).to(torch.int32)
    e = torch.where(part > 0, e, -126).clamp(-126, 121)
    inv = torch.exp2(-e.to(torch.float64)).to(torch.float32)
    codes = torch.round(v * inv.unsqueeze(-1)).clamp(-127, 127)
    codes = torch.where(bad.unsqueeze(-1), 0.0, codes).to(torch.int8)
    exps = torch.where(bad, 255, e + 127).to(torch.uint8)
    return codes.view(*lead, blocks * BLOCK8)[..., :d].contiguous(), exps


def unpack8(
    codes: torch.Tensor,
    exponents: torch.Tensor,
    dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """The values that 8 bit codes stand for."""
    scale = torch.exp2(exponents.to(torch.float64) - 127).to(torch.float32)
    scale = torch.where(exponents == 255, torch.nan, scale)
    scale = scale.repeat_interleave(BLOCK8, dim=-1)[..., : codes.shape[-1]]
    return (codes.to(torch.float32) * scale).to(dtype)


def _gelu_gate(x: torch.Tensor) -> torch.Tensor:
    u = math.sqrt(8 / math.pi) * (x + 0.044715 * x * x * x)
    return 1 / (1 + torch.exp(-u))


def gelu(x: torch.Tensor, approximate: str) -> torch.Tensor:
    """x * P(x), P the normal distribution function or its tanh form."""
    v = x.to(torch.float32)
    if approximate == 'tanh':
        return (v * _gelu_gate(v)).to(x.dtype)
    return (v * 0.5 * torch.erfc(-v * math.sqrt(0.5))).to(x.dtype)


def gelu_backward(
    dy: torch.Tensor,
    x: torch.Tensor,
    approximate: str,
) -> torch.Tensor:
    """dy times GELU's slope at x, in dy's type."""
    v = x.to(torch.float32)
    if approximate == 'tanh':
        p = _gelu_gate(v)
        # p (1 - p) is 0 beyond |x| = 30, where x^2 may overflow
        c = v.clamp(-30, 30)
        slope = math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * c * c)
        d = p + c * p * (1 - p) * slope
    else:
        d = 0.5 * torch.erfc(-v * math.sqrt(0.5)) + v * torch.exp(
            -0.5 * v * v,
        ) / math.sqrt(2 * math.pi)
    return (dy.to(torch.float32) * d).to(dy.dtype)


def weight_grad(
    g: torch.Tensor,
    a: torch.Tensor,
    bias: bool,
    dtype: torch.dtype,
    bias_dtype: torch.dtype,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(g^T a, column sums of g) over all rows, summed in fp32."""
    g32 = g.to(torch.float32).reshape(-1, g.shape[-1])
    a32 = a.to(torch.float32).reshape(-1, a.shape[-1])
    db = g32.sum(0).to(bias_dtype) if bias else None
    # autocast would multiply in its own type
    with torch.autocast(g.device.type, enabled=False):
        dw = g32.t() @ a32
    return dw.to(dtype), db


def layer_norm_forward(
    x: torch.Tensor,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    eps: float,
    residual: torch.Tensor | None,
    out_dtype: torch.dtype,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, total, mean, rstd); the statistics are flat, one a row."""
    total = x
    if residual is not None:
        total = (x.to(torch.float32) + residual.to(torch.float32)).to(x.dtype)
    t = total.to(torch.float32)
    mean = t.mean(-1, keepdim=True)
    var = (t - mean).square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    y = (t - mean) * rstd
    if weight is not None:
        y = y * weight.to(torch.float32)
    if bias is not None:
        y = y + bias.to(torch.float32)
    return y.to(out_dtype), total, mean.reshape(-1), rstd.reshape(-1)


def layer_norm_backward(
    dy: torch.Tensor,
    total: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor | None,
    grad_total: torch.Tensor | None,
    dtype: torch.dtype,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias), the parameters' gradients in fp32."""
    d = dy.shape[-1]
    g = dy.to(torch.float32).reshape(-1, d)
    s = rstd.unsqueeze(-1)
    h = (total.to(torch.float32).reshape(-1, d) - mean.unsqueeze(-1)) * s
    q = g if weight is None else g * weight.to(torch.float32)
    dx = s * (
        q - q.mean(-1, keepdim=True) - h * (q * h).mean(-1, keepdim=True)
    )
    if grad_total is not None:
        dx = dx + grad_total.to(torch.float32).reshape(-1, d)
    return dx.to(dtype).view(dy.shape), (g * h).sum(0), g.sum(0)
