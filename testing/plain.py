"""Plain 64 bit forms of the transformer block's operators, for tests.

Written from the formulas, apart from kfac_amd.ops.reference. Bounds say how
far a float32 computation with one final rounding may be from them.
"""

from __future__ import annotations

import math

import torch

UNIT = 2.0**-24  # half a step of float32, relative


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Largest absolute error of one rounding below the normal range."""
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def values8(x: torch.Tensor) -> torch.Tensor:
    """What a tensor is after a pass through 8 bits, in float64."""
    out = []
    for part in x.double().split(64, dim=-1):
        top = part.abs().amax(-1, keepdim=True)
        bad = ~part.isfinite().all(-1, keepdim=True)
        # log2 of a double tells 127 * 2^k from its float32 neighbours
        e = torch.ceil(torch.log2(top / 127)).clamp(-126, 121)
        step = torch.exp2(torch.where(bad, 0.0, e))
        v = (part / step).round().clamp(-127, 127) * step
        out.append(torch.where(bad, math.nan, v))
    return torch.cat(out, -1)


def gelu(x: torch.Tensor, approximate: str) -> torch.Tensor:
    """GELU of a float64 tensor."""
    if approximate == 'tanh':
        u = math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)
        return 0.5 * x * (1 + torch.tanh(u))
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))


def gelu_slope(x: torch.Tensor, approximate: str) -> torch.Tensor:
    """GELU's derivative at a float64 tensor."""
    if approximate == 'tanh':
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (x + 0.044715 * x**3))
        return 0.5 * (1 + th) + 0.5 * x * (1 - th**2) * c * (
            1 + 3 * 0.044715 * x**2
        )
    density = torch.exp(-0.5 * x**2) / math.sqrt(2 * math.pi)
    return 0.5 * torch.special.erfc(-x / math.sqrt(2)) + x * density


def norm(
    t: torch.Tensor,
    w: torch.Tensor | None,
    b: torch.Tensor | None,
    eps: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd, bound of a float32 computation's error in y)."""
    t = t.double()
    d = t.shape[-1]
    mean = t.mean(-1, keepdim=True)
    rstd = ((t - mean).square().mean(-1, keepdim=True) + eps) ** -0.5
    h = (t - mean) * rstd
    w = torch.ones_like(h[..., :1]) if w is None else w.double()
    b = torch.zeros_like(h[..., :1]) if b is None else b.double()
    y = h * w + b
    # A sum of D values passes through at most 16 + D / 8192 additions in a
    # lane and 10 across lanes. The mean is off by that many roundings of
    # the mean magnitude, rstd by half as many of itself and the mean's
    # error (second order), and a handful of roundings follow.
    k = 32 + d / 8192
    off = k * (rstd * t.abs().mean(-1, keepdim=True) + h.abs()) * w.abs()
    off = UNIT * (off + 2 * (h * w).abs() + 2 * b.abs())
    # Below 2^-126 float32 numbers are 2^-149 apart: a centred square there
    # is off by up to 2^-150, and so is their mean, the variance 1 / rstd^2;
    # rstd is then off by half of 2^-150 * rstd^2, relative. It tells only
    # where the spread is below 1e-17 and eps is 0 (1e-20: 4e-6).
    off = off + (h * w).abs() * 2.0**-151 * rstd**2
    return y, mean, rstd, off


def norm_grads(
    dy: torch.Tensor,
    t: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    w: torch.Tensor | None,
    dt: torch.Tensor | None,
) -> dict[str, tuple[torch.Tensor, torch.Tensor]]:
    """{name: (gradient, bound of a float32 computation's error)}."""
    d = t.shape[-1]
    g, t = dy.double().reshape(-1, d), t.double().reshape(-1, d)
    m, s = mean.double().reshape(-1, 1), rstd.double().reshape(-1, 1)
    h = (t - m) * s
    q = g if w is None else g * w.double()
    s1 = q.mean(-1, keepdim=True)
    s2 = (q * h).mean(-1, keepdim=True)
    dx = s * (q - s1 - h * s2)
    k = 40 + d / 8192  # additions of a sum, and the roundings around it
    off = s * (
        q.abs()
        + q.abs().mean(-1, keepdim=True)
        + h.abs() * (q * h).abs().mean(-1, keepdim=True)
    )
    if dt is not None:
        dx = dx + dt.double().reshape(-1, d)
        off = off + dt.double().reshape(-1, d).abs() / k
    r = t.shape[0]
    return {
        'dx': (dx.view(dy.shape), (UNIT * k * off).view(dy.shape)),
        # R additions in whatever order, 4 roundings in each product
        'dw': ((g * h).sum(0), UNIT * (r + 4) * (g * h).abs().sum(0)),
        'db': (g.sum(0), UNIT * (r + 4) * g.abs().sum(0)),
    }


def weight_grads(
    g: torch.Tensor,
    a: torch.Tensor,
) -> dict[str, tuple[torch.Tensor, torch.Tensor]]:
    """{name: (gradient, bound of a float32 sum's error)}; a in float64."""
    g = g.double().reshape(-1, g.shape[-1])
    a = a.double().reshape(-1, a.shape[-1])
    m = g.shape[0]
    # Products are exact. A matrix core adds them in its own order and may
    # cut where a rounding would be half as far off: twice the unit for
    # each of M additions, of up to three parts of g.
    k = 2 * UNIT * (3 * m + 8)
    return {
        'dw': (g.t() @ a, k * (g.abs().t() @ a.abs())),
        'db': (g.sum(0), k * g.abs().sum(0)),
    }


def assert_same(got: torch.Tensor, want: torch.Tensor) -> None:
    """Equal values, NaN in the same places."""
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


def assert_within(
    got: torch.Tensor,
    want: torch.Tensor,
    off: torch.Tensor | float = 0.0,
) -> None:
    """``got`` is ``want`` but for ``off`` and one rounding to its type."""
    assert got.shape == want.shape, (got.shape, want.shape)
    got64 = got.double()
    room = (
        off
        + half_step(got.dtype) * (want.abs() + off)
        + tiny(got.dtype)
    )
    top = torch.finfo(got.dtype).max
    same = (got64.isnan() & want.isnan()) | (got64 == want)
    # beyond the type's range: infinite
    over = (want.abs() + room >= top) & got64.isinf()
    over &= got64.sign() == want.sign()
    ok = same | over | ((got64 - want).abs() <= room)
    if not bool(ok.all()):
        at = tuple(int(i) for i in (~ok).nonzero()[0])
        room = room if isinstance(room, float) else room.expand_as(want)[at]
        raise AssertionError(
            f'{int((~ok).sum())} of {ok.numel()} values are off, the first '
            f'at {at}: {got64[at].item()!r}, not {want[at].item()!r} within '
            f'{float(room):.3g}',
        )
