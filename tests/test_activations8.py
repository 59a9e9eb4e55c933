"""Activations in 8 bits on the CPU: values, gradients, refusals."""

from __future__ import annotations

import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

from kfac_amd import ops
from testing import plain

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _seed_rng() -> None:
    torch.manual_seed(0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1,), (3, 63), (2, 3, 65), (0, 5), (4, 200)])
def test_pack8_values(dtype, shape) -> None:
    x = (torch.randn(shape) * torch.exp(4 * torch.randn(shape))).to(dtype)
    p = ops.pack8(x)
    assert p.codes.shape == x.shape
    assert p.exponents.shape == (*shape[:-1], -(-shape[-1] // 64))
    got = ops.unpack8(p)
    # (fp16 values of this spread hold infinities: their blocks are NaN)
    plain.assert_same(got.double(), plain.values8(x))
    # exact in bfloat16
    plain.assert_same(ops.unpack8(p, torch.bfloat16).float(), got)


def test_pack8_edges() -> None:
    edge = 127 * 2.0**-3
    rows = {
        'zeros': torch.zeros(64),
        'edge': torch.full((64,), edge),
        'above the edge': torch.full((64,), edge * (1 + 2.0**-23)),
        'ties': torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5]),
        'least': torch.tensor([2.0**-126, 2.0**-127, 2.0**-149]),
        'largest': torch.tensor([torch.finfo(torch.float32).max, -1.0]),
    }
    for name, x in rows.items():
        got = ops.unpack8(ops.pack8(x)).double()
        assert torch.equal(got, plain.values8(x)), name
        assert got.isfinite().all(), name


@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
def test_pack8_not_finite(bad) -> None:
    x = torch.randn(2, 130)
    x[0, 70] = bad
    got = ops.unpack8(ops.pack8(x))
    assert got[0, 64:128].isnan().all()
    clean = torch.cat([got[0, :64], got[0, 128:], got[1]])
    assert clean.isfinite().all()


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
@pytest.mark.parametrize('dtype', TYPES)
def test_gelu8(dtype, approximate) -> None:
    x = (3 * torch.randn(5, 100)).to(dtype).requires_grad_()
    y, packed = ops.gelu8(x, approximate=approximate, packed_output=True)
    want = plain.gelu(x.detach().double(), approximate)
    # 8 roundings of values no larger than x
    off = 8 * plain.UNIT * (1 + x.detach().double().abs())
    plain.assert_within(y.detach(), want, off)
    again = ops.pack8(y.detach())
    assert torch.equal(packed.codes, again.codes)
    assert torch.equal(packed.exponents, again.exponents)
    dy = torch.randn(5, 100).to(dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    x8 = plain.values8(x.detach())
    want = dy.double() * plain.gelu_slope(x8, approximate)
    off = 16 * plain.UNIT * dy.double().abs() * (1 + x8.abs())
    plain.assert_within(dx, want, off)
    # without a gradient to compute the input is not packed
    with torch.no_grad():
        y2, packed2 = ops.gelu8(x, approximate=approximate)
    assert torch.equal(y2, y) and packed2 is None


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
def test_gelu8_gradient_against_differences(approximate) -> None:
    x = torch.linspace(-6, 6, 200)
    f = ops.gelu8_forward(x, approximate=approximate)
    dx = ops.gelu8_backward(
        torch.ones(200), f.packed_input, approximate=approximate,
    )
    at = ops.unpack8(f.packed_input).double()
    step = 1e-5
    diff = (
        plain.gelu(at + step, approximate) - plain.gelu(at - step, approximate)
    ) / (2 * step)
    # the difference's own error: step^2 / 6 times the third derivative
    # (below 3), and 64 bit rounding over the step
    torch.testing.assert_close(dx.double(), diff, rtol=0, atol=2e-6)


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
def test_gelu8_far_values(approximate) -> None:
    x = torch.tensor([1e20, -1e20, 40.0, -40.0, 0.0])
    f = ops.gelu8_forward(x.view(5, 1), approximate=approximate)
    want = torch.tensor([1e20, 0.0, 40.0, 0.0, 0.0])
    assert torch.equal(f.y.flatten().abs(), want)
    dx = ops.gelu8_backward(
        torch.ones(5, 1), f.packed_input, approximate=approximate,
    )
    assert torch.equal(dx.flatten(), torch.tensor([1.0, 0, 1, 0, 0.5]))


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('needs_grad', [False, True])
@pytest.mark.parametrize('packed_output', [False, True])
def test_gelu8_forward_mode(
    dtype, approximate, needs_grad, packed_output,
) -> None:
    x = (3 * torch.randn(5, 100)).to(dtype)
    dx = torch.randn(5, 100).to(dtype)
    want = dx.double() * plain.gelu_slope(x.double(), approximate)
    off = 16 * plain.UNIT * dx.double().abs() * (1 + x.double().abs())
    alone, _ = ops.gelu8(x, approximate=approximate)
    x.requires_grad_(needs_grad)
    with fwAD.dual_level():
        y, packed = ops.gelu8(
            fwAD.make_dual(x, dx),
            approximate=approximate,
            packed_output=packed_output,
        )
        y, dy = fwAD.unpack_dual(y)
    assert torch.equal(y, alone)
    assert y.requires_grad == needs_grad
    assert (packed is not None) == packed_output
    plain.assert_within(dy.detach(), want, off)


def test_other_forward_mode() -> None:
    x, dx, w = torch.randn(5, 64), torch.randn(5, 64), torch.randn(3, 64)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, dx)
        dy = fwAD.unpack_dual(ops.linear8(dual, w)).tangent
        # no tangent is dropped in silence
        with pytest.raises(RuntimeError):
            ops.linear8(dual, w.clone().requires_grad_())
        with pytest.raises(RuntimeError):
            ops.layer_norm(dual)
    assert torch.equal(dy, F.linear(dx, w))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('out', TYPES)
def test_weight_grad8(dtype, out) -> None:
    x = torch.randn(2, 19, 70)
    g = torch.randn(2, 19, 33).to(dtype)
    packed = ops.pack8(x)
    dw, db = ops.weight_grad8(g, packed, dtype=out)
    want = plain.weight_grads(g, plain.values8(x))
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])
    assert ops.weight_grad8(g, packed, bias=False)[1] is None


def test_weight_grad8_no_rows() -> None:
    dw, db = ops.weight_grad8(torch.zeros(0, 5), ops.pack8(torch.zeros(0, 7)))
    assert torch.equal(dw, torch.zeros(5, 7))
    assert torch.equal(db, torch.zeros(5))


def test_linear8_matches_linear() -> None:
    x = torch.randn(4, 6, 70, requires_grad=True)
    w = torch.randn(33, 70, requires_grad=True)
    b = torch.randn(33, requires_grad=True)
    g = torch.randn(4, 6, 33)
    y = ops.linear8(x, w, b)
    want = F.linear(x, w, b)
    assert torch.equal(y, want)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    wx, _, _ = torch.autograd.grad(want, (x, w, b), g)
    torch.testing.assert_close(dx, wx)
    exact = plain.weight_grads(g, plain.values8(x.detach()))
    plain.assert_within(dw, *exact['dw'])
    plain.assert_within(db, *exact['db'])


def test_linear8_gradient_against_differences() -> None:
    # x of whole numbers up to 127 is its own 8 bit form, so the gradients
    # are those of the plain product
    x = torch.randint(-127, 128, (5, 64)).float()
    x[:, 0] = 127
    w = torch.randn(3, 64, requires_grad=True)
    c = torch.randn(5, 3)
    (ops.linear8(x, w) * c).sum().backward()
    base = w.detach().double()
    for n, k in ((0, 0), (1, 17), (2, 63)):
        step = torch.zeros(3, 64, dtype=torch.float64)
        step[n, k] = 1e-3
        up = ((x.double() @ (base + step).t()) * c.double()).sum()
        down = ((x.double() @ (base - step).t()) * c.double()).sum()
        diff = (up - down) / 2e-3
        # linear: only rounding, of 5 terms up to 127 * |c|
        assert abs(float(diff) - float(w.grad[n, k])) < 1e-3


@pytest.mark.parametrize('m,n,k', [(1, 3, 5), (4096, 33, 70)])
def test_parameters_of_two_types(m, n, k) -> None:
    # each gradient is the float32 sum, rounded once to its own type
    f32, bf16, f16 = TYPES
    x, g = torch.randn(m, k), 1 + torch.randn(m, n)
    for xt, bt in ((bf16, f32), (f32, bf16), (f16, bf16)):
        p = ops.pack8(x.to(xt))
        want = plain.weight_grads(g.to(xt), ops.unpack8(p).double())
        w = torch.randn(n, k).to(xt).requires_grad_()
        b = torch.randn(n).to(bt).requires_grad_()
        ops.linear8(x.to(xt), w, b).backward(g.to(xt))
        assert (w.grad.dtype, b.grad.dtype) == (xt, bt)
        plain.assert_within(w.grad, *want['dw'])
        plain.assert_within(b.grad, *want['db'])
        dw, db = ops.weight_grad8(g.to(xt), p, dtype=xt, bias_dtype=bt)
        assert torch.equal(dw, w.grad) and torch.equal(db, b.grad)
    # of a type that the operators do not have: from the float32 sum
    b = torch.randn(n).double().requires_grad_()
    ops.linear8(x, w.detach().float().requires_grad_(), b).backward(g)
    assert b.grad.dtype == torch.float64
    want = plain.weight_grads(g, ops.unpack8(p).double())
    plain.assert_within(b.grad.float(), *want['db'])
    with pytest.raises(TypeError):
        ops.weight_grad8(g, p, bias_dtype=torch.float64)
    dw, db = ops.weight_grad8(
        g[:0], ops.pack8(x[:0]), dtype=f16, bias_dtype=f32,
    )
    assert (dw.dtype, db.dtype) == (f16, f32)
    assert not dw.any() and not db.any()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('bias', [*TYPES, torch.float64])
def test_linear8_bias_type_without_gradients(dtype, bias) -> None:
    x, w = torch.randn(4, 8).to(dtype), torch.randn(3, 8).to(dtype).requires_grad_()
    b = torch.randn(3).to(bias).requires_grad_()
    y = ops.linear8(x, w, b)
    with torch.no_grad():
        assert torch.equal(ops.linear8(x, w, b), y)
    assert torch.equal(ops.linear8(x, w.detach(), b.detach()), y)
    kind = x.device.type
    with torch.autocast(kind, dtype=torch.bfloat16):
        y = ops.linear8(x, w, b)
        with torch.no_grad():
            assert torch.equal(ops.linear8(x, w, b), y)
    assert y.dtype == torch.bfloat16


def test_linear8_some_gradients() -> None:
    x = torch.randn(4, 8)
    w, b = torch.randn(3, 8), torch.randn(3)
    for flags in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1), (0, 0, 0)):
        args = [
            t.clone().requires_grad_(bool(f)) for t, f in zip((x, w, b), flags)
        ]
        y = ops.linear8(*args)
        assert y.requires_grad == any(flags)
        if any(flags):
            y.sum().backward()
        for t, f in zip(args, flags):
            assert (t.grad is not None) == bool(f)
    with torch.no_grad():
        y = ops.linear8(x, w.requires_grad_(), b)
    assert not y.requires_grad


def test_linear8_autocast() -> None:
    x = torch.randn(4, 8, requires_grad=True)
    w = torch.randn(3, 8, requires_grad=True)
    b = torch.randn(3, requires_grad=True)
    with torch.autocast('cpu', dtype=torch.bfloat16):
        y = ops.linear8(x, w, b)
        want = F.linear(x, w, b)
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, want)
    y.float().sum().backward()
    assert (x.grad.dtype, w.grad.dtype) == (torch.float32, torch.float32)
    xb = x.detach().bfloat16()
    exact = plain.weight_grads(torch.ones(4, 3), plain.values8(xb))
    plain.assert_within(w.grad, *exact['dw'])


def test_autocast_around_everything() -> None:
    # autocast chooses linear8's type and nothing else
    x, g = torch.randn(50, 70), torch.randn(50, 33)
    w = torch.randn(33, 70, requires_grad=True)
    b = torch.randn(33, requires_grad=True)
    norm = torch.randn(70), torch.randn(70)

    def passes() -> list[torch.Tensor]:
        p = ops.pack8(x)
        out = [*p, ops.unpack8(p), *ops.weight_grad8(g, p)]
        for form in ('none', 'tanh'):
            f = ops.gelu8_forward(x, approximate=form)
            out += [f.y, ops.gelu8_backward(x, p, approximate=form)]
        n = ops.layer_norm_forward(x, *norm)
        out += [n.y, n.mean, n.rstd]
        return out + [
            *ops.layer_norm_backward(x, p, n.mean, n.rstd, norm[0]),
        ]

    def gradients(inside: bool) -> tuple[torch.Tensor, ...]:
        with torch.autocast('cpu', dtype=torch.bfloat16):
            y = ops.linear8(x, w, b)
            if inside:
                return torch.autograd.grad(y, (w, b), g.to(y.dtype))
        return torch.autograd.grad(y, (w, b), g.to(y.dtype))

    want = passes()
    with torch.autocast('cpu', dtype=torch.bfloat16):
        got = passes()
    for i, (p, q) in enumerate(zip(got, want)):
        assert torch.equal(p, q), i
    for p, q in zip(gradients(True), gradients(False)):
        assert torch.equal(p, q)


def test_linear8_takes_packed_input() -> None:
    x = torch.randn(4, 70)
    w = torch.randn(3, 70, requires_grad=True)
    (a,) = torch.autograd.grad(ops.linear8(x, w).sum(), w)
    (b,) = torch.autograd.grad(
        ops.linear8(x, w, packed=ops.pack8(x)).sum(), w,
    )
    assert torch.equal(a, b)


def test_no_second_derivative() -> None:
    x = torch.randn(3, 8, requires_grad=True)
    y, _ = ops.gelu8(x)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_refusals() -> None:
    x = torch.randn(4, 70)
    p = ops.pack8(x)
    with pytest.raises(TypeError):
        ops.pack8(x.double())
    with pytest.raises(TypeError):
        ops.pack8(torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.pack8(torch.tensor(1.0))
    with pytest.raises(ValueError):
        ops.pack8(torch.zeros(3, 0))
    with pytest.raises(TypeError):
        ops.unpack8(p, torch.float64)
    with pytest.raises(TypeError):
        ops.unpack8(ops.Packed8(p.codes.int(), p.exponents))
    with pytest.raises(ValueError):
        ops.unpack8(ops.Packed8(p.codes, p.exponents[:, :1]))
    with pytest.raises(ValueError):
        ops.unpack8(ops.Packed8(p.codes[:3], p.exponents))
    with pytest.raises(ValueError):
        ops.gelu8_forward(x, approximate='sigmoid')
    with pytest.raises(ValueError):
        ops.gelu8_backward(x[:, :69], p)
    with pytest.raises(TypeError):
        ops.gelu8_backward(x.double(), p)
    with pytest.raises(ValueError):
        ops.weight_grad8(torch.zeros(3, 5), p)
    with pytest.raises(ValueError):
        ops.weight_grad8(torch.zeros(2, 2, 5), p)
    with pytest.raises(TypeError):
        ops.weight_grad8(torch.zeros(4, 5), p, dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.linear8(x, torch.zeros(3, 69))
    with pytest.raises(TypeError):
        ops.linear8(x, torch.zeros(3, 70).bfloat16())
    with pytest.raises(ValueError):
        ops.linear8(x, torch.zeros(3, 70), packed=ops.pack8(x[:3]))
