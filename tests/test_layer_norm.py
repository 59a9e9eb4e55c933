"""Layer norm on the CPU: values, gradients, refusals."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from kfac_amd import ops
from testing import plain

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAIRS = [
    (F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32),
    (F16, F16), (F16, F32),
]


@pytest.fixture(autouse=True)
def _seed_rng() -> None:
    torch.manual_seed(0)


@pytest.mark.parametrize('inner,outer', PAIRS)
@pytest.mark.parametrize('keep8', [False, True])
def test_layer_norm(inner, outer, keep8) -> None:
    x = (2 * torch.randn(3, 5, 70) + 1).to(inner).requires_grad_()
    r = torch.randn(3, 5, 70).to(inner).requires_grad_()
    w = torch.randn(70, requires_grad=True)
    b = torch.randn(70, requires_grad=True)
    out = ops.layer_norm(
        x, w, b, residual=r, out_dtype=outer, keep8=keep8,
        packed_output=True,
    )
    total = x.detach() + r.detach()
    assert out.y.dtype == outer and out.total.dtype == inner
    assert torch.equal(out.total, total)
    y, mean, rstd, off = plain.norm(total, w.detach(), b.detach(), 1e-5)
    plain.assert_within(out.y.detach(), y, off)
    again = ops.pack8(out.y.detach())
    assert torch.equal(out.packed_output.codes, again.codes)
    assert torch.equal(out.packed_output.exponents, again.exponents)
    dy = torch.randn(3, 5, 70).to(outer)
    dt = torch.randn(3, 5, 70).to(inner)
    dx, dr, dw, db = torch.autograd.grad(
        (out.y, out.total), (x, r, w, b), (dy, dt),
    )
    n = ops.layer_norm_forward(
        x.detach(), w.detach(), b.detach(), residual=r.detach(),
    )
    kept = plain.values8(total) if keep8 else total
    want = plain.norm_grads(dy, kept, n.mean, n.rstd, w.detach(), dt)
    plain.assert_within(dx, *want['dx'])
    assert torch.equal(dr, dx)
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])


def test_matches_torch() -> None:
    x = torch.randn(7, 33, requires_grad=True)
    w = torch.randn(33, requires_grad=True)
    b = torch.randn(33, requires_grad=True)
    g = torch.randn(7, 33)
    y = ops.layer_norm(x, w, b).y
    want = F.layer_norm(x, (33,), w, b)
    torch.testing.assert_close(y, want)
    for a, e in zip(
        torch.autograd.grad(y, (x, w, b), g),
        torch.autograd.grad(want, (x, w, b), g),
    ):
        torch.testing.assert_close(a, e, rtol=1e-5, atol=1e-5)


def test_gradient_against_differences() -> None:
    x = torch.randn(2, 9)
    w, b, c = torch.randn(9), torch.randn(9), torch.randn(2, 9)
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    (ops.layer_norm(*args).y * c).sum().backward()

    def loss(x64, w64, b64):
        return (plain.norm(x64, w64, b64, 1e-5)[0] * c.double()).sum()

    step = 1e-6
    for i in range(3):
        base = [t.double() for t in (x, w, b)]
        for j in range(base[i].numel()):
            sides = []
            for sign in (1, -1):
                moved = [t.clone() for t in base]
                moved[i].view(-1)[j] += sign * step
                sides.append(float(loss(*moved)))
            diff = (sides[0] - sides[1]) / (2 * step)
            # step^2 of third derivatives, 1e-15 / step of rounding, and
            # float32's roundings of gradients of order 10
            assert abs(diff - float(args[i].grad.view(-1)[j])) < 2e-5


def test_optional_parts() -> None:
    x = torch.randn(4, 10, requires_grad=True)
    w = torch.randn(10, requires_grad=True)
    b = torch.randn(10, requires_grad=True)
    for args in ((None, None), (w, None), (None, b), (w, b)):
        out = ops.layer_norm(x, *args)
        assert out.total is x and out.packed_output is None
        y, _, _, off = plain.norm(
            x.detach(), *(None if t is None else t.detach() for t in args),
            1e-5,
        )
        plain.assert_within(out.y.detach(), y, off)
        given = [t for t in (x, *args) if t is not None]
        for t, grad in zip(given, torch.autograd.grad(out.y.sum(), given)):
            assert grad.shape == t.shape


def test_unused_outputs() -> None:
    x = torch.randn(4, 10, requires_grad=True)
    r = torch.randn(4, 10, requires_grad=True)
    w = torch.randn(10, requires_grad=True)
    out = ops.layer_norm(x, w, residual=r)
    (out.total * 2).sum().backward()
    assert torch.equal(x.grad, torch.full((4, 10), 2.0))
    assert torch.equal(r.grad, x.grad)
    out = ops.layer_norm(x, w, residual=r)
    gx, gr = torch.autograd.grad(out.y.sum(), (x, r))
    assert torch.equal(gx, gr)


def test_narrow_residual_gets_its_own_type() -> None:
    x = torch.randn(4, 10, requires_grad=True)
    r = torch.randn(4, 10).bfloat16().requires_grad_()
    out = ops.layer_norm(x, residual=r, out_dtype=BF16)
    out.y.float().square().sum().backward()
    assert r.grad.dtype == BF16
    assert torch.equal(r.grad, x.grad.bfloat16())


def test_no_rows_and_constant_rows() -> None:
    w, b = torch.randn(5), torch.randn(5)
    n = ops.layer_norm_forward(torch.zeros(0, 5), w, b, packed_output=True)
    assert n.y.shape == (0, 5) and n.mean.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(
        torch.zeros(0, 5), n.total, n.mean, n.rstd, w,
    )
    assert dx.shape == (0, 5)
    assert torch.equal(dw, torch.zeros(5)) and torch.equal(db, dw)
    n = ops.layer_norm_forward(torch.full((2, 5), 3.0), w, b)
    assert torch.equal(n.y, b.expand(2, 5))


@pytest.mark.parametrize('rows', [1, 4096])
@pytest.mark.parametrize('width', [70])
def test_parameters_of_two_types(rows, width) -> None:
    # each gradient is the float32 sum, rounded once to its own type
    x, dy = torch.randn(rows, width), 1 + torch.randn(rows, width)
    for wt, bt in ((BF16, F32), (F32, BF16), (F16, BF16)):
        w, b = torch.randn(width).to(wt), torch.randn(width).to(bt)
        n = ops.layer_norm_forward(x, w, b)
        want = plain.norm_grads(dy, x, n.mean, n.rstd, w, None)
        w.requires_grad_(), b.requires_grad_()
        ops.layer_norm(x, w, b).y.backward(dy)
        assert (w.grad.dtype, b.grad.dtype) == (wt, bt)
        plain.assert_within(w.grad, *want['dw'])
        plain.assert_within(b.grad, *want['db'])
        _, dw, db = ops.layer_norm_backward(
            dy, x, n.mean, n.rstd, w.detach(), bias_dtype=bt,
        )
        assert torch.equal(dw, w.grad) and torch.equal(db, b.grad)
    _, dw, db = ops.layer_norm_backward(
        dy, x, n.mean, n.rstd, bias_dtype=BF16,
    )
    assert dw is None and db.dtype == BF16
    plain.assert_within(db, *want['db'])
    with pytest.raises(TypeError):
        ops.layer_norm_backward(
            dy, x, n.mean, n.rstd, bias_dtype=torch.float64,
        )
    none = ops.layer_norm_backward(
        dy[:0], x[:0], n.mean[:0], n.rstd[:0], w.detach(), bias_dtype=F32,
    )
    assert none[1].dtype == F16 and none[2].dtype == F32
    assert not none[1].any() and not none[2].any()


@pytest.mark.parametrize('width', [70])
@pytest.mark.parametrize('rows', [0, 3, 700])
def test_frozen_parameters(rows, width, monkeypatch) -> None:
    from kfac_amd.ops import norm

    made = []
    backward = norm.layer_norm_backward

    def spy(*args, **kwargs):
        made.append(backward(*args, **kwargs))
        return made[-1]

    monkeypatch.setattr(norm, 'layer_norm_backward', spy)
    x, dy = torch.randn(rows, width), torch.randn(rows, width)
    w, b = torch.randn(width), torch.randn(width)
    grads = []
    for frozen in ((), (w,), (b,), (w, b)):
        x.requires_grad_()
        for t in (w, b):
            t.requires_grad_(all(t is not f for f in frozen))
            t.grad = x.grad = None
        ops.layer_norm(x, w, b).y.backward(dy)
        grads.append((x.grad, w.grad, b.grad))
    for (dx, dw, db), got, skip in zip(
        grads, made, ((), (1,), (2,), (1, 2)),
    ):
        for i, (p, q) in enumerate(zip((dx, dw, db), got)):
            if i in skip:
                assert p is None and q is None
            else:
                assert torch.equal(p, grads[0][i]) and torch.equal(q, p)


def test_refusals() -> None:
    x = torch.randn(4, 10)
    w = torch.randn(10)
    n = ops.layer_norm_forward(x, w)
    for bad in (x.double(), x.int()):
        with pytest.raises(TypeError):
            ops.layer_norm_forward(bad)
    for bad in (torch.tensor(1.0), torch.zeros(3, 0)):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(bad)
    for bad in (torch.zeros(9), torch.zeros(1, 10)):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(x, bad)
        with pytest.raises(ValueError):
            ops.layer_norm_forward(x, w, bad)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x, w.double())
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x.bfloat16(), out_dtype=F16)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x.bfloat16(), residual=x)
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x, residual=x[:, :1])
    args = (x, n.total, n.mean, n.rstd, w)
    for i, bad in (
        (0, x[:3]), (1, x[:3]), (2, n.mean[:3]), (3, n.rstd.view(4, 1)),
        (4, w[:9]),
    ):
        with pytest.raises(ValueError):
            ops.layer_norm_backward(*args[:i], bad, *args[i + 1:])
    with pytest.raises(ValueError):
        ops.layer_norm_backward(
            x, ops.pack8(x[:3]), n.mean, n.rstd, w,
        )
    with pytest.raises(TypeError):
        ops.layer_norm_backward(*args, dtype=BF16)
    with pytest.raises(TypeError):
        ops.layer_norm_backward(*args, grad_total=x.bfloat16())
    with pytest.raises(ValueError):
        ops.layer_norm_backward(*args, grad_total=x[:3])
