"""Layer norm on the GPU, against plain 64 bit forms."""

from __future__ import annotations

import math

import pytest
import torch

from kfac_amd import ops
from testing import plain

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAIRS = [
    (F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32),
    (F16, F16), (F16, F32),
]
# around the widths where a row takes more lanes, and beyond registers
WIDTHS = [
    1, 2, 7, 8, 9, 15, 63, 65, 71, 129, 256, 511, 512, 513, 768, 1001, 1024, 1025, 2047,
    2048, 2049, 2304, 3001, 4095, 4096, 4097, 4160, 6001, 8191, 8192, 8193, 12001, 16384,
    16385, 20001, 33000,
]


@pytest.fixture(autouse=True)
def _gpu() -> None:
    assert ops.extension_available()
    torch.manual_seed(0)


def rand(*shape: int) -> torch.Tensor:
    return torch.randn(*shape, device='cuda')


def check(
    x, w, b, *, r=None, out=None, keep8=False, pack=False, dt=None, eps=1e-5,
):
    """Both passes against the plain form; the forward pass's result."""
    n = ops.layer_norm_forward(
        x, w, b, eps, residual=r, out_dtype=out, packed_input=keep8,
        packed_output=pack,
    )
    total = x if r is None else (x.float() + r.float()).to(x.dtype)
    assert torch.equal(n.total, total)
    y, mean, rstd, off = plain.norm(total, w, b, eps)
    plain.assert_within(n.y, y, off)
    for p, t in ((n.packed_input, n.total), (n.packed_output, n.y)):
        if p is not None:
            q = ops.pack8(t)
            assert torch.equal(p.codes, q.codes)
            assert torch.equal(p.exponents, q.exponents)
    assert (n.packed_input is not None) == keep8
    assert (n.packed_output is not None) == pack
    dy = rand(*x.shape).to(n.y.dtype)
    dx, dw, db = ops.layer_norm_backward(
        dy, n.packed_input if keep8 else n.total, n.mean, n.rstd, w,
        bias=b is not None, grad_total=dt, dtype=x.dtype,
    )
    kept = plain.values8(total) if keep8 else total
    want = plain.norm_grads(dy, kept, n.mean, n.rstd, w, dt)
    plain.assert_within(dx, *want['dx'])
    assert dx.dtype == x.dtype
    if w is None:
        assert dw is None
    else:
        plain.assert_within(dw, *want['dw'])
        assert dw.dtype == w.dtype
    if b is None:
        assert db is None
    else:
        plain.assert_within(db, *want['db'])
    return n


@pytest.mark.parametrize('width', WIDTHS)
@pytest.mark.parametrize('rows', [1, 3, 37])
def test_widths(width, rows) -> None:
    x = 2 * rand(rows, width) + 1
    w, b = rand(width), rand(width)
    check(x, w, b)
    check(
        x, w, b, r=rand(rows, width).bfloat16(), out=BF16, keep8=True,
        pack=True, dt=rand(rows, width),
    )


@pytest.mark.parametrize('inner,outer', PAIRS)
@pytest.mark.parametrize('width', [40, 768, 1001, 3000, 9000, 17000])
def test_types(inner, outer, width) -> None:
    x = (2 * rand(11, width) - 3).to(inner)
    r = rand(11, width).to(inner)
    w, b = rand(width), rand(width)
    check(x, w, b, out=outer, keep8=True, pack=True)
    check(x, w, b, r=r, out=outer, dt=rand(11, width).to(inner))
    # parameters of other types
    check(x, w.bfloat16(), b.half(), out=outer)


@pytest.mark.parametrize('rows', [1, 16, 17, 63, 64, 65, 4096, 5000, 20000])
@pytest.mark.parametrize('width', [24, 64, 100, 250, 256, 600, 1500])
def test_rows(rows, width) -> None:
    check(rand(rows, width), rand(width), rand(width))


def test_optional_parts() -> None:
    x = rand(5, 300)
    w, b = rand(300), rand(300)
    check(x, None, None)
    check(x, w, None)
    check(x, None, b)
    check(x, w, b, eps=0.0)
    check(x.view(5, 3, 100), w[:100], b[:100])
    check(rand(300), w, b)


def test_strides_and_offsets() -> None:
    base = rand(64, 400)
    w, b = rand(802)[1:401], rand(800)[::2]
    check(base.t().contiguous().t(), w, b)
    check(base[:, 1:301], w[:300], b[:300])
    n = ops.layer_norm_forward(base, w, b)
    dy = rand(400, 64).t()
    got = ops.layer_norm_backward(dy, n.total, n.mean, n.rstd, w)
    want = plain.norm_grads(dy, base, n.mean, n.rstd, w, None)
    for g, name in zip(got, ('dx', 'dw', 'db')):
        plain.assert_within(g, *want[name])


def test_far_mean_and_small_spread() -> None:
    # the centred squares, not a difference of large sums: fp32 holds 1e4
    # to within 1e-3, so the values themselves carry the spread exactly
    x = 1e4 + rand(9, 768)
    check(x, rand(768), rand(768))
    check((1e-20 * rand(9, 768)), rand(768), rand(768), eps=0.0)


def test_constant_and_broken_rows() -> None:
    w, b = rand(100), rand(100)
    x = rand(6, 100)
    x[1] = 3
    x[2, 5] = math.nan
    x[4, 7] = math.inf
    n = ops.layer_norm_forward(x, w, b)
    assert torch.equal(n.y[1], b)
    assert n.y[2].isnan().all() and n.y[4].isnan().all()
    clean = [0, 1, 3, 5]
    y, _, _, off = plain.norm(x[clean], w, b, 1e-5)
    plain.assert_within(n.y[clean], y, off)
    dy = rand(6, 100)
    dx, dw, db = ops.layer_norm_backward(dy, n.total, n.mean, n.rstd, w)
    assert dx[2].isnan().all() and dx[clean].isfinite().all()
    assert dw.isnan().all() and db.isfinite().all()


def test_no_rows() -> None:
    w = rand(5).bfloat16()
    n = ops.layer_norm_forward(
        torch.zeros(0, 5, device='cuda'), w, packed_input=True,
    )
    dx, dw, db = ops.layer_norm_backward(
        n.y, n.packed_input, n.mean, n.rstd, w,
    )
    assert dx.shape == (0, 5)
    zero = torch.zeros(5, device='cuda', dtype=BF16)
    assert torch.equal(dw, zero) and torch.equal(db, zero)


@pytest.mark.parametrize('width', [768, 3000, 9000, 17000])
def test_same_bits_each_time(width) -> None:
    x, w, b, dy = rand(3000, width), rand(width), rand(width), rand(3000, width)
    n = ops.layer_norm_forward(x, w, b)
    first = ops.layer_norm_backward(dy, x, n.mean, n.rstd, w)
    for _ in range(3):
        again = ops.layer_norm_backward(dy, x, n.mean, n.rstd, w)
        for p, q in zip(first, again):
            assert torch.equal(p, q)


def test_another_stream() -> None:
    x, w, b = rand(500, 768), rand(768), rand(768)
    n = ops.layer_norm_forward(x, w, b)
    grads = ops.layer_norm_backward(x, n.total, n.mean, n.rstd, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m = ops.layer_norm_forward(x, w, b)
        again = ops.layer_norm_backward(x, m.total, m.mean, m.rstd, w)
    torch.cuda.current_stream().wait_stream(side)
    for t in (m.y, *again):
        t.record_stream(torch.cuda.current_stream())
    assert torch.equal(m.y, n.y)
    for p, q in zip(grads, again):
        assert torch.equal(p, q)


def test_captured_and_replayed() -> None:
    x, w, b, dy = rand(999, 768), rand(768), rand(768), rand(999, 768)

    def step():
        n = ops.layer_norm_forward(x, w, b, packed_input=True)
        return (
            n.y,
            *ops.layer_norm_backward(dy, n.packed_input, n.mean, n.rstd, w),
        )

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        x.copy_(rand(999, 768))
        dy.copy_(rand(999, 768))
        want = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for p, q in zip(out, want):
                assert torch.equal(p, q), i


def test_offsets_beyond_31_bits() -> None:
    rows, width = 2_200_000, 1000  # 2.2e9 values
    x = torch.zeros(rows, width, device='cuda', dtype=BF16)
    tail = rand(300, width).bfloat16()
    x[-300:] = tail
    w, b = rand(width), rand(width)
    n = ops.layer_norm_forward(x, w, b, packed_input=True)
    y, _, _, off = plain.norm(tail, w, b, 1e-5)
    plain.assert_within(n.y[-300:], y, off)
    assert torch.equal(n.y[0], b.bfloat16())
    dy = torch.zeros_like(x)
    dy[-300:] = rand(300, width).bfloat16()
    dx, dw, db = ops.layer_norm_backward(
        dy, n.packed_input, n.mean, n.rstd, w,
    )
    want = plain.norm_grads(
        dy[-300:], plain.values8(tail), n.mean[-300:], n.rstd[-300:], w, None,
    )
    plain.assert_within(dx[-300:], *want['dx'])
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])
    assert not dx[:-300].any()


def test_autograd_block() -> None:
    x = rand(4, 50, 256).requires_grad_()
    r = rand(4, 50, 256).bfloat16().requires_grad_()
    w, b = rand(256).requires_grad_(), rand(256).requires_grad_()
    out = ops.layer_norm(
        x, w, b, residual=r, out_dtype=BF16, keep8=True, packed_output=True,
    )
    dy, dt = rand(4, 50, 256).bfloat16(), rand(4, 50, 256)
    dx, dr, dw, db = torch.autograd.grad(
        (out.y, out.total), (x, r, w, b), (dy, dt),
    )
    n = ops.layer_norm_forward(
        x.detach(), w.detach(), b.detach(), residual=r.detach(),
    )
    want = plain.norm_grads(
        dy, plain.values8(n.total), n.mean, n.rstd, w.detach(), dt,
    )
    plain.assert_within(dx, *want['dx'])
    assert torch.equal(dr, dx.bfloat16())
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])


def test_expanded_gradient() -> None:
    # what the backward pass of a sum hands over: strides of 0
    x = rand(30, 100).requires_grad_()
    w, b = rand(100).requires_grad_(), rand(100).requires_grad_()
    ops.layer_norm(x, w, b).y.sum().backward()
    n = ops.layer_norm_forward(x.detach(), w.detach(), b.detach())
    want = plain.norm_grads(
        torch.ones(30, 100, device='cuda'), n.total, n.mean, n.rstd,
        w.detach(), None,
    )
    plain.assert_within(x.grad, *want['dx'])
    plain.assert_within(w.grad, *want['dw'])
    plain.assert_within(b.grad, *want['db'])


@pytest.mark.parametrize('rows', [1, 40, 4096])
@pytest.mark.parametrize('width', [5, 70, 768, 1001, 3000, 17000])
def test_parameters_of_two_types(rows, width) -> None:
    # each gradient is the float32 sum, rounded once to its own type
    x, dy = rand(rows, width), 1 + rand(rows, width)
    for wt, bt in ((BF16, F32), (F32, BF16), (F16, BF16)):
        w, b = rand(width).to(wt), rand(width).to(bt)
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


@pytest.mark.parametrize('width', [5, 70, 768, 3000, 17000])
@pytest.mark.parametrize('rows', [0, 3, 700])
def test_frozen_parameters(rows, width, monkeypatch) -> None:
    from kfac_amd.ops import norm

    made = []
    backward = norm.layer_norm_backward

    def spy(*args, **kwargs):
        made.append(backward(*args, **kwargs))
        return made[-1]

    monkeypatch.setattr(norm, 'layer_norm_backward', spy)
    x, dy = rand(rows, width), rand(rows, width)
    w, b = rand(width), rand(width)
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
    x, w = rand(4, 10), rand(10)
    n = ops.layer_norm_forward(x, w)
    for bad in (x.double(), x.int()):
        with pytest.raises(TypeError):
            ops.layer_norm_forward(bad)
    for bad in (torch.tensor(1.0).cuda(), torch.zeros(3, 0).cuda()):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(bad)
    for bad in (w[:9], w.view(1, 10), w.cpu()):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(x, bad)
        with pytest.raises(ValueError):
            ops.layer_norm_forward(x, w, bad)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x, w.double())
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x.bfloat16(), out_dtype=F16)
    for bad in (x, x.half(), x.double()):
        with pytest.raises(TypeError):
            ops.layer_norm_forward(x.bfloat16(), residual=bad)
    for bad in (x[:, :1], x.cpu()):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(x, residual=bad)
    args = (x, n.total, n.mean, n.rstd, w)
    for i, bad in (
        (0, x[:3]), (1, x[:3]), (1, x.cpu()), (2, n.mean[:3]),
        (2, n.mean.cpu()), (3, n.rstd.view(4, 1)), (3, n.rstd.double()),
        (4, w[:9]), (1, ops.pack8(x[:3])),
    ):
        with pytest.raises(ValueError):
            ops.layer_norm_backward(*args[:i], bad, *args[i + 1:])
    with pytest.raises(TypeError):
        ops.layer_norm_backward(*args, dtype=BF16)
    with pytest.raises(TypeError):
        ops.layer_norm_backward(
            x, ops.pack8(x), n.mean, n.rstd, dtype=torch.float64,
        )
    with pytest.raises(TypeError):
        ops.layer_norm_backward(
            x.half(), ops.pack8(x), n.mean, n.rstd, dtype=BF16,
        )
    with pytest.raises(TypeError):
        ops.layer_norm_backward(*args, grad_total=x.bfloat16())
    with pytest.raises(ValueError):
        ops.layer_norm_backward(*args, grad_total=x[:3])
