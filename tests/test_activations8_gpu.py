"""Activations in 8 bits on the GPU, against plain 64 bit forms."""

from __future__ import annotations

import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

from kfac_amd import ops
from testing import plain

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
SHAPES = [
    (1,), (1, 1), (3, 7), (3, 63), (2, 64), (5, 65), (2, 3, 100), (0, 5),
    (129, 1001), (300, 768), (17, 2304),
]


@pytest.fixture(autouse=True)
def _gpu() -> None:
    assert ops.extension_available()
    torch.manual_seed(0)


def rand(*shape: int) -> torch.Tensor:
    return torch.randn(*shape, device='cuda')


def same_packed(a: ops.Packed8, b: ops.Packed8) -> None:
    assert torch.equal(a.codes, b.codes)
    assert torch.equal(a.exponents, b.exponents)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_pack8(dtype, shape) -> None:
    x = (rand(*shape) * torch.exp(2 * rand(*shape))).to(dtype)
    p = ops.pack8(x)
    same_packed(p, ops.Packed8(*(t.cuda() for t in ops.pack8(x.cpu()))))
    want = plain.values8(x)
    plain.assert_same(ops.unpack8(p).double(), want)
    plain.assert_same(ops.unpack8(p, BF16).double(), want)
    plain.assert_same(ops.unpack8(p, F16), want.to(F16))


def test_pack8_edges() -> None:
    x = torch.zeros(9, 64, device='cuda')
    edge = 127 * 2.0**-3
    x[1] = edge
    x[2] = edge * (1 + 2.0**-23)
    x[3, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5])
    x[4, :3] = torch.tensor([2.0**-126, 2.0**-127, 2.0**-149])
    x[5, 0] = torch.finfo(F32).max
    x[6, 5] = math.inf
    x[7, 63] = math.nan
    x[8, 0] = -math.inf
    p = ops.pack8(x)
    same_packed(p, ops.Packed8(*(t.cuda() for t in ops.pack8(x.cpu()))))
    got = ops.unpack8(p)
    plain.assert_same(got.double(), plain.values8(x))
    assert got[:6].isfinite().all() and got[6:].isnan().all()


def test_strides_and_offsets() -> None:
    base = rand(70, 300).bfloat16()
    for x in (
        base.t(), base[:, 1:], base[::2, 3:203], base.flatten()[1:1001],
        base[:, :1].expand(70, 130),
    ):
        plain.assert_same(
            ops.unpack8(ops.pack8(x)).double(), plain.values8(x),
        )
    g = rand(300, 70).t()
    p = ops.pack8(base[:, 5:100])
    p = ops.Packed8(p.codes, p.exponents)
    dw, db = ops.weight_grad8(g, p)
    want = plain.weight_grads(g, plain.values8(base[:, 5:100]))
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_gelu8(dtype, approximate, shape) -> None:
    x = (3 * rand(*shape)).to(dtype)
    f = ops.gelu8_forward(x, approximate=approximate, packed_output=True)
    want = plain.gelu(x.double(), approximate)
    # 8 roundings of values no larger than x
    plain.assert_within(f.y, want, 8 * plain.UNIT * (1 + x.double().abs()))
    same_packed(f.packed_input, ops.pack8(x))
    same_packed(f.packed_output, ops.pack8(f.y))
    less = ops.gelu8_forward(x, approximate=approximate, packed_input=False)
    assert torch.equal(less.y, f.y)
    assert less.packed_input is None and less.packed_output is None
    dy = rand(*shape).to(dtype)
    dx = ops.gelu8_backward(dy, f.packed_input, approximate=approximate)
    x8 = plain.values8(x)
    want = dy.double() * plain.gelu_slope(x8, approximate)
    off = 16 * plain.UNIT * dy.double().abs() * (1 + x8.abs())
    plain.assert_within(dx, want, off)


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
@pytest.mark.parametrize('dtype', TYPES)
def test_gelu8_every_sixteen_bit_value(dtype, approximate) -> None:
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).cuda()
    x = bits.view(F16 if dtype == F16 else BF16).to(dtype)
    x = x[x.isfinite()].view(-1, 1)
    f = ops.gelu8_forward(x, approximate=approximate)
    want = plain.gelu(x.double(), approximate)
    # beyond |x| = 40 the gate is 0 or 1 to the last bit
    off = 8 * plain.UNIT * (1 + x.double().abs().clamp(max=40))
    plain.assert_within(f.y, want.nan_to_num(0.0, math.inf, 0.0), off)
    x8 = plain.values8(x)
    dx = ops.gelu8_backward(
        torch.ones_like(x), f.packed_input, approximate=approximate,
    )
    slope = plain.gelu_slope(x8.clamp(-1e6, 1e6), approximate)
    off = 16 * plain.UNIT * (1 + x8.abs().clamp(max=40))
    plain.assert_within(dx, slope, off)


def test_gelu8_tail() -> None:
    # Relative errors, in units of 2^-24, where the values themselves are
    # small. The exponential's argument -x^2 / 2 is rounded three times (a
    # square and two factors): 1.5 x^2 units, and the instruction is off by 2.
    # The polynomial is off by 1.4e-7 (3 units), its 7 fmas by at most 2.2
    # units each (sum of |terms| over their sum), and its argument t by 4,
    # which t m'(t) / m(t) < 2.5 makes 10: 28. One more for the product.
    x = torch.linspace(-10, -1, 9001, device='cuda').view(-1, 1)
    y = ops.gelu8_forward(x).y
    want = plain.gelu(x.double(), 'none')
    off = plain.UNIT * (31 + 1.5 * x.double().square()) * want.abs()
    plain.assert_within(y, want, off)
    # The slope q - |x| e / sqrt(2 pi), q the tail, from -2 down: the
    # exponential's errors are common to both terms, 31 units of each others'
    # (3 roundings of the second) grow by (x^2 + 1) / (x^2 - 1) <= 5 / 3.
    x = -torch.arange(16, 81, device='cuda').view(-1, 1) / 8  # 7 bits each
    f = ops.gelu8_forward(x)
    assert torch.equal(ops.unpack8(f.packed_input), x)
    dx = ops.gelu8_backward(torch.ones_like(x), f.packed_input)
    want = plain.gelu_slope(x.double(), 'none')
    off = plain.UNIT * (54 + 1.5 * x.double().square()) * want.abs()
    plain.assert_within(dx, want, off)


@pytest.mark.parametrize('approximate', ['none', 'tanh'])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('needs_grad', [False, True])
@pytest.mark.parametrize('packed_output', [False, True])
def test_gelu8_forward_mode(
    dtype, approximate, needs_grad, packed_output,
) -> None:
    x = (3 * rand(5, 100)).to(dtype)
    dx = rand(5, 100).to(dtype)
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
    x, dx, w = rand(5, 64), rand(5, 64), rand(3, 64)
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
@pytest.mark.parametrize(
    'm,n,k',
    [
        (1, 1, 1), (1, 5, 64), (2, 128, 128), (31, 33, 65), (64, 256, 256),
        (65, 129, 127), (200, 8, 1000), (1000, 517, 8), (1280, 256, 256),
        (4099, 300, 200), (777, 1001, 333), (3000, 768, 768),
        (33, 2304, 768), (20000, 16, 16), (5000, 32, 4096), (3001, 12, 3415),
        (700, 33, 1025), (9, 64, 6144), (4097, 1, 2000), (16384, 63, 519),
    ],
)
def test_weight_grad8(dtype, m, n, k) -> None:
    p = ops.pack8(rand(m, k) * torch.exp(rand(m, 1)))
    g = (1e-2 * rand(m, n)).to(dtype)
    g[::3] = 0
    dw, db = ops.weight_grad8(g, p)
    want = plain.weight_grads(g, ops.unpack8(p).double())
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])
    again, _ = ops.weight_grad8(g, p, bias=False)
    assert torch.equal(again, dw)
    assert _ is None
    for out in (BF16, F16):
        dw2, db2 = ops.weight_grad8(g, p, dtype=out)
        # the sums, rounded once
        assert torch.equal(dw2, dw.to(out))
        assert torch.equal(db2, db.to(out))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
def test_weight_grad8_not_finite(dtype, bad) -> None:
    m, n, k = 130, 70, 150
    x = rand(m, k)
    x[7, 100] = bad  # block 64..127 of token 7
    g = rand(m, n).to(dtype)
    g[40, 3] = bad
    p = ops.pack8(x)
    dw, db = ops.weight_grad8(g, p)
    a = ops.unpack8(p).double()
    # 64 bit products, with the columns that hold no number apart
    want = plain.weight_grads(g, a)
    assert dw[:, 64:128].isnan().all()
    row = torch.where(
        a[40] == 0, math.nan, a[40].sign() * bad,
    )
    plain.assert_same(dw[3, :64].double(), row[:64])
    plain.assert_same(dw[3, 128:].double(), row[128:])
    clean = torch.arange(n, device='cuda') != 3
    off = want['dw'][1][clean].nan_to_num(0)
    keep = [*range(64), *range(128, k)]
    plain.assert_within(
        dw[clean][:, keep], want['dw'][0][clean][:, keep], off[:, keep],
    )
    plain.assert_same(db[3].double(), torch.full_like(db[3].double(), bad))
    assert db[clean].isfinite().all()


@pytest.mark.parametrize('dtype', TYPES)
def test_weight_grad8_far_values(dtype) -> None:
    # the largest and the least that the types hold
    info = torch.finfo(dtype)
    g = torch.zeros(40, 3, device='cuda', dtype=dtype)
    g[0, 0], g[1, 1], g[2, 2] = info.max, info.tiny, 1
    x = torch.zeros(40, 64, device='cuda')
    x[0], x[1], x[2] = 0.5, 127.0, 2.0**-20
    p = ops.pack8(x)
    dw, db = ops.weight_grad8(g, p)
    want = plain.weight_grads(g, ops.unpack8(p).double())
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])


def test_no_rows() -> None:
    p = ops.pack8(torch.zeros(0, 7, device='cuda'))
    assert ops.unpack8(p).shape == (0, 7)
    dw, db = ops.weight_grad8(torch.zeros(0, 5, device='cuda'), p, dtype=BF16)
    assert torch.equal(dw, torch.zeros(5, 7, device='cuda', dtype=BF16))
    assert torch.equal(db, torch.zeros(5, device='cuda', dtype=BF16))


@pytest.mark.parametrize('m,n,k', [(1, 3, 5), (4096, 33, 70), (16384, 63, 519), (300, 768, 768)])
def test_parameters_of_two_types(m, n, k) -> None:
    # each gradient is the float32 sum, rounded once to its own type
    f32, bf16, f16 = TYPES
    x, g = rand(m, k), 1 + rand(m, n)
    for xt, bt in ((bf16, f32), (f32, bf16), (f16, bf16)):
        p = ops.pack8(x.to(xt))
        want = plain.weight_grads(g.to(xt), ops.unpack8(p).double())
        w = rand(n, k).to(xt).requires_grad_()
        b = rand(n).to(bt).requires_grad_()
        ops.linear8(x.to(xt), w, b).backward(g.to(xt))
        assert (w.grad.dtype, b.grad.dtype) == (xt, bt)
        plain.assert_within(w.grad, *want['dw'])
        plain.assert_within(b.grad, *want['db'])
        dw, db = ops.weight_grad8(g.to(xt), p, dtype=xt, bias_dtype=bt)
        assert torch.equal(dw, w.grad) and torch.equal(db, b.grad)
    # of a type that the operators do not have: from the float32 sum
    b = rand(n).double().requires_grad_()
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
    x, w = rand(4, 8).to(dtype), rand(3, 8).to(dtype).requires_grad_()
    b = rand(3).to(bias).requires_grad_()
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


def test_linear8_training_step() -> None:
    x = rand(64, 20, 256).requires_grad_()
    w = (rand(512, 256) / 16).requires_grad_()
    b = rand(512).requires_grad_()
    with torch.autocast('cuda', dtype=BF16):
        y = ops.linear8(x, w, b)
        want = torch.nn.functional.linear(x, w, b)
    assert torch.equal(y, want)
    g = rand(64, 20, 512).bfloat16()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    (ex,) = torch.autograd.grad(want, x, g)
    assert torch.equal(dx, ex)
    exact = plain.weight_grads(g, plain.values8(x.detach().bfloat16()))
    plain.assert_within(dw, *exact['dw'])
    plain.assert_within(db, *exact['db'])


def test_linear8_backward_under_autocast() -> None:
    x, g = rand(200, 256), rand(200, 300).bfloat16()
    w, b = rand(300, 256).requires_grad_(), rand(300).requires_grad_()
    with torch.autocast('cuda', dtype=BF16):
        y = ops.linear8(x, w, b)
        inside = torch.autograd.grad(y, (w, b), g, retain_graph=True)
    for p, q in zip(inside, torch.autograd.grad(y, (w, b), g)):
        assert torch.equal(p, q)


def test_expanded_gradient() -> None:
    x = rand(30, 100).requires_grad_()
    w, b = rand(70, 100).requires_grad_(), rand(70).requires_grad_()
    y, packed = ops.gelu8(x, packed_output=True)
    ops.linear8(y, w, b, packed=packed).sum().backward()
    g = torch.ones(30, 70, device='cuda')
    want = plain.weight_grads(g, plain.values8(y.detach()))
    plain.assert_within(w.grad, *want['dw'])
    plain.assert_within(b.grad, *want['db'])
    dy = (g.double() @ w.detach().double()).float()
    x8 = plain.values8(x.detach())
    slope = plain.gelu_slope(x8, 'none')
    # 70 additions in dy, 16 roundings in the slope
    off = plain.UNIT * (
        (70 + 4) * (g.double() @ w.detach().double().abs()) * slope.abs()
        + 16 * dy.double().abs() * (1 + x8.abs())
    )
    plain.assert_within(x.grad, dy.double() * slope, off)


def test_two_threads_and_streams() -> None:
    import threading

    x, g = rand(2000, 512), rand(2000, 300)
    want = ops.weight_grad8(g, ops.pack8(x))
    torch.cuda.synchronize()
    results: dict[int, list] = {}

    def work(i: int) -> None:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [ops.weight_grad8(g, ops.pack8(x)) for _ in range(20)]
            stream.synchronize()
        results[i] = got

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(results) == 4
    for got in results.values():
        for dw, db in got:
            assert torch.equal(dw, want[0]) and torch.equal(db, want[1])


def test_another_stream() -> None:
    x, g = rand(500, 256), rand(500, 300)
    p = ops.pack8(x)
    dw, _ = ops.weight_grad8(g, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p2 = ops.pack8(x)
        dw2, _ = ops.weight_grad8(g, p2)
    torch.cuda.current_stream().wait_stream(side)
    for t in (*p2, dw2):
        t.record_stream(torch.cuda.current_stream())
    same_packed(p, p2)
    assert torch.equal(dw, dw2)


def test_captured_and_replayed() -> None:
    x, g, dy = rand(700, 256), rand(700, 300), rand(700, 256)

    def step():
        f = ops.gelu8_forward(x, packed_output=True)
        dx = ops.gelu8_backward(dy, f.packed_input)
        dw, db = ops.weight_grad8(g, f.packed_output)
        return f.y, dx, dw, db

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
        x.copy_(rand(700, 256))
        g.copy_(rand(700, 300))
        want = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b), i


def test_offsets_beyond_31_bits() -> None:
    # 2.2e9 values of 16 bits: byte offsets pass 32 bits, value offsets 31
    rows, n = 2_200_000, 1000
    g = torch.zeros(rows, n, device='cuda', dtype=BF16)
    tail = rand(512, n).bfloat16()
    g[-512:] = tail
    p = ops.pack8(g)
    plain.assert_same(
        ops.unpack8(ops.Packed8(p.codes[-512:], p.exponents[-512:])).double(),
        plain.values8(tail),
    )
    assert not p.codes[:-512].any()
    a = torch.zeros(rows, 64, device='cuda')
    a[-512:] = rand(512, 64)
    pa = ops.pack8(a)
    dw, db = ops.weight_grad8(g, pa)
    want = plain.weight_grads(tail, plain.values8(a[-512:]))
    plain.assert_within(dw, *want['dw'])
    plain.assert_within(db, *want['db'])
    # and as the input that was kept
    small = torch.zeros(rows, 16, device='cuda', dtype=BF16)
    small[-512:] = rand(512, 16).bfloat16()
    dw, _ = ops.weight_grad8(small, p)
    want = plain.weight_grads(small[-512:], plain.values8(tail))
    plain.assert_within(dw, *want['dw'])
    dx = ops.gelu8_backward(g, p)
    x8 = plain.values8(tail)
    want = tail.double() * plain.gelu_slope(x8, 'none')
    off = 16 * plain.UNIT * tail.double().abs() * (1 + x8.abs())
    plain.assert_within(dx[-512:], want, off)


def test_refusals() -> None:
    x = rand(4, 70)
    p = ops.pack8(x)
    with pytest.raises(TypeError):
        ops.pack8(x.double())
    with pytest.raises(TypeError):
        ops.pack8(torch.zeros(4, 4, dtype=torch.int32, device='cuda'))
    with pytest.raises(ValueError):
        ops.pack8(torch.tensor(1.0, device='cuda'))
    with pytest.raises(ValueError):
        ops.pack8(torch.zeros(3, 0, device='cuda'))
    with pytest.raises(TypeError):
        ops.unpack8(p, torch.float64)
    with pytest.raises(TypeError):
        ops.unpack8(ops.Packed8(p.codes.int(), p.exponents))
    for exps in (
        p.exponents[:, :1], p.exponents[:3], p.exponents.view(2, 2, 2),
        p.exponents.cpu(),
    ):
        with pytest.raises(ValueError):
            ops.unpack8(ops.Packed8(p.codes, exps))
        with pytest.raises(ValueError):
            ops.weight_grad8(x, ops.Packed8(p.codes, exps))
        with pytest.raises(ValueError):
            ops.gelu8_backward(x, ops.Packed8(p.codes, exps))
    with pytest.raises(ValueError):
        ops.gelu8_forward(x, approximate='sigmoid')
    with pytest.raises(ValueError):
        ops.gelu8_backward(x[:, :69], p)
    with pytest.raises(TypeError):
        ops.gelu8_backward(x.double(), p)
    with pytest.raises(ValueError):
        ops.gelu8_backward(x.cpu(), p)
    for g in (x[:3], x.view(2, 2, 70), x.cpu()):
        with pytest.raises(ValueError):
            ops.weight_grad8(g, p)
    with pytest.raises(TypeError):
        ops.weight_grad8(x.double(), p)
    with pytest.raises(TypeError):
        ops.weight_grad8(x, p, dtype=torch.float64)
