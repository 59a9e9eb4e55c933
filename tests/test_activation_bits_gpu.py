"""A decoder that keeps its activations in 8 bits, as a whole (GPU)."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import kfac_amd
from kfac_amd import ops
from kfac_amd.models import GELU8
from kfac_amd.models import GPTNeoXModel
from kfac_amd.models import LayerNorm8
from kfac_amd.models import Linear8
from kfac_amd.models.gptneox import KFAC_SKIP_LAYERS

pytestmark = pytest.mark.gpu

SIZES = dict(vocab=997, d=256, n_layers=2, n_heads=4, ffn=640, max_seq=128)


@pytest.fixture(autouse=True)
def _gpu() -> None:
    assert ops.extension_available()
    torch.manual_seed(0)


def models() -> tuple[GPTNeoXModel, GPTNeoXModel]:
    exact = GPTNeoXModel(**SIZES)
    eight = GPTNeoXModel(**SIZES, activation_bits=8)
    eight.load_state_dict(exact.state_dict())
    return exact, eight


def test_matches_the_cpu() -> None:
    _, model = models()
    tokens = torch.randint(0, 997, (3, 100))
    weight = torch.randn(3, 100, 997)
    out = model(tokens)
    (out * weight).sum().backward()
    want = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    model.cuda()
    got = model(tokens.cuda())
    (got * weight.cuda()).sum().backward()
    torch.testing.assert_close(got.cpu(), out, rtol=1e-3, atol=1e-3)
    for n, p in model.named_parameters():
        # values that the two float32 paths round to the two sides of a
        # code's border move by 1/64 of their block's largest, one in some
        # 1e4: 1/64 / sqrt(1e4), a few times over
        off = float((p.grad.cpu() - want[n]).norm() / want[n].norm())
        assert off < 1e-3, (n, off)


def test_autocast_near_the_exact_model() -> None:
    exact, eight = (m.cuda() for m in models())
    tokens = torch.randint(0, 997, (4, 128), device='cuda')
    for m in (exact, eight):
        with torch.autocast('cuda', dtype=torch.bfloat16):
            logits = m(tokens[:, :-1])
        F.cross_entropy(
            logits.float().reshape(-1, 997), tokens[:, 1:].reshape(-1),
        ).backward()
    for (n, p), (_, q) in zip(
        exact.named_parameters(), eight.named_parameters(),
    ):
        assert q.grad.dtype == torch.float32
        # 1.2 % from each of up to 8 kept tensors, and bf16's steps in both
        off = float((p.grad - q.grad).norm() / p.grad.norm())
        assert off < 0.012 * math.sqrt(8) + 0.02, (n, off)


def test_kfac_trains_it_and_holds_no_inputs() -> None:
    _, model = models()
    model.cuda()
    precon = kfac_amd.KFACPreconditioner(
        model, skip_layers=KFAC_SKIP_LAYERS, lr=0.1,
    )
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    tokens = torch.randint(0, 997, (4, 128), device='cuda')
    for _ in range(3):
        opt.zero_grad()
        with torch.autocast('cuda', dtype=torch.bfloat16):
            logits = model(tokens[:, :-1])
            loss = F.cross_entropy(
                logits.reshape(-1, 997), tokens[:, 1:].reshape(-1),
            )
        loss.backward()
        for _, layer in precon._layers.values():
            assert layer._pending_inputs
            assert all(t.numel() == 0 for t in layer._pending_inputs)
        precon.step()
        for n, p in model.named_parameters():
            assert p.grad.isfinite().all(), n
        opt.step()


def test_kfac_factors_match_the_exact_model() -> None:
    tokens = torch.randint(0, 997, (4, 128), device='cuda')
    factors = []
    for m in models():
        m.cuda()
        precon = kfac_amd.KFACPreconditioner(m, skip_layers=KFAC_SKIP_LAYERS)
        m(tokens).square().mean().backward()
        torch.cuda.synchronize()
        factors.append(
            {n: layer.a_factor for n, layer in precon._layers.values()},
        )
    for n, a in factors[0].items():
        torch.testing.assert_close(a, factors[1][n], rtol=1e-3, atol=1e-4)


def test_kfac_output_factors_match_the_exact_model() -> None:
    # attention's output projection too: its output gradient is the residual
    # stream's, into which the norm's gradient is added later
    tokens = torch.randint(0, 997, (16, 128), device='cuda')
    factors = []
    for m in models():
        m.cuda()
        precon = kfac_amd.KFACPreconditioner(m, skip_layers=['embed_out'])
        names = {name for name, _ in precon._layers.values()}
        assert 'layers.0.attention.dense' in names
        for i in range(3):
            m(tokens).square().mean().backward()
            for _, layer in precon._layers.values():
                assert len(layer._pending_grads) == 1
                assert layer._pending_grads[0].numel() > 0
            if i < 2:
                precon.step()
                for _, layer in precon._layers.values():
                    assert not layer._pending_grads
                m.zero_grad()
        torch.cuda.synchronize()
        factors.append(
            {n: layer.g_factor for n, layer in precon._layers.values()},
        )
    # An output gradient g is off by d = 1.2 % from each of the up to 8 kept
    # tensors behind it, at random: entries of g^T g over M = 2048 tokens by
    # d * sqrt(2 M) of a product where the diagonal has M of them, and with
    # N < 800 columns the whole by d * sqrt(2 N / M) < d, and d^2 on the
    # diagonal. The identity that a factor starts from is left out.
    for n, g in factors[0].items():
        eye = 0.95**3 * torch.eye(g.shape[0], device='cuda')
        off = float((g - factors[1][n]).norm() / (g - eye).norm())
        assert off < 2 * 0.012 * math.sqrt(8), (n, off)


def test_keeps_less_memory() -> None:
    tokens = torch.randint(0, 997, (16, 128), device='cuda')
    kept = []
    for m in models():
        m.cuda()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autocast('cuda', dtype=torch.bfloat16):
            out = m(tokens)
        size = out.numel() * out.element_size()
        kept.append(torch.cuda.memory_allocated() - before - size)
        del out
    # per token and layer, exact: two norms' fp32 inputs (8 d) and their
    # bf16 outputs (4 d), qkv (6 d), attention's output (2 d), GELU's input
    # and output (4 ffn); in 8 bits all but qkv and attention's own copy of
    # its output at a byte: less than 0.65 of it with ffn = 2.5 d
    assert kept[1] < 0.65 * kept[0], kept


def test_training_step_captured_and_replayed() -> None:
    norm, up = LayerNorm8(256).cuda(), Linear8(256, 640).cuda()
    act, down = GELU8().cuda(), Linear8(640, 256).cuda()
    params = [*norm.parameters(), *up.parameters(), *down.parameters()]
    x = torch.randn(300, 256, device='cuda', requires_grad=True)
    r = torch.randn(300, 256, device='cuda')
    dy = torch.randn(300, 256, device='cuda')

    def step():
        n = norm(x, r)
        h, packed = act(up(n.y, packed=n.packed_output))
        y = down(h, packed=packed) + n.total
        return torch.autograd.grad(y, [x, *params], dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(300, 256, device='cuda'))
        r.copy_(torch.randn(300, 256, device='cuda'))
        dy.copy_(torch.randn(300, 256, device='cuda'))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
