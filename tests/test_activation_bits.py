"""A decoder that keeps its activations in 8 bits, as a whole (CPU).

Its gradients are compared with a float64 model whose backward pass reads
rounded values at the same places, and with the exact model's.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import kfac_amd
from kfac_amd.models import GELU8
from kfac_amd.models import GPTNeoXModel
from kfac_amd.models import LayerNorm8
from kfac_amd.models import Linear8
from kfac_amd.models.gptneox import KFAC_SKIP_LAYERS
from testing import plain

SIZES = dict(vocab=97, d=64, n_layers=2, n_heads=4, ffn=160, max_seq=32)


@pytest.fixture(autouse=True)
def _seed_rng() -> None:
    torch.manual_seed(0)


def models() -> tuple[GPTNeoXModel, GPTNeoXModel]:
    exact = GPTNeoXModel(**SIZES)
    eight = GPTNeoXModel(**SIZES, activation_bits=8)
    eight.load_state_dict(exact.state_dict())
    return exact, eight


def linear64(x, w, b):
    """x w^T + b; w's gradient comes from the 8 bit values of x."""
    x8 = plain.values8(x.detach())
    y = x @ w.detach().t() + (x8 @ w.t() - x8 @ w.detach().t())
    return y if b is None else y + b


def gelu64(x):
    slope = plain.gelu_slope(plain.values8(x.detach()), 'none')
    return plain.gelu(x.detach(), 'none') + slope * (x - x.detach())


class Norm64(torch.autograd.Function):
    @staticmethod
    def forward(ctx, t, w, b):
        y, mean, rstd, _ = plain.norm(t, w, b, 1e-5)
        ctx.save_for_backward(t, w, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        t, w, mean, rstd = ctx.saved_tensors
        g = plain.norm_grads(dy, plain.values8(t), mean, rstd, w, None)
        return g['dx'][0], g['dw'][0], g['db'][0]


def forward64(p, tokens, sizes):
    """The decoder in float64 on a dict of parameters."""
    d, heads = sizes['d'], sizes['n_heads']
    b, s = tokens.shape
    x = p['embed_in.weight'][tokens] + p['embed_pos.weight'][:s]
    mask = torch.full((s, s), -math.inf, dtype=torch.float64).triu(1)
    for i in range(sizes['n_layers']):
        def get(name, i=i):
            return p[f'layers.{i}.{name}.weight'], p[f'layers.{i}.{name}.bias']

        y = Norm64.apply(x, *get('input_layernorm'))
        qkv = linear64(y, *get('attention.query_key_value'))
        q, k, v = (
            t.view(b, s, heads, d // heads).transpose(1, 2)
            for t in qkv.chunk(3, -1)
        )
        a = (q @ k.transpose(-1, -2)) / math.sqrt(d // heads) + mask
        a = (a.softmax(-1) @ v).transpose(1, 2).reshape(b, s, d)
        x = x + linear64(a, *get('attention.dense'))
        y = Norm64.apply(x, *get('post_attention_layernorm'))
        h = gelu64(linear64(y, *get('mlp.dense_h_to_4h')))
        x = x + linear64(h, *get('mlp.dense_4h_to_h'))
    x = Norm64.apply(x, p['final_layer_norm.weight'], p['final_layer_norm.bias'])
    return x @ p['embed_in.weight'].t()


def test_gradients_are_those_of_the_rounded_model() -> None:
    _, model = models()
    tokens = torch.randint(0, 97, (3, 20))
    weight = torch.randn(3, 20, 97)
    out = model(tokens)
    (out * weight).sum().backward()
    p = {
        n: q.detach().double().requires_grad_()
        for n, q in model.named_parameters()
    }
    want = forward64(p, tokens, SIZES)
    (want * weight.double()).sum().backward()
    off = (out - want).detach().norm() / want.detach().norm()
    assert float(off) < 1e-5
    for n, q in model.named_parameters():
        # A value that float32 rounds to the other side of a code's border
        # moves by a step, 1/64 of its block's largest: one in some 1e4
        # values (1e-6 relative error, 127 borders), so 1/64 / sqrt(1e4) of
        # the gradient at most, a few times over for the layers above.
        off = float((q.grad - p[n].grad).norm() / p[n].grad.norm())
        assert off < 1e-3, (n, off)


def test_gradients_are_near_the_exact_model() -> None:
    exact, eight = models()
    tokens = torch.randint(0, 97, (3, 20))
    a, b = exact(tokens), eight(tokens)
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
    a.square().mean().backward()
    b.square().mean().backward()
    for (n, p), (_, q) in zip(
        exact.named_parameters(), eight.named_parameters(),
    ):
        # a kept value is off by 2^e / sqrt(12) in the mean, 2^e at most
        # 1/63.5 of the largest of 64, itself about 2.5 times the mean
        # value: 1.2 %, from each of the up to 8 tensors behind a gradient
        off = float((p.grad - q.grad).norm() / p.grad.norm())
        assert off < 0.012 * math.sqrt(8), (n, off)


def test_state_dicts_are_the_same() -> None:
    exact, eight = models()
    assert exact.state_dict().keys() == eight.state_dict().keys()
    with pytest.raises(ValueError):
        GPTNeoXModel(**SIZES, activation_bits=4)


def test_no_grad_matches() -> None:
    exact, eight = models()
    tokens = torch.randint(0, 97, (2, 5))
    with torch.no_grad():
        torch.testing.assert_close(
            exact(tokens), eight(tokens), rtol=1e-4, atol=1e-4,
        )


def test_autocast() -> None:
    exact, eight = models()
    tokens = torch.randint(0, 97, (2, 20))
    grads = []
    for m in (exact, eight):
        with torch.autocast('cpu', dtype=torch.bfloat16):
            out = m(tokens)
        out.float().square().mean().backward()
        grads.append({n: p.grad for n, p in m.named_parameters()})
    for n, g in grads[0].items():
        assert grads[1][n].dtype == g.dtype
        # bf16 steps of 2^-8 in both, besides the 8 bits
        off = float((g - grads[1][n]).norm() / g.norm())
        assert off < 0.06, (n, off)


def test_kfac_trains_it() -> None:
    _, model = models()
    precon = kfac_amd.KFACPreconditioner(
        model, skip_layers=KFAC_SKIP_LAYERS, lr=0.1,
    )
    names = {name for name, _ in precon._layers.values()}
    assert names == {
        f'layers.{i}.mlp.{n}'
        for i in range(2)
        for n in ('dense_h_to_4h', 'dense_4h_to_h')
    }
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    tokens = torch.randint(0, 97, (3, 20))
    for _ in range(2):
        opt.zero_grad()
        logits = model(tokens[:, :-1])
        F.cross_entropy(
            logits.reshape(-1, 97), tokens[:, 1:].reshape(-1),
        ).backward()
        precon.step()
        for n, p in model.named_parameters():
            assert p.grad.isfinite().all(), n
        opt.step()


def test_kfac_factors_see_the_exact_input() -> None:
    exact, eight = models()
    tokens = torch.randint(0, 97, (3, 20))
    factors = []
    for m in (exact, eight):
        precon = kfac_amd.KFACPreconditioner(m, skip_layers=KFAC_SKIP_LAYERS)
        m(tokens).square().mean().backward()
        factors.append(
            {n: layer.a_factor for n, layer in precon._layers.values()},
        )
    for n, a in factors[0].items():
        torch.testing.assert_close(a, factors[1][n], rtol=1e-4, atol=1e-5)


class Residual(torch.nn.Module):
    """A block whose output's gradient goes to its linear and past it."""

    def __init__(self) -> None:
        super().__init__()
        self.norm = LayerNorm8(64)
        self.lin = Linear8(64, 64)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        self.stream = x * 1
        return self.stream + self.lin(self.norm(self.stream).y)


def test_output_gradient_stays_until_the_step() -> None:
    # A covariance may read a linear's output gradient long after the hook:
    # what the layer holds of it must keep autograd from adding the norm's
    # gradient into the same tensor, which it does where it has the only
    # reference.
    model = Residual()
    precon = kfac_amd.KFACPreconditioner(model)
    ((_, layer),) = precon._layers.values()
    seen = {}

    def accumulate(g, *args) -> None:
        seen['at'], seen['values'] = g.data_ptr(), g.clone()
        layer._hold_grad(g)

    layer.module.accumulate_g_factor = accumulate
    x = torch.randn(5, 64, requires_grad=True)
    y = model(x)
    model.stream.register_hook(lambda g: seen.update(total=g.data_ptr()))
    (y * torch.randn(5, 64)).sum().backward()
    assert seen['total'] != seen['at']
    (held,) = layer._pending_grads
    assert held.data_ptr() == seen['at'] and held._version == 0
    assert torch.equal(held, seen['values'])
    layer.clear_pending()
    assert not layer._pending_grads


def test_packs_what_is_read(monkeypatch) -> None:
    from kfac_amd.ops import norm

    asked = []
    forward = norm.layer_norm_forward

    def spy(*args, **kwargs):
        asked.append((kwargs['packed_input'], kwargs['packed_output']))
        return forward(*args, **kwargs)

    monkeypatch.setattr(norm, 'layer_norm_forward', spy)
    _, model = models()
    tokens = torch.randint(0, 97, (2, 5))
    model(tokens)
    # two norms a block, whose results linears keep, and the last one
    assert asked == [(True, True)] * 4 + [(True, False)]


def test_keeps_nothing_without_a_gradient(monkeypatch) -> None:
    from kfac_amd.ops import norm

    asked = []
    forward = norm.layer_norm_forward

    def spy(*args, **kwargs):
        asked.append((kwargs['packed_input'], kwargs['packed_output']))
        return forward(*args, **kwargs)

    monkeypatch.setattr(norm, 'layer_norm_forward', spy)
    _, model = models()
    tokens = torch.randint(0, 97, (2, 5))
    model.requires_grad_(False)
    model(tokens)
    with torch.no_grad():
        model.requires_grad_(True)(tokens)
    assert not any(packed_input for packed_input, _ in asked)
    x = torch.randn(3, 8)
    for i in range(4):
        args = [x, torch.randn(8), torch.randn(8), x.clone()]
        args[i].requires_grad_()
        asked.clear()
        norm.layer_norm(*args[:3], residual=args[3], keep8=True)
        assert asked == [(True, False)]
        x = x.detach()


def test_modules_refuse() -> None:
    with pytest.raises(ValueError):
        LayerNorm8((4, 8))
    with pytest.raises(ValueError):
        LayerNorm8(8)(torch.randn(3, 4))
    with pytest.raises(ValueError):
        Linear8(8, 4)(torch.randn(3, 4))


def test_modules_stand_alone() -> None:
    x = torch.randn(5, 70, requires_grad=True)
    norm, lin, act = LayerNorm8(70), Linear8(70, 30), GELU8('tanh')
    n = norm(x)
    assert n.total is x
    y, packed = act(lin(n.y, packed=n.packed_output))
    y.sum().backward()
    assert packed.codes.shape == (5, 30)
    assert x.grad.shape == x.shape and lin.weight.grad.shape == (30, 70)
    plainly = LayerNorm8(70, elementwise_affine=False)
    torch.testing.assert_close(
        plainly(x.detach()).y, F.layer_norm(x.detach(), (70,)),
    )
