"""What the operators of a transformer block's training path are measured on.

Four operators: layer norm (``norm``), the 8 bit form of an activation
(``pack``), GELU whose input is kept in 8 bits (``gelu``) and a linear
layer's weight and bias gradient from an input kept in 8 bits (``wgrad``).

``own`` false computes the plain form: elementary torch operations in 32
bits, rounded once at the end. ``own`` true makes the calls that a program
makes of ``kfac_amd.ops``.
"""

from __future__ import annotations

import math
import random
from typing import Any

import torch

own = False

BLOCK = 64  # values of a row that share one power of two
EPS = 1e-5
TYPES = {
    'f32': torch.float32,
    'bf16': torch.bfloat16,
    'f16': torch.float16,
}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}
PACKED = 1.0 + 1.0 / BLOCK  # bytes that a value takes in 8 bit form


def listed() -> list[dict[str, Any]]:
    return [
        # one token of a small LM (width 256): a forward pass alone, where
        # nothing but the call's latency counts
        dict(name='norm_token', op='norm', rows=1, cols=256, x='f32',
             y='f32', residual=False, keep8=False, out8=False, train=False),
        # the LM example's batch (64 x 20 tokens, width 256) in fp32
        dict(name='norm_lm', op='norm', rows=1280, cols=256, x='f32',
             y='f32', residual=True, keep8=False, out8=False, train=True),
        # the 125M decoder's block (8 x 2048 tokens, width 768) under bf16
        # autocast: fp32 residual stream, the sum with a branch, bf16 out,
        # everything kept in 8 bits
        dict(name='norm_decoder8', op='norm', rows=16384, cols=768, x='f32',
             y='bf16', residual=True, keep8=True, out8=True, train=True),
        # a ragged batch of an odd width in fp16
        dict(name='norm_odd', op='norm', rows=4099, cols=1001, x='f16',
             y='f16', residual=False, keep8=False, out8=False, train=True),
        # a wide model in pure bf16
        dict(name='norm_wide', op='norm', rows=16384, cols=8192, x='bf16',
             y='bf16', residual=False, keep8=False, out8=False, train=True),
        # one sequence of the LM example, to 8 bits and back
        dict(name='pack_lm', op='pack', rows=64, cols=256, x='f32'),
        # the 125M decoder's qkv output
        dict(name='pack_decoder', op='pack', rows=16384, cols=2304,
             x='bf16'),
        # the LM example's hidden layer
        dict(name='gelu_lm', op='gelu', rows=1280, cols=256, x='f32',
             tanh=False, out8=False),
        # a hidden layer of 4 x 1024 under bf16 autocast, its output
        # packed for the second linear's gradient
        dict(name='gelu_hidden', op='gelu', rows=16384, cols=4096, x='bf16',
             tanh=False, out8=True),
        # the LM example's hidden layer in fp32
        dict(name='wgrad_lm', op='wgrad', rows=1280, inputs=256,
             outputs=256, g='f32'),
        # the 125M decoder's qkv projection
        dict(name='wgrad_qkv', op='wgrad', rows=16384, inputs=768,
             outputs=2304, g='bf16'),
        # a wide square projection
        dict(name='wgrad_wide', op='wgrad', rows=16384, inputs=8192,
             outputs=4096, g='bf16'),
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    """An integer spread over the logarithm of [low, high]."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(high, max(low, v))


def draw(rng: random.Random) -> dict[str, Any]:
    op = rng.choice(['norm', 'norm', 'pack', 'gelu', 'wgrad', 'wgrad'])
    rows = _log(rng, 1, 16384)
    if op == 'wgrad':
        inputs, outputs = _log(rng, 8, 6144), _log(rng, 8, 4096)
        if rng.random() < 0.5:
            inputs, outputs = -(-inputs // 64) * 64, -(-outputs // 64) * 64
        return dict(op=op, rows=rows, inputs=inputs, outputs=outputs,
                    g=rng.choice(['bf16', 'bf16', 'f16', 'f32']))
    # half the values of the widest listed case, at most
    cols = _log(rng, 8, min(8192, 2 ** 26 // rows))
    if rng.random() < 0.5:
        cols = -(-cols // 64) * 64
    x = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'pack':
        return dict(op=op, rows=rows, cols=cols, x=x)
    if op == 'gelu':
        return dict(op=op, rows=rows, cols=cols, x=x,
                    tanh=rng.random() < 0.5,
                    out8=x != 'f32' and rng.random() < 0.5)
    y = rng.choice(['f32', 'bf16']) if x == 'f32' else x
    keep8 = rng.random() < 0.5
    return dict(op=op, rows=rows, cols=cols, x=x, y=y,
                residual=rng.random() < 0.5, keep8=keep8,
                out8=y != 'f32' and rng.random() < 0.5,
                train=keep8 or rng.random() < 0.7)


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, device='cuda', generator=gen)

    rows = case['rows']
    state: dict[str, Any] = dict(case)
    if case['op'] == 'wgrad':
        # activations in 8 bits; a loss's gradients, a row in sixteen
        # without any (padding)
        x = normal(rows, case['inputs'])
        state['codes'], state['exponents'] = _pack(x.bfloat16().float())
        live = torch.rand(rows, 1, device='cuda', generator=gen) > 1 / 16
        g = normal(rows, case['outputs']) * live * 1e-3
        state['g'] = g.to(TYPES[case['g']])
        return state
    cols, t = case['cols'], TYPES[case['x']]
    # channels of different spread, a few of them far out
    spread = torch.exp(0.5 * normal(cols))
    state['x'] = (normal(rows, cols) * spread + 0.1 * normal(cols)).to(t)
    if case['op'] == 'gelu':
        state['dy'] = (1e-2 * normal(rows, cols)).to(t)
    if case['op'] == 'norm':
        state['weight'] = 1 + 0.1 * normal(cols)
        state['bias'] = 0.1 * normal(cols)
        if case['residual']:
            state['r'] = (0.3 * normal(rows, cols)).to(TYPES[case['y']])
        if case['train']:
            state['dy'] = (1e-2 * normal(rows, cols)).to(TYPES[case['y']])
            if case['residual']:
                # what flows past the norm along the residual stream
                state['dt'] = (1e-2 * normal(rows, cols)).to(t)
    return state


# -- the plain form --------------------------------------------------------


def _pack(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, exponents + 127) of the rows of a finite fp32 matrix."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    padded = torch.zeros(rows, blocks * BLOCK, device=x.device)
    padded[:, :cols] = x
    padded = padded.view(rows, blocks, BLOCK)
    part, power = torch.frexp(padded.abs().amax(-1))  # part in [0.5, 1)
    e = power - 7 + (part > 127 / 128).int()
    e = torch.clamp(torch.where(part > 0, e, -126), -126, 121)
    scale = torch.exp2(-e.double()).float()
    codes = torch.clamp(torch.round(padded * scale[..., None]), -127, 127)
    codes = codes.view(rows, -1)[:, :cols].to(torch.int8).contiguous()
    return codes, (e + 127).to(torch.uint8)


def _unpack(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    rows, cols = codes.shape
    scale = torch.exp2(exponents.double() - 127).float()
    scale = scale.repeat_interleave(BLOCK, dim=1)[:, :cols]
    return codes.float() * scale


def _plain_norm(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    xt, yt = s['x'].dtype, TYPES[s['y']]
    t = s['x'].float()
    if s['residual']:
        t = (t + s['r'].float()).to(xt).float()
    mean = t.mean(-1, keepdim=True)
    rstd = ((t - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = ((t - mean) * rstd * s['weight'] + s['bias']).to(yt)
    out = {'y': y}
    if s['out8']:
        out['y8'] = _unpack(*_pack(y.float())).to(yt)
    if s['residual']:
        out['total'] = t.to(xt)
    if s['train']:
        if s['keep8']:
            t = _unpack(*_pack(t))
        h = (t - mean) * rstd
        dy = s['dy'].float()
        q = dy * s['weight']
        dx = rstd * (
            q
            - q.mean(-1, keepdim=True)
            - h * (q * h).mean(-1, keepdim=True)
        )
        if s['residual']:
            dx = dx + s['dt'].float()
        out['dx'] = dx.to(xt)
        out['dweight'] = (dy * h).sum(0)
        out['dbias'] = dy.sum(0)
    return out


def _plain_gelu(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    x, t = s['x'].float(), s['x'].dtype

    def cdf(v: torch.Tensor) -> torch.Tensor:
        # erfc holds the small values of the left tail
        return 0.5 * torch.erfc(-v * math.sqrt(0.5))

    x8 = _unpack(*_pack(x))
    if s['tanh']:
        c = math.sqrt(2 / math.pi)

        # 0.5 * (1 + tanh(u)) written as a sigmoid of 2u
        def gate(v: torch.Tensor) -> torch.Tensor:
            return 1 / (1 + torch.exp(-2 * c * (v + 0.044715 * v * v * v)))

        y = x * gate(x)
        p = gate(x8)
        slope = 2 * c * (1 + 3 * 0.044715 * x8 * x8)
        d = p + x8 * p * (1 - p) * slope
    else:
        y = x * cdf(x)
        d = cdf(x8) + x8 * torch.exp(-0.5 * x8 * x8) / math.sqrt(2 * math.pi)
    y = y.to(t)
    out = {'y': y, 'dx': (s['dy'].float() * d).to(t)}
    if s['out8']:
        out['y8'] = _unpack(*_pack(y.float())).to(t)
    return out


def run(state: dict[str, Any]) -> dict[str, torch.Tensor]:
    op = state['op']
    if own:
        return _own(state)
    if op == 'norm':
        return _plain_norm(state)
    if op == 'gelu':
        return _plain_gelu(state)
    if op == 'pack':
        x = state['x']
        return {'x8': _unpack(*_pack(x.float())).to(x.dtype)}
    g = state['g'].float()
    values = _unpack(state['codes'], state['exponents'])
    return {'dweight': g.t() @ values, 'dbias': g.sum(0)}


def _own(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    from kfac_amd import ops

    if s['op'] == 'pack':
        x = s['x']
        return {'x8': ops.unpack8(ops.pack8(x), x.dtype)}
    if s['op'] == 'wgrad':
        dw, db = ops.weight_grad8(
            s['g'], ops.Packed8(s['codes'], s['exponents']),
        )
        return {'dweight': dw, 'dbias': db}
    if s['op'] == 'gelu':
        f = ops.gelu8_forward(
            s['x'],
            approximate='tanh' if s['tanh'] else 'none',
            packed_output=s['out8'],
        )
        dx = ops.gelu8_backward(
            s['dy'],
            f.packed_input,
            approximate='tanh' if s['tanh'] else 'none',
        )
        out = {'y': f.y, 'dx': dx}
        if s['out8']:
            out['y8'] = ops.unpack8(f.packed_output, f.y.dtype)
        return out
    n = ops.layer_norm_forward(
        s['x'],
        s['weight'],
        s['bias'],
        EPS,
        residual=s['r'] if s['residual'] else None,
        out_dtype=TYPES[s['y']],
        packed_input=s['keep8'],
        packed_output=s['out8'],
    )
    out = {'y': n.y}
    if s['out8']:
        out['y8'] = ops.unpack8(n.packed_output, n.y.dtype)
    if s['residual']:
        out['total'] = n.total
    if s['train']:
        out['dx'], out['dweight'], out['dbias'] = ops.layer_norm_backward(
            s['dy'],
            n.packed_input if s['keep8'] else n.total,
            n.mean,
            n.rstd,
            s['weight'],
            grad_total=s['dt'] if s['residual'] else None,
            dtype=s['x'].dtype,
        )
    return out


# -- the definition, in 64 bits --------------------------------------------


def _through8(x: torch.Tensor) -> torch.Tensor:
    """The values that a finite matrix has after a pass through 8 bits."""
    out = []
    for part in x.double().split(BLOCK, dim=1):
        top = part.abs().max(dim=1, keepdim=True).values
        step = torch.exp2(torch.ceil(torch.log2(top / 127)).clamp(-126, 121))
        out.append((part / step).round().clamp(-127, 127) * step)
    return torch.cat(out, dim=1)


def exact(case: dict[str, Any], seed: int) -> dict[str, torch.Tensor]:
    s = prepare(case, seed)
    if case['op'] == 'pack':
        return {'x8': _through8(s['x'])}
    if case['op'] == 'wgrad':
        power = torch.exp2(s['exponents'].double() - 127)
        a = s['codes'].double()
        for k in range(power.shape[1]):
            a[:, k * BLOCK:(k + 1) * BLOCK] *= power[:, k:k + 1]
        g = s['g'].double()
        return {'dweight': torch.mm(g.t(), a), 'dbias': torch.sum(g, 0)}
    x = s['x'].double()
    if case['op'] == 'gelu':
        x8, dy = _through8(x), s['dy'].double()
        if case['tanh']:
            def f(v: torch.Tensor) -> torch.Tensor:
                return math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)

            y = x / 2 * (1 + torch.tanh(f(x)))
            th = torch.tanh(f(x8))
            inner = math.sqrt(2 / math.pi) * (1 + 0.134145 * x8 ** 2)
            d = (1 + th) / 2 + x8 / 2 * (1 - th ** 2) * inner
        else:
            y = x / 2 * torch.special.erfc(-x / math.sqrt(2))
            density = torch.exp(-x8 ** 2 / 2) / math.sqrt(2 * math.pi)
            d = torch.special.erfc(-x8 / math.sqrt(2)) / 2 + x8 * density
        out = {'y': y, 'dx': dy * d}
        if case['out8']:
            out['y8'] = _through8(y.to(TYPES[case['x']]))
        return out
    if case['residual']:
        x = (x + s['r'].double()).to(TYPES[case['x']]).double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sigma = torch.sqrt(var + EPS)
    w = s['weight'].double()
    y = torch.addcmul(s['bias'].double(), (x - mean) / sigma, w)
    out = {'y': y}
    if case['out8']:
        out['y8'] = _through8(y.to(TYPES[case['y']]))
    if case['residual']:
        out['total'] = x
    if case['train']:
        h = ((_through8(x) if case['keep8'] else x) - mean) / sigma
        dy, n = s['dy'].double(), case['cols']
        q = dy * w
        inner = torch.sum(q * h, dim=1, keepdim=True)
        dx = (n * q - torch.sum(q, dim=1, keepdim=True) - h * inner)
        dx = dx / (n * sigma)
        if case['residual']:
            dx = dx + s['dt'].double()
        out['dx'] = dx
        out['dweight'] = torch.sum(dy * h, 0)
        out['dbias'] = torch.sum(dy, 0)
    return out


def work(case: dict[str, Any]) -> dict[str, float]:
    rows = case['rows']
    if case['op'] == 'wgrad':
        k, n = case['inputs'], case['outputs']
        read = rows * (n * SIZE[case['g']] + k * PACKED)
        return {'bytes': read + 4 * n * (k + 1), 'flops': 2 * rows * n * k}
    size = rows * case['cols']
    sx = SIZE[case['x']]
    if case['op'] == 'pack':
        return {'bytes': size * 2 * sx, 'flops': 4 * size}
    if case['op'] == 'gelu':
        each = 4 * sx + (sx if case['out8'] else 0)
        return {'bytes': size * each, 'flops': 30 * size}
    sy = SIZE[case['y']]
    each = sx + sy + (sy if case['out8'] else 0)
    if case['residual']:
        each += sy + sx
    flops = 8
    if case['train']:
        each += sy + sx + (sx if case['residual'] else 0)
        flops += 12
    params = 8 * case['cols'] * (2 if case['train'] else 1)
    return {'bytes': size * each + params, 'flops': flops * size}
