"""GPT-NeoX-style decoder LM (125M default) for the LM benchmark.

Matches the BASELINE.json config "GPT-NeoX 125M (kfac/gpt_neox
Linear-only layers) synthetic seq=2048": K-FAC preconditions the MLP
linears (named mlp.dense_h_to_4h / mlp.dense_4h_to_h like GPT-NeoX);
attention, embeddings and the LM head are skip-listed by the caller.
Attention uses torch's fused scaled_dot_product_attention.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from kfac_amd.models.modules import GELU8
from kfac_amd.models.modules import LayerNorm8
from kfac_amd.models.modules import Linear8
from kfac_amd.ops import Packed8


class MLP(nn.Module):
    def __init__(self, d: int, ffn: int):
        super().__init__()
        self.dense_h_to_4h = nn.Linear(d, ffn)
        self.dense_4h_to_h = nn.Linear(ffn, d)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.dense_4h_to_h(F.gelu(self.dense_h_to_4h(x)))


class Attention(nn.Module):
    linear: type[nn.Linear] = nn.Linear

    def __init__(self, d: int, n_heads: int):
        super().__init__()
        self.n_heads = n_heads
        self.query_key_value = self.linear(d, 3 * d)
        self.dense = self.linear(d, d)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.dense(self.attend(self.query_key_value(x)))

    def attend(self, qkv: torch.Tensor) -> torch.Tensor:
        b, s, d3 = qkv.shape
        d = d3 // 3
        q, k, v = qkv.chunk(3, dim=-1)
        hd = d // self.n_heads

        def heads(t: torch.Tensor) -> torch.Tensor:
            return t.view(b, s, self.n_heads, hd).transpose(1, 2)

        out = F.scaled_dot_product_attention(
            heads(q), heads(k), heads(v), is_causal=True,
        )
        return out.transpose(1, 2).reshape(b, s, d)


class Block(nn.Module):
    def __init__(self, d: int, n_heads: int, ffn: int):
        super().__init__()
        self.input_layernorm = nn.LayerNorm(d)
        self.attention = Attention(d, n_heads)
        self.post_attention_layernorm = nn.LayerNorm(d)
        self.mlp = MLP(d, ffn)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x + self.attention(self.input_layernorm(x))
        return x + self.mlp(self.post_attention_layernorm(x))


class MLP8(nn.Module):
    """:class:`MLP` with its activations kept in 8 bits."""

    def __init__(self, d: int, ffn: int):
        super().__init__()
        self.dense_h_to_4h = Linear8(d, ffn)
        self.gelu = GELU8()
        self.dense_4h_to_h = Linear8(ffn, d)

    def forward(
        self,
        x: torch.Tensor,
        packed: Packed8 | None,
    ) -> torch.Tensor:
        h, packed = self.gelu(self.dense_h_to_4h(x, packed=packed))
        return self.dense_4h_to_h(h, packed=packed)


class Attention8(Attention):
    """:class:`Attention` whose projections keep their input in 8 bits."""

    linear = Linear8

    def forward(  # type: ignore[override]
        self,
        x: torch.Tensor,
        packed: Packed8 | None,
    ) -> torch.Tensor:
        return self.dense(
            self.attend(self.query_key_value(x, packed=packed)),
        )


class Block8(nn.Module):
    """:class:`Block` with its activations kept in 8 bits.

    A branch's result joins the residual stream in the next norm, so a block
    takes the stream and the last branch, and returns the same.
    """

    def __init__(self, d: int, n_heads: int, ffn: int):
        super().__init__()
        self.input_layernorm = LayerNorm8(d)
        self.attention = Attention8(d, n_heads)
        self.post_attention_layernorm = LayerNorm8(d)
        self.mlp = MLP8(d, ffn)

    def forward(
        self,
        x: torch.Tensor,
        branch: torch.Tensor | None,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        y, x, packed = self.input_layernorm(x, branch)
        branch = self.attention(y, packed)
        y, x, packed = self.post_attention_layernorm(x, branch)
        return x, self.mlp(y, packed)


class GPTNeoXModel(nn.Module):
    """Decoder-only LM; (batch, seq) int tokens -> (batch, seq, vocab).

    ``activation_bits=8`` keeps the activations of norms, linears and GELU in
    8 bits for the backward pass. Parameters and their names are the same.
    """

    def __init__(
        self,
        vocab: int = 50304,
        d: int = 768,
        n_layers: int = 12,
        n_heads: int = 12,
        ffn: int = 3072,
        max_seq: int = 2048,
        activation_bits: int | None = None,
    ):
        super().__init__()
        if activation_bits not in (None, 8):
            raise ValueError(
                f'activation_bits must be None or 8, got {activation_bits}',
            )
        self.activation_bits = activation_bits
        block = Block if activation_bits is None else Block8
        self.embed_in = nn.Embedding(vocab, d)
        self.embed_pos = nn.Embedding(max_seq, d)
        self.layers = nn.ModuleList(
            block(d, n_heads, ffn) for _ in range(n_layers)
        )
        if activation_bits is None:
            self.final_layer_norm = nn.LayerNorm(d)
        else:
            # embed_out keeps its input as it is
            self.final_layer_norm = LayerNorm8(d, packed_output=False)
        self.embed_out = nn.Linear(d, vocab, bias=False)
        # weight tying -> 125.3M parameters total at the default config
        self.embed_out.weight = self.embed_in.weight

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        b, s = tokens.shape
        pos = torch.arange(s, device=tokens.device)
        x = self.embed_in(tokens) + self.embed_pos(pos)[None]
        if self.activation_bits is not None:
            branch = None
            for layer in self.layers:
                x, branch = layer(x, branch)
            return self.embed_out(self.final_layer_norm(x, branch).y)
        for layer in self.layers:
            x = layer(x)
        return self.embed_out(self.final_layer_norm(x))


def gptneox_125m(
    vocab: int = 50304,
    activation_bits: int | None = None,
) -> GPTNeoXModel:
    """~125M-parameter configuration."""
    return GPTNeoXModel(
        vocab=vocab,
        d=768,
        n_layers=12,
        n_heads=12,
        ffn=3072,
        activation_bits=activation_bits,
    )


# skip-list for K-FAC: precondition MLP linears only (reference LM
# example skips embedding/decoder/attention, torch_language_model.py:162-167)
KFAC_SKIP_LAYERS = ['.*attention.*', 'embed.*', '.*embed_out.*']
