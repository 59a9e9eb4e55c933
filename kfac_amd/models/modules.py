"""Modules of a transformer block that keep their activations in 8 bits.

Subclasses of torch's, with the same parameters and state dict keys
(checkpoints load either way), built on the operators of kfac_amd.ops.
Linear8 stands in for a linear layer as it is. LayerNorm8 and GELU8 return
tuples: besides the result the 8 bit form of it, which the next linear layer
then does not have to make, and LayerNorm8 the sum that it took the norm of.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from kfac_amd import ops
from kfac_amd.ops import NormOutput
from kfac_amd.ops import Packed8


class LayerNorm8(nn.LayerNorm):
    """Layer norm of ``x + residual`` over the last dimension.

    Keeps the sum in 8 bits for the backward pass. Under autocast the result
    has autocast's type, which the next linear layer computes in.
    ``packed_output=False`` leaves out the result's 8 bit form, for a norm
    that no :class:`Linear8` follows.
    """

    def __init__(
        self,
        normalized_shape: int,
        eps: float = 1e-5,
        elementwise_affine: bool = True,
        bias: bool = True,
        packed_output: bool = True,
    ):
        super().__init__(normalized_shape, eps, elementwise_affine, bias)
        if len(self.normalized_shape) != 1:
            raise ValueError('LayerNorm8 takes the last dimension only')
        self.packed_output = packed_output

    def forward(  # type: ignore[override]
        self,
        x: torch.Tensor,
        residual: torch.Tensor | None = None,
    ) -> NormOutput:
        """(y, total, packed y); see :func:`kfac_amd.ops.layer_norm`."""
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(
                f'rows of {x.shape[-1]} values do not fit a norm of '
                f'{self.normalized_shape[0]}',
            )
        out_dtype = x.dtype
        if torch.is_autocast_enabled(x.device.type):
            out_dtype = torch.get_autocast_dtype(x.device.type)
        return ops.layer_norm(
            x,
            self.weight,
            self.bias,
            self.eps,
            residual=residual,
            out_dtype=out_dtype,
            keep8=True,
            packed_output=self.packed_output and torch.is_grad_enabled(),
        )


class Linear8(nn.Linear):
    """Linear layer that keeps its input in 8 bits.

    The weight's gradient is computed from the 8 bit input. K-FAC registers
    it like any other linear layer; its factors see the exact input.
    """

    # read by KFACBaseLayer: inputs are not held until the step
    keeps_codes = True

    def forward(  # type: ignore[override]
        self,
        x: torch.Tensor,
        packed: Packed8 | None = None,
    ) -> torch.Tensor:
        """``x @ weight.T + bias``; packed: the 8 bit form of x, if made."""
        return ops.linear8(x, self.weight, self.bias, packed=packed)


class GELU8(nn.GELU):
    """GELU that keeps its input in 8 bits and packs its output."""

    def forward(  # type: ignore[override]
        self,
        x: torch.Tensor,
    ) -> tuple[torch.Tensor, Packed8 | None]:
        """(y, packed y)."""
        return ops.gelu8(
            x,
            approximate=self.approximate,
            packed_output=torch.is_grad_enabled(),
        )
