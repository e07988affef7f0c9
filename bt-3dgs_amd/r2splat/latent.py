"""A latent decoder of the Gaussian table, from the operators of ``ops.latent``.

The reference trains 11 free numbers per Gaussian.  ``LatentDecoder`` gives
each Gaussian a code instead: a row of a shared codebook, mixed along the
table's order by a gated recurrence both ways, and mapped to 11 numbers by one
weight per tree level.  A split appends its children in their parents' order,
first all of one side, then all of the other, so the recurrence mixes each
generation in the order of the one before; siblings lie far apart.
Its output is added to a base table, so a decoder at its initial weights
leaves the base as it is.  No reference counterpart.

One training step, with the trainer's explicit backward in the middle::

    raw = decoder(codes, rows, offsets)                  # [N, 11]
    means, quats, scales, opacities = decoder.leaves(base, raw)
    state = explicit.prepare_explicit_gaussians(quats, scales, opacities, ...)
    image = explicit.explicit_rasterize(state, means, ...).image
    loss(image).backward()
    explicit.explicit_backward(state, means, quats, scales, opacities)
    decoder.backward(raw, means, quats, scales, opacities)
    optimizer.step()                                     # r2splat.optim.Adam

``rows, offsets = ops.latent.group_rows(level, n_levels)`` stay as they are
until a densification changes the table.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from .ops import latent
from .scenes import RawGaussians

__all__ = ["LatentDecoder"]

_WIDTHS = (3, 4, 3, 1)  # means, quats, raw scales, raw opacities


class LatentDecoder(torch.nn.Module):
    """Codes and tree levels of N Gaussians -> [N, 11] raw parameters.

    n_codes rows of ``width`` channels in the codebook and as many in the
    gates' table, n_levels weights of 11 x width and as many biases."""

    def __init__(self, n_codes: int, n_levels: int, width: int = 64,
                 generator: Optional[torch.Generator] = None, dtype=torch.float32):
        super().__init__()

        def normal(*shape, scale):
            return torch.nn.Parameter(
                (torch.randn(*shape, generator=generator) * scale).to(dtype))

        # Codes are stored at 1 / sqrt(width) and scaled back by the lookup, so
        # that one learning rate serves tables of any width.
        self.scale = math.sqrt(width)
        self.codebook = normal(n_codes, width, scale=1.0 / self.scale)
        self.gates = normal(n_codes, width, scale=1.0 / self.scale)
        self.weight = torch.nn.Parameter(torch.zeros(n_levels, sum(_WIDTHS), width, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(n_levels, sum(_WIDTHS), dtype=dtype))

    def forward(self, codes: Tensor, rows: Tensor, offsets: Tensor) -> Tensor:
        """[N, 11] of codes [N] (one outside the codebook: no code) and the
        Gaussians' grouping by level."""
        x = latent.embedding_lookup(self.codebook, codes, self.scale)
        gate = latent.embedding_lookup(self.gates, codes, self.scale)
        down, _ = latent.gated_scan(x[None], gate[None])
        up, _ = latent.gated_scan(x[None], gate[None], reverse=True)
        return latent.grouped_matmul(x + down[0] + up[0], self.weight, offsets, rows=rows,
                                     bias=self.bias)

    @staticmethod
    def leaves(base: RawGaussians, raw: Tensor) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
        """base + raw as (means, quats, raw scales, raw opacities): float32
        leaves that the explicit backward stores its gradients in."""
        parts = [p.detach().float() for p in raw.split(_WIDTHS, dim=1)]
        table = (base.means, base.quats, base.raw_scales, base.raw_opacities)
        return tuple((t + p.reshape(t.shape)).contiguous().requires_grad_(True)
                     for t, p in zip(table, parts))

    @staticmethod
    def backward(raw: Tensor, *leaves: Tensor) -> None:
        """The leaves' gradients on to the decoder's parameters."""
        raw.backward(torch.cat([t.grad.reshape(raw.shape[0], -1) for t in leaves],
                               dim=1).to(raw.dtype))
