"""A latent decoder of the Gaussian table, from the operators of ``ops.latent``.

The reference trains 11 free numbers per Gaussian.  ``LatentDecoder`` gives
each Gaussian a code instead: a row of a shared codebook, mixed along the
table's order by a gated recurrence both ways, and mapped to 11 numbers by one
weight per tree level.  A split appends its children in their parents' order,
first all of one side, then all of the other, so the recurrence mixes each
generation in the order of the one before; siblings lie far apart.
Its output is added to a base table, so a decoder at its initial weights
leaves the base as it is.  ``blocks`` of attention with a decay for each head mix
the table further, half of the heads along its order and half against it, with
the Gaussians' means as positions.  No reference counterpart.

One training step, with the trainer's explicit backward in the middle::

    raw = decoder(codes, rows, offsets)                  # [N, 11]
    means, quats, scales, opacities = decoder.leaves(base, raw)
    state = explicit.prepare_explicit_gaussians(quats, scales, opacities, ...)
    image = explicit.explicit_rasterize(state, means, ...).image
    loss(image).backward()
    explicit.explicit_backward(state, means, quats, scales, opacities)
    decoder.backward(raw, means, quats, scales, opacities)
    optimizer.step()                       # r2splat.optim.Adam, or AdamW for 16 bits

``rows, offsets = ops.latent.group_rows(level, n_levels)`` stay as they are
until a densification changes the table.  A decoder with blocks is called with the
base's means besides: ``decoder(codes, rows, offsets, base.means)``.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from .ops import latent
from .scenes import RawGaussians

__all__ = ["LatentDecoder", "MixingBlock"]

_WIDTHS = (3, 4, 3, 1)  # means, quats, raw scales, raw opacities


def _normal(*shape, scale, generator, dtype):
    return torch.nn.Parameter((torch.randn(*shape, generator=generator) * scale).to(dtype))


class MixingBlock(torch.nn.Module):
    """One block of a decoder: normalised tokens [N, width] and their positions
    [N, 3] -> (update, gate), both [N, width], for ``ops.latent.residual_norm``.

    Of ``heads`` heads (an even number) the first half attends to the tokens
    before each, the others to those behind; their memories reach from 32 to 4096
    tokens.  Queries and keys are turned by the positions, a third of a head's
    pairs for each axis."""

    def __init__(self, width: int, heads: int = 4, generator: Optional[torch.Generator] = None,
                 dtype=torch.float32):
        super().__init__()
        if heads < 2 or heads % 2 or width % heads or width // heads < 6:
            raise ValueError(f"{width} channels do not make {heads} heads: an even number of "
                             "heads, of 6 channels or more")
        self.heads = heads
        pairs = width // heads // 2
        self.sections = tuple(pairs // 3 + (axis < pairs % 3) for axis in range(3))
        new = lambda *shape: _normal(*shape, scale=shape[1] ** -0.5,  # noqa: E731
                                     generator=generator, dtype=dtype)
        self.inward = new(4 * width, width)  # queries, keys, values, gates
        self.outward = new(width, width)
        self.post = torch.nn.Parameter(torch.ones(width, dtype=dtype))
        reach = torch.linspace(5.0, 12.0, heads // 2, dtype=torch.float32).repeat(2)
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-reach)), persistent=False)

    def _apply(self, fn, *args, **kwargs):
        """Decays are float32 whatever the module is cast to: in eight bits a memory
        of 4096 tokens would be one of another length, and the operator takes no other."""
        decays = self.log_decay
        super()._apply(fn, *args, **kwargs)
        if self.log_decay.dtype != decays.dtype:
            self.log_decay = decays.to(self.log_decay.device)
        return self

    def forward(self, u: Tensor, positions: Tensor) -> Tuple[Tensor, Tensor]:
        n, width = u.shape
        q, k, v, gate = torch.nn.functional.linear(u, self.inward).split(width, dim=1)
        q, k, v = (t.reshape(n, self.heads, width // self.heads) for t in (q, k, v))
        q, k = latent.rotary_axes(q, k, positions, self.sections)
        half = self.heads // 2
        mixed = [latent.decay_attention(*(t[None, :, part] for t in (q, k, v)),
                                        self.log_decay[part], reverse=back)[0][0]
                 for part, back in ((slice(0, half), False), (slice(half, None), True))]
        update = torch.nn.functional.linear(torch.cat(mixed, 1).reshape(n, width), self.outward)
        return update, gate


class LatentDecoder(torch.nn.Module):
    """Codes and tree levels of N Gaussians -> [N, 11] raw parameters.

    n_codes rows of ``width`` channels in the codebook and as many in the
    gates' table, n_levels weights of 11 x width and as many biases; ``blocks``
    MixingBlocks of ``heads`` heads between them, which see the means times
    ``position_scale``."""

    def __init__(self, n_codes: int, n_levels: int, width: int = 64,
                 generator: Optional[torch.Generator] = None, dtype=torch.float32,
                 blocks: int = 0, heads: int = 4, position_scale: float = 64.0):
        super().__init__()
        normal = lambda *shape, scale: _normal(*shape, scale=scale,  # noqa: E731
                                               generator=generator, dtype=dtype)

        # Codes are stored at 1 / sqrt(width) and scaled back by the lookup, so
        # that one learning rate serves tables of any width.
        self.scale = math.sqrt(width)
        self.codebook = normal(n_codes, width, scale=1.0 / self.scale)
        self.gates = normal(n_codes, width, scale=1.0 / self.scale)
        self.weight = torch.nn.Parameter(torch.zeros(n_levels, sum(_WIDTHS), width, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(n_levels, sum(_WIDTHS), dtype=dtype))
        self.position_scale = position_scale
        self.blocks = torch.nn.ModuleList(MixingBlock(width, heads, generator, dtype)
                                          for _ in range(blocks))
        # The norm before each block.
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width, dtype=dtype))
                                            for _ in range(blocks))

    def forward(self, codes: Tensor, rows: Tensor, offsets: Tensor,
                means: Optional[Tensor] = None) -> Tensor:
        """[N, 11] of codes [N] (one outside the codebook: no code), the Gaussians'
        grouping by level and, for a decoder with blocks, their means [N, 3]."""
        x = latent.embedding_lookup(self.codebook, codes, self.scale)
        gate = latent.embedding_lookup(self.gates, codes, self.scale)
        down, _ = latent.gated_scan(x[None], gate[None])
        up, _ = latent.gated_scan(x[None], gate[None], reverse=True)
        x = x + down[0] + up[0]
        if self.blocks:
            x = self._mix(x, means)
        return latent.grouped_matmul(x, self.weight, offsets, rows=rows, bias=self.bias)

    def _mix(self, x: Tensor, means: Optional[Tensor]) -> Tensor:
        if means is None:
            raise RuntimeError("a decoder with blocks needs the means")
        positions = means.detach().float() * self.position_scale
        # The blocks' updates together are as large as one's.
        scale = 1.0 / math.sqrt(len(self.blocks))
        u = latent.pre_norm(x, self.norms[0])
        for block, following in zip(self.blocks, [*self.norms[1:], None]):
            update, gate = block(u, positions)
            x, u = latent.residual_norm(x, update, gate, block.post, following, scale=scale)
        return x

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
