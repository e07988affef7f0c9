"""Operators of a latent decoder: row lookup, gated scan, products per group.

A latent-coded Gaussian model keeps a shared codebook instead of free
parameters for every Gaussian and decodes them: rows looked up by code and
by tree level, mixed along the table's order, and mapped to raw parameters
by one weight per tree level.  These are the differentiable operators such
a decoder is built from (``r2splat.latent`` is one); the reference has none
of them.

* ``embedding_lookup``  rows of a table by id, scaled; the table's gradient
  sums the positions of each id in a fixed order, without atomics;
* ``gated_scan``        h_t = a_t h_{t-1} + (1 - a_t) x_t with
  a_t = sigmoid(gate_t), over equal or ragged sequences of any length, and
  ``gated_scan_step`` for one more token of running sequences;
* ``grouped_matmul``    one weight per group of rows, groups of any size, the
  groups' rows anywhere in the table; ``group_rows`` finds them.

Activations, tables and weights are float32, bfloat16 or float16 CUDA
tensors; sums and states are float32.  Gradients come from HIP kernels; they
are not differentiable again, and forward-mode tangents are refused.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ..cuda import _wrapper as W

__all__ = ["embedding_lookup", "gated_scan", "gated_scan_step", "grouped_matmul", "group_rows"]


def _wants_grad(*tensors) -> bool:
    """Whether the call goes through its autograd function: for a gradient, and
    for a forward-mode tangent, which that function refuses (the kernels would
    drop it)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    # Outside a dual level there is none to look for; looking costs 0.3 us a tensor.
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _index32(t: Optional[Tensor]) -> Optional[Tensor]:
    if t is None:
        return None
    return (t if t.dtype == torch.int32 else t.to(torch.int32)).contiguous()


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.n_rows, ctx.scale = table.shape[0], scale
        return W.embedding_fwd(table, ids, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return W.embedding_bwd(grad, ids, ctx.n_rows, ctx.scale), None, None


def embedding_lookup(table: Tensor, ids: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``: [*ids.shape, D] of a table [V, D].  An id outside
    [0, V) gives a zero row and no gradient (a Gaussian without a code)."""
    if not _wants_grad(table):
        return W.embedding_fwd(table, ids, scale)
    return _Lookup.apply(table, ids, float(scale))


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, offsets, reverse):
        ctx.set_materialize_grads(False)
        y, final, kept = W.gated_scan_fwd(x, gate, initial, offsets, reverse)
        ctx.save_for_backward(x, gate, initial, offsets, kept)
        ctx.reverse = reverse
        return y, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, v_y, v_final):
        x, gate, initial, offsets, kept = ctx.saved_tensors
        if v_y is None:
            v_y = torch.zeros_like(x)
        v_x, v_gate, v_initial = W.gated_scan_bwd(x, gate, initial, offsets, kept, v_y, v_final,
                                                  ctx.reverse)
        return v_x, v_gate, v_initial if ctx.needs_input_grad[2] else None, None, None


def gated_scan(x: Tensor, gate: Tensor, initial: Optional[Tensor] = None,
               offsets: Optional[Tensor] = None, reverse: bool = False) -> Tuple[Tensor, Tensor]:
    """(y, final) of ``h_t = a_t h_{t-1} + (1 - a_t) x_t``, ``a_t = sigmoid(gate_t)``,
    for every channel on its own.

    x, gate: [B, L, D], or ragged sequences one behind the other, [N, D] with
    ``offsets`` [S + 1] (integers that ascend from 0 to N; equal ones are empty
    sequences).  ``initial`` [B or S, D] float32 is each sequence's history
    (zeros by default), ``final`` float32 its last state, y the states in x's
    type.  ``reverse`` runs each sequence from its last token.  A gate of +inf
    holds the state whatever x is; one of -inf forgets it; finite gates beyond
    87.3, whose smaller factor leaves float32's normal range, do the same.  A
    NaN or infinity elsewhere reaches the later states of its channel and
    sequence until a gate forgets it."""
    offsets = _index32(offsets)
    if not _wants_grad(x, gate, initial):
        return W.gated_scan_fwd(x, gate, initial, offsets, reverse, keep=False)[:2]
    return _GatedScan.apply(x, gate, initial, offsets, bool(reverse))


def gated_scan_step(x: Tensor, gate: Tensor, state: Tensor) -> Tuple[Tensor, Tensor]:
    """(y, next state) after one more token of each of B sequences: x, gate
    [B, D], state [B, D] float32."""
    if state is None:
        raise RuntimeError("state must be given")
    if not _wants_grad(x, gate, state):
        return W.gated_scan_step(x, gate, state)
    y, final = gated_scan(x[:, None], gate[:, None], state)
    return y[:, 0], final


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, rows):
        ctx.save_for_backward(x, weight, offsets, rows)
        return W.grouped_matmul_fwd(x, weight, bias, offsets, rows)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, v_y):
        x, weight, offsets, rows = ctx.saved_tensors
        need = ctx.needs_input_grad
        v_x, v_weight, v_bias = W.grouped_matmul_bwd(x, weight, offsets, rows, v_y, need[2],
                                                     need[0], need[1])
        return v_x, v_weight, v_bias, None, None


def grouped_matmul(x: Tensor, weight: Tensor, offsets: Tensor, rows: Optional[Tensor] = None,
                   bias: Optional[Tensor] = None) -> Tensor:
    """y [N, M] with ``y[r] = weight[e] @ x[r] + bias[e]`` for the rows r of each
    group e: ``rows[offsets[e]:offsets[e + 1]]``, or those numbers themselves
    without ``rows``; rows in no group give zeros.  x [N, K], weight [E, M, K],
    bias [E, M]; offsets [E + 1] ascend from 0 to at most N and ``rows`` is a
    permutation of 0..N-1, as ``group_rows`` returns them."""
    offsets, rows = _index32(offsets), _index32(rows)
    if not _wants_grad(x, weight, bias):
        return W.grouped_matmul_fwd(x, weight, bias, offsets, rows)
    return _GroupedMatmul.apply(x, weight, bias, offsets, rows)


def group_rows(ids: Tensor, n_groups: int) -> Tuple[Tensor, Tensor]:
    """(rows [N], offsets [n_groups + 1]), int32: the positions of ids [N] in
    stable order of their id, those of ids outside [0, n_groups) last."""
    return W.group_rows(ids, n_groups)
