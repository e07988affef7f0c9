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
  groups' rows anywhere in the table; ``group_rows`` finds them;
* ``decay_attention``   linear attention whose state every head forgets at its
  own rate, over equal or ragged sequences of any length, and
  ``decay_attention_step`` for one more token of running sequences;
* ``rotary_axes``       queries and keys turned by their positions along several
  axes;
* ``pre_norm``, ``residual_norm``  the norms before and after a block, with its
  gate and the residual stream between them.

Activations, tables and weights are float32, bfloat16 or float16 CUDA
tensors; sums and states are float32.  Gradients come from HIP kernels; they
are not differentiable again, and forward-mode tangents are refused.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ..cuda import _wrapper as W

__all__ = ["embedding_lookup", "gated_scan", "gated_scan_step", "grouped_matmul", "group_rows",
           "decay_attention", "decay_attention_step", "rotary_axes", "pre_norm", "residual_norm"]


def _wants_grad(*tensors) -> bool:
    """Whether the call goes through its autograd function: for a gradient, and
    for a forward-mode tangent, which that function refuses (the kernels would
    drop it)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
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


def _refuse_grad(t, name: str) -> None:
    """For an input that the kernels give no derivative for."""
    if _wants_grad(t):
        raise NotImplementedError(f"{name} must not require a gradient")


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.plan = plan
        return W.rotary_axes(q, k, positions, *plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, v_q, v_k):
        (positions,) = ctx.saved_tensors
        if v_q is None:  # alone, the keys' gradient takes the queries' place
            v_k, _ = (None, None) if v_k is None else W.rotary_axes(
                v_k, None, positions, *ctx.plan, inverse=True)
            return None, v_k, None, None
        return (*W.rotary_axes(v_q, v_k, positions, *ctx.plan, inverse=True), None, None)


def rotary_axes(q: Tensor, k: Optional[Tensor], positions: Tensor, sections: Sequence[int],
                base: float = 1e4, interleaved: bool = False, shared: bool = False
                ) -> Tuple[Tensor, Optional[Tensor]]:
    """(q', k'): pairs (a, b) of each head's channels turned to
    ``(a cos t - b sin t, b cos t + a sin t)``, so that the product of a query and
    a key depends on where they are to each other along each axis.

    q [..., H, D], k [..., Hk, D] (or None), positions [..., A] int32, int64 or
    float32, the tokens' places on A axes.  ``sections[a]`` pairs belong to axis
    a; pair i of its m has ``t = position[a] base^(-i / m)``, or with ``shared``
    i and m count all pairs of all axes.  With R pairs in all, pair j is channels
    j and R + j, or with ``interleaved`` 2j and 2j + 1; channels from 2R on stay
    as they are.  Angles are exact to a float32 turn for positions up to 2^31.
    Positions have no gradient."""
    _refuse_grad(positions, "positions")
    plan = (tuple(sections), float(base), bool(interleaved), bool(shared))
    if not _wants_grad(q, k):
        return W.rotary_axes(q, k, positions, *plan)
    return _Rotary.apply(q, k, positions, plan)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, update, gate, update_weight, weight, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, update, gate, update_weight, weight)
        ctx.plan = plan
        y, u = W.residual_norm_fwd(x, update, gate, update_weight, weight, *plan)
        return (u,) if update is None else (y,) if weight is None else (y, u)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, update, gate, update_weight, weight = ctx.saved_tensors
        v_y, v_u = (None, *grads) if update is None else (*grads, None)[:2]
        if v_y is None and v_u is None:
            return (None,) * 6
        return (*W.residual_norm_bwd(x, update, gate, update_weight, weight, v_y, v_u, *ctx.plan,
                                     want=ctx.needs_input_grad[:5]), None)


def pre_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, centered: bool = False) -> Tensor:
    """``norm(x) * weight`` over the last dimension (at most 8192 channels):
    ``norm(x) = x / sqrt(mean(x^2) + eps)``, with ``centered`` of x less its mean.
    x [..., D], weight [D]."""
    if weight is None:
        raise RuntimeError("weight must be given")
    plan = (1.0, float(eps), bool(centered))
    if not _wants_grad(x, weight):
        return W.residual_norm_fwd(x, None, None, None, weight, *plan)[1]
    return _ResidualNorm.apply(x, None, None, None, weight, plan)[0]


def residual_norm(x: Tensor, update: Tensor, gate: Optional[Tensor] = None,
                  update_weight: Optional[Tensor] = None, weight: Optional[Tensor] = None,
                  scale: float = 1.0, eps: float = 1e-6, centered: bool = False
                  ) -> Tuple[Tensor, Optional[Tensor]]:
    """(y, u): a block's output joined to the stream, and the norm before the
    next block, in one pass::

        y = x + scale * sigmoid(gate) * norm(update) * update_weight
        u = norm(y) * weight

    x, update [..., D]; gate of their shape or [D] for all rows (none: 1); without
    ``update_weight`` the update is not normalised, without ``weight`` u is None.
    ``norm`` is that of ``pre_norm``; u is made from y before y is rounded to its
    type."""
    if update is None:
        raise RuntimeError("update must be given")
    plan = (float(scale), float(eps), bool(centered))
    if not _wants_grad(x, update, gate, update_weight, weight):
        return W.residual_norm_fwd(x, update, gate, update_weight, weight, *plan)
    out = _ResidualNorm.apply(x, update, gate, update_weight, weight, plan)
    return out if weight is not None else (out[0], None)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, offsets, reverse, scale):
        ctx.set_materialize_grads(False)
        y, final, kept = W.decay_attention_fwd(q, k, v, log_decay, initial, offsets, reverse, scale)
        ctx.save_for_backward(q, k, v, log_decay, initial, offsets, kept)
        ctx.reverse, ctx.scale = reverse, scale
        return y, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, v_y, v_final):
        q, k, v, log_decay, initial, offsets, kept = ctx.saved_tensors
        if v_y is None:
            v_y = torch.zeros_like(v)
        v_q, v_k, v_v, v_initial = W.decay_attention_bwd(q, k, v, log_decay, initial, offsets, kept,
                                                         v_y, v_final, ctx.reverse, ctx.scale)
        return (v_q, v_k, v_v, None, v_initial if ctx.needs_input_grad[4] else None, None, None,
                None)


def decay_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor,
                    initial: Optional[Tensor] = None, offsets: Optional[Tensor] = None,
                    reverse: bool = False, scale: Optional[float] = None
                    ) -> Tuple[Tensor, Tensor]:
    """(y, final) of linear attention with a decay for each head::

        S_t = exp(log_decay) S_{t-1} + k_t v_t^T,    y_t = scale S_t^T q_t

    q, k: [B, L, H, Dk], v: [B, L, H, Dv], or ragged sequences one behind the
    other, [N, H, D] with ``offsets`` [S + 1] (integers that ascend from 0 to at
    most N; equal ones are empty sequences; tokens behind the last give zeros).
    Dk and Dv up to 256.  ``log_decay`` [H] float32 holds the natural logarithms
    of the decays, at most 0 (-inf: every token alone); it has no gradient.
    ``initial`` [B or S, H, Dk, Dv] float32 is each sequence's first state (zeros
    by default), ``final`` its last.  ``scale`` is Dk^-0.5 by default; ``reverse``
    runs each sequence from its last token.  A NaN or infinity reaches later
    tokens of its head and sequence, never earlier ones."""
    _refuse_grad(log_decay, "log_decay")
    offsets = _index32(offsets)
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.shape[-1] else 1.0
    if not _wants_grad(q, k, v, initial):
        return W.decay_attention_fwd(q, k, v, log_decay, initial, offsets, bool(reverse),
                                     float(scale), keep=False)[:2]
    return _DecayAttention.apply(q, k, v, log_decay, initial, offsets, bool(reverse), float(scale))


def decay_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor,
                         scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """(y, next state) after one more token of each of B sequences: q, k
    [B, H, Dk], v [B, H, Dv], state [B, H, Dk, Dv] float32."""
    if state is None:
        raise RuntimeError("state must be given")
    _refuse_grad(log_decay, "log_decay")
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.shape[-1] else 1.0
    if not _wants_grad(q, k, v, state):
        return W.decay_attention_step(q, k, v, log_decay, state, float(scale))
    y, final = decay_attention(q[:, None], k[:, None], v[:, None], log_decay, state, scale=scale)
    return y[:, 0], final
