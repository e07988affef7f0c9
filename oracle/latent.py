"""The latent decoder's operators in numpy float64, from their formulas.

Each function returns the exact value and, beside it, what a bound on a
float32 evaluation needs: sums of absolute terms, and for the recurrence the
sum of terms weighted by the number of roundings that each has gone through.
No reference counterpart (the reference has no such operators).
"""

from __future__ import annotations

import numpy as np


def lookup(table, ids, scale):
    out = np.zeros((*ids.shape, table.shape[1]))
    known = (ids >= 0) & (ids < table.shape[0])
    out[known] = scale * table[ids[known]]
    return out


def lookup_grad(v_out, ids, n_rows, scale):
    """(gradient [V, D], the same of |v_out|, entries of each row [V])."""
    grad = np.zeros((n_rows, v_out.shape[-1]))
    mass = np.zeros_like(grad)
    count = np.zeros(n_rows, np.int64)
    flat = v_out.reshape(-1, v_out.shape[-1])
    for i, v in enumerate(ids.reshape(-1)):
        if 0 <= v < n_rows:
            grad[v] += flat[i]
            mass[v] += np.abs(flat[i])
            count[v] += 1
    return scale * grad, abs(scale) * mass, count


def groups(ids, n_groups):
    inside = (ids >= 0) & (ids < n_groups)
    key = np.where(inside, ids, n_groups)
    rows = np.argsort(key, kind="stable")
    return rows, np.searchsorted(key[rows], np.arange(n_groups + 1))


def sigmoid(g):
    with np.errstate(over="ignore"):
        return np.where(g >= 0, 1.0 / (1.0 + np.exp(-np.abs(g))),
                        np.exp(-np.abs(g)) / (1.0 + np.exp(-np.abs(g))))


def _drop(factor, value):
    """factor * value, nothing where the factor is 0."""
    with np.errstate(invalid="ignore"):
        return np.where(factor == 0, 0.0, factor * value)


class Scan:
    """h_t = a_t h_{t-1} + (1 - a_t) x_t over x [N, D], sequences
    [bounds[s], bounds[s + 1])."""

    def __init__(self, x, gate, bounds, initial=None, reverse=False):
        self.x, self.a, self.b = x, sigmoid(gate), sigmoid(-gate)
        self.bounds, self.reverse = bounds, reverse
        s = len(bounds) - 1
        self.state = np.zeros((s, x.shape[1])) if initial is None else initial
        self.h, self.prior = np.zeros_like(x), np.zeros_like(x)
        self.final = np.array(self.state, dtype=np.float64, copy=True)
        # Sums of |terms|, and of |terms| times the steps each went through.
        self.mass, self.steps = np.zeros_like(x), np.zeros_like(x)
        self.prior_steps, self.final_steps = np.zeros_like(x), np.zeros_like(self.final)
        for q in range(s):
            now, mass, steps = self.state[q], np.abs(self.state[q]), np.zeros(x.shape[1])
            for t in self._order(q):
                a, b = self.a[t], self.b[t]
                self.prior[t], self.prior_steps[t] = now, steps
                new = _drop(b, x[t])
                now = _drop(a, now) + new
                steps = _drop(a, steps + mass) + np.abs(new)
                mass = _drop(a, mass) + np.abs(new)
                self.h[t], self.mass[t], self.steps[t] = now, mass, steps
            self.final[q], self.final_steps[q] = now, steps

    def _order(self, q):
        lo, hi = int(self.bounds[q]), int(self.bounds[q + 1])
        return range(hi - 1, lo - 1, -1) if self.reverse else range(lo, hi)

    def grad(self, v_y, v_final):
        """(v_x, v_gate, v_initial, flow, flow_steps): flow_t the gradient that
        reaches the state after token t."""
        flow, steps_at = np.zeros_like(self.x), np.zeros_like(self.x)
        v_initial = np.array(v_final, dtype=np.float64, copy=True)
        initial_steps = np.zeros_like(v_initial)
        for q in range(len(self.bounds) - 1):
            now, mass = v_final[q], np.abs(v_final[q])
            steps = np.zeros(self.x.shape[1])
            for t in reversed(self._order(q)):
                now = now + v_y[t]
                mass = mass + np.abs(v_y[t])
                steps = steps + mass
                flow[t], steps_at[t] = now, steps
                now, mass, steps = (_drop(self.a[t], z) for z in (now, mass, steps + mass))
            v_initial[q], initial_steps[q] = now, steps
        with np.errstate(invalid="ignore"):
            v_x = _drop(self.b, flow)
            v_gate = _drop(self.a * self.b, flow * (self.prior - self.x))
        return v_x, v_gate, v_initial, flow, steps_at, initial_steps


def grouped(x, weight, bias, offsets, rows):
    """(y, sums of |terms|)."""
    n = x.shape[0]
    rows = np.arange(n) if rows is None else rows
    y, mass = np.zeros((n, weight.shape[1])), np.zeros((n, weight.shape[1]))
    for e in range(weight.shape[0]):
        r = rows[offsets[e]:offsets[e + 1]]
        y[r], mass[r] = x[r] @ weight[e].T, np.abs(x[r]) @ np.abs(weight[e]).T
        if bias is not None:
            y[r] += bias[e]
            mass[r] += np.abs(bias[e])
    return y, mass


def grouped_grad(x, weight, offsets, rows, v_y):
    """((v_x, mass), (v_weight, mass), (v_bias, mass), rows of each group)."""
    n = x.shape[0]
    rows = np.arange(n) if rows is None else rows
    v_x, m_x = np.zeros_like(x), np.zeros_like(x)
    v_w, m_w = np.zeros_like(weight), np.zeros_like(weight)
    v_b, m_b = np.zeros(weight.shape[:2]), np.zeros(weight.shape[:2])
    sizes = np.zeros(weight.shape[0], np.int64)
    for e in range(weight.shape[0]):
        r = rows[offsets[e]:offsets[e + 1]]
        sizes[e] = len(r)
        v_x[r], m_x[r] = v_y[r] @ weight[e], np.abs(v_y[r]) @ np.abs(weight[e])
        v_w[e], m_w[e] = v_y[r].T @ x[r], np.abs(v_y[r]).T @ np.abs(x[r])
        v_b[e], m_b[e] = v_y[r].sum(0), np.abs(v_y[r]).sum(0)
    return (v_x, m_x), (v_w, m_w), (v_b, m_b), sizes
