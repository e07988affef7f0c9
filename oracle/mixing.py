"""Rotary positions, norms around a block and 8-bit AdamW states in numpy
float64, from their formulas.

``Bounded`` carries beside each value a bound on the error of any float32
evaluation of the same expression: every operation adds the rounding it makes
and hands on what its operands bring (u = 2^-24; a sum of m terms in any order
is off by at most m u times the sum of their absolute values).  No reference
counterpart (the reference has no such operators).
"""

from __future__ import annotations

import numpy as np

U = 2.0 ** -24


class Bounded:
    def __init__(self, v, e=0.0):
        self.v = np.asarray(v, np.float64)
        self.e = np.broadcast_to(np.asarray(e, np.float64), self.v.shape)

    @staticmethod
    def of(x):
        return x if isinstance(x, Bounded) else Bounded(x)

    def _rounded(self, v, e):
        return Bounded(v, e * (1 + U) + U * np.abs(v))

    def __add__(self, o):
        o = Bounded.of(o)
        return self._rounded(self.v + o.v, self.e + o.e)

    def __sub__(self, o):
        o = Bounded.of(o)
        return self._rounded(self.v - o.v, self.e + o.e)

    def __mul__(self, o):
        o = Bounded.of(o)
        return self._rounded(self.v * o.v, np.abs(self.v) * o.e + np.abs(o.v) * self.e
                             + self.e * o.e)

    __rmul__ = __mul__
    __radd__ = __add__

    def sum(self, axis, keepdims=False):
        m = self.v.shape[axis]
        mass = (np.abs(self.v) + self.e).sum(axis, keepdims=keepdims)
        return Bounded(self.v.sum(axis, keepdims=keepdims),
                       self.e.sum(axis, keepdims=keepdims) + m * U * mass)

    def mean(self):
        """Over the last axis, kept; one product with a rounded 1 / m more."""
        s = self.sum(-1, keepdims=True)
        v = s.v / self.v.shape[-1]
        return Bounded(v, s.e / self.v.shape[-1] + 2 * U * (np.abs(v) + s.e))

    def rsqrt(self):
        """1 / sqrt: a root and a quotient, one unit each."""
        v = 1.0 / np.sqrt(self.v)
        low = np.maximum(self.v - self.e, 1e-300)
        return Bounded(v, np.abs(1.0 / np.sqrt(low) - v) + 3 * U * v)


def sigmoid(g):
    """(sigmoid, 1 - sigmoid) of exact g: exp of a float32 is off by 2 units at
    most, then a sum, a quotient and a product."""
    a = np.exp(-np.abs(g))
    big, small = 1.0 / (1.0 + a), a / (1.0 + a)
    up = Bounded(np.where(g >= 0, big, small), 8 * U * np.where(g >= 0, big, small))
    down = Bounded(np.where(g >= 0, small, big), 8 * U * np.where(g >= 0, small, big))
    return up, down


def norm(x, eps, centered):
    """(normalised rows, factor)."""
    x = Bounded.of(x)
    if centered:
        x = x - x.mean()
    factor = ((x * x).mean() + eps).rsqrt()
    return x * factor, factor


def norm_grad(v, unit, factor, centered):
    along = (v * unit).mean()
    inner = v - v.mean() if centered else v
    return (inner - unit * along) * factor


def residual_norm(x, update, gate, w1, w2, v_y, v_u, scale, eps, centered):
    """{name: Bounded} of y, u and the gradients; None stands for what is not
    there (v_y, v_u: zeros)."""
    one = np.ones(x.shape[-1])
    out = {}
    y = Bounded(x)
    if update is not None:
        h, h_factor = norm(update, eps, centered) if w1 is not None else (Bounded(update), None)
        up, down = sigmoid(gate) if gate is not None else (Bounded(one), Bounded(0 * one))
        # The scale itself is rounded to float32.
        s = Bounded(scale, U * abs(scale))
        y = Bounded(x) + (s * up) * (h * (w1 if w1 is not None else one))
        out["y"] = y
    v = Bounded(np.zeros_like(x) if v_y is None else v_y)
    if w2 is not None:
        z, z_factor = norm(y, eps, centered)
        out["u"] = z * w2
        vu = np.zeros_like(x) if v_u is None else v_u
        v = v + norm_grad(Bounded(vu) * w2, z, z_factor, centered)
        out["v_w2"] = (Bounded(vu) * z).sum(0)
    out["v_x"] = v
    if update is not None:
        weight = w1 if w1 is not None else one
        v_h = (s * v) * up
        if gate is not None:
            v_gate = (s * v) * (h * weight) * (up * down)
            out["v_gate"] = v_gate if gate.ndim == x.ndim else v_gate.sum(0)
        out["v_update"] = v_h
        if w1 is not None:
            out["v_w1"] = (v_h * h).sum(0)
            out["v_update"] = norm_grad(v_h * w1, h, h_factor, centered)
    return out


def rotary(x, positions, sections, base, interleaved, shared, inverse=False):
    """(turned [N, H, D], bound).  The angle: a product in float64 of a position
    and a frequency, each off by a few 2^-53 of it, then 2^-24 of half a turn; sine
    and cosine off by 2 units; two products and a sum."""
    n, _, d = x.shape
    pairs = sum(sections)
    rate = []
    for m in sections:
        rate += [i / m for i in range(m)]
    if shared:
        rate = [i / pairs for i in range(pairs)]
    axis = np.repeat(np.arange(len(sections)), sections)
    # Turns in extended precision: float64 angles of far positions would be this
    # oracle's own error.
    turns = positions.astype(np.longdouble)[:, axis] * \
        np.longdouble(base) ** -np.asarray(rate, np.longdouble) / (2 * np.longdouble(np.pi))
    frac = (turns - np.rint(turns)).astype(np.float64)
    angle = 2 * np.pi * frac[:, None] * (-1 if inverse else 1)
    slack = (16 * 2.0 ** -53 * 2 * np.pi * np.abs(turns).astype(np.float64))[:, None] + 4 * U
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    out, bound = x.copy(), np.zeros_like(x)
    parts = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    off = (np.abs(a) + np.abs(b)) * (slack + 3 * U)
    if interleaved:
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = parts
        bound[..., 0:2 * pairs:2] = bound[..., 1:2 * pairs:2] = off
    else:
        out[..., :pairs], out[..., pairs:2 * pairs] = parts
        bound[..., :pairs] = bound[..., pairs:2 * pairs] = off
    return out, bound


# ---------------------------------------------------------- 8-bit states --

RUN, MOST, LEAST, LEAST_NORMAL = 256, 448.0, 2.0 ** -9, 2.0 ** -6


def chance(n, step):
    """The 32-bit chances of n elements at a step."""
    with np.errstate(over="ignore"):
        h = np.arange(n, dtype=np.uint32) + np.uint32(step) * np.uint32(0x9E3779B9)
        h ^= h >> np.uint32(16)
        h *= np.uint32(0x6A09E667)
        h ^= h >> np.uint32(15)
        h *= np.uint32(0xBB67AE85)
        return h ^ (h >> np.uint32(16))


def code_step(y):
    """Distance of float8 e4m3 codes at y (0 to 448)."""
    exponent = np.maximum(np.floor(np.log2(np.maximum(y, 2.0 ** -30))), -6)
    return 2.0 ** (exponent - 3)


def quantize(x, r, root):
    """(values of the codes over their scale, scales) of x [n] with chances r / 2^16."""
    runs = -(-len(x) // RUN)
    padded = np.zeros(runs * RUN)
    padded[:len(x)] = x
    most = np.where(np.isfinite(padded), np.abs(padded), 0.0).reshape(runs, RUN).max(1)
    scale = np.maximum(most / MOST, 2.0 ** -126)
    y = np.minimum(np.abs(x) / np.repeat(scale, RUN)[:len(x)], MOST)
    step = code_step(y)
    code = np.minimum(np.floor(y / step + r / 65536.0) * step, MOST)
    if root:
        code = np.where((x > 0) & (code == 0), LEAST, code)
    return np.where(np.isfinite(x), np.copysign(code, x), np.nan), scale


# ------------------------------------------------------- decay attention --


class DecayAttention:
    """S_t = g S_{t-1} + k_t v_t^T, y_t = scale S_t^T q_t over q, k [N, H, Dk],
    v [N, H, Dv], sequences [bounds[s], bounds[s + 1]), token after token.

    Beside y, the final states and the gradients it keeps the same sums of absolute
    terms (``*_mass``): an evaluation by products of c-token chunks in float32 makes
    sums of at most dk + dv + c terms and powers of g off by a few units, and walks
    length / c steps, each of which rounds the state once more."""

    def __init__(self, q, k, v, log_decay, bounds, initial=None, reverse=False, scale=1.0):
        self.q, self.k, self.v, self.scale = q, k, v, scale
        self.g = np.exp(log_decay)[:, None, None]
        self.bounds, self.reverse = bounds, reverse
        s, h = len(bounds) - 1, q.shape[1]
        zeros = np.zeros((s, h, q.shape[2], v.shape[2]))
        self.initial = zeros if initial is None else initial

    def _walk(self, q, k, v, start, early, reverse):
        """y and last states of the recurrence that all the outputs are."""
        y, last = np.zeros(v.shape), start.copy()
        with np.errstate(invalid="ignore"):
            for s in range(len(self.bounds) - 1):
                state = start[s].copy()
                order = range(self.bounds[s], self.bounds[s + 1])
                for t in reversed(order) if reverse else order:
                    if not early:
                        state = self.g * state
                    state = state + k[t][:, :, None] * v[t][:, None, :]
                    y[t] = (q[t][:, :, None] * state).sum(1)
                    if early:
                        state = self.g * state
                last[s] = state
        return y, last

    def _both(self, q, k, v, start, early, reverse):
        exact = self._walk(q, k, v, start, early, reverse)
        mass = self._walk(*(np.abs(a) for a in (q, k, v, start)), early, reverse)
        return (*exact, *mass)

    def forward(self):
        """(y, final, y_mass, final_mass)."""
        y, final, ym, fm = self._both(self.q, self.k, self.v, self.initial, False, self.reverse)
        return self.scale * y, final, abs(self.scale) * ym, fm

    def backward(self, v_y, v_final=None):
        """{name: (gradient, mass)}."""
        turn = lambda a: a.swapaxes(-1, -2)  # noqa: E731
        last = np.zeros_like(self.initial) if v_final is None else v_final
        g = self.scale * v_y
        v_q, _, qm, _ = self._both(g, self.v, self.k, turn(self.initial), False, self.reverse)
        v_v, start, vm, sm = self._both(self.k, self.q, g, last, True, not self.reverse)
        v_k, _, km, _ = self._both(self.v, g, self.q, turn(last), True, not self.reverse)
        return dict(v_q=(v_q, qm), v_k=(v_k, km), v_v=(v_v, vm), v_initial=(start, sm))
