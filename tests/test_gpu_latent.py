"""The latent decoder's operators on the GPU against float64.

Tolerances are bounds on a float32 evaluation, from the roundings it makes
(u = 2^-24 each), plus the one rounding to the output's type:

* a sum of m products:  (m + 2) u sum |terms|;
* the recurrence: a term that has gone through j steps carries j factors, each
  with the error of a gate (exponent 2 |g| u, exp2 and reciprocal one unit in
  the last place each, two more roundings) and of its product: j (2 |g| + 9) u
  of the term, summed over the terms (oracle.latent.Scan keeps that sum).
"""

import numpy as np
import pytest
import torch

from oracle import latent as ref
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _close(got, exact, bound, dtype, what):
    got = _np(got)
    assert got.shape == exact.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(exact)), what
    tol = bound + ROUND[dtype] * (np.abs(exact) + bound) + TINY[dtype]
    err = np.abs(got - exact)
    bad = ~(err <= tol) & ~np.isnan(exact) & (got != exact)
    assert not bad.any(), (what, float(np.nanmax(err / tol)), np.argwhere(bad)[:4].tolist())


# ------------------------------------------------------------- group_rows --


@pytest.mark.parametrize("n,groups", [(0, 3), (1, 1), (5, 0), (777, 1), (4097, 18), (70_001, 2047),
                                      (70_001, 2048), (9000, 100_000)])
@pytest.mark.parametrize("wide", [False, True])
def test_group_rows(n, groups, wide):
    ids = torch.randint(-2, groups + 2, (n,), generator=_gen(n + groups))
    ids = ids.to(torch.int64 if wide else torch.int32)
    rows, offsets = latent.group_rows(ids.to(DEV), groups)
    e_rows, e_offsets = ref.groups(ids.numpy().astype(np.int64), groups)
    assert np.array_equal(rows.cpu().numpy(), e_rows)
    assert np.array_equal(offsets.cpu().numpy(), e_offsets)


def test_group_rows_of_ids_beyond_32_bits():
    ids = torch.tensor([1, 2 ** 32, 0, -2 ** 40, 2 ** 32 + 1, 1], device=DEV)
    rows, offsets = latent.group_rows(ids, 2)
    assert rows.tolist() == [2, 0, 5, 1, 3, 4] and offsets.tolist() == [0, 1, 3]


# ----------------------------------------------------------------- lookup --


def _lookup_case(n, v, d, dtype, seed, kind="any"):
    g = _gen(seed)
    ids = torch.randint(0, max(v, 1), (n,), generator=g)
    if kind == "any" and n:
        ids[torch.rand(n, generator=g) < 0.1] = -1
        ids[torch.rand(n, generator=g) < 0.05] = v
    elif kind == "one":
        ids[:] = v // 2
    return _randn(g, v, d, dtype=dtype), ids, _randn(g, n, d, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d,kind", [
    (0, 5, 4, "any"), (1, 1, 1, "all"), (3, 0, 6, "any"), (65, 7, 3, "any"), (1000, 33, 45, "any"),
    (4111, 18, 64, "all"), (5000, 3, 16, "one"), (2500, 3001, 256, "any"), (300, 9, 600, "any"),
    (33, 40, 1030, "all")])
def test_lookup(n, v, d, kind, dtype):
    table, ids, v_out = _lookup_case(n, v, d, dtype, n + 7 * v + d, kind)
    scale = 1.7
    out = latent.embedding_lookup(table.to(DEV), ids.to(DEV), scale)
    exact = ref.lookup(_np(table), ids.numpy(), scale)
    _close(out, exact, 2 * U * np.abs(exact), dtype, "out")  # scale and product
    grad = W.embedding_bwd(v_out.to(DEV), ids.to(DEV), v, scale)
    exact, mass, count = ref.lookup_grad(_np(v_out), ids.numpy(), v, scale)
    _close(grad, exact, (count[:, None] + 3) * U * mass, dtype, "v_table")
    again = W.embedding_bwd(v_out.to(DEV), ids.to(DEV), v, scale)
    assert torch.equal(grad, again)


def test_lookup_ids_of_any_shape_and_32_bits():
    table, ids, v_out = _lookup_case(120, 11, 8, torch.float32, 0)
    ids = ids.reshape(4, 30)
    out = latent.embedding_lookup(table.to(DEV), ids.to(DEV))
    assert out.shape == (4, 30, 8)
    assert torch.equal(out, latent.embedding_lookup(table.to(DEV), ids.to(torch.int32).to(DEV)))
    a = W.embedding_bwd(v_out.reshape(4, 30, 8).to(DEV), ids.to(DEV), 11)
    assert torch.equal(a, W.embedding_bwd(v_out.to(DEV), ids.reshape(-1).to(torch.int32).to(DEV),
                                          11))


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_of_strided_and_unaligned_rows(dtype):
    table, ids, v_out = _lookup_case(200, 20, 24, dtype, 3)
    base = latent.embedding_lookup(table.to(DEV), ids.to(DEV))
    grad = W.embedding_bwd(v_out.to(DEV), ids.to(DEV), 20)
    for lead, width in ((0, 40), (1, 41), (2, 30), (4, 32)):
        wide = torch.full((20, width), 9.0, dtype=dtype, device=DEV)
        wide[:, lead:lead + 24] = table.to(DEV)
        assert torch.equal(latent.embedding_lookup(wide[:, lead:lead + 24], ids.to(DEV)), base)
        wide = torch.full((200, width), 9.0, dtype=dtype, device=DEV)
        wide[:, lead:lead + 24] = v_out.to(DEV)
        assert torch.equal(W.embedding_bwd(wide[:, lead:lead + 24], ids.to(DEV), 20), grad)
    assert torch.equal(latent.embedding_lookup(table.t().contiguous().to(DEV).t(), ids.to(DEV)),
                       base)
    # One gradient row for every position (a summed output's).
    shared = v_out[:1].to(DEV).expand(200, 24)
    assert torch.equal(W.embedding_bwd(shared, ids.to(DEV), 20),
                       W.embedding_bwd(shared.contiguous(), ids.to(DEV), 20))


def test_lookup_autograd():
    table, ids, v_out = _lookup_case(500, 40, 12, torch.float32, 5)
    t = table.to(DEV).requires_grad_(True)
    out = latent.embedding_lookup(t, ids.to(DEV), scale=0.5)
    out.backward(v_out.to(DEV))
    assert torch.equal(t.grad, W.embedding_bwd(v_out.to(DEV), ids.to(DEV), 40, 0.5))
    # A difference of the (linear) forward along one direction.
    e = _randn(_gen(9), 40, 12)
    lhs = (ref.lookup(_np(e), ids.numpy(), 0.5) * _np(v_out)).sum()
    _, mass, count = ref.lookup_grad(_np(v_out), ids.numpy(), 40, 0.5)
    tol = ((count[:, None] + 3) * U * mass * np.abs(_np(e))).sum()
    assert abs((_np(t.grad) * _np(e)).sum() - lhs) <= tol


def test_lookup_keeps_nonfinite_rows_apart():
    table = torch.ones(4, 8, device=DEV)
    table[1] = float("nan")
    table[2] = float("inf")
    out = latent.embedding_lookup(table, torch.tensor([0, -1, 1, 2, 3, 4], device=DEV))
    assert torch.isnan(out[2]).all() and torch.isinf(out[3]).all()
    assert (out[[0, 4]] == 1).all() and (out[[1, 5]] == 0).all()
    grad = W.embedding_bwd(out, torch.tensor([0, 0, -1, 9, 2, 2], device=DEV), 3)
    assert torch.equal(grad, torch.tensor([1.0, 0.0, 1.0], device=DEV)[:, None].expand(3, 8))


# ------------------------------------------------------------------- scan --


def _bounds(kind, n, g):
    if kind == "one":
        return [0, n]
    if kind == "ones":
        return list(range(n + 1))
    cuts = torch.randint(0, n + 1, (max(1, n // 40) + 6,), generator=g)
    cuts[:3] = n // 2  # empty sequences inside, at the start and at the end
    return sorted([0, 0] + cuts.tolist() + [n, n, n])


def _scan_case(n, d, kind, dtype, seed, gate_scale=1.5):
    g = _gen(seed)
    x, gate = _randn(g, n, d, dtype=dtype), _randn(g, n, d, dtype=dtype, scale=gate_scale, shift=1.5)
    bounds = _bounds(kind, n, g)
    s = len(bounds) - 1
    return (x, gate, torch.tensor(bounds, dtype=torch.int32), _randn(g, s, d),
            _randn(g, n, d, dtype=dtype), _randn(g, s, d))


def _check_scan(x, gate, offsets, initial, v_y, v_final, reverse, got):
    y, final, v_x, v_gate, v_initial = got
    dtype = x.dtype
    s = offsets.numel() - 1
    scan = ref.Scan(_np(x), _np(gate), offsets.numpy(), _np(initial), reverse)
    finite = np.abs(_np(gate))
    finite = finite[np.isfinite(finite)]
    kappa = (2 * (finite.max() if finite.size else 0.0) + 9) * U
    _close(y, scan.h, kappa * scan.steps, dtype, "y")
    _close(final, scan.final, kappa * scan.final_steps, torch.float32, "final")
    if v_x is None:
        return
    vf = np.zeros((s, x.shape[1])) if v_final is None else _np(v_final)
    e_x, e_g, e_i, flow, steps, i_steps = scan.grad(_np(v_y), vf)
    ab = scan.a * scan.b
    with np.errstate(invalid="ignore"):
        gap = np.abs(scan.prior) + np.abs(_np(x))
        _close(v_x, e_x, ref._drop(scan.b, kappa * (steps + np.abs(flow))), dtype, "v_x")
        b_g = ref._drop(ab, kappa * (np.abs(scan.prior - _np(x)) * steps
                                     + np.abs(flow) * scan.prior_steps
                                     + 2 * np.abs(flow) * gap))
    _close(v_gate, e_g, b_g, dtype, "v_gate")
    _close(v_initial, e_i, kappa * (i_steps + np.abs(e_i)), torch.float32, "v_initial")


def _run_scan(x, gate, offsets, initial, v_y, v_final, reverse):
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    x, gate, offsets, initial, v_y, v_final = map(dev, (x, gate, offsets, initial, v_y, v_final))
    y, final, carries = W.gated_scan_fwd(x, gate, initial, offsets, reverse)
    return (y, final, *W.gated_scan_bwd(x, gate, initial, offsets, carries, v_y, v_final, reverse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("n,d,kind", [
    (1, 1, "one"), (17, 5, "ragged"), (300, 64, "one"), (129, 33, "ragged"), (2049, 7, "ragged"),
    (1500, 99, "ragged"), (700, 130, "ones"), (5000, 2, "one"), (257, 300, "ragged")])
def test_scan(n, d, kind, reverse, dtype):
    case = _scan_case(n, d, kind, dtype, 11 * n + d)
    _check_scan(*case, reverse, _run_scan(*case, reverse))


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_without_states_or_their_gradients(dtype):
    x, gate, offsets, _, v_y, _ = _scan_case(333, 40, "ragged", dtype, 1)
    case = (x, gate, offsets, None, v_y, None)
    _check_scan(*case, False, _run_scan(*case, False))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,l,d", [(1, 1, 3), (5, 1, 64), (3, 2, 10), (4, 130, 66), (70, 9, 32)])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_equal_sequences(b, l, d, reverse, dtype):
    g = _gen(b + l + d)
    x, gate = _randn(g, b, l, d, dtype=dtype), _randn(g, b, l, d, dtype=dtype, scale=2.0)
    initial, v_final = _randn(g, b, d), _randn(g, b, d)
    v_y = _randn(g, b, l, d, dtype=dtype)
    y, final, carries = W.gated_scan_fwd(x.to(DEV), gate.to(DEV), initial.to(DEV), None, reverse)
    grads = W.gated_scan_bwd(x.to(DEV), gate.to(DEV), initial.to(DEV), None, carries, v_y.to(DEV),
                             v_final.to(DEV), reverse)
    flat = lambda t: t.reshape(b * l, d)  # noqa: E731
    _check_scan(flat(x), flat(gate), torch.arange(0, b * l + 1, l), initial, flat(v_y), v_final,
                reverse, (flat(y), final, flat(grads[0]), flat(grads[1]), grads[2]))


def test_scan_without_tokens():
    x = torch.zeros(0, 6, device=DEV)
    offsets = torch.zeros(4, dtype=torch.int32, device=DEV)
    initial, v_final = torch.randn(3, 6, device=DEV), torch.randn(3, 6, device=DEV)
    y, final, carries = W.gated_scan_fwd(x, x, initial, offsets)
    assert y.shape == (0, 6) and torch.equal(final, initial)
    v_x, v_gate, v_initial = W.gated_scan_bwd(x, x, initial, offsets, carries, x, v_final)
    assert v_x.shape == v_gate.shape == (0, 6) and torch.equal(v_initial, v_final)
    z = torch.zeros(2, 0, 6, device=DEV)
    y, final = latent.gated_scan(z, z, initial[:2])
    assert y.shape == (2, 0, 6) and torch.equal(final, initial[:2])
    assert latent.gated_scan(z, z)[1].abs().sum() == 0
    assert latent.gated_scan(z[:0], z[:0])[0].shape == (0, 0, 6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_gates_of_infinity_hold_and_forget(reverse, dtype):
    x, gate, offsets, initial, v_y, v_final = _scan_case(900, 34, "ragged", dtype, 21)
    g = _gen(4)
    hold, forget = torch.rand(900, 34, generator=g) < 0.3, torch.rand(900, 34, generator=g) < 0.1
    gate[forget] = float("-inf")
    gate[hold] = float("inf")
    clean = (x.clone(), gate, offsets, initial, v_y, v_final)
    got = _run_scan(*clean, reverse)
    _check_scan(*clean, reverse, got)
    # What a held token's input holds does not matter.
    x[hold] = float("nan")
    y, final, v_x, _, _ = _run_scan(x, gate, offsets, initial, v_y, v_final, reverse)
    assert torch.equal(y, got[0]) and torch.equal(final, got[1]) and torch.equal(v_x, got[2])


def test_scan_forgets_a_state_that_is_not_finite():
    x = torch.ones(1, 400, 8, device=DEV)
    gate = torch.zeros(1, 400, 8, device=DEV)
    x[0, 3], x[0, 200] = float("nan"), float("inf")
    gate[0, 100] = gate[0, 203] = float("-inf")
    y, _ = latent.gated_scan(x, gate)
    assert torch.isfinite(y[0, :3]).all() and torch.isnan(y[0, 3:100]).all()
    assert (y[0, 100:200] == 1).all() and torch.isinf(y[0, 200:203]).all()
    assert (y[0, 203:] == 1).all()


@pytest.mark.parametrize("value", [-3.0e38, 3.0e38])
def test_scan_of_the_largest_gates(value):
    x, gate, offsets, initial, v_y, v_final = _scan_case(200, 16, "ragged", torch.float32, 8)
    gate[torch.rand(200, 16, generator=_gen(1)) < 0.5] = value
    case = (x, gate, offsets, initial, v_y, v_final)
    got = _run_scan(*case, False)
    assert all(torch.isfinite(t).all() for t in got)
    limit = gate.clone()
    limit[gate.abs() > 1e38] = float("inf") if value > 0 else float("-inf")
    for a, b in zip(got, _run_scan(x, limit, offsets, initial, v_y, v_final, False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_of_strided_and_unaligned_rows(dtype):
    x, gate, offsets, initial, v_y, v_final = (t.to(DEV) for t in
                                               _scan_case(260, 22, "ragged", dtype, 2))
    base = _run_scan(x, gate, offsets, initial, v_y, v_final, False)

    def wide(t, lead, width):
        w = torch.full((260, width), 7.0, dtype=dtype, device=DEV)
        w[:, lead:lead + 22] = t
        return w[:, lead:lead + 22]

    for lead, width in ((0, 44), (22, 44), (1, 23), (2, 27)):
        got = _run_scan(wide(x, lead, width), wide(gate, lead, width), offsets, initial,
                        wide(v_y, lead, width), v_final, False)
        for a, b in zip(got, base):
            assert torch.equal(a, b)
    shared = v_y[:1].expand(260, 22)  # a broadcast gradient
    for a, b in zip(_run_scan(x, gate, offsets, initial, shared, v_final, False),
                    _run_scan(x, gate, offsets, initial, shared.contiguous(), v_final, False)):
        assert torch.equal(a, b)


def test_scan_steps_equal_the_sequence():
    g = _gen(0)
    x, gate = _randn(g, 6, 20, 48), _randn(g, 6, 20, 48, scale=2.0)
    initial = _randn(g, 6, 48)
    state, ys = initial.to(DEV), []
    for t in range(20):
        y, state = latent.gated_scan_step(x[:, t].to(DEV), gate[:, t].to(DEV), state)
        ys.append(y)
    flat = lambda t: t.reshape(120, 48)  # noqa: E731
    _check_scan(flat(x), flat(gate), torch.arange(0, 121, 20), initial, None, None, False,
                (flat(torch.stack(ys, 1)), state, None, None, None))


def test_scan_autograd_and_differences():
    case = _scan_case(90, 6, "ragged", torch.float32, 13)
    x, gate, offsets, initial, v_y, v_final = case
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gate, initial)]
    y, final = latent.gated_scan(*leaves, offsets=offsets.to(DEV).to(torch.int64), reverse=True)
    ((y * v_y.to(DEV)).sum() + (final * v_final.to(DEV)).sum()).backward()
    grads = [t.grad for t in leaves]
    _check_scan(*case, True, (y, final, *grads))

    def loss(xv, gv, iv):
        s = ref.Scan(xv, gv, offsets.numpy(), iv, True)
        return (s.h * _np(v_y)).sum() + (s.final * _np(v_final)).sum()

    point = [_np(t) for t in (x, gate, initial)]
    rng = np.random.default_rng(0)
    for i in range(3):
        e = rng.standard_normal(point[i].shape)
        step = 1e-5
        hi, lo = list(point), list(point)
        hi[i], lo[i] = point[i] + step * e, point[i] - step * e
        diff = (loss(*hi) - loss(*lo)) / (2 * step)
        # Third derivatives of order one over 90 tokens: 1e-10 of their sum;
        # float32 sums of a few hundred terms: 1e-4 of it at the very most.
        scale = np.abs(_np(grads[i]) * e).sum()
        assert abs((_np(grads[i]) * e).sum() - diff) <= 1e-4 * scale, i
    # An output that receives no gradient.
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gate)]
    latent.gated_scan(*leaves, offsets=offsets.to(DEV))[1].sum().backward()
    assert all(torch.isfinite(t.grad).all() for t in leaves)


# ---------------------------------------------------------------- grouped --


def _grouped_case(n, k, m, e, dtype, seed, routed, rest=0):
    g = _gen(seed)
    x, weight = _randn(g, n, k, dtype=dtype), _randn(g, e, m, k, dtype=dtype)
    bias, v_y = _randn(g, e, m, dtype=dtype), _randn(g, n, m, dtype=dtype)
    ids = torch.randint(0, max(1, e), (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.4] = 0  # ragged: many in one, some groups empty
    ids[ids == 2] = 1
    if rest or e == 0:
        ids[:n // 5 if e else n] = -1
    rows, offsets = ref.groups(ids.numpy(), e)
    rows = torch.from_numpy(rows).to(torch.int32) if routed else None
    return x, weight, bias, torch.from_numpy(offsets).to(torch.int32), rows, v_y


def _check_grouped(case, got):
    x, weight, bias, offsets, rows, v_y = case
    y, v_x, v_weight, v_bias = got
    r = None if rows is None else rows.numpy()
    k, m = x.shape[1], weight.shape[1]
    exact, mass = ref.grouped(_np(x), _np(weight), _np(bias), offsets.numpy(), r)
    _close(y, exact, (k + 2) * U * mass, x.dtype, "y")
    (e_x, m_x), (e_w, m_w), (e_b, m_b), sizes = ref.grouped_grad(_np(x), _np(weight),
                                                                 offsets.numpy(), r, _np(v_y))
    _close(v_x, e_x, (m + 2) * U * m_x, x.dtype, "v_x")
    _close(v_weight, e_w, (sizes[:, None, None] + 2) * U * m_w, x.dtype, "v_weight")
    if v_bias is not None:
        _close(v_bias, e_b, (sizes[:, None] + 2) * U * m_b, x.dtype, "v_bias")


def _run_grouped(x, weight, bias, offsets, rows, v_y):
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    x, weight, bias, offsets, rows, v_y = map(dev, (x, weight, bias, offsets, rows, v_y))
    y = W.grouped_matmul_fwd(x, weight, bias, offsets, rows)
    return (y, *W.grouped_matmul_bwd(x, weight, offsets, rows, v_y, bias is not None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("routed", [False, True])
@pytest.mark.parametrize("n,k,m,e", [
    (1, 1, 1, 1), (7, 3, 5, 9), (64, 64, 64, 4), (200, 45, 11, 10), (1000, 128, 96, 6),
    (333, 17, 130, 70), (2600, 64, 72, 3), (513, 200, 40, 5), (90, 260, 264, 8), (0, 8, 8, 2),
    (40, 0, 8, 3), (5000, 32, 32, 2)])
def test_grouped(n, k, m, e, routed, dtype):
    case = _grouped_case(n, k, m, e, dtype, n + k + m + e, routed)
    _check_grouped(case, _run_grouped(*case))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("routed", [False, True])
def test_grouped_rows_in_no_group(routed, dtype):
    case = _grouped_case(700, 48, 80, 5, dtype, 1, routed, rest=1)
    got = _run_grouped(*case)
    _check_grouped(case, got)
    none = case[4][case[3][-1]:].long() if routed else torch.arange(int(case[3][-1]), 700)
    assert len(none) and (got[0][none.to(DEV)] == 0).all() and (got[1][none.to(DEV)] == 0).all()
    # No group at all.
    case = _grouped_case(70, 16, 8, 0, dtype, 2, routed)
    y, v_x, v_weight, v_bias = _run_grouped(*case)
    assert y.abs().sum() == 0 and v_x.abs().sum() == 0 and v_weight.numel() == 0


def test_grouped_keeps_nonfinite_rows_apart():
    x, weight, bias, offsets, rows, v_y = _grouped_case(300, 40, 24, 4, torch.bfloat16, 5, True)
    clean = _run_grouped(x, weight, bias, offsets, rows, v_y)
    x[7], weight[3] = float("nan"), float("inf")
    y, v_x, v_weight, _ = _run_grouped(x, weight, bias, offsets, rows, v_y)
    group = torch.empty(300, dtype=torch.long)
    for e in range(4):
        group[rows[offsets[e]:offsets[e + 1]].long()] = e
    other = (group != 3) & (torch.arange(300) != 7)
    assert torch.isnan(y[7]).all() and torch.equal(y[other.to(DEV)], clean[0][other.to(DEV)])
    assert torch.equal(v_x[(group != 3).to(DEV)], clean[1][(group != 3).to(DEV)])
    for e in range(4):
        assert torch.isnan(v_weight[e]).all() == (e == int(group[7]))
        assert e == int(group[7]) or torch.equal(v_weight[e], clean[2][e])


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_of_strided_and_unaligned_rows(dtype):
    case = _grouped_case(210, 24, 40, 4, dtype, 6, True)
    x, weight, bias, offsets, rows, v_y = (t.to(DEV) for t in case)
    base = _run_grouped(x, weight, bias, offsets, rows, v_y)

    def wide(t, lead, width):
        w = torch.full((210, width), 7.0, dtype=dtype, device=DEV)
        w[:, lead:lead + t.shape[1]] = t
        return w[:, lead:lead + t.shape[1]]

    for lead, width in ((0, 64), (8, 56), (1, 47), (2, 42)):
        got = _run_grouped(wide(x, lead, width), weight, bias, offsets, rows,
                           wide(v_y, lead, width))
        for a, b in zip(got, base):
            assert torch.equal(a, b)
    flipped = weight.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(_run_grouped(x, flipped, bias, offsets, rows, v_y)[0], base[0])
    # A broadcast gradient, and only some of the gradients.
    shared = v_y[:1].expand(210, 40)
    full = W.grouped_matmul_bwd(x, weight, offsets, rows, shared.contiguous(), True)
    for a, b in zip(W.grouped_matmul_bwd(x, weight, offsets, rows, shared, True), full):
        assert torch.equal(a, b)
    only = W.grouped_matmul_bwd(x, weight, offsets, rows, shared, False, False, True)
    assert only[0] is None and only[2] is None and torch.equal(only[1], full[1])
    only = W.grouped_matmul_bwd(x, weight, offsets, rows, shared, True, True, False)
    assert only[1] is None and torch.equal(only[0], full[0]) and torch.equal(only[2], full[2])


def test_grouped_autograd_and_differences():
    case = _grouped_case(150, 20, 12, 4, torch.float32, 9, True)
    x, weight, bias, offsets, rows, v_y = case
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, weight, bias)]
    y = latent.grouped_matmul(leaves[0], leaves[1], offsets.to(DEV), rows=rows.to(DEV).long(),
                              bias=leaves[2])
    y.backward(v_y.to(DEV))
    grads = [t.grad for t in leaves]
    _check_grouped(case, (y, *grads))
    rng = np.random.default_rng(1)
    point = [_np(t) for t in (x, weight, bias)]
    (_, m_x), (_, m_w), (_, m_b), sizes = ref.grouped_grad(point[0], point[1], offsets.numpy(),
                                                           rows.numpy(), _np(v_y))
    bounds = ((12 + 3) * U * m_x, (sizes[:, None, None] + 3) * U * m_w,
              (sizes[:, None] + 3) * U * m_b)
    for i in range(3):
        e = rng.standard_normal(point[i].shape)
        hi, lo = list(point), list(point)
        hi[i], lo[i] = point[i] + e, point[i] - e  # each input alone is linear
        loss = [(ref.grouped(*z, offsets.numpy(), rows.numpy())[0] * _np(v_y)).sum()
                for z in (hi, lo)]
        tol = (bounds[i] * np.abs(e)).sum()
        assert abs((_np(grads[i]) * e).sum() - (loss[0] - loss[1]) / 2) <= tol, i


# ------------------------------------------------- streams, graphs, sizes --


def _all_operators(dtype):
    table, ids, v_out = _lookup_case(3000, 50, 64, dtype, 3)
    scan = _scan_case(1200, 64, "ragged", dtype, 4)
    grouped = _grouped_case(900, 64, 48, 6, dtype, 5, True)
    dev = [t.to(DEV) for t in (table, ids, v_out, *scan, *grouped)]

    def call():
        table, ids, v_out = dev[:3]
        out = [W.embedding_fwd(table, ids, 2.0), W.embedding_bwd(v_out, ids, 50, 2.0)]
        out += _run_scan(*dev[3:9], True)
        out += _run_grouped(*dev[9:])
        out += W.group_rows(ids, 50)
        return out

    return call


def test_operators_run_on_the_current_stream():
    call = _all_operators(torch.bfloat16)
    base = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(again, base):
        assert torch.equal(a, b)


def test_operators_replay_from_a_graph():
    call = _all_operators(torch.float16)
    base = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, base):
            assert torch.equal(a, b)
        call()  # eager work between the replays


def test_scan_beyond_32_bit_elements():
    n, d = 2 ** 25 + 300, 64  # 2^31 elements and some
    tail = 700
    x = torch.zeros(n, d, dtype=torch.float16, device=DEV)
    gate = torch.zeros(n, d, dtype=torch.float16, device=DEV)
    g = _gen(0)
    xt, gt = _randn(g, tail, d, dtype=torch.float16), _randn(g, tail, d, dtype=torch.float16)
    vt = _randn(g, tail, d, dtype=torch.float16)
    x[-tail:], gate[-tail:] = xt.to(DEV), gt.to(DEV)
    v_y = torch.zeros_like(x)
    v_y[-tail:] = vt.to(DEV)
    y, final, carries = W.gated_scan_fwd(x[None], gate[None])
    v_x, v_gate, _ = W.gated_scan_bwd(x[None], gate[None], None, None, carries, v_y[None])
    assert y[0, :-tail].abs().max() == 0
    small = _run_scan(xt, gt, torch.tensor([0, tail], dtype=torch.int32), None, vt, None, False)
    scan = ref.Scan(_np(xt), _np(gt), [0, tail])
    kappa = (2 * np.abs(_np(gt)).max() + 9) * U
    _close(y[0, -tail:], scan.h, kappa * scan.steps, torch.float16, "y")
    _close(final, scan.final, kappa * scan.final_steps, torch.float32, "final")
    for big, part in ((v_x, small[2]), (v_gate, small[3])):
        # The same formulas over tiles that begin elsewhere.
        err = (big[0, -tail:].float() - part.float()).abs()
        assert (err <= 2.0 ** -9 * part.float().abs() + 1e-5).all()


def test_lookup_and_grouped_beyond_32_bit_elements():
    n, d = 2 ** 25 + 77, 64
    ids = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    tail = torch.arange(50, device=DEV, dtype=torch.int32)
    ids[-50:] = tail
    table = torch.randn(64, d, device=DEV).to(torch.bfloat16)
    out = latent.embedding_lookup(table, ids)
    assert torch.equal(out[-50:], table[:50]) and out[-50 - 2 ** 16:-50].abs().sum() == 0
    grad = W.embedding_bwd(out, ids, 64)
    assert torch.equal(grad[:50], table[:50]) and grad[50:].abs().sum() == 0
    eye = torch.eye(d, device=DEV, dtype=torch.bfloat16)[None].expand(2, d, d).contiguous()
    rows, offsets = latent.group_rows((ids >= 0).to(torch.int32), 2)
    y = latent.grouped_matmul(out, eye, offsets, rows=rows)
    assert torch.equal(y[-2 ** 16:], out[-2 ** 16:])
    v_x, v_weight, _ = W.grouped_matmul_bwd(out, eye, offsets, rows, out)
    assert torch.equal(v_x[-2 ** 16:], out[-2 ** 16:])
    t = table[:50].double()
    assert v_weight[0].abs().sum() == 0
    assert ((v_weight[1].double() - t.T @ t).abs() <= 2.0 ** -8 * (t.T @ t).abs() + 1e-4).all()


# --------------------------------------------------------------- refusals --


def test_refusals():
    f = torch.zeros(4, 8, device=DEV)
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    off = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    x3 = f[None]
    w = torch.zeros(1, 6, 8, device=DEV)
    bad = [
        (lambda: W.embedding_fwd(f.cpu(), ids), "table must be a CUDA tensor"),
        (lambda: W.embedding_fwd(f.double(), ids), "not implemented for"),
        (lambda: W.embedding_fwd(f, ids.float()), "ids must be int32 or int64"),
        (lambda: W.embedding_fwd(f[0], ids), "table must be"),
        (lambda: W.embedding_bwd(f[:3], ids, 4), "v_out must be"),
        (lambda: W.embedding_bwd(f, ids, -1), "n_rows must not be negative"),
        (lambda: W.group_rows(f, 3), "ids must be"),
        (lambda: W.group_rows(ids, -1), "n_groups must not be negative"),
        (lambda: W.gated_scan_fwd(f, f), r"x must be \[B, L, D\]"),
        (lambda: W.gated_scan_fwd(x3, x3, None, off), r"x must be \[N, D\]"),
        (lambda: W.gated_scan_fwd(x3, x3.bfloat16()), "gate must be torch.float32"),
        (lambda: W.gated_scan_fwd(x3, x3[:, :2]), "gate must have the shape of x"),
        (lambda: W.gated_scan_fwd(x3, x3, f), "initial must be"),
        (lambda: W.gated_scan_fwd(x3, x3, f[:1].bfloat16()), "initial must be torch.float32"),
        (lambda: W.gated_scan_fwd(f, f, None, off.long()), "offsets must be torch.int32"),
        (lambda: W.gated_scan_fwd(f, f, None, off[:1]), "offsets name no sequence"),
        (lambda: W.gated_scan_bwd(x3, x3, None, None, f[:0], x3), "kept is not that"),
        (lambda: W.grouped_matmul_fwd(f, w[:, :, :7], None, off), "x must be"),
        (lambda: W.grouped_matmul_fwd(f, w.half(), None, off), "weight must be torch.float32"),
        (lambda: W.grouped_matmul_fwd(f, w, f, off), "bias must be"),
        (lambda: W.grouped_matmul_fwd(f, w, None, off[:1]), "offsets must be"),
        (lambda: W.grouped_matmul_fwd(f, w, None, off, off), "rows must be"),
        (lambda: W.grouped_matmul_bwd(f, w, off, None, f), "v_y must be"),
    ]
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()


# ------------------------------------------------------------ the decoder --


def test_decoder_fits_a_projection():
    """Operators, rasterizer, explicit backward and Adam in one loop: a decoder
    at its start leaves its base alone, and training brings its image closer to
    another scene's."""
    from r2splat import geometry, optim, scenes
    from r2splat.latent import LatentDecoder
    from r2splat.ops import explicit

    n, levels, width = 1500, 5, 24
    g = _gen(0)
    base = scenes.random_gaussians(n, g, -3.4, 0.3, extent=0.6).to(DEV)
    other = scenes.random_gaussians(n, g, -3.2, 0.3, extent=0.6).to(DEV)
    views, Ks = (t.to(DEV) for t in geometry.cone_beam_views([0.4], 48))
    codes = torch.randint(-1, 64, (n,), generator=g).to(DEV)
    rows, offsets = latent.group_rows(torch.randint(0, levels, (n,), generator=g).to(DEV), levels)
    decoder = LatentDecoder(64, levels, width, g).to(DEV)
    optimizer = optim.Adam(decoder.parameters(), lr=1e-2)

    def render(means, quats, scales, opacities):
        state = explicit.prepare_explicit_gaussians(quats, scales, opacities, scale_min=5e-4,
                                                    scale_max=1.0)
        return state, explicit.explicit_rasterize(state, means, views, Ks, img_w=48, img_h=48,
                                                  tile_size=16, eps2d=1e-8, radius_clip=3.0,
                                                  absgrad=True).image

    target = render(other.means, other.quats, other.raw_scales, other.raw_opacities)[1].detach()
    losses = []
    for _ in range(12):
        optimizer.zero_grad()
        raw = decoder(codes, rows, offsets)
        if not losses:
            assert raw.abs().max() == 0  # zero weights: the base itself
        leaves = decoder.leaves(base, raw)
        state, image = render(*leaves)
        loss = (image - target).square().mean()
        loss.backward()
        explicit.explicit_backward(state, *leaves)
        decoder.backward(raw, *leaves)
        optimizer.step()
        losses.append(loss.item())
    assert all(torch.isfinite(p).all() for p in decoder.parameters())
    assert losses[-1] < 0.9 * losses[0], losses


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_step_equals_its_general_form(dtype):
    g = _gen(3)
    x, gate = (_randn(g, 37, 50, dtype=dtype).to(DEV) for _ in range(2))
    state = _randn(g, 37, 50).to(DEV)
    wide = torch.cat([x, gate], 1)
    y, final = latent.gated_scan_step(wide[:, :50], wide[:, 50:], state)
    e_y, e_final, _ = W.gated_scan_fwd(x[:, None], gate[:, None], state)
    assert torch.equal(y, e_y[:, 0]) and torch.equal(final, e_final)
    x.requires_grad_(True)
    latent.gated_scan_step(x, gate, state)[1].sum().backward()
    assert torch.allclose(x.grad.float(), torch.sigmoid(-gate.float()).to(dtype).float(),
                          rtol=2 * ROUND[dtype], atol=1e-6)
    with pytest.raises(RuntimeError, match="state must be"):
        W.gated_scan_step(x.detach(), gate, state[:3])
