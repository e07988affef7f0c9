"""The latent decoder's operators at their edges: rows of one vector, states
that are not finite through long sequences, groups of one part and of many.
Same restatement and bounds as test_gpu_latent.py."""

import numpy as np
import pytest
import torch

from oracle import latent as ref
from r2splat.cuda import _lib, _ops
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent
from test_gpu_latent import (DEV, TYPES, U, _check_scan, _close, _lookup_case, _np, _run_scan,
                             _scan_case)
from test_gpu_latent_paths import _check_equal, _equal_case, _run_equal

pytestmark = pytest.mark.gpu


# Every width from one element to more than a vector, over several blocks of
# rows, into memory that holds NaNs: a row that is not written shows.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16, 17])
def test_lookup_writes_every_row(d, wide, dtype):
    n, v, scale = 5003, 37, 1.7
    table, ids, v_out = _lookup_case(n, v, d, dtype, n + d)
    t, i = table.to(DEV), ids.to(torch.int64 if wide else torch.int32).to(DEV)
    lib = _lib.load()
    out = torch.full((n, d), float("nan"), dtype=dtype, device=DEV)
    assert lib.r2s_embedding_fwd(t.data_ptr(), d, i.data_ptr(), int(wide), scale,
                                 _ops._LATENT_TYPES[dtype], n, v, d, out.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream) == 0
    exact = ref.lookup(_np(table), ids.numpy(), scale)
    _close(out, exact, 2 * U * np.abs(exact), dtype, "out")  # scale and product
    assert torch.equal(latent.embedding_lookup(t, i, scale), out)
    grad = W.embedding_bwd(v_out.to(DEV), i, v, scale)
    exact, mass, count = ref.lookup_grad(_np(v_out), ids.numpy(), v, scale)
    _close(grad, exact, (count[:, None] + 3) * U * mass, dtype, "v_table")


# Groups around the ends of a part of 128 rows: none, one and several parts in
# one call, and as many groups of two as the rows can fill.  The workspace is
# exactly as long as the query says; what follows it stays.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("routed", [False, True])
@pytest.mark.parametrize("want", ["both", "weight", "bias"])
@pytest.mark.parametrize("sizes", [
    [0, 1, 127, 128, 129, 0, 255, 256, 257, 385, 2, 0], [129] * 20, [0] * 70 + [300] + [0] * 70,
    [128] * 9 + [129], [3] * 130])
def test_grouped_parts_of_ragged_groups(sizes, want, routed, dtype):
    n, e, k, m = sum(sizes) + 5, len(sizes), 40, 24
    g = torch.Generator().manual_seed(e)
    x, v_y = (torch.randn(n, d, generator=g).to(dtype) for d in (k, m))
    weight = torch.zeros(e, m, k, dtype=dtype)
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    rows = torch.randperm(n, generator=g) if routed else None
    r = None if rows is None else rows.numpy()
    _, (e_w, m_w), (e_b, m_b), count = ref.grouped_grad(_np(x), _np(weight), offsets, r, _np(v_y))
    lib, code = _lib.load(), _ops._LATENT_TYPES[dtype]
    need = lib.r2s_grouped_matmul_bwd_workspace_bytes(n, k, m, e, code, want != "bias")
    ws = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device=DEV)
    v_weight = torch.full((e, m, k), float("nan"), dtype=dtype, device=DEV)
    v_bias = torch.full((e, m), float("nan"), dtype=dtype, device=DEV)
    on = [t.to(DEV) for t in (x, v_y, torch.from_numpy(offsets).int())]
    order = None if rows is None else rows.int().to(DEV)
    assert lib.r2s_grouped_matmul_bwd(
        on[0].data_ptr(), k, None, on[2].data_ptr(), None if order is None else order.data_ptr(),
        on[1].data_ptr(), m, n, k, m, e, code, None,
        None if want == "bias" else v_weight.data_ptr(),
        None if want == "weight" else v_bias.data_ptr(), ws.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (ws[need:] == 0xAB).all()
    if want != "bias":
        _close(v_weight, e_w, (count[:, None, None] + 2) * U * m_w, dtype, "v_weight")
    if want != "weight":
        _close(v_bias, e_b, (count[:, None] + 2) * U * m_b, dtype, "v_bias")


# A state that is not finite stays so to its sequence's end, however small the
# product of the gates after it gets, whatever form the launch takes, until a
# gate forgets it; its gradient, the other way, likewise.
def _spoil(x, gate, v_y, seed):
    g = torch.Generator().manual_seed(seed)
    n, d = x.shape
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t in (x, v_y):
            t[torch.randint(0, n, (3,), generator=g), torch.randint(0, d, (3,), generator=g)] = bad
    gate[torch.rand(n, d, generator=g) < 1.0 / 900.0] = -float("inf")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("n,d,kind", [(6000, 10, "one"), (9000, 64, "one"), (7000, 33, "ragged"),
                                      (5000, 130, "one")])
def test_scan_keeps_what_is_not_finite(n, d, kind, reverse, dtype):
    x, gate, offsets, initial, v_y, v_final = _scan_case(n, d, kind, dtype, n + d)
    _spoil(x, gate, v_y, d)
    case = (x, gate, offsets, initial, v_y, v_final)
    _check_scan(*case, reverse, _run_scan(*case, reverse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("b,l,d", [(192, 600, 6), (1, 3000, 5), (2, 5000, 70)])
def test_scan_of_equal_sequences_keeps_what_is_not_finite(b, l, d, reverse, dtype):
    x, gate, initial, v_y, v_final = _equal_case(b, l, d, dtype, b + l + d)
    _spoil(x.view(b * l, d), gate.view(b * l, d), v_y.view(b * l, d), l)
    case = (x, gate, initial, v_y, v_final)
    _check_equal(case, reverse, _run_equal(*case, reverse))


def test_scan_ends_as_its_steps_do_after_a_nan():
    x, gate = torch.ones(3, 900, 8, device=DEV), torch.full((3, 900, 8), -1.0, device=DEV)
    x[1, 4], x[2, 4] = float("nan"), float("inf")
    _, final = latent.gated_scan(x, gate)
    state = torch.zeros(3, 8, device=DEV)
    for t in range(900):
        _, state = latent.gated_scan_step(x[:, t], gate[:, t], state)
    assert torch.isnan(final[1]).all() and torch.isinf(final[2]).all()
    assert torch.isnan(state[1]).all() and torch.isinf(state[2]).all()
    assert torch.isfinite(final[0]).all()
