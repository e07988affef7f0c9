"""The latent decoder's operators at sizes where a launch takes another form:
scans in rounds, wide lane groups, chunks with many sequences, product tiles of
both widths, weights' gradients in parts, short and long lists of ids.  Same
restatement and bounds as test_gpu_latent.py."""

import numpy as np
import pytest
import torch

from oracle import latent as ref
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent
from test_gpu_latent import (DEV, TYPES, _check_grouped, _check_scan, _gen, _grouped_case, _randn,
                             _run_grouped, _run_scan, _scan_case)

pytestmark = pytest.mark.gpu


def _equal_case(b, l, d, dtype, seed):
    g = _gen(seed)
    x, gate = _randn(g, b, l, d, dtype=dtype), _randn(g, b, l, d, dtype=dtype, scale=1.5, shift=1.0)
    return x, gate, _randn(g, b, d), _randn(g, b, l, d, dtype=dtype), _randn(g, b, d)


def _run_equal(x, gate, initial, v_y, v_final, reverse):
    b, l, d = x.shape
    x, gate, initial, v_y, v_final = (t.to(DEV) for t in (x, gate, initial, v_y, v_final))
    y, final, kept = W.gated_scan_fwd(x, gate, initial, None, reverse)
    v_x, v_gate, v_initial = W.gated_scan_bwd(x, gate, initial, None, kept, v_y, v_final, reverse)
    flat = lambda t: t.reshape(b * l, d)  # noqa: E731
    return flat(y), final, flat(v_x), flat(v_gate), v_initial


def _check_equal(case, reverse, got):
    x, gate, initial, v_y, v_final = case
    b, l, d = x.shape
    flat = lambda t: t.reshape(b * l, d)  # noqa: E731
    _check_scan(flat(x), flat(gate), torch.arange(0, b * l + 1, l), initial, flat(v_y), v_final,
                reverse, got)


# A block per sequence with 64 and 128 bytes of a row, one round and several,
# lengths that end inside a chunk, and all of a few sequences in one block.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("b,l,d", [(200, 131, 17), (260, 137, 33), (24, 1100, 130), (3, 300, 6),
                                   (1, 129, 1)])
def test_scan_in_rounds(b, l, d, reverse, dtype):
    case = _equal_case(b, l, d, dtype, b + l + d)
    _check_equal(case, reverse, _run_equal(*case, reverse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_in_rounds_holds_and_forgets(reverse, dtype):
    case = list(_equal_case(192, 290, 16, dtype, 5))
    g = _gen(6)
    hold, forget = (torch.rand(case[0].shape, generator=g) < r for r in (0.2, 0.1))
    case[1][forget] = float("-inf")
    case[1][hold] = float("inf")
    got = _run_equal(*case, reverse)
    _check_equal(case, reverse, got)
    case[0] = case[0].clone()
    case[0][hold] = float("nan")
    again = _run_equal(*case, reverse)
    assert all(torch.equal(again[i], got[i]) for i in (0, 1, 2))


# Bits do not depend on the sequence's place, its neighbours or the run.
def test_scan_in_rounds_is_the_same_for_equal_inputs():
    x, gate, initial, v_y, v_final = _equal_case(1, 517, 40, torch.float32, 9)
    many = [t.expand(250, *t.shape[1:]).contiguous() for t in (x, gate, initial, v_y, v_final)]
    a, b = (_run_equal(*many, False) for _ in range(2))
    for u, v in zip(a, b):
        assert torch.equal(u, v)
        rows = u.reshape(250, -1)
        assert torch.equal(rows, rows[:1].expand_as(rows))


# More sequences in a chunk of eight tokens than its lanes look at together,
# most of them empty, in narrow and wide rows.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("d", [1, 2, 9, 64, 128, 200])
def test_scan_of_many_empty_sequences(d, reverse, dtype):
    n = 333
    x, gate, _, _, v_y, _ = _scan_case(n, d, "one", dtype, d)
    bounds = [0] * 40 + [1] * 30 + [2, 3, 3, 3, 9] + [50] * 100 + [51, 58] + [200] * 17 + [n] * 33
    s = len(bounds) - 1
    g = _gen(7)
    case = (x, gate, torch.tensor(bounds, dtype=torch.int32), _randn(g, s, d), v_y,
            _randn(g, s, d))
    _check_scan(*case, reverse, _run_scan(*case, reverse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("n,d", [(4000, 127), (2500, 260)])
def test_scan_of_ragged_wide_rows(n, d, reverse, dtype):
    case = _scan_case(n, d, "ragged", dtype, n + d)
    _check_scan(*case, reverse, _run_scan(*case, reverse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("b,l,d", [(40, 17, 256), (20, 128, 70), (9, 8, 64)])
def test_scan_of_short_equal_sequences(b, l, d, reverse, dtype):
    case = _equal_case(b, l, d, dtype, b + l + d)
    _check_equal(case, reverse, _run_equal(*case, reverse))


# Tiles of 128 columns (enough groups for 385 blocks), and weights' gradients of
# many tiles whose groups are cut into parts.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("routed", [False, True])
@pytest.mark.parametrize("n,k,m,e", [(1200, 72, 130, 300), (1200, 130, 70, 400),
                                     (1700, 300, 390, 2), (1100, 264, 136, 1)])
def test_grouped_tiles_and_parts(n, k, m, e, routed, dtype):
    case = _grouped_case(n, k, m, e, dtype, n + k + m + e, routed)
    _check_grouped(case, _run_grouped(*case))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n,groups", [(2048, 5), (2049, 5), (2047, 30_000), (2000, 40_000),
                                      (31, 200_000), (32, 0), (33, 1), (4096, 4000),
                                      (4097, 4000), (4000, 20_000)])
def test_group_rows_of_short_lists(n, groups, wide):
    ids = torch.randint(-2, max(groups + 2, 1), (n,), generator=_gen(n + groups))
    ids[n // 2:] = ids[:n - n // 2].flip(0)  # equal ids far apart
    ids = ids.to(torch.int64 if wide else torch.int32)
    rows, offsets = latent.group_rows(ids.to(DEV), groups)
    e_rows, e_offsets = ref.groups(ids.numpy().astype(np.int64), groups)
    assert np.array_equal(rows.cpu().numpy(), e_rows)
    assert np.array_equal(offsets.cpu().numpy(), e_offsets)
