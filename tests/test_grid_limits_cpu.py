"""Sizes that a launch's grid (fewer than 2^32 threads along a side) does not take, by
the C entries' refusals: no device is touched."""

import ctypes

import pytest

from r2splat.cuda import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_adamw_of_more_elements_than_a_grid_holds(lib):
    t = _lib.AdamwTensor(param=256, grad=256, exp_avg=256, second=256,
                         n=(2 ** 32 // 256 - 1) * 4096 + 1)
    assert lib.r2s_adamw_step(ctypes.byref(t), 1, None) == 1002
    assert b"tensor 0 is too large: more than 68719472640 elements" in lib.r2s_last_error()


FAKE = ctypes.c_void_p(4096)  # never dereferenced: the checks fail first
LARGE = 1 << 60  # bytes that a workspace is said to have


def _refused(lib, rc, message):
    assert rc == 1002 and message in lib.r2s_last_error(), (rc, lib.r2s_last_error())


def test_lookups_of_more_rows_than_a_grid_holds(lib):
    """A block to a row of 16 KB; 16 lanes to a row of the table's gradient."""
    rc = lib.r2s_embedding_fwd(FAKE, 4096, FAKE, 0, 1.0, 0, 1 << 24, 100, 4096, FAKE, None)
    _refused(lib, rc, b"output too large")
    for n, n_rows, width in ((0, 1 << 28, 33), (1 << 20, (1 << 31) - 2, 5)):
        rc = lib.r2s_embedding_bwd(FAKE, width, FAKE, 0, 1.0, 0, n, n_rows, width, FAKE, FAKE, LARGE,
                                   None)
        _refused(lib, rc, b"2^32 threads")


def test_scans_of_more_states_than_a_grid_holds(lib):
    def fwd(sequences, length, width, type_=0, ragged=False, n=None):
        return lib.r2s_gated_scan_fwd(
            FAKE, width, FAKE, width, None, FAKE if ragged else None, sequences, length,
            sequences * length if n is None else n, width, type_, 0, FAKE, FAKE, FAKE, FAKE, LARGE,
            None)

    _refused(lib, fwd(1 << 25, 1, 128), b"too many tokens")        # a step, a thread an element
    _refused(lib, fwd(1 << 25, 2, 128), b"too many tokens")        # a thread a channel
    _refused(lib, fwd((1 << 26) + 1, 0, 64), b"more states")       # sequences without a token
    _refused(lib, fwd((1 << 26) + 1, 0, 64, ragged=True, n=1000), b"more states")
    rc = lib.r2s_gated_scan_bwd(FAKE, 128, FAKE, 128, None, None, FAKE, FAKE, 128, None, 1 << 25, 2,
                                1 << 26, 128, 0, 0, FAKE, FAKE, FAKE, FAKE, LARGE, None)
    _refused(lib, rc, b"too many tokens")


def test_grouped_products_of_more_tiles_than_a_grid_holds(lib):
    n = (1 << 31) - 1  # 2^24 tiles of 128 rows
    rc = lib.r2s_grouped_matmul_fwd(FAKE, 1, FAKE, None, FAKE, None, n, 1, 1, 3, 0, FAKE, None)
    _refused(lib, rc, b"too many tiles")
    rc = lib.r2s_grouped_matmul_bwd(FAKE, 1, FAKE, FAKE, None, FAKE, 1, n, 1, 1, 3, 0, FAKE, None,
                                    None, FAKE, LARGE, None)
    _refused(lib, rc, b"too many tiles")
