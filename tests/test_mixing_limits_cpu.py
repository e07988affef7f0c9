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
