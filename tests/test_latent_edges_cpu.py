"""The latent decoder's operators at their edges, without a GPU."""

import pytest

from r2splat.cuda import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_grouped_workspace_does_not_grow_with_the_groups(lib):
    size = lib.r2s_grouped_matmul_bwd_workspace_bytes
    # 4096 rows cannot fill more than a few parts of groups that have several,
    # whatever the number of groups: 16 MiB of float32 each.
    slab = 4 * 2048 * 2048
    assert size(4096, 2048, 2048, 256, _lib.TYPE_BF16, 1) <= 10 * slab
    assert size(4096, 2048, 2048, 65535, _lib.TYPE_BF16, 1) <= 10 * slab
    # Fewer rows than a part: no group has two.
    for kind in (_lib.TYPE_F32, _lib.TYPE_BF16, _lib.TYPE_F16):
        assert size(100, 2048, 2048, 1000, kind, 1) <= 1 << 16
        assert size(0, 2048, 2048, 1000, kind, 1) <= 1 << 16
    # Parts of a row of the bias alone where the weights' gradient is not wanted.
    assert size(1 << 20, 1024, 1024, 64, _lib.TYPE_BF16, 0) <= 1 << 22
    assert size(1 << 20, 1024, 1024, 64, _lib.TYPE_BF16, 1) > 1 << 28
    assert size(10, 8, 8, 2, 7, 1) == 0 and size(-1, 8, 8, 2, 0, 1) == 0
