"""The latent decoder's operators at their edges, without a GPU."""

import pytest
import torch
from torch.autograd import forward_ad

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


def _plain_wrapper(monkeypatch):
    """ops.latent over stand-ins of its kernels that carry no derivative."""
    from r2splat.ops import latent

    class Plain:
        @staticmethod
        def embedding_fwd(table, ids, scale):
            return scale * table.detach()[ids]

        @staticmethod
        def gated_scan_fwd(x, gate, initial, offsets, reverse, keep=True):
            return x.detach().clone(), torch.zeros(x.shape[0], x.shape[-1]), torch.zeros(1)

        @staticmethod
        def gated_scan_step(x, gate, state):
            return x.detach().clone(), torch.zeros(x.shape)

        @staticmethod
        def grouped_matmul_fwd(x, weight, bias, offsets, rows):
            return x.detach() @ weight.detach()[0].T

    monkeypatch.setattr(latent, "W", Plain)
    return latent


def test_tangents_are_refused_rather_than_lost(monkeypatch):
    latent = _plain_wrapper(monkeypatch)
    t, ids = torch.randn(4, 4), torch.zeros(4, dtype=torch.int64)
    off = torch.tensor([0, 4], dtype=torch.int32)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(t, torch.ones(4, 4))
        calls = [lambda: latent.embedding_lookup(d, ids),
                 lambda: latent.gated_scan(d[None], t[None]),
                 lambda: latent.gated_scan(t[None], d[None]),
                 lambda: latent.gated_scan(t[None], t[None], d[:1]),
                 lambda: latent.gated_scan_step(t, d, t),
                 lambda: latent.grouped_matmul(d, t[None], off),
                 lambda: latent.grouped_matmul(t, d[None], off),
                 lambda: latent.grouped_matmul(t, t[None], off, bias=d[:1])]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward mode AD"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode AD"):
                call()  # no_grad leaves tangents alone
        # Inputs without one are taken as ever.
        assert latent.embedding_lookup(t, ids, 2.0).equal(2.0 * t[ids])
        assert latent.grouped_matmul(t, t[None], off).equal(t @ t.T)


def test_scan_step_needs_its_state_with_and_without_gradients(monkeypatch):
    latent = _plain_wrapper(monkeypatch)
    for wanted in (False, True):
        x = torch.randn(4, 4, requires_grad=wanted)
        with pytest.raises(RuntimeError, match="state must be given"):
            latent.gated_scan_step(x, x, None)
        y, _ = latent.gated_scan_step(x, x, torch.zeros(4, 4))
        assert y.shape == (4, 4)
