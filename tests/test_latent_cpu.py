"""The latent decoder's operators without a GPU: the C ABI's refusals, which
come before any device is touched, the float64 restatement against plain
formulas and differences, and the import contract."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import latent as ref
from r2splat.cuda import _lib

FAKE = ctypes.c_void_p(256)  # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _refused(lib, rc, code, message):
    assert rc == code and message in lib.r2s_last_error(), lib.r2s_last_error()


def test_group_rows_arguments(lib):
    _refused(lib, lib.r2s_group_rows(FAKE, 0, -1, 3, FAKE, FAKE, None, 0, None), 1001, b"negative")
    _refused(lib, lib.r2s_group_rows(FAKE, 0, 1 << 31, 3, FAKE, FAKE, None, 0, None), 1002,
             b"2^31 - 1")
    _refused(lib, lib.r2s_group_rows(None, 0, 5, 3, FAKE, FAKE, FAKE, 1 << 20, None), 1001,
             b"null ids")
    _refused(lib, lib.r2s_group_rows(FAKE, 0, 5, 3, FAKE, FAKE, None, 0, None), 1004,
             b"workspace")
    assert lib.r2s_group_rows_workspace_bytes(0, 3) == 0
    small = lib.r2s_group_rows_workspace_bytes(1000, 100)
    # More than 511 groups take two passes and a pair of buffers.
    assert 0 < small < lib.r2s_group_rows_workspace_bytes(1000, 600) \
        and lib.r2s_group_rows_workspace_bytes(1 << 20, 600) >= 12 * (1 << 20)


def test_embedding_arguments(lib):
    fwd, bwd = lib.r2s_embedding_fwd, lib.r2s_embedding_bwd
    _refused(lib, fwd(FAKE, 8, FAKE, 0, 1.0, 7, 4, 4, 8, FAKE, None), 1001, b"element type 7")
    _refused(lib, fwd(FAKE, 7, FAKE, 0, 1.0, 0, 4, 4, 8, FAKE, None), 1001, b"row stride")
    _refused(lib, fwd(FAKE, 8, None, 0, 1.0, 0, 4, 4, 8, FAKE, None), 1001, b"null ids")
    _refused(lib, fwd(None, 8, FAKE, 0, 1.0, 0, 4, 4, 8, FAKE, None), 1001, b"null table")
    _refused(lib, fwd(FAKE, 8, FAKE, 0, 1.0, 0, 4, -4, 8, FAKE, None), 1001, b"negative")
    _refused(lib, fwd(FAKE, 8, FAKE, 0, 1.0, 0, 1 << 31, 4, 8, FAKE, None), 1002, b"2^31 - 1")
    assert fwd(None, 8, None, 0, 1.0, 0, 0, 4, 8, None, None) == 0  # nothing to do
    _refused(lib, bwd(FAKE, 8, FAKE, 0, 1.0, 0, 4, 4, 8, FAKE, None, 0, None), 1004, b"workspace")
    _refused(lib, bwd(FAKE, 8, FAKE, 0, 1.0, 0, 4, 4, 8, None, FAKE, 1 << 20, None), 1001,
             b"null gradient")
    assert bwd(FAKE, 8, FAKE, 0, 1.0, 0, 4, 0, 8, None, None, 0, None) == 0


def test_gated_scan_arguments(lib):
    def fwd(x=FAKE, xs=8, offsets=None, s=2, length=5, n=10, d=8, kind=0, final=FAKE, ws=None,
            size=0):
        return lib.r2s_gated_scan_fwd(x, xs, FAKE, 8, None, offsets, s, length, n, d, kind, 0,
                                      FAKE, final, FAKE, ws, size, None)

    _refused(lib, fwd(kind=3), 1001, b"element type")
    _refused(lib, fwd(n=11), 1001, b"11 tokens are not 2 sequences of 5")
    _refused(lib, fwd(s=-1), 1001, b"negative")
    _refused(lib, fwd(xs=7), 1001, b"rows overlap")
    _refused(lib, fwd(offsets=FAKE, s=0), 1001, b"without a sequence")
    _refused(lib, fwd(final=None), 1001, b"null final")
    _refused(lib, fwd(x=None), 1001, b"null tokens")
    _refused(lib, fwd(n=1 << 31, length=1 << 30), 1002, b"tokens")
    _refused(lib, fwd(xs=1 << 40, length=1000, n=2000), 1002, b"too far apart")
    _refused(lib, fwd(x=ctypes.c_void_p(258), kind=1), 1001, b"multiples of 4 bytes")
    # A ragged call beyond one block's reach goes through maps in a workspace.
    assert lib.r2s_gated_scan_workspace_bytes(0, 1, 4, 0, 100_000, 64) > 0
    _refused(lib, fwd(offsets=FAKE, s=4, n=100_000), 1004, b"workspace")
    assert fwd(s=0, n=0) == 0 and fwd(d=0) == 0
    # Kept states: one for each eight tokens of a strip.
    assert lib.r2s_gated_scan_kept_rows(0, 0, 8, 4096, 8 * 4096, 1024) >= 8 * 4096 // 8
    rc = lib.r2s_gated_scan_bwd(FAKE, 8, FAKE, 8, None, None, None, FAKE, 8, None, 2, 5, 10, 8, 0,
                                0, FAKE, FAKE, None, None, 0, None)
    _refused(lib, rc, 1001, b"kept states")


def test_grouped_matmul_arguments(lib):
    def fwd(x=FAKE, xs=8, w=FAKE, offsets=FAKE, n=4, k=8, m=8, e=2, kind=0, y=FAKE):
        return lib.r2s_grouped_matmul_fwd(x, xs, w, None, offsets, None, n, k, m, e, kind, y, None)

    _refused(lib, fwd(kind=-1), 1001, b"element type")
    _refused(lib, fwd(offsets=None), 1001, b"null offsets")
    _refused(lib, fwd(xs=7), 1001, b"rows overlap")
    _refused(lib, fwd(w=None), 1001, b"null input, weight or output")
    _refused(lib, fwd(k=-1), 1001, b"negative")
    _refused(lib, fwd(e=65536), 1002, b"65535 groups")
    assert fwd(n=0) == 0 and fwd(m=0) == 0
    bwd = lib.r2s_grouped_matmul_bwd
    rc = bwd(FAKE, 8, FAKE, FAKE, None, FAKE, 8, 4, 8, 8, 2, 0, None, FAKE, None, None, 0, None)
    _refused(lib, rc, 1004, b"workspace")
    rc = bwd(FAKE, 8, FAKE, FAKE, None, FAKE, 7, 4, 8, 8, 2, 0, None, FAKE, None, None, 0, None)
    _refused(lib, rc, 1001, b"rows overlap")
    assert bwd(FAKE, 8, FAKE, FAKE, None, FAKE, 8, 4, 8, 8, 2, 0, None, None, None, None, 0,
               None) == 0  # no gradient wanted


def test_restatement_against_torch():
    g = torch.Generator().manual_seed(0)
    table = torch.randn(9, 5, generator=g, dtype=torch.float64)
    ids = torch.randint(0, 9, (40,), generator=g)
    v = torch.randn(40, 5, generator=g, dtype=torch.float64)
    t = table.clone().requires_grad_(True)
    out = 0.3 * t[ids]
    out.backward(v)
    assert np.allclose(ref.lookup(table.numpy(), ids.numpy(), 0.3), out.detach().numpy())
    assert np.allclose(ref.lookup_grad(v.numpy(), ids.numpy(), 9, 0.3)[0], t.grad.numpy())

    x, gate = (torch.randn(30, 4, generator=g, dtype=torch.float64).requires_grad_(True)
               for _ in range(2))
    initial = torch.randn(3, 4, generator=g, dtype=torch.float64).requires_grad_(True)
    bounds = [0, 11, 11, 30]
    v_y = torch.randn(30, 4, generator=g, dtype=torch.float64)
    v_final = torch.randn(3, 4, generator=g, dtype=torch.float64)
    for reverse in (False, True):
        ys, finals = [None] * 30, []
        for q in range(3):
            h = initial[q]
            order = range(bounds[q], bounds[q + 1])
            for i in (reversed(order) if reverse else order):
                a = torch.sigmoid(gate[i])
                h = a * h + (1 - a) * x[i]
                ys[i] = h
            finals.append(h)
        y, final = torch.stack(ys), torch.stack(finals)
        grads = torch.autograd.grad((y * v_y).sum() + (final * v_final).sum(), (x, gate, initial))
        scan = ref.Scan(x.detach().numpy(), gate.detach().numpy(), bounds,
                        initial.detach().numpy(), reverse)
        assert np.allclose(scan.h, y.detach().numpy())
        assert np.allclose(scan.final, final.detach().numpy())
        for mine, theirs in zip(scan.grad(v_y.numpy(), v_final.numpy()), grads):
            assert np.allclose(mine, theirs.numpy())

    x = torch.randn(20, 6, generator=g, dtype=torch.float64).requires_grad_(True)
    w = torch.randn(4, 3, 6, generator=g, dtype=torch.float64).requires_grad_(True)
    b = torch.randn(4, 3, generator=g, dtype=torch.float64).requires_grad_(True)
    ids = torch.randint(0, 4, (20,), generator=g)
    rows, offsets = ref.groups(ids.numpy(), 4)
    y = torch.stack([w[e] @ x[i] + b[e] for i, e in enumerate(ids.tolist())])
    v = torch.randn(20, 3, generator=g, dtype=torch.float64)
    grads = torch.autograd.grad((y * v).sum(), (x, w, b))
    args = [t.detach().numpy() for t in (x, w)]
    assert np.allclose(ref.grouped(*args, b.detach().numpy(), offsets, rows)[0],
                       y.detach().numpy())
    for mine, theirs in zip(ref.grouped_grad(*args, offsets, rows, v.numpy())[:3], grads):
        assert np.allclose(mine[0], theirs.numpy())


def test_modules_import_without_the_library():
    from r2splat import latent as model
    from r2splat.cuda import _wrapper
    from r2splat.ops import latent

    for name in latent.__all__:
        assert callable(getattr(latent, name))
    for name in ("group_rows", "embedding_fwd", "embedding_bwd", "gated_scan_fwd",
                 "gated_scan_step", "gated_scan_bwd", "grouped_matmul_fwd", "grouped_matmul_bwd"):
        assert callable(getattr(_wrapper, name))
    decoder = model.LatentDecoder(10, 3, 16)
    assert sum(p.numel() for p in decoder.parameters()) == 2 * 160 + 3 * 11 * 17
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="unavailable"):
            latent.embedding_lookup(torch.zeros(2, 2), torch.zeros(1, dtype=torch.int64))
