"""Rotary positions and the norms around a block on the GPU against float64.

Tolerances come with the values: oracle.mixing bounds the error of any float32
evaluation of the same expressions, operation by operation; the output's own
rounding is added here.
"""

import numpy as np
import pytest
import torch

from oracle import mixing as ref
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _cuda(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _close(got, exact, bound, dtype, what):
    got = _np(got)
    assert got.shape == exact.shape, what
    # A rounding is off by half a step, relative to the value that is rounded.
    tol = bound + HALF[dtype] * (np.abs(exact) + bound) + TINY[dtype]
    bad = ~(np.abs(got - exact) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], exact[bad][:4])


# ---------------------------------------------------------------- rotary --


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,h,hk,d,sections,interleaved,shared", [
    (1, 1, 0, 2, (1,), False, False), (1, 8, 2, 64, (32,), False, False),
    (37, 3, 3, 33, (5, 6, 5), True, False), (130, 2, 1, 64, (10, 11, 9), False, True),
    (2500, 5, 5, 16, (2, 0, 3), False, False), (1025, 1, 1, 7, (1, 1, 1), True, True),
    (64, 17, 1, 130, (20, 21, 22), True, False), (9, 2, 2, 512, (256,), False, False),
    (300, 4, 2, 24, (0, 0), False, False)])
def test_rotary(n, h, hk, d, sections, interleaved, shared, dtype):
    g = _gen(n + d)
    q, k = _randn(g, n, h, d, dtype=dtype), _randn(g, n, hk, d, dtype=dtype) if hk else None
    axes = len(sections)
    kinds = [torch.randint(-(2 ** 20), 2 ** 20, (n, axes), generator=g),
             torch.randint(0, 2 ** 31, (n, axes), generator=g, dtype=torch.int64),
             torch.randint(-5, 500, (n, axes), generator=g, dtype=torch.int32),
             _randn(g, n, axes, scale=1000.0)]
    for positions in kinds:
        got = latent.rotary_axes(*_cuda(q, k, positions), sections, 1000.0, interleaved, shared)
        back = W.rotary_axes(*_cuda(q, k, positions), sections, 1000.0, interleaved, shared, True)
        for x, y, z in zip((q, k), got, back):
            if x is None:
                assert y is None and z is None
                continue
            for out, inverse in ((y, False), (z, True)):
                exact, bound = ref.rotary(_np(x), positions.numpy(), sections, 1000.0,
                                          interleaved, shared, inverse)
                _close(out, exact, bound, dtype, (positions.dtype, inverse))
                rest = 2 * sum(sections)
                assert torch.equal(out[..., rest:].cpu(), x[..., rest:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_strides_gradients_and_empty(dtype):
    g = _gen(3)
    # Slices of one projection, and heads before tokens.
    fused = _randn(g, 50, 3, 4, 20, dtype=dtype).to(DEV)
    positions = _randn(g, 50, 2, scale=30.0).to(DEV)
    swapped = fused[:, 1].transpose(0, 1).contiguous().transpose(0, 1)
    odd = fused[..., 1:18][:, 0]  # a head of 17 at odd elements
    want = latent.rotary_axes(fused[:, 0].contiguous(), fused[:, 1].contiguous(), positions, (4, 6))
    for q, k in ((fused[:, 0], fused[:, 1]), (fused[:, 0], swapped)):
        for a, b in zip(latent.rotary_axes(q, k, positions, (4, 6)), want):
            assert torch.equal(a, b)
    a, _ = latent.rotary_axes(odd, None, positions, (3, 5))
    assert torch.equal(a, latent.rotary_axes(odd.contiguous(), None, positions, (3, 5))[0])
    every = fused[:1, 0].expand(50, 4, 20)  # one token's heads, turned to 50 places
    assert torch.equal(latent.rotary_axes(every, None, positions, (4, 6))[0],
                       latent.rotary_axes(every.contiguous(), None, positions, (4, 6))[0])
    # Batches, and gradients by the turn back.
    q, k = (fused[:, i].reshape(5, 10, 4, 20).detach().requires_grad_(True) for i in (0, 1))
    p = positions.reshape(5, 10, 2)
    out = latent.rotary_axes(q, k, p, (4, 6))
    assert torch.equal(out[0].reshape(50, 4, 20), want[0])
    v = [torch.randn_like(t) for t in out]
    grads = torch.autograd.grad(out, (q, k), v)
    for a, b in zip(grads, W.rotary_axes(*v, p, (4, 6), inverse=True)):
        assert torch.equal(a, b)
    out = latent.rotary_axes(q, k, p, (4, 6))
    (only,) = torch.autograd.grad(out[1], (k,), v[1])
    assert torch.equal(only, grads[1])
    alone, none = latent.rotary_axes(q, None, p, (4, 6))
    assert none is None
    (only,) = torch.autograd.grad(alone, (q,), v[0])
    assert torch.equal(only, grads[0])
    # Turning is linear: <turn(q), v> = <q, turn back(v)>.
    if dtype == torch.float32:
        left = float((out[0].detach() * v[0]).sum())
        right = float((q.detach() * grads[0]).sum())
        mass = float((q.detach().abs() * v[0].abs()).sum()) * 2
        assert abs(left - right) <= 1100 * 2.0 ** -23 * mass
    for shape in ((0, 4, 20), (5, 0, 20)):
        e = torch.empty(shape, dtype=dtype, device=DEV)
        out, none = latent.rotary_axes(e, None, positions[:shape[0]], (4, 6))
        assert out.shape == shape and none is None


def test_rotary_positions_that_are_not_finite_stay_in_their_token():
    q = torch.randn(6, 2, 8, device=DEV)
    p = torch.zeros(6, 1, device=DEV)
    p[2], p[4] = float("inf"), float("nan")
    out, _ = latent.rotary_axes(q, None, p, (4,))
    assert torch.isnan(out[[2, 4]]).all() and torch.equal(out[[0, 1, 3, 5]], q[[0, 1, 3, 5]])


# ----------------------------------------------------------------- norms --


def _norm_case(n, d, gate, dtype, seed, normed=True, following=True):
    g = _gen(seed)
    x, update = _randn(g, n, d, dtype=dtype), _randn(g, n, d, shift=0.5, scale=2.0, dtype=dtype)
    shape = {"rows": (n, d), "channels": (d,), "none": None}[gate]
    gate = None if shape is None else _randn(g, *shape, scale=3.0, dtype=dtype)
    w1 = _randn(g, d, dtype=dtype) if normed else None
    w2 = _randn(g, d, dtype=dtype) if following else None
    return x, update, gate, w1, w2, _randn(g, n, d, dtype=dtype), _randn(g, n, d, dtype=dtype)


NAMES = ("v_x", "v_update", "v_gate", "v_w1", "v_w2")


def _check_norm(case, scale, eps, centered, dtype):
    x, update, gate, w1, w2, v_y, v_u = case
    if w2 is None:
        v_u = None
    exact = ref.residual_norm(*(_np(t) for t in (x, update, gate, w1, w2, v_y, v_u)), scale, eps,
                              centered)
    dev = _cuda(x, update, gate, w1, w2)
    y, u = W.residual_norm_fwd(*dev, scale, eps, centered)
    grads = W.residual_norm_bwd(*dev, *_cuda(v_y, v_u), scale, eps, centered)
    found = dict(zip(NAMES, grads), u=u, y=y if update is not None else None)
    for name, got in found.items():
        if name not in exact:
            assert got is None, name
            continue
        _close(got, exact[name].v, exact[name].e, dtype, name)
    return dev, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (5, 3), (300, 45), (1000, 64), (77, 129), (40, 513),
                                 (33, 1024), (20, 1500), (9, 2600), (5, 8192), (3, 4097)])
def test_residual_norm(n, d, dtype):
    for i, gate in enumerate(("rows", "channels", "none")):
        _check_norm(_norm_case(n, d, gate, dtype, n + d + i), 0.7, 1e-6, bool(i % 2), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_residual_norm_without_parts(dtype):
    case = _norm_case(70, 50, "rows", dtype, 1, normed=False)
    _check_norm(case, -1.5, 1e-5, False, dtype)
    _check_norm(_norm_case(70, 50, "channels", dtype, 2, following=False), 1.0, 1e-5, True, dtype)
    _check_norm(_norm_case(70, 50, "none", dtype, 3, normed=False, following=False), 2.0, 1e-5,
                False, dtype)
    x, *_, w2, v_y, v_u = _norm_case(70, 50, "none", dtype, 4)
    for centered in (False, True):
        _check_norm((x, None, None, None, w2, v_y, v_u), 1.0, 1e-5, centered, dtype)
        exact = ref.residual_norm(_np(x), None, None, None, _np(w2), None, None, 1.0, 1e-5,
                                  centered)["u"]
        _close(latent.pre_norm(x.to(DEV), w2.to(DEV), 1e-5, centered), exact.v, exact.e, dtype, "u")


def test_residual_norm_many_rows_and_the_same_bits():
    """More rows than lane groups: sums over rows in a fixed order."""
    case = _norm_case(60_001, 40, "channels", torch.float32, 5)
    dev, grads = _check_norm(case, 0.5, 1e-6, True, torch.float32)
    again = W.residual_norm_bwd(*dev, *_cuda(*case[5:]), 0.5, 1e-6, True)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_residual_norm_gradients_through_autograd_and_differences():
    dtype = torch.float32
    x, update, gate, w1, w2, v_y, v_u = _norm_case(6, 10, "channels", dtype, 6)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, update, gate, w1, w2)]
    # Batches, and rows that are not dense.
    wide = torch.zeros(2, 3, 16, device=DEV)
    wide[..., :10] = x.to(DEV).reshape(2, 3, 10)
    batched = wide[..., :10].detach().requires_grad_(True)
    y, u = latent.residual_norm(batched, leaves[1].reshape(2, 3, 10), *leaves[2:], scale=0.7)
    total = (y * v_y.to(DEV).reshape(2, 3, 10)).sum() + (u * v_u.to(DEV).reshape(2, 3, 10)).sum()
    grads = torch.autograd.grad(total, [batched, *leaves[1:]])
    direct = W.residual_norm_bwd(*(t.detach() for t in leaves), *_cuda(v_y, v_u), 0.7)
    for a, b in zip(grads, direct):
        assert torch.equal(a.reshape(b.shape), b)

    def value(*args):
        out = ref.residual_norm(*args, _np(v_y), _np(v_u), 0.7, 1e-6, False)
        return (out["y"].v * _np(v_y)).sum() + (out["u"].v * _np(v_u)).sum()

    args = [_np(t) for t in (x, update, gate, w1, w2)]
    for which, grad in enumerate(direct):
        flat = _np(grad).reshape(-1)
        for i in range(0, flat.size, max(1, flat.size // 5)):
            h = 1e-5
            ends = []
            for sign in (1, -1):
                moved = [a.copy() for a in args]
                moved[which].reshape(-1)[i] += sign * h
                ends.append(value(*moved))
            # Central differences: h^2 / 6 of a third derivative (below 1e3 here) and
            # 2^-52 of the value (below 1e2) over h.
            assert abs((ends[0] - ends[1]) / (2 * h) - flat[i]) < 1e-4 * (1 + abs(flat[i]))


def test_residual_norm_only_what_is_wanted():
    case = _norm_case(30, 24, "rows", torch.float32, 7)
    leaves = [t.to(DEV) for t in case[:5]]
    full = W.residual_norm_bwd(*leaves, *_cuda(*case[5:]))
    for i in range(5):
        want = tuple(j == i for j in range(5))
        only = W.residual_norm_bwd(*leaves, *_cuda(*case[5:]), want=want)
        assert [t is not None for t in only] == list(want) and torch.equal(only[i], full[i])
    # One of the two outputs alone.
    leaves = [t.requires_grad_(True) for t in leaves]
    y, u = latent.residual_norm(*leaves)
    got = torch.autograd.grad(u, leaves, case[6].to(DEV), retain_graph=True)
    want = W.residual_norm_bwd(*(t.detach() for t in leaves), None, case[6].to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(y, leaves[:4], case[5].to(DEV))
    want = W.residual_norm_bwd(*(t.detach() for t in leaves), case[5].to(DEV), None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_residual_norm_empty_and_not_finite():
    w = torch.ones(8, device=DEV)
    e = torch.empty(0, 8, device=DEV)
    y, u = latent.residual_norm(e, e, e, w, w)
    assert y.shape == u.shape == (0, 8)
    grads = W.residual_norm_bwd(e, e, w, w, w, e, e)
    assert grads[0].shape == (0, 8) and all(not g.any() for g in grads[2:])
    x, f, gate = (torch.randn(40, 8, device=DEV) for _ in range(3))
    x[3, 2], f[17, 5] = float("nan"), float("inf")
    gate[5] = -200.0  # a closed gate
    gate[6] = 200.0
    y, u = latent.residual_norm(x, f, gate, w, w)
    assert torch.equal(y[5], x[5])
    bad = torch.isnan(u).any(1)
    assert bad[3] and bad[17] and int(bad.sum()) == 2
    grads = W.residual_norm_bwd(x, f, gate, w, w, torch.ones_like(x), torch.ones_like(x))
    assert not torch.isnan(grads[1][5]).any() and not grads[2][5].any()


# ---------------------------------------------- streams, graphs, refusals --


def test_mixing_captured_and_on_another_stream():
    x, f, gate = (torch.randn(200, 64, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    p = torch.arange(400, device=DEV, dtype=torch.int32).reshape(200, 2)

    def work():
        y, u = W.residual_norm_fwd(x, f, gate, w, w)
        q, _ = W.rotary_axes(u.reshape(200, 4, 16), None, p, (4, 4))
        return (y, u, q, *W.residual_norm_bwd(x, f, gate, w, w, y, u))

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for seed in range(3):
        torch.manual_seed(seed)
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, work()))


def test_mixing_refusals():
    q = torch.randn(5, 2, 8, device=DEV)
    p = torch.zeros(5, 2, device=DEV)
    bad = [(lambda: latent.rotary_axes(q.cpu(), None, p, (2, 2)), "CUDA"),
           (lambda: latent.rotary_axes(q.double(), None, p, (2, 2)), "not implemented"),
           (lambda: latent.rotary_axes(q, q.half(), p, (2, 2)), "k must be torch.float32"),
           (lambda: latent.rotary_axes(q, q[:4], p, (2, 2)), "k must be"),
           (lambda: latent.rotary_axes(q, None, p.double(), (2, 2)), "positions must be"),
           (lambda: latent.rotary_axes(q, None, p, (2,)), "positions must be"),
           (lambda: latent.rotary_axes(q, None, p, (2, 3)), "not pairs"),
           (lambda: latent.rotary_axes(q, None, p, (-1, 3)), "not pairs"),
           (lambda: latent.rotary_axes(q, None, p, ()), "1 to 8 axes"),
           (lambda: latent.rotary_axes(q, None, p, (2, 2), base=0.0), "base"),
           (lambda: latent.rotary_axes(q[:, 0, 0], None, p, (2, 2)), r"\[..., H, D\]")]
    x, w = torch.randn(5, 8, device=DEV), torch.ones(8, device=DEV)
    big = torch.zeros(2, 8193, device=DEV)
    bad += [(lambda: latent.pre_norm(x, None), "weight must be given"),
            (lambda: latent.residual_norm(x, None), "update must be given"),
            (lambda: latent.pre_norm(x, w[:7]), r"weight must be \[8\]"),
            (lambda: latent.pre_norm(x, w.half()), "weight must be torch.float32"),
            (lambda: latent.pre_norm(big, big[0]), "8192 channels"),
            (lambda: latent.residual_norm(x, x[:4]), "shape of x"),
            (lambda: latent.residual_norm(x, x, x[:4]), "shape of x"),
            (lambda: W.residual_norm_fwd(x, None, x, None, w), "needs an update"),
            (lambda: W.residual_norm_bwd(x, x, None, None, None, x, x), "needs the weight")]
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()
    with pytest.raises(NotImplementedError, match="positions"):
        latent.rotary_axes(q, None, p.requires_grad_(True), (2, 2))
