"""Rotary positions, the norms around a block and AdamW without a GPU: the C
ABI's refusals, which come before any device is touched, and the restatement
against torch and differences."""

import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import mixing as ref
from r2splat import optim
from r2splat.cuda import _lib

FAKE = ctypes.c_void_p(256)  # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _refused(lib, rc, code, message):
    assert rc == code and message in lib.r2s_last_error(), lib.r2s_last_error()


def test_rotary_arguments(lib):
    def call(q=FAKE, qs=(32, 8), hq=4, hk=0, positions=FAKE, kind=0, sections=(2, 2), base=1e4,
             type_=0, n=5, head=8, out=FAKE):
        axes = len(sections)
        return lib.r2s_rotary_axes(q, *qs, hq, None, 0, 0, hk, positions, kind,
                                   (ctypes.c_int32 * max(axes, 1))(*sections), axes, 0, base, 0, 0,
                                   type_, n, head, out, None, None)

    _refused(lib, call(type_=3), 1001, b"element type 3")
    _refused(lib, call(n=-1), 1001, b"negative")
    _refused(lib, call(kind=3), 1001, b"position type")
    _refused(lib, call(sections=()), 1001, b"1 to 8 axes")
    _refused(lib, call(sections=(1,) * 9), 1001, b"1 to 8 axes")
    _refused(lib, call(sections=(3, 2)), 1001, b"5 pairs do not fit a head of 8")
    _refused(lib, call(sections=(3, -1)), 1001, b"section 1 is negative")
    _refused(lib, call(base=0.0), 1001, b"base")
    _refused(lib, call(base=float("nan")), 1001, b"base")
    _refused(lib, call(n=1 << 31), 1002, b"tokens")
    _refused(lib, call(head=4096), 1002, b"2048 channels")
    _refused(lib, call(positions=None), 1001, b"null positions")
    _refused(lib, call(q=None), 1001, b"null q")
    _refused(lib, call(hk=1), 1001, b"null k")
    _refused(lib, call(qs=(1 << 58, 8)), 1001, b"bad stride")
    assert call(n=0) == 0 and call(hq=0) == 0 and call(head=0, sections=(0,)) == 0


def test_residual_norm_arguments(lib):
    def fwd(x=FAKE, xs=8, f=FAKE, fs=8, gate=None, kind=0, w1=None, w2=FAKE, type_=0, n=4, d=8,
            y=FAKE, u=FAKE):
        return lib.r2s_residual_norm_fwd(x, xs, f, fs, gate, 8, kind, w1, w2, 1.0, 1e-6, 0, type_,
                                         n, d, y, u, None)

    _refused(lib, fwd(type_=-1), 1001, b"element type")
    _refused(lib, fwd(n=-1), 1001, b"negative")
    _refused(lib, fwd(kind=3), 1001, b"gate kind")
    _refused(lib, fwd(d=8193, xs=8193, fs=8193), 1002, b"8192 channels")
    _refused(lib, fwd(x=None), 1001, b"null x")
    _refused(lib, fwd(xs=7), 1001, b"rows overlap")
    _refused(lib, fwd(kind=1), 1001, b"null gate")
    _refused(lib, fwd(f=None, w1=FAKE, y=None), 1001, b"without an update")
    _refused(lib, fwd(f=None), 1001, b"y goes with an update")
    _refused(lib, fwd(w2=None), 1001, b"u with a weight")
    assert fwd(n=0) == 0 and fwd(d=0) == 0 and fwd(f=None, w2=None, y=None, u=None) == 0
    size = lib.r2s_residual_norm_bwd_workspace_bytes
    assert size(0, 0, 8) == size(7, 5, 8) == size(0, 5, 9000) == 0
    assert size(1, 1 << 20, 1024) <= 768 * 3 * 4 * 1024

    def bwd(f=FAKE, w1=FAKE, w2=FAKE, kind=0, v_u=FAKE, grads=(FAKE,) * 5, ws=FAKE, room=1 << 20):
        return lib.r2s_residual_norm_bwd(FAKE, 8, f, 8, FAKE, 8, kind, w1, w2, FAKE, 8, v_u, 8, 1.0,
                                         1e-6, 0, 0, 4, 8, *grads, ws, room, None)

    _refused(lib, bwd(f=None, w1=None), 1001, b"update that is not there")
    _refused(lib, bwd(w1=None), 1001, b"null update weight")
    _refused(lib, bwd(w2=None), 1001, b"null weight")
    _refused(lib, bwd(), 1001, b"no gate")
    _refused(lib, bwd(w2=None, grads=(FAKE, FAKE, None, FAKE, None)), 1001, b"without a weight")
    _refused(lib, bwd(kind=2, ws=None, room=0), 1004, b"workspace")


def test_adamw_arguments(lib):
    def call(**fields):
        t = _lib.AdamwTensor(**{**dict(param=256, grad=256, exp_avg=256, second=256, n=8), **fields})
        return lib.r2s_adamw_step(ctypes.byref(t), 1, None)

    _refused(lib, lib.r2s_adamw_step(None, 1, None), 1001, b"bad tensor list")
    _refused(lib, call(n=-1), 1001, b"negative")
    _refused(lib, call(type=3), 1001, b"element type 3")
    _refused(lib, call(grad=None), 1001, b"null pointer")
    _refused(lib, call(type=1), 1001, b"master")
    _refused(lib, call(master=256), 1001, b"master")
    _refused(lib, call(exp_avg_scale=256), 1001, b"one scale of two")
    _refused(lib, call(n=1 << 41), 1002, b"too large")
    assert call(n=0, grad=None) == 0 and lib.r2s_adamw_step(None, 0, None) == 0


def test_adamw_options():
    p = torch.zeros(4, requires_grad=True)
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0),
               dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    with pytest.raises(NotImplementedError, match="float lr"):
        optim.AdamW([p], lr=torch.tensor(1e-3))
    opt = optim.AdamW([p])
    opt.step()  # nothing has a gradient
    p.grad = torch.ones(4)
    with pytest.raises(NotImplementedError, match="CUDA parameters"):
        opt.step()


def test_norm_restatement_against_autograd():
    g = torch.Generator().manual_seed(0)
    draw = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    for centered in (False, True):
        for shape in ((7, 5), (5,)):
            x, f, w1, w2 = draw(7, 5), draw(7, 5), draw(5), draw(5)
            gate, v_y, v_u = draw(*shape), draw(7, 5), draw(7, 5)
            leaves = [t.requires_grad_(True) for t in (x, f, gate, w1, w2)]

            def norm(z):
                z = z - z.mean(-1, keepdim=True) if centered else z
                return z / torch.sqrt(z.square().mean(-1, keepdim=True) + 1e-5)

            y = x + 0.7 * torch.sigmoid(gate) * norm(f) * w1
            u = norm(y) * w2
            want = torch.autograd.grad((y * v_y).sum() + (u * v_u).sum(), leaves)
            out = ref.residual_norm(*(t.detach().numpy() for t in (*leaves, v_y, v_u)), 0.7, 1e-5,
                                    centered)
            assert np.allclose(out["y"].v, y.detach()) and np.allclose(out["u"].v, u.detach())
            for name, grad in zip(("v_x", "v_update", "v_gate", "v_w1", "v_w2"), want):
                assert np.allclose(out[name].v, grad), name
                assert (out[name].e > 0).all()


def test_bounds_hold_for_float32_evaluations():
    """The bounds' own check: numpy's float32 stays inside them."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 300)).astype(np.float32)
    for centered in (False, True):
        z = x - x.mean(-1, keepdims=True, dtype=np.float32) if centered else x
        z = z / np.sqrt((z * z).mean(-1, keepdims=True, dtype=np.float32) + np.float32(1e-6))
        exact, _ = ref.norm(x.astype(np.float64), 1e-6, centered)
        assert (np.abs(z - exact.v) <= exact.e).all()
        assert exact.e.max() < 1e-4


def test_rotary_restatement():
    rng = np.random.default_rng(1)
    x, p = rng.standard_normal((6, 2, 11)), rng.integers(0, 50, (6, 2))
    for interleaved in (False, True):
        for shared in (False, True):
            y, _ = ref.rotary(x, p, (2, 3), 100.0, interleaved, shared)
            back, _ = ref.rotary(y, p, (2, 3), 100.0, interleaved, shared, inverse=True)
            assert np.allclose(back, x)
            for j, (axis, rate) in enumerate([(0, 0), (0, 1 / 2), (1, 0), (1, 1 / 3), (1, 2 / 3)]):
                rate = j / 5 if shared else rate
                angle = p[:, axis] * 100.0 ** -rate
                a, b = (2 * j, 2 * j + 1) if interleaved else (j, 5 + j)
                z = (x[:, 1, a] + 1j * x[:, 1, b]) * np.exp(1j * angle)
                assert np.allclose(y[:, 1, a], z.real) and np.allclose(y[:, 1, b], z.imag)
            assert (y[..., 10:] == x[..., 10:]).all()


def test_quantized_values_are_float8_codes_and_right_on_average():
    rng = np.random.default_rng(2)
    x = rng.standard_normal(20_000) * np.exp(rng.standard_normal(20_000) * 3)
    total = np.zeros_like(x)
    for step in range(64):
        codes, scale = ref.quantize(x, (ref.chance(len(x), step) & 0xFFFF).astype(float), False)
        as_float8 = torch.tensor(codes).to(torch.float8_e4m3fn).double().numpy()
        assert (as_float8 == codes).all() and np.abs(codes).max() <= 448
        total += codes
    scale = np.repeat(scale, 256)[:len(x)]
    step = ref.code_step(np.abs(x) / scale)
    error = (total / 64 - x / scale) / step
    # Means of 64 errors of at most half a step's deviation, 20,000 of them: 6 deviations.
    assert np.abs(error).max() < 6 * 0.5 / 8 and abs(error.mean()) < 6 * 0.5 / 8 / 141
    root, _ = ref.quantize(np.abs(x), np.zeros(len(x)), True)
    assert (root > 0).all()


def test_chances_are_spread():
    h = ref.chance(1 << 16, 12345)
    for part in (h & 0xFFFF, h >> 16):
        counts = np.bincount(part >> 8, minlength=256)
        # 256 draws to each of 256 cells: 6 deviations.
        assert abs(counts - 256).max() < 6 * 16
    bits = np.unpackbits((h ^ ref.chance(1 << 16, 12346)).view(np.uint8))
    assert abs(bits.mean() - 0.5) < 0.01  # steps side by side
    assert abs(np.corrcoef(h & 0xFFFF, h >> 16)[0, 1]) < 0.03


def test_tangents_are_refused_rather_than_lost(monkeypatch):
    from r2splat.ops import latent

    class Plain:
        @staticmethod
        def rotary_axes(q, k, *args, **kw):
            return q.detach().clone(), None if k is None else k.detach().clone()

        @staticmethod
        def residual_norm_fwd(x, update, gate, w1, w2, *args):
            return x.detach().clone(), x.detach().clone()

        @staticmethod
        def decay_attention_fwd(q, k, v, *args, **kw):
            return v.detach().clone(), torch.zeros(1), torch.zeros(1)

        @staticmethod
        def decay_attention_step(q, k, v, *args):
            return v.detach().clone(), torch.zeros(1)

    monkeypatch.setattr(latent, "W", Plain)
    t, w, p = torch.randn(4, 2, 6), torch.ones(6), torch.zeros(4, 1)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(t, torch.ones_like(t))
        dw = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: latent.rotary_axes(d, None, p, (3,)),
                     lambda: latent.rotary_axes(t, d, p, (3,)),
                     lambda: latent.pre_norm(d, w), lambda: latent.pre_norm(t, dw),
                     lambda: latent.residual_norm(d, t, weight=w),
                     lambda: latent.residual_norm(t, d, weight=w),
                     lambda: latent.residual_norm(t, t, gate=d, weight=w),
                     lambda: latent.residual_norm(t, t, update_weight=dw)):
            with pytest.raises(NotImplementedError, match="forward mode AD"):
                call()
        with pytest.raises(NotImplementedError, match="positions"):
            latent.rotary_axes(t, None, forward_ad.make_dual(p, torch.ones_like(p)), (3,))
        g = torch.zeros(2)
        state = torch.zeros(4, 2, 6, 6)
        for args in ((d, t, t), (t, d, t), (t, t, d)):
            with pytest.raises(NotImplementedError, match="forward mode AD"):
                latent.decay_attention(*(a[None] for a in args), g)
            with pytest.raises(NotImplementedError, match="forward mode AD"):
                latent.decay_attention_step(*args, g, state)
        with pytest.raises(NotImplementedError, match="log_decay"):
            latent.decay_attention(t[None], t[None], t[None],
                                   forward_ad.make_dual(g, torch.ones(2)))


def test_functions_are_there_without_the_library():
    from r2splat.cuda import _wrapper
    from r2splat.ops import latent

    for name in ("decay_attention", "decay_attention_step", "rotary_axes", "pre_norm",
                 "residual_norm"):
        assert name in latent.__all__ and callable(getattr(latent, name))
    for name in ("decay_attention_fwd", "decay_attention_bwd", "decay_attention_step",
                 "rotary_axes", "residual_norm_fwd", "residual_norm_bwd"):
        assert callable(getattr(_wrapper, name))
    if not torch.cuda.is_available():
        q = torch.zeros(1, 1, 1, 2)
        with pytest.raises(RuntimeError, match="unavailable"):
            latent.decay_attention(q, q, q, torch.zeros(1))


def test_decay_attention_arguments(lib):
    def fwd(q=FAKE, qs=(80, 16, 8), offsets=None, s=2, length=5, n=10, h=2, dk=8, dv=8, type_=0,
            final=FAKE, kept=FAKE, decay=FAKE):
        return lib.r2s_decay_attention_fwd(q, *qs, FAKE, 80, 16, 8, FAKE, 80, 16, 8, decay, None,
                                           offsets, s, length, n, h, dk, dv, 1.0, type_, 0, FAKE,
                                           final, kept, None, 0, None)

    _refused(lib, fwd(type_=9), 1001, b"element type")
    _refused(lib, fwd(h=-1), 1001, b"negative")
    _refused(lib, fwd(dk=257), 1002, b"256 channels")
    _refused(lib, fwd(n=1 << 31), 1002, b"tokens")
    _refused(lib, fwd(n=11), 1001, b"11 tokens are not 2 sequences of 5")
    _refused(lib, fwd(offsets=FAKE, s=0), 1001, b"without a sequence")
    _refused(lib, fwd(decay=None), 1001, b"null decays")
    _refused(lib, fwd(final=None), 1001, b"null final")
    _refused(lib, fwd(q=None), 1001, b"null tokens")
    _refused(lib, fwd(qs=(-1, 16, 8)), 1001, b"bad stride")
    _refused(lib, fwd(qs=(80, 1 << 58, 8)), 1001, b"bad stride")
    _refused(lib, fwd(s=1, length=100_000, n=100_000, kept=None), 1001, b"null kept")
    _refused(lib, fwd(offsets=FAKE, n=100_000), 1004, b"workspace")
    assert fwd(s=0, n=0) == 0 and fwd(h=0) == 0 and fwd(dv=0) == 0
    kept, room = lib.r2s_decay_attention_kept_states, lib.r2s_decay_attention_workspace_bytes
    # Short sequences carry nothing; a long one's states are few beside its tokens.
    assert kept(0, 0, 8, 200, 1600, 4, 16, 16) == 0 and room(0, 0, 8, 200, 1600, 4, 16, 16, 1) == 0
    states = kept(1, 0, 1, 500_000, 500_000, 4, 16, 16)
    assert 0 < states <= 500_000 // 256
    assert room(1, 0, 1, 500_000, 500_000, 4, 16, 16, 0) == 0
    assert room(1, 0, 1, 500_000, 500_000, 4, 16, 16, 1) == states * 4 * 16 * 16 * 4
    # Ragged calls have a table of their spans, and no state for each sequence.
    assert kept(0, 1, 100_000, 0, 100_000, 4, 16, 16) <= 100_000 // 256
    assert 4 * 100_000 < room(0, 1, 100_000, 0, 100_000, 4, 16, 16, 0) < 1 << 20
    assert kept(7, 0, 1, 9, 9, 1, 1, 1) == 0 and room(0, 0, 1, 9, 8, 1, 1, 1, 1) == 0
    rc = lib.r2s_decay_attention_bwd(FAKE, 80, 16, 8, FAKE, 80, 16, 8, FAKE, 80, 16, 8, FAKE, None,
                                     None, None, FAKE, 80, 16, 8, None, 2, 5, 10, 2, 8, 8, 1.0, 0,
                                     0, None, FAKE, FAKE, None, None, 0, None)
    _refused(lib, rc, 1001, b"null tokens")
    rc = lib.r2s_decay_attention_step(FAKE, 16, 8, FAKE, 16, 8, FAKE, 16, 8, FAKE, None, 2, 2, 8, 8,
                                      1.0, 0, FAKE, FAKE, None)
    _refused(lib, rc, 1001, b"null pointer")


def test_decay_attention_restatement_against_autograd():
    g = torch.Generator().manual_seed(3)
    draw = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    bounds = [0, 7, 7, 20]
    for reverse in (False, True):
        q, k, v, state = draw(20, 2, 4), draw(20, 2, 4), draw(20, 2, 3), draw(3, 2, 4, 3)
        v_y, v_final, log_decay = draw(20, 2, 3), draw(3, 2, 4, 3), -draw(2).abs()
        leaves = [t.requires_grad_(True) for t in (q, k, v, state)]
        gamma, ys, finals = log_decay.exp()[:, None, None], [None] * 20, []
        for s in range(3):
            now = state[s]
            order = range(bounds[s], bounds[s + 1])
            for t in reversed(order) if reverse else order:
                now = gamma * now + k[t][:, :, None] * v[t][:, None]
                ys[t] = 0.4 * (q[t][:, :, None] * now).sum(1)
            finals.append(now)
        y, final = torch.stack(ys), torch.stack(finals)
        want = torch.autograd.grad((y * v_y).sum() + (final * v_final).sum(), leaves)
        exact = ref.DecayAttention(*(t.detach().numpy() for t in (q, k, v, log_decay)), bounds,
                                   state.detach().numpy(), reverse, 0.4)
        ey, ef, _, _ = exact.forward()
        assert np.allclose(ey, y.detach()) and np.allclose(ef, final.detach())
        found = exact.backward(v_y.numpy(), v_final.numpy())
        for name, grad in zip(("v_q", "v_k", "v_v", "v_initial"), want):
            assert np.allclose(found[name][0], grad), name
