"""Linear attention with a decay for each head on the GPU against float64, token
after token.

Tolerances, u = 2^-24: an output is a sum of products of three inputs and a power
of the decay.  A chunked float32 evaluation rounds each of its terms by at most
(dk + dv + 64) u in the sums of products, by 8 u and by 2 u |log2(weight)| in the
power (exponents up to 126 before a weight underflows, so by less than that
times the weight, of which w |log2 w| < 0.54), and by 2 u for each of the length / 32
chunks that the state is carried through, which is capped by the decay but not
counted on; 16-bit operands' rest parts add 2^-16 (the square of a half step of
bfloat16's 2^-8).  All of the sum of the terms' absolute values."""

import math

import numpy as np
import pytest
import torch

from oracle.mixing import DecayAttention
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _tolerance(dtype, dk, dv, longest):
    share = (dk + dv + 64 + 16 + 2 * longest / 32) * U
    return share + (0 if dtype == torch.float32 else 2.0 ** -15)


def _close(got, exact, mass, share, dtype, what):
    got = _np(got)
    assert got.shape == exact.shape, what
    bound = share * mass
    tol = bound + (HALF[dtype] * (np.abs(exact) + bound) if dtype is not None else 0) + TINY[dtype]
    bad = ~(np.abs(got - exact) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], exact[bad][:4],
                           (np.abs(got - exact) / np.maximum(mass, 1e-30)).max() / share)


def _case(n, heads, dk, dv, sequences, dtype, seed, initial=True):
    g = _gen(seed)
    q, k, v = (_randn(g, n, heads, d, dtype=dtype) for d in (dk, dk, dv))
    # From a memory of one token to one without an end.
    log_decay = torch.log1p(-torch.exp2(-torch.linspace(0.5, 10, heads)))
    if heads > 1:
        log_decay[-1] = 0.0
    state = _randn(g, sequences, heads, dk, dv) if initial else None
    return q, k, v, log_decay, state, _randn(g, n, heads, dv, dtype=dtype), \
        _randn(g, sequences, heads, dk, dv)


def _check(case, bounds, reverse, dtype, ragged, scale=0.3):
    q, k, v, log_decay, state, v_y, v_final = case
    sequences = len(bounds) - 1
    dev = [None if t is None else t.to(DEV) for t in case]
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV) if ragged else None
    shape = (lambda t: t) if ragged else (lambda t: t.reshape(sequences, -1, *t.shape[1:]))
    tokens = [shape(t) for t in dev[:3]]
    y, final, kept = W.decay_attention_fwd(*tokens, dev[3], dev[4], offsets, reverse, scale)
    grads = W.decay_attention_bwd(*tokens, dev[3], dev[4], offsets, kept, shape(dev[5]), dev[6],
                                  reverse, scale)
    exact = DecayAttention(*(_np(t) for t in (q, k, v, log_decay)), bounds, _np(state), reverse,
                           scale)
    longest = max(b - a for a, b in zip(bounds, bounds[1:])) if sequences else 0
    share = _tolerance(dtype, q.shape[2], v.shape[2], longest)
    ey, ef, ym, fm = exact.forward()
    _close(y.reshape(ey.shape), ey, ym, share, dtype, "y")
    _close(final, ef, fm, share, torch.float32, "final")
    want = exact.backward(_np(v_y), _np(v_final))
    for name, got in zip(("v_q", "v_k", "v_v", "v_initial"), grads):
        value, mass = want[name]
        _close(got.reshape(value.shape), value, mass, share,
               torch.float32 if name == "v_initial" else dtype, name)
    return (y, final, *grads)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,length,heads,dk,dv", [
    (1, 1, 1, 1, 1), (3, 1, 2, 16, 16), (2, 63, 2, 16, 16), (2, 64, 1, 64, 64), (1, 65, 2, 33, 45),
    (3, 130, 3, 64, 16), (1, 200, 2, 128, 128), (1, 97, 2, 20, 100), (2, 100, 1, 256, 256),
    (1, 70, 1, 130, 7), (1, 33, 1, 5, 200), (5, 40, 2, 32, 32)])
def test_equal_sequences(b, length, heads, dk, dv, dtype):
    for reverse in (False, True):
        case = _case(b * length, heads, dk, dv, b, dtype, length + dk + reverse, bool(reverse))
        _check(case, list(range(0, b * length + 1, length)), reverse, dtype, False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dk,dv", [(2, 16, 16), (1, 64, 64), (1, 33, 45)])
def test_ragged_sequences(heads, dk, dv, dtype):
    bounds = [0, 0, 5, 69, 70, 70, 200, 201, 264, 300, 300]
    for reverse in (False, True):
        case = _case(300, heads, dk, dv, 10, dtype, dk + reverse)
        _check(case, bounds, reverse, dtype, True)


@pytest.mark.parametrize("dtype,heads,dk,dv", [
    (torch.float32, 1, 17, 20), (torch.bfloat16, 2, 16, 16), (torch.float16, 1, 32, 64)])
def test_sequences_of_several_spans(dtype, heads, dk, dv):
    n = 3001
    for reverse in (False, True):
        case = _case(n, heads, dk, dv, 1, dtype, 1 + reverse)
        _check(case, [0, n], reverse, dtype, False)
        bounds = [0, 3, 3, 1500, 1500, 1756, 2012, 2900, 3001, 3001]
        case = _case(n, heads, dk, dv, len(bounds) - 1, dtype, 3 + reverse)
        _check(case, bounds, reverse, dtype, True)


def test_a_long_sequence_in_its_pieces():
    """A sequence at once, and in two calls through the state between them."""
    n, heads, d = 50_000, 2, 32
    q, k, v, log_decay, _, _, _ = _case(n, heads, d, d, 1, torch.float32, 9)
    q, k, v, log_decay = (t.to(DEV) for t in (q, k, v, log_decay))
    y, final = latent.decay_attention(q[None], k[None], v[None], log_decay)
    a, b = (slice(None, 20_001), slice(20_001, None))
    y1, middle = latent.decay_attention(*(t[None, a] for t in (q, k, v)), log_decay)
    y2, last = latent.decay_attention(*(t[None, b] for t in (q, k, v)), log_decay, middle)
    both = torch.cat([y1, y2], 1)
    share = _tolerance(torch.float32, d, d, n)
    mass, end = latent.decay_attention(*(t[None].abs() for t in (q, k, v)), log_decay)
    assert ((both - y).abs() <= 2 * share * mass + 1e-30).all()
    assert ((last - final).abs() <= 2 * share * end + 1e-30).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,heads,dk,dv", [(1, 1, 1, 1), (7, 3, 16, 16), (64, 8, 64, 64),
                                           (3, 2, 33, 45), (2, 1, 256, 256), (5, 2, 130, 7)])
def test_step(b, heads, dk, dv, dtype):
    case = _case(b, heads, dk, dv, b, dtype, b + dk)
    q, k, v, log_decay, state = case[:5]
    y, final = latent.decay_attention_step(*(t.to(DEV) for t in (q, k, v, log_decay, state)))
    exact = DecayAttention(*(_np(t) for t in (q, k, v, log_decay)), list(range(b + 1)), _np(state),
                           False, dk ** -0.5)
    ey, ef, ym, fm = exact.forward()
    share = _tolerance(torch.float32, dk, dv, 1)
    _close(y, ey, ym, share, dtype, "y")
    _close(final, ef, fm, share, torch.float32, "final")
    wide = torch.zeros(b, heads, dk, dv + 1, device=DEV)
    wide[..., 1:] = state.to(DEV)
    fused = torch.randn(b, heads, 2 * dk + dv, device=DEV).to(dtype)
    again = latent.decay_attention_step(fused[..., :dk], fused[..., dk:2 * dk], fused[..., 2 * dk:],
                                        log_decay.to(DEV), wide[..., 1:])
    plain = latent.decay_attention_step(*(t.contiguous() for t in fused.split((dk, dk, dv), -1)),
                                        log_decay.to(DEV), state.to(DEV))
    assert all(torch.equal(s, t) for s, t in zip(again, plain))


def test_strides():
    g = _gen(4)
    b, length, h, d = 3, 90, 4, 24
    fused = _randn(g, b, length, 3, h, d, dtype=torch.bfloat16).to(DEV)
    log_decay = -torch.rand(h, generator=g).to(DEV)
    q, k, v = fused.unbind(2)
    want = latent.decay_attention(*(t.contiguous() for t in (q, k, v)), log_decay)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = torch.zeros(b, length, h, d + 1, device=DEV, dtype=torch.bfloat16)
    odd[..., 1:] = k
    across = v.transpose(2, 3).contiguous().transpose(2, 3)  # a head's elements lie apart
    for args in ((q, k, v), heads_first, (q, odd[..., 1:], across)):
        got = latent.decay_attention(*args, log_decay)
        assert all(torch.equal(s, t) for s, t in zip(got, want))
    # One query for every token and head.
    one = q[:, :1, :1].expand(b, length, h, d)
    got = latent.decay_attention(one, k, v, log_decay)
    want = latent.decay_attention(one.contiguous(), k, v, log_decay)
    assert all(torch.equal(s, t) for s, t in zip(got, want))


def test_gradients_through_autograd_and_differences():
    g = _gen(5)
    n, h, dk, dv = 21, 2, 4, 3
    bounds = [0, 8, 8, 20]  # the last token is in no sequence
    q, k, v = (_randn(g, n, h, d) for d in (dk, dk, dv))
    state, v_y, v_final = _randn(g, 3, h, dk, dv), _randn(g, n, h, dv), _randn(g, 3, h, dk, dv)
    log_decay = torch.tensor([-0.3, -0.01])
    offsets = torch.tensor(bounds, device=DEV)  # int64 is taken
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, state)]
    y, final = latent.decay_attention(*leaves[:3], log_decay.to(DEV), leaves[3], offsets)
    assert not y[20].any()
    total = (y * v_y.to(DEV)).sum() + (final * v_final.to(DEV)).sum()
    grads = torch.autograd.grad(total, leaves)

    def value(q, k, v, state):
        y, final, _, _ = DecayAttention(q, k, v, _np(log_decay), bounds, state, False,
                                        dk ** -0.5).forward()
        return (y * _np(v_y)).sum() + (final * _np(v_final)).sum()

    args = [_np(t) for t in (q, k, v, state)]
    for which, grad in enumerate(grads):
        flat = _np(grad).reshape(-1)
        for i in range(0, flat.size, max(1, flat.size // 12)):
            ends = []
            for sign in (1, -1):
                moved = [a.copy() for a in args]
                moved[which].reshape(-1)[i] += sign * 1e-4
                ends.append(value(*moved))
            # Linear in each input: no error of the difference but 2^-52 of the value
            # (below 1e3) over 1e-4; the gradient's own is below 200 u of 1e3.
            assert abs((ends[0] - ends[1]) / 2e-4 - flat[i]) < 2e-2 * (1 + abs(flat[i])) * 1e-1
    # One output's gradient alone, and through the step.
    only = torch.autograd.grad(latent.decay_attention(*leaves[:3], log_decay.to(DEV), leaves[3],
                                                      offsets)[1].sum(), leaves, allow_unused=True)
    assert not only[0].any() and only[1].any()
    one = [t[:3].detach().requires_grad_(True) for t in leaves[:3]]
    y, final = latent.decay_attention_step(*one, log_decay.to(DEV), leaves[3])
    plain = latent.decay_attention_step(*(t.detach() for t in one), log_decay.to(DEV),
                                        leaves[3].detach())
    assert torch.allclose(y, plain[0], rtol=1e-5, atol=1e-5)
    assert all(t is not None for t in torch.autograd.grad((y.sum() + final.sum()),
                                                          [*one, leaves[3]]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [16, 64])
def test_values_that_are_not_finite_reach_later_tokens_alone(d, dtype):
    n, h = 400, 2
    q, k, v, log_decay, _, v_y, _ = _case(n, h, d, d, 1, dtype, 6, False)
    q, k, v, v_y, log_decay = (t.to(DEV) for t in (q, k, v, v_y, log_decay))
    clean, _ = latent.decay_attention(q[None], k[None], v[None], log_decay)
    for which, value in (("v", float("nan")), ("v", float("inf")), ("k", float("nan")),
                         ("q", float("inf"))):
        for reverse in (False, True):
            t = {"q": q, "k": k, "v": v}[which].clone()
            t[203, 1, 3] = value
            args = [t if which == name else x for name, x in (("q", q), ("k", k), ("v", v))]
            if reverse:
                args = [a.flip(0) for a in args]
            y, final = latent.decay_attention(*(a[None] for a in args), log_decay, reverse=reverse)
            y = y[0].flip(0) if reverse else y[0]
            bad = ~torch.isfinite(y)
            assert not bad[:, 0].any() and not bad[:203].any(), (which, value)
            assert bad[203, 1].any()
            near = (y - clean[0])[:203].float().abs()
            assert (near <= 1e-2 * (1 + clean[0][:203].float().abs())).all()
            if which == "q":
                assert not bad[204:].any() and torch.isfinite(final).all()
            else:
                assert bad[204:, 1].any(1).all() and not torch.isfinite(final[0, 1]).all()
    # Gradients run the other way, and the queries' on.
    y, final, kept = W.decay_attention_fwd(q[None], k[None], v[None], log_decay)
    for which, behind in (("q", ("v_k", "v_v")), ("k", ("v_v",)), ("v", ("v_k",))):
        t = {"q": q, "k": k, "v": v}[which].clone()
        t[203, 1, 3] = float("inf")
        args = [t if which == name else x for name, x in (("q", q), ("k", k), ("v", v))]
        kept = W.decay_attention_fwd(*(a[None] for a in args), log_decay)[2]
        grads = dict(zip(("v_q", "v_k", "v_v"), W.decay_attention_bwd(
            *(a[None] for a in args), log_decay, None, None, kept, v_y[None])))
        for name, grad in grads.items():
            bad = ~torch.isfinite(grad[0]).all(-1)
            assert not bad[:, 0].any(), (which, name)
            if which == "q":  # reaches the tokens before, not its own gradient
                assert not bad[204:].any() and bool(bad[:203, 1].all()) == (name != "v_q")
            else:  # what it was multiplied with: behind it the queries, at it the other
                assert not bad[:203].any() and bad[203:, 1].any() == (name in (*behind, "v_q"))
                assert name == "v_q" or not bad[204:].any()
    y, final, kept = W.decay_attention_fwd(q[None], k[None], v[None], log_decay)
    v_y[203, 0, 2] = float("nan")
    y, final, kept = W.decay_attention_fwd(q[None], k[None], v[None], log_decay)
    v_q, v_k, v_v, _ = W.decay_attention_bwd(q[None], k[None], v[None], log_decay, None, None, kept,
                                             v_y[None])
    assert torch.isnan(v_q[0, 203, 0]).any() and int(torch.isnan(v_q).any(-1).sum()) == 1
    for grad in (v_k, v_v):
        bad = torch.isnan(grad[0]).any(-1)
        assert bad[:204, 0].all() and not bad[204:].any() and not bad[:, 1].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_decays_at_their_ends(dtype):
    n, d = 150, 16
    q, k, v = (_randn(_gen(i), 1, n, 4, d, dtype=dtype).to(DEV) for i in range(3))
    log_decay = torch.tensor([-float("inf"), -200.0, 0.0, -1e-7], device=DEV)
    y, final = latent.decay_attention(q, k, v, log_decay, scale=1.0)
    assert torch.isfinite(y).all()
    alone = (q.float() * k.float()).sum(-1, keepdim=True) * v.float()
    tol = 40 * U * (q.float() * k.float()).abs().sum(-1, keepdim=True) * v.float().abs()
    for head in (0, 1):
        far = (y.float() - alone)[:, :, head].abs()
        assert (far <= (tol + 2 * HALF[dtype] * alone.abs() + 2.0 ** -15 * tol / (40 * U) + 1e-7)
                [:, :, head]).all()
        # One exact product, rounded; float16's two bfloat16 parts leave out that of
        # both rests, each at most half a step (2^-8) of its value.
        last = torch.outer(k[0, -1, head].float(), v[0, -1, head].float())
        off = 2 * U if dtype == torch.float32 else 2 * U + 2.0 ** -16
        assert ((final[0, head] - last).abs() <= off * last.abs()).all()
    total = torch.einsum("nk,nv->kv", k[0, :, 2].double(), v[0, :, 2].double())
    mass = torch.einsum("nk,nv->kv", k[0, :, 2].double().abs(), v[0, :, 2].double().abs())
    assert ((final[0, 2] - total).abs() <= 300 * U * mass + 2.0 ** -15 * mass).all()


def test_float16_states_and_scores_beyond_its_range():
    n, d = 300, 16
    g = _gen(8)
    q, k = (_randn(g, 1, n, 1, d, dtype=torch.float16, scale=300.0).to(DEV) for _ in range(2))
    v = _randn(g, 1, n, 1, d, dtype=torch.float16, scale=300.0).to(DEV)
    log_decay = torch.tensor([-0.001], device=DEV)
    y, final = latent.decay_attention(q, k, v, log_decay, scale=2.0 ** -24)
    exact = DecayAttention(*(_np(t[0]) for t in (q, k, v)), _np(log_decay), [0, n], None, False,
                           2.0 ** -24)
    ey, ef, ym, fm = exact.forward()
    share = _tolerance(torch.float16, d, d, n)
    assert np.abs(ef).max() > 65504
    _close(y[0], ey, ym, share, torch.float16, "y")
    _close(final, ef, fm, share, torch.float32, "final")


def test_empty():
    log_decay = torch.zeros(2, device=DEV)
    e = lambda *s: torch.zeros(s, device=DEV)  # noqa: E731
    state = torch.randn(3, 2, 4, 5, device=DEV)
    y, final = latent.decay_attention(e(3, 0, 2, 4), e(3, 0, 2, 4), e(3, 0, 2, 5), log_decay, state)
    assert y.shape == (3, 0, 2, 5) and torch.equal(final, state)
    off = torch.zeros(4, dtype=torch.int32, device=DEV)
    y, final, kept = W.decay_attention_fwd(e(0, 2, 4), e(0, 2, 4), e(0, 2, 5), log_decay, state, off)
    assert y.shape == (0, 2, 5) and torch.equal(final, state)
    grads = W.decay_attention_bwd(e(0, 2, 4), e(0, 2, 4), e(0, 2, 5), log_decay, state, off, kept, y,
                                  state)
    assert torch.equal(grads[3], state)
    # Tokens in no sequence: zeros, and no gradient.
    q, v = torch.randn(700, 2, 4, device=DEV), torch.randn(700, 2, 5, device=DEV)
    y, final, kept = W.decay_attention_fwd(q, q, v, log_decay, state, off)
    assert not y.any() and torch.equal(final, state)
    grads = W.decay_attention_bwd(q, q, v, log_decay, state, off, kept, v, state)
    assert not any(t.any() for t in grads[:3]) and torch.equal(grads[3], state)
    y, final = latent.decay_attention(e(2, 9, 2, 0), e(2, 9, 2, 0), e(2, 9, 2, 5) + 1, log_decay)
    assert not y.any() and final.shape == (2, 2, 0, 5)
    y, final = latent.decay_attention_step(e(0, 2, 4), e(0, 2, 4), e(0, 2, 5), log_decay, state[:0])
    assert y.shape == (0, 2, 5) and final.shape == (0, 2, 4, 5)
    y, final = latent.decay_attention(e(1, 9, 2, 4) + 1, e(1, 9, 2, 4), e(1, 9, 2, 0), log_decay)
    assert y.shape == (1, 9, 2, 0)


def test_offsets_that_do_not_ascend_stay_in_bounds():
    """Whatever they say, nothing is read or written outside the tensors."""
    n = 2000
    q, v = torch.randn(n, 1, 8, device=DEV), torch.randn(n, 1, 8, device=DEV)
    log_decay = torch.full((1,), -0.1, device=DEV)
    for bounds in ([0, n, 0, n, 0, n], [5, -100, 3 * n, 7], [n, n, 0], [0, -1], [1, 2]):
        off = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        y, final, kept = W.decay_attention_fwd(q, q, v, log_decay, None, off)
        grads = W.decay_attention_bwd(q, q, v, log_decay, None, off, kept, v)
        torch.cuda.synchronize()
        assert y.shape == v.shape and grads[0].shape == q.shape


@pytest.mark.parametrize("dtype,d", [(torch.float32, 128), (torch.bfloat16, 256)])
def test_large_heads_captured(dtype, d):
    """More LDS than a launch has without asking."""
    q, k, v, log_decay, _, v_y, _ = (
        None if t is None else t.to(DEV) for t in _case(700, 1, d, d, 1, dtype, 11, False))
    q, k, v, v_y = (t[None] for t in (q, k, v, v_y))

    def work():
        y, final, kept = W.decay_attention_fwd(q, k, v, log_decay)
        return (y, final, *W.decay_attention_bwd(q, k, v, log_decay, None, None, kept, v_y))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for seed in range(2):
        torch.manual_seed(seed)
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, work()))


def test_captured_and_on_another_stream():
    n, h, d = 3000, 2, 16
    q, k, v, log_decay, state, v_y, v_final = (
        t.to(DEV) for t in _case(n, h, d, d, 4, torch.bfloat16, 10))
    offsets = torch.tensor([0, 1000, 1000, 2700, 2990], dtype=torch.int32, device=DEV)

    def work():
        y, final, kept = W.decay_attention_fwd(q, k, v, log_decay, state, offsets)
        s, _ = W.decay_attention_step(q[:4], k[:4], v[:4], log_decay, final)
        return (y, final, s, *W.decay_attention_bwd(q, k, v, log_decay, state, offsets, kept, v_y,
                                                    v_final))

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
    for seed, bounds in enumerate(([0, 10, 600, 1300, 3000], [0, 0, 0, 0, 3000],
                                   [0, 700, 1400, 2100, 2800])):
        torch.manual_seed(seed)
        v.copy_(torch.randn(n, h, d, device=DEV))
        offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, work()))


def test_refusals():
    q, v = torch.randn(2, 5, 3, 8, device=DEV), torch.randn(2, 5, 3, 6, device=DEV)
    g = torch.zeros(3, device=DEV)
    state = torch.zeros(2, 3, 8, 6, device=DEV)
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    f = latent.decay_attention
    big = torch.zeros(1, 1, 1, 257, device=DEV)
    for call, message in (
            (lambda: f(q.cpu(), q, v, g), "CUDA"), (lambda: f(q.double(), q, v, g), "implemented"),
            (lambda: f(q, q.half(), v, g), "k must be torch.float32"),
            (lambda: f(q, q[:, :4], v, g), "k must be"), (lambda: f(q, q, v[..., 0, :], g), "v must"),
            (lambda: f(q[0], q[0], v[0], g), r"\[B, L, H, Dk\] without"),
            (lambda: f(q, q, v, g, offsets=off), r"\[N, H, Dk\] with"),
            (lambda: f(q, q, v, g[:2]), "log_decay must be"),
            (lambda: f(q, q, v, g.double()), "log_decay must be"),
            (lambda: f(q, q, v, g, state[:1]), "initial must be"),
            (lambda: f(q, q, v, g, state.half()), "initial must be"),
            (lambda: f(q[0], q[0], v[0], g, offsets=off[:1]), "no sequence"),
            (lambda: f(big, big, big, g[:1]), "256 channels"),
            (lambda: latent.decay_attention_step(q[:, 0], q[:, 0], v[:, 0], g, None), "must be given"),
            (lambda: latent.decay_attention_step(q, q, v, g, state), r"\[B, H, Dk\]")):
        with pytest.raises(RuntimeError, match=message):
            call()
    with pytest.raises(NotImplementedError, match="log_decay"):
        f(q, q, v, g.requires_grad_(True))
    y, final, kept = W.decay_attention_fwd(q, q, v, g.detach())
    with pytest.raises(RuntimeError, match="kept"):
        W.decay_attention_bwd(q, q, v, g.detach(), None, None, state, v)


@pytest.mark.parametrize("lengths", [
    [0, 1, 255, 256, 257, 40, 600, 128] * 6,   # whole spans and rests of every eighth
    [0, 1, 3, 2, 0, 5] * 250 + [700, 0],       # more sequences than a block has threads
    [700, 3]], ids=["mixed", "many", "few"])
@pytest.mark.parametrize("heads,dk,dv,dtype", [(5, 16, 16, torch.bfloat16),
                                               (3, 33, 45, torch.float32),
                                               (2, 64, 64, torch.float16)])
def test_ragged_spans_taken_out_of_order(lengths, heads, dk, dv, dtype):
    bounds = np.cumsum([0] + lengths).tolist()
    case = _case(bounds[-1] + 7, heads, dk, dv, len(lengths), dtype, len(lengths) + dk)
    exact = tuple(None if t is None else t[:bounds[-1]] if t.shape[0] == bounds[-1] + 7 else t
                  for t in case)
    got = _check(exact, bounds, True, dtype, True)
    # Tokens behind the last sequence change nothing and get zeros.
    q, k, v, log_decay, state, v_y, v_final = (t.to(DEV) for t in case)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    y, final, kept = W.decay_attention_fwd(q, k, v, log_decay, state, offsets, True, 0.3)
    grads = W.decay_attention_bwd(q, k, v, log_decay, state, offsets, kept, v_y, v_final, True, 0.3)
    for a, b in zip(got, (y, final, *grads)):
        assert torch.equal(a, b[:a.shape[0]])
        assert not bool(b[a.shape[0]:].any())
