"""AdamW on the GPU: float32 states against torch's bit for bit, 16-bit
parameters through their masters, 8-bit states against numpy."""

import copy

import numpy as np
import pytest
import torch

from oracle import mixing as ref
from r2splat import optim

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _params(shapes, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(DEV).requires_grad_(True) for s in shapes]


def _grads(params, seed, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(p.shape, generator=g) * scale).to(p.dtype).to(DEV) for p in params]


SHAPES = [(4096, 64), (33, 7), (1,), (), (0, 5), (5000,), (257,)] + [(10 + i, 3) for i in range(70)]


@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_float32_states_as_torch(decay):
    mine, theirs = _params(SHAPES, torch.float32), _params(SHAPES, torch.float32)
    kw = dict(lr=3e-3, betas=(0.8, 0.95), eps=1e-7, weight_decay=decay)
    a, b = optim.AdamW(mine, **kw), torch.optim.AdamW(theirs, **kw)
    for step in range(4):
        for p, q, g in zip(mine, theirs, _grads(mine, step)):
            p.grad, q.grad = g, g.clone()
        mine[1].grad = theirs[1].grad = None if step == 1 else mine[1].grad
        a.step(), b.step()
        for p, q in zip(mine, theirs):
            assert torch.equal(p, q)
            if p.numel():
                for name in ("exp_avg", "exp_avg_sq"):
                    assert torch.equal(a.state[p][name], b.state[q][name])
    assert float(a.state[mine[1]]["step"]) == 3.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16_bit_parameters_are_their_masters_roundings(dtype):
    mine = _params(SHAPES, dtype)
    full = [p.detach().float().requires_grad_(True) for p in mine]
    a, b = optim.AdamW(mine, lr=1e-4), torch.optim.AdamW(full, lr=1e-4)
    for step in range(4):
        for p, q, g in zip(mine, full, _grads(mine, step)):
            p.grad, q.grad = g, g.float()
        a.step(), b.step()
    for p, q in zip(mine, full):
        assert torch.equal(p, q.to(dtype)) and torch.equal(a.state[p]["master"], q)


def test_unaligned_parameters():
    """Views that start at any element are stepped the same."""
    flat = torch.randn(20_000, device=DEV)
    for bits in (32, 8):
        for off in (0, 1, 3):
            p = flat[off:off + 9001].detach().requires_grad_(True)
            q = flat[off:off + 9001].clone().requires_grad_(True)
            assert p.data_ptr() % 16 == off * 4 % 16
            a, b = (optim.AdamW([t], lr=0.0, weight_decay=0.0, state_bits=bits) for t in (p, q))
            for step in range(2):
                p.grad = _grads([p], step)[0]
                q.grad = torch.zeros(9002, device=DEV)[1:].copy_(p.grad)
                a.step(), b.step()
            assert a.state[p].pop("step") == b.state[q].pop("step") == 2
            for name, t in a.state[p].items():
                other = b.state[q][name]
                view = (lambda z: z.view(torch.uint8)) if t.element_size() == 1 else (lambda z: z)
                assert torch.equal(view(t), view(other)), name


def _expected(p, g, mean, root, step, lr, beta1, beta2, eps, decay):
    """(p, mean, root) after a step, in float64."""
    mean = beta1 * mean + (1 - beta1) * g
    root = np.sqrt(beta2 * root ** 2 + (1 - beta2) * g ** 2)
    p = p * (1 - lr * decay) - lr / (1 - beta1 ** step) * mean / (
        root / np.sqrt(1 - beta2 ** step) + eps)
    return p, mean, root


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [4096, 5000, 100_003])
def test_8_bit_states(n, dtype):
    lr, betas, eps, decay = 1e-2, (0.9, 0.99), 1e-8, 0.05
    (p,) = _params([(n,)], dtype, n)
    opt = optim.AdamW([p], lr, betas, eps, decay, state_bits=8)
    for step in range(1, 6):
        (g,) = _grads([p], step)
        # Runs of very different sizes, and one of zeros.
        g[: n // 3] *= 1e-3
        g[256:512] = 0
        p.grad = g
        if step == 1:
            before, mean, root = p.detach().float().clone(), np.zeros(n), np.zeros(n)
        else:
            before = state["master" if dtype != torch.float32 else "p"].clone()
            wide = lambda name: np.repeat(  # noqa: E731
                state[name + "_scale"].cpu().double().numpy(), 256)[:n]
            mean = state["exp_avg"].float().cpu().double().numpy() * wide("exp_avg")
            root = state["exp_avg_sq_root"].float().cpu().double().numpy() \
                * wide("exp_avg_sq_root")
        opt.step()
        state = dict(opt.state[p], p=p.detach().clone())
        want, mean, root = _expected(before.cpu().double().numpy(), g.cpu().double().numpy(), mean,
                                     root, step, lr, *betas, eps, decay)
        got = state["master" if dtype != torch.float32 else "p"].cpu().double().numpy()
        # A step is a product of a dozen float32 operations whose scalars are rounded:
        # 24 u of it, and two roundings of the parameter.  The mean's two terms may
        # cancel; the root is at least sqrt(1 - beta2) = 0.1 of |g| and so of each.
        change = lr / (1 - betas[0] ** step) * (np.abs(mean) + np.abs(g.cpu().double().numpy())) / (
            root / np.sqrt(1 - betas[1] ** step) + eps)
        assert (np.abs(got - want) <= 24 * U * change + 3 * U * np.abs(want) + 1e-30).all()
        if dtype != torch.float32:
            assert torch.equal(p.detach(), state["master"].to(dtype))
        r = ref.chance(n, step)
        for name, exact, chance, is_root in (("exp_avg", mean, r & 0xFFFF, False),
                                             ("exp_avg_sq_root", root, r >> 16, True)):
            codes, scales = ref.quantize(exact, chance.astype(np.float64), is_root)
            found = state[name + "_scale"].cpu().double().numpy()
            # The largest of a run is off by the roundings of its own sums.
            assert (np.abs(found - scales) <= 1e-5 * scales).all(), name
            held = state[name].float().cpu().double().numpy()
            size = np.abs(exact) / np.repeat(scales, 256)[:n]
            # A value next to where chance cuts may fall on the other side: one code off.
            assert (np.abs(held - codes) <= 2 * ref.code_step(size) * (held != codes)).all()
            assert (held != codes).mean() < 1e-3, name
            if is_root:
                assert (held[exact > 0] > 0).all()
            # Rounding by chance is right on average: the errors' mean is that of n
            # independent ones below a step each, 5 deviations at most.
            step_size = ref.code_step(size)
            off = (held - size * np.sign(exact) if not is_root else held - size) / step_size
            inside = (exact != 0) & (size > 2.0 ** -6) & (size < 440)
            assert abs(off[inside].mean()) < 5 * 0.5 / np.sqrt(inside.sum()), name


def test_8_bit_averages_move_when_a_step_is_less_than_half_a_code():
    n = 8192
    p = torch.zeros(n, device=DEV, requires_grad=True)
    opt = optim.AdamW([p], lr=0.0, betas=(0.9, 0.99), state_bits=8)
    g = torch.full((n,), 1.0, device=DEV)
    g[::256] = 4.0  # holds the scale
    for _ in range(300):
        p.grad = g
        opt.step()
    s = opt.state[p]
    root = s["exp_avg_sq_root"].float() * s["exp_avg_sq_root_scale"].repeat_interleave(256)
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[::256] = False
    # sqrt(1 - 0.99^300) = 0.975; to nearest it would stay at the first code whose
    # step 1 % of the way does not leave.
    assert abs(float(root[rest].mean()) - 0.975) < 0.03


def test_gradients_that_are_not_finite_stay_in_their_element():
    p = torch.zeros(8192, device=DEV, requires_grad=True)
    opt = optim.AdamW([p], lr=1e-2, state_bits=8)
    for _ in range(2):
        p.grad = torch.ones_like(p)
        p.grad[700], p.grad[701] = float("nan"), float("inf")
        opt.step()
    bad = torch.zeros(8192, dtype=torch.bool, device=DEV)
    bad[700:702] = True
    assert torch.equal(torch.isfinite(p.detach()), ~bad)
    for name in ("exp_avg", "exp_avg_sq_root"):
        assert torch.equal(torch.isnan(opt.state[p][name].float()), bad)
        assert torch.isfinite(opt.state[p][name + "_scale"]).all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_and_loaded_states_go_on_the_same(bits, dtype):
    shapes = [(100, 50), (7, 3)]
    mine = _params(shapes, dtype)
    opt = optim.AdamW(mine, state_bits=bits)
    for step in range(2):
        for p, g in zip(mine, _grads(mine, step)):
            p.grad = g
        opt.step()
    other = [p.detach().clone().requires_grad_(True) for p in mine]
    again = optim.AdamW(other, state_bits=bits)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    for step in range(2, 4):
        for p, q, g in zip(mine, other, _grads(mine, step)):
            p.grad, q.grad = g, g
        opt.step(), again.step()
    for p, q in zip(mine, other):
        assert torch.equal(p, q)
        assert opt.state[p].pop("step") == again.state[q].pop("step") == 4
        for name, t in opt.state[p].items():
            o = again.state[q][name]
            assert o.dtype == t.dtype
            if t.element_size() == 1:
                t, o = t.view(torch.uint8), o.view(torch.uint8)
            assert torch.equal(t, o), name


def test_two_groups_on_another_stream():
    mine, theirs = _params([(300, 20), (5,)], torch.float32), _params([(300, 20), (5,)],
                                                                      torch.float32)
    side = torch.cuda.Stream()
    groups = lambda ps: [dict(params=ps[:1], lr=1e-2), dict(params=ps[1:], eps=1e-4)]  # noqa: E731
    a, b = optim.AdamW(groups(mine)), torch.optim.AdamW(groups(theirs))
    for p, q, g in zip(mine, theirs, _grads(mine, 0)):
        p.grad, q.grad = g, g.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(mine, theirs))


def test_refusals():
    p = torch.zeros(5000, device=DEV, requires_grad=True)
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p], state_bits=8)
    with pytest.raises(RuntimeError, match="captured"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    opt.state[p]["exp_avg_scale"] = opt.state[p]["exp_avg_scale"][:3]
    with pytest.raises(RuntimeError, match="'exp_avg_scale' does not match"):
        opt.step()
    for q, kind in ((torch.zeros(4, 4, device=DEV).t()[:, :2], "contiguous"),
                    (torch.zeros(4), "CUDA"), (torch.zeros(4, device=DEV).double(), "float32")):
        q = q.detach().requires_grad_(True)
        q.grad = torch.ones_like(q)
        with pytest.raises(NotImplementedError, match=kind):
            optim.AdamW([q]).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_changed_after_a_step(bits):
    """The same parameter object with other memory behind it: another address is
    followed, another type or device refused before anything is launched."""
    p = torch.nn.Parameter(torch.ones(8192, device="cuda"))
    optimizer = optim.AdamW([p], lr=1e-2, state_bits=bits)
    p.grad = torch.ones_like(p)
    optimizer.step()
    before, old = p.detach().clone(), p.data
    p.data = old.clone()
    optimizer.step()
    assert torch.equal(old, before) and bool((p < before).all())
    p.data = p.data.half()
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="master"):
        optimizer.step()
    p.data = p.data.float().cpu()
    p.grad = torch.ones_like(p)
    with pytest.raises(NotImplementedError):
        optimizer.step()
    p.data = old
    p.grad = torch.ones_like(p)
    optimizer.state[p]["exp_avg"].data = torch.zeros(4096, device="cuda")
    with pytest.raises(RuntimeError, match="exp_avg"):
        optimizer.step()
