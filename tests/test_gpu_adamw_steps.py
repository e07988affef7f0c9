"""AdamW on the GPU: steps that are refused, and what they leave as it was."""

import pytest
import torch

from r2splat import optim

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _held(opt):
    """Every state's values, by parameter."""
    return [{name: t.clone() if isinstance(t, torch.Tensor) else t
             for name, t in opt.state.get(p, {}).items()}
            for group in opt.param_groups for p in group["params"]]


def _same(a, b):
    bits = lambda t: t.view(torch.uint8) if t.element_size() == 1 else t  # noqa: E731
    return len(a) == len(b) and all(
        x.keys() == y.keys() and all(
            torch.equal(bits(x[k]), bits(y[k])) if isinstance(x[k], torch.Tensor) else x[k] == y[k]
            for k in x)
        for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_refused_step_leaves_counts_states_and_parameters(dtype, bits):
    """A later parameter is refused: the earlier ones, with and without a state, are
    as they were, and going on after the mend is as if the step had not been tried."""
    def make():
        ps = [torch.full((n,), 0.5, device=DEV).to(dtype).requires_grad_(True)
              for n in (6000, 50, 6000, 7)]
        return ps, optim.AdamW([dict(params=ps[:2]), dict(params=ps[2:], lr=1e-2)],
                               state_bits=bits)

    (ps, opt), (others, other) = make(), make()
    for qs, o in ((ps, opt), (others, other)):
        for q in qs[::2]:
            q.grad = torch.ones_like(q)
        o.step()
        for q in qs:  # two have no state yet
            q.grad = torch.full_like(q, 0.25)
    before, values = _held(opt), [p.detach().clone() for p in ps]
    assert [bool(s) for s in before] == [True, False, True, False]

    def refused(error, match):
        with pytest.raises(error, match=match):
            opt.step()
        assert _same(_held(opt), before)
        assert len(opt.state) == 2
        assert all(torch.equal(p, v) for p, v in zip(ps, values))

    good, ps[3].grad = ps[3].grad, None
    ps[3].grad = torch.sparse_coo_tensor([[1]], [1.0], (7,), device=DEV).to(dtype)
    refused(RuntimeError, "sparse")
    ps[3].grad = good
    opt.param_groups[1]["eps"] = torch.tensor(1e-8)
    refused(NotImplementedError, "float eps")
    opt.param_groups[1]["eps"] = 1e-8
    kept = opt.state[ps[2]]["exp_avg"]
    opt.state[ps[2]]["exp_avg"] = before[2]["exp_avg"] = kept[:10]
    refused(RuntimeError, "'exp_avg' does not match")
    opt.state[ps[2]]["exp_avg"] = kept
    for o in (opt, other):
        o.step()
    assert _same(_held(opt), _held(other))
    assert all(torch.equal(p, q) for p, q in zip(ps, others))
    assert [opt.state[p]["step"] for p in ps] == [2, 1, 2, 1]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [50, 6001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_is_written_to_a_16_bit_parameter_is_taken_up(dtype, n, bits):
    """Between steps some elements are written, by whatever way, and the others keep
    their copies' bits; a step after that goes on from the written values."""
    g = torch.Generator().manual_seed(n + bits)
    p = torch.randn(n, generator=g).to(dtype).to(DEV).requires_grad_(True)
    opt = optim.AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
    for _ in range(3):
        p.grad = torch.randn(n, generator=g).to(dtype).to(DEV)
        opt.step()
    master = opt.state[p]["master"]
    assert not torch.equal(master, p.detach().float())  # holds more than the parameter
    opt.param_groups[0]["lr"] = 0.0  # the step alone writes nothing now
    p.grad = torch.zeros_like(p)
    held, value = master.clone(), p.detach().clone()
    opt.step()
    assert torch.equal(master, held) and torch.equal(p.detach(), value)
    written = torch.arange(n, device=DEV) % 7 == 3
    with torch.no_grad():
        p[written] = -2.5
    p.data[0] = 0.0
    p.data[5] = float("nan")
    written[0] = written[5] = True
    value = p.detach().clone()
    opt.step()
    want = torch.where(written, value.float(), held)
    assert torch.equal(master.nan_to_num(9.0), want.nan_to_num(9.0))
    assert torch.equal(p.detach().nan_to_num(9.0), value.nan_to_num(9.0))
    # A model's checkpoint, loaded after the optimizer's.
    fresh = torch.linspace(-3, 3, n, device=DEV).to(dtype)
    with torch.no_grad():
        p.copy_(fresh)
    opt.step()
    assert torch.equal(p.detach(), fresh)
    same = held.to(dtype) == fresh  # there is nothing to tell these by
    assert torch.equal(master[~same], fresh.float()[~same])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_finite_gradients_leave_8_bit_states_finite(dtype):
    """The square of a gradient beyond 1.8e19 is none of float32's numbers, its root is:
    sqrt(beta2) to a step of it, times the codes' step at the least."""
    p = torch.zeros(8192, device=DEV, dtype=dtype, requires_grad=True)
    opt = optim.AdamW([p], lr=1e-2, betas=(0.9, 0.99), weight_decay=0.0, state_bits=8)
    large = torch.tensor([1e19, 2e19, 1e25, 1e30, -3e38], device=DEV)
    at = torch.tensor([300, 1000, 2001, 4100, 8000], device=DEV)  # runs of their own
    root = torch.zeros(5, device=DEV, dtype=torch.float64)
    mean = torch.zeros(5, device=DEV, dtype=torch.float64)
    for step in range(3):
        p.grad = torch.ones_like(p)
        p.grad[at] = large.to(dtype) if step < 2 else torch.ones(5, device=DEV, dtype=dtype)
        g = p.grad[at].double()
        opt.step()
        s = opt.state[p]
        root = (0.99 * root ** 2 + 0.01 * g ** 2).sqrt()
        mean = 0.9 * mean + 0.1 * g
        for name, exact in (("exp_avg", mean), ("exp_avg_sq_root", root)):
            assert torch.isfinite(s[name].float()).all() and torch.isfinite(s[name + "_scale"]).all()
            found = s[name].float()[at].double() * s[name + "_scale"][at // 256].double()
            # The largest of its run has the largest code, 448, and no chance: what is
            # off is the scale's roundings alone, a few units of float32 a step.
            assert ((found - exact).abs() <= (step + 1) * 16 * 2.0 ** -24 * exact.abs()).all(), name
        assert torch.isfinite(p.detach()).all()
    # lr mean / root, corrected: 0.1 / 0.1 in the first step.  (A root beyond 2^126 has
    # no reciprocal among float32's normal numbers: no step.)
    assert (p.detach()[at[:4]].float().abs() > 0.5e-2).all()
