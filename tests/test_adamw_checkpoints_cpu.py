"""AdamW's bookkeeping without a GPU: what a refused step leaves behind."""

import pytest
import torch

from r2splat import optim


def test_a_refused_step_makes_no_state():
    """A parameter that the kernel does not take is refused before it has a state."""
    p = torch.zeros(5000, requires_grad=True)
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p], state_bits=8)
    with pytest.raises(NotImplementedError, match="CUDA parameters"):
        opt.step()
    assert not opt.state


def _torch_checkpoint(kind=torch.optim.AdamW, second=False, **options):
    """torch's state of two parameters, the second with or without a gradient."""
    ps = [torch.nn.Parameter(torch.ones(6)), torch.nn.Parameter(torch.ones(5000))]
    opt = kind(ps, lr=0.25, **options)
    for p in ps[:1 + second]:
        p.grad = torch.full_like(p, 0.5)
    opt.step()
    return opt.state_dict()


def _mine(**options):
    ps = [torch.nn.Parameter(torch.ones(6)), torch.nn.Parameter(torch.ones(5000))]
    return ps, optim.AdamW(ps, **options)


def test_a_checkpoint_of_torch_keeps_the_states_bits():
    """torch's groups know no state_bits: a parameter that had no gradient before the
    save gets the states that this optimizer was made with."""
    ps, opt = _mine(state_bits=8)
    opt.load_state_dict(_torch_checkpoint())
    (group,) = opt.param_groups
    assert group["state_bits"] == 8 and group["lr"] == 0.25
    assert set(opt.state[ps[0]]) == {"step", "exp_avg", "exp_avg_sq"} and ps[1] not in opt.state
    assert torch.equal(opt.state[ps[0]]["exp_avg"], torch.full((6,), 0.5 * (1 - 0.9)))
    # The kernel is not there for CPU parameters, and nothing else is amiss.
    ps[1].grad = torch.ones(5000)
    with pytest.raises(NotImplementedError, match="CUDA parameters"):
        opt.step()
    # One's own checkpoint brings its own.
    _, other = _mine(state_bits=32)
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["state_bits"] == 8


@pytest.mark.parametrize("option", ["amsgrad", "maximize", "capturable", "differentiable"])
def test_what_the_step_does_not_do_is_refused_and_not_dropped(option):
    checkpoint = _torch_checkpoint()
    checkpoint["param_groups"][0][option] = True
    ps, opt = _mine()
    before = opt.state_dict()
    with pytest.raises(NotImplementedError, match=option):
        opt.load_state_dict(checkpoint)
    assert opt.state_dict() == before and not opt.state
    # Nor by a group of its own, from the start or later on.
    extra = torch.nn.Parameter(torch.ones(3))
    with pytest.raises(NotImplementedError, match=option):
        optim.AdamW([{"params": [extra], option: True}])
    with pytest.raises(NotImplementedError, match=option):
        opt.add_param_group({"params": [extra], option: True})
    assert len(opt.param_groups) == 1
    opt.param_groups[0][option] = True
    with pytest.raises(NotImplementedError, match=option):
        opt.step()


def test_coupled_decay_is_refused_where_there_is_any():
    _, opt = _mine()
    with pytest.raises(NotImplementedError, match="decoupled_weight_decay"):
        opt.load_state_dict(_torch_checkpoint(torch.optim.Adam, weight_decay=0.1))
    opt.load_state_dict(_torch_checkpoint(torch.optim.Adam))  # without, Adam is AdamW


def test_bits_of_a_group():
    p = torch.nn.Parameter(torch.ones(3))
    with pytest.raises(ValueError, match="state_bits must be 8 or 32, got 16"):
        optim.AdamW([{"params": [p], "state_bits": 16}])
    _, opt = _mine()
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group({"params": [p], "state_bits": 4})
    checkpoint = opt.state_dict()
    checkpoint["param_groups"][0]["state_bits"] = None
    with pytest.raises(ValueError, match="state_bits"):
        opt.load_state_dict(checkpoint)
    opt.add_param_group({"params": [p], "state_bits": 8})
    assert [g["state_bits"] for g in opt.param_groups] == [32, 8]


def test_hooks_of_loading_see_and_change_what_is_loaded():
    ps, opt = _mine()
    seen = []

    def half(optimizer, state_dict):
        """The caller's own change, in a dictionary of its own."""
        states = {i: {k: t * 0.5 if k == "exp_avg" else t for k, t in s.items()}
                  for i, s in state_dict["state"].items()}
        groups = [{**g, "lr": 7.0} for g in state_dict["param_groups"]]
        return {**state_dict, "state": states, "param_groups": groups}

    opt.register_load_state_dict_pre_hook(half)
    opt.register_load_state_dict_post_hook(
        lambda optimizer: seen.append({p: dict(s) for p, s in optimizer.state.items()}))
    checkpoint = _torch_checkpoint(second=True)
    wanted = {i: s["exp_avg"].clone() * 0.5 for i, s in checkpoint["state"].items()}
    for times in (1, 2):  # nothing of a load stays behind for the next
        opt.load_state_dict(checkpoint)
        assert opt.param_groups[0]["lr"] == 7.0
        for i, p in enumerate(ps):
            assert torch.equal(opt.state[p]["exp_avg"], wanted[i])
            assert opt.state[p]["exp_avg"] is seen[-1][p]["exp_avg"]
        assert len(seen) == times

    def bad(optimizer, state_dict):
        state_dict["param_groups"] = [{**g, "maximize": True} for g in state_dict["param_groups"]]

    handle = opt.register_load_state_dict_pre_hook(bad)
    with pytest.raises(NotImplementedError, match="maximize"):
        opt.load_state_dict(checkpoint)
    handle.remove()
    opt.load_state_dict(checkpoint)
    assert len(seen) == 3 and not checkpoint["param_groups"][0]["maximize"]


def test_post_hooks_see_the_types_that_were_saved():
    """A 16-bit parameter's states are float32, before and after the hooks."""
    def make():
        p = torch.nn.Parameter(torch.ones(4, dtype=torch.bfloat16))
        return p, optim.AdamW([p])

    p, opt = make()
    saved = opt.state_dict()
    saved["state"] = {0: {"step": 3, "master": torch.full((4,), 1 + 2.0 ** -12),
                          "exp_avg": torch.full((4,), 2.0 ** -20 + 1),
                          "exp_avg_sq": torch.full((4,), 0.5)}}
    q, other = make()
    types = []
    other.register_load_state_dict_post_hook(
        lambda o: types.extend((k, t.dtype) for k, t in o.state[q].items() if k != "step"))
    other.load_state_dict(saved)
    assert types and all(t == torch.float32 for _, t in types)
    assert torch.equal(other.state[q]["master"], saved["state"][0]["master"])
    assert other.state[q]["master"] is not saved["state"][0]["master"]
