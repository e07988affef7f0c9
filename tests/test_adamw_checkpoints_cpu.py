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
