"""A latent decoder with blocks on the GPU, cast after it was made and over an empty
table."""

import pytest
import torch

from r2splat.latent import LatentDecoder
from r2splat.ops import latent

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(n, levels, dtype):
    g = torch.Generator().manual_seed(n)
    codes = torch.randint(0, 16, (n,), generator=g).to(DEV)
    level = torch.randint(0, levels, (n,), generator=g).to(DEV)
    means = torch.rand(n, 3, generator=g).to(DEV)
    return codes, *latent.group_rows(level, levels), means


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cast_after_it_was_made(dtype):
    """As one that was made in the type."""
    g = torch.Generator().manual_seed(3)
    decoder = LatentDecoder(16, 3, width=24, heads=4, blocks=2, generator=g)
    with torch.no_grad():
        decoder.weight.normal_(generator=g)
    made = LatentDecoder(16, 3, width=24, heads=4, blocks=2, dtype=dtype).to(DEV)
    decoder = decoder.to(DEV).to(dtype)
    made.load_state_dict(decoder.state_dict())
    args = _inputs(200, 3, dtype)
    out = [m(*args) for m in (decoder, made)]
    assert out[0].dtype == dtype and torch.equal(*out) and bool(out[0].any())
    grads = [torch.autograd.grad(o.float().square().sum(), list(m.parameters()))
             for o, m in zip(out, (decoder, made))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("blocks", [0, 2])
def test_an_empty_table(blocks):
    decoder = LatentDecoder(16, 3, width=24, heads=4, blocks=blocks).to(DEV)
    out = decoder(*_inputs(0, 3, torch.float32))
    assert out.shape == (0, 11)
    grads = torch.autograd.grad(out.sum(), list(decoder.parameters()))
    assert all(g.shape == p.shape and not g.any() for g, p in zip(grads, decoder.parameters()))
    with torch.no_grad():
        assert decoder(*_inputs(0, 3, torch.float32)).shape == (0, 11)
