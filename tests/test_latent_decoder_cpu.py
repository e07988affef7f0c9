"""A latent decoder's blocks without a GPU: what casting the module does to them."""

import copy

import pytest
import torch

from r2splat.latent import LatentDecoder


def _decays(decoder):
    return [b.log_decay for b in decoder.blocks]


@pytest.mark.parametrize("cast", [
    lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
    lambda m: m.bfloat16().float(), lambda m: m.type(torch.float16), lambda m: copy.deepcopy(m).half(),
    lambda m: torch.nn.Sequential(m).half()[0]],
    ids=["to", "half", "double", "there-and-back", "type", "copied", "inside"])
def test_decays_stay_float32_whatever_the_module_is_cast_to(cast):
    decoder = LatentDecoder(4, 2, width=24, heads=4, blocks=2)
    want = [d.clone() for d in _decays(decoder)]
    decoder.blocks[1].log_decay.mul_(0.5)  # one's own decays are kept as well
    want[1] *= 0.5
    cast_to = cast(decoder)
    for d, w in zip(_decays(cast_to), want):
        assert d.dtype == torch.float32 and torch.equal(d, w)
    assert "blocks.0.log_decay" in dict(cast_to.named_buffers())


def test_decays_are_float32_under_another_default_type():
    want = _decays(LatentDecoder(4, 2, width=24, heads=4, blocks=1))[0]
    torch.set_default_dtype(torch.float64)
    try:
        got = _decays(LatentDecoder(4, 2, width=24, heads=4, blocks=1))[0]
    finally:
        torch.set_default_dtype(torch.float32)
    assert got.dtype == torch.float32 and torch.equal(got, want)
