"""Decay attention on the GPU: last states to float32's own precision, and calls whose
offsets ask for more than there is, which write nothing outside their tensors."""

import numpy as np
import pytest
import torch

from oracle.mixing import DecayAttention
from r2splat.cuda import _wrapper as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [16, 33, 64, 128])
@pytest.mark.parametrize("length", [1, 2, 4])
def test_states_are_float32_with_16_bit_inputs(length, d, dtype):
    """Sequences so short that rounding the decayed values to two 16-bit parts would
    show: to nearest, a part of 8 bits leaves half a step, 2^-8 of the value, two leave
    2^-8 half a step of that rest's power of two, 2^-17 = 128 u.  The states' own error
    is less: a power of the decay, 4 u and 2 u |log2| of it (weights above 2^-6 here:
    12 u at most, and less of w |log2 w|), two scales and a product of 3 u, what three
    parts leave, 1 u, and a sum of at most 5 products of parts a token, 5 u each."""
    b, h = 50, 2
    g = torch.Generator().manual_seed(d + length)
    q, k, v, v_y = (torch.randn(b * length, h, d, generator=g).to(dtype) for _ in range(4))
    log_decay = -torch.rand(h, generator=g)
    exact = DecayAttention(*(_np(t) for t in (q, k, v, log_decay)),
                           list(range(0, b * length + 1, length)), None, False, 0.3)
    share = (20 + 5 * length) * U
    dev = [t.reshape(b, length, h, d).to(DEV) for t in (q, k, v)]
    y, final, kept = W.decay_attention_fwd(*dev, log_decay.to(DEV), None, None, False, 0.3)
    _, ef, _, fm = exact.forward()
    assert (np.abs(_np(final) - ef) <= share * fm).all()
    v_initial = W.decay_attention_bwd(*dev, log_decay.to(DEV), None, None, kept,
                                      v_y.reshape(b, length, h, d).to(DEV), None, False, 0.3)[3]
    value, mass = exact.backward(_np(v_y))["v_initial"]
    assert (np.abs(_np(v_initial) - value) <= share * mass).all()


class _Margins:
    """torch.empty whose tensors lie inside larger ones full of a pattern."""

    bytes = 1 << 20

    def __init__(self):
        self.held, self.empty = [], torch.empty

    def __call__(self, *shape, dtype=torch.float32, device=None, **kw):
        shape = shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape
        size = int(np.prod(shape, dtype=np.int64)) * torch.tensor([], dtype=dtype).element_size()
        held = self.empty(size + 2 * self.bytes, dtype=torch.uint8, device=device).fill_(0x5A)
        self.held.append((held, size))
        return held[self.bytes:self.bytes + size].view(dtype).view(shape)

    def untouched(self):
        return all(bool((t[:self.bytes] == 0x5A).all())
                   and bool((t[self.bytes + size:] == 0x5A).all()) for t, size in self.held)


@pytest.mark.parametrize("h,dk,dv,dtype", [(1, 8, 8, torch.float32), (5, 16, 16, torch.bfloat16),
                                           (2, 33, 45, torch.float32), (1, 64, 64, torch.float16)])
@pytest.mark.parametrize("bounds", [
    [0, 2000, 0, 2000, 0, 2000], [5, -100, 6000, 7], [2000, 2000, 0], [0, -1], [1, 2],
    [0, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [2000, 0] * 20, [0, 700, 300, 2000]])
def test_offsets_that_do_not_ascend_write_nothing_outside(bounds, h, dk, dv, dtype, monkeypatch):
    n = 2000
    g = torch.Generator().manual_seed(1)
    q, k, v, v_y = (torch.randn(n, h, d, generator=g).to(dtype).to(DEV) for d in (dk, dk, dv, dv))
    inputs = [t.clone() for t in (q, k, v, v_y)]
    log_decay = torch.full((h,), -0.1, device=DEV)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    state = torch.randn(len(bounds) - 1, h, dk, dv, generator=g).to(DEV)
    margins = _Margins()
    monkeypatch.setattr(torch, "empty", margins)
    for reverse in (False, True):
        y, final, kept = W.decay_attention_fwd(q, k, v, log_decay, state, offsets, reverse)
        W.decay_attention_bwd(q, k, v, log_decay, state, offsets, kept, v_y, state, reverse)
    torch.cuda.synchronize()
    assert len(margins.held) >= 14 and margins.untouched()
    assert all(torch.equal(a, b) for a, b in zip(inputs, (q, k, v, v_y)))
