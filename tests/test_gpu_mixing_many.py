"""The mixing operators where their blocks are more than one launch's grid has room
for (2^32 threads): the same bits as the same call in two halves."""

import pytest
import torch

from r2splat.cuda import _wrapper as W
from r2splat.ops import latent

pytestmark = pytest.mark.gpu
DEV = "cuda"
GRID = 2 ** 32 // 256  # blocks of 256 threads that one launch does not hold


@pytest.mark.parametrize("dv,dtype", [(4, torch.bfloat16), (1, torch.float32)])
def test_step_of_more_states_than_a_grid_holds(dv, dtype):
    h, dk = 8, 4
    b = GRID // h + 3
    torch.manual_seed(0)
    q, k = (torch.randn(b, h, dk, device=DEV, dtype=dtype) for _ in range(2))
    v = torch.randn(b, h, dv, device=DEV, dtype=dtype)
    state = torch.randn(b, h, dk, dv, device=DEV)
    log_decay = -torch.rand(h, device=DEV)
    y, final = latent.decay_attention_step(q, k, v, log_decay, state)
    for part in (slice(None, b // 2), slice(b // 2, None)):
        y_part, final_part = latent.decay_attention_step(q[part], k[part], v[part], log_decay,
                                                         state[part])
        assert torch.equal(y[part], y_part) and torch.equal(final[part], final_part)
    # The last sequence's, whose states are in the second launch.
    want = torch.exp(log_decay)[:, None, None] * state[-1] + (
        k[-1, :, :, None].float() * v[-1, :, None].float())
    assert torch.allclose(final[-1], want, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_rotary_of_more_tokens_than_a_grid_holds(dtype):
    """A block to a token from 513 pairs on.  One row of queries for all tokens, so
    that only the outputs (34 GB) are large."""
    n, pairs = GRID + 40, 513
    torch.manual_seed(1)
    row = torch.randn(1, 1, 2 * pairs, device=DEV, dtype=dtype)
    places = torch.randint(0, 1000, (n, 1), device=DEV, dtype=torch.int32)
    out, _ = latent.rotary_axes(row.expand(n, 1, 2 * pairs), None, places, (pairs,))
    for part in (slice(0, 50), slice(GRID // 2, GRID // 2 + 50), slice(GRID - 30, None)):
        count = places[part].shape[0]
        want, _ = latent.rotary_axes(row.expand(count, 1, 2 * pairs), None, places[part], (pairs,))
        assert torch.equal(out[part], want)
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("ragged", [False, True])
def test_attention_of_more_sequences_than_a_grid_holds(ragged):
    b, d = GRID + 21, 2
    torch.manual_seed(2)
    q, k, v, v_y = (torch.randn(b, 1, d, device=DEV) for _ in range(4))
    log_decay, scale = torch.tensor([-0.3], device=DEV), 0.7

    def both(part):
        """Outputs, last states and gradients of some of the sequences, of a token each."""
        args = [t[part] for t in (q, k, v, v_y)]
        count = args[0].shape[0]
        offsets = torch.arange(count + 1, device=DEV, dtype=torch.int32) if ragged else None
        args = args if ragged else [t[:, None] for t in args]
        y, final, kept = W.decay_attention_fwd(*args[:3], log_decay, None, offsets, False, scale)
        grads = W.decay_attention_bwd(*args[:3], log_decay, None, offsets, kept, args[3], None,
                                      False, scale)
        return [t.reshape(count, -1) for t in (y, final, *grads)]

    got = both(slice(None))
    for part in (slice(None, b // 2), slice(b // 2, None)):
        assert all(torch.equal(a[part], w) for a, w in zip(got, both(part)))
    score = scale * (q * k).sum(-1)
    assert torch.allclose(got[0], score * v[:, 0], rtol=1e-5, atol=1e-5)
    assert torch.allclose(got[4], score * v_y[:, 0], rtol=1e-5, atol=1e-5)
