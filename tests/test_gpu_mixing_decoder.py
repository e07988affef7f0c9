"""The decoder with mixing blocks, and its operators together as it uses them, on
the GPU against a float64 restatement in elementary torch.

A gradient has gone through a dozen operators; how far float32 takes it is not
written down term by term but measured: the same restatement in float32 on the CPU
shows it, and the kernels may be eight times as far (they round elsewhere, and
their sums run in another order)."""

import math

import pytest
import torch

from r2splat import geometry, optim, scenes
from r2splat.latent import LatentDecoder
from r2splat.ops import explicit, latent

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _norm(x):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def _turn(x, positions, sections):
    pairs = sum(sections)
    rate = torch.cat([torch.tensor([1e4 ** (-i / m) for i in range(m)], dtype=torch.float64)
                      for m in sections])
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    angle = (positions.double()[:, axis] * rate)[:, None].to(x.dtype)
    a, b, rest = x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]
    cos, sin = torch.cos(angle), torch.sin(angle)
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _attend(q, k, v, log_decay, back):
    """Every pair of tokens at once."""
    n = q.shape[0]
    apart = torch.arange(n)[:, None] - torch.arange(n)
    apart = -apart if back else apart
    weight = torch.where(apart[None] >= 0, torch.exp(
        log_decay.double()[:, None, None] * apart.clamp(min=0)), 0.0).to(q.dtype)
    scores = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * weight
    return torch.matmul(scores, v.transpose(0, 1).contiguous()).transpose(0, 1) \
        * q.shape[-1] ** -0.5


def _scan(x, gate, back):
    a, h, out = torch.sigmoid(gate), torch.zeros_like(x[0]), [None] * x.shape[0]
    order = range(x.shape[0])
    for t in (reversed(order) if back else order):
        h = a[t] * h + (1 - a[t]) * x[t]
        out[t] = h
    return torch.stack(out)


def _restated(decoder, p, codes, levels, means):
    """The decoder's formulas, with parameters p by name."""
    x, gate = decoder.scale * p["codebook"][codes], decoder.scale * p["gates"][codes]
    x = x + _scan(x, gate, False) + _scan(x, gate, True)
    positions = means.float() * decoder.position_scale
    for i, block in enumerate(decoder.blocks):
        u = _norm(x) * p[f"norms.{i}"]
        n, width = u.shape
        q, k, v, gate = (u @ p[f"blocks.{i}.inward"].T).split(width, dim=1)
        q, k, v = (t.reshape(n, block.heads, -1) for t in (q, k, v))
        q, k = (_turn(t, positions, block.sections) for t in (q, k))
        half, decay = block.heads // 2, block.log_decay.cpu()
        mixed = torch.cat([_attend(q[:, :half], k[:, :half], v[:, :half], decay[:half], False),
                           _attend(q[:, half:], k[:, half:], v[:, half:], decay[half:], True)], 1)
        update = mixed.reshape(n, width) @ p[f"blocks.{i}.outward"].T
        x = x + torch.sigmoid(gate) * _norm(update) * p[f"blocks.{i}.post"] \
            / math.sqrt(len(decoder.blocks))
    return torch.einsum("nmk,nk->nm", p["weight"][levels], x) + p["bias"][levels]


def _decoder(n, levels, width, heads, seed):
    g = torch.Generator().manual_seed(seed)
    decoder = LatentDecoder(50, levels, width, g, blocks=2, heads=heads)
    with torch.no_grad():
        decoder.weight.copy_(torch.randn(decoder.weight.shape, generator=g) * 0.2)
        decoder.norms[1].copy_(1 + 0.2 * torch.randn(width, generator=g))
    codes = torch.randint(0, 50, (n,), generator=g)
    level = torch.randint(0, levels, (n,), generator=g)
    return decoder, codes, level, torch.randn(n, 3, generator=g), torch.randn(n, 11, generator=g)


@pytest.mark.parametrize("n,width,heads", [(1, 12, 2), (150, 24, 2), (333, 64, 4)])
def test_decoder_and_its_gradients_against_float64(n, width, heads):
    decoder, codes, level, means, v = _decoder(n, 3, width, heads, n)
    found = {}
    for dtype in (torch.float64, torch.float32):
        p = {name: t.detach().to(dtype).requires_grad_(True)
             for name, t in decoder.named_parameters()}
        raw = _restated(decoder, p, codes, level, means)
        grads = torch.autograd.grad((raw * v.to(dtype)).sum(), list(p.values()))
        found[dtype] = {"raw": raw.detach(), **dict(zip(p, grads))}
    decoder = decoder.to(DEV)
    rows, offsets = latent.group_rows(level.to(DEV), 3)
    raw = decoder(codes.to(DEV), rows, offsets, means.to(DEV))
    raw.backward(v.to(DEV))
    got = {"raw": raw.detach(), **{name: t.grad for name, t in decoder.named_parameters()}}
    exact, single = found[torch.float64], found[torch.float32]
    for name, t in got.items():
        size = float(exact[name].norm())
        far = float((t.cpu().double() - exact[name]).norm())
        plain = float((single[name].double() - exact[name]).norm())
        assert far <= 8 * plain + 1e-6 * size, (name, far / size, plain / size)


def test_decoder_without_blocks_is_as_it_was():
    a = LatentDecoder(10, 3, 16, torch.Generator().manual_seed(1))
    b = LatentDecoder(10, 3, 16, torch.Generator().manual_seed(1), blocks=1, heads=2)
    for name, p in a.named_parameters():
        assert torch.equal(p, dict(b.named_parameters())[name])
    assert set(dict(a.named_parameters())) == {"codebook", "gates", "weight", "bias"}


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_training_steps_through_the_renderer(dtype, bits):
    """Decode, render, the explicit backward and AdamW, a few times over."""
    n, levels, width = 2000, 3, 64
    g = torch.Generator().manual_seed(7)
    base = scenes.random_gaussians(n, g, -3.2, 0.3).to(DEV)
    views, Ks = (t.to(DEV) for t in geometry.cone_beam_views([0.3], 64))
    codes = torch.randint(0, 80, (n,), generator=g).to(DEV)
    rows, offsets = latent.group_rows(torch.randint(0, levels, (n,), generator=g).to(DEV), levels)
    decoder = LatentDecoder(80, levels, width, g, dtype=dtype, blocks=2).to(DEV)
    opt = optim.AdamW(decoder.parameters(), lr=3e-3, state_bits=bits)
    before = [p.detach().clone() for p in decoder.parameters()]
    for step in range(3):
        opt.zero_grad()
        raw = decoder(codes, rows, offsets, base.means)
        if step == 0:
            assert not raw.any()  # the base as it is
        leaves = decoder.leaves(base, raw)
        means, quats, scales, opacities = leaves
        state = explicit.prepare_explicit_gaussians(quats, scales, opacities, scale_min=5e-4,
                                                    scale_max=1.0)
        image = explicit.explicit_rasterize(state, means, views, Ks, img_w=64, img_h=64,
                                            tile_size=16, eps2d=1e-8, radius_clip=3.0,
                                            absgrad=True).image
        image.square().mean().backward()
        explicit.explicit_backward(state, means, quats, scales, opacities)
        decoder.backward(raw, *leaves)
        for name, p in decoder.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all(), name
        opt.step()
    assert all(torch.isfinite(p).all() for p in decoder.parameters())
    # The first step's gradient stops at the zero output weights; by the third
    # all parameters have moved.
    assert all(not torch.equal(a, p) for a, p in zip(before, decoder.parameters()))


def test_decoder_refuses_what_does_not_fit():
    with pytest.raises(ValueError, match="do not make"):
        LatentDecoder(10, 3, 16, blocks=1, heads=3)
    with pytest.raises(ValueError, match="do not make"):
        LatentDecoder(10, 3, 16, blocks=1, heads=4)
    decoder = LatentDecoder(10, 3, 12, blocks=1, heads=2).to(DEV)
    codes = torch.zeros(5, dtype=torch.int64, device=DEV)
    rows, offsets = latent.group_rows(codes, 3)
    with pytest.raises(RuntimeError, match="needs the means"):
        decoder(codes, rows, offsets)
