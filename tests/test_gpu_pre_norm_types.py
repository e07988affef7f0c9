"""pre_norm and its gradients in every type against float64, bounds by the oracle's
count of float32 roundings and half a step of the output's type."""

import pytest
import torch

from oracle import mixing as ref
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def _close(got, exact, dtype, what):
    got, half = got.detach().cpu().double().numpy(), torch.finfo(dtype).eps / 2
    tol = exact.e + half * (abs(exact.v) + exact.e) + TINY[dtype]
    assert got.shape == exact.v.shape and (abs(got - exact.v) <= tol).all(), what


@pytest.mark.parametrize("centered", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (70, 50), (300, 64), (9, 1030), (4, 8192)])
def test_pre_norm_and_gradients(n, d, dtype, centered):
    g = torch.Generator().manual_seed(n + d)
    x = (torch.randn(n, d, generator=g) * 3 + 1).to(dtype)
    weight, v_u = (torch.randn(*s, generator=g).to(dtype) for s in ((d,), (n, d)))
    exact = ref.residual_norm(x.double().numpy(), None, None, None, weight.double().numpy(), None,
                              v_u.double().numpy(), 1.0, 1e-5, centered)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, weight)]
    u = latent.pre_norm(*leaves, 1e-5, centered)
    _close(u, exact["u"], dtype, "u")
    v_x, v_weight = torch.autograd.grad(u, leaves, v_u.to(DEV))
    _close(v_x, exact["v_x"], dtype, "v_x")
    _close(v_weight, exact["v_w2"], dtype, "v_weight")
    plain = W.residual_norm_fwd(x.to(DEV), None, None, None, weight.to(DEV), 1.0, 1e-5, centered)
    assert torch.equal(plain[1], u) and plain[0].dtype == dtype
