"""The latent decoder's operators at their edges: rows of one vector, states
that are not finite through long sequences, groups of one part and of many.
Same restatement and bounds as test_gpu_latent.py."""

import numpy as np
import pytest
import torch

from oracle import latent as ref
from r2splat.cuda import _lib, _ops
from r2splat.cuda import _wrapper as W
from r2splat.ops import latent
from test_gpu_latent import DEV, TYPES, U, _close, _lookup_case, _np

pytestmark = pytest.mark.gpu


# Every width from one element to more than a vector, over several blocks of
# rows, into memory that holds NaNs: a row that is not written shows.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16, 17])
def test_lookup_writes_every_row(d, wide, dtype):
    n, v, scale = 5003, 37, 1.7
    table, ids, v_out = _lookup_case(n, v, d, dtype, n + d)
    t, i = table.to(DEV), ids.to(torch.int64 if wide else torch.int32).to(DEV)
    lib = _lib.load()
    out = torch.full((n, d), float("nan"), dtype=dtype, device=DEV)
    assert lib.r2s_embedding_fwd(t.data_ptr(), d, i.data_ptr(), int(wide), scale,
                                 _ops._LATENT_TYPES[dtype], n, v, d, out.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream) == 0
    exact = ref.lookup(_np(table), ids.numpy(), scale)
    _close(out, exact, 2 * U * np.abs(exact), dtype, "out")  # scale and product
    assert torch.equal(latent.embedding_lookup(t, i, scale), out)
    grad = W.embedding_bwd(v_out.to(DEV), i, v, scale)
    exact, mass, count = ref.lookup_grad(_np(v_out), ids.numpy(), v, scale)
    _close(grad, exact, (count[:, None] + 3) * U * mass, dtype, "v_table")
