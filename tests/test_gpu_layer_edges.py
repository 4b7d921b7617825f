"""The block-sparse layer operators at the edges of their ranges."""
import numpy as np
import pytest

import lm_reference as ref
import varblockspmm_b200 as vb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("size", [(8, 8), (24, 40), (64, 32), (40, 64), (64, 64)])
def test_ortho_zero_and_not_finite_blocks_are_whole(cuda, size, steps):
    """A block of zeros gives zeros whatever eps is, one with a NaN or an infinity gives NaN everywhere, and
    their neighbours (two of them share a CTA) what they give alone."""
    torch = cuda
    h, w = size
    m = ref.matrix(6, 2, 1, 3, row_size=[h] * 6, col_size=[w] * 2)
    v = m.values.copy().reshape(6, h * w)
    v[0] = 0.0
    v[2, 3] = np.nan
    v[3, -1] = -np.inf
    v[5] = 0.0
    v[5, 1] = np.nan
    plan = vb.OrthoPlan(vb.Matrix(m))
    for eps in (0.0, 1e-44, 1e-38, 9e-38, 1e-7):
        out = torch.full((m.values.size,), 7.0, device="cuda")
        plan.execute(torch.from_numpy(v.reshape(-1)).cuda(), out, steps=steps, eps=eps)
        plan.check_status()
        out = out.cpu().numpy().reshape(6, h * w)
        assert (out[0] == 0).all(), eps
        for k in (2, 3, 5):
            assert np.isnan(out[k]).all(), (k, eps)
        alone = torch.empty(m.values.size, device="cuda")
        plan.execute(torch.from_numpy(m.values).cuda(), alone, steps=steps, eps=eps)
        alone = alone.cpu().numpy().reshape(6, h * w)
        for k in (1, 4):
            assert np.isfinite(out[k]).all() and np.array_equal(out[k], alone[k]), (k, eps)
