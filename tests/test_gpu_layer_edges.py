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


@pytest.mark.parametrize("tokens", [2, 40, 300])
@pytest.mark.parametrize("low", [100, 96, 90])
def test_weight_gradients_of_activations_near_the_largest_number(cuda, tokens, low):
    """A token of 2^127 with small gradients beside one of 2^low with large ones, whose products are larger: the
    first one's count in full."""
    torch = cuda
    m = ref.matrix(5, 6, 3, 4)
    M, K = m.scalar_rows(), m.scalar_cols()
    rng = np.random.default_rng(tokens)
    X = np.zeros((tokens, K), dtype=np.float32)
    dH = np.zeros((tokens, M), dtype=np.float32)
    X[0], dH[0] = 2.0 ** 127 * rng.uniform(0.5, 1, K), 2.0 ** -30 * rng.uniform(0.5, 1, M)
    X[1], dH[1] = 2.0 ** low * rng.uniform(0.5, 1, K), 2.0 ** (115 - low) * rng.uniform(0.5, 1, M)
    ones = torch.ones(tokens, M, device="cuda")  # relu: dG = dU = dH
    plan = vb.GatedPlan(vb.Matrix(m), vb.Matrix(m), vb.Activation.ReLU)
    out = [torch.full((len(m.values),), float("nan"), device="cuda") for _ in range(2)]
    plan.backward(torch.from_numpy(X).cuda(), ones, ones, torch.from_numpy(dH).cuda(), None, *out)
    plan.check_status()
    want = dH.astype(np.float64).T @ X.astype(np.float64)
    # all terms are positive, so the bound of a sum of two products is relative
    tol = ref.sampled(m, ref.product_tolerance(2, want))
    want = ref.sampled(m, want)
    for got in out:
        assert np.all(np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol)
