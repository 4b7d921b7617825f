"""How far the block-sparse layer operators are from 64 bits in the 2-norm, where bounds per element are too wide to
notice a lost cross term or a sum that is no longer promoted."""
import numpy as np
import pytest

import lm_reference as ref
import varblockspmm_b200 as vb

pytestmark = pytest.mark.gpu


def limit(n):
    """Relative 2-norm of the error of sums of n products of random sign. An accumulation chunk is at most 8 steps
    of 16 products, each of which cuts off at most 2^-23 of the running sum, on average half of that: 8 2^-24.
    Operands held to 2^-23 and the left-out term of 2^-22, at random: 2 2^-24 at most. Then n / 128 chunks are added
    with a rounding each, of 0.58 2^-24 of the sum so far on average (square root), a sum that grows with its
    square root: 0.41 sqrt(n / 128) 2^-24."""
    return (10 + 0.41 * np.sqrt(n / 128)) * 2.0 ** -24


def off(got, want):
    got = got.cpu().numpy().astype(np.float64).reshape(want.shape)
    return np.linalg.norm(got - want) / np.linalg.norm(want)


SHAPES = {"long_rows": (6, 400, 300), "long_columns": (400, 6, 4), "square": (60, 60, 30)}


@pytest.mark.parametrize("tokens", [1, 20, 100, 700])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_gated_products(cuda, name, tokens):
    torch = cuda
    rows, cols, degree = SHAPES[name]
    gate = ref.matrix(rows, cols, degree, 11)
    up = ref.matrix(rows, cols, max(1, degree // 2), 12, row_size=gate.row_size, col_size=gate.col_size)
    M, K = gate.scalar_rows(), gate.scalar_cols()
    rng = np.random.default_rng(tokens)
    X = rng.standard_normal((tokens, K)).astype(np.float32)
    dH = rng.standard_normal((tokens, M)).astype(np.float32)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up), vb.Activation.ReLU)
    H, G, U = (torch.full((tokens, M), float("nan"), device="cuda") for _ in range(3))
    plan.execute(torch.from_numpy(X).cuda(), H, G, U)
    n = ref.max_row_products(gate)
    A = [ref.dense(gate), ref.dense(up)]
    X64 = X.astype(np.float64)
    assert off(G, X64 @ A[0].T) <= limit(n)
    assert off(U, X64 @ A[1].T) <= limit(n)
    # gradients from given G and U, so that dG and dU are exact products of two numbers, rounded once or twice
    g, u = (np.abs(rng.standard_normal((tokens, M))).astype(np.float32) for _ in range(2))
    out = [torch.full((k,), float("nan"), device="cuda") for k in (tokens * K, len(gate.values), len(up.values))]
    plan.backward(*(torch.from_numpy(t).cuda() for t in (X, g, u, dH)), *out)
    plan.check_status()
    dG, dU = dH.astype(np.float64) * u, dH.astype(np.float64) * g
    n = ref.max_col_products(gate) + ref.max_col_products(up)
    assert off(out[0], dG @ A[0] + dU @ A[1]) <= limit(n)
    for got, m, d in ((out[1], gate, dG), (out[2], up, dU)):
        assert off(got, ref.sampled(m, d.T @ X64)) <= limit(tokens)


SIZES = (8, 16, 24, 32, 40, 48, 56, 64)


@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e25, 1e36])
def test_ortho_blocks_of_any_magnitude(cuda, scale):
    """The median and the worst block against float32 arithmetic on values of about one, where that neither over- nor
    underflows: the scale is divided out before the first step. Operands are held to 2^-23 where float32 arithmetic
    rounds to 2^-24, so twice its error in the median; per block four times, or 16 roundings."""
    torch = cuda
    m = ref.matrix(16, 16, 16, 41, row_size=SIZES * 2, col_size=SIZES * 2)
    v = m.values * np.float32(scale)
    base = v.astype(np.float64) / scale
    assert np.isfinite(v).all()
    out = torch.full((len(v),), float("nan"), device="cuda")
    plan = vb.OrthoPlan(vb.Matrix(m, structure_only=True))
    plan.execute(torch.from_numpy(v).cuda(), out, steps=5, eps=0.0)
    plan.check_status()
    got = out.cpu().numpy().astype(np.float64)
    coef = (3.4445, -4.7750, 2.0315)
    want = ref.newton_schulz(m, base, 5, 0.0, coef, np.float64)
    plain = ref.newton_schulz(m, base.astype(np.float32), 5, 0.0, coef, np.float32)
    err = np.array([[np.linalg.norm(x[p] - want[p]) / np.linalg.norm(want[p]) for x in (got, plain)]
                    for _, _, _, p, _, _ in ref.blocks(m)])
    ours, theirs = np.median(err, axis=0)
    assert ours <= 2 * theirs, (ours, theirs)
    assert np.all(err[:, 0] <= np.maximum(4 * err[:, 1], 16 * 2.0 ** -24)), err.max(axis=0)
