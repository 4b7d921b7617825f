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


@pytest.mark.parametrize("kind", [vb.Activation.SiLU, vb.Activation.Sigmoid])
def test_activations_and_derivatives_in_their_tails(cuda, kind):
    """act(G) U and act'(G) over the whole range of G, against 64 bits. Sigmoids of x and -x are each off by
    (6 + 1.2 |x|) 2^-23 of themselves (see act_both), a product of them with one another or with x by the sum and
    a rounding; dB passes through a product with the unit matrix, which holds values to 2^-23 twice, and, as a
    token's gradients of gate and up share one power of two, to no better than 2^-50 of the largest of both:
    that one is in [2^14, 2^15) as the high half, half a step of the low half's smallest numbers is
    2^-25 2^-11 = 2^-36."""
    torch = cuda
    unit = vb.HostMatrix(1, 1, [0, 1], [0], [8], [8], [0, 8], [0, 8], [0, 64], np.eye(8, dtype=np.float32).reshape(-1))
    none = vb.HostMatrix(1, 1, [0, 0], [], [8], [8], [0, 8], [0, 8], [0], [])
    x = np.concatenate([np.linspace(-80, 80, 2001), np.linspace(-3, 3, 600), [0.0, -1e-30, 1e-30]]).astype(np.float32)
    T = len(x)
    G = torch.from_numpy(np.repeat(x[:, None], 8, axis=1)).cuda()  # a value to a token: each has its own scale
    ones, dB = torch.ones(T, 8, device="cuda"), torch.full((T, 8), float("nan"), device="cuda")
    # backward, up without blocks: dB = act'(G)
    plan = vb.GatedPlan(vb.Matrix(unit), vb.Matrix(none), kind)
    plan.backward(ones, G, ones, ones, dB)
    plan.check_status()
    x64 = x.astype(np.float64)
    s, c = np.exp(-np.logaddexp(0, -x64)), np.exp(-np.logaddexp(0, x64))
    rel = (6 + 1.2 * np.abs(x64)) * 2.0 ** -23
    if kind == vb.Activation.Sigmoid:
        want, size = s * c, s * c
    else:
        want, size = s * (1 + x64 * c), s * (1 + np.abs(x64) * c)
    a64 = s if kind == vb.Activation.Sigmoid else np.abs(x64) * s  # dU
    tol = (2 * rel + 6 * 2.0 ** -23) * size + 2.0 ** -50 * np.maximum(a64, np.abs(want)) + 1e-37
    got = dB.cpu().numpy().astype(np.float64)
    over = np.abs(got - want[:, None]) / tol[:, None]
    assert over.max() <= 1, (x[over.max(axis=1).argmax()], over.max())
    # forward, gate and up the unit matrix: H = act(G) U with the G and U that it returns
    plan = vb.GatedPlan(vb.Matrix(unit), vb.Matrix(unit), kind)
    H, Gf, Uf = (torch.full((T, 8), float("nan"), device="cuda") for _ in range(3))
    plan.execute(G, H, Gf, Uf)
    plan.check_status()
    g, u = Gf.cpu().numpy().astype(np.float64), Uf.cpu().numpy().astype(np.float64)
    s = np.exp(-np.logaddexp(0, -g))
    want = (s if kind == vb.Activation.Sigmoid else g * s) * u
    tol = ((6 + 1.2 * np.abs(g)) * 2.0 ** -23 + 2 * 2.0 ** -24) * np.abs(want) + 1e-37
    assert np.all(np.abs(H.cpu().numpy() - want) <= tol)


def by_clusters(tokens, K):
    """Which panels Int8Plan quantises by clusters of CTAs that hold two tokens each; others take two kernels."""
    return K <= 38400 and (tokens <= max(128, K // 24) or K > 16384)


@pytest.mark.parametrize("tokens,K,held", [
    (1, 968, True), (128, 960, True), (129, 960, False),  # one piece of the lanes' registers, just full and over
    (128, 2048, True), (129, 2048, False), (129, 3096, True), (341, 8184, True), (342, 8184, False),
    (682, 16384, True), (683, 16384, False), (683, 16392, True),  # longer ones: any number of tokens
    (3, 20008, True), (33, 30712, True), (131, 30728, True),
    (2, 38400, True), (259, 38400, True), (2, 38408, False), (259, 38408, False)])
@pytest.mark.parametrize("offset", [0, 1])
def test_int8_every_way_of_quantising(cuda, tokens, K, held, offset):
    """Panels on both sides of every border of the choice, one token with a NaN, one with an infinity, one of
    zeros, at aligned and unaligned places."""
    torch = cuda
    assert by_clusters(tokens, K) == held
    col_size = [64] * (K // 64) + ([K % 64] if K % 64 else [])
    m = ref.matrix(5, len(col_size), min(25, len(col_size)), 71, row_size=[8, 24, 64, 8, 16], col_size=col_size)
    m.block_col[m.row_ptr[1] - 1] = len(col_size) - 1  # the last columns are read
    m = vb.HostMatrix(m.block_rows, m.block_cols, m.row_ptr, m.block_col, m.row_size, m.col_size, m.row_scalar_off,
                      m.col_scalar_off, np.concatenate([[0], np.cumsum(np.repeat(m.row_size, np.diff(m.row_ptr)) *
                                                                       m.col_size[m.block_col])]), [])
    rng = np.random.default_rng(tokens)
    q = rng.integers(-128, 128, int(m.value_off[-1])).astype(np.int8)
    rs = (rng.random(m.scalar_rows()) + 0.1).astype(np.float32)
    X = (rng.standard_normal((tokens, K)) * np.exp(rng.standard_normal((tokens, 1)))).astype(np.float32)
    bad = []
    if tokens > 2:
        X[tokens - 1, K - 1], X[1, 0], X[0] = np.nan, -np.inf, 0.0
        bad = [1, tokens - 1]
    with np.errstate(all="ignore"):
        ts = np.abs(X).max(axis=1) * (np.float32(1) / np.float32(127))
        Q = np.clip(np.where(ts[:, None] > 0, np.rint(X.astype(np.float64) / ts[:, None].astype(np.float64)), 0),
                    -127, 127)
        want = (np.where(np.isfinite(Q), Q, 0) @ ref.dense(m, q).T) * (ts[:, None].astype(np.float64) * rs)
    buf = torch.zeros(tokens * K + 8, device="cuda")
    x = buf[offset:offset + tokens * K]
    x.copy_(torch.from_numpy(X).cuda().reshape(-1))
    plan = vb.Int8Plan(vb.Matrix(m, structure_only=True), torch.from_numpy(q).cuda(), torch.from_numpy(rs).cuda())
    C = torch.full((tokens, m.scalar_rows()), 7.0, device="cuda")
    plan.execute_panel(x, C)
    plan.check_status()
    got = C.cpu().numpy().astype(np.float64)
    good = np.setdiff1d(np.arange(tokens), bad)
    # the sum, the product of the scales and the result round once each
    assert np.all(np.abs(got[good] - want[good]) <= 4 * ref.U * np.abs(want[good]))
    assert np.isnan(got[bad]).all()


def long_case(torch, tokens, rows, cols, degree, seed):
    m = ref.matrix(rows, cols, degree, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    X = torch.randn(tokens, m.scalar_cols(), generator=g, device="cuda")
    return m, X, g


@pytest.mark.parametrize("tokens,rows,cols,degree", [
    (4096, 12, 14, 6), (4097, 3, 4, 2), (65535, 2, 3, 2), (70001, 3, 4, 2), (1 << 22, 1, 1, 1)])
def test_many_tokens(cuda, tokens, rows, cols, degree):
    """Up to the largest number of tokens: all three directions and both ways of giving 8-bit activations."""
    torch = cuda
    m, X, g = long_case(torch, tokens, rows, cols, degree, 5 if tokens < 1 << 22 else 6)
    M, K = m.scalar_rows(), m.scalar_cols()
    A = torch.from_numpy(ref.dense(m)).cuda()
    absA = A.abs()
    bare, w = vb.Matrix(m, structure_only=True), torch.from_numpy(m.values).cuda()
    plan = vb.GatedPlan(bare, bare, vb.Activation.ReLU)
    plan.set_values(w, -w)
    H, G, U = (torch.full((tokens, M), float("nan"), device="cuda") for _ in range(3))
    plan.execute(X, H, G, U)
    plan.check_status()
    step = 1 << 16  # compared in pieces, in 64 bits

    def held(got, want, tol):
        assert bool(((got.double() - want).abs() <= tol + 1e-37).all())

    n = ref.max_row_products(m)
    for t in range(0, tokens, step):
        x = X[t:t + step].double()
        want = x @ A.T
        tol = ref.product_tolerance(n, x.abs() @ absA.T)
        held(G[t:t + step], want, tol)
        held(U[t:t + step], -want, tol)
        held(H[t:t + step], G[t:t + step].double().clamp(min=0) * U[t:t + step].double(), 2e-7 * want.square() + 1e-30)
    dH = 1e-3 * torch.randn(tokens, M, generator=g, device="cuda")
    dX = torch.full_like(X, float("nan"))
    dw = [torch.full((len(m.values),), float("nan"), device="cuda") for _ in range(2)]
    plan.backward(X, G, U, dH, dX, *dw)
    plan.check_status()
    sums, mags = [torch.zeros(M, K, dtype=torch.float64, device="cuda") for _ in range(2)], \
        [torch.zeros(M, K, dtype=torch.float64, device="cuda") for _ in range(2)]
    n = 2 * ref.max_col_products(m)
    for t in range(0, tokens, step):
        x, gg, u, dh = (v[t:t + step].double() for v in (X, G, U, dH))
        d = [dh * u * (gg > 0), dh * gg.clamp(min=0)]
        # dG and dU are rounded twice, then their product's bound
        size = (d[0].abs() + d[1].abs()) @ absA
        held(dX[t:t + step], (d[0] - d[1]) @ A, ref.product_tolerance(n, size) + 2 * ref.U * size)
        for i in range(2):
            sums[i] += d[i].T @ x
            mags[i] += d[i].abs().T @ x.abs()
    for i in range(2):
        want, mag = ref.sampled(m, sums[i].cpu().numpy()), ref.sampled(m, mags[i].cpu().numpy())
        got = dw[i].cpu().numpy().astype(np.float64)
        # tokens are added 64 at a time
        tol = ref.product_tolerance(min(tokens, 64) + tokens / 64, mag) + 2 * ref.U * mag
        assert np.all(np.abs(got - want) <= tol), i
    # 8 bits
    q = torch.from_numpy(np.random.default_rng(1).integers(-127, 128, len(m.values)).astype(np.int8)).cuda()
    rs = torch.rand(M, device="cuda") + 0.1
    i8 = vb.Int8Plan(bare, q, rs)
    C, C2, Q, ts = (torch.zeros(tokens, M, device="cuda"), torch.zeros(tokens, M, device="cuda"),
                    torch.zeros(tokens, K, dtype=torch.int8, device="cuda"), torch.zeros(tokens, device="cuda"))
    i8.execute_panel(X, C)
    vb.quantize_panel(X, Q, ts, K)
    i8.execute(Q, ts, C2)
    i8.check_status()
    assert torch.equal(C, C2)
    Aq = torch.from_numpy(ref.dense(m, q.cpu().numpy())).cuda()
    for t in range(0, tokens, step):
        x = X[t:t + step]
        want_ts = x.abs().amax(1) * torch.tensor(np.float32(1) / np.float32(127), device="cuda")
        assert torch.equal(ts[t:t + step], want_ts)
        want_q = torch.round(x.double() / want_ts.double()[:, None])
        assert torch.equal(Q[t:t + step].double(), want_q)
        want = (want_q @ Aq.T) * (want_ts.double()[:, None] * rs.double())
        held(C[t:t + step], want, 4 * ref.U * want.abs())


@pytest.mark.parametrize("tokens", [700, 4099])
def test_int8_many_long_tokens(cuda, tokens):
    """Clusters of held tokens, more than the GPU holds at once."""
    torch = cuda
    m = ref.matrix(4, 400, 30, 9, row_size=[8, 16, 64, 24], col_size=[48] * 400)
    K = m.scalar_cols()
    assert by_clusters(tokens, K)
    X = torch.randn(tokens, K, device="cuda")
    q = torch.from_numpy(np.random.default_rng(2).integers(-127, 128, len(m.values)).astype(np.int8)).cuda()
    rs = torch.rand(m.scalar_rows(), device="cuda") + 0.1
    plan = vb.Int8Plan(vb.Matrix(m, structure_only=True), q, rs)
    C = torch.zeros(tokens, m.scalar_rows(), device="cuda")
    plan.execute_panel(X, C)
    plan.check_status()
    ts = X.abs().amax(1) * torch.tensor(np.float32(1) / np.float32(127), device="cuda")
    want = torch.round(X.double() / ts.double()[:, None]) @ torch.from_numpy(ref.dense(m, q.cpu().numpy())).cuda().T
    want = want * (ts.double()[:, None] * rs.double())
    assert bool(((C.double() - want).abs() <= 4 * ref.U * want.abs()).all())
