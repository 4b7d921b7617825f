"""The operators for block-sparse layers on the GPU, against plain 64-bit implementations: the gated
feed-forward block and its gradients, the 8-bit product, the orthogonalised block update."""
import numpy as np
import pytest

import lm_reference as ref
import varblockspmm_b200 as vb

pytestmark = pytest.mark.gpu

SIZES = (8, 16, 24, 32, 40, 48, 56, 64)
# name: gate, up matrix
PAIRS = {
    "mixed": lambda: (ref.matrix(9, 11, 4, 1, empty=(2,), skip_cols=(5,)),
                      ref.matrix(9, 11, 3, 2, empty=(0, 2), skip_cols=(5,))),
    "one_block": lambda: (ref.matrix(1, 1, 1, 3, sizes=(8,)), ref.matrix(1, 1, 1, 4, sizes=(8,))),
    "largest_blocks": lambda: (ref.matrix(3, 5, 5, 5, sizes=(64,)), ref.matrix(3, 5, 2, 6, sizes=(64,))),
    "smallest_blocks": lambda: (ref.matrix(40, 70, 7, 7, sizes=(8,)), ref.matrix(40, 70, 60, 8, sizes=(8,))),
    "repeated": lambda: (ref.matrix(4, 3, 7, 9, repeat=True), ref.matrix(4, 3, 5, 10, repeat=True)),
    "one_long_row": lambda: (ref.matrix(1, 300, 290, 11), ref.matrix(1, 300, 1, 12)),
    "no_blocks": lambda: (ref.matrix(3, 4, 0, 13), ref.matrix(3, 4, 0, 14)),
    "tall": lambda: (ref.matrix(200, 2, 1, 15), ref.matrix(200, 2, 2, 16)),
}


def pair(name):
    gate, up = PAIRS[name]()
    # one partition for both
    up = ref.matrix(up.block_rows, up.block_cols, int(np.diff(up.row_ptr).max()), 77,
                    empty=tuple(np.flatnonzero(np.diff(up.row_ptr) == 0)),
                    skip_cols=tuple(np.setdiff1d(np.arange(up.block_cols), up.block_col))
                    if up.nnzb > up.block_cols else (), repeat=name == "repeated",
                    row_size=gate.row_size, col_size=gate.col_size, scale=0.5)
    return gate, up


def activations(tokens, features, seed):
    """Token sizes over orders of magnitude, a few large features, a token of zeros."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((tokens, features)) * np.exp(rng.standard_normal((tokens, 1)))
    x[:, ::37] *= 30.0
    if tokens > 3:
        x[2] = 0.0
    return (0.1 * x).astype(np.float32)


class Gated:
    """The forward quantities in float64 with their error bounds."""

    def __init__(self, gate, up, kind, X, kept=None):
        self.A = [ref.dense(gate), ref.dense(up)]
        X64 = X.astype(np.float64)
        n = [ref.max_row_products(gate), ref.max_row_products(up)]
        self.Y = [X64 @ a.T for a in self.A]
        self.tol = [ref.product_tolerance(n[i], np.abs(X64) @ ref.dense(m, np.abs(m.values)).T)
                    for i, m in enumerate((gate, up))]
        self.G, self.U = self.Y
        a, _ = ref.act(kind, self.G)
        self.H = a * self.U
        # |act'| <= 1.13 for every kind; its evaluation is off by a few roundings of |G|
        ta = 1.13 * self.tol[0] + 8 * ref.U * (np.abs(self.G) + (kind == vb.Activation.Sigmoid))
        self.H_tol = ta * (np.abs(self.U) + self.tol[1]) + np.abs(a) * self.tol[1] + 2 * ref.U * np.abs(self.H)


def close(got, want, tol, what):
    got = got.detach().cpu().numpy().astype(np.float64).reshape(want.shape)
    assert np.all(np.isfinite(got)), f"{what}: not finite"
    over = np.abs(got - want) > tol + 1e-37
    assert not over.any(), (what, int(over.sum()), float(np.max(np.abs(got - want) / (tol + 1e-37))))


def run_forward(torch, plan, X, M, keep=True):
    dX = torch.from_numpy(X).cuda()
    out = [torch.full((len(X), M), float("nan"), device="cuda") for _ in range(3)]
    plan.execute(dX, out[0], *(out[1:] if keep else ()), stream=torch.cuda.current_stream())
    plan.check_status()
    return dX, out


def check_backward(torch, plan, gate, up, kind, X, seed=5, padded=()):
    M, K, T = gate.scalar_rows(), gate.scalar_cols(), len(X)
    dX_in, (H, G, U) = run_forward(torch, plan, X, M)
    rng = np.random.default_rng(seed)
    dH = (1e-3 * rng.standard_normal((T, M))).astype(np.float32)
    dH[list(padded)] = 0.0
    dB = torch.full((T, K), float("nan"), device="cuda")
    dw = [torch.full((len(m.values),), float("nan"), device="cuda") for m in (gate, up)]
    plan.backward(dX_in, G, U, torch.from_numpy(dH).cuda(), dB, *dw, stream=torch.cuda.current_stream())
    plan.check_status()
    # the formula on the kept pre-activations
    G64, U64, X64 = (t.cpu().numpy().astype(np.float64) for t in (G, U, dX_in))
    a, da = ref.act(kind, G64)
    dY = [dH * U64 * da, dH * a]
    dY_tol = [np.abs(dH) * np.abs(U64) * 16 * ref.U * (1 + np.abs(G64)),
              np.abs(dH) * 8 * ref.U * (1 + np.abs(G64))]
    want, tol = np.zeros((T, K)), np.zeros((T, K))
    n = ref.max_col_products(gate) + ref.max_col_products(up)
    for m, d, t in zip((gate, up), dY, dY_tol):
        A, absA = ref.dense(m), ref.dense(m, np.abs(m.values))
        want += d @ A
        tol += t @ absA + ref.product_tolerance(n, (np.abs(d) + t) @ absA)
    close(dB, want, tol, "dB")
    for m, d, t, got, name in zip((gate, up), dY, dY_tol, dw, ("dgate", "dup")):
        mag = (np.abs(d) + t).T @ np.abs(X64)
        close(got, ref.sampled(m, d.T @ X64),
              ref.sampled(m, t.T @ np.abs(X64) + ref.product_tolerance(T, mag)), name)


@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 16, 33, 64, 65, 128, 129, 300, 1000])
@pytest.mark.parametrize("name", ["mixed", "one_long_row"])
def test_gated_lengths(cuda, name, tokens):
    gate, up = pair(name)
    X = activations(tokens, gate.scalar_cols(), tokens)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up), vb.Activation.SiLU)
    want = Gated(gate, up, vb.Activation.SiLU, X)
    _, (H, G, U) = run_forward(cuda, plan, X, gate.scalar_rows())
    close(G, want.G, want.tol[0], "G")
    close(U, want.U, want.tol[1], "U")
    close(H, want.H, want.H_tol, "H")
    _, (H2, _, _) = run_forward(cuda, plan, X, gate.scalar_rows(), keep=False)
    assert np.array_equal(H2.cpu().numpy(), H.cpu().numpy())
    check_backward(cuda, plan, gate, up, vb.Activation.SiLU, X)


@pytest.mark.parametrize("kind", list(vb.Activation))
@pytest.mark.parametrize("name", sorted(PAIRS))
def test_gated_structures(cuda, name, kind):
    gate, up = pair(name)
    X = activations(19, gate.scalar_cols(), 3)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up), kind)
    want = Gated(gate, up, kind, X)
    _, (H, G, U) = run_forward(cuda, plan, X, gate.scalar_rows())
    close(G, want.G, want.tol[0], "G")
    close(U, want.U, want.tol[1], "U")
    close(H, want.H, want.H_tol, "H")
    check_backward(cuda, plan, gate, up, kind, X)


@pytest.mark.parametrize("tokens", [1, 40, 130])
def test_many_work_items_per_sm(cuda, tokens):
    """Matrices with far more block rows and columns than the GPU has SMs, short rows and empty ones."""
    torch = cuda
    rng = np.random.default_rng(6)
    rows, cols = 2500, 60
    rs = rng.choice((8, 16, 24, 64), rows, p=(0.5, 0.3, 0.1, 0.1))
    cs = rng.choice((8, 16, 40), cols)
    empty = tuple(np.flatnonzero(rng.random(rows) < 0.2))
    gate = ref.matrix(rows, cols, 5, 61, row_size=rs, col_size=cs, empty=empty)
    up = ref.matrix(rows, cols, 30, 62, row_size=rs, col_size=cs, empty=empty[::2])
    X = activations(tokens, gate.scalar_cols(), tokens)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up))
    want = Gated(gate, up, vb.Activation.SiLU, X)
    for _ in range(3):
        _, (H, G, U) = run_forward(torch, plan, X, gate.scalar_rows())
        close(G, want.G, want.tol[0], "G")
        close(U, want.U, want.tol[1], "U")
        close(H, want.H, want.H_tol, "H")
    check_backward(torch, plan, gate, up, vb.Activation.SiLU, X)
    tall = ref.matrix(cols, rows, 300, 63, row_size=cs, col_size=rs)  # many block columns
    wide = ref.matrix(cols, rows, 200, 64, row_size=cs, col_size=rs)
    X2 = activations(tokens, tall.scalar_cols(), 3)
    check_backward(torch, vb.GatedPlan(vb.Matrix(tall), vb.Matrix(wide)), tall, wide,
                   vb.Activation.SiLU, X2)
    q, sc = int8_weights(up, 7)
    C = torch.empty(tokens, up.scalar_rows(), device="cuda")
    i8 = vb.Int8Plan(vb.Matrix(up), torch.from_numpy(q).cuda(), torch.from_numpy(sc).cuda())
    Q, ts = quantized(X)
    want8 = (Q @ ref.dense(up, q).T) * ts[:, None].astype(np.float64) * sc
    for _ in range(3):
        C.fill_(float("nan"))
        i8.execute_panel(torch.from_numpy(X).cuda(), C)
        i8.check_status()
        close(C, want8, 4 * ref.U * np.abs(want8), "C")


@pytest.mark.parametrize("size", SIZES)
def test_gated_every_block_height_and_width(cuda, size):
    for rows, cols in (((size,), SIZES), (SIZES, (size,))):
        gate = ref.matrix(8, 16, 5, size, sizes=SIZES, row_size=np.resize(rows, 8),
                          col_size=np.resize(cols, 16))
        up = ref.matrix(8, 16, 6, size + 1, row_size=gate.row_size, col_size=gate.col_size)
        X = activations(21, gate.scalar_cols(), size)
        plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up), vb.Activation.GELU)
        want = Gated(gate, up, vb.Activation.GELU, X)
        _, (H, G, U) = run_forward(cuda, plan, X, gate.scalar_rows())
        close(G, want.G, want.tol[0], "G")
        close(H, want.H, want.H_tol, "H")
        check_backward(cuda, plan, gate, up, vb.Activation.GELU, X)


def test_gated_gradient_against_differences(cuda):
    """The gradients along random directions against central differences of the 64-bit forward."""
    torch = cuda
    gate, up = pair("mixed")
    kind, T, M = vb.Activation.SiLU, 6, gate.scalar_rows()
    X = activations(T, gate.scalar_cols(), 8)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up), kind)
    dX, (H, G, U) = run_forward(torch, plan, X, M)
    rng = np.random.default_rng(2)
    dH = rng.standard_normal((T, M)).astype(np.float32)
    got = [torch.empty_like(dX), torch.empty(len(gate.values), device="cuda"),
           torch.empty(len(up.values), device="cuda")]
    plan.backward(dX, G, U, torch.from_numpy(dH).cuda(), *got)
    torch.cuda.synchronize()

    def loss(x, vg, vu):
        a, _ = ref.act(kind, x @ ref.dense(gate, vg).T)
        return float((a * (x @ ref.dense(up, vu).T) * dH).sum())

    base = [X.astype(np.float64), gate.values.astype(np.float64), up.values.astype(np.float64)]
    for i in range(3):
        d = rng.standard_normal(base[i].shape) * np.abs(base[i]).mean()
        h = 1e-5  # the differences are off by about h^2 and 2^-52 / h, both below 1e-9
        at = [[b + s * h * d if j == i else b for j, b in enumerate(base)] for s in (1, -1)]
        want = (loss(*at[0]) - loss(*at[1])) / (2 * h)
        g = got[i].cpu().numpy().astype(np.float64).reshape(d.shape)
        # fp32 gradients: sums of at most 1200 terms, each to 1200 * 2^-24 of its magnitude
        assert abs((g * d).sum() - want) <= 1200 * ref.U * np.abs(g * d).sum() + 1e-6 * abs(want), i


def test_gated_set_values_parts_and_zero_tokens(cuda):
    torch = cuda
    gate, up = pair("mixed")
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up))
    other = [m.copy() for m in (gate, up)]
    for m in other:
        m.values = (m.values[::-1] * 3).copy()
    plan.set_values(*(torch.from_numpy(m.values).cuda() for m in other))
    X = activations(12, gate.scalar_cols(), 4)
    want = Gated(*other, vb.Activation.SiLU, X)
    dX, (H, G, U) = run_forward(torch, plan, X, gate.scalar_rows())
    close(H, want.H, want.H_tol, "H")
    # either part of the backward alone gives what both give
    dH = torch.full_like(H, 1e-3)
    full = [torch.empty_like(dX), torch.empty(len(gate.values), device="cuda"),
            torch.empty(len(up.values), device="cuda")]
    plan.backward(dX, G, U, dH, *full)
    part = [torch.empty_like(t) for t in full]
    plan.backward(dX, G, U, dH, part[0])
    plan.backward(dX, G, U, dH, None, part[1], part[2])
    torch.cuda.synchronize()
    for a, b in zip(full, part):
        assert torch.equal(a, b)
    # no tokens: weight gradients are zero, nothing else is touched
    none = torch.empty(0, gate.scalar_cols(), device="cuda")
    empty = torch.empty(0, gate.scalar_rows(), device="cuda")
    plan.execute(none, empty)
    plan.backward(none, empty, empty, empty, none, part[1], part[2])
    torch.cuda.synchronize()
    assert not part[1].any() and not part[2].any()
    plan.backward(none, empty, empty, empty, none)


@pytest.mark.parametrize("offset", [0, 1, 2])
def test_gated_unaligned_panels_and_rows_behind(cuda, offset):
    """Panels at any float offset; what lies behind the last token stays as it was."""
    torch = cuda
    gate, up = pair("mixed")
    M, K, T = gate.scalar_rows(), gate.scalar_cols(), 9
    X = activations(T, K, 6)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up))
    want = Gated(gate, up, vb.Activation.SiLU, X)
    buf = torch.zeros(T * K + 8, device="cuda")
    buf[offset:offset + T * K] = torch.from_numpy(X).cuda().reshape(-1)
    outs = [torch.full((T * M + 64,), 7.0, device="cuda") for _ in range(3)]
    v = [t[offset:offset + T * M] for t in outs]
    plan.execute(buf[offset:offset + T * K], *v)
    dout = [torch.full((n + 64,), 7.0, device="cuda") for n in (T * K, len(gate.values), len(up.values))]
    d = [t[offset:offset + n] for t, n in zip(dout, (T * K, len(gate.values), len(up.values)))]
    plan.backward(buf[offset:offset + T * K], v[1], v[2], v[0].clone(), *d)
    plan.check_status()
    close(v[0], want.H, want.H_tol, "H")
    for t, inner in list(zip(outs, v)) + list(zip(dout, d)):
        assert (t[:offset] == 7).all() and (t[offset + inner.numel():] == 7).all()
        assert torch.isfinite(inner).all()


def test_gated_scales(cuda):
    """Weights, activations and gradients far from one: nothing over- or underflows on the way."""
    torch = cuda
    gate, up = pair("mixed")
    X = activations(10, gate.scalar_cols(), 9)
    for sw, sx in ((1e-12, 1e8), (1e10, 1e-14), (1e-18, 1e18)):
        g, u = gate.copy(), up.copy()
        g.values, u.values = (g.values * np.float32(sw)), (u.values * np.float32(sw))
        x = (X * np.float32(sx)).astype(np.float32)
        plan = vb.GatedPlan(vb.Matrix(g), vb.Matrix(u), vb.Activation.ReLU)
        want = Gated(g, u, vb.Activation.ReLU, x)
        _, (H, G, U) = run_forward(torch, plan, x, g.scalar_rows())
        close(G, want.G, want.tol[0], "G")
        close(H, want.H, want.H_tol, "H")
        check_backward(torch, plan, g, u, vb.Activation.ReLU, x)


@pytest.mark.parametrize("name,tokens", [("mixed", 9), ("mixed", 70), ("mixed", 300), ("one_long_row", 3),
                                         ("one_long_row", 200), ("largest_blocks", 129)])
def test_gated_tokens_of_unlike_size(cuda, name, tokens):
    """A token 2^50 times the others (a padded place, whose dH is zero) and one 2^60 below them: every
    token has its own accuracy, forward and backward, and the padded one takes no accuracy from the
    weight gradients."""
    torch = cuda
    gate, up = pair(name)
    kind = vb.Activation.SiLU
    X = activations(tokens, gate.scalar_cols(), 31)
    X[1] *= np.float32(2.0 ** 50)
    X[tokens - 1] *= np.float32(2.0 ** -60)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up), kind)
    want = Gated(gate, up, kind, X)
    _, (H, G, U) = run_forward(torch, plan, X, gate.scalar_rows())
    close(G, want.G, want.tol[0], "G")
    close(U, want.U, want.tol[1], "U")
    check_backward(torch, plan, gate, up, kind, X, padded=(1,))


def test_gated_not_finite_stays_in_its_token(cuda):
    """A NaN or an infinity in one token leaves the other tokens as they were, and reaches only the
    rows that read its feature."""
    torch = cuda
    gate, up = pair("mixed")
    K, M = gate.scalar_cols(), gate.scalar_rows()
    X = activations(20, K, 10)
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up))
    want = Gated(gate, up, vb.Activation.SiLU, X)
    reads = [np.abs(ref.dense(m)) for m in (gate, up)]
    for bad in (np.nan, np.inf, -np.inf):
        x = X.copy()
        x[4, 3] = bad
        _, (H, G, U) = run_forward(torch, plan, x, M)
        for got, w, tol, a in ((G, want.G, want.tol[0], reads[0]), (U, want.U, want.tol[1], reads[1])):
            got = got.cpu().numpy()
            others = np.arange(20) != 4
            assert np.all(np.abs(got[others] - w[others]) <= tol[others] + 1e-37)
            touched = a[:, 3] > 0
            assert not np.isfinite(got[4][touched]).any()
            same = ~touched & (np.abs(a).sum(1) == 0)
            assert np.all(got[4][same] == 0)


def test_gated_streams_and_graphs(cuda):
    """Two calls at once on two streams, and two captured graphs replayed together."""
    torch = cuda
    gate, up = pair("mixed")
    M, K = gate.scalar_rows(), gate.scalar_cols()
    plan = vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up))
    Xs = [activations(t, K, t) for t in (40, 17)]
    dXs = [torch.from_numpy(x).cuda() for x in Xs]
    want = [Gated(gate, up, vb.Activation.SiLU, x) for x in Xs]
    outs = [[torch.zeros(len(x), M, device="cuda") for _ in range(3)] for x in Xs]
    grads = [[torch.zeros(len(x), K, device="cuda"), torch.zeros(len(gate.values), device="cuda"),
              torch.zeros(len(up.values), device="cuda")] for x in Xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in Xs]

    def step(i, s):
        plan.execute(dXs[i], *outs[i], stream=s)
        plan.backward(dXs[i], outs[i][1], outs[i][2], outs[i][0], *grads[i], stream=s)

    for _ in range(5):
        for i, s in enumerate(streams):
            step(i, s)
    torch.cuda.synchronize()
    eager = [[t.clone() for t in outs[i] + grads[i]] for i in range(2)]
    for i in range(2):
        close(outs[i][0], want[i].H, want[i].H_tol, "H")
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(i, torch.cuda.current_stream())
        graphs.append(g)
    for i in range(2):
        for t in outs[i] + grads[i]:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    plan.check_status()
    for i in range(2):
        for a, b in zip(eager[i], outs[i] + grads[i]):
            assert torch.equal(a, b)


# ---- 8-bit product -------------------------------------------------------------------------------

def quantized(x, axis=1):
    """(integers, float32 scales) of the definition, the quotient in 64 bits."""
    with np.errstate(all="ignore"):
        s = np.abs(x).max(axis=axis, initial=0).astype(np.float32) * (np.float32(1) / np.float32(127))
        q = np.rint(x.astype(np.float64) / np.expand_dims(s.astype(np.float64), axis))
    return np.clip(np.where(np.expand_dims(s, axis) > 0, q, 0), -127, 127), s


def int8_weights(m, seed):
    rng = np.random.default_rng(seed)
    q = rng.integers(-127, 128, len(m.values)).astype(np.int8)
    q[:: 5] = np.where(q[:: 5] > 0, 127, -128)  # the type's own extremes too
    return q, (rng.random(m.scalar_rows()) + 0.1).astype(np.float32)


@pytest.mark.parametrize("tokens", [1, 5, 8, 17, 64, 65, 128, 200])
@pytest.mark.parametrize("name", sorted(PAIRS))
def test_int8_product(cuda, name, tokens):
    torch = cuda
    m, _ = PAIRS[name]()
    q, rs = int8_weights(m, 1)
    X = activations(tokens, m.scalar_cols(), tokens + 1)
    plan = vb.Int8Plan(vb.Matrix(m), torch.from_numpy(q).cuda(), torch.from_numpy(rs).cuda())
    Q, ts = quantized(X)
    want = (Q @ ref.dense(m, q).T) * ts[:, None].astype(np.float64) * rs
    tol = 4 * ref.U * np.abs(want)  # the sum, the product of the scales and the result round once
    C = torch.full((tokens, m.scalar_rows()), float("nan"), device="cuda")
    plan.execute_panel(torch.from_numpy(X).cuda(), C)
    plan.check_status()
    close(C, want, tol, "C")
    dQ, dts = torch.from_numpy(Q.astype(np.int8)).cuda(), torch.from_numpy(ts).cuda()
    C2 = torch.full_like(C, float("nan"))
    plan.execute(dQ, dts, C2)
    plan.check_status()
    assert torch.equal(C, C2)


@pytest.mark.parametrize("tokens", [9, 70, 140])
@pytest.mark.parametrize("offset", [1, 2])
def test_int8_unaligned_panels_and_rows_behind(cuda, offset, tokens):
    torch = cuda
    m = ref.matrix(5, 220, 30, 41)  # long enough rows for every way of quantising a panel
    M, K = m.scalar_rows(), m.scalar_cols()
    q, rs = int8_weights(m, 3)
    plan = vb.Int8Plan(vb.Matrix(m), torch.from_numpy(q).cuda(), torch.from_numpy(rs).cuda())
    X = activations(tokens, K, 4)
    Q, ts = quantized(X)
    want = (Q @ ref.dense(m, q).T) * ts[:, None].astype(np.float64) * rs
    xb = torch.zeros(tokens * K + 8, device="cuda")
    x = xb[offset:offset + tokens * K]
    x.copy_(torch.from_numpy(X).cuda().reshape(-1))
    qb = torch.zeros(tokens * K + 8, dtype=torch.int8, device="cuda")
    qx = qb[offset:offset + tokens * K]
    qx.copy_(torch.from_numpy(Q.astype(np.int8)).cuda().reshape(-1))
    for call in (lambda c: plan.execute_panel(x, c),
                 lambda c: plan.execute(qx, torch.from_numpy(ts).cuda(), c)):
        out = torch.full((tokens * M + 64,), 7.0, device="cuda")
        c = out[offset:offset + tokens * M]
        call(c)
        plan.check_status()
        close(c, want, 4 * ref.U * np.abs(want), "C")
        assert (out[:offset] == 7).all() and (out[offset + tokens * M:] == 7).all()


@pytest.mark.parametrize("tokens,cols", [(130, 260), (257, 260), (260, 240), (129, 1400)])
def test_int8_long_tokens(cuda, tokens, cols):
    """Tokens long and many enough to be quantised by clusters; one holds an infinity, one zeros."""
    torch = cuda
    m = ref.matrix(40, cols, 12, 42)
    q, rs = int8_weights(m, 5)
    plan = vb.Int8Plan(vb.Matrix(m), torch.from_numpy(q).cuda(), torch.from_numpy(rs).cuda())
    assert m.scalar_cols() >= 8192
    X = activations(tokens, m.scalar_cols(), 9)
    X[7, 11] = -np.inf
    Q, ts = quantized(X)
    want = (Q @ ref.dense(m, q).T) * ts[:, None].astype(np.float64) * rs
    C = torch.full((tokens, m.scalar_rows()), 7.0, device="cuda")
    plan.execute_panel(torch.from_numpy(X).cuda(), C)
    plan.check_status()
    assert torch.isnan(C[7]).all()
    keep = np.arange(tokens) != 7
    close(C[torch.from_numpy(keep).cuda()], want[keep], 4 * ref.U * np.abs(want[keep]), "C")


@pytest.mark.parametrize("K", [1, 7, 8, 100, 4096, 40009])
def test_quantize_panel(cuda, K):
    torch = cuda
    X = activations(7, K, K)
    X[1] = np.float32(1e-41) * np.sign(X[1])  # denormal: the scale is a few steps or zero
    X[3] = np.where(np.arange(K) % 2 == 0, 127.0, np.arange(K) % 127 + 0.5)  # exact halves
    X[4, 0], X[5, K - 1] = np.nan, -np.inf
    Q = torch.full((7, K), 99, dtype=torch.int8, device="cuda")
    s = torch.full((7,), -1.0, device="cuda")
    vb.quantize_panel(torch.from_numpy(X).cuda(), Q, s, K)
    torch.cuda.synchronize()
    Q, s = Q.cpu().numpy(), s.cpu().numpy()
    want, ws = quantized(X)
    ok = np.isfinite(X).all(axis=1)
    assert np.array_equal(s[ok], ws[ok]) and np.array_equal(Q[ok], want[ok])
    assert np.isnan(s[~ok]).all() and not Q[~ok].any()


def test_int8_widest_row(cuda):
    """The largest sum that 32 bits have to hold: -128 times -128 over the widest row that is not refused."""
    torch = cuda
    m = ref.matrix(1, 2048, 2048, 52, sizes=(64,), row_size=(8,), col_size=(64,) * 2047 + (56,))
    K, width = m.scalar_cols(), 131064
    assert K == width
    low = torch.full((len(m.values),), -128, dtype=torch.int8, device="cuda")
    plan = vb.Int8Plan(vb.Matrix(m), low, torch.ones(8, device="cuda"))
    for tokens in (1, 130):
        C = torch.zeros(tokens, 8, device="cuda")
        plan.execute(torch.full((tokens, K), -128, dtype=torch.int8, device="cuda"),
                     torch.ones(tokens, device="cuda"), C)
        plan.check_status()
        assert (C.cpu() == np.float32(width * 128 * 128)).all()
    wide = ref.matrix(1, 2048, 2048, 53, sizes=(64,), row_size=(8,))
    with pytest.raises(vb.InvalidArgument, match="overflow"):
        vb.Int8Plan(vb.Matrix(wide), torch.zeros(len(wide.values), dtype=torch.int8, device="cuda"),
                    torch.ones(8, device="cuda"))


def test_quantize_values_and_product(cuda):
    torch = cuda
    m = ref.matrix(9, 11, 4, 21, empty=(3,))
    M = vb.Matrix(m)
    q, s = vb.quantize_values(M)
    torch.cuda.synchronize()
    A = ref.dense(m)
    want, ws = quantized(A.astype(np.float32))
    assert np.array_equal(s.cpu().numpy(), ws)
    assert np.array_equal(q.cpu().numpy(), ref.sampled(m, want))
    X = activations(9, m.scalar_cols(), 2)
    C = torch.empty(9, m.scalar_rows(), device="cuda")
    vb.Int8Plan(M, q, s).execute_panel(torch.from_numpy(X).cuda(), C)
    torch.cuda.synchronize()
    # each weight and activation is off by at most half a step of its scale
    ex, ew = np.abs(X).max(1, keepdims=True) / 254, np.abs(A).max(1) / 254
    tol = np.abs(X) @ (ew[:, None] * (A != 0)).T + ex * np.abs(A).sum(1) + ex * ew * (A != 0).sum(1)
    close(C, X.astype(np.float64) @ A.T, tol * (1 + 1e-5), "C")


def test_int8_not_finite_zero_tokens_and_graph(cuda):
    torch = cuda
    m, _ = PAIRS["mixed"]()
    q, rs = int8_weights(m, 2)
    plan = vb.Int8Plan(vb.Matrix(m), torch.from_numpy(q).cuda(), torch.from_numpy(rs).cuda())
    X = activations(6, m.scalar_cols(), 3)
    C = torch.empty(6, m.scalar_rows(), device="cuda")
    plan.execute_panel(torch.from_numpy(X).cuda(), C)
    bad = X.copy()
    bad[1, 5] = np.inf
    dbad = torch.from_numpy(bad).cuda()
    C2 = torch.empty_like(C)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.execute_panel(dbad, C2, stream=torch.cuda.current_stream())
    g.replay()
    torch.cuda.synchronize()
    plan.check_status()
    assert torch.isnan(C2[1]).all()
    keep = torch.arange(6) != 1
    assert torch.equal(C[keep], C2[keep])
    plan.execute_panel(torch.empty(0, m.scalar_cols(), device="cuda"),
                       torch.empty(0, m.scalar_rows(), device="cuda"))


# ---- orthogonalised update -----------------------------------------------------------------------

def check_ortho(m, values, got, steps=5, eps=1e-7, coef=(3.4445, -4.7750, 2.0315)):
    """Products are held to 2^-22 where float32 arithmetic rounds to 2^-24, so the result may be four
    times as far from the 64-bit one as float32 arithmetic is, block by block in the 2-norm; where
    that happens to be small, 2^-24 per rounding of a sum of 64 and a growth of 3.98 a step (the
    polynomial's steepest slope on its range) bound it."""
    want = ref.newton_schulz(m, values, steps, eps, coef, np.float64)
    plain = ref.newton_schulz(m, values, steps, eps, coef, np.float32)
    floor = 8 * ref.U * 3.98 ** min(steps, 5)
    for _, _, _, p, h, w in ref.blocks(m):
        off, ref_off = (np.linalg.norm(x[p] - want[p]) for x in (got.astype(np.float64), plain))
        assert off <= 4 * ref_off + floor * np.linalg.norm(want[p]), (h, w, off, ref_off)


@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("scale", [1.0, 1e-20, 1e25])
def test_ortho_all_block_sizes(cuda, steps, scale):
    torch = cuda
    m = ref.matrix(8, 8, 8, 31, row_size=SIZES, col_size=SIZES, scale=scale)
    eps = 1e-7 if scale > 1e-10 else 0.0
    plan = vb.OrthoPlan(vb.Matrix(m))
    v = torch.from_numpy(m.values).cuda()
    out = torch.full_like(v, float("nan"))
    plan.execute(v, out, steps=steps, eps=eps)
    inplace = v.clone()
    plan.execute(inplace, inplace, steps=steps, eps=eps)
    torch.cuda.synchronize()
    assert torch.equal(out, inplace)
    norm = m.values.astype(np.float64) / np.float64(scale)
    check_ortho(m, (norm if eps == 0.0 else m.values.astype(np.float64)), out.cpu().numpy(), steps,
                eps)


@pytest.mark.parametrize("count", [1, 2, 3, 700])
def test_ortho_counts(cuda, count):
    """One block, an odd number, and many of one size, large and small."""
    torch = cuda
    for h, w in ((64, 40), (48, 56), (24, 64), (8, 16)):
        m = ref.matrix(count, 3, 1, count, row_size=[h] * count, col_size=[w] * 3)
        plan = vb.OrthoPlan(vb.Matrix(m))
        v = torch.from_numpy(m.values).cuda()
        out = torch.full_like(v, float("nan"))
        plan.execute(v, out, stream=torch.cuda.current_stream())
        plan.check_status()
        check_ortho(m, m.values, out.cpu().numpy())


def test_ortho_rank_one_zero_and_not_finite_blocks(cuda):
    torch = cuda
    m = ref.matrix(12, 6, 4, 33, sizes=(8, 24, 32, 64))
    v = m.values.copy()
    bl = list(ref.blocks(m))
    for k, (_, _, _, p, h, w) in enumerate(bl):
        if k % 5 == 0:
            v[p] = 0.0
        elif k % 5 == 1:  # one direction: the other singular values are zero
            v[p] = np.outer(np.linspace(1, 2, w), np.linspace(-1, 1, h)).reshape(-1)
        elif k % 5 == 2:  # already orthogonal
            x = np.zeros((w, h))
            np.fill_diagonal(x, 1.0)
            v[p] = x.reshape(-1)
    m.values = v
    bad = v.copy()
    poisoned = [bl[3], bl[7]]
    bad[poisoned[0][3].start] = np.nan
    bad[poisoned[1][3].stop - 1] = np.inf
    plan = vb.OrthoPlan(vb.Matrix(m))
    outs = []
    for x in (v, bad):
        out = torch.empty(len(x), device="cuda")
        plan.execute(torch.from_numpy(x).cuda(), out)
        outs.append(out.cpu().numpy())
    check_ortho(m, v, outs[0])
    for k, (_, _, _, p, _, _) in enumerate(bl):
        if k % 5 == 0:
            assert not outs[0][p].any()
        if k in (3, 7):
            assert np.isnan(outs[1][p]).any()
        else:
            assert np.array_equal(outs[0][p], outs[1][p])


def test_training_step_and_serving_together(cuda):
    """The operators as they are used together: forward, backward, orthogonalised update of both
    weights, the new weights in the plan, then the updated gate served in 8 bits."""
    torch = cuda
    gate, up = pair("mixed")
    M, K, T = gate.scalar_rows(), gate.scalar_cols(), 50
    X = activations(T, K, 12)
    mats = [vb.Matrix(gate), vb.Matrix(up)]
    plan, ortho = vb.GatedPlan(*mats), [vb.OrthoPlan(m) for m in mats]
    dX, (H, G, U) = run_forward(torch, plan, X, M)
    grads = [torch.empty(len(m.values), device="cuda") for m in (gate, up)]
    plan.backward(dX, G, U, torch.ones_like(H), None, *grads)
    new = []
    for o, g, m in zip(ortho, grads, (gate, up)):
        upd = torch.empty_like(g)
        o.execute(g, upd)
        check_ortho(m, g.cpu().numpy(), upd.cpu().numpy())
        w = torch.from_numpy(m.values).cuda() - 0.02 * upd
        new.append(m.copy())
        new[-1].values = w.cpu().numpy()
    plan.set_values(*(torch.from_numpy(m.values).cuda() for m in new))
    want = Gated(*new, vb.Activation.SiLU, X)
    _, (H2, _, _) = run_forward(torch, plan, X, M)
    close(H2, want.H, want.H_tol, "H")
    assert not torch.equal(H, H2)
    served = vb.Matrix(new[0])
    q, s = vb.quantize_values(served)
    C = torch.empty(T, M, device="cuda")
    vb.Int8Plan(served, q, s).execute_panel(dX, C)
    torch.cuda.synchronize()
    rel = np.linalg.norm(C.cpu().numpy() - want.G) / np.linalg.norm(want.G)
    A = ref.dense(new[0])
    ex, ew = np.abs(X).max(1, keepdims=True) / 254, np.abs(A).max(1) / 254
    tol = np.abs(X) @ (ew[:, None] * (A != 0)).T + ex * np.abs(A).sum(1) + ex * ew * (A != 0).sum(1)
    close(C, want.G, tol * (1 + 1e-5), "C")
    assert rel < 0.2


# ---- refusals ------------------------------------------------------------------------------------

def test_refusals_on_device_objects(cuda):
    torch = cuda
    gate, up = pair("mixed")
    g, u = vb.Matrix(gate), vb.Matrix(up)
    with pytest.raises(vb.InvalidArgument, match="partitions"):
        vb.GatedPlan(g, vb.Matrix(ref.matrix(9, 11, 2, 50, sizes=(64,))))
    with pytest.raises(vb.InvalidArgument, match="activation"):
        vb.GatedPlan(g, u, 9)
    plan = vb.GatedPlan(g, u)
    M, K = gate.scalar_rows(), gate.scalar_cols()
    X, H = torch.zeros(4, K, device="cuda"), torch.full((4, M), 5.0, device="cuda")
    bad = [
        (dict(B=X.cpu(), H=H), "CUDA"), (dict(B=X.half(), H=H), "float32"),
        (dict(B=X, H=H[:3]), "expected"), (dict(B=X, H=H, G=H), "together"),
        (dict(B=X.T, H=H), "contiguous"), (dict(B=X.T.contiguous(), H=H), "shape"),
        (dict(B=X.reshape(-1)[:-1], H=H), "multiple"), (dict(B=X.data_ptr(), H=H), "tokens"),
        (dict(B=X, H=H, tokens=-1), "tokens"),
        (dict(B=X.data_ptr(), H=H.data_ptr(), tokens=-1, workspace=(0, 0)), "tokens"),
        (dict(B=X.data_ptr(), H=H.data_ptr(), tokens=1 << 23, workspace=(0, 0)), "tokens"),
        (dict(B=0, H=H, tokens=4), "null"),
    ]
    for kw, msg in bad:
        with pytest.raises(vb.InvalidArgument, match=msg):
            plan.execute(**kw)
    need = plan.workspace_bytes(4, backward=True)
    small = torch.empty(max(0, need - 1), dtype=torch.uint8, device="cuda")
    back = dict(B=X, G=H, U=H, dH=H, dB=torch.empty_like(X))
    with pytest.raises(vb.InvalidArgument, match="workspace too small"):
        plan.backward(**back, workspace=small)
    with pytest.raises(vb.InvalidArgument, match="aligned"):
        plan.backward(**back, workspace=torch.empty(need + 512, dtype=torch.uint8, device="cuda")[1:])
    with pytest.raises(vb.InvalidArgument, match="together"):
        plan.backward(**back, dgate=torch.empty(len(gate.values), device="cuda"))
    with pytest.raises(vb.InvalidArgument, match="no output"):
        plan.backward(X, H, H, H)
    assert (H == 5).all()
    with pytest.raises(vb.InvalidArgument, match="int8"):
        vb.Int8Plan(g, torch.zeros(len(gate.values), device="cuda"), torch.zeros(M, device="cuda"))
    with pytest.raises(vb.InvalidArgument, match="row_scale"):
        vb.Int8Plan(g, torch.zeros(len(gate.values), dtype=torch.int8, device="cuda"),
                    torch.zeros(M - 1, device="cuda"))
    wide = ref.matrix(1, 2050, 2050, 51, sizes=(64,), row_size=(8,))
    with pytest.raises(vb.InvalidArgument, match="overflow"):
        vb.Int8Plan(vb.Matrix(wide), torch.zeros(len(wide.values), dtype=torch.int8, device="cuda"),
                    torch.zeros(8, device="cuda"))
    o = vb.OrthoPlan(g)
    v = torch.zeros(len(gate.values), device="cuda")
    for kw, msg in ((dict(steps=-1), "steps"), (dict(steps=65), "steps"), (dict(eps=-1.0), "eps"),
                    (dict(eps=float("nan")), "eps"), (dict(coefficients=(1.0,)), "three")):
        with pytest.raises(vb.InvalidArgument, match=msg):
            o.execute(v, v, **kw)
    with pytest.raises(vb.InvalidArgument, match="elements"):
        o.execute(v[:-1], v)
