"""Plans of the block-sparse layers: what they keep of a matrix, when they have weights, and what orders
their creation with other work on the GPU."""
import numpy as np
import pytest

import lm_reference as ref
import varblockspmm_b200 as vb

pytestmark = pytest.mark.gpu


def structure(m):
    """A matrix of m's structure without its values."""
    bare = m.copy()
    bare.values = bare.values[:0]
    return vb.Matrix(bare, structure_only=True)


def pair():
    gate = ref.matrix(9, 11, 4, 1, empty=(2,))
    return gate, ref.matrix(9, 11, 3, 2, row_size=gate.row_size, col_size=gate.col_size)


def panel(torch, tokens, features, seed):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((tokens, features)).astype(np.float32)).cuda()


def test_gated_plan_from_structure_alone(cuda):
    """No weights until set_values, then the results of a plan made from whole matrices, bit by bit."""
    torch = cuda
    gate, up = pair()
    M, K, T = gate.scalar_rows(), gate.scalar_cols(), 12
    X = panel(torch, T, K, 3)
    dH = 1e-3 * panel(torch, T, M, 4)
    dev = [torch.from_numpy(m.values).cuda() for m in (gate, up)]

    def results(plan):
        H, G, U = (torch.full((T, M), float("nan"), device="cuda") for _ in range(3))
        out = [torch.full_like(t, float("nan")) for t in (X, *dev)]
        plan.execute(X, H, G, U)
        plan.backward(X, G, U, dH, *out)
        plan.check_status()
        return [H, G, U, *out]

    want = results(vb.GatedPlan(vb.Matrix(gate), vb.Matrix(up)))
    for mats in ((structure(gate), structure(up)), (vb.Matrix(gate), structure(up))):
        plan = vb.GatedPlan(*mats)
        H = torch.full((T, M), 5.0, device="cuda")
        with pytest.raises(vb.InvalidArgument, match="no weights"):
            plan.execute(X, H)
        with pytest.raises(vb.InvalidArgument, match="no weights"):
            plan.backward(X, H, H, H, torch.empty_like(X))
        torch.cuda.synchronize()
        assert (H == 5).all()
        plan.set_values(*dev)
        for a, b in zip(want, results(plan)):
            assert torch.equal(a, b)


def test_plans_outlive_their_matrices(cuda):
    torch = cuda
    gate, up = pair()
    mats = [vb.Matrix(gate), vb.Matrix(up), structure(gate)]
    plan, ortho = vb.GatedPlan(*mats[:2]), vb.OrthoPlan(mats[2])
    X, v = panel(torch, 7, gate.scalar_cols(), 5), torch.from_numpy(gate.values).cuda()
    H, upd = torch.empty(7, gate.scalar_rows(), device="cuda"), torch.empty_like(v)
    plan.execute(X, H)
    ortho.execute(v, upd)
    torch.cuda.synchronize()
    first = [H.clone(), upd.clone()]
    for m in mats:
        m.close()
    # the matrices' memory is taken over by others
    other = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(4)]
    plan.set_values(v, torch.from_numpy(up.values).cuda())
    plan.execute(X, H)
    ortho.execute(v, upd)
    torch.cuda.synchronize()
    assert torch.equal(H, first[0]) and torch.equal(upd, first[1]) and len(other) == 4


def test_gated_plan_without_blocks_has_its_weights(cuda):
    torch = cuda
    m = ref.matrix(3, 4, 0, 13)
    plan = vb.GatedPlan(structure(m), structure(m), vb.Activation.Sigmoid)
    H = torch.full((5, m.scalar_rows()), 7.0, device="cuda")
    plan.execute(panel(torch, 5, m.scalar_cols(), 1), H)
    plan.check_status()
    assert (H == 0).all()


def int8_case(torch, tokens=19, seed=6):
    m = ref.matrix(9, 11, 5, seed, empty=(4,))
    rng = np.random.default_rng(seed)
    q = [torch.from_numpy(rng.integers(-128, 128, len(m.values)).astype(np.int8)).cuda() for _ in range(2)]
    s = [torch.from_numpy((rng.random(m.scalar_rows()) + 0.1).astype(np.float32)).cuda() for _ in range(2)]
    Q = torch.from_numpy(rng.integers(-127, 128, (tokens, m.scalar_cols())).astype(np.int8)).cuda()
    ts = torch.from_numpy((rng.random(tokens) + 0.1).astype(np.float32)).cuda()
    want = [(Q.cpu().numpy().astype(np.float64) @ ref.dense(m, q[i].cpu().numpy()).T) *
            (ts.cpu().numpy()[:, None].astype(np.float64) * s[i].cpu().numpy()) for i in range(2)]
    return m, q, s, Q, ts, want


def int8_close(C, want):
    """The sum, the product of the scales and the result round once each."""
    got = C.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= 4 * ref.U * np.abs(want))


def test_int8_plan_from_structure_and_other_weights(cuda):
    """No weights until set_values; set_values replaces them, captured and replayed too."""
    torch = cuda
    m, q, s, Q, ts, want = int8_case(torch)
    plan = vb.Int8Plan(structure(m))
    C = torch.full((len(Q), m.scalar_rows()), 5.0, device="cuda")
    for call in (lambda: plan.execute(Q, ts, C), lambda: plan.execute_panel(Q.float(), C)):
        with pytest.raises(vb.InvalidArgument, match="no weights"):
            call()
    torch.cuda.synchronize()
    assert (C == 5).all()
    for i in (0, 1, 0):
        plan.set_values(q[i], s[i])
        plan.execute(Q, ts, C)
        plan.check_status()
        int8_close(C, want[i])
    g = torch.cuda.CUDAGraph()
    values, scales = q[0].clone(), s[0].clone()
    with torch.cuda.graph(g):
        plan.set_values(values, scales, stream=torch.cuda.current_stream())
        plan.execute(Q, ts, C, stream=torch.cuda.current_stream())
    for i in (1, 0):
        values.copy_(q[i])
        scales.copy_(s[i])
        g.replay()
        torch.cuda.synchronize()
        int8_close(C, want[i])


@pytest.mark.parametrize("offset", [1, 4, 8])
def test_int8_weights_at_any_alignment(cuda, offset):
    torch = cuda
    m, q, s, Q, ts, want = int8_case(torch, 5, 8)
    buf = torch.zeros(len(q[0]) + 16, dtype=torch.int8, device="cuda")
    v = buf[offset:offset + len(q[0])]
    v.copy_(q[0])
    plan = vb.Int8Plan(structure(m), v, s[0])
    C = torch.full((len(Q), m.scalar_rows()), float("nan"), device="cuda")
    plan.execute(Q, ts, C)
    plan.check_status()
    int8_close(C, want[0])


@pytest.mark.parametrize("size", [8, 16, 24, 40, 56, 64])
def test_int8_layout_of_every_block_width(cuda, size):
    torch = cuda
    sizes = (8, 16, 24, 32, 40, 48, 56, 64)
    m = ref.matrix(8, 8, 5, size, row_size=sizes, col_size=[size] * 8, repeat=True)
    rng = np.random.default_rng(size)
    q = rng.integers(-128, 128, len(m.values)).astype(np.int8)
    Q = rng.integers(-127, 128, (3, m.scalar_cols())).astype(np.int8)
    plan = vb.Int8Plan(structure(m), torch.from_numpy(q).cuda(), torch.ones(m.scalar_rows(), device="cuda"))
    C = torch.full((3, m.scalar_rows()), float("nan"), device="cuda")
    plan.execute(torch.from_numpy(Q).cuda(), torch.ones(3, device="cuda"), C)
    plan.check_status()
    # whole numbers below 2^24: exact
    assert np.array_equal(C.cpu().numpy().astype(np.float64), Q.astype(np.float64) @ ref.dense(m, q).T)


def test_int8_creation_waits_for_weights_made_on_another_stream(cuda):
    """Weights whose quantisation is still behind other work on a side stream when the plan is made."""
    torch = cuda
    m = ref.matrix(9, 11, 5, 7)
    M = vb.Matrix(m)
    q, s = vb.quantize_values(M)
    torch.cuda.synchronize()
    X = panel(torch, 6, m.scalar_cols(), 9)
    want = torch.empty(6, m.scalar_rows(), device="cuda")
    vb.Int8Plan(M, q, s).execute_panel(X, want)
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(40):  # some tens of ms
                busy = (busy @ busy).clamp_(-1, 1)
        q2, s2 = vb.quantize_values(M, stream=side)
        C = torch.empty_like(want)
        vb.Int8Plan(M, q2, s2).execute_panel(X, C)
        torch.cuda.synchronize()
        assert torch.equal(C, want)


def test_new_plans_are_usable_from_any_stream_at_once(cuda):
    """A plan's tables are complete when its creation returns, whatever stream runs its first call."""
    torch = cuda
    m = ref.matrix(300, 40, 12, 31)
    bare, v = structure(m), torch.from_numpy(m.values).cuda()
    X, dH = panel(torch, 9, m.scalar_cols(), 1), panel(torch, 9, m.scalar_rows(), 2)
    rng = np.random.default_rng(3)
    q = torch.from_numpy(rng.integers(-127, 128, len(m.values)).astype(np.int8)).cuda()
    scale = torch.ones(m.scalar_rows(), device="cuda")
    want = None
    torch.cuda.synchronize()
    for k in range(12):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            out = [torch.zeros_like(v) for _ in range(3)] + [torch.zeros_like(dH) for _ in range(4)]
            vb.OrthoPlan(bare).execute(v, out[0], stream=s)
            plan = vb.GatedPlan(bare, bare)
            plan.set_values(v, v, stream=s)
            plan.execute(X, *out[3:6], stream=s)
            plan.backward(X, out[4], out[5], dH, None, out[1], out[2], stream=s)
            i8 = vb.Int8Plan(bare)
            i8.set_values(q, scale, stream=s)
            i8.execute_panel(X, out[6], stream=s)
        s.synchronize()
        want = want or [t.clone() for t in out]
        for a, b in zip(want, out):
            assert torch.equal(a, b), k
