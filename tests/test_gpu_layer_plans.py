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
