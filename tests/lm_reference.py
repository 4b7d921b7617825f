"""Plain 64-bit restatements of the block-sparse layer operators, and the matrices their tests use."""
import numpy as np
import torch

import varblockspmm_b200 as vb

U = 2.0 ** -24  # half a step of float32


def matrix(rows, cols, degree, seed, sizes=(8, 16, 24, 32, 40, 48, 56, 64), empty=(), skip_cols=(),
           repeat=False, row_size=None, col_size=None, scale=1.0):
    """A random host matrix: `degree` blocks per block row in random order (repeat: the same block
    column may come twice), no blocks in the rows `empty` and the columns `skip_cols`."""
    rng = np.random.default_rng(seed)
    rs = np.asarray(rng.choice(sizes, rows) if row_size is None else row_size, dtype=np.int32)
    cs = np.asarray(rng.choice(sizes, cols) if col_size is None else col_size, dtype=np.int32)
    allowed = np.setdiff1d(np.arange(cols), np.asarray(skip_cols, dtype=int))
    row_ptr, block_col, value_off = [0], [], [0]
    for i in range(rows):
        n = 0 if i in empty else (degree if repeat else min(degree, len(allowed)))
        for c in rng.choice(allowed, n, replace=repeat):
            block_col.append(int(c))
            value_off.append(value_off[-1] + int(rs[i]) * int(cs[c]))
        row_ptr.append(len(block_col))
    values = rng.standard_normal(value_off[-1]).astype(np.float32) * np.float32(scale)
    m = vb.HostMatrix(rows, cols, row_ptr, block_col, rs, cs, np.concatenate([[0], np.cumsum(rs)]),
                      np.concatenate([[0], np.cumsum(cs)]), value_off, values)
    m.validate()
    return m


def blocks(m):
    """(block, rows slice, columns slice, packed slice, h, w) of every block."""
    for i in range(m.block_rows):
        for b in range(m.row_ptr[i], m.row_ptr[i + 1]):
            c = m.block_col[b]
            yield (b, slice(m.row_scalar_off[i], m.row_scalar_off[i + 1]),
                   slice(m.col_scalar_off[c], m.col_scalar_off[c + 1]),
                   slice(m.value_off[b], m.value_off[b + 1]), int(m.row_size[i]), int(m.col_size[c]))


def dense(m, values=None):
    """The M x K matrix in float64 (repeated blocks add up)."""
    v = (m.values if values is None else np.asarray(values)).astype(np.float64)
    a = np.zeros((m.scalar_rows(), m.scalar_cols()))
    for _, r, c, p, h, w in blocks(m):
        a[r, c] += v[p].reshape(w, h).T
    return a


def sampled(m, full):
    """The packed values of an M x K matrix at the blocks of m."""
    out = np.zeros(int(m.value_off[-1]))
    for _, r, c, p, h, w in blocks(m):
        out[p] = full[r, c].T.reshape(-1)
    return out


def act(kind, x):
    """The activation and its derivative in float64."""
    x = torch.from_numpy(x).requires_grad_()
    f = {vb.Activation.SiLU: lambda t: t * torch.sigmoid(t),
         vb.Activation.GELU: torch.nn.functional.gelu,
         vb.Activation.ReLU: torch.relu, vb.Activation.Sigmoid: torch.sigmoid}[kind]
    y = f(x)
    y.sum().backward()
    return y.detach().numpy(), x.grad.numpy()


def product_tolerance(n, magnitude):
    """Bound of an fp32-accurate sum of n products of total magnitude `magnitude`: the operands are
    held to 2^-23, a product that leaves out lo * lo is off by 2^-22, and each of n additions rounds
    by at most 2^-24 of the partial sums."""
    return (4 * 2 ** -23 + n * U) * magnitude


def max_row_products(m):
    """The largest number of columns that a block row of m sums over."""
    w = m.col_size[m.block_col].astype(np.int64)
    return max([int(w[m.row_ptr[i]:m.row_ptr[i + 1]].sum()) for i in range(m.block_rows)] + [1])


def max_col_products(m):
    """The largest number of rows that a block column of m sums over."""
    s = np.zeros(m.block_cols, dtype=np.int64)
    for i in range(m.block_rows):
        np.add.at(s, m.block_col[m.row_ptr[i]:m.row_ptr[i + 1]], int(m.row_size[i]))
    return max(int(s.max()), 1)


def newton_schulz(m, values, steps, eps, coef, dtype):
    """Every block of the packed array orthogonalised, in numpy arithmetic of `dtype`."""
    out = np.zeros(len(values), dtype=dtype)
    a, b, c = (dtype(x) for x in coef)
    for _, _, _, p, h, w in blocks(m):
        x = np.asarray(values[p], dtype=dtype).reshape(w, h).T
        x = x if h <= w else x.T
        x = x / (np.sqrt((x * x).sum(dtype=dtype)) + dtype(eps)) if x.any() else x
        for _ in range(steps):
            g = x @ x.T
            x = a * x + (b * g + c * (g @ g)) @ x
        out[p] = (x if h <= w else x.T).T.reshape(-1)
    return out
