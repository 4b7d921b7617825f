"""Measured cases of the block-sparse operators for language models: the gated feed-forward block
with its backward pass (GatedPlan), the 8-bit integer product (Int8Plan) and the orthogonalised block
update (OrthoPlan).

Activations are [tokens, features] row-major, which is the engine's column-major features x tokens
panel. Weights are VBSR matrices; `values` is the packed reference layout (blocks in row order, each
column-major). Block sizes follow the engine's four distributions.
"""
import math

import numpy as np
import torch

own = False

_SIZES = {
    "uniform": ([8, 16, 24, 32, 40, 48, 56, 64], None),
    "low": ([24, 32, 40], [0.25, 0.5, 0.25]),
    "high": ([8, 16, 56, 64], [0.3, 0.2, 0.2, 0.3]),
    "bimodal": ([8, 64], [0.5, 0.5]),
}
_MEAN = {"uniform": 36.0, "low": 32.0, "high": 35.2, "bimodal": 36.0}
_COEF = (3.4445, -4.7750, 2.0315)
_EPS = 1e-7
_STEPS = 5


def _case(name, op, rows, cols, degree, dist, tokens=0, act="silu", empty=0.0):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "degree": degree, "dist": dist,
            "tokens": tokens, "act": act, "empty": empty}


def listed():
    return [
        # the gated block on the engine's 256-row correctness matrix, a handful of tokens: latency
        _case("gated 256r d4 8 tokens", "gated", 256, 256, 4, "uniform", 8, "gelu", 0.05),
        # one token decoded through the wide-panel matrix: streams both weights once
        _case("gated 1024r d16 1 token", "gated", 1024, 1024, 16, "bimodal", 1),
        # a serving batch on the headline matrix (4096 block rows, degree 8)
        _case("gated 4096r d8 32 tokens", "gated", 4096, 4096, 8, "high", 32),
        # a prompt of an odd length
        _case("gated 1024r d16 517 tokens", "gated", 1024, 512, 16, "uniform", 517),
        # a training step (weights re-laid, forward, backward), small batch
        _case("train 1024r d8 256 tokens", "train", 1024, 1024, 8, "low", 256),
        # a training step, ragged token count, some block rows pruned away
        _case("train 512r d16 1000 tokens", "train", 512, 512, 16, "uniform", 1000, "gelu", 0.05),
        # 8-bit decoding of one token, headline matrix
        _case("int8 4096r d8 1 token", "int8", 4096, 4096, 8, "high", 1),
        # 8-bit serving batch, wide-panel matrix
        _case("int8 1024r d16 64 tokens", "int8", 1024, 1024, 16, "bimodal", 64),
        # 8-bit prompt of an odd length
        _case("int8 1024r d16 777 tokens", "int8", 1024, 1024, 16, "uniform", 777, "silu", 0.05),
        # update of a small matrix: latency
        _case("ortho 256r d4", "ortho", 256, 256, 4, "uniform"),
        # update of the headline matrix, of the wide-panel matrix (8 x 8 to 64 x 64 blocks)
        _case("ortho 4096r d8", "ortho", 4096, 4096, 8, "high"),
        _case("ortho 1024r d16", "ortho", 1024, 1024, 16, "bimodal"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Block rows and columns 48..4096, degree 1..32, tokens 1..1200, every block-size distribution
    and activation; values and values x tokens stay below the largest listed ones."""
    op = rng.choice(["gated", "gated", "train", "int8", "int8", "ortho"])
    dist = rng.choice(sorted(_SIZES))
    while True:
        rows, cols = _log_int(rng, 48, 4096), _log_int(rng, 48, 4096)
        degree = _log_int(rng, 1, 32)
        tokens = 0 if op == "ortho" else _log_int(rng, 16 if op == "train" else 1, 1200)
        values = rows * degree * _MEAN[dist] ** 2
        if 1e5 <= values <= 3.6e7 and values * max(tokens, 1) <= 9e9 and rows * cols <= 1 << 23 and (
                op != "train" or values * tokens <= 6e9):
            break
    return {"op": op, "rows": rows, "cols": cols, "degree": degree, "dist": dist, "tokens": tokens,
            "act": rng.choice(["silu", "gelu", "relu", "sigmoid"]) if op in ("gated", "train") else "silu",
            "empty": rng.choice([0.0, 0.0, 0.05])}


# ---- inputs ----------------------------------------------------------------------------------


def _structure(case, g, row_size, col_size, rng):
    """A VBSR structure: `degree` distinct block columns per block row (sorted), a share `empty` of
    the block rows without blocks."""
    rows, cols = case["rows"], case["cols"]
    degree = min(case["degree"], cols)
    pick = torch.rand(rows, cols, generator=g, device="cuda").topk(degree, dim=1).indices
    block_col = pick.sort(dim=1).values.cpu().numpy().astype(np.int32)
    keep = rng.random(rows) >= case["empty"]
    keep[0] = True
    count = np.where(keep, degree, 0)
    block_col = block_col[keep].reshape(-1)
    row_ptr = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    block_row = np.repeat(np.arange(rows, dtype=np.int32), count)
    h, w = row_size[block_row].astype(np.int64), col_size[block_col].astype(np.int64)
    value_off = np.concatenate([[0], np.cumsum(h * w)])
    return {"row_ptr": row_ptr, "block_col": block_col, "block_row": block_row, "h": h, "w": w,
            "value_off": value_off, "row_size": row_size, "col_size": col_size,
            "row_off": np.concatenate([[0], np.cumsum(row_size.astype(np.int64))]),
            "col_off": np.concatenate([[0], np.cumsum(col_size.astype(np.int64))])}


def _sub_blocks(st):
    """The matrix as 8 x 8 sub-blocks: their row and column in units of 8, and the packed positions
    of their values, [S, 8 columns, 8 rows]."""
    nh, nw = st["h"] // 8, st["w"] // 8
    n = nh * nw
    b = np.repeat(np.arange(len(n)), n)
    i = np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n)
    r8, c8 = i % nh[b], i // nh[b]
    row8 = st["row_off"][st["block_row"][b]] // 8 + r8
    col8 = st["col_off"][st["block_col"][b]] // 8 + c8
    base = st["value_off"][b] + 8 * r8 + 8 * c8 * st["h"][b]
    dev = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (row8, col8, base, st["h"][b])]
    k = torch.arange(8, device="cuda")
    at = dev[2][:, None, None] + dev[3][:, None, None] * k[None, :, None] + k[None, None, :]
    return {"row8": dev[0], "col8": dev[1], "at": at}


def _values(st, g):
    """Weights of variance 1 / fan-in, as trained layers have them."""
    fan = max(1.0, float(st["w"].sum()) / max(1, len(st["row_size"])))
    return torch.randn(int(st["value_off"][-1]), generator=g, device="cuda") / math.sqrt(fan)


def _activations(tokens, features, g):
    """Tokens of differing size with a few large features, as the residual stream has them."""
    x = torch.randn(tokens, features, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(tokens, 1, generator=g, device="cuda"))
    x[:, :: 97] *= 12.0
    return x


def _matrix(vb, st):
    """The structure alone: plans are made before there are values."""
    host = vb.HostMatrix(len(st["row_size"]), len(st["col_size"]), st["row_ptr"], st["block_col"],
                         st["row_size"], st["col_size"], st["row_off"], st["col_off"], st["value_off"])
    return vb.Matrix(host, structure_only=True)


def _inputs(case, seed):
    # the structure belongs to the case, the numbers in it come from the seed
    rng = np.random.default_rng([case["rows"], case["cols"], case["degree"]])
    sg, g = torch.Generator(device="cuda"), torch.Generator(device="cuda")
    sg.manual_seed(case["rows"] + 7 * case["cols"])
    g.manual_seed(seed)
    sizes, p = _SIZES[case["dist"]]
    row_size = rng.choice(sizes, case["rows"], p=p).astype(np.int32)
    col_size = rng.choice(sizes, case["cols"], p=p).astype(np.int32)
    op, T = case["op"], case["tokens"]
    st = _structure(case, sg, row_size, col_size, rng)
    M, K = int(st["row_off"][-1]), int(st["col_off"][-1])
    s = {"case": case, "st": st, "M": M, "K": K}
    if op in ("gated", "train"):
        s["st_up"] = _structure(case, sg, row_size, col_size, rng)
        s["gate"], s["up"] = _values(st, g), _values(s["st_up"], g)
        s["X"] = _activations(T, K, g)
        if op == "train":
            s["dH"] = 1e-3 * torch.randn(T, M, generator=g, device="cuda")
    elif op == "int8":
        s["values"] = torch.randint(-127, 128, (int(st["value_off"][-1]),), generator=g,
                                    device="cuda", dtype=torch.int8)
        s["row_scale"] = torch.rand(M, generator=g, device="cuda") * 1e-3 + 1e-4
        s["X"] = _activations(T, K, g)
    else:
        # gradients of a batch smaller than the block: a few strong directions over noise
        n = int(st["value_off"][-1])
        s["grad"] = 1e-4 * torch.randn(n, generator=g, device="cuda")
        s["grad"] *= 1.0 + 3.0 * torch.rand(n, generator=g, device="cuda").square()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    op, T, M, K, st = case["op"], case["tokens"], s["M"], s["K"], s["st"]
    dev = "cuda"
    if own:
        import varblockspmm_b200 as vb
        if op in ("gated", "train"):
            act = {"silu": vb.Activation.SiLU, "gelu": vb.Activation.GELU, "relu": vb.Activation.ReLU,
                   "sigmoid": vb.Activation.Sigmoid}[case["act"]]
            s["plan"] = vb.GatedPlan(_matrix(vb, st), _matrix(vb, s["st_up"]), act)
            s["H"] = torch.empty(T, M, device=dev)
            need = s["plan"].workspace_bytes(T, backward=op == "train")
            s["workspace"] = torch.empty(need, dtype=torch.uint8, device=dev)
            if op == "train":
                s["G"], s["U"] = torch.empty(T, M, device=dev), torch.empty(T, M, device=dev)
                s["dX"] = torch.empty(T, K, device=dev)
                s["dgate"], s["dup"] = torch.empty_like(s["gate"]), torch.empty_like(s["up"])
        elif op == "int8":
            s["plan"] = vb.Int8Plan(_matrix(vb, st))
            s["C"] = torch.empty(T, M, device=dev)
            s["workspace"] = torch.empty(s["plan"].workspace_bytes(T), dtype=torch.uint8, device=dev)
        else:
            s["plan"] = vb.OrthoPlan(_matrix(vb, st))
            s["out"] = torch.empty_like(s["grad"])
    elif op in ("gated", "train"):
        s["sub"], s["sub_up"] = _sub_blocks(st), _sub_blocks(s["st_up"])
    elif op == "int8":
        s["sub"] = _sub_blocks(st)
    else:
        # every block as a 64 x 64 tile, zeros outside it: packed position or -1
        h, w = (torch.from_numpy(st[k]).cuda() for k in ("h", "w"))
        off = torch.from_numpy(st["value_off"][:-1]).cuda()
        k = torch.arange(64, device=dev)
        r, c = k[None, :, None], k[None, None, :]
        h, w, off = h[:, None, None], w[:, None, None], off[:, None, None]
        s["at"] = torch.where((r < h) & (c < w), off + r + c * h, -1)
    return s


# ---- one pass --------------------------------------------------------------------------------


def _groups(x):
    """[T, features] as [features / 8, T, 8]."""
    return x.reshape(x.shape[0], -1, 8).permute(1, 0, 2)


def _panel(x8):
    return x8.permute(1, 0, 2).reshape(x8.shape[1], -1)


def _product(sub, values, x, features):
    """A x for the sub-blocks of A: [T, features]."""
    y = torch.bmm(_groups(x)[sub["col8"]], values[sub["at"]])
    out = torch.zeros(features // 8, x.shape[0], 8, device=x.device)
    return _panel(out.index_add_(0, sub["row8"], y))


def _product_t(sub, values, dy, features):
    """A^T dy: [T, features]."""
    y = torch.bmm(_groups(dy)[sub["row8"]], values[sub["at"]].transpose(1, 2))
    out = torch.zeros(features // 8, dy.shape[0], 8, device=dy.device)
    return _panel(out.index_add_(0, sub["col8"], y))


def _sampled(sub, dy, x, like):
    """dy x^T at the blocks of A, packed."""
    d = torch.bmm(_groups(x)[sub["col8"]].transpose(1, 2), _groups(dy)[sub["row8"]])
    out = torch.empty_like(like)
    out[sub["at"]] = d
    return out


def _act(name, g):
    """The activation and its derivative."""
    if name == "relu":
        return g * (g > 0), (g > 0).to(g.dtype)
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


def _newton_schulz(x):
    a = torch.bmm(x, x.transpose(1, 2))
    return _COEF[0] * x + torch.bmm(_COEF[1] * a + _COEF[2] * torch.bmm(a, a), x)


def run(s):
    op = s["case"]["op"]
    if own:
        # the weights are packed values, as for the plain form: what the kernels make of them is part of the pass
        stream = torch.cuda.current_stream()
        if op == "gated":
            s["plan"].set_values(s["gate"], s["up"], stream=stream)
            s["plan"].execute(s["X"], s["H"], workspace=s["workspace"], stream=stream)
            return s["H"]
        if op == "train":
            s["plan"].set_values(s["gate"], s["up"], stream=stream)
            s["plan"].execute(s["X"], s["H"], s["G"], s["U"], workspace=s["workspace"], stream=stream)
            s["plan"].backward(s["X"], s["G"], s["U"], s["dH"], s["dX"], s["dgate"], s["dup"],
                               workspace=s["workspace"], stream=stream)
            return {"H": s["H"], "dX": s["dX"], "dgate": s["dgate"], "dup": s["dup"]}
        if op == "int8":
            s["plan"].set_values(s["values"], s["row_scale"], stream=stream)
            s["plan"].execute_panel(s["X"], s["C"], workspace=s["workspace"], stream=stream)
            return s["C"]
        s["plan"].execute(s["grad"], s["out"], steps=_STEPS, eps=_EPS, coefficients=_COEF, stream=stream)
        return s["out"]
    if op == "gated":
        g = _product(s["sub"], s["gate"], s["X"], s["M"])
        u = _product(s["sub_up"], s["up"], s["X"], s["M"])
        return _act(s["case"]["act"], g)[0] * u
    if op == "train":
        g = _product(s["sub"], s["gate"], s["X"], s["M"])
        u = _product(s["sub_up"], s["up"], s["X"], s["M"])
        a, da = _act(s["case"]["act"], g)
        dg, du = s["dH"] * u * da, s["dH"] * a
        dx = _product_t(s["sub"], s["gate"], dg, s["K"]) + _product_t(s["sub_up"], s["up"], du, s["K"])
        return {"H": a * u, "dX": dx, "dgate": _sampled(s["sub"], dg, s["X"], s["gate"]),
                "dup": _sampled(s["sub_up"], du, s["X"], s["up"])}
    if op == "int8":
        # the token scale is a 32-bit number; the quotient is rounded in 64 bits (values next to a half)
        scale = s["X"].abs().amax(dim=1, keepdim=True) / 127.0
        q = torch.where(scale > 0, torch.round(s["X"].double() / scale.double()), 0.0).float()
        # sums of 8 products of 8-bit numbers are exact in 32-bit floats, their sums in 32-bit integers
        y = torch.bmm(_groups(q)[s["sub"]["col8"]], s["values"][s["sub"]["at"]].float()).to(torch.int32)
        acc = torch.zeros(s["M"] // 8, q.shape[0], 8, dtype=torch.int32, device=q.device)
        acc = _panel(acc.index_add_(0, s["sub"]["row8"], y))
        return acc.float() * (scale * s["row_scale"])
    x = torch.where(s["at"] >= 0, s["grad"][s["at"].clamp(min=0)], 0.0)
    x = x / (x.square().sum(dim=(1, 2), keepdim=True).sqrt() + _EPS)
    x = _newton_schulz(_newton_schulz(_newton_schulz(_newton_schulz(_newton_schulz(x)))))
    inside = s["at"] >= 0
    out = torch.empty_like(s["grad"])
    out[s["at"][inside]] = x[inside]
    return out


def work(case):
    op, T = case["op"], case["tokens"]
    mean = _MEAN[case["dist"]]
    blocks = case["rows"] * min(case["degree"], case["cols"]) * (1.0 - case["empty"])
    n = blocks * mean * mean
    M, K = case["rows"] * mean, case["cols"] * mean
    if op == "gated":
        return {"bytes": 8 * n + 4 * T * (K + M), "flops": 4 * n * T}
    if op == "train":
        # weights read, re-laid, read by the products both ways, gradients written; X, G, U, dH, H, dX
        return {"bytes": 8 * n * 2 + 4 * T * (3 * K + 6 * M), "flops": 12 * n * T}
    if op == "int8":
        return {"bytes": n + 4 * T * (K + M), "flops": 2 * n * T}
    sizes, p = _SIZES[case["dist"]]
    p = p or [1.0 / len(sizes)] * len(sizes)
    per = sum(ph * pw * (4 * min(h, w) * h * w + 2 * min(h, w) ** 3)
              for h, ph in zip(sizes, p) for w, pw in zip(sizes, p))
    return {"bytes": 8 * n, "flops": blocks * per * _STEPS}


# ---- the definitions in 64 bits --------------------------------------------------------------
# A block row's packed values are one [columns, h] matrix, columns in the order of its blocks.


def _rows64(st, values):
    """Per non-empty block row: (first row, h, its scalar columns, its [columns, h] values)."""
    for i in np.flatnonzero(np.diff(st["row_ptr"])):
        b0, b1 = st["row_ptr"][i], st["row_ptr"][i + 1]
        h = int(st["row_size"][i])
        cols = np.concatenate([np.arange(st["col_off"][c], st["col_off"][c + 1])
                               for c in st["block_col"][b0:b1]])
        v0, v1 = int(st["value_off"][b0]), int(st["value_off"][b1])
        yield int(st["row_off"][i]), h, torch.from_numpy(cols).cuda(), values[v0:v1].double().view(-1, h)


def _exact_product(st, values, xt, rows):
    y = torch.zeros(rows, xt.shape[1], dtype=torch.float64, device="cuda")
    for r0, h, cols, a in _rows64(st, values):
        y[r0:r0 + h] = a.T @ xt[cols]
    return y


def _exact_backward(st, values, xt, dyt, dxt):
    d = torch.zeros(values.numel(), dtype=torch.float64, device="cuda")
    at = 0
    for r0, h, cols, a in _rows64(st, values):
        dxt[cols] += a @ dyt[r0:r0 + h]
        d[at:at + a.numel()] = (xt[cols] @ dyt[r0:r0 + h].T).reshape(-1)
        at += a.numel()
    return d


def exact(case, seed):
    s = _inputs(case, seed)
    op, st = case["op"], s["st"]
    if op in ("gated", "train"):
        xt = s["X"].double().T.contiguous()
        g = _exact_product(st, s["gate"], xt, s["M"])
        u = _exact_product(s["st_up"], s["up"], xt, s["M"])
        if case["act"] == "relu":
            a, da = torch.clamp(g, min=0), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device="cuda"))
        elif case["act"] == "gelu":
            phi = torch.special.ndtr(g)
            a, da = g * phi, phi + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        elif case["act"] == "sigmoid":
            a = torch.sigmoid(g)
            da = a - a.square()
        else:
            p = torch.sigmoid(g)
            a, da = g * p, p + g * (p - p.square())
        if op == "gated":
            return (a * u).T.contiguous()
        dht = s["dH"].double().T
        dxt = torch.zeros_like(xt)
        dgate = _exact_backward(st, s["gate"], xt, dht * u * da, dxt)
        dup = _exact_backward(s["st_up"], s["up"], xt, dht * a, dxt)
        return {"H": (a * u).T.contiguous(), "dX": dxt.T.contiguous(), "dgate": dgate, "dup": dup}
    if op == "int8":
        scale = (s["X"].abs().amax(dim=1) / 127.0).double()[:, None]
        q = torch.nan_to_num(torch.round(s["X"].double() / scale), nan=0.0)
        c = _exact_product(st, s["values"], q.T.contiguous(), s["M"]).T
        return c * scale * s["row_scale"].double()
    out = torch.empty(s["grad"].numel(), dtype=torch.float64, device="cuda")
    grad = s["grad"].double()
    for h, w in sorted({(int(h), int(w)) for h, w in zip(st["h"], st["w"])}):
        off = torch.from_numpy(st["value_off"][:-1][(st["h"] == h) & (st["w"] == w)]).cuda()
        at = off[:, None] + torch.arange(h * w, device="cuda")[None, :]
        x = grad[at].view(-1, w, h)  # the transposed block: the formula commutes with transposition
        x = x / (torch.linalg.matrix_norm(x)[:, None, None] + _EPS)
        for _ in range(_STEPS):
            a = x @ x.transpose(1, 2)
            x = _COEF[0] * x + (_COEF[1] * a + _COEF[2] * (a @ a)) @ x
        out[at] = x.reshape(-1, h * w)
    return out
