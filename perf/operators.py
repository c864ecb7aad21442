"""Cases, plain forms and 64-bit values of the training-side operators.

Operators (all over ``[B, H, S, D]`` tensors, block lists as segmented CSR):

* ``rope``: rotary positions on q and k, text tokens left alone; ``inverse``
  is the gradient of the rotation (the transposed one).
* ``fwd``: block-sparse attention that also returns the row log-sum-exp.
* ``bwd``: its gradient, from q, k, v, the output, the log-sum-exp and the
  output's gradient.

The plain forms evaluate each listed block as one small matrix product in
32 bits; rows that see no key give zeros (log-sum-exp -inf).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _attn(name, op, dtype, B, H, Sq, Sk, D, bm, bn, density, text=0, grid=(0, 0, 0), empty=0, strided=False):
    """``text``: leading tokens whose row and column blocks are all live;
    ``grid``: (frames, height, width) of the video tokens that follow, (0, 0, 0)
    for values without a spatial structure; ``empty``: every so many-th row
    block sees nothing (0: none); ``strided``: ``[B, S, H, D]`` storage."""
    return {"name": name, "op": op, "dtype": dtype, "B": B, "H": H, "Sq": Sq, "Sk": Sk, "D": D, "bm": bm, "bn": bn,
            "density": density, "text": text, "frames": grid[0], "height": grid[1], "width": grid[2],
            "empty": empty, "strided": strided}


def _rope(name, dtype, B, H, D, R, text, grid, layout, inverse, factor=1.0, strided=False):
    """``R``: rotated channels of the head; ``factor``: positions divided by it."""
    return {"name": name, "op": "rope", "dtype": dtype, "B": B, "H": H, "D": D, "R": R, "text": text,
            "frames": grid[0], "height": grid[1], "width": grid[2], "layout": layout, "inverse": inverse,
            "factor": factor, "strided": strided}


def listed():
    return [
        # the framework's smoke geometry: two heads of a short clip, one call's latency
        _rope("rope_short", "bf16", 1, 2, 64, 64, 130, (4, 10, 16), "interleaved", False),
        # one layer of the default video geometry, both halves of the guidance batch
        _rope("rope_layer", "bf16", 2, 30, 64, 64, 226, (13, 30, 45), "interleaved", False),
        # the gradient at the largest geometry: half layout on half of the head, stretched positions, q and k
        # straight from a [B, S, H, D] projection
        _rope("rope_back_large", "f16", 1, 30, 64, 32, 224, (11, 48, 85), "half", True, 2.0, True),
        # one query against a short context: the least a call can cost
        _attn("fwd_one_token", "fwd", "f16", 1, 2, 1, 200, 64, 128, 128, 1.0),
        # short clip, 64-token blocks
        _attn("fwd_short", "fwd", "bf16", 1, 2, 770, 770, 64, 64, 64, 0.25, 130, (4, 10, 16)),
        # the training forward of one layer at the default geometry and density
        _attn("fwd_layer", "fwd", "bf16", 2, 30, 17776, 17776, 64, 128, 128, 0.10, 226, (13, 30, 45)),
        # the fp32 check configuration
        _attn("fwd_f32", "fwd", "f32", 1, 2, 2048, 2048, 64, 64, 64, 0.25),
        # gradients of the same three, and of what a user's masks and shards look like
        _attn("bwd_short", "bwd", "bf16", 1, 2, 770, 770, 64, 64, 64, 0.25, 130, (4, 10, 16)),
        # cross lengths, neither a multiple of its block, unlike block sizes, rows that see nothing
        _attn("bwd_ragged", "bwd", "bf16", 2, 3, 1500, 1111, 64, 64, 128, 0.35, 0, (0, 0, 0), 5),
        # one of eight GPUs' heads of the long geometry, straight from a [B, S, H, D] projection
        _attn("bwd_long_share", "bwd", "f16", 1, 4, 33976, 33976, 64, 128, 128, 0.10, 226, (25, 30, 45), 0, True),
        # one layer at the default geometry and density: the largest
        _attn("bwd_layer", "bwd", "bf16", 2, 30, 17776, 17776, 64, 128, 128, 0.10, 226, (13, 30, 45)),
        # the fp32 check configuration
        _attn("bwd_f32", "bwd", "f32", 1, 2, 2048, 2048, 64, 64, 64, 0.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "fwd", "bwd", "bwd"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    B, H = rng.randint(1, 2), _log(rng, 1, 30)
    if op == "rope":
        grid = (rng.randint(1, 13), rng.randint(3, 40), rng.randint(3, 60))
        D = rng.choice([64, 128])
        case = _rope("", dtype, B, H, D, rng.choice([D, D // 2, 24]), rng.randint(0, 300), grid,
                     rng.choice(["interleaved", "half"]), rng.random() < 0.5, rng.choice([1.0, 1.5, 4.0]),
                     rng.random() < 0.5)
    else:
        f32 = dtype == "f32"
        S = _log(rng, 1, 4096 if f32 else 16000)
        H = min(H, 4) if f32 else H
        cross = rng.random() < 0.4
        blocks = [64, 128]
        case = _attn("", op, dtype, B, H, S, _log(rng, 1, 2 * S) if cross else S,
                     rng.choice([64, 128]) if f32 else 64, rng.choice(blocks), rng.choice(blocks),
                     rng.choice([0.1, 0.2, 1.0 if S < 1500 else 0.15]), 0 if cross else rng.choice([0, rng.randint(0, min(S, 250))]),
                     (0, 0, 0), rng.choice([0, 0, 3, 7]), rng.random() < 0.4)
    del case["name"]
    return case


# --------------------------------------------------------------------------- inputs

def _blocks(case):
    """Row blocks, column blocks, dense rows, dense columns, picked columns a row."""
    nbq, nbk = -(-case["Sq"] // case["bm"]), -(-case["Sk"] // case["bn"])
    tq = min(nbq, -(-case["text"] // case["bm"]))
    tk = min(nbk, -(-case["text"] // case["bn"]))
    return nbq, nbk, tq, tk, min(nbk - tk, math.ceil(case["density"] * nbk))


def _randn(g, shape, strided):
    """N(0, 1) values ``[B, H, S, D]``, optionally a view of ``[B, S, H, D]`` storage."""
    B, H, S, D = shape
    if strided:
        return torch.randn(B, S, H, D, generator=g, device="cuda").transpose(1, 2)
    return torch.randn(B, H, S, D, generator=g, device="cuda")


def _field(case, x, g):
    """Adds to the video rows of ``x`` what neighbouring tokens share: one value
    for each (2, 4, 4) cell of the grid and channel, twice the size of the rest."""
    F, h, w = case["frames"], case["height"], case["width"]
    B, H, S, D = x.shape
    if F == 0:
        return x
    coarse = torch.randn(B, H, -(-F // 2), -(-h // 4), -(-w // 4), D, generator=g, device="cuda")
    at = torch.arange(max(F, h, w), device="cuda")
    fine = coarse[:, :, at[:F] // 2][:, :, :, at[:h] // 4][:, :, :, :, at[:w] // 4].reshape(B, H, F * h * w, D)
    x[:, :, S - F * h * w:].mul_(0.5).add_(fine)
    return x


def _means(x, b):
    S = x.shape[2]
    n = -(-S // b)
    y = torch.nn.functional.pad(x.float(), (0, 0, 0, n * b - S))
    return y.reshape(*x.shape[:2], n, b, x.shape[3]).sum(3)


def _list(case, q, k):
    """Segmented CSR of the live blocks: the columns of the highest block-mean
    scores of every row block, dense text rows and columns, rows left empty."""
    nbq, nbk, tq, tk, top = _blocks(case)
    B, H = case["B"], case["H"]
    score = torch.matmul(_means(q, case["bm"]), _means(k, case["bn"]).transpose(-1, -2))
    score[..., :tk] = -math.inf
    mask = torch.zeros(B, H, nbq, nbk, dtype=torch.bool, device="cuda")
    if top:
        mask.scatter_(-1, score.topk(top, dim=-1).indices, True)
    mask[..., :tk] = True
    mask[:, :, :tq] = True
    if case["empty"]:
        mask[:, :, case["empty"] - 1::case["empty"]] = False
    m = mask.reshape(B * H, nbq, nbk)
    row_ptr = torch.zeros(B * H, nbq + 1, dtype=torch.int64, device="cuda")
    row_ptr[:, 1:] = m.sum(-1).cumsum(-1)
    at = m.reshape(B * H, -1).cumsum(-1) - 1
    live = m.reshape(B * H, -1)
    start = torch.arange(B * H, device="cuda")[:, None] * (nbq * nbk)
    col_idx = torch.zeros(B * H * nbq * nbk, dtype=torch.int32, device="cuda")
    col = torch.arange(nbk, dtype=torch.int32, device="cuda").repeat(B * H, nbq)
    col_idx[(at + start)[live]] = col[live]
    return (row_ptr + start).to(torch.int32), col_idx, int(live.sum())


def _table(case):
    """cos and sin of every video token's angles, ``[tokens, R / 2]``: the
    rotated channels shared out over (t, h, w) as 1 : 1.5 : 1.5."""
    R, grid = case["R"], (case["frames"], case["height"], case["width"])
    rt = R // 8 * 2
    dims = (rt, (R - rt) // 4 * 2, R - rt - (R - rt) // 4 * 2)
    angles = [torch.arange(n, dtype=torch.float64, device="cuda")[:, None] / case["factor"]
              * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / max(d, 1))
              for n, d in zip(grid, dims)]
    F, h, w = grid
    a = torch.cat([angles[0][:, None, None].expand(F, h, w, -1), angles[1][None, :, None].expand(F, h, w, -1),
                   angles[2][None, None].expand(F, h, w, -1)], dim=-1).reshape(F * h * w, R // 2)
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "rope":
        S = case["text"] + case["frames"] * case["height"] * case["width"]
        shape = (case["B"], case["H"], S, case["D"])
        q, k = (_randn(g, shape, case["strided"]).to(dt) for _ in range(2))
        cos, sin = _table(case)
        return {"case": case, "q": q, "k": k, "cos": cos, "sin": sin}
    B, H, D, strided = case["B"], case["H"], case["D"], case["strided"]
    q = _field(case, _randn(g, (B, H, case["Sq"], D), strided), g).to(dt)
    k = _field(case, _randn(g, (B, H, case["Sk"], D), strided), g).to(dt)
    v = _randn(g, (B, H, case["Sk"], D), strided).to(dt)
    row_ptr, col_idx, live = _list(case, q, k)
    state = {"case": case, "q": q, "k": k, "v": v, "row_ptr": row_ptr, "col_idx": col_idx, "live": live,
             "scale": 1.0 / math.sqrt(D)}
    if case["op"] == "bwd":
        done = _plain_fwd(state)
        # the forward's output has the layout of q, as the framework's own has
        state["out"] = torch.empty_like(q).copy_(done["out"])
        state["lse"] = done["lse"]
        state["dout"] = _randn(g, (B, H, case["Sq"], D), strided).to(dt)
    return state


# --------------------------------------------------------------------------- plain forms

def _plain_rope(state):
    case, cos, sin = state["case"], state["cos"], state["sin"]
    R, t = case["R"], case["text"]
    sign = -1.0 if case["inverse"] else 1.0

    def turn(x):
        y = x.float()
        z = y[:, :, t:]
        if case["layout"] == "interleaved":
            a, b = z[..., 0:R:2], z[..., 1:R:2]
            r = torch.stack([a * cos - sign * (b * sin), b * cos + sign * (a * sin)], dim=-1).flatten(-2)
        else:
            a, b = z[..., :R // 2], z[..., R // 2:R]
            r = torch.cat([a * cos - sign * (b * sin), b * cos + sign * (a * sin)], dim=-1)
        z = torch.cat([r, z[..., R:]], dim=-1)
        return torch.cat([y[:, :, :t], z], dim=2).to(x.dtype)

    return {"q": turn(state["q"]), "k": turn(state["k"])}


def _pairs(state):
    """Row block and column block (both counted over all heads) of every listed block."""
    case, row_ptr = state["case"], state["row_ptr"].long()
    nbq, nbk = _blocks(case)[:2]
    n = (row_ptr[:, 1:] - row_ptr[:, :-1]).reshape(-1)
    rows = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=state["live"])
    within = torch.arange(state["live"], device="cuda") - (n.cumsum(0) - n)[rows]
    cols = state["col_idx"][row_ptr[:, :-1].reshape(-1)[rows] + within].long()
    return rows, cols, rows // nbq * nbk + cols


def _cut(x, b):
    """``[B, H, S, D]`` as blocks ``[B * H * n, b, D]`` in 32 bits, zeros past the end."""
    B, H, S, D = x.shape
    n = -(-S // b)
    return torch.nn.functional.pad(x.float(), (0, 0, 0, n * b - S)).reshape(B * H * n, b, D)


def _join(x, like):
    B, H, S, D = like.shape
    return x.reshape(B, H, -1, D)[:, :, :S].to(like.dtype)


def _scores(state, rows, cols, at):
    """Scaled products of every listed block, -inf past the last key."""
    case = state["case"]
    s = torch.bmm(_cut(state["q"], case["bm"])[rows], _cut(state["k"], case["bn"])[at].transpose(1, 2))
    s.mul_(state["scale"])
    past = cols[:, None] * case["bn"] + torch.arange(case["bn"], device="cuda") >= case["Sk"]
    return s.masked_fill_(past[:, None], -math.inf)


def _plain_fwd(state):
    case, q = state["case"], state["q"]
    B, H, Sq, D = q.shape
    rows, cols, at = _pairs(state)
    n = B * H * _blocks(case)[0]
    s = _scores(state, rows, cols, at)
    top = torch.full((n, case["bm"]), -math.inf, device="cuda").index_reduce_(0, rows, s.amax(-1), "amax")
    s.sub_(top[rows][..., None]).exp_()
    total = torch.zeros(n, case["bm"], device="cuda").index_add_(0, rows, s.sum(-1))
    o = torch.zeros(n, case["bm"], D, device="cuda").index_add_(
        0, rows, torch.bmm(s, _cut(state["v"], case["bn"])[at]))
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    return {"out": _join(o, q), "lse": (top + total.log()).reshape(B, H, -1)[:, :, :Sq]}


def _plain_bwd(state):
    case, q, k = state["case"], state["q"], state["k"]
    B, H, Sq, D = q.shape
    bm, bn = case["bm"], case["bn"]
    rows, cols, at = _pairs(state)
    nbq, nbk = _blocks(case)[:2]
    p = _scores(state, rows, cols, at)
    lse = torch.nn.functional.pad(state["lse"], (0, nbq * bm - Sq)).reshape(B * H * nbq, bm)
    p.sub_(lse[rows][..., None]).exp_()
    do = _cut(state["dout"], bm)
    delta = (do * _cut(state["out"], bm)).sum(-1)
    do = do[rows]
    dv = torch.zeros(B * H * nbk, bn, D, device="cuda").index_add_(0, at, torch.bmm(p.transpose(1, 2), do))
    ds = torch.bmm(do, _cut(state["v"], bn)[at].transpose(1, 2)).sub_(delta[rows][..., None]).mul_(p)
    del p, do
    ds.mul_(state["scale"])
    dq = torch.zeros(B * H * nbq, bm, D, device="cuda").index_add_(0, rows, torch.bmm(ds, _cut(k, bn)[at]))
    dk = torch.zeros(B * H * nbk, bn, D, device="cuda").index_add_(
        0, at, torch.bmm(ds.transpose(1, 2), _cut(q, bm)[rows]))
    return {"dq": _join(dq, q), "dk": _join(dk, k), "dv": _join(dv, k)}


# --------------------------------------------------------------------------- the framework's calls

def _own(state):
    from sparseattnfunctions_b200 import kernels

    case = state["case"]
    if case["op"] == "rope":
        q, k = kernels.rope(state["q"], state["k"], state["cos"], state["sin"], text_len=case["text"],
                            layout=case["layout"], inverse=case["inverse"])
        return {"q": q, "k": k}
    nbq, nbk, tq = _blocks(case)[:3]
    csr = kernels.BlockCSR(state["row_ptr"], state["col_idx"], case["B"], case["H"], nbq, nbk, case["bm"],
                           case["bn"], dense_rows=tq)
    if case["op"] == "fwd":
        out, lse = kernels.bsa_fwd_lse(state["q"], state["k"], state["v"], csr, state["scale"])
        return {"out": out, "lse": lse}
    dq, dk, dv = kernels.bsa_bwd(state["dout"], state["q"], state["k"], state["v"], state["out"], state["lse"],
                                 csr, state["scale"])
    return {"dq": dq, "dk": dk, "dv": dv}


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "fwd": _plain_fwd, "bwd": _plain_bwd}[state["case"]["op"]](state)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "rope":
        video = case["frames"] * case["height"] * case["width"]
        n = case["B"] * case["H"] * (case["text"] + video) * case["D"]
        return {"bytes": 4 * n * e + 4 * video * case["R"], "flops": 6 * case["B"] * case["H"] * video * case["R"]}
    nbq, nbk, tq, tk, top = _blocks(case)
    every = case["empty"]
    gone = nbq // every if every else 0
    gone_text = tq // every if every else 0
    share = ((tq - gone_text) * nbk + (nbq - tq - gone + gone_text) * (tk + top)) / (nbq * nbk)
    heads = case["B"] * case["H"]
    pairs = heads * share * case["Sq"] * case["Sk"]
    nq, nk = heads * case["Sq"] * case["D"], heads * case["Sk"] * case["D"]
    if case["op"] == "fwd":
        return {"bytes": (2 * nq + 2 * nk) * e + 4 * heads * case["Sq"], "flops": 4 * case["D"] * pairs}
    return {"bytes": (4 * nq + 4 * nk) * e + 4 * heads * case["Sq"], "flops": 10 * case["D"] * pairs}


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions, head by head over whole rows with a token mask."""
    state = prepare(case, seed)
    q, k = state["q"].double(), state["k"].double()
    if case["op"] == "rope":
        R, t = case["R"], case["text"]
        turn = torch.complex(state["cos"].double(), state["sin"].double())
        turn = turn.conj() if case["inverse"] else turn
        got = {}
        for name, x in (("q", q), ("k", k)):
            y, z = x.clone(), x[:, :, t:, :R]
            if case["layout"] == "interleaved":
                r = torch.complex(z[..., 0::2], z[..., 1::2]) * turn
                y[:, :, t:, 0:R:2], y[:, :, t:, 1:R:2] = r.real, r.imag
            else:
                r = torch.complex(z[..., :R // 2], z[..., R // 2:]) * turn
                y[:, :, t:, :R // 2], y[:, :, t:, R // 2:R] = r.real, r.imag
            got[name] = y
        return got
    v = state["v"].double()
    B, H, Sq, D = q.shape
    Sk, nbq, nbk = k.shape[2], *_blocks(case)[:2]
    ptr, col = state["row_ptr"].cpu().tolist(), state["col_idx"].cpu()
    got = {"out": torch.zeros_like(q), "lse": torch.full((B, H, Sq), -math.inf, dtype=torch.float64, device="cuda")}
    if case["op"] == "bwd":
        got = {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    for b in range(B):
        for h in range(H):
            p = ptr[b * H + h]
            mask = torch.zeros(nbq, nbk, dtype=torch.bool)
            for i in range(nbq):
                mask[i, col[p[i]:p[i + 1]].long()] = True
            mask = mask.cuda().repeat_interleave(case["bm"], 0).repeat_interleave(case["bn"], 1)[:Sq, :Sk]
            for r in range(0, Sq, 8192):  # in strips of rows: the long geometries
                rows = slice(r, min(Sq, r + 8192))
                s = (q[b, h, rows] @ k[b, h].T * state["scale"]).masked_fill_(~mask[rows], -math.inf)
                if case["op"] == "fwd":
                    seen = mask[rows].any(-1)
                    got["lse"][b, h, rows] = torch.logsumexp(s, -1)
                    got["out"][b, h, rows][seen] = torch.softmax(s[seen], -1) @ v[b, h]
                    continue
                lse = state["lse"][b, h, rows].double()
                a = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[:, None])
                do = state["dout"][b, h, rows].double()
                delta = (do * state["out"][b, h, rows].double()).sum(-1, keepdim=True)
                got["dv"][b, h] += a.T @ do
                ds = a * (do @ v[b, h].T - delta) * state["scale"]
                got["dq"][b, h, rows] = ds @ k[b, h]
                got["dk"][b, h] += ds.T @ q[b, h, rows]
    return got
