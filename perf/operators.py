"""Timed cases of the expert-dispatch and MXFP4-product operators.

Five passes, as a mixture-of-experts layer with packed 4-bit weights makes them:

  dispatch  the pairs of a routing sorted by expert (moe_sort) and every pair's token row copied
            into expert order (moe_permute); with `grad` also the tokens' gradient
            (moe_permute_bwd)
  combine   each token's rows summed with its routing weights (moe_unpermute); with `grad` also
            the gradients of the rows and of the weights (moe_unpermute_bwd)
  linear    activations quantised to MXFP4 (mxfp4_quant) and multiplied with one packed matrix
            (mxfp4_mm)
  experts   sort, token rows quantised straight into expert order (moe_permute_mxfp4), and the
            product of each expert's rows with its own packed matrix (mxfp4_mm with offsets)
  dgrad     the gradient of that product with respect to its activations (mxfp4_mm_bwd)

Packed weights are in the layout mxfp4_pack makes: E2M1 codes [matrix][row][in/2] (low nibble =
even element) and E8M0 scales in 512-byte atoms of 128 rows x 4 groups of 32 elements, the scale
of row r (of the atom's 128) and group g at byte 16*(r % 32) + 4*(r / 32) + g.
"""
import math

import torch

own = False

HIDDEN, INTER, TOPK, EXPERTS = 7168, 2048, 8, 384
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # a decode batch of 16 requests through the full expert set: pure latency
        dict(name="dispatch_decode", op="dispatch", T=16, k=TOPK, ids=EXPERTS, E=EXPERTS, H=HIDDEN, dtype="bf16",
             grad=False),
        # one expert-parallel rank: 48 of 384 experts are held here, the other pairs go elsewhere;
        # an odd width in fp32, forward and backward
        dict(name="dispatch_shard", op="dispatch", T=777, k=TOPK, ids=EXPERTS, E=48, H=1003, dtype="f32", grad=True),
        # a training micro-batch: bandwidth
        dict(name="dispatch_train", op="dispatch", T=4096, k=TOPK, ids=EXPERTS, E=EXPERTS, H=HIDDEN, dtype="bf16",
             grad=True),
        # the same three steps of a layer's way back
        dict(name="combine_decode", op="combine", T=16, k=TOPK, ids=EXPERTS, E=EXPERTS, H=HIDDEN, dtype="bf16",
             grad=False),
        dict(name="combine_train", op="combine", T=4096, k=TOPK, ids=EXPERTS, E=EXPERTS, H=HIDDEN, dtype="bf16",
             grad=True),
        # one token through a square projection: the weights' bytes
        dict(name="linear_token", op="linear", M=1, N=HIDDEN, K=HIDDEN, dtype="bf16", out="bf16"),
        # a prompt's ragged last chunk, fp32 in and out, sides that fill no tile
        dict(name="linear_chunk", op="linear", M=333, N=2080, K=3616, dtype="f32", out="f32"),
        # a long prompt: the tensor cores
        dict(name="linear_prompt", op="linear", M=8192, N=HIDDEN, K=HIDDEN, dtype="bf16", out="bf16"),
        # 16 requests through the gate/up matrices of 64 experts, two rows or so each
        dict(name="experts_decode", op="experts", T=16, k=TOPK, E=64, N=2 * INTER, K=HIDDEN, dtype="bf16", out="bf16"),
        # a prompt through the gate/up matrices of the 48 experts that a rank holds
        dict(name="experts_prompt", op="experts", T=4096, k=TOPK, E=48, N=2 * INTER, K=HIDDEN, dtype="bf16",
             out="bf16"),
        # a short sequence's gradient through narrow experts
        dict(name="dgrad_ragged", op="dgrad", T=300, k=TOPK, E=48, N=1432, K=992, out="f32"),
        # a micro-batch's gradient through the down matrices
        dict(name="dgrad_train", op="dgrad", T=4096, k=TOPK, E=48, N=HIDDEN, K=INTER, out="bf16"),
    ]


def draw(rng):
    def log(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(step, int(round(v / step)) * step)

    op = rng.choice(["dispatch", "combine", "linear", "experts", "dgrad"])
    if op in ("dispatch", "combine"):
        ids = log(8, EXPERTS)
        k = rng.choice([1, 2, 4, 6, 8])
        dtype = rng.choice(["bf16", "f32"])
        H = log(64, HIDDEN if dtype == "bf16" else HIDDEN // 2, rng.choice([1, 8, 64]))
        return dict(op=op, T=log(1, 4096), k=k, ids=ids, E=rng.choice([ids, max(1, ids // 4)]), H=H, dtype=dtype,
                    grad=rng.random() < 0.5)
    if op == "linear":
        return dict(op=op, M=log(1, 8192), N=log(64, HIDDEN, rng.choice([1, 16, 128])), K=log(64, HIDDEN, 32),
                    dtype=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
    k = rng.choice([1, 2, 4, 8])
    E = max(k, log(2, 48))
    T = log(1, 4096 * 8 // k if op == "experts" else 2048)
    T = min(T, 4096)
    if op == "experts":
        return dict(op=op, T=T, k=k, E=E, N=log(64, 2 * INTER, rng.choice([1, 16, 128])), K=log(64, HIDDEN, 32),
                    dtype=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
    return dict(op=op, T=T, k=k, E=E, N=log(64, HIDDEN, 8), K=log(64, INTER, 32), out=rng.choice(["bf16", "f32"]))


# ------------------------------------------------------------------------------ inputs
def routing(g, T, k, ids):
    """Top-k ids of scores with popular and rare experts, and renormalised weights."""
    s = torch.randn(T, ids, generator=g, device="cuda") + torch.linspace(0.8, -0.8, ids, device="cuda")
    top = torch.sigmoid(s).topk(k, dim=1)
    return top.indices.to(torch.int32), top.values / top.values.sum(1, keepdim=True)


def offsets(idx, E):
    """(off [E+1], pos [T][k]) of a routing, with ids >= E dropped."""
    flat = idx.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = key.argsort(stable=True)
    count = torch.bincount(key, minlength=E + 1)
    off = torch.zeros(E + 1, dtype=torch.int32, device=idx.device)
    off[1:] = count[:E].cumsum(0)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=idx.device)
    pos = torch.where(key < E, pos, -1).to(torch.int32).reshape(idx.shape)
    return off, pos, int(count[:E].max())


def weights(g, E, N, K):
    """Packed matrices: uniform codes, scale bytes 118..124, as 4-bit checkpoints carry."""
    codes = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, generator=g, device="cuda")
    Np, Kp = -(-N // 128) * 128, -(-K // 128) * 128
    rows = torch.full((E, Np, Kp // 32), 127, dtype=torch.uint8, device="cuda")
    rows[:, :N, :K // 32] = torch.randint(118, 125, (E, N, K // 32), dtype=torch.uint8, generator=g, device="cuda")
    atoms = rows.view(E, Np // 128, 4, 32, Kp // 128, 4).permute(0, 1, 4, 3, 2, 5).contiguous()
    return codes, atoms.view(E, Np // 128, Kp // 128, 512)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def randn(*shape, dtype):
        return torch.randn(*shape, generator=g, device="cuda").to(DTYPES[dtype])

    s = {"case": dict(case)}
    if op == "dispatch":
        T, k, H, dt = case["T"], case["k"], case["H"], case["dtype"]
        s["idx"], _ = routing(g, T, k, case["ids"])
        s["x"] = randn(T, H, dtype=dt)
        s["drows"] = randn(T * k, H, dtype=dt) if case["grad"] else None
        s["rows"] = torch.zeros(T * k, H, dtype=DTYPES[dt], device="cuda")   # rows past the last stay zero
    elif op == "combine":
        T, k, H, dt = case["T"], case["k"], case["H"], case["dtype"]
        idx, s["wt"] = routing(g, T, k, case["ids"])
        _, s["pos"], _ = offsets(idx, case["E"])
        s["y"] = randn(T * k, H, dtype=dt)
        s["dout"] = randn(T, H, dtype=dt) if case["grad"] else None
        s["dy"] = torch.zeros(T * k, H, dtype=DTYPES[dt], device="cuda") if case["grad"] else None
    elif op == "linear":
        s["x"] = randn(case["M"], case["K"], dtype=case["dtype"])
        s["codes"], s["atoms"] = weights(g, 1, case["N"], case["K"])
    else:
        T, k, E = case["T"], case["k"], case["E"]
        s["idx"], _ = routing(g, T, k, E)
        s["off"], s["pos"], s["cap"] = offsets(s["idx"], E)
        if op == "experts":
            s["x"] = randn(T, case["K"], dtype=case["dtype"])
        else:
            s["dy"] = randn(T * k, case["N"], dtype="bf16")
        s["codes"], s["atoms"] = weights(g, E, case["N"], case["K"])
    return s


# ------------------------------------------------------------------------------ the plain form
def plain_sort(idx, E):
    flat = idx.reshape(-1).long()
    P = flat.numel()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = key.argsort(stable=True)
    off = torch.searchsorted(key[order], torch.arange(E + 1, device=idx.device)).to(torch.int32)
    r = torch.arange(P, device=idx.device)
    pos = torch.empty_like(order)
    pos[order] = r
    pos = torch.where(key < E, pos, -1).to(torch.int32).reshape(idx.shape)
    pair = torch.where(r < off[E], order, -1).to(torch.int32)
    return pos, pair, off


def plain_quant(x):
    """The values that x, quantised to MXFP4, stands for (fp32): per 32 elements the power of two
    floor(log2 max|x|) - 2, elements to the nearest of 0 .5 1 1.5 2 3 4 6, ties to the even code."""
    v = x.float().reshape(x.shape[0], -1, 32)
    e = (torch.frexp(v.abs().amax(-1, keepdim=True)).exponent - 3).clamp(-127, 127)
    a = torch.ldexp(v.abs(), -e)
    q = (0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75) + 1.0 * (a > 2.5)
         + 1.0 * (a >= 3.5) + 2.0 * (a > 5.0))
    return torch.ldexp(torch.copysign(q, v), e).reshape(x.shape)


def plain_weights(codes, atoms):
    """[E][N][K] fp32 values of packed matrices."""
    E, N, K2 = codes.shape
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(-1).int()
    v = table.index_select(0, c).view(E, N, -1, 32)
    sc = atoms.view(E, atoms.shape[1], atoms.shape[2], 32, 4, 4).permute(0, 1, 4, 3, 2, 5)
    sc = sc.reshape(E, atoms.shape[1] * 128, -1)[:, :N, :K2 // 16].float() - 127
    v.mul_(torch.exp2(sc).unsqueeze(-1))
    return v.view(E, N, 2 * K2)


def plain(s):
    c = s["case"]
    op = c["op"]
    if op == "dispatch":
        pos, pair, off = plain_sort(s["idx"], c["E"])
        live = (pair >= 0).unsqueeze(1)
        rows = s["x"].index_select(0, pair.clamp(min=0) // c["k"]) * live
        got = {"pos": pos, "pair": pair, "off": off, "rows": rows}
        if c["grad"]:
            d = s["drows"][pos.clamp(min=0).long()].float() * (pos >= 0).unsqueeze(-1)
            got["dx"] = d.sum(1).to(s["x"].dtype)
        return got
    if op == "combine":
        pos, dt = s["pos"], s["y"].dtype
        live = (pos >= 0).unsqueeze(-1)
        at = pos.clamp(min=0).long()
        y = s["y"][at].float() * live
        got = {"out": (y * s["wt"].unsqueeze(-1)).sum(1).to(dt)}
        if c["grad"]:
            do = s["dout"].float().unsqueeze(1)
            got["dwt"] = (y * do).sum(-1)
            dy = torch.zeros(y.shape[0] * y.shape[1] + 1, y.shape[2], dtype=dt, device=y.device)
            put = torch.where(pos >= 0, pos, dy.shape[0] - 1).long().reshape(-1)
            dy[put] = (s["wt"].unsqueeze(-1) * do).to(dt).view(-1, y.shape[2])
            got["dy"] = dy[:-1]
        return got
    W = plain_weights(s["codes"], s["atoms"])
    out = DTYPES[c["out"]]
    if op == "linear":
        return {"y": (plain_quant(s["x"]) @ W[0].T).to(out)}
    idx = s["idx"].long()
    if op == "experts":
        pos, _, off = plain_sort(s["idx"], c["E"])
        slot = (pos - off[idx]).long()
        a = torch.zeros(c["E"], s["cap"], c["K"], device=W.device)
        a[idx, slot] = plain_quant(s["x"]).unsqueeze(1).expand(-1, c["k"], -1)
        y = torch.empty(pos.numel(), c["N"], dtype=out, device=W.device)
        y[pos.long().view(-1)] = torch.bmm(a, W.transpose(1, 2))[idx, slot].view(-1, c["N"]).to(out)
        return {"y": y, "pos": pos, "off": off}
    slot = (s["pos"] - s["off"][idx]).long()
    at = s["pos"].long()
    a = torch.zeros(c["E"], s["cap"], c["N"], device=W.device)
    a[idx, slot] = s["dy"][at].float()
    da = torch.empty(at.numel(), c["K"], dtype=out, device=W.device)
    da[at.view(-1)] = torch.bmm(a, W)[idx, slot].view(-1, c["K"]).to(out)
    return {"da": da}


# ------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return framework(s)
    return plain(s)


def framework(s):
    from __graft_entry__ import load_package
    k3 = load_package()
    c = s["case"]
    op = c["op"]
    if op == "dispatch":
        pos, pair, off = k3.moe_sort(s["idx"], c["E"])
        got = {"pos": pos, "pair": pair, "off": off, "rows": k3.moe_permute(s["x"], pos, out=s["rows"])}
        if c["grad"]:
            got["dx"] = k3.moe_permute_bwd(s["drows"], pos)
        return got
    if op == "combine":
        got = {"out": k3.moe_unpermute(s["y"], s["pos"], s["wt"])}
        if c["grad"]:
            got["dy"], got["dwt"] = k3.moe_unpermute_bwd(s["dout"], s["y"], s["pos"], s["wt"], dy=s["dy"])
        return got
    if op == "linear":
        a, sa = k3.mxfp4_quant(s["x"])
        return {"y": k3.mxfp4_mm(a, sa, k3.Mxfp4Mat(s["codes"], s["atoms"]), out_dtype=DTYPES[c["out"]])}
    W = k3.Mxfp4Mat(s["codes"], s["atoms"])
    if op == "experts":
        pos, _, off = k3.moe_sort(s["idx"], c["E"])
        a, sa = k3.moe_permute_mxfp4(s["x"], pos)
        return {"y": k3.mxfp4_mm(a, sa, W, off=off, out_dtype=DTYPES[c["out"]]), "pos": pos, "off": off}
    return {"da": k3.mxfp4_mm_bwd(s["dy"], W, off=s["off"], out_dtype=DTYPES[c["out"]])}


# ------------------------------------------------------------------------------ what a pass needs
def work(case):
    op = case["op"]
    if op in ("dispatch", "combine"):
        T, k, H, b = case["T"], case["k"], case["H"], BYTES[case["dtype"]]
        P = T * k
        n = P * case["E"] / case["ids"]   # pairs whose expert is held
        nbytes = (T + n) * H * b
        if op == "dispatch":
            nbytes += 4 * (3 * P + case["E"] + 1)
            flops = 0
            if case["grad"]:
                nbytes += (T + n) * H * b
                flops = n * H
        else:
            nbytes += 8 * P
            flops = 2 * n * H
            if case["grad"]:
                nbytes += (T + n) * H * b + 4 * P   # y and the routing are the forward's
                flops += 3 * n * H
        return {"bytes": nbytes, "flops": flops}
    N, K = case["N"], case["K"]
    mat = N * K * 17 / 32
    if op == "linear":
        M = case["M"]
        return {"bytes": M * K * BYTES[case["dtype"]] + mat + M * N * BYTES[case["out"]], "flops": 2 * M * N * K}
    T, k, E = case["T"], case["k"], case["E"]
    P = T * k
    met = E * (1 - (1 - k / E) ** T)   # experts that some token chose
    if op == "experts":
        nbytes = T * K * BYTES[case["dtype"]] + met * mat + P * N * BYTES[case["out"]] + 8 * P + 4 * E
    else:
        nbytes = P * N * 2 + met * mat + P * K * BYTES[case["out"]] + 4 * E
    return {"bytes": nbytes, "flops": 2 * P * N * K}


# ------------------------------------------------------------------------------ 64 bits
def exact_quant(x):
    """MXFP4 values from the definition: the step of an element's binade, half to even."""
    v = x.double().reshape(x.shape[0], -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -126))) - 2).clamp(min=2.0 ** -127)
    a = v.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(v) * (torch.round(a / step) * step).clamp(max=6) * unit).reshape(x.shape)


def exact_matrix(codes, atoms):
    """[N][K] in 64 bits: each element from its nibble's fields and its own scale byte."""
    N, K2 = codes.shape
    n = torch.arange(N, device=codes.device).unsqueeze(1)
    i = torch.arange(2 * K2, device=codes.device).unsqueeze(0)
    nib = (codes.long().repeat_interleave(2, dim=1) >> (4 * (i % 2))) & 15
    ex, m = (nib >> 1) & 3, (nib & 1).double()
    mag = torch.where(ex == 0, 0.5 * m, torch.exp2(ex.double() - 1) * (1 + 0.5 * m))
    g = torch.arange(K2 // 16, device=codes.device).unsqueeze(0)
    byte = atoms[n // 128, g // 4, 16 * (n % 32) + 4 * (n % 128 // 32) + g % 4]
    sc = torch.exp2(byte.double() - 127).repeat_interleave(32, dim=1)
    return torch.where(nib >= 8, -mag, mag) * sc


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "dispatch":
        idx, E, k = s["idx"].cpu().reshape(-1).tolist(), case["E"], case["k"]
        lists = [[] for _ in range(E)]
        for p, e in enumerate(idx):
            if 0 <= e < E:
                lists[e].append(p)
        order = [p for ps in lists for p in ps]
        off = torch.tensor([0] + [len(ps) for ps in lists], dtype=torch.int32).cumsum(0).int()
        n = len(order)
        r = torch.tensor(order, dtype=torch.int64, device="cuda")
        pos = torch.full((len(idx),), -1, dtype=torch.int32, device="cuda")
        pos[r] = torch.arange(n, dtype=torch.int32, device="cuda")
        pair = torch.full((len(idx),), -1, dtype=torch.int32, device="cuda")
        pair[:n] = r.int()
        rows = torch.zeros(len(idx), case["H"], dtype=torch.float64, device="cuda")
        rows[:n] = s["x"][r // k].double()
        got = {"pos": pos.view(-1, k), "pair": pair, "off": off.cuda(), "rows": rows}
        if case["grad"]:
            got["dx"] = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
            got["dx"].index_add_(0, r // k, s["drows"][:n].double())
        return got
    if op == "combine":
        T, k, H = case["T"], case["k"], case["H"]
        pos = s["pos"].long().view(-1)
        p = torch.nonzero(pos >= 0).view(-1)
        r, t = pos[p], p // k
        w = s["wt"].double().view(-1)[p].unsqueeze(1)
        out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        out.index_add_(0, t, w * s["y"][r].double())
        got = {"out": out}
        if case["grad"]:
            do = s["dout"][t].double()
            got["dy"] = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
            got["dy"][r] = w * do
            dwt = torch.zeros(T * k, dtype=torch.float64, device="cuda")
            dwt[p] = (do * s["y"][r].double()).sum(1)
            got["dwt"] = dwt.view(T, k)
        return got
    if op == "linear":
        return {"y": exact_quant(s["x"]) @ exact_matrix(s["codes"][0], s["atoms"][0]).T}
    off, idx = s["off"].tolist(), s["idx"].reshape(-1).long()
    name, width = ("y", case["N"]) if op == "experts" else ("da", case["K"])
    res = torch.zeros(idx.numel(), width, dtype=torch.float64, device="cuda")
    x = exact_quant(s["x"]) if op == "experts" else None
    for e in range(case["E"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        W = exact_matrix(s["codes"][e], s["atoms"][e])
        if op == "experts":
            tokens = torch.nonzero(idx == e).view(-1) // case["k"]
            res[lo:hi] = x[tokens] @ W.T
        else:
            res[lo:hi] = s["dy"][lo:hi].double() @ W
    return {"y": res, "pos": s["pos"], "off": s["off"]} if op == "experts" else {"da": res}
