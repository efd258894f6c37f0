"""MXFP4 quantisation (k3c_mxfp4_quant), packing and the products k3c_mxfp4_mm and
k3c_mxfp4_mm_bwd against plain 64-bit arithmetic on the same codes.

Tolerances. Quantisation and packing are exact. In the products every term is exact in fp32 (E2M1
x E2M1 under powers of two; bf16 x E2M1 under a power of two). A 64-wide (mm) or 16-wide (mm_bwd)
step adds its terms to the accumulator with at most one unit (2^-23, a truncation) of the running
magnitude, which sum|terms| bounds; 8 more units stand for the additions within steps. Rounding
to bf16 adds 2^-8 of the result, to fp32 nothing."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


@pytest.fixture(scope="module")
def dev():
    import torch
    return torch.device("cuda:0")


def quant_plain(v):
    """v [rows][in] float64 (finite or not, no NaN) -> (codes 0..15 [rows][in], scale bytes): the
    nearest grid value by distance, the even code on ties."""
    rows, n = v.shape
    G = -(-n // 32)
    pad = np.zeros((rows, G * 32))
    pad[:, :n] = v
    g = pad.reshape(rows, G, 32)
    top = np.abs(g).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(np.isinf(top), 128, np.floor(np.log2(np.where(np.isinf(top), 1, top))))
    byte = np.clip(np.where(top == 0, -1000, e) - 2 + 127, 0, 254)
    a = np.minimum(np.abs(g) / 2.0 ** (byte - 127)[..., None], 6.0)
    d = np.abs(a[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    near = d == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code + 8 * np.signbit(g)
    return code.reshape(rows, -1)[:, :n].astype(np.uint8), byte.astype(np.uint8)


def values(codes, byte):
    """float64 values of codes [rows][in] (0..15) under scale bytes [rows][in/32 rounded up]."""
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    sc = 2.0 ** (byte.astype(np.float64) - 127)
    return v * np.repeat(sc, 32, axis=1)[:, :codes.shape[1]]


def pack_nibbles(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n,pad", [(1, 2, 0), (1, 32, 0), (3, 34, 0), (5, 96, 1), (7, 1000, 24), (64, 7168, 0),
                                        (513, 352, 32)])
def test_quant(k3, dev, rows, n, pad, dtype):
    import torch
    g = np.random.default_rng(rows + n)
    x = g.standard_normal((rows, n + pad)) * 2.0 ** g.integers(-140, 120, (rows, 1))
    x[:, ::7] = g.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0, 0.0, -0.0], x[:, ::7].shape)   # ties
    x[0, :] = 0
    t = torch.from_numpy(x).float()
    t = t.bfloat16() if dtype == "bf16" else t
    packed, scales = k3.mxfp4_quant(t.to(dev)[:, :n])
    codes, byte = quant_plain(t.double().numpy()[:, :n])
    assert np.array_equal(scales.cpu().numpy(), byte)
    assert np.array_equal(unpack(packed.cpu().numpy())[:, :n], codes)


def test_quant_borders_of_the_range(k3, dev):
    """Subnormal groups, the largest finite value, infinities (read back as infinities) and NaN
    (scale byte 255, zero codes)."""
    import torch
    x = torch.zeros(7, 32)
    x[0, 3] = 2.0 ** -149
    x[1, :] = 2.0 ** -127
    x[2, 5], x[2, 6] = torch.finfo(torch.float32).max, 1.0
    x[3, 0], x[3, 1], x[3, 2] = float("inf"), -float("inf"), 3.0
    x[4, 31], x[4, 0] = float("nan"), 5.0
    x[5, :] = torch.linspace(-1.9e-38, 1.9e-38, 32)
    x[6, 0], x[6, 1] = 2.0 ** -125, -2.0 ** -127
    packed, scales = k3.mxfp4_quant(x.to(dev))
    ok = [0, 1, 2, 3, 5, 6]
    codes, byte = quant_plain(x.double().numpy()[ok])
    assert np.array_equal(scales.cpu().numpy()[ok], byte)
    assert np.array_equal(unpack(packed.cpu().numpy())[ok], codes)
    assert scales[4, 0] == 255 and (packed[4] == 0).all()
    back = k3.mxfp4_dequant(packed, scales).cpu()
    assert back[3, 0] == float("inf") and back[3, 1] == -float("inf") and torch.isfinite(back[2, 6])


@pytest.mark.parametrize("n,rows,in_", [(1, 1, 32), (3, 130, 96), (2, 256, 4128)])
def test_pack(k3, dev, n, rows, in_):
    import torch
    g = np.random.default_rng(in_)
    p = g.integers(0, 256, (n, rows, in_ // 2), dtype=np.uint8)
    s = g.integers(0, 256, (n, rows, in_ // 32), dtype=np.uint8)
    s[:, ::3, 0] = 255
    codes, atoms = (t.cpu().numpy() for t in k3.mxfp4_pack(torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev)))
    want = np.full_like(atoms, 127)
    for r in range(rows):
        for q in range(in_ // 32):
            b = s[:, r, q]
            want[:, r // 128, q // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + q % 4] = np.where(b == 255, 127, b)
    assert np.array_equal(atoms, want)
    skip = np.repeat(s == 255, 16, axis=2)
    assert np.array_equal(codes, np.where(skip, 0, p))


def operand(seed, rows, in_, lo=116, hi=132):
    g = np.random.default_rng(seed)
    codes = g.integers(0, 16, (rows, in_), dtype=np.uint8)
    byte = g.integers(lo, hi, (rows, in_ // 32), dtype=np.uint8)
    return codes, byte


def to_dev(dev, *arrays):
    import torch
    return [torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays]


def check(got, want, mag, steps, bf16):
    lim = (steps + 8) * 2.0 ** -23 * mag + (2.0 ** -8 * np.abs(want) if bf16 else 0)
    bad = np.abs(got - want) > lim
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / np.maximum(lim, 1e-300)).max()))


def matrices(k3, dev, seed, n, rows, in_):
    """n packed matrices: (Mxfp4Mat, float64 values [n][rows][in])."""
    cs, bs, vs = [], [], []
    for i in range(n):
        c, b = operand(seed + i, rows, in_)
        cs.append(pack_nibbles(c))
        bs.append(b)
        vs.append(values(c, b))
    return k3.Mxfp4Mat(*k3.mxfp4_pack(*to_dev(dev, np.stack(cs), np.stack(bs)))), np.stack(vs)


DENSE = [(1, 1, 32), (1, 64, 64), (2, 65, 96), (1, 7168, 2048), (31, 130, 160), (33, 200, 256), (127, 384, 288),
         (128, 128, 512), (129, 257, 1056), (300, 1000, 3616), (64, 7168, 7168), (1000, 640, 352), (2200, 4100, 64),
         (2100, 2304, 1056), (256, 19000, 256), (900, 4100, 4128), (4300, 4100, 1312),
         (300, 4100, 1056), (5000, 4100, 2080)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", DENSE)
def test_mm(k3, dev, M, N, K, out):
    import torch
    W, w = matrices(k3, dev, 5, 1, N, K)
    c, b = operand(6, M, K)
    a, s = to_dev(dev, pack_nibbles(c), b)
    y = k3.mxfp4_mm(a, s, W, out_dtype=torch.float32 if out == "f32" else torch.bfloat16)
    av = torch.from_numpy(values(c, b)).to(dev)
    wv = torch.from_numpy(w[0]).to(dev)
    check(y.double().cpu().numpy(), (av @ wv.T).cpu().numpy(), (av.abs() @ wv.abs().T).cpu().numpy(), -(-K // 64),
          out == "bf16")
    assert torch.equal(y, k3.mxfp4_mm(a, s, W, out_dtype=y.dtype))      # the same bits again


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [m for m in DENSE if m[1] % 8 == 0]
                         + [(4000, 72, 2592), (128, 200, 60000), (300, 136, 19232), (2200, 4096, 64), (2700, 4096, 1824)])
def test_mm_bwd(k3, dev, M, N, K, out):
    import torch
    W, w = matrices(k3, dev, 7, 1, N, K)
    g = torch.Generator().manual_seed(M + N)
    dy = torch.randn((M, N), generator=g).bfloat16().to(dev)
    da = k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32 if out == "f32" else torch.bfloat16)
    wv = torch.from_numpy(w[0]).to(dev)
    check(da.double().cpu().numpy(), (dy.double() @ wv).cpu().numpy(), (dy.double().abs() @ wv.abs()).cpu().numpy(),
          -(-N // 16), out == "bf16")
    assert torch.equal(da, k3.mxfp4_mm_bwd(dy, W, out_dtype=da.dtype))


# rows per group: empty groups at both ends and in the middle, groups that end inside a tile, one
# row, several tiles
GROUPS = [[0], [1], [0, 0, 5, 0], [1] * 9, [130, 0, 1, 257, 32], [0, 40, 33, 128, 129, 1, 0, 300, 0], [2300, 1]]
# and sizes that reach every tile shape of both products
SHAPES = [(g, N, K) for g in GROUPS for N, K in ((64, 32), (200, 416), (520, 1056))] + [
    ([700, 0, 900, 1300] + [300] * 30, 1304, 1312), ([1000, 0] + [1000] * 7, 2104, 1312), ([9] * 100, 200, 2080),
    ([100] * 100, 72, 1056), ([1400, 1, 0, 1290], 4104, 1824)]


@pytest.mark.parametrize("sizes,N,K", SHAPES, ids=lambda v: "-".join(map(str, v[:8])) if isinstance(v, list) else str(v))
def test_grouped_products(k3, dev, sizes, N, K):
    """Both products over ragged groups; rows behind the last group stay as they were."""
    import torch
    G, n = len(sizes), sum(sizes)
    M = n + 3
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    W, w = matrices(k3, dev, 11, G, N, K)
    c, b = operand(12, M, K)
    a, s, po = to_dev(dev, pack_nibbles(c), b, off)
    y = torch.full((M, N), 7.0, device=dev)
    k3.mxfp4_mm(a, s, W, off=po, out=y)
    g = torch.Generator().manual_seed(N)
    dy = torch.randn((M, N), generator=g).bfloat16().to(dev)
    da = torch.full((M, K), 7.0, device=dev)
    k3.mxfp4_mm_bwd(dy, W, off=po, out=da)
    assert (y[n:] == 7).all() and (da[n:] == 7).all()
    av, dv = values(c, b), dy.double().cpu().numpy()
    for e in range(G):
        r = slice(off[e], off[e + 1])
        check(y[r].double().cpu().numpy(), av[r] @ w[e].T, np.abs(av[r]) @ np.abs(w[e]).T, -(-K // 64), False)
        check(da[r].double().cpu().numpy(), dv[r] @ w[e], np.abs(dv[r]) @ np.abs(w[e]), -(-N // 16), False)


def test_matrix_map_and_strided_rows(k3, dev):
    """mat_of picks each group's matrix, an index without one gives zeros; out and dy rows may be
    strided, with an odd stride or base (element stores) or an even one; columns beside them stay."""
    import torch
    N, K, M = 72, 96, 50
    W, w = matrices(k3, dev, 21, 3, N, K)
    mat_of = [2, -1, 0, 0, 3]
    off = [0, 20, 30, 30, 45, 50]
    W = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=torch.tensor(mat_of, dtype=torch.int32, device=dev))
    assert W.groups == 5
    c, b = operand(22, M, K)
    a, s = to_dev(dev, pack_nibbles(c), b)
    po = torch.tensor(off, dtype=torch.int32, device=dev)
    dyb = torch.randn((M, N + 24), device=dev).bfloat16()
    dy = dyb[:, 8:8 + N]
    av, dv = values(c, b), dy.double().cpu().numpy()
    for pad, dt in ((0, torch.float32), (5, torch.float32), (8, torch.float32), (3, torch.bfloat16), (8, torch.bfloat16)):
        yb = torch.full((M, N + 2 * pad), 7.0, dtype=dt, device=dev)
        db = torch.full((M, K + 2 * pad), 7.0, dtype=dt, device=dev)
        k3.mxfp4_mm(a, s, W, off=po, out=yb[:, pad:pad + N])
        k3.mxfp4_mm_bwd(dy, W, off=po, out=db[:, pad:pad + K])
        assert (yb[:, :pad] == 7).all() and (yb[:, pad + N:] == 7).all()
        assert (db[:, :pad] == 7).all() and (db[:, pad + K:] == 7).all()
        y, d = yb[:, pad:pad + N].double().cpu().numpy(), db[:, pad:pad + K].double().cpu().numpy()
        for g, m in enumerate(mat_of):
            r = slice(off[g], off[g + 1])
            if not 0 <= m < 3:
                assert (y[r] == 0).all() and (d[r] == 0).all()
                continue
            check(y[r], av[r] @ w[m].T, np.abs(av[r]) @ np.abs(w[m]).T, 2, dt == torch.bfloat16)
            check(d[r], dv[r] @ w[m], np.abs(dv[r]) @ np.abs(w[m]), 5, dt == torch.bfloat16)


def test_offsets_outside_the_rows_are_clamped(k3, dev):
    """Bad offsets (negative, descending, past the rows) touch nothing outside the result."""
    import torch
    N, K, M = 64, 64, 40
    W, w = matrices(k3, dev, 31, 4, N, K)
    c, b = operand(32, M, K)
    a, s = to_dev(dev, pack_nibbles(c), b)
    buf = torch.full((M + 2, N), 7.0, device=dev)
    off = torch.tensor([-5, 10, 4, 30, 10 ** 9], dtype=torch.int32, device=dev)
    k3.mxfp4_mm(a, s, W, off=off, out=buf[1:M + 1])
    assert (buf[0] == 7).all() and (buf[M + 1] == 7).all()
    got, av = buf[1:M + 1].double().cpu().numpy(), values(c, b)
    for r, e in ((slice(0, 4), 0), (slice(30, M), 3)):   # scales span 30 binades: not exact in fp32
        check(got[r], av[r] @ w[e].T, np.abs(av[r]) @ np.abs(w[e]).T, 1, False)


def test_nan_scale_makes_its_row_nan(k3, dev):
    """An activation group with scale 255 (the format's NaN) makes its row NaN and no other row;
    infinities pass through as the reference's arithmetic has them."""
    import torch
    x = torch.randn(5, 256, device=dev)
    x[2, 100] = float("nan")
    W, w = matrices(k3, dev, 41, 1, 200, 256)
    y = k3.mxfp4_mm(*k3.mxfp4_quant(x), W, out_dtype=torch.float32)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all()


def test_infinity_is_the_largest_value(k3, dev):
    """An infinite activation enters a product as 6 * 2^126, exactly: infinite only where the result
    leaves fp32's range, and no other row sees it."""
    import torch
    N, K = 40, 96
    c, b = operand(141, N, K)
    for wb in (90, 140):
        wbyte = np.full_like(b, wb)
        W = k3.Mxfp4Mat(*k3.mxfp4_pack(*to_dev(dev, pack_nibbles(c)[None], wbyte[None])))
        x = torch.zeros(3, K)
        x[0], x[2] = 1.0, 2.0
        x[1, 40], x[1, 41] = -float("inf"), 5.0
        y = k3.mxfp4_mm(*k3.mxfp4_quant(x.to(dev)), W, out_dtype=torch.float32).double().cpu().numpy()
        v = x.double().numpy().copy()
        v[1, 40], v[1, 41] = -6 * 2.0 ** 126, 0
        want = v @ values(c, wbyte).T
        with np.errstate(over="ignore"):
            assert np.array_equal(y, want.astype(np.float32))


def test_scales_over_the_whole_range(k3, dev):
    """Scale bytes 0..254 on either side; results inside fp32's range are right, and the widened
    weights of mm_bwd keep subnormal scales."""
    import torch
    N, K = 64, 64
    c, b = operand(51, N, K)
    for wb, ab in ((0, 254), (1, 250), (254, 0), (200, 30), (127, 127)):
        wbyte = np.full_like(b, wb)
        W = k3.Mxfp4Mat(*k3.mxfp4_pack(*to_dev(dev, pack_nibbles(c)[None], wbyte[None])))
        ac, _ = operand(52, 9, K)
        abyte = np.full((9, K // 32), ab, np.uint8)
        a, s = to_dev(dev, pack_nibbles(ac), abyte)
        y = k3.mxfp4_mm(a, s, W, out_dtype=torch.float32).double().cpu().numpy()
        assert np.array_equal(y, values(ac, abyte) @ values(c, wbyte).T)
        if wb > 251:
            continue        # 6 * 2^(wb - 127) exceeds fp32: infinities, as in the reference's flat path
        dy = (torch.randint(-3, 4, (9, N), device=dev).double() * 2.0 ** (100 if wb < 100 else 0)).bfloat16()
        da = k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32).double().cpu().numpy()
        assert np.array_equal(da, dy.double().cpu().numpy() @ values(c, wbyte))


def test_gradient_is_the_adjoint(k3, dev):
    """<dY, mm(A)> = <mm_bwd(dY), A>, and one code changed moves the product by that column of W:
    small integers everywhere, so both hold exactly."""
    import torch
    N, K, M = 136, 160, 21
    g = np.random.default_rng(3)
    c = g.choice([2, 4, 6, 10, 12, 0], (N, K)).astype(np.uint8)      # +-1, 2, 4
    one = np.full((N, K // 32), 127, np.uint8)
    W = k3.Mxfp4Mat(*k3.mxfp4_pack(*to_dev(dev, pack_nibbles(c)[None], one[None])))
    ac = g.choice([2, 4, 10, 12, 0], (M, K)).astype(np.uint8)
    a, s = to_dev(dev, pack_nibbles(ac), one[:M, :])
    dy = torch.randint(-4, 5, (M, N), device=dev).bfloat16()
    y = k3.mxfp4_mm(a, s, W, out_dtype=torch.float32)
    da = k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32)
    av = torch.from_numpy(values(ac, one[:M])).to(dev)
    assert (dy.double() * y.double()).sum() == (da.double() * av).sum()
    ac2 = ac.copy()
    ac2[:, 77] = np.where(ac[:, 77] == 2, 4, 2)
    y2 = k3.mxfp4_mm(to_dev(dev, pack_nibbles(ac2))[0], s, W, out_dtype=torch.float32)
    step = values(ac2, one[:M])[:, 77] - values(ac, one[:M])[:, 77]
    assert np.array_equal((y2 - y).double().cpu().numpy(), step[:, None] * values(c, one)[:, 77][None])


def test_captured_and_on_two_streams(k3, dev):
    import torch
    W, _ = matrices(k3, dev, 61, 6, 384, 512)
    off = torch.tensor([0, 100, 100, 350, 351, 380, 400], dtype=torch.int32, device=dev)

    def chain(x, dy):
        y = k3.mxfp4_mm(*k3.mxfp4_quant(x), W, off=off)
        return y, k3.mxfp4_mm_bwd(dy, W, off=off)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return torch.randn((400, 512), generator=g).to(dev), torch.randn((400, 384), generator=g).bfloat16().to(dev)
    a, b = inputs(1), inputs(2)
    wa, wb = chain(*a), chain(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            ga = chain(*a)
        with torch.cuda.stream(s2):
            gb = chain(*b)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ga + gb, wa + wb))
    held = [t.clone() for t in a]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = chain(*held)
    for src, want in ((b, wb), (a, wa)):
        for h, t in zip(held, src):
            h.copy_(t)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_experts_of_a_pool_layer_together(k3, dev):
    """The operators as a layer uses them, on a pool layer's own arena and run table: router, sort,
    quantising permute, gate/up product, SwiGLU, quantise, down product, weighted sum -- each
    step against 64 bits on the step's own inputs; then back through every step."""
    import torch
    H, I, E, K, T = 512, 256, 12, 3, 37
    g = k3.synth.rng(77)
    experts = [k3.synth.expert(g, H, I) for _ in range(E)]
    _, wb = k3.synth.router_weights(g, E, H)
    Wr = torch.from_numpy(wb.view(np.int16)).to(dev).view(torch.bfloat16)
    pl = k3.PoolMoeLayer.pack([k3.DeviceExpert.from_host(e, dev) for e in experts], None, Wr, None, H, I, K, dev)
    pl.run_of[5] = -1                                   # an expert that is not resident
    _, xb = k3.synth.activations(g, T, H)
    x = torch.from_numpy(xb.view(np.int16)).to(dev).view(torch.bfloat16)
    idx, wt, _ = k3.router(x, Wr, None, K)
    pos, pair, off = k3.moe_sort(idx, E)
    GU, D = k3.Mxfp4Mat.from_pool(pl, "gate_up"), k3.Mxfp4Mat.from_pool(pl, "down")
    a, sa = k3.moe_permute_mxfp4(x, pos)
    gu = k3.mxfp4_mm(a, sa, GU, off=off, out_dtype=torch.float32)
    blocks = gu.view(T * K, I // 64, 2, 64)
    gate, up = blocks[:, :, 0].reshape(T * K, I), blocks[:, :, 1].reshape(T * K, I)
    h = torch.nn.functional.silu(gate) * up
    b, sb = k3.mxfp4_quant(h)
    y = k3.mxfp4_mm(b, sb, D, off=off, out_dtype=torch.float32)
    out = k3.moe_unpermute(y, pos, wt)

    def mat(e, name):
        return values(unpack(e[name + "_p"]), e[name + "_s"])

    av, bv = values(unpack(a.cpu().numpy()), sa.cpu().numpy()), values(unpack(b.cpu().numpy()), sb.cpu().numpy())
    offn, idn, pn, wn = off.cpu().numpy(), idx.cpu().numpy(), pos.cpu().numpy(), wt.double().cpu().numpy()
    assert offn[-1] == T * K
    yn = y.double().cpu().numpy()
    dout = torch.randn((T, H), device=dev)
    dy, dwt = k3.moe_unpermute_bwd(dout, y, pos, wt)
    dh = k3.mxfp4_mm_bwd(dy.bfloat16(), D, off=off, out_dtype=torch.float32)
    sg = torch.sigmoid(gate)
    dgate, dup = dh * up * sg * (1 + gate * (1 - sg)), dh * gate * sg
    dgu = torch.stack([dgate.view(T * K, I // 64, 64), dup.view(T * K, I // 64, 64)], 2).reshape(T * K, 2 * I).bfloat16()
    da = k3.mxfp4_mm_bwd(dgu, GU, off=off, out_dtype=torch.float32)
    dx = k3.moe_permute_bwd(da, pos)
    for e in range(E):
        r = slice(offn[e], offn[e + 1])
        if e == 5:
            assert (gu[r] == 0).all() and (yn[r] == 0).all() and (da[r] == 0).all()
            continue
        wg, wu, wd = mat(experts[e], "gate"), mat(experts[e], "up"), mat(experts[e], "down")
        check(gate[r].double().cpu().numpy(), av[r] @ wg.T, np.abs(av[r]) @ np.abs(wg).T, H // 64, False)
        check(up[r].double().cpu().numpy(), av[r] @ wu.T, np.abs(av[r]) @ np.abs(wu).T, H // 64, False)
        check(yn[r], bv[r] @ wd.T, np.abs(bv[r]) @ np.abs(wd).T, I // 64, False)
        d = dy[r].bfloat16().double().cpu().numpy()
        check(dh[r].double().cpu().numpy(), d @ wd, np.abs(d) @ np.abs(wd), H // 16, False)
        wgu = np.stack([wg.reshape(I // 64, 64, H), wu.reshape(I // 64, 64, H)], 1).reshape(2 * I, H)
        d = dgu[r].double().cpu().numpy()
        check(da[r].double().cpu().numpy(), d @ wgu, np.abs(d) @ np.abs(wgu), 2 * I // 16, False)
    want = (wn[:, :, None] * yn[pn]).sum(1)
    lim = (K + 2) * 2.0 ** -24 * (np.abs(wn)[:, :, None] * np.abs(yn[pn])).sum(1)
    assert (np.abs(out.double().cpu().numpy() - want) <= lim).all()
    want = da.double().cpu().numpy()[pn]
    assert (np.abs(dx.double().cpu().numpy() - want.sum(1)) <= (K + 2) * 2.0 ** -24 * np.abs(want).sum(1)).all()


def test_experts_of_a_latent_layer(k3, dev):
    """A latent layer's own 896 experts at the latent width, 16 a token: both of its matrices from its
    arena and run table, each against 64 bits, and the gradient through the first."""
    import torch
    g = k3.synth.rng(79)
    H, Lw, I, E, K, T = 512, 256, 128, 896, 16, 40
    lat = k3.synth.latent_layer(g, H, Lw, I, 5, 4, n_shared=1, wdt=1)
    few = lat["experts"]
    lat.update(experts=[few[e % 5] for e in range(E)], topk=K, router_w=np.zeros((E, H), np.float32),
               router_bias=np.zeros(E, np.float32))
    layer = k3.LatentMoeLayer.from_host(lat, dev)
    gn = torch.Generator().manual_seed(3)
    idx = torch.stack([torch.randperm(E, generator=gn)[:K] for _ in range(T)]).int().to(dev)
    pos, _, off = k3.moe_sort(idx, E)
    row_e = np.zeros(T * K, int)
    row_e[pos.cpu().numpy()] = idx.cpu().numpy() % 5

    def mat(e, name):
        return values(unpack(e[name + "_p"]), e[name + "_s"])
    gate_up = np.stack([np.stack([mat(e, "gate").reshape(I // 64, 64, Lw), mat(e, "up").reshape(I // 64, 64, Lw)], 1)
                        .reshape(2 * I, Lw) for e in few])
    down = np.stack([mat(e, "down") for e in few])
    for which, w in (("gate_up", gate_up), ("down", down)):
        x = torch.randn((T, w.shape[2]), generator=gn).to(dev)
        a, s = k3.moe_permute_mxfp4(x, pos)
        W = k3.Mxfp4Mat.from_pool(layer, which)
        y = k3.mxfp4_mm(a, s, W, off=off, out_dtype=torch.float32).double().cpu().numpy()
        av = values(unpack(a.cpu().numpy()), s.cpu().numpy())
        check(y, np.einsum("mk,mnk->mn", av, w[row_e]), np.einsum("mk,mnk->mn", np.abs(av), np.abs(w[row_e])),
              w.shape[2] // 64, False)
        dy = torch.randn((T * K, w.shape[1]), generator=gn).bfloat16().to(dev)
        da = k3.mxfp4_mm_bwd(dy, W, off=off, out_dtype=torch.float32).double().cpu().numpy()
        dv = dy.double().cpu().numpy()
        check(da, np.einsum("mn,mnk->mk", dv, w[row_e]), np.einsum("mn,mnk->mk", np.abs(dv), np.abs(w[row_e])),
              w.shape[1] // 16, False)
    with pytest.raises(k3.K3CError, match="no pool-format runs"):
        k3.Mxfp4Mat.from_pool(lat, "down")


def test_products_match_the_gemv_and_dequant(k3, dev):
    """The same codes through the framework's own fp32-activation GEMV and dequantiser."""
    import torch
    N, K = 96, 256
    c, b = operand(71, N, K, 118, 125)
    p, s = to_dev(dev, pack_nibbles(c), b)
    x = torch.randn((5, K), device=dev)
    a, sa = k3.mxfp4_quant(x)
    y = k3.mxfp4_mm(a, sa, k3.Mxfp4Mat(*k3.mxfp4_pack(p, s)), out_dtype=torch.float32)
    ref = k3.mxfp4_gemv(k3.mxfp4_dequant(a, sa), p, s)
    mag = np.abs(values(unpack(a.cpu().numpy()), sa.cpu().numpy())) @ np.abs(values(c, b)).T
    assert (np.abs((y - ref).double().cpu().numpy()) <= (K + 16) * 2.0 ** -23 * mag).all()


def test_results_past_32_bits(k3, dev):
    """Product and gradient rows more than 4 GiB from the first, against the same rows alone."""
    import torch
    M, N, K = 600000, 4096, 64
    W, _ = matrices(k3, dev, 81, 1, N, K)
    g = torch.Generator(device=dev).manual_seed(1)
    a, s = k3.mxfp4_quant(torch.randn(M, K, generator=g, device=dev))
    y = k3.mxfp4_mm(a, s, W)
    assert torch.equal(y[-300:], k3.mxfp4_mm(a[-300:].contiguous(), s[-300:].contiguous(), W))
    assert torch.equal(y[:300], k3.mxfp4_mm(a[:300].contiguous(), s[:300].contiguous(), W))
    da = k3.mxfp4_mm_bwd(y, W)
    assert torch.equal(da[-300:], k3.mxfp4_mm_bwd(y[-300:], W)) and torch.equal(da[:300], k3.mxfp4_mm_bwd(y[:300], W))


def test_large_products_on_two_streams(k3, dev):
    """Kernels of CTA pairs from two streams at once, both products, eager and captured."""
    import torch
    W, _ = matrices(k3, dev, 91, 1, 4096, 2048)
    g = torch.Generator().manual_seed(4)
    x = [torch.randn((5000, 2048), generator=g).to(dev) for _ in range(2)]

    def chain(t):
        y = k3.mxfp4_mm(*k3.mxfp4_quant(t), W)
        return y, k3.mxfp4_mm_bwd(y, W)
    want = [chain(t) for t in x]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        cap = chain(x[0])
    for _ in range(5):
        got = []
        for t, q in zip(x, st):
            with torch.cuda.stream(q):
                got.append(chain(t))
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(got + [cap], want + [want[0]]):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_one_mapped_matrix_for_all_rows_and_no_rows(k3, dev):
    """Without offsets the rows multiply matrix mat_of[0]; no rows give empty results."""
    import torch
    N, K = 72, 96
    W, w = matrices(k3, dev, 101, 3, N, K)
    W = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=torch.tensor([2, 0], dtype=torch.int32, device=dev))
    c, b = operand(102, 10, K)
    a, s = to_dev(dev, pack_nibbles(c), b)
    dy = torch.randn(10, N, device=dev).bfloat16()
    av, dv = values(c, b), dy.double().cpu().numpy()
    check(k3.mxfp4_mm(a, s, W, out_dtype=torch.float32).double().cpu().numpy(), av @ w[2].T, np.abs(av) @ np.abs(w[2]).T, 2, False)
    check(k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32).double().cpu().numpy(), dv @ w[2], np.abs(dv) @ np.abs(w[2]), 5, False)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    for o in (None, off):
        assert k3.mxfp4_mm(a[:0], s[:0], W, off=o).shape == (0, N)
        assert k3.mxfp4_mm_bwd(dy[:0], W, off=o).shape == (0, K)
    assert k3.mxfp4_quant(torch.empty(0, 64, device=dev))[1].shape == (0, 2)


@pytest.mark.parametrize("G", [512, 896, 1024])
def test_the_most_groups(k3, dev, G):
    """Up to 1024 groups, most of them empty, sharing three matrices."""
    import torch
    N, K, M = 136, 160, 700
    g = np.random.default_rng(5)
    cuts = np.sort(np.concatenate([np.repeat(g.integers(0, M + 1, G // 4 - 8), 4), np.zeros(20, int), np.full(11, M)]))
    off = np.concatenate([[0], cuts, [M]]).astype(np.int32)
    assert off.size == G + 1
    mat_of = g.integers(0, 3, G).astype(np.int32)
    W, w = matrices(k3, dev, 111, 3, N, K)
    c, b = operand(112, M, K)
    a, s, po, pm = to_dev(dev, pack_nibbles(c), b, off, mat_of)
    W = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=pm)
    y = k3.mxfp4_mm(a, s, W, off=po, out_dtype=torch.float32).double().cpu().numpy()
    dy = torch.randn(M, N, device=dev).bfloat16()
    da = k3.mxfp4_mm_bwd(dy, W, off=po, out_dtype=torch.float32).double().cpu().numpy()
    row_w = w[np.repeat(mat_of, np.diff(off))]          # [M][N][K]
    av, dv = values(c, b), dy.double().cpu().numpy()
    check(y, np.einsum("mk,mnk->mn", av, row_w), np.einsum("mk,mnk->mn", np.abs(av), np.abs(row_w)), 3, False)
    check(da, np.einsum("mn,mnk->mk", dv, row_w), np.einsum("mn,mnk->mk", np.abs(dv), np.abs(row_w)), 9, False)


@pytest.mark.parametrize("K", [32, 96, 160, 512, 1056, 2016])
@pytest.mark.parametrize("first", [0, 1, 3, 5, 8])
def test_scale_rows_on_any_boundary(k3, dev, first, K):
    """a_scales at every kind of address, for row lengths of odd and even bytes; nothing beside the
    array is read as a scale (its neighbours hold the NaN byte)."""
    import torch
    N = 64
    W, w = matrices(k3, dev, 121, 1, N, K)
    for M in (1, 2, 33, 129):
        c, b = operand(122, M, K)
        a = to_dev(dev, pack_nibbles(c))[0]
        buf = torch.full((first + b.size + 40,), 255, dtype=torch.uint8, device=dev)
        s = buf[first:first + b.size].view(M, K // 32)
        s.copy_(torch.from_numpy(b))
        av = values(c, b)
        y = k3.mxfp4_mm(a, s, W, out_dtype=torch.float32).double().cpu().numpy()
        check(y, av @ w[0].T, np.abs(av) @ np.abs(w[0]).T, -(-K // 64), False)


def test_result_may_not_be_the_rows(k3, dev):
    import torch
    W, _ = matrices(k3, dev, 131, 1, 64, 64)
    dy = torch.randn(9, 64, device=dev).bfloat16()
    a, s = k3.mxfp4_quant(dy)
    with pytest.raises(k3.K3CError, match="may not be an input"):
        k3.mxfp4_mm_bwd(dy, W, out=dy)
    with pytest.raises(k3.K3CError, match="may not be an input"):
        k3.mxfp4_mm(a[:8], s[:8], k3.Mxfp4Mat(*k3.mxfp4_pack(*k3.mxfp4_quant(dy[:8]))), out=a.view(-1)[:256].view(torch.float32).view(8, 8))
    with pytest.raises(k3.K3CError, match="n_experts"):
        k3.moe_sort(torch.zeros(2, 2, dtype=torch.int32, device=dev), (1 << 32) + 4)


def test_pack_in_place(k3, dev):
    """The codes written over the packed nibbles they come from."""
    import torch
    g = np.random.default_rng(8)
    n, rows, in_ = 3, 70, 160
    p, s = to_dev(dev, g.integers(0, 256, (n, rows, in_ // 2), dtype=np.uint8), g.integers(250, 256, (n, rows, in_ // 32), dtype=np.uint8))
    codes, atoms = k3.mxfp4_pack(p, s)
    mine = torch.empty_like(atoms)
    assert k3.lib().k3c_mxfp4_pack(p.data_ptr(), mine.data_ptr(), p.data_ptr(), s.data_ptr(), n, rows, in_,
                                   torch.cuda.current_stream(dev).cuda_stream) == 0
    assert torch.equal(p, codes) and torch.equal(mine, atoms)


def test_offsets_that_name_rows_again_and_again(k3, dev):
    """Descending offsets that let 512 groups name all rows each: more tiles than 32 bits count. The
    first of them is done, and nothing outside the result is touched."""
    import torch
    torch.cuda.empty_cache()
    G, M, N, K = 1024, (1 << 29) + 384, 1, 32
    W, _ = matrices(k3, dev, 151, 1, N, K)
    W = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=torch.zeros(G, dtype=torch.int32, device=dev))
    g = torch.Generator(device=dev).manual_seed(2)
    a = torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, device=dev, generator=g)
    s = torch.full((M, 1), 127, dtype=torch.uint8, device=dev)
    off = torch.zeros(G + 1, dtype=torch.int32, device=dev)
    off[1::2] = M
    buf = torch.full((M + 256, N), 7.0, dtype=torch.bfloat16, device=dev)
    k3.mxfp4_mm(a, s, W, off=off, out=buf[128:M + 128])
    assert (buf[:128] == 7).all() and (buf[M + 128:] == 7).all()
    assert torch.equal(buf[128:M + 128], k3.mxfp4_mm(a, s, W))


def test_result_may_not_overlap_what_is_read(k3, dev):
    """A product's result in part of its rows, scales, offsets, matrices or map is refused; columns
    of one buffer side by side are not."""
    import torch
    N, K, M = 64, 64, 40
    W, w = matrices(k3, dev, 161, 2, N, K)
    big = torch.zeros(1 << 16, dtype=torch.uint8, device=dev)
    raw = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=big[4096:4104].view(torch.int32))
    c, b = operand(162, M, K)
    a, s = to_dev(dev, pack_nibbles(c), b)

    def put(t, at):
        v = big[at:at + t.nbytes].view(t.dtype).view(t.shape)
        v.copy_(t)
        return v

    off = torch.tensor([0, 20, M], dtype=torch.int32, device=dev)
    nb = M * N * 2
    out = big[8192:8192 + nb].view(torch.bfloat16).view(M, N)
    dy = torch.randn(M, N, device=dev).bfloat16()
    codes, atoms = W.keep[0], W.keep[1]
    for call in (lambda: k3.mxfp4_mm(put(a, 8192 + nb - 16), s, W, out=out),
                 lambda: k3.mxfp4_mm(a, put(s, 8192 - s.nbytes + 1), W, out=out),
                 lambda: k3.mxfp4_mm(a, s, W, off=put(off, 8192 + 400), out=out),
                 lambda: k3.mxfp4_mm(a, s, k3.Mxfp4Mat(put(codes, 8192 + nb - 16), atoms), out=out),
                 lambda: k3.mxfp4_mm(a, s, k3.Mxfp4Mat(codes, put(atoms, 8192 - 512)), out=out),
                 lambda: k3.mxfp4_mm(a, s, raw, off=off, out=big[4100:4100 + nb].view(torch.bfloat16).view(M, N)),
                 lambda: k3.mxfp4_mm_bwd(put(dy, 8192 + nb - 32), W, out=out),
                 lambda: k3.mxfp4_mm_bwd(dy, W, off=put(off, 8192 - 4), out=out)):
        with pytest.raises(k3.K3CError, match="may not be an input"):
            call()
    want = k3.mxfp4_mm(a, s, W), k3.mxfp4_mm_bwd(dy, W)
    wide = torch.full((M, 3 * N), 7.0, dtype=torch.bfloat16, device=dev)
    wide[:, N:2 * N].copy_(dy)
    k3.mxfp4_mm_bwd(wide[:, N:2 * N], W, out=wide[:, 2 * N:])
    assert torch.equal(wide[:, 2 * N:], want[1]) and torch.equal(wide[:, N:2 * N], dy) and (wide[:, :N] == 7).all()
    with pytest.raises(k3.K3CError, match="may not be an input"):
        k3.mxfp4_mm_bwd(wide[:, N:2 * N], W, out=wide[:, 2 * N - 8:3 * N - 8])
    assert torch.equal(k3.mxfp4_mm(put(a, 8192 + nb), put(s, 8192 - s.nbytes), W, out=out), want[0])


def test_the_longest_sums(k3, dev):
    """A gradient over 2^29 weight rows, 8.4 million K blocks of one tile (2.5 s, longer than a wait
    inside the kernel may take otherwise), and a product over the longest rows there may be. All but
    some elements are 0 and the others small integers: every sum is exact."""
    import torch
    torch.cuda.empty_cache()
    g = torch.Generator(device=dev).manual_seed(6)

    def ones(n):       # n places and +-1 there
        at = torch.cat([torch.randint(0, n, (200,), generator=g, device=dev), torch.tensor([0, n - 1], device=dev)]).unique()
        return at, torch.randint(0, 2, at.shape, generator=g, device=dev).double() * 2 - 1
    N, K = (1 << 29) + 40, 32
    codes = torch.randint(0, 256, (1, N, K // 2), dtype=torch.uint8, device=dev, generator=g) & 0x66    # 0, 1, 2, 4
    atoms = torch.full((1, -(-N // 128), 1, 512), 127, dtype=torch.uint8, device=dev)
    at, v = ones(N)
    dy = torch.zeros(1, N, dtype=torch.bfloat16, device=dev)
    dy[0, at] = v.bfloat16()
    da = k3.mxfp4_mm_bwd(dy, k3.Mxfp4Mat(codes, atoms), out_dtype=torch.float32)
    grid = torch.tensor(GRID, device=dev)
    rows = grid[torch.stack([codes[0, at] & 7, codes[0, at] >> 4 & 7], -1).reshape(len(at), K).long()]
    assert torch.equal(da[0].double(), v @ rows)
    del codes, atoms, dy
    K = (1 << 31) - 1024
    a = torch.zeros(1, K // 2, dtype=torch.uint8, device=dev)
    at, v = ones(K // 2)
    a[0, at] = torch.where(v > 0, 0x22, 0x2A).to(torch.uint8)          # 1, 1 and -1, 1
    codes = torch.randint(0, 256, (1, 1, K // 2), dtype=torch.uint8, device=dev, generator=g) & 0x66
    W = k3.Mxfp4Mat(codes, torch.full((1, 1, K // 128, 512), 127, dtype=torch.uint8, device=dev))
    y = k3.mxfp4_mm(a, torch.full((1, K // 32), 127, dtype=torch.uint8, device=dev), W, out_dtype=torch.float32)
    w = grid[torch.stack([codes[0, 0, at] & 7, codes[0, 0, at] >> 4 & 7], -1).long()]
    assert y.item() == (v * w[:, 0] + w[:, 1]).sum().item()


@pytest.mark.parametrize("N", [1, 7, 65, 257, 4095])
def test_gradient_of_padded_rows(k3, dev, N):
    """dy of any number of columns in rows whose stride is a multiple of 8, one row (contiguous to
    torch) and several, beside values that are NaN."""
    import torch
    K = 96
    W, w = matrices(k3, dev, 171, 1, N, K)
    ld = -(-N // 8) * 8 + 16
    for M in (1, 2, 33):
        buf = torch.full((M + 1, ld), float("nan"), dtype=torch.bfloat16, device=dev)
        dy = buf[:M, :N]
        dy.copy_(torch.randn((M, N), generator=torch.Generator().manual_seed(M)))
        da = k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32).double().cpu().numpy()
        dv = dy.double().cpu().numpy()
        check(da, dv @ w[0], np.abs(dv) @ np.abs(w[0]), -(-N // 16), False)


@pytest.mark.parametrize("N", [1, 7, 65, 257, 4095, 4104])
def test_gradient_of_rows_on_any_boundary(k3, dev, N):
    """dy as the product's own result has it, contiguous whatever its width, and rows at odd addresses
    and strides; grouped, with rows behind the last group left as they were, eager and captured."""
    import torch
    K, G = 160, 3
    W, w = matrices(k3, dev, 181, G, N, K)
    for M, sizes in ((0, [0, 0, 0]), (1, [0, 1, 0]), (2, [1, 0, 1]), (40, [3, 0, 30])):
        off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        po = to_dev(dev, off)[0]
        for first, pad in ((0, 0), (1, 0), (3, 2), (8, 3)):
            buf = torch.full(((N + pad) * M + first + 9,), float("nan"), dtype=torch.bfloat16, device=dev)
            dy = buf[first:first + (N + pad) * M].view(M, N + pad)[:, :N]
            dy.copy_(torch.randn((M, N), generator=torch.Generator().manual_seed(M)))
            da = torch.full((M, K), 7.0, device=dev)
            k3.mxfp4_mm_bwd(dy, W, off=po, out=da)
            assert (da[off[-1]:] == 7).all()
            got, dv = da.double().cpu().numpy(), dy.double().cpu().numpy()
            for e in range(G):
                r = slice(off[e], off[e + 1])
                check(got[r], dv[r] @ w[e], np.abs(dv[r]) @ np.abs(w[e]), -(-N // 16), False)
    held = torch.zeros_like(dy)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap = k3.mxfp4_mm_bwd(held, W, off=po, out=torch.zeros_like(da))
    held.copy_(dy)
    g.replay()
    assert torch.equal(cap[:off[-1]], da[:off[-1]])
    flat = torch.randn(33 * max(N, K) + 8, device=dev).bfloat16()       # a copied dy is no less an input
    with pytest.raises(k3.K3CError, match="may not be an input"):
        k3.mxfp4_mm_bwd(flat[1:1 + 33 * N].view(33, N), W, out=flat[:33 * K].view(33, K))


def test_under_autograd(k3, dev):
    """Inputs that require grad are refused by name; inside autograd functions the calls and their
    gradients make a differentiable layer of frozen experts, whose gradients are the calls' own."""
    import torch
    T, K, E, H, I = 40, 3, 7, 96, 64
    g = torch.Generator().manual_seed(9)
    W, _ = matrices(k3, dev, 191, E, I, H)
    idx = torch.randint(0, E, (T, K), generator=g).int().to(dev)
    pos, _, off = k3.moe_sort(idx, E)
    x0, wt0 = torch.randn((T, H), generator=g).to(dev), torch.rand((T, K), generator=g).to(dev)
    x, wt = x0.clone().requires_grad_(), wt0.clone().requires_grad_()
    y0, d0 = torch.randn((T * K, I), generator=g).to(dev), torch.randn((T, I), generator=g).to(dev)
    y, d = y0.clone().requires_grad_(), d0.clone().requires_grad_()
    bf = torch.zeros((T * K, I), dtype=torch.bfloat16, device=dev, requires_grad=True)
    rows = torch.zeros((T * K, H), device=dev, requires_grad=True)
    for name, call in (("x", lambda: k3.moe_permute(x, pos)), ("x", lambda: k3.moe_permute_mxfp4(x, pos)),
                       ("x", lambda: k3.mxfp4_quant(x)), ("out", lambda: k3.moe_permute(x0, pos, out=rows)),
                       ("drows", lambda: k3.moe_permute_bwd(y, pos)), ("y", lambda: k3.moe_unpermute(y, pos, wt0)),
                       ("wt", lambda: k3.moe_unpermute(y0, pos, wt)), ("dout", lambda: k3.moe_unpermute_bwd(d, y0, pos, wt0)),
                       ("dy", lambda: k3.mxfp4_mm_bwd(bf, W, off=off))):
        with pytest.raises(k3.K3CError, match=f"^{name}: requires grad"):
            call()

    class Layer(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, wt):
            y = k3.mxfp4_mm(*k3.moe_permute_mxfp4(x, pos), W, off=off, out_dtype=torch.float32)
            ctx.save_for_backward(y, wt)
            return k3.moe_unpermute(y, pos, wt)

        @staticmethod
        def backward(ctx, dout):
            y, wt = ctx.saved_tensors
            dy, dwt = k3.moe_unpermute_bwd(dout.contiguous(), y, pos, wt)
            return k3.moe_permute_bwd(k3.mxfp4_mm_bwd(dy.bfloat16(), W, off=off, out_dtype=torch.float32), pos), dwt

    Layer.apply(x, wt).backward(d0)
    y = k3.mxfp4_mm(*k3.moe_permute_mxfp4(x0, pos), W, off=off, out_dtype=torch.float32)
    dy, dwt = k3.moe_unpermute_bwd(d0, y, pos, wt0)
    assert torch.equal(wt.grad, dwt)
    assert torch.equal(x.grad, k3.moe_permute_bwd(k3.mxfp4_mm_bwd(dy.bfloat16(), W, off=off, out_dtype=torch.float32), pos))


def test_an_empty_map_is_refused(k3, dev):
    import torch
    W, _ = matrices(k3, dev, 201, 2, 64, 64)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    with pytest.raises(k3.K3CError, match="mat_of"):
        k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=none)
    a, s = k3.mxfp4_quant(torch.randn(4, 64, device=dev))
    with pytest.raises(k3.K3CError, match="off"):
        k3.mxfp4_mm(a, s, W, off=none)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_finite_elements_beside_an_infinity(k3, dev, dtype):
    """Byte 253 for the group, finite elements rounded under it: 0 up to 2^124, a code above, and from
    3.5 * 2^126 on the code 4, which is 2^128 to the dequantiser."""
    import torch
    near = [2.0 ** 124, 2.0 ** 124 * 1.01, 1.5 * 2.0 ** 125, 3e38, -2.0 ** 127, 2.0 ** 123, -2.0 ** 124, 1.0]
    x = torch.zeros(3, 40)
    x[:, 3] = torch.tensor([float("inf"), -float("inf"), float("inf")])
    x[:, 4:12] = torch.tensor(near)
    x[2] = x[2].roll(30)                                   # in a short group
    x = x.bfloat16() if dtype == "bf16" else x
    packed, scales = k3.mxfp4_quant(x.to(dev))
    codes, byte = quant_plain(x.double().numpy())
    assert np.array_equal(scales.cpu().numpy(), byte) and (byte == 253).sum() == 3
    assert np.array_equal(unpack(packed.cpu().numpy())[:, :40], codes)
    assert codes[0, 4] == 0 and codes[0, 5] == 1 and codes[0, 7] == 6
    wide = torch.zeros(1, 64)
    wide[0, 32:35] = torch.tensor([float("inf"), 3e38, -2.0 ** 127])
    back = k3.mxfp4_dequant(*k3.mxfp4_quant(wide.to(dev))).cpu()
    assert back[0, 32:35].tolist() == [float("inf"), float("inf"), -2.0 ** 127]


@pytest.mark.parametrize("byte", [252, 253, 254])
def test_gradient_of_the_largest_weights(k3, dev, byte):
    """Every code under the last scale bytes, finite as long as its magnitude is below 2^128 (all of
    them under 252), by one weight row whose gradient is the row itself."""
    import torch
    c = (np.arange(32, dtype=np.uint8) % 16)[None]
    b = np.full((1, 1), byte, np.uint8)
    W = k3.Mxfp4Mat(*k3.mxfp4_pack(*to_dev(dev, pack_nibbles(c), b)))
    v = values(c, b)
    v[np.abs(v) >= 2.0 ** 128] = np.inf * np.sign(v[np.abs(v) >= 2.0 ** 128])
    assert np.isfinite(v).all() == (byte == 252)
    dy = torch.tensor([[2.0 ** -20], [-3.0], [0.25]], device=dev).bfloat16()
    da = k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32).double().cpu().numpy()
    want = dy.double().cpu().numpy() * v
    want[np.abs(want) >= 2.0 ** 128] = np.inf * np.sign(want[np.abs(want) >= 2.0 ** 128])
    assert np.array_equal(da, want)
    N, K = 64, 64                                          # and sums of them
    c, b = operand(211, N, K)
    b[:] = byte
    if byte == 252:
        W = k3.Mxfp4Mat(*k3.mxfp4_pack(*to_dev(dev, pack_nibbles(c), b)))
        dy = (torch.randint(-3, 4, (9, N), device=dev).double() * 2.0 ** -20).bfloat16()
        da = k3.mxfp4_mm_bwd(dy, W, out_dtype=torch.float32).double().cpu().numpy()
        assert np.array_equal(da, dy.double().cpu().numpy() @ values(c, b))


# ragged groups, and the tiles (rows, columns) that the product and its gradient take for them
TILED = [([1400, 1, 0, 1290], 4104, 1824, (256, 256), (512, 256)),
         ([700, 0, 900, 1300] + [300] * 30, 1304, 1312, (128, 256), (256, 256)),
         ([100, 9, 0, 130] * 12, 200, 2080, (128, 128), (128, 256)),
         ([40, 30, 1, 0, 33, 9, 20, 60], 520, 1056, (128, 64), (128, 128))]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("roll", [0, 4, 7])
@pytest.mark.parametrize("sizes,N,K,tile,tile_bwd", TILED, ids=["%dx%d" % t[3] for t in TILED])
def test_groups_without_a_matrix_in_every_tile(k3, dev, sizes, N, K, tile, tile_bwd, roll, out):
    """Both products in every tile shape, where groups at the start, at the end and side by side have
    no matrix: zeros for those, the others' results beside them, rows behind the last group as they
    were; with roll 7 the offsets leave the rows at both ends."""
    import torch
    G, n = len(sizes), sum(sizes)
    M = n if roll == 7 else n + 3
    L = k3.lib()
    assert divmod(L.k3c_mxfp4_mm_tile(M, G, 1, N, K, 0), 65536) == tile
    assert divmod(L.k3c_mxfp4_mm_tile(M, G, 1, N, K, 1), 65536) == tile_bwd
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    mat_of = np.roll(np.array([-1, 0, 7, 1, -1, -3, 2, 0], np.int32), -roll)[np.arange(G) % 8]
    given = off.copy()
    if roll == 7:
        given[0], given[-1] = -9, n + 10 ** 6
    W, w = matrices(k3, dev, 221, 3, N, K)
    c, b = operand(222, M, K)
    a, s, po, pm = to_dev(dev, pack_nibbles(c), b, given, mat_of)
    W = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=pm)
    dt = torch.float32 if out == "f32" else torch.bfloat16
    y = torch.full((M, N), 7.0, dtype=dt, device=dev)
    da = torch.full((M, K), 7.0, dtype=dt, device=dev)
    dy = torch.randn((M, N), generator=torch.Generator().manual_seed(N)).bfloat16().to(dev)
    k3.mxfp4_mm(a, s, W, off=po, out=y)
    k3.mxfp4_mm_bwd(dy, W, off=po, out=da)
    assert (y[n:] == 7).all() and (da[n:] == 7).all()
    av, wv = to_dev(dev, values(c, b), w)
    dv = dy.double()
    for e in range(G):
        r = slice(off[e], off[e + 1])
        if not 0 <= mat_of[e] < 3:
            assert (y[r] == 0).all() and (da[r] == 0).all()
            continue
        m = wv[mat_of[e]]
        check(*(t.double().cpu().numpy() for t in (y[r], av[r] @ m.T, av[r].abs() @ m.abs().T)), -(-K // 64), out == "bf16")
        check(*(t.double().cpu().numpy() for t in (da[r], dv[r] @ m, dv[r].abs() @ m.abs())), -(-N // 16), out == "bf16")


def test_experts_of_a_pool_that_are_loaded_and_evicted(k3, dev):
    """The matrices of a layer over an ExpertPool's slots: each product takes what the run table names
    when it runs, zeros for experts that are not resident."""
    import torch
    H, I, NE, NS = 256, 128, 8, 4
    g = k3.synth.rng(83)
    experts = [k3.synth.expert(g, H, I) for _ in range(NE)]
    run = torch.empty(k3.pool_run_bytes(H, I), dtype=torch.uint8, device=dev)
    host = []
    for e in experts:
        k3.pool_pack(run, k3.DeviceExpert.from_host(e, dev).q(), H, I)
        host.append(run.cpu().pin_memory())
    pool = k3.ExpertPool(H, I, 1, NE, NS, lambda layer, e: host[e])
    run_of = pool.run_table()
    Wr = torch.zeros((NE, H), dtype=torch.bfloat16, device=dev)
    layer = pool.layer(Wr, H, I, 2, NE, run_of)
    D, GU = k3.Mxfp4Mat.from_pool(layer, "down"), k3.Mxfp4Mat.from_pool(layer, "gate_up")
    assert (D.rows, D.in_, GU.rows, GU.in_, D.groups) == (H, I, 2 * I, H, NE)
    idx = torch.arange(24, dtype=torch.int32, device=dev).view(12, 2) % NE
    pos, _, off = k3.moe_sort(idx, NE)
    gn = torch.Generator().manual_seed(1)
    x = torch.randn((12, H), generator=gn).to(dev)
    h, dy = torch.randn((24, I), generator=gn).to(dev), torch.randn((24, H), generator=gn).bfloat16().to(dev)
    a, sa = k3.moe_permute_mxfp4(x, pos)
    b, sb = k3.mxfp4_quant(h)
    av, bv = values(unpack(a.cpu().numpy()), sa.cpu().numpy()), values(unpack(b.cpu().numpy()), sb.cpu().numpy())
    dv, offn = dy.double().cpu().numpy(), off.cpu().numpy()

    def mat(e, name):
        return values(unpack(e[name + "_p"]), e[name + "_s"])
    for ids in ([0, 3, 5, 6], [7, 1, 3]):
        pool.acquire(0, ids, run_of)
        table = run_of.cpu().numpy()
        gu = k3.mxfp4_mm(a, sa, GU, off=off, out_dtype=torch.float32).double().cpu().numpy()
        y = k3.mxfp4_mm(b, sb, D, off=off, out_dtype=torch.float32).double().cpu().numpy()
        dh = k3.mxfp4_mm_bwd(dy, D, off=off, out_dtype=torch.float32).double().cpu().numpy()
        assert all(table[e] >= 0 for e in ids) and (table < 0).sum() >= NE - NS
        for e in range(NE):
            r = slice(offn[e], offn[e + 1])
            if table[e] < 0:
                assert (gu[r] == 0).all() and (y[r] == 0).all() and (dh[r] == 0).all()
                continue
            wg, wu, wd = mat(experts[e], "gate"), mat(experts[e], "up"), mat(experts[e], "down")
            blocks = gu[r].reshape(-1, I // 64, 2, 64)
            check(blocks[:, :, 0].reshape(-1, I), av[r] @ wg.T, np.abs(av[r]) @ np.abs(wg).T, H // 64, False)
            check(blocks[:, :, 1].reshape(-1, I), av[r] @ wu.T, np.abs(av[r]) @ np.abs(wu).T, H // 64, False)
            check(y[r], bv[r] @ wd.T, np.abs(bv[r]) @ np.abs(wd).T, I // 64, False)
            check(dh[r], dv[r] @ wd, np.abs(dv[r]) @ np.abs(wd), H // 16, False)
        pool.release(0, ids)
    torch.cuda.synchronize()
    pool.close()


# 60 groups of 0 to 181 rows with a matrix in most of them
RAGGED = [39, 17, 2, 44, 72, 48, 7, 20, 2, 29, 18, 76, 63, 56, 1, 56, 72, 8, 80, 8, 35, 31, 181, 8, 4, 101, 7, 23, 42, 13, 2,
          29, 20, 14, 31, 6, 23, 5, 35, 39, 9, 41, 17, 6, 75, 13, 4, 0, 14, 14, 55, 2, 37, 71, 28, 13, 3, 6, 3, 61]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("sizes,N,K", [t[:3] for t in TILED] + [(RAGGED, 819, 1440), ([1100], 832, 2048)],
                         ids=["%dx%d" % t[3] for t in TILED] + ["ragged", "dense"])
def test_slow_stores_change_no_result(k3, dev, sizes, N, K, out):
    """Results in rows on odd addresses, which are stored element by element, are those in rows that are
    not, bit for bit and every time: the epilogue's slow stores hold up whatever shares their way to
    memory, so that waits which fast ones never test are."""
    import torch
    G, M = len(sizes), sum(sizes)
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    mat_of = np.array([0, 1, 2, 0, -1], np.int32)[np.arange(G) % 5]
    W, _ = matrices(k3, dev, 231, 3, N, K)
    c, b = operand(232, M, K)
    a, s, po, pm = to_dev(dev, pack_nibbles(c), b, off, mat_of)
    W = k3.Mxfp4Mat(W.keep[0], W.keep[1], mat_of=pm)
    dt = torch.float32 if out == "f32" else torch.bfloat16
    dy = torch.randn((M, N), generator=torch.Generator().manual_seed(N)).bfloat16().to(dev)
    want = k3.mxfp4_mm(a, s, W, off=po, out_dtype=dt), k3.mxfp4_mm_bwd(dy, W, off=po, out_dtype=dt)
    got = [torch.zeros(M * (n + 1) + 1, dtype=dt, device=dev)[1:].view(M, n + 1)[:, :n] for n in (N, K)]
    bad = torch.zeros((), dtype=torch.int64, device=dev)
    for _ in range(25):
        k3.mxfp4_mm(a, s, W, off=po, out=got[0])
        k3.mxfp4_mm_bwd(dy, W, off=po, out=got[1])
        for g, w in zip(got, want):
            bad += (g != w).sum()
            g.zero_()
    assert bad.item() == 0


def test_quantising_and_packing_past_32_bits(k3, dev):
    """More than 2^32 elements in and bytes out: the last rows and matrices as they come out alone."""
    import torch
    torch.cuda.empty_cache()
    g = torch.Generator(device=dev).manual_seed(7)
    H = 7168
    x = torch.randn((600008, H + 8), device=dev, generator=g, dtype=torch.bfloat16)
    for v in (x.view(-1)[:600000 * H].view(600000, H), x[:, :H], x[:, 1:H + 1], x[:, :H - 2]):
        p, s = k3.mxfp4_quant(v)
        for i in (slice(0, 300), slice(-300, None)):
            wp, ws = k3.mxfp4_quant(v[i].contiguous())
            assert torch.equal(p[i], wp) and torch.equal(s[i], ws)
        del p, s
    T, K = 80000, 16
    idx = torch.randint(0, 5, (T, K), device=dev, generator=g, dtype=torch.int32)
    pos, pair, _ = k3.moe_sort(idx, 5)
    p, s = k3.moe_permute_mxfp4(x[:T, :H], pos)
    wp, ws = k3.mxfp4_quant(x[:T, :H])
    for i in (slice(0, 300), slice(-300, None)):
        tok = (pair[i] // K).long()
        assert torch.equal(p[i], wp[tok]) and torch.equal(s[i], ws[tok])
    del p, s, wp, ws, x
    n, rows = 320, 4096
    p = torch.randint(0, 256, (n, rows, H // 2), dtype=torch.uint8, device=dev, generator=g)
    s = torch.randint(118, 256, (n, rows, H // 32), dtype=torch.uint8, device=dev, generator=g)
    codes, atoms = k3.mxfp4_pack(p, s)
    for i in (0, n - 1):
        wc, wa = k3.mxfp4_pack(p[i], s[i])
        assert torch.equal(codes[i], wc[0]) and torch.equal(atoms[i], wa[0])
    a, sa = k3.mxfp4_quant(torch.randn((40, H), device=dev, generator=g))
    off = torch.zeros(n + 1, dtype=torch.int32, device=dev)
    off[n:] = 40                                    # all rows at the last matrix
    W = k3.Mxfp4Mat(codes, atoms)
    y = k3.mxfp4_mm(a, sa, W, off=off)
    last = k3.Mxfp4Mat(wc, wa)
    assert torch.equal(y.view(torch.int16), k3.mxfp4_mm(a, sa, last).view(torch.int16))      # the bits: infinities and NaN
    assert torch.equal(k3.mxfp4_mm_bwd(y, W, off=off).view(torch.int16), k3.mxfp4_mm_bwd(y, last).view(torch.int16))
    del p, s, codes, atoms, W
    torch.cuda.empty_cache()
