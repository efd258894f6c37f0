"""Tokens sorted by expert and back (k3c_moe_sort, k3c_moe_permute, k3c_moe_permute_mxfp4,
k3c_moe_unpermute and their gradients) against plain numpy in 64 bits.

Tolerances. Copies and integers are exact. A sum of k terms in fp32, each term rounded once and
added once, is within (k + 1) * 2^-24 * sum|terms| of the exact sum; rounding the result to bf16
adds 2^-8 of its magnitude, to fp32 2^-24. dwt sums H products: at most ceil(H/256) * 8 fused
adds per thread, 5 warp steps and 8 partial sums, each off by 2^-24 of the sum of magnitudes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


@pytest.fixture(scope="module")
def dev():
    import torch
    return torch.device("cuda:0")


def torch_dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def rand(shape, dtype, seed, dev):
    import torch
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(torch_dtype(dtype)).to(dev)


def plain_sort(idx, E):
    T, K = idx.shape
    flat = idx.reshape(-1)
    rows = [p for e in range(E) for p in np.nonzero(flat == e)[0]]
    pos = np.full(T * K, -1, np.int32)
    pair = np.full(T * K, -1, np.int32)
    for r, p in enumerate(rows):
        pos[p] = r
        pair[r] = p
    off = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(E)])]).astype(np.int32)
    return pos.reshape(T, K), pair, off


def routing(T, K, E, kind, seed):
    g = np.random.default_rng(seed)
    if kind == "distinct":        # with fewer experts than choices the rest are dropped
        return np.argsort(g.random((T, max(E, K))), axis=1)[:, :K].astype(np.int32)
    if kind == "repeats":         # a token may name an expert twice
        return g.integers(0, E, (T, K)).astype(np.int32)
    if kind == "one":             # every pair at the last expert
        return np.full((T, K), E - 1, np.int32)
    if kind == "none":            # every pair dropped
        return np.where(g.random((T, K)) < 0.5, -1, E + 7).astype(np.int32)
    if kind == "holes":           # dropped pairs, extreme ids, and tokens without any row
        idx = g.integers(-2, E + 2, (T, K)).astype(np.int32)
        idx[g.random((T, K)) < 0.1] = np.iinfo(np.int32).min
        idx[g.random((T, K)) < 0.1] = np.iinfo(np.int32).max
        idx[::3] = -1
        return idx
    raise AssertionError(kind)


@pytest.mark.parametrize("kind", ["distinct", "repeats", "one", "none", "holes"])
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 8, 384), (3, 5, 7), (128, 8, 32), (129, 8, 33), (512, 8, 384),
                                   (1024, 8, 384), (1025, 8, 384), (2053, 6, 1500), (5000, 1, 2048), (9001, 7, 13),
                                   (513, 64, 7), (1000, 64, 383)])
def test_sort(k3, dev, T, K, E, kind):
    import torch
    idx = routing(T, K, E, kind, T + K + E)
    pos, pair, off = k3.moe_sort(torch.from_numpy(idx).to(dev), E)
    wpos, wpair, woff = plain_sort(idx, E)
    assert np.array_equal(off.cpu().numpy(), woff)
    assert np.array_equal(pos.cpu().numpy(), wpos)
    assert np.array_equal(pair.cpu().numpy(), wpair)


def test_sort_many_pairs(k3, dev):
    """More pairs than one pass of every block: 128 blocks of several passes."""
    import torch
    T, K, E = 90001, 8, 61
    idx = np.random.default_rng(3).integers(-1, E, (T, K)).astype(np.int32)
    pos, pair, off = (t.cpu().numpy() for t in k3.moe_sort(torch.from_numpy(idx).to(dev), E))
    flat = idx.reshape(-1)
    order = np.argsort(np.where(flat < 0, E, flat), kind="stable")
    n = int((flat >= 0).sum())
    assert np.array_equal(pair[:n], order[:n]) and (pair[n:] == -1).all()
    assert np.array_equal(off, np.searchsorted(np.sort(flat[flat >= 0]), np.arange(E + 1)))
    assert np.array_equal(pos.reshape(-1)[order[:n]], np.arange(n)) and (pos.reshape(-1)[flat < 0] == -1).all()


SHAPES = [(1, 1, 1, 8), (1, 8, 384, 7168), (3, 5, 7, 33), (17, 4, 6, 1000), (40, 9, 12, 64), (33, 64, 70, 40),
          (130, 2, 5, 2056)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["repeats", "none", "holes"])
@pytest.mark.parametrize("T,K,E,H", SHAPES)
def test_permute_and_gradient(k3, dev, T, K, E, H, kind, dtype):
    import torch
    idx = routing(T, K, E, kind, T + H)
    pos, pair, off = k3.moe_sort(torch.from_numpy(idx).to(dev), E)
    n = int(off[-1])
    x = rand((T, H), dtype, 1, dev)
    rows = torch.full((T * K, H), 7.0, dtype=x.dtype, device=dev)
    k3.moe_permute(x, pos, out=rows)
    assert torch.equal(rows[:n], x[(pair[:n] // K).long()])
    assert (rows[n:] == 7).all()                       # rows behind the last pair stay
    d = rand((T * K, H), dtype, 2, dev)
    got = k3.moe_permute_bwd(d, pos).double().cpu().numpy()
    dn, pn = d.double().cpu().numpy(), pos.cpu().numpy()
    for t in range(T):
        at = pn[t][pn[t] >= 0]
        want = dn[at].sum(0)
        lim = (len(at) + 1) * 2.0 ** -24 * np.abs(dn[at]).sum(0) + HALF[dtype] * np.abs(want)
        assert (np.abs(got[t] - want) <= lim).all()


@pytest.mark.parametrize("y_dtype,out_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("kind", ["repeats", "none", "holes"])
@pytest.mark.parametrize("T,K,E,H", SHAPES)
def test_unpermute_and_gradients(k3, dev, T, K, E, H, kind, y_dtype, out_dtype):
    import torch
    idx = routing(T, K, E, kind, T + H + 1)
    pos, _, off = k3.moe_sort(torch.from_numpy(idx).to(dev), E)
    n = int(off[-1])
    y = rand((T * K, H), y_dtype, 3, dev)
    y[n:] = float("nan")                               # nothing reads the rows behind the last pair
    wt = rand((T, K), "f32", 4, dev)
    wt[pos < 0] = float("nan")                         # nor a dropped pair's weight
    out = k3.moe_unpermute(y, pos, wt, out_dtype=torch_dtype(out_dtype)).double().cpu().numpy()
    dout = rand((T, H), out_dtype, 5, dev)
    dy = torch.full_like(y, 7.0)
    dwt = torch.full_like(wt, 7.0)
    k3.moe_unpermute_bwd(dout, y, pos, wt, dy=dy, dwt=dwt)
    assert (dy[n:] == 7).all()
    yn, wn, pn, dn = (a.double().cpu().numpy() for a in (y, wt, pos, dout))
    gy, gw = dy.double().cpu().numpy(), dwt.double().cpu().numpy()
    depth = -(-H // 256) * 8 + 13
    for t in range(T):
        on = pn[t] >= 0
        r = pn[t][on].astype(int)
        terms = wn[t][on][:, None] * yn[r]
        want = terms.sum(0)
        lim = (len(r) + 1) * 2.0 ** -24 * np.abs(terms).sum(0) + HALF[out_dtype] * np.abs(want)
        assert (np.abs(out[t] - want) <= lim).all()
        want = wn[t][on][:, None] * dn[t][None]
        assert (np.abs(gy[r] - want) <= (2.0 ** -24 + HALF[y_dtype]) * np.abs(want) + 1e-40).all()
        prod = yn[r] * dn[t][None]
        assert (np.abs(gw[t][on] - prod.sum(1)) <= depth * 2.0 ** -24 * np.abs(prod).sum(1)).all()
        assert (gw[t][~on] == 0).all()


def test_unpermute_keeps_the_order_of_the_sum(k3, dev):
    """fp32 rows and sums: products and additions rounded one by one in top-k order, bit for bit
    (the order of the MoE layers' combine, src/core/k3_ops.c:641-642)."""
    import torch
    T, K, E, H = 37, 8, 20, 516
    idx = routing(T, K, E, "distinct", 9)
    pos, _, _ = k3.moe_sort(torch.from_numpy(idx).to(dev), E)
    y, wt = rand((T * K, H), "f32", 1, dev), rand((T, K), "f32", 2, dev)
    got = k3.moe_unpermute(y, pos, wt).cpu().numpy()
    yn, wn, pn = y.cpu().numpy(), wt.cpu().numpy(), pos.cpu().numpy()
    want = np.zeros((T, H), np.float32)
    for j in range(K):
        want = want + wn[:, j:j + 1] * yn[pn[:, j]]
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_gradients_against_differences(k3, dev):
    """unpermute(permute(x)) is linear in x and in wt: a difference of two passes along a direction
    is the inner product with the gradient. fp32, so both sides carry about 1e-6 of the magnitudes'
    sum; steps of 1 make the differences as exact as the passes."""
    import torch
    T, K, E, H = 23, 4, 9, 136
    idx = routing(T, K, E, "holes", 5)
    pos, _, _ = k3.moe_sort(torch.from_numpy(idx).to(dev), E)
    x, v = rand((T, H), "f32", 1, dev), rand((T, H), "f32", 2, dev)
    wt, u = rand((T, K), "f32", 3, dev), rand((T, K), "f32", 4, dev)
    c = rand((T, H), "f32", 5, dev)

    def loss(x, wt):
        return (k3.moe_unpermute(k3.moe_permute(x, pos, out=torch.zeros((T * K, H), device=dev)), pos, wt).double()
                * c.double()).sum().item()

    rows = k3.moe_permute(x, pos, out=torch.zeros((T * K, H), device=dev))
    dy, dwt = k3.moe_unpermute_bwd(c, rows, pos, wt, dy=torch.zeros_like(rows))
    dx = k3.moe_permute_bwd(dy, pos)
    mag = (k3.moe_unpermute(k3.moe_permute(x.abs() + v.abs(), pos, out=torch.zeros((T * K, H), device=dev)), pos,
                            wt.abs() + u.abs()) * c.abs()).double().sum().item()
    lim = (2 * K + 16 + 8) * 2.0 ** -24 * mag
    assert abs((loss(x + v, wt) - loss(x - v, wt)) / 2 - (dx.double() * v.double()).sum().item()) <= lim
    assert abs((loss(x, wt + u) - loss(x, wt - u)) / 2 - (dwt.double() * u.double()).sum().item()) <= lim


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,K,E,H", [(1, 1, 1, 32), (1, 8, 384, 7168), (19, 3, 5, 96), (70, 8, 12, 2080)])
def test_permute_mxfp4_is_quant_then_permute(k3, dev, T, K, E, H, dtype):
    import torch
    idx = routing(T, K, E, "holes" if T > 1 else "repeats", H)
    pos, pair, off = k3.moe_sort(torch.from_numpy(idx).to(dev), E)
    n = int(off[-1])
    x = rand((T, H + 5 * (T > 1)), dtype, 1, dev)[:, :H]      # strided rows, not 16-byte aligned
    packed, scales = k3.moe_permute_mxfp4(x, pos)
    wp, ws = k3.mxfp4_quant(x)
    tok = (pair[:n] // K).long()
    assert torch.equal(packed[:n], wp[tok]) and torch.equal(scales[:n], ws[tok])


def test_no_tokens(k3, dev):
    import torch
    pos, pair, off = k3.moe_sort(torch.empty((0, 8), dtype=torch.int32, device=dev), 5)
    assert pos.shape == (0, 8) and pair.numel() == 0 and off.cpu().tolist() == [0] * 6
    x = torch.empty((0, 64), device=dev)
    assert k3.moe_permute(x, pos).shape == (0, 64)
    assert k3.moe_permute_bwd(torch.empty((0, 64), device=dev), pos).shape == (0, 64)
    assert k3.moe_permute_mxfp4(x, pos)[0].shape == (0, 32)
    wt = torch.empty((0, 8), device=dev)
    assert k3.moe_unpermute(x, pos, wt).shape == (0, 64)
    assert k3.moe_unpermute_bwd(x, x, pos, wt)[1].shape == (0, 8)


def test_captured_and_on_two_streams(k3, dev):
    """A captured sort + permute + unpermute replayed on new inputs, and two eager chains at once
    on streams of their own, give what one after another gives."""
    import torch
    T, K, E, H = 1500, 8, 40, 512
    def chain(idx, x, wt):
        pos, _, _ = k3.moe_sort(idx, E)
        return k3.moe_unpermute(k3.moe_permute(x, pos), pos, wt)

    def inputs(seed):
        return (torch.from_numpy(routing(T, K, E, "repeats", seed)).to(dev), rand((T, H), "bf16", seed, dev),
                rand((T, K), "f32", seed + 1, dev))
    a, b = inputs(1), inputs(2)
    want_a, want_b = chain(*a), chain(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = {}
    for _ in range(5):
        with torch.cuda.stream(s1):
            got["a"] = chain(*a)
        with torch.cuda.stream(s2):
            got["b"] = chain(*b)
    torch.cuda.synchronize()
    assert torch.equal(got["a"], want_a) and torch.equal(got["b"], want_b)
    held = [t.clone() for t in a]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = chain(*held)
    for src, want in ((b, want_b), (a, want_a)):
        for h, t in zip(held, src):
            h.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_outputs_may_not_be_inputs(k3, dev):
    import torch
    pos = torch.arange(6, dtype=torch.int32, device=dev).view(6, 1)
    x, wt = torch.randn(6, 32, device=dev), torch.ones(6, 1, device=dev)
    for call in (lambda: k3.moe_permute(x, pos, out=x), lambda: k3.moe_permute_bwd(x, pos, out=x),
                 lambda: k3.moe_unpermute(x, pos, wt, out=x), lambda: k3.moe_unpermute_bwd(x, x.clone(), pos, wt, dy=x),
                 lambda: k3.moe_unpermute_bwd(x, x.clone(), pos, wt, dwt=wt)):
        with pytest.raises(k3.K3CError, match="may not be an input"):
            call()


def test_offsets_past_32_bits(k3, dev):
    """Rows more than 4 GiB from the first: 40000 x 8 rows of 14336 bytes."""
    import torch
    T, K, E, H = 40000, 8, 3, 7168
    g = torch.Generator(device=dev).manual_seed(1)
    idx = torch.randint(0, E, (T, K), generator=g, device=dev, dtype=torch.int32)
    x = torch.randn(T, H, generator=g, device=dev).bfloat16()
    pos, pair, off = k3.moe_sort(idx, E)
    rows = k3.moe_permute(x, pos)
    last = pair[-2000:].long()
    assert torch.equal(rows[-2000:], x[last // K])
    assert torch.equal(rows[pos[::997].long()], x[::997].unsqueeze(1).expand(-1, K, -1))
    wt = torch.full((T, K), 0.125, device=dev)          # eight equal rows: exact
    assert torch.equal(k3.moe_unpermute(rows, pos, wt), x)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("first,pad", [(0, 8), (0, 3), (1, 7), (8, 0)])
def test_permute_of_strided_rows(k3, dev, first, pad, dtype):
    """x as a slice of wider rows: aligned and odd strides and bases."""
    import torch
    T, K, E, H = 50, 3, 6, 72
    pos, pair, off = k3.moe_sort(torch.from_numpy(routing(T, K, E, "holes", 8)).to(dev), E)
    n = int(off[-1])
    x = rand((T, first + H + pad), dtype, 1, dev)[:, first:first + H]
    assert torch.equal(k3.moe_permute(x, pos)[:n], x[(pair[:n] // K).long()])


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_gradient_of_the_sum_alone(k3, dev, dtype, first):
    """k3c_moe_unpermute_bwd with dy or dwt left out gives the other as with both (y is not read
    without dwt); rows on odd addresses (first = 1) and a width no vector divides among them."""
    import torch
    L, st = k3.lib(), torch.cuda.current_stream(dev).cuda_stream
    code = {"bf16": k3.K3C_BF16, "f32": k3.K3C_F32}[dtype]
    T, K, E = 21, 5, 9
    pos, _, _ = k3.moe_sort(torch.from_numpy(routing(T, K, E, "holes", 4)).to(dev), E)
    wt = rand((T, K), "f32", 6, dev)
    for H in (64, 4097):
        def odd(rows, seed):
            return rand((rows * H + first,), dtype, seed, dev)[first:].view(rows, H)
        y, dout = odd(T * K, 7), odd(T, 8)
        both = [torch.full_like(y, 3.0), torch.full((T, K), 3.0, device=dev)]
        k3.moe_unpermute_bwd(dout, y, pos, wt, dy=both[0], dwt=both[1])
        dy, dwt = odd(T * K, 9).fill_(3.0), torch.full((T, K), 3.0, device=dev)
        for a, b, yy in ((dy, None, None), (None, dwt, y)):
            rc = L.k3c_moe_unpermute_bwd(*(None if t is None else t.data_ptr() for t in (a, b)), dout.data_ptr(), code,
                                         None if yy is None else yy.data_ptr(), code, wt.data_ptr(), pos.data_ptr(), T, K, H, st)
            assert rc == 0
        assert torch.equal(dy, both[0])
        # the sums' split over threads goes with the width alone, but not over vectors and elements
        want = (dout[:, None].double() * y[pos.clamp(min=0).long()].double())
        lim = (H // 256 * 8 + 32) * 2.0 ** -24 * want.abs().sum(-1) * (pos >= 0)
        assert ((dwt.double() - want.sum(-1) * (pos >= 0)).abs() <= lim).all()


@pytest.mark.parametrize("n", [0, 2049, -(1 << 32) + 2048, (1 << 32) + 1])
def test_expert_counts_the_sort_refuses(k3, dev, n):
    import torch
    with pytest.raises(k3.K3CError, match="n_experts"):
        k3.moe_sort(torch.zeros((4, 2), dtype=torch.int32, device=dev), n)
    assert k3.moe_sort(torch.zeros((4, 2), dtype=torch.int32, device=dev), 2048)[2].shape == (2049,)


def test_outputs_may_not_overlap_inputs(k3, dev):
    """A result that shares part of its memory with any input is refused, one that lies beside them in
    the same buffer is not."""
    import torch
    T, K, H = 6, 2, 32
    buf = torch.zeros(4 * T * K * H, device=dev)
    pos = torch.arange(T * K, dtype=torch.int32, device=dev).view(T, K)
    wt = torch.ones(T, K, device=dev)

    def at(first, rows, cols=H):
        return buf[first:first + rows * cols].view(rows, cols)

    n, one = T * K * H, T * H
    ip = pos.view(torch.float32)
    for call in (lambda: k3.moe_permute(at(n - 1, T), pos, out=at(0, T * K)),
                 lambda: k3.moe_permute(at(0, T), pos, out=at(one - 1, T * K)),
                 lambda: k3.moe_permute(buf[:T * 2 * H].view(T, 2 * H)[:, H:], pos, out=at(H, T * K)),
                 lambda: k3.moe_permute_bwd(at(one - 1, T * K), pos, out=at(0, T)),
                 lambda: k3.moe_unpermute(at(H, T * K), pos, wt, out=at(0, T)),
                 lambda: k3.moe_unpermute(at(0, T * K), pos, at(n + 3, T, K), out=at(n, T)),
                 lambda: k3.moe_unpermute(torch.zeros(T * K, K, device=dev), pos, wt, out=ip),
                 lambda: k3.moe_unpermute_bwd(at(0, T), at(one, T * K), pos, wt, dy=at(one + n - 1, T * K)),
                 lambda: k3.moe_unpermute_bwd(at(0, T), at(one, T * K), pos, wt, dwt=at(one - 1, T, K)),
                 lambda: k3.moe_unpermute_bwd(at(0, T), at(one, T * K), pos, wt, dy=at(one + n, T * K), dwt=at(one + 2 * n - 2, T, K))):
        with pytest.raises(k3.K3CError, match="may not be an input"):
            call()
    x = torch.randn(T, H, device=dev)
    wide = torch.zeros(T * K, 4 * H, device=dev)     # side by side
    at(0, T).copy_(x)
    assert torch.equal(k3.moe_permute(at(0, T), pos, out=at(one, T * K)), x.repeat_interleave(K, 0))
    src = wide[:T, H:2 * H]
    src.copy_(x)
    assert torch.equal(k3.moe_permute(src, pos, out=at(one, T * K)), x.repeat_interleave(K, 0))
    gap = buf[:2 * T * 2 * K * H].view(T, 4 * K * H)       # x's rows in the first columns, one token's rows behind them
    gap[:1, :H].copy_(x[:1])
    assert torch.equal(k3.moe_permute(gap[:2, :H][:1], pos[:1], out=gap.view(-1)[H:H + K * H].view(K, H)), x[:1].repeat_interleave(K, 0))


@pytest.mark.parametrize("kind", ["missing", "other arguments", "another result"])
def test_results_without_the_short_allocation(k3, dev, kind, monkeypatch):
    """torch's private short way to a new tensor missing or changed: results come from its public one."""
    import torch
    guards = torch._C._dynamo.guards
    if kind == "missing":
        monkeypatch.delattr(guards, "_empty_strided_cuda", raising=False)
    else:
        def other(size, stride, dtype, *more):
            if kind == "other arguments":
                raise TypeError("four arguments")
            return torch.empty(size)
        monkeypatch.setattr(guards, "_empty_strided_cuda", other, raising=False)
    monkeypatch.setattr(k3, "_rt", k3._Runtime())
    idx = torch.tensor([[1, 0], [1, 5]], dtype=torch.int32, device=dev)
    pos, pair, off = k3.moe_sort(idx, 2)
    assert pos.tolist() == [[1, 0], [2, -1]] and pair.tolist() == [1, 0, 2, -1] and off.tolist() == [0, 1, 3]


def test_the_most_pairs(k3, dev):
    """As many pairs as 32 bits allow, with rows of one element: pair p goes to expert p % 3 - 1, the
    first third of them nowhere."""
    import torch
    torch.cuda.empty_cache()
    K, E = 8, 2
    T = ((1 << 31) - (1 << 19) - 1) // K
    P = T * K
    idx = torch.arange(P, dtype=torch.int32, device=dev).remainder_(3).sub_(1).view(T, K)
    pos, pair, off = k3.moe_sort(idx, E)
    n = [(P - e - 1 + 2) // 3 for e in range(E)]
    assert off.tolist() == [0, n[0], n[0] + n[1]]
    pos = pos.view(-1)
    x = (torch.arange(T, dtype=torch.int32, device=dev) % 251).bfloat16().view(T, 1)
    rows = k3.moe_permute(x, pos.view(T, K))
    out = k3.moe_permute_bwd(rows, pos.view(T, K))
    for lo in range(0, P, 1 << 27):
        p = torch.arange(lo, min(lo + (1 << 27), P), dtype=torch.int32, device=dev)
        e = p % 3 - 1
        want = torch.where(e < 0, -1, p // 3 + torch.where(e == 1, n[0], 0))
        assert torch.equal(pos[p[0]:p[-1] + 1], want)
        live = want >= 0
        assert torch.equal(pair[want[live].long()], p[live])
        assert torch.equal(rows.view(-1)[want[live].long()], x.view(-1)[(p[live] // K).long()])
        t = p[::K] // K
        held = (idx.view(-1)[lo:lo + p.numel()].view(-1, K) >= 0).sum(1)
        assert torch.equal(out.view(-1)[t[0]:t[-1] + 1], (x.view(-1)[t[0]:t[-1] + 1].float() * held).bfloat16())
    assert (pair[n[0] + n[1]:] == -1).all()
    with pytest.raises(k3.K3CError, match="32 bits"):
        k3.moe_sort(torch.empty((T + 1, K), dtype=torch.int32, device=dev), E)
    del idx, pos, pair, rows, out, x
    torch.cuda.empty_cache()


def test_two_threads(k3, dev):
    """Threads with streams of their own, each through all the calls, get what one alone does."""
    import threading
    import torch
    T, K, E, H, N = 700, 4, 19, 96, 72
    g = torch.Generator(device=dev).manual_seed(5)
    codes = torch.randint(0, 256, (E, N, H // 2), dtype=torch.uint8, device=dev, generator=g)
    W = k3.Mxfp4Mat(*k3.mxfp4_pack(codes, torch.randint(118, 125, (E, N, H // 32), dtype=torch.uint8, device=dev, generator=g)))

    def layer(idx, x, wt):
        pos, _, off = k3.moe_sort(idx, E)
        y = k3.mxfp4_mm(*k3.moe_permute_mxfp4(x, pos), W, off=off)
        out = k3.moe_unpermute(y, pos, wt)
        dy, dwt = k3.moe_unpermute_bwd(out, y, pos, wt)
        return out, dwt, k3.moe_permute_bwd(k3.mxfp4_mm_bwd(dy, W, off=off), pos)

    ins = [(torch.randint(0, E, (T, K), device=dev, generator=g, dtype=torch.int32), torch.randn(T, H, device=dev, generator=g),
            torch.rand(T, K, device=dev, generator=g)) for _ in range(4)]
    want = [layer(*i) for i in ins]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = layer(*ins[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
