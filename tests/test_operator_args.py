"""Refusals of the sort / permute / MXFP4-product entry points, without a GPU: the C functions
validate before any CUDA call, and the Python wrappers refuse tensors of the wrong type, shape,
layout or place."""
import ctypes as C

import pytest

BUF = 1 << 20            # an aligned address nothing dereferences


def err(k3):
    return k3.lib().k3c_last_error().decode()


def mat(k3, **kw):
    d = dict(codes=BUF, atoms=BUF, code_stride=64 * 16, atom_stride=512, n_mats=1, rows=64, in_=32, mat_of=None)
    d.update(kw)
    return k3.Mxfp4MatC(*(d[n] for n in ("codes", "atoms", "code_stride", "atom_stride", "n_mats", "rows", "in_", "mat_of")))


def test_sort_refusals(k3):
    L = k3.lib()
    for args, word in (((BUF, BUF, BUF, BUF, -1, 8, 4, None, 0, None), "ntok"),
                       ((BUF, BUF, BUF, BUF, 4, 0, 4, None, 0, None), "topk"),
                       ((BUF, BUF, BUF, BUF, 4, 65, 4, None, 0, None), "topk"),
                       ((BUF, BUF, BUF, BUF, 4, 8, 0, None, 0, None), "n_experts"),
                       ((BUF, BUF, BUF, BUF, 4, 8, 2049, None, 0, None), "n_experts"),
                       ((BUF, BUF, BUF, BUF, 1 << 30, 8, 4, None, 0, None), "32 bits"),
                       ((None, BUF, BUF, BUF, 4, 8, 4, None, 0, None), "NULL"),
                       ((BUF, BUF, None, BUF, 0, 8, 4, None, 0, None), "NULL"),
                       ((BUF, BUF, BUF, BUF, 4096, 8, 4, None, 0, None), "scratch"),
                       ((BUF, BUF, BUF, BUF, 4096, 8, 4, BUF, 8, None), "scratch"),
                       ((BUF, BUF, BUF, BUF, 4096, 8, 4, BUF + 1, 1 << 20, None), "scratch")):
        assert L.k3c_moe_sort(*args) == -1 and word in err(k3), (args, err(k3))
    assert L.k3c_moe_sort_scratch(16, 8, 384) == 0
    assert L.k3c_moe_sort_scratch(1024, 8, 384) == 0
    assert L.k3c_moe_sort_scratch(4096, 8, 384) == 16 * 384 * 4
    assert L.k3c_moe_sort_scratch(-1, 8, 384) == 0


def test_permute_refusals(k3):
    L = k3.lib()
    assert L.k3c_moe_permute(BUF, BUF, 2, 64, BUF, 4, 2, 64, None) == -1 and "dtype" in err(k3)
    assert L.k3c_moe_permute(BUF, BUF, 0, 63, BUF, 4, 2, 64, None) == -1 and "ldx" in err(k3)
    assert L.k3c_moe_permute(BUF, BUF, 0, 64, BUF, 4, 2, 0, None) == -1 and "hidden" in err(k3)
    assert L.k3c_moe_permute(None, BUF, 0, 64, BUF, 4, 2, 64, None) == -1 and "NULL" in err(k3)
    assert L.k3c_moe_permute_bwd(BUF, BUF, 7, BUF, 4, 2, 64, None) == -1 and "dtype" in err(k3)
    assert L.k3c_moe_permute_bwd(BUF, BUF, 0, None, 4, 2, 64, None) == -1 and "NULL" in err(k3)
    assert L.k3c_moe_permute_mxfp4(BUF, BUF, BUF, 0, 48, BUF, 4, 2, 48, None) == -1 and "multiple of 32" in err(k3)
    assert L.k3c_moe_permute_mxfp4(BUF + 8, BUF, BUF, 0, 64, BUF, 4, 2, 64, None) == -1 and "aligned" in err(k3)
    assert L.k3c_moe_unpermute(BUF, 0, BUF, 3, BUF, BUF, 4, 2, 64, None) == -1 and "dtype" in err(k3)
    assert L.k3c_moe_unpermute(BUF, 0, BUF, 0, None, BUF, 4, 2, 64, None) == -1 and "NULL" in err(k3)
    assert L.k3c_moe_unpermute_bwd(BUF, BUF, BUF, 0, None, 0, BUF, BUF, 4, 2, 64, None) == -1 and "NULL" in err(k3)
    assert L.k3c_moe_unpermute_bwd(BUF, BUF, BUF, -1, BUF, 0, BUF, BUF, 4, 2, 64, None) == -1 and "dtype" in err(k3)


def test_quant_and_pack_refusals(k3):
    L = k3.lib()
    assert L.k3c_mxfp4_quant(BUF, BUF, BUF, 0, 33, 4, 33, None) == -1 and "even" in err(k3)
    assert L.k3c_mxfp4_quant(BUF, BUF, BUF, 0, 32, 4, 34, None) == -1 and "ldx" in err(k3)
    assert L.k3c_mxfp4_quant(BUF, BUF, BUF, 9, 32, 4, 32, None) == -1 and "dtype" in err(k3)
    assert L.k3c_mxfp4_quant(BUF, BUF, None, 0, 32, 4, 32, None) == -1 and "NULL" in err(k3)
    assert L.k3c_mxfp4_pack(BUF, BUF, BUF, BUF, 1, 4, 48, None) == -1 and "multiple of 32" in err(k3)
    assert L.k3c_mxfp4_pack(BUF, BUF, BUF, BUF, 0, 4, 64, None) == -1 and "n_mats" in err(k3)
    assert L.k3c_mxfp4_pack(BUF + 4, BUF, BUF, BUF, 1, 4, 64, None) == -1 and "aligned" in err(k3)
    assert L.k3c_mxfp4_atom_bytes(129, 160) == 4 * 512 and L.k3c_mxfp4_atom_bytes(0, 32) == 0


def test_mm_refusals(k3):
    L = k3.lib()

    def mm(W, y=BUF, dt=0, ldy=64, a=BUF, M=4, off=None, G=1):
        return L.k3c_mxfp4_mm(y, dt, ldy, a, BUF, M, None if W is None else C.byref(W), off, G, None)

    def bwd(W, da=BUF, dt=0, ld=64, dy=BUF, lddy=64, M=4, off=None, G=1):
        return L.k3c_mxfp4_mm_bwd(da, dt, ld, dy, lddy, M, None if W is None else C.byref(W), off, G, None)

    for f in (mm, bwd):
        for W, word in ((None, "matrix"), (mat(k3, in_=48), "multiple of 32"), (mat(k3, rows=0), "rows"),
                        (mat(k3, codes=BUF + 8), "aligned"), (mat(k3, n_mats=2, atom_stride=520), "aligned"),
                        (mat(k3, n_mats=2, code_stride=512), "strides"), (mat(k3, n_mats=0), "n_mats")):
            assert f(W) == -1 and word in err(k3), (word, err(k3))
        assert f(mat(k3), M=-1) == -1 and "M=" in err(k3)
        assert f(mat(k3), G=2) == -1 and "n_groups" in err(k3)
        assert f(mat(k3), off=BUF, G=0) == -1 and "n_groups" in err(k3)
        assert f(mat(k3, n_mats=2000, mat_of=BUF), off=BUF, G=1025) == -1 and "n_groups" in err(k3)
        assert f(mat(k3), off=BUF, G=2) == -1 and "matrices" in err(k3)
        assert f(mat(k3), dt=4) == -1 and "dtype" in err(k3)
        assert f(mat(k3), M=0) == 0
    assert mm(mat(k3), ldy=63) == -1 and "ldy" in err(k3)
    assert mm(mat(k3), a=BUF + 8) == -1 and "aligned" in err(k3)
    assert mm(mat(k3), y=None) == -1 and "NULL" in err(k3)
    assert bwd(mat(k3), ld=31) == -1 and "ldda" in err(k3)
    assert bwd(mat(k3), lddy=60) == -1 and "lddy" in err(k3)
    assert bwd(mat(k3), lddy=68) == -1 and "lddy" in err(k3)
    assert bwd(mat(k3), dy=BUF + 2) == -1 and "aligned" in err(k3)


def test_wrappers_refuse(k3):
    import torch
    i32, f = torch.zeros((4, 2), dtype=torch.int32), torch.zeros((4, 64))
    for call in (lambda: k3.moe_sort(i32, 8),                       # not on a GPU
                 lambda: k3.moe_sort(i32.long(), 8), lambda: k3.moe_sort(i32[0], 8),
                 lambda: k3.moe_permute(f, i32), lambda: k3.moe_permute(f.half(), i32),
                 lambda: k3.moe_permute_bwd(f, i32), lambda: k3.moe_permute_mxfp4(f, i32),
                 lambda: k3.moe_unpermute(f, i32, f[:, :2]), lambda: k3.moe_unpermute_bwd(f, f, i32, f),
                 lambda: k3.mxfp4_quant(f), lambda: k3.mxfp4_quant(f.double()),
                 lambda: k3.mxfp4_pack(f, f), lambda: k3.Mxfp4Mat(f, f)):
        with pytest.raises(k3.K3CError):
            call()


def test_extents_past_32_bits_are_refused(k3):
    """Extents that the C arguments could not hold are refused, not cut; and those whose sums with a
    tile's would not fit."""
    import torch
    L = k3.lib()
    big = (1 << 31) + 32
    for rows, n in ((big, 32), (1, big), (big, 2)):
        t = torch.empty((rows, n), dtype=torch.bfloat16, device="meta")
        for f in (lambda: k3._rows_arg(t, "x", -1, (torch.bfloat16,)), lambda: k3._mat_arg(t, "x", -1, (torch.bfloat16,))):
            with pytest.raises(k3.K3CError, match="32 bits"):
                f()
        assert k3._rows_arg(t[:5, :2], "x", -1, (torch.bfloat16,))[:2] == (min(rows, 5), 2)
    top = (1 << 31) - 1024
    assert L.k3c_mxfp4_mm(BUF, 0, 64, BUF, BUF, top + 1, C.byref(mat(k3)), None, 1, None) == -1 and "M=" in err(k3)
    assert L.k3c_mxfp4_mm_bwd(BUF, 0, 64, BUF, 64, top + 1, C.byref(mat(k3)), None, 1, None) == -1 and "M=" in err(k3)
    for kw in (dict(rows=top + 1), dict(in_=top + 32)):
        assert L.k3c_mxfp4_mm(BUF, 0, top + 64, BUF, BUF, 4, C.byref(mat(k3, **kw)), None, 1, None) == -1 and "matrix" in err(k3)
    assert L.k3c_mxfp4_quant(BUF, BUF, BUF, 0, top + 32, 1, top + 2, None) == -1 and "in=" in err(k3)
    assert L.k3c_mxfp4_pack(BUF, BUF, BUF, BUF, 1, top + 1, 32, None) == -1 and "rows=" in err(k3)
    # more tiles than 32 bits count: 2^31 - 2^12 rows times as many columns
    n = (1 << 31) - 4096
    assert L.k3c_mxfp4_mm(BUF, 0, n, BUF, BUF, n, C.byref(mat(k3, rows=n)), None, 1, None) == -1 and "tiles" in err(k3)
    assert L.k3c_mxfp4_mm_bwd(BUF, 0, n, BUF, 64, n, C.byref(mat(k3, in_=n)), None, 1, None) == -1 and "tiles" in err(k3)


def test_mat_struct_layout_matches_header(k3, tmp_path):
    import os
    import subprocess
    from conftest import ROOT
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "k3c.h"\nint main(void) { printf("%zu %zu %zu %zu\\n",'
                   ' sizeof(k3c_mxfp4_mat), offsetof(k3c_mxfp4_mat, code_stride), offsetof(k3c_mxfp4_mat, rows),'
                   ' offsetof(k3c_mxfp4_mat, mat_of)); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True).stdout.split()]
    m = k3.Mxfp4MatC
    assert got == [C.sizeof(m), m.code_stride.offset, m.rows.offset, m.mat_of.offset]


@pytest.mark.parametrize("n", [0, -1, 2049, 1 << 31, (1 << 32) + 4, -(1 << 32) + 2048, -(1 << 33) + 1, 1 << 64])
def test_sort_refuses_expert_counts_before_it_allocates(k3, n):
    """Counts outside 1..2048, those among them that 32 bits would cut to one inside: off is as
    long as the count given, the entry point would write as many as the count it sees."""
    import torch
    with pytest.raises(k3.K3CError, match="n_experts"):
        k3.moe_sort(torch.zeros((4, 2), dtype=torch.int32), n)


def test_memory_in_common_is_found():
    """_share against the sets of bytes themselves: contiguous pieces, rows of one stride (slices of
    one buffer, side by side or one inside the other) and of two."""
    import random
    import __graft_entry__ as ge
    k3 = ge.load_package()
    rng = random.Random(1)

    def bytes_of(t):
        p, r, w, s = t
        return {p + i * s + j for i in range(r) for j in range(w)}
    met = [0, 0]
    for _ in range(4000):
        s = rng.randint(1, 12)
        two = []
        for _ in range(2):
            if rng.random() < 0.4:
                s = rng.randint(1, 12)
            two.append((rng.randint(0, 40), rng.randint(0, 5), rng.randint(0, s), s))
        want = bool(bytes_of(two[0]) & bytes_of(two[1]))
        assert k3._share(*two) == want and k3._share(*two[::-1]) == want, two
        met[want] += 1
        if want:
            with pytest.raises(k3.K3CError, match="may not be an input"):
                k3._apart("out", two[0], (10 ** 6, 1, 4, 4), two[1])
        else:
            k3._apart("out", *two)
    assert min(met) > 500


def test_tensors_that_require_grad_are_refused(k3):
    """In gradient mode, whose record would lack them; not where it is off, as in autograd functions."""
    import torch
    t = torch.zeros((4, 6), requires_grad=True)
    for f in (lambda: k3._mat_arg(t, "x", -1, (torch.float32,)), lambda: k3._rows_arg(t, "x", -1, (torch.float32,)),
              lambda: k3._rows_arg(t[:, :3], "x", -1, (torch.float32,))):
        with pytest.raises(k3.K3CError, match="x: requires grad"):
            f()
        with torch.no_grad():
            assert f()[0] == 4


def test_lengths_of_vectors(k3):
    """off and mat_of hold 1 element to 2^31 - 1: the entry points take an empty one, whose address is
    NULL, for none (every group its own matrix), and cut a longer one's length."""
    import torch
    for n in (0, 1 << 31, (1 << 32) + 3):
        with pytest.raises(k3.K3CError, match="mat_of.*32 bits"):
            k3._vec_arg(torch.empty(n, dtype=torch.int32, device="meta"), "mat_of", -1, torch.int32)
    assert k3._vec_arg(torch.empty(5, dtype=torch.int32, device="meta"), "mat_of", -1, torch.int32) == 5


# Each wrapper's valid call, and per tensor the defects that its own check has to find: another type,
# another rank, one more row or column, elements or rows that are not as they have to lie.
T, K, E, H, ROWS, IN, M = 4, 2, 3, 64, 6, 64, 5
PAIRS = {"x": ("f32", T, H), "pos": ("i32", T, K), "wt": ("f32", T, K), "y": ("f32", T * K, H), "drows": ("f32", T * K, H),
         "dout": ("bf16", T, H), "dy": ("f32", T * K, H), "dwt": ("f32", T, K)}
ANY = "type rank stride"                 # extents that this argument itself sets
OWN = ANY + " rows cols"
CALLS = {
    "moe_sort": (dict(idx=("i32", T, K)), (E,), dict(idx=ANY)),
    "moe_permute": (dict(x=PAIRS["x"], pos=PAIRS["pos"], out=("f32", T * K, H)), (),
                    dict(x=ANY + " overlap", pos=ANY + " rows", out=OWN)),
    "moe_permute_bwd": (dict(drows=PAIRS["drows"], pos=PAIRS["pos"], out=("f32", T, H)), (),
                        dict(drows=ANY + " rows", pos=ANY, out=OWN)),
    "moe_permute_mxfp4": (dict(x=PAIRS["x"], pos=PAIRS["pos"]), (), dict(x=ANY + " overlap", pos=ANY + " rows")),
    "moe_unpermute": (dict(y=PAIRS["y"], pos=PAIRS["pos"], wt=PAIRS["wt"], out=("bf16", T, H)), (),
                      dict(y=ANY + " rows", pos=ANY, wt=OWN, out=OWN)),
    "moe_unpermute_bwd": (dict(dout=PAIRS["dout"], y=PAIRS["y"], pos=PAIRS["pos"], wt=PAIRS["wt"], dy=PAIRS["dy"],
                               dwt=PAIRS["dwt"]), (),
                          dict(dout=OWN, y=ANY + " rows", pos=ANY, wt=OWN, dy=OWN, dwt=OWN)),
    "mxfp4_quant": (dict(x=("bf16", M, IN)), (), dict(x=ANY + " overlap")),
    "mxfp4_pack": (dict(packed=("u8", 2, ROWS, IN // 2), scales=("u8", 2, ROWS, IN // 32)), (),
                   dict(packed="type rank stride", scales="type rank stride rows cols mats")),
    "Mxfp4Mat": (dict(codes=("u8", 2, ROWS, IN // 2), atoms=("u8", 2, 1, 1, 512), mat_of=("i32", 4)), (),
                 dict(codes="type rank stride", atoms="type rank stride rows cols mats", mat_of="type rank stride")),
    "mxfp4_mm": (dict(a=("u8", M, IN // 2), a_scales=("u8", M, IN // 32), W=None, off=("i32", 3), out=("bf16", M, ROWS)), (),
                 dict(a=ANY + " cols", a_scales=OWN, off="type rank stride cols", out=OWN + " overlap")),
    "mxfp4_mm_bwd": (dict(dy=("bf16", M, ROWS), W=None, off=("i32", 3), out=("f32", M, IN)), (),
                     dict(dy=ANY + " cols overlap", off="type rank stride cols", out=OWN + " overlap")),
}
CASES = [(f, a, d) for f, (_, _, own) in CALLS.items() for a, ds in own.items() for d in ds.split()]


def one_defect(torch, dev, spec, defect):
    """A tensor of the spec with one defect, or None of them."""
    types = {"f32": torch.float32, "bf16": torch.bfloat16, "i32": torch.int32, "u8": torch.uint8}
    other = {"f32": torch.float16, "bf16": torch.float64, "i32": torch.int64, "u8": torch.int8}
    name, *shape = spec
    dt = types[name]
    if defect == "type":
        dt = other[name]
    elif defect == "rank":
        shape.append(1)
    elif defect in ("rows", "cols", "mats"):
        shape[{"rows": max(len(shape) - 2, 0), "cols": len(shape) - 1, "mats": 0}[defect]] += 1
    if defect == "stride":
        return torch.zeros(*shape[:-1], 2 * shape[-1], dtype=dt, device=dev)[..., ::2]
    if defect == "overlap":
        return torch.zeros(1, shape[-1], dtype=dt, device=dev).expand(*shape)
    return torch.zeros(*shape, dtype=dt, device=dev)


def refused(k3, torch, dev, case, monkeypatch):
    """The call with that one defect raises by the argument's name, and reaches no entry point; the
    same call without it does."""
    fn, arg, defect = case
    specs, rest, _ = CALLS[fn]
    launched = []

    def kept(n, *a):
        launched.append(n)
    monkeypatch.setattr(k3, "_launch", lambda rt, name, *a: kept(name))
    W = k3.Mxfp4Mat(*(one_defect(torch, dev, s, None) for s in (("u8", 2, ROWS, IN // 2), ("u8", 2, 1, 1, 512))))

    def call(bad):
        args = {n: W if s is None else one_defect(torch, dev, s, defect if n == bad else None) for n, s in specs.items()}
        if fn == "mxfp4_mm" and bad == "off" and defect == "cols":
            assert args["off"].shape == (4,)               # three groups, two matrices
        return getattr(k3, fn)(*list(args.values())[:1], *rest, **dict(list(args.items())[1:]))
    with pytest.raises(k3.K3CError, match=f"^{arg}: "):
        call(arg)
    assert not launched
    call(None)
    assert launched or fn == "Mxfp4Mat"


@pytest.mark.parametrize("case", CASES, ids="-".join)
def test_one_defect_is_refused_by_name(k3, case, monkeypatch):
    """On the CPU: the wrappers with tensors and a runtime of no device."""
    import types
    import torch
    rt = types.SimpleNamespace(
        torch=torch, lib=None, floats=(torch.float32, torch.bfloat16), code={torch.float32: 0, torch.bfloat16: 1},
        size={torch.float32: 4, torch.bfloat16: 2}, i32=torch.int32, u8=torch.uint8, f32=torch.float32, device=lambda: -1,
        empty=lambda size, stride, dtype: torch.empty_strided(size, stride, dtype=dtype))
    monkeypatch.setattr(k3, "_runtime", lambda t: rt)
    refused(k3, torch, "cpu", case, monkeypatch)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids="-".join)
def test_one_defect_is_refused_by_name_on_a_gpu(k3, case, monkeypatch):
    import torch
    refused(k3, torch, "cuda", case, monkeypatch)


@pytest.mark.gpu
@pytest.mark.parametrize("fn,arg", [(f, a) for f, (s, _, _) in CALLS.items() for a in list(s)[1:] if s[a]])
def test_a_tensor_elsewhere_is_refused(k3, fn, arg, monkeypatch):
    """The first argument on the GPU, one of the others on the CPU."""
    import torch
    monkeypatch.setattr(k3, "_launch", lambda *a: pytest.fail("launched"))
    W = k3.Mxfp4Mat(*(one_defect(torch, "cuda", s, None) for s in (("u8", 2, ROWS, IN // 2), ("u8", 2, 1, 1, 512))))
    specs, rest, _ = CALLS[fn]
    args = {n: W if s is None else one_defect(torch, "cpu" if n == arg else "cuda", s, None) for n, s in specs.items()}
    with pytest.raises(k3.K3CError, match=f"^{arg}: |a CUDA tensor expected"):    # y leads moe_unpermute_bwd
        getattr(k3, fn)(*list(args.values())[:1], *rest, **dict(list(args.items())[1:]))


def test_a_gpu_is_asked_for(k3):
    import torch
    for t in (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)):
        with pytest.raises(k3.K3CError, match="a CUDA tensor expected"):
            k3._runtime(t)


def test_products_tests_reach_every_tile(k3):
    """The sizes of the products' GPU tests take all four tile shapes of each product, dense and
    grouped: a changed rule that leaves one of them untested shows here."""
    import test_gpu_mxfp4_mm as mm
    L = k3.lib()

    def tile(*a):
        return divmod(L.k3c_mxfp4_mm_tile(*a), 65536)
    dense, grouped = mm.DENSE, [(s, n, k) for s, n, k, *_ in mm.TILED]
    both = {0: {(256, 256), (128, 256), (128, 128), (128, 64)}, 1: {(512, 256), (256, 256), (128, 256), (128, 128)}}
    more = [(128, 200, 60000), (300, 136, 19232)]      # the gradient's own
    for gradient in (0, 1):
        assert {tile(m, 1, 0, n, k, gradient) for m, n, k in dense + more * gradient} == both[gradient]
        assert {tile(sum(s), len(s), 1, n, k, gradient) for s, n, k in grouped} == both[gradient]
    for bad in ((0, 1, 0, 64, 64, 0), (4, 0, 0, 64, 64, 0), (4, 1025, 1, 64, 64, 0), (4, 1, 0, 0, 64, 0), (4, 1, 0, 64, 16, 1)):
        assert L.k3c_mxfp4_mm_tile(*bad) == -1 and "mxfp4_mm_tile" in err(k3)
