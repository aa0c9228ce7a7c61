"""Norm and rotation, the paged MX cache and attention over it, against plain 64-bit forms (serving_plain.py)."""
import importlib.util
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import serving_plain as P  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(t):
    return torch.finfo(t).eps / 2


def rnd(g, *shape, dtype=BF16, amp=1.0):
    return (torch.randn(*shape, generator=g) * amp).to(dtype)


def laid_out(x, layout, how="dense"):
    """CPU tensor [B,H,L,D] -> the CUDA tensor a caller passes for `layout`, in memory as `how` says."""
    B, H, L, D = x.shape
    y = x if layout == "HND" else x.transpose(1, 2)
    if how == "dense":
        return y.contiguous().cuda()
    if how == "padded":                      # rows with a gap behind them
        z = torch.full((*y.shape[:-1], D + 16), float("nan"), dtype=x.dtype, device="cuda")[..., :D]
    elif how == "transposed":                # the other layout's memory
        z = torch.empty_like(y.transpose(1, 2).contiguous(), device="cuda").transpose(1, 2)
    elif how == "shifted":                   # a base that is off by one element
        z = torch.empty(y.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(y.shape)
    elif how == "odd":                       # rows of an odd pitch
        z = torch.empty((*y.shape[:-1], D + 1), dtype=x.dtype, device="cuda")[..., :D]
    elif how == "strided":                   # every second element
        z = torch.empty((*y.shape[:-1], 2 * D), dtype=x.dtype, device="cuda")[..., ::2]
    z.copy_(y.cuda())
    return z


def logical(y, layout):
    return (y if layout == "HND" else y.transpose(1, 2)).cpu()


# ------------------------------------------------------------------------------------------------------- norm and rotation
def _angles(rows, half):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return ang.cos().float(), ang.sin().float()


ROPE = [
    # B, L, Hq, Hkv, D, dtype, layout, norm, rot, axes, interleaved, memory
    (1, 1, 1, 1, 128, BF16, "HND", "head", 128, 1, False, "dense"),
    (3, 17, 8, 2, 128, BF16, "HND", "head", 128, 1, True, "padded"),
    (2, 333, 5, 5, 64, FP16, "NHD", "head", 64, 1, False, "transposed"),
    (2, 31, 4, 1, 64, FP32, "HND", "head", 32, 1, False, "dense"),
    (1, 70, 40, 40, 128, BF16, "NHD", "across", 128, 3, True, "dense"),
    (2, 19, 12, 3, 128, FP16, "HND", "across", 128, 2, False, "shifted"),
    (1, 5, 128, 7, 128, FP32, "NHD", "across", 64, 1, True, "odd"),
    (2, 9, 33, 20, 64, BF16, "NHD", "across", 64, 4, False, "strided"),
    (4, 6, 3, 2, 128, BF16, "HND", None, 128, 4, False, "strided"),
    (1, 300, 2, 1, 64, BF16, "NHD", None, 48, 1, True, "odd"),
    (1, 45, 6, 2, 128, BF16, "HND", "head", 0, 1, False, "dense"),
    (1, 7000, 3, 1, 128, FP16, "HND", "head", 104, 2, True, "shifted"),
]


@pytest.mark.parametrize("pos64", [False, True])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_norm_rope(case, pos64):
    import mpsa
    B, L, Hq, Hkv, D, dtype, layout, norm, rot, axes, inter, how = case
    g = torch.Generator().manual_seed(L + D)
    q, k = rnd(g, B, Hq, L, D, dtype=dtype), rnd(g, B, Hkv, L, D, dtype=dtype, amp=3.0)
    half, rows = rot // 2, 500
    kw, rowpos, cos, sin = {}, None, None, None
    if rot:
        cos, sin = _angles(rows, half)
        kw["rope"] = (cos.cuda(), sin.cuda())
        pos = torch.randint(0, rows, (B, L, axes), generator=g)
        pos[0, L // 2] = rows - 1
        sections = None
        axis = torch.zeros(half, dtype=torch.long)
        if axes > 1:
            cut = sorted(int(x) for x in torch.randint(0, half + 1, (axes - 1,), generator=g))
            sections = tuple(b - a for a, b in zip([0, *cut], [*cut, half]))
            axis = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections))
        rowpos = pos[..., axis]
        kw["sections"] = sections
        p = (pos if axes > 1 else pos[..., 0]).to(torch.int64 if pos64 else torch.int32).cuda()
        if B == 1:
            p = p[0]
        kw["positions"] = p
    weights = [None, None]
    if norm:
        kw["eps"] = 1e-5
        kw["across_heads"] = norm == "across"
        for i, H in enumerate((Hq, Hkv)):
            weights[i] = (1 + 0.3 * torch.randn((H, D) if norm == "across" else (D,), generator=g)).to(FP32 if pos64 else dtype)
    else:
        kw["norm"] = False
    out = mpsa.norm_rope(laid_out(q, layout, how), laid_out(k, layout, how), q_weight=None if weights[0] is None else weights[0].cuda(),
                         k_weight=None if weights[1] is None else weights[1].cuda(), interleaved=inter, tensor_layout=layout, **kw)
    # fp32 arithmetic behind the one rounding: a sum of n positive terms is off by its depth in additions (8 in a lane, 4 or 5 across lanes;
    # across heads 32, 5 and 16), which the root halves; reciprocal root 2, two products, product and sum of the rotation 2
    deep = {None: 0, "head": 13, "across": 53}[norm]
    c = (deep / 2 + 6) * 2.0 ** -24
    for x, w, y in zip((q, k), weights, out):
        assert y.dtype == dtype and y.is_contiguous()
        if w is not None:
            w = w.double().reshape(1, -1, 1, D) if norm == "across" else w.double()
        ref, size = P.norm_rope(x, w, norm, 1e-5, cos, sin, rowpos, inter)
        err = (logical(y, layout).double() - ref).abs()
        assert bool((err <= half_step(dtype) * ref.abs() + c * size * 1.01 + 1e-30 + (2.0 ** -25 if dtype == FP16 else 0)).all()), float(err.max())


def test_norm_rope_one_operand_default_positions_and_outside_the_table():
    import mpsa
    g = torch.Generator().manual_seed(3)
    q = rnd(g, 2, 4, 20, 128)
    cos, sin = _angles(20, 64)
    rope = (cos.cuda(), sin.cuda())
    y = mpsa.norm_rope(q.cuda(), rope=rope)
    pos = torch.arange(20, dtype=torch.int32).cuda()
    assert torch.equal(y, mpsa.norm_rope(q.cuda(), rope=rope, positions=pos))
    for bad in (-1, 20, 2 ** 31 - 1, -2 ** 31):
        p = pos.clone()
        p[7] = bad
        z = mpsa.norm_rope(q.cuda(), rope=rope, positions=p)
        assert bool(torch.isnan(z[:, :, 7]).all())
        assert torch.equal(torch.cat((z[:, :, :7], z[:, :, 8:]), 2), torch.cat((y[:, :, :7], y[:, :, 8:]), 2))
    p = pos.long()
    p[3] = 2 ** 40
    cos, sin = _angles(20, 32)
    z = mpsa.norm_rope(q.cuda(), rope=(cos.cuda(), sin.cuda()), positions=p)
    assert bool(torch.isnan(z[:, :, 3, :64]).all()) and not bool(torch.isnan(z[:, :, 3, 64:]).any())


def test_norm_rope_non_finite_rows_stay_in_their_rows():
    import mpsa
    g = torch.Generator().manual_seed(4)
    q = rnd(g, 1, 3, 40, 128)
    y = mpsa.norm_rope(q.cuda())
    q[0, 1, 5, 3], q[0, 2, 6, 9] = float("nan"), float("inf")
    z = mpsa.norm_rope(q.cuda())
    keep = torch.ones(3, 40, dtype=torch.bool)
    keep[1, 5] = keep[2, 6] = False
    assert torch.equal(z[0][keep.cuda()], y[0][keep.cuda()])
    assert bool(torch.isnan(z[0, 1, 5]).all()) and bool(torch.isnan(z[0, 2, 6, 9]))
    zero = mpsa.norm_rope(torch.zeros(1, 1, 2, 64, device="cuda", dtype=BF16))
    assert bool((zero == 0).all())


# -------------------------------------------------------------------------------------------------------------- the cache
def filled(g, pages, H, page, D, elem):
    """A cache with finite bytes left by others everywhere."""
    import mpsa
    c = mpsa.kv_cache(pages, H, D, page_size=page, elem=elem)
    for t in (c.k, c.v):
        t.copy_(torch.randint(0, 112 if elem != "e2m1" else 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.randint(110, 125, t.shape, generator=g, dtype=torch.uint8))
    return c


def table_of(g, B, m, pages):
    return torch.randperm(pages, generator=g)[: B * m].to(torch.int32).reshape(B, m)


def codes_of(c, name):
    """fp64 values in units of the scales, and the scale codes, of a whole cache buffer."""
    code, scale = getattr(c, name).cpu(), getattr(c, name + "_scale").cpu()
    if c.elem == "e2m1":
        code = torch.stack((code & 15, code >> 4), -1).flatten(-2)
    return P.element_table(c.elem)[code.long()].reshape(*scale.shape, 32), scale.long()


APPEND = [
    # B, T, starts up to, Hkv, D, elem, page, dtype, layout, memory
    (1, 1, 0, 1, 64, "e4m3", 16, BF16, "HND", "dense"),
    (3, 37, 50, 2, 128, "e4m3", 16, BF16, "NHD", "dense"),
    (2, 130, 100, 3, 64, "e5m2", 64, FP16, "HND", "padded"),
    (5, 9, 33, 8, 128, "e2m1", 32, BF16, "HND", "transposed"),
    (2, 33, 7, 1, 64, "e2m1", 128, FP32, "NHD", "shifted"),
    (1, 600, 900, 4, 128, "e4m3", 1024, FP32, "HND", "odd"),
    (2, 21, 3, 2, 128, "e5m2", 16, FP32, "NHD", "strided"),
]


@pytest.mark.parametrize("counted", [False, True])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append_is_the_rounding_and_leaves_the_rest(case, counted):
    import mpsa
    B, T, most, H, D, elem, page, dtype, layout, how = case
    g = torch.Generator().manual_seed(T + D)
    m = -(-(most + T) // page)
    c = filled(g, B * m + 2, H, page, D, elem)
    before = {n: getattr(c, n).cpu().clone() for n in ("k", "v", "k_scale", "v_scale")}
    table = table_of(g, B, m, B * m + 2)
    start = torch.randint(0, most + 1, (B,), generator=g, dtype=torch.int32)
    counts = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32) if counted else None
    x = {}
    for n in ("k", "v"):
        t = rnd(g, B, H, T, D, dtype=FP32) * torch.exp2(torch.randint(-12, 6, (B, H, T, 1), generator=g).float())
        t[0, 0, 0, :32] = 0
        if T > 4:
            t[0, -1, 1, 32:64] = torch.randn(32, generator=g) * 1e-6
            t[-1, 0, 2, 5] = P.LARGEST[elem] * 2.0 ** -3                    # the largest element exactly, and just above it
            t[-1, 0, 3, 40] = P.LARGEST[elem] * 2.0 ** -3 * (1 + 2.0 ** -7)
            t[0, 0, 4, 1] = -0.0
        x[n] = t.to(dtype)
    mpsa.kv_cache_append(c, laid_out(x["k"], layout, how), laid_out(x["v"], layout, how), table.cuda(), start.cuda(),
                         counts=None if counts is None else counts.cuda(), tensor_layout=layout)
    written = torch.zeros(c.k.shape[:3], dtype=torch.bool)
    for n in ("k", "v"):
        y, e = P.quantise(x[n], elem)
        got, gots = codes_of(c, n)
        for b in range(B):
            for t in range(T if counts is None else int(counts[b])):
                p = int(start[b]) + t
                at = int(table[b, p // page]), slice(None), p % page
                written[at] = True
                assert torch.equal(got[at], y[b, :, t]) and torch.equal(gots[at], e[b, :, t])
        for part in (n, n + "_scale"):
            assert torch.equal(getattr(c, part).cpu()[~written], before[part][~written])


@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_append_of_non_finite_tiny_and_huge_values(elem):
    import mpsa
    g = torch.Generator().manual_seed(1)
    c = filled(g, 2, 1, 16, 128, elem)
    k = rnd(g, 1, 1, 8, 128, dtype=FP32)
    k[0, 0, 0, 3], k[0, 0, 1, 40], k[0, 0, 2, 70] = float("nan"), float("inf"), -float("inf")
    k[0, 0, 3] *= 1e-42
    k[0, 0, 4] *= 3e37
    k[0, 0, 5, :32] = 3.4028234e38
    k[0, 0, 6] *= 2.0 ** -126
    table = torch.tensor([[1]], dtype=torch.int32).cuda()
    mpsa.kv_cache_append(c, k.cuda(), k.cuda(), table, torch.tensor([3], dtype=torch.int32).cuda())
    y, e = P.quantise(k, elem)
    for n in ("k", "v"):
        got, gots = codes_of(c, n)
        assert torch.equal(gots[1, 0, 3:11], e[0, 0]) and torch.equal(got[1, 0, 3:11], y[0, 0])
    back, _ = mpsa.kv_cache_read(c, table, torch.tensor([11], dtype=torch.int32).cuda(), out_dtype=FP32)
    nan = torch.isnan(back[0, 0].cpu()).reshape(16, 4, 32)
    assert bool(nan[3, 0].all()) and bool(nan[4, 1].all()) and bool(nan[5, 2].all()) and int(nan.sum()) == 96


@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("D,page,dtype", [(64, 16, BF16), (128, 64, FP16), (128, 16, FP32), (64, 128, FP32)])
def test_read_back(elem, D, page, dtype):
    import mpsa
    g = torch.Generator().manual_seed(D + page)
    B, H, m = 4, 3, 5
    c = filled(g, B * m, H, page, D, elem)
    table = table_of(g, B, m, B * m)
    table[2, 1] = -1
    table[3, 0] = B * m
    lengths = torch.tensor([m * page, 0, 3 * page - 5, 2 * page + 1], dtype=torch.int32)
    for n in (None, 2 * page + 3, 1):
        k, v = mpsa.kv_cache_read(c, table.cuda(), lengths.cuda(), max_len=n, out_dtype=dtype)
        N = m * page if n is None else n
        assert k.shape == v.shape == (B, H, N, D)
        for name, got in (("k", k), ("v", v)):
            ref = torch.zeros(B, H, N, D, dtype=torch.float64)
            for b in range(B):
                L = min(int(lengths[b]), N)
                x = P.values(P.gather(getattr(c, name), table[b].clamp(0, B * m - 1), L), P.gather(getattr(c, name + "_scale"), table[b].clamp(0, B * m - 1), L), elem)
                there = ((table[b] >= 0) & (table[b] < B * m)).repeat_interleave(page)[:L]
                ref[b, :, :L] = torch.where(there[:, None], x, 0.0)
            assert torch.equal(got.cpu(), ref.to(dtype)), name
    # a length beyond the table, and lengths below zero
    k, _ = mpsa.kv_cache_read(c, table.cuda(), torch.tensor([10 ** 9, -7, 0, 0], dtype=torch.int32).cuda(), max_len=m * page + 9, out_dtype=dtype)
    assert bool((k[0, :, m * page:] == 0).all()) and bool((k[1] == 0).all()) and not bool((k[0, :, :m * page] == 0).all())


def test_pages_that_do_not_exist_are_not_written():
    import mpsa
    g = torch.Generator().manual_seed(2)
    c = filled(g, 4, 2, 16, 64, "e4m3")
    before = [getattr(c, n).clone() for n in ("k", "v", "k_scale", "v_scale")]
    x = rnd(g, 3, 2, 40, 64).cuda()
    table = torch.tensor([[-1, 4, 7], [2 ** 31 - 1, -2 ** 31, 1000], [-1, -1, -1]], dtype=torch.int32).cuda()
    mpsa.kv_cache_append(c, x, x, table, torch.tensor([0, 3, 2 ** 31 - 1], dtype=torch.int32).cuda())
    mpsa.kv_cache_append(c, x, x, table.clamp(0, 3), torch.tensor([48, -40, -2 ** 31], dtype=torch.int32).cuda())       # beyond the table, before the start
    mpsa.kv_cache_append(c, x, x, table.clamp(0, 3), torch.zeros(3, dtype=torch.int32).cuda(), counts=torch.tensor([0, -5, 0], dtype=torch.int32).cuda())
    assert all(torch.equal(a, getattr(c, n)) for a, n in zip(before, ("k", "v", "k_scale", "v_scale")))


# -------------------------------------------------------------------------------------------------------------- attention
def real_cache(g, B, lens, H, page, D, elem, amp=1.0, spare=2):
    """A cache whose sequences hold quantised values, scattered over pages; everything else is NaN codes and NaN scales."""
    import mpsa
    m = max(1, -(-max(lens) // page))
    c = mpsa.kv_cache(B * m + spare, H, D, page_size=page, elem=elem)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        t.fill_(255)
    table = table_of(g, B, m, B * m + spare)
    if max(lens) > 0:
        T = max(lens)
        wide = 1 + 3 * (torch.rand(1, H, 1, D, generator=g) > 0.95).float()
        k, v = (rnd(g, B, H, T, D) * wide * amp).to(BF16), rnd(g, B, H, T, D)
        mpsa.kv_cache_append(c, k.cuda(), v.cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32).cuda(), counts=torch.tensor(lens, dtype=torch.int32).cuda())
    return c, table


def check_attention(c, table, lens, q, out, lse, q_lens=None, mask=None, sm=None, absent=None):
    """out, lse of kv_cache_attention (logical [B,Hq,T,D]) against the plain form.

    A score is a sum of D products in fp32, scaled per block: off by at most (D + 8) 2^-23 of the sum of its terms' magnitudes (a matrix
    instruction may cut off instead of rounding), which moves log2 of a probability by that times log2(e), and the exponential adds 2^-22.
    P is rounded to fp16 (2^-11), sums of n fp32 terms to n 2^-24 at worst, n up to a few hundred in one accumulator (2^-16); the output is rounded once.
    What is rounded is P times a block scale, in units in which the row's largest such product is 2^7 at least: fp16 steps of 2^-24 below 2^-14 add
    2^-25 for each key, 2^-32 of the largest product.  An element is at most the type's largest value L times its scale, and the largest element of a
    block more than L/2 times it (the scale is the smallest one that does), so that is 2^-31 of the row's largest p |v|, for each of n keys."""
    B, Hq, T, D = q.shape
    sm = D ** -0.5 if sm is None else sm
    for b in range(B):
        n = lens[b]
        t = T if q_lens is None else q_lens[b]
        k, v = (P.values(P.gather(getattr(c, x), table[b], n), P.gather(getattr(c, x + "_scale"), table[b], n), c.elem) for x in ("k", "v"))
        seen = torch.ones(t, n, dtype=torch.bool)
        if t and n >= t:
            seen[:, n - t:] = torch.ones(t, t).tril().bool() if mask is None else (mask if mask.dim() == 2 else mask[b])[:t, :t]
        if absent is not None:
            seen &= ~absent[b][:n]
        o, l, a, mag, big = P.attention(q[b, :, :t].double(), k, v, seen, sm)
        ds = (D + 8) * 2.0 ** -23 * mag.unsqueeze(-1) + 2.0 ** -22
        got, gl = out[b, :, :t].double(), lse[b, :, :t].double()
        assert torch.equal(torch.isnan(got), torch.isnan(o)), b
        fine = ~torch.isnan(o)
        err, tol = (got - o).abs(), half_step(q.dtype) * o.abs() * 1.01 + (2 * ds + 2.0 ** -11 + 2.0 ** -16) * a + n * 2.0 ** -31 * big.unsqueeze(-1) + 2.0 ** -24
        assert bool((err[fine] <= tol[fine]).all()), (b, float((err[fine] / tol[fine]).max()))
        real = torch.isfinite(l)
        assert torch.equal(gl[~real & ~torch.isnan(l)], l[~real & ~torch.isnan(l)])
        lt = 1.4427 * 1.01 * ds.squeeze(-1) + 2.0 ** -16 + 2.0 ** -23 * l.abs()
        assert bool(((gl - l).abs()[real] <= lt[real]).all())
        assert bool((out[b, :, t:] == 0).all()) and bool((lse[b, :, t:] == -math.inf).all())


def tree_mask(g, T):
    m = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        if i:
            m[i] = m[int(torch.randint(max(0, i - 5), i, (1,), generator=g))]
        m[i, i] = True
    return m


ATTEND = [
    # lens, T, Hq, Hkv, D, elem, page, dtype, layout, memory of q, q_lens, mask
    ([1], 1, 1, 1, 64, "e4m3", 16, BF16, "HND", "dense", None, None),
    ([1, 2, 15, 16, 17, 0], 1, 4, 1, 128, "e4m3", 16, BF16, "HND", "dense", None, None),
    ([31, 32, 33, 127, 128, 129, 255, 257], 1, 8, 2, 128, "e5m2", 64, FP16, "NHD", "padded", None, None),
    ([700, 3, 0, 1501], 1, 12, 12, 64, "e2m1", 32, BF16, "HND", "transposed", None, None),
    ([4097, 100], 1, 10, 2, 128, "e2m1", 128, FP16, "HND", "shifted", None, None),
    ([9000], 1, 8, 1, 64, "e5m2", 1024, BF16, "NHD", "odd", None, None),
    ([40, 600, 5], 5, 6, 3, 128, "e4m3", 16, BF16, "HND", "dense", None, None),
    ([40, 600, 9, 77], 9, 4, 2, 64, "e4m3", 64, FP16, "NHD", "strided", [9, 1, 9, 0], None),
    ([64, 1000, 33], 33, 8, 2, 128, "e4m3", 32, BF16, "HND", "dense", [33, 17, 2], "tree"),
    ([65, 300], 64, 8, 1, 128, "e5m2", 64, BF16, "NHD", "dense", None, "tree"),
    ([100, 500, 64], 64, 4, 4, 64, "e2m1", 16, FP16, "HND", "dense", [64, 40, 64], "shared"),
    ([300, 1100], 130, 14, 2, 128, "e4m3", 64, BF16, "HND", "dense", None, None),
    ([20, 21], 20, 3, 1, 128, "e2m1", 16, BF16, "HND", "dense", None, "empty"),
    ([5000, 1100], 1024, 2, 2, 64, "e4m3", 128, BF16, "NHD", "dense", [1024, 1000], None),
    ([2048, 129], 128, 4, 4, 128, "e2m1", 64, BF16, "HND", "padded", None, "tree"),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_attention(case):
    import mpsa
    lens, T, Hq, Hkv, D, elem, page, dtype, layout, how, q_lens, kind = case
    g = torch.Generator().manual_seed(sum(lens) + T)
    B = len(lens)
    c, table = real_cache(g, B, lens, Hkv, page, D, elem)
    q = rnd(g, B, Hq, T, D, dtype=dtype)
    mask = None
    if kind == "tree":
        mask = torch.stack([tree_mask(g, T) for _ in range(B)])
    elif kind == "shared":
        mask = tree_mask(g, T)
    elif kind == "empty":                      # rows that see none of the drafted tokens, and with no keys before them nothing at all
        mask = torch.zeros(B, T, T, dtype=torch.bool)
        mask[:, ::2] = tree_mask(g, T)[::2]
    out, lse = mpsa.kv_cache_attention(laid_out(q, layout, how), c, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                       q_lens=None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32).cuda(),
                                       mask=None if mask is None else mask.cuda(), return_lse=True, tensor_layout=layout)
    assert out.dtype == dtype and out.is_contiguous()
    check_attention(c, table, lens, q, logical(out, layout), lse.cpu(), q_lens, mask)


@pytest.mark.parametrize("elem,D", [("e4m3", 128), ("e2m1", 128), ("e5m2", 64)])
def test_attention_of_a_long_sequence_among_short_ones(elem, D):
    import mpsa
    g = torch.Generator().manual_seed(8)
    lens = [5, 33000, 0, 260, 1]
    c, table = real_cache(g, 5, lens, 2, 64, D, elem, amp=0.5)
    q = rnd(g, 5, 8, 1, D)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    check_attention(c, table, lens, q, out.cpu(), lse.cpu())


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("T", [1, 40])
def test_attention_with_scores_that_grow_and_values_of_many_sizes(elem, T):
    import mpsa
    g = torch.Generator().manual_seed(9)
    n, D, Hq, Hkv = 1500, 128, 4, 1
    c = mpsa.kv_cache(30, Hkv, D, elem=elem)
    table = table_of(g, 1, 30, 30)
    k = rnd(g, 1, Hkv, n, D, dtype=FP32) * torch.linspace(0.1, 8, n)[:, None]
    v = rnd(g, 1, Hkv, n, D, dtype=FP32) * torch.exp2(torch.randint(-9, 9, (1, Hkv, n, 1), generator=g).float())
    mpsa.kv_cache_append(c, k.cuda(), v.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32).cuda())
    for scale in (1.0, 2.0 ** -30, 3.0):
        q = rnd(g, 1, Hq, T, D) * scale
        out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), return_lse=True)
        check_attention(c, table, [n], q, out.cpu(), lse.cpu())
    q = rnd(g, 1, Hq, T, D)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), return_lse=True, sm_scale=0.01)
    check_attention(c, table, [n], q, out.cpu(), lse.cpu(), sm=0.01)


@pytest.mark.parametrize("T,Hq", [(1, 4), (6, 4), (40, 8)])
def test_what_is_masked_has_no_part_whatever_it_is(T, Hq):
    """NaN among keys and values that some rows do not see reaches the rows that do, and no others."""
    import mpsa
    g = torch.Generator().manual_seed(10)
    lens, D, Hkv = [90, 300], 128, 2
    c, table = real_cache(g, 2, lens, Hkv, 16, D, "e4m3")
    x = rnd(g, 2, Hkv, T, D)
    bad = x.clone()
    bad[:, :, T // 2, 70] = float("nan")                    # one drafted token's block
    start = torch.tensor([n - T for n in lens], dtype=torch.int32).cuda()
    mpsa.kv_cache_append(c, x.cuda(), bad.cuda(), table.cuda(), start)
    mask = torch.eye(T, dtype=torch.bool)
    mask[T - 1, 0] = True
    q = rnd(g, 2, Hq, T, D)
    for kind in ("v", "k"):
        if kind == "k":
            mpsa.kv_cache_append(c, bad.cuda(), x.cuda(), table.cuda(), start)
        out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), mask=mask.cuda(), return_lse=True)
        hit = torch.isnan(out.cpu()).any(-1)
        assert bool(hit[:, :, T // 2].all()) and int(hit.sum()) == 2 * Hq
        if kind == "v":                                      # (only that block of the depth)
            assert bool(torch.isnan(out[:, :, T // 2, 64:96]).all()) and not bool(torch.isnan(out[:, :, T // 2, :64]).any())
            check_attention(c, table, lens, q, out.cpu(), lse.cpu(), mask=mask)


def test_attention_of_non_finite_queries_stays_in_its_row():
    import mpsa
    g = torch.Generator().manual_seed(11)
    c, table = real_cache(g, 1, [200], 2, 16, 64, "e4m3")
    q = rnd(g, 1, 8, 3, 64)
    args = (c, table.cuda(), torch.tensor([200], dtype=torch.int32).cuda())
    ref = mpsa.kv_cache_attention(q.cuda(), *args)
    q[0, 2, 1, 5], q[0, 7, 0, 60] = float("nan"), float("inf")
    out = mpsa.kv_cache_attention(q.cuda(), *args)
    keep = torch.ones(8, 3, dtype=torch.bool)
    keep[2, 1] = keep[7, 0] = False
    assert torch.equal(out[0][keep.cuda()], ref[0][keep.cuda()])
    assert bool(torch.isnan(out[0, 2, 1]).all()) and bool(torch.isnan(out[0, 7, 0]).all())
    zero = torch.zeros(1, 8, 3, 64, dtype=BF16)
    out, lse = mpsa.kv_cache_attention(zero.cuda(), *args, return_lse=True)
    check_attention(c, table, [200], zero, out.cpu(), lse.cpu())


@pytest.mark.parametrize("T", [1, 40])
def test_pages_that_do_not_exist_are_not_seen(T):
    import mpsa
    g = torch.Generator().manual_seed(12)
    lens = [250, 100, 64]
    c, table = real_cache(g, 3, lens, 2, 16, 128, "e4m3")
    q = rnd(g, 3, 4, T, 128)
    holes = table.clone()
    holes[0, 3], holes[0, 7], holes[1, :] = -1, c.k.shape[0], 2 ** 31 - 1
    absent = [((h < 0) | (h >= c.k.shape[0])).repeat_interleave(16) for h in holes]
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, holes.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    check_attention(c, table, lens, q, out.cpu(), lse.cpu(), absent=absent)
    # lengths that the table cannot hold, and below zero
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor([2 ** 31 - 1, -5, 64], dtype=torch.int32).cuda(), return_lse=True)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


# ------------------------------------------------------------------------------------------------------------- run together
def _generate(g, c, table, D, Hq, Hkv, dtype, graph=False):
    """A prompt in two chunks, three single tokens, a tree of drafts, the accepted ones written again: yields (inputs, outputs)."""
    import mpsa
    B = table.shape[0]
    cos, sin = _angles(400, D // 2)
    rope = (cos.cuda(), sin.cuda())
    wq, wk = ((1 + 0.1 * torch.randn(D, generator=g)).cuda() for _ in range(2))
    lengths = torch.zeros(B, dtype=torch.int32).cuda()
    steps = [(50, None, None), (13, None, None), (1, None, None), (1, None, None), (1, None, None), (7, tree_mask(g, 7), [0, 2, 5]), (1, None, None)]
    for T, mask, kept in steps:
        raw = [rnd(g, B, H, T, D, dtype=dtype).cuda() for H in (Hq, Hkv, Hkv)]
        depth = torch.arange(T) if mask is None else mask.sum(1) - 1
        pos = (lengths[:, None] + depth.cuda()[None]).to(torch.int32)
        q, k = mpsa.norm_rope(raw[0], raw[1], q_weight=wq, k_weight=wk, rope=rope, positions=pos)
        mpsa.kv_cache_append(c, k, raw[2], table, lengths)
        o = mpsa.kv_cache_attention(q, c, table, lengths + T, mask=None if mask is None else mask.cuda())
        yield T, mask, kept, raw, pos, (wq, wk, cos, sin), o
        if kept is not None:                     # the accepted drafts follow each other
            mpsa.kv_cache_append(c, k[:, :, kept].contiguous(), raw[2][:, :, kept].contiguous(), table, lengths)
            T = len(kept)
        lengths += T


@pytest.mark.parametrize("elem,D,dtype", [("e4m3", 128, BF16), ("e2m1", 64, FP16)])
def test_a_run_of_all_of_them(elem, D, dtype):
    import mpsa
    g = torch.Generator().manual_seed(13)
    B, Hq, Hkv = 3, 6, 2
    c = mpsa.kv_cache(20, Hkv, D, page_size=32, elem=elem)
    table = table_of(g, B, 4, 20).cuda()
    held = [torch.zeros(B, Hkv, 0, D, dtype=torch.float64) for _ in range(2)]
    for T, mask, kept, raw, pos, (wq, wk, cos, sin), o in _generate(g, c, table, D, Hq, Hkv, dtype):
        rows = pos.cpu().long().unsqueeze(-1).expand(B, T, D // 2)
        q, _ = P.norm_rope(raw[0].cpu(), wq.cpu().double(), "head", 1e-6, cos, sin, rows, False)
        k, _ = P.norm_rope(raw[1].cpu(), wk.cpu().double(), "head", 1e-6, cos, sin, rows, False)
        new = []
        for x in (k.to(dtype), raw[2].cpu()):
            y, e = P.quantise(x, elem)
            new.append(torch.ldexp(y, (e - 127).unsqueeze(-1)).flatten(-2))
        n = held[0].shape[2]
        seen = torch.ones(T, n + T, dtype=torch.bool)
        seen[:, n:] = torch.ones(T, T).tril().bool() if mask is None else mask
        for b in range(B):
            ref = P.attention(q[b].to(dtype).double(), torch.cat((held[0][b], new[0][b]), 1), torch.cat((held[1][b], new[1][b]), 1), seen, D ** -0.5)[0]
            # a norm that rounds the other way moves a key or a query by a step of its type, and an element of the cache by a step of its own
            step = {"e4m3": 2.0 ** -3, "e2m1": 2.0 ** -1}[elem]
            err = (o[b].cpu().double() - ref).norm() / ref.norm()
            assert float(err) < 4 * half_step(dtype) + 0.02 * step, float(err)
        keep = kept if kept is not None else list(range(T))
        held = [torch.cat((h, x[:, :, keep]), 2) for h, x in zip(held, new)]
        assert held[0].shape[2] <= 128


def test_captured_and_replayed_and_on_two_streams():
    import mpsa
    g = torch.Generator().manual_seed(14)
    B, Hq, Hkv, D = 4, 8, 2, 128
    lens = [300, 4000, 17, 1]
    c, table = real_cache(g, B, [n + 40 for n in lens], Hkv, 64, D, "e4m3")
    table = table.cuda()
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    q, k, v = rnd(g, B, Hq, 1, D).cuda(), rnd(g, B, Hkv, 1, D).cuda(), rnd(g, B, Hkv, 1, D).cuda()
    cos, sin = (t.cuda() for t in _angles(5000, 64))

    def step():
        y, z = mpsa.norm_rope(q, k, rope=(cos, sin), positions=lengths[:, None])
        mpsa.kv_cache_append(c, z, v, table, lengths)
        return mpsa.kv_cache_attention(y, c, table, lengths + 1, return_lse=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(3):
        lengths += i
        q.copy_(rnd(g, B, Hq, 1, D))
        graph.replay()
        a = out.clone(), lse.clone()
        b = step()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # two calls in flight at once, each on its own stream
    side = [torch.cuda.Stream() for _ in range(2)]
    qs = [rnd(g, B, Hq, 1, D).cuda() for _ in range(2)]
    alone = [mpsa.kv_cache_attention(x, c, table, lengths) for x in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x, s in zip(qs, side):
            with torch.cuda.stream(s):
                got.append(mpsa.kv_cache_attention(x, c, table, lengths))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


def test_parts_merge():
    """Two caches' results over different keys, merged through their denominators."""
    import mpsa
    g = torch.Generator().manual_seed(15)
    c, table = real_cache(g, 1, [640], 2, 64, 128, "e4m3")
    q = rnd(g, 1, 8, 1, 128)
    whole, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor([640], dtype=torch.int32).cuda(), return_lse=True)
    parts = [mpsa.kv_cache_attention(q.cuda(), c, t.contiguous().cuda(), torch.tensor([n], dtype=torch.int32).cuda(), return_lse=True)
             for t, n in ((table[:, :4], 256), (table[:, 4:], 384))]
    acc, l = parts[0][0].float(), parts[0][1].clone()
    mpsa.attention_merge(acc, l, parts[1][0], parts[1][1])
    assert float((acc - whole.float()).abs().max()) <= 2 * half_step(BF16) * float(whole.abs().max()) and float((l - lse).abs().max()) < 1e-4


@pytest.mark.parametrize("elem,D", [("e4m3", 128), ("e2m1", 64), ("e5m2", 64), ("e2m1", 128)])
@pytest.mark.parametrize("T,Hq", [(1, 8), (3, 8), (7, 8), (40, 8)])
def test_attention_whose_units_are_cut_anywhere(elem, D, T, Hq):
    """Tables that are long enough for runs of equal length: units begin and end in the middle of them, some CTAs have several, some none."""
    import mpsa
    g = torch.Generator().manual_seed(T + D)
    lens = [3000, T, 800, 0, 61, 4100, 33]
    q_lens = [T, T, max(1, T - 2), 0, T, T, 1]
    lens = [max(n, t) for n, t in zip(lens, q_lens)]
    c, table = real_cache(g, 7, lens, 2, 64, D, elem, amp=0.7)
    table = torch.cat((table, torch.full((7, 256), -1, dtype=torch.int32)), 1)            # room for more than they have
    q = rnd(g, 7, Hq, T, D)
    args = (q.cuda(), c, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    kw = dict(q_lens=torch.tensor(q_lens, dtype=torch.int32).cuda(), return_lse=True)
    out, lse = mpsa.kv_cache_attention(*args, **kw)
    check_attention(c, table, lens, q, out.cpu(), lse.cpu(), q_lens)
    again = mpsa.kv_cache_attention(*args, **kw)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    mpsa.check_status()


def test_many_sequences():
    import mpsa
    g = torch.Generator().manual_seed(20)
    B = 300
    lens = [int(x) for x in torch.randint(0, 90, (B,), generator=g)]
    lens[7], lens[250] = 1500, 700
    c, table = real_cache(g, B, lens, 1, 16, 64, "e4m3")
    for T, Hq in ((1, 2), (2, 20)):
        q = rnd(g, B, Hq, T, 64)
        q_lens = [min(T, n) for n in lens]
        out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
        check_attention(c, table, lens, q, out.cpu(), lse.cpu(), q_lens)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_captured_beside_another_stream(T):
    """Graphs of two calls replayed at once on two streams, with new lengths, and an eager call between them."""
    import mpsa
    g = torch.Generator().manual_seed(21)
    lens = [3000, 40, 7000]
    c, table = real_cache(g, 3, [7100] * 3, 2, 64, 128, "e4m3")
    table = table.cuda()
    qs = [rnd(g, 3, 8, T, 128).cuda() for _ in range(2)]
    lengths = [torch.tensor(lens, dtype=torch.int32).cuda() for _ in range(2)]
    mpsa.kv_cache_attention(qs[0], c, table, lengths[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, n in zip(qs, lengths):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(mpsa.kv_cache_attention(q, c, table, n))
        graphs.append(graph)
    side = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        lengths[0].add_(i)
        lengths[1].copy_(torch.tensor([T + i, 7000 - 3 * i, 900], dtype=torch.int32))
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = [mpsa.kv_cache_attention(q, c, table, n) for q, n in zip(qs, lengths)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    mpsa.check_status()


def test_long_chains_of_calls_see_what_was_written_before():
    """Append, read and attention one behind the other without a host wait: each overlaps the launch of the one before."""
    import mpsa
    g = torch.Generator().manual_seed(22)
    c = mpsa.kv_cache(64, 2, 128, page_size=16)
    table = table_of(g, 2, 32, 64).cuda()
    lengths = torch.zeros(2, dtype=torch.int32).cuda()
    ks, vs = rnd(g, 2, 2, 60, 128).cuda(), rnd(g, 2, 2, 60, 128).cuda()
    got = []
    for t in range(60):
        mpsa.kv_cache_append(c, ks[:, :, t:t + 1], vs[:, :, t:t + 1], table, lengths)
        lengths += 1
        got.append((mpsa.kv_cache_read(c, table, lengths, max_len=60), mpsa.kv_cache_attention(ks[:, :, t:t + 1], c, table, lengths)))
    k, v = mpsa.kv_cache_read(c, table, lengths, max_len=60)
    for t, ((a, b), o) in enumerate(got):
        assert torch.equal(a[:, :, :t + 1], k[:, :, :t + 1]) and torch.equal(b[:, :, :t + 1], v[:, :, :t + 1]) and bool((a[:, :, t + 1:] == 0).all())
        again = mpsa.kv_cache_attention(ks[:, :, t:t + 1], c, table, torch.full((2,), t + 1, dtype=torch.int32).cuda())
        assert torch.equal(o, again)


def test_the_long_way_gives_the_same(monkeypatch):
    """Without the native module every call goes through the Python checks and ctypes."""
    import mpsa
    from mpsa import _lib
    g = torch.Generator().manual_seed(23)
    q, k, v = rnd(g, 2, 8, 5, 128).cuda(), rnd(g, 2, 2, 5, 128).cuda(), rnd(g, 2, 2, 5, 128).cuda()
    cos, sin = (t.cuda() for t in _angles(64, 64))
    lengths = torch.tensor([7, 30], dtype=torch.int32).cuda()
    mask = tree_mask(g, 5).cuda()

    def everything():
        c = mpsa.kv_cache(8, 2, 128, page_size=16, elem="e5m2")
        table = torch.arange(8, dtype=torch.int32).reshape(2, 4).cuda()
        y = mpsa.norm_rope(q, k, q_weight=cos[0].repeat(2).contiguous(), rope=(cos, sin), positions=lengths[:, None] + torch.arange(5, dtype=torch.int32).cuda())
        mpsa.kv_cache_append(c, y[1], v, table, lengths, counts=torch.tensor([5, 4], dtype=torch.int32).cuda())
        r = mpsa.kv_cache_read(c, table, lengths + 5)
        return (*y, c.k, c.v_scale, *r, *mpsa.kv_cache_attention(y[0], c, table, lengths + 5, mask=mask, return_lse=True), mpsa.norm_rope(q))

    native = everything()
    monkeypatch.setattr(_lib, "_native", _lib._LongWay)
    assert all(torch.equal(a, b) for a, b in zip(native, everything()))


def test_a_cache_keeps_its_buffers():
    import dataclasses

    import mpsa
    c = mpsa.kv_cache(4, 1, 64)
    with pytest.raises(dataclasses.FrozenInstanceError):
        c.k = torch.zeros_like(c.k)
    assert (c.num_kv_heads, c.page_size, c.head_dim) == (1, 64, 64) and mpsa.kv_cache(4, 3, 128, page_size=16, elem="e2m1").head_dim == 128
    x = torch.zeros(1, 1, 2, 64, device="cuda", dtype=BF16, requires_grad=True)
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    for f in (lambda: mpsa.kv_cache_append(c, x, x, i[None], i), lambda: mpsa.kv_cache_attention(x, c, i[None], i + 2)):
        with pytest.raises(ValueError):
            f()
        with torch.no_grad():
            f()


# ------------------------------------------------------------------------------------------------------------------ model hook
class _Rms(torch.nn.Module):
    def __init__(self, dim):
        super().__init__()
        self.eps, self.weight = 1e-5, torch.nn.Parameter(1 + 0.2 * torch.randn(dim))

    def forward(self, x):
        return (x.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + self.eps) * self.weight.double()).to(x.dtype)


@pytest.mark.parametrize("normed", [True, False])
def test_wan_block_with_norm_and_rotation_in_one_pass(normed):
    from mpsa import model_hooks as H
    spec = importlib.util.spec_from_file_location("_hooks_cpu", os.path.join(os.path.dirname(__file__), "test_model_hooks_cpu.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    torch.manual_seed(3)
    heads, d, L, grid = 3, 128, 200, (4, 6, 8)
    model = mod._Wan(dim=heads * d, heads=heads, n=1)
    att = model.blocks[0].self_attn
    if normed:
        att.norm_q, att.norm_k = _Rms(heads * d), _Rms(heads * d)
    model = model.cuda()
    ang = torch.arange(64, dtype=torch.float64)[:, None] * torch.cat([1e4 ** (-torch.arange(n, dtype=torch.float64) / n) for n in (22, 21, 21)])
    freqs = torch.polar(torch.ones_like(ang), ang)
    H.set_mpsa_attn_wan(model, fused_norm_rope=True)
    seen = []

    class Recorder(torch.nn.Module):
        def forward(self, q, k, v, **kw):
            seen.append((q, k, kw))
            return v

    att.inner_attention = Recorder()
    x = torch.randn(1, L, heads * d, device="cuda")
    att(x, torch.tensor([L]), torch.tensor([grid]), freqs)
    (q, k, kw), = seen
    assert kw == dict(is_causal=False, tensor_layout="NHD") and q.dtype == BF16
    f, h, w = grid
    i = torch.arange(f * h * w)
    turn = torch.cat((freqs[i // (h * w), :22], freqs[i // w % h, 22:43], freqs[i % w, 43:]), 1)[None, :, None]
    for got, lin, norm in ((q, att.q, att.norm_q), (k, att.k, att.norm_k)):
        y = norm(lin(x).detach()).double().cpu().reshape(1, L, heads, d)
        z = torch.view_as_complex(y[:, :f * h * w].reshape(1, -1, heads, 64, 2).contiguous()) * turn
        y[:, :f * h * w] = torch.view_as_real(z).flatten(-2)
        # fp32 throughout (2^-24 of a few operations of elements of size 6 at most; the norm above rounds to fp32 once more), then bf16
        assert bool(((got.double().cpu() - y).abs() <= half_step(BF16) * y.abs() * 1.01 + 2.0 ** -17).all())


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    import mpsa
    x = torch.zeros(2, 4, 3, 128, dtype=BF16, device="cuda")
    cos, sin = (t.cuda() for t in _angles(16, 64))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = mpsa.kv_cache(8, 2, 128)
    kv = torch.zeros(2, 2, 3, 128, dtype=BF16, device="cuda")
    tab = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    w = torch.ones(128, device="cuda", requires_grad=True)
    bad = [
        lambda: mpsa.norm_rope(x.cpu()), lambda: mpsa.norm_rope(x.double()), lambda: mpsa.norm_rope(x[0]), lambda: mpsa.norm_rope(x[..., :96]),
        lambda: mpsa.norm_rope(x, x[:1]), lambda: mpsa.norm_rope(x, x.half()), lambda: mpsa.norm_rope(x, tensor_layout="LHD"),
        lambda: mpsa.norm_rope(x, q_weight=w), lambda: mpsa.norm_rope(x, q_weight=torch.ones(64, device="cuda")),
        lambda: mpsa.norm_rope(x, norm=False, q_weight=torch.ones(128, device="cuda")), lambda: mpsa.norm_rope(x, k_weight=torch.ones(128, device="cuda")),
        lambda: mpsa.norm_rope(x, rope=(cos, sin[:8])), lambda: mpsa.norm_rope(x, rope=(cos.half(), sin.half())), lambda: mpsa.norm_rope(x, rope=(cos[:2], sin[:2])),
        lambda: mpsa.norm_rope(x, rope=(cos[:, :6].contiguous(), sin[:, :6].contiguous())), lambda: mpsa.norm_rope(x, positions=i32(0, 1, 2)),
        lambda: mpsa.norm_rope(x, rope=(cos, sin), positions=i32(0, 1)), lambda: mpsa.norm_rope(x, rope=(cos, sin), positions=i32(0, 1, 2).float()),
        lambda: mpsa.norm_rope(x, rope=(cos, sin), sections=(32, 32)), lambda: mpsa.norm_rope(x, rope=(cos, sin), positions=i32(0, 1, 2), sections=(32, 33)),
        lambda: mpsa.norm_rope(x, eps=-1.0), lambda: mpsa.norm_rope(x, eps=float("nan")), lambda: mpsa.norm_rope(x[:, :, :0]),
        lambda: mpsa.norm_rope(torch.zeros(1, 129, 1, 128, device="cuda"), across_heads=True),
        lambda: mpsa.kv_cache(8, 2, 96), lambda: mpsa.kv_cache(8, 2, 128, page_size=48), lambda: mpsa.kv_cache(8, 2, 128, page_size=8),
        lambda: mpsa.kv_cache(0, 2, 128), lambda: mpsa.kv_cache(8, 2, 128, elem="int8"), lambda: mpsa.kv_cache(8, 2, 128, device="cpu"),
        lambda: mpsa.KVCache(c.k, c.k_scale, c.v, c.v_scale[:4]), lambda: mpsa.KVCache(c.k, c.k_scale, c.v.view(torch.int8), c.v_scale),
        lambda: mpsa.KVCache(c.k[:, :, ::2], c.k_scale[:, :, ::2], c.v[:, :, ::2], c.v_scale[:, :, ::2]),
        lambda: mpsa.kv_cache_append(c, kv, kv.half(), tab, i32(0, 0)), lambda: mpsa.kv_cache_append(c, kv, kv[:, :, :2], tab, i32(0, 0)),
        lambda: mpsa.kv_cache_append(c, x, x, tab, i32(0, 0)), lambda: mpsa.kv_cache_append(c, kv, kv, tab.long(), i32(0, 0)),
        lambda: mpsa.kv_cache_append(c, kv, kv, tab[:1], i32(0, 0)), lambda: mpsa.kv_cache_append(c, kv, kv, tab, i32(0)),
        lambda: mpsa.kv_cache_append(c, kv, kv, tab, i32(0, 0).long()), lambda: mpsa.kv_cache_append(c, kv, kv, tab, i32(0, 0), counts=i32(1)),
        lambda: mpsa.kv_cache_append(c, kv[:, :, :0], kv[:, :, :0], tab, i32(0, 0)), lambda: mpsa.kv_cache_append(c, kv, kv, tab.t().contiguous().t(), i32(0, 0)),
        lambda: mpsa.kv_cache_append(c, kv, kv, tab.cpu(), i32(0, 0)),
        lambda: mpsa.kv_cache_read(c, tab, i32(1)), lambda: mpsa.kv_cache_read(c, tab, i32(1, 1), max_len=0),
        lambda: mpsa.kv_cache_read(c, tab, i32(1, 1), out_dtype=torch.float64),
        lambda: mpsa.kv_cache_attention(x.float(), c, tab, i32(3, 3)), lambda: mpsa.kv_cache_attention(x[:, :3], c, tab, i32(3, 3)),
        lambda: mpsa.kv_cache_attention(x[..., :64], c, tab, i32(3, 3)), lambda: mpsa.kv_cache_attention(x, c, tab, i32(3)),
        lambda: mpsa.kv_cache_attention(x, c, tab, i32(3, 3), q_lens=i32(1)), lambda: mpsa.kv_cache_attention(x, c, tab, i32(3, 3), sm_scale=0.0),
        lambda: mpsa.kv_cache_attention(x, c, tab, i32(3, 3), sm_scale=float("nan")), lambda: mpsa.kv_cache_attention(x, c, tab, i32(3, 3), sm_scale=-1.0),
        lambda: mpsa.kv_cache_attention(x, c, tab, i32(3, 3), mask=torch.ones(3, 3, device="cuda")),
        lambda: mpsa.kv_cache_attention(x, c, tab, i32(3, 3), mask=torch.ones(3, 2, dtype=torch.bool, device="cuda")),
        lambda: mpsa.kv_cache_attention(x[:, :, :0], c, tab, i32(3, 3)), lambda: mpsa.kv_cache_attention(x[:0], c, tab[:0], i32()),
        lambda: mpsa.kv_cache_attention(torch.zeros(1, 2, 1025, 128, dtype=BF16, device="cuda"), c, tab[:1], i32(3)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("taken:", i)
    with torch.no_grad():
        mpsa.norm_rope(x, q_weight=w)
