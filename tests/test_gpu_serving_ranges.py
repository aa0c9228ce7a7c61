"""Attention over the paged MX cache where keys and values of one sequence differ in size by far, or are nothing at all: for few query rows of a KV
head (T = 1, 6) and for many (T = 40), which are two kernels, against the plain 64-bit form (serving_plain.py)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import serving_plain as P  # noqa: E402
from test_gpu_serving import BF16, FP32, check_attention, half_step, rnd, table_of, tree_mask  # noqa: E402

pytestmark = pytest.mark.gpu


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache_of_rows(g, k, v, elem, page=64):
    """A cache that holds the rows of k, v [B,H,n,D], and its table."""
    import mpsa
    B, H, n, D = k.shape
    m = -(-n // page)
    c = mpsa.kv_cache(B * m, H, D, page_size=page, elem=elem)
    table = table_of(g, B, m, B * m)
    mpsa.kv_cache_append(c, k.cuda(), v.cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32).cuda())
    return c, table


@pytest.mark.parametrize("written", [True, False])
@pytest.mark.parametrize("place", [5, 20000])
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("elem,gap", [("e2m1", 12), ("e4m3", 16), ("e5m2", 24)])
def test_keys_without_values_keep_their_weight(elem, gap, T, place, written):
    """One key with values and 40 000 whose values (and keys) are zero, written as such or left as a new pool has them: their scores are `gap` below
    the one's in log2, and they are in the denominator all the same."""
    import mpsa
    g = torch.Generator().manual_seed(gap)
    n, D, Hq = 40001, 64, 2
    k, v = torch.zeros(1, 1, n, D), torch.zeros(1, 1, n, D)
    k[0, 0, place, 0], v[0, 0, place] = 4.0, 1.0
    if written:
        c, table = cache_of_rows(g, k.to(BF16), v.to(BF16), elem)
    else:
        m = -(-n // 64)
        c, table = mpsa.kv_cache(m, 1, D, elem=elem), table_of(g, 1, m, m)
        mpsa.kv_cache_append(c, k[:, :, place:place + 1].to(BF16).cuda(), v[:, :, place:place + 1].to(BF16).cuda(), table.cuda(), i32(place))
    q = torch.zeros(1, Hq, T, D, dtype=BF16)
    q[..., 0] = 1.0
    sm = gap / 4.0 / math.log2(math.e)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), sm_scale=sm, return_lse=True)
    check_attention(c, table, [n], q, out.cpu(), lse.cpu(), sm=sm)


@pytest.mark.parametrize("octaves", [16, 26, 40, 60])
@pytest.mark.parametrize("T", [6, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_large_values_of_keys_that_a_row_does_not_see(elem, T, octaves):
    """A drafted token's values are larger than all others' by far: the drafts that do not see it have the same result as without it, over few keys
    and over many."""
    import mpsa
    g = torch.Generator().manual_seed(octaves)
    D, Hq, Hkv = 64, 2, 1
    for n in (T + 90, 32768 + T):
        k, v = rnd(g, 1, Hkv, n, D), rnd(g, 1, Hkv, n, D)
        v[:, :, n - T + 2] *= 2.0 ** octaves
        c, table = cache_of_rows(g, k, v, elem)
        q = rnd(g, 1, Hq, T, D)
        mask = tree_mask(g, T)
        mask[:, 2] = False
        mask[2, 2] = True
        args = (q.cuda(), c, table.cuda(), i32(n))
        out, lse = mpsa.kv_cache_attention(*args, mask=mask.cuda(), return_lse=True)
        check_attention(c, table, [n], q, out.cpu(), lse.cpu(), mask=mask)


@pytest.mark.parametrize("place", [3, 700])
@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_large_values_of_improbable_keys(elem, T, place):
    """A key whose score is 120 below the others' in log2 has values that are 2^60 larger: with its weight it is nothing, and it takes nothing from
    the keys beside it."""
    import mpsa
    g = torch.Generator().manual_seed(place)
    n, D, Hq = 1000, 64, 4
    k, v = rnd(g, 1, 1, n, D), rnd(g, 1, 1, n, D)
    k[..., 0] = 0.0
    k[:, :, place] = 0.0
    k[:, :, place, 0] = -16.0
    v[:, :, place] *= 2.0 ** 60
    q = rnd(g, 1, Hq, T, D)
    q[..., 0] = 120.0 / 16.0 / math.log2(math.e) * 8.0 * 1.01
    c, table = cache_of_rows(g, k, v, elem)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), return_lse=True)
    check_attention(c, table, [n], q, out.cpu(), lse.cpu())


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_a_block_of_a_key_that_is_larger_than_its_others(elem, T):
    """All keys' values are 2^26 larger in their first 32 depth elements: the others keep the bits that 2^-32 of a key's largest product leaves."""
    import mpsa
    g = torch.Generator().manual_seed(5)
    n, D, Hq = 700, 128, 4
    k, v = rnd(g, 1, 1, n, D), 1.0 + torch.rand(1, 1, n, D, generator=g)
    v[..., :32] *= 2.0 ** 26
    c, table = cache_of_rows(g, k, v.to(BF16), elem)
    q = rnd(g, 1, Hq, T, D, amp=0.1)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), return_lse=True)
    check_attention(c, table, [n], q, out.cpu(), lse.cpu())
    k, v = (P.values(P.gather(getattr(c, x), table[0], n), P.gather(getattr(c, x + "_scale"), table[0], n), elem) for x in ("k", "v"))
    # P times the block's scale and, with many rows, the element in units of its key's largest are held to 2^-25 of what is 2^7 for the largest
    # product of the row: 2^-32 of it each, and at most twice that with elements of up to twice the others in size; of 700 keys at most
    seen = torch.ones(T, n, dtype=torch.bool)
    seen[:, n - T:] = torch.ones(T, T).tril().bool()
    o, _, a, _, big = P.attention(q[0].double(), k, v, seen, D ** -0.5)
    err = (out[0].cpu().double() - o).abs()[..., 32:]
    tol = (half_step(BF16) * o.abs() * 1.01 + 2.0 ** -10 * a + n * 2.0 ** -30 * big.unsqueeze(-1))[..., 32:]
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("octaves", [10, 24, 27, 32, 40, 60, 100])
@pytest.mark.parametrize("T", [1, 6, 40])
def test_scores_of_any_size(T, octaves, sign):
    """Scores so large that neighbouring fp32 numbers are further apart than the logarithms of two weights: the largest key has all the weight, and
    the row is not empty.  Keys have one element and differ by an eighth at least, so that the largest one is so in any rounding."""
    import mpsa
    g = torch.Generator().manual_seed(octaves)
    n, D, Hq = 700, 64, 4
    k, v = torch.zeros(1, 1, n, D), rnd(g, 1, 1, n, D)
    size = torch.randint(2, 9, (n,), generator=g).float() / 16
    size[n - T] = size[0] = size[320] = 0.25                   # (what the first draft sees at the least, and what is seen with it)
    best = 333
    size[best] = 0.625 if sign > 0 else 0.0625
    k[0, 0, :, 0] = size * sign
    q = rnd(g, 1, Hq, T, D)
    q[..., 0] = 1.40625 * 2.0 ** octaves
    c, table = cache_of_rows(g, k.to(BF16), v, "e4m3")
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), return_lse=True)
    if octaves == 10:                                          # (scores that still matter)
        check_attention(c, table, [n], q, out.cpu(), lse.cpu())
        return
    held = P.values(P.gather(c.v, table[0], n), P.gather(c.v_scale, table[0], n), "e4m3")[0, best]
    # the weight of the one key is exactly 1 where all others' are 0: P is a power of two then or has its rounding to fp16, 2^-11
    assert bool(((out[0].cpu().double() - held).abs() <= (half_step(BF16) * 1.01 + 2.0 ** -11) * held.abs() + 2.0 ** -24).all())
    s = 1.40625 * 2.0 ** octaves * float(k[0, 0, best, 0]) * D ** -0.5 * math.log2(math.e)
    assert bool(((lse.cpu().double() - s).abs() <= 2.0 ** -20 * abs(s) + 2.0 ** -16).all())


def check_by_key(c, table, n, q, out, lse, mask=None):
    """As check_attention for one sequence, with each key's score held to its own size.

    Score j is off by (D + 8) 2^-23 of the sum of its own terms' magnitudes, and by what an operand cannot hold: 2^-31 of the key's largest element and
    2^-25 of the row's largest query element in each term.  That moves P_j by a factor exp(d_j); out = sum P v / sum P then moves by at most
    sum |dP_j| (|v_j| + |out|) / sum P.  The rest is check_attention's."""
    T, D = q.shape[2], q.shape[3]
    G = q.shape[1] // c.num_kv_heads
    k, v = (P.values(P.gather(getattr(c, x), table[0], n), P.gather(getattr(c, x + "_scale"), table[0], n), c.elem).repeat_interleave(G, 0) for x in ("k", "v"))
    seen = torch.ones(T, n, dtype=torch.bool)
    seen[:, n - T:] = torch.ones(T, T).tril().bool() if mask is None else mask
    x, sm = q[0].double(), D ** -0.5
    s = torch.where(seen, x @ k.transpose(1, 2) * sm, float("-inf"))
    d = (D + 8) * 2.0 ** -23 * (x.abs() @ k.abs().transpose(1, 2)) + 2.0 ** -31 * x.abs().sum(-1, keepdim=True) * k.abs().amax(-1).unsqueeze(1)
    d = (d + 2.0 ** -25 * x.abs().amax(-1, keepdim=True) * k.abs().sum(-1).unsqueeze(1)) * sm + 2.0 ** -22
    l = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - l)
    move = torch.where(seen, torch.exp(torch.minimum(s - l + d, torch.tensor(700.0, dtype=torch.float64))) - p, 0.0)
    o, a = p @ v, p @ v.abs()
    got, gl = out[0].double(), lse[0].double()
    tol = half_step(q.dtype) * o.abs() * 1.01 + (2.0 ** -11 + 2.0 ** -16) * a + 1.01 * (move @ v.abs() + o.abs() * move.sum(-1, keepdim=True))
    tol = tol + n * 2.0 ** -31 * (p * v.abs().amax(-1).unsqueeze(1)).amax(-1, keepdim=True) + 2.0 ** -24
    assert bool(((got - o).abs() <= tol).all()), float(((got - o).abs() / tol).max())
    l = l.squeeze(-1) * math.log2(math.e)
    assert bool(((gl - l).abs() <= torch.log2(1 + move.sum(-1)) * 1.01 + 2.0 ** -16 + 2.0 ** -23 * l.abs()).all())
    return float((tol < 0.1 * a + 1e-3).double().mean())       # (where a score is held to less than a bit nothing is tested)


@pytest.mark.parametrize("octaves", [12, 26, 40, 60])
@pytest.mark.parametrize("T", [6, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_large_keys_that_a_row_does_not_see(elem, T, octaves):
    import mpsa
    g = torch.Generator().manual_seed(octaves + 1)
    D, Hq, Hkv, n = 64, 4, 2, T + 90
    k, v = rnd(g, 1, Hkv, n, D), rnd(g, 1, Hkv, n, D)
    k[:, :, n - T + 2] *= 2.0 ** octaves
    c, table = cache_of_rows(g, k, v, elem)
    q = rnd(g, 1, Hq, T, D)
    mask = tree_mask(g, T)
    mask[:, 2] = False
    mask[2, 2] = True
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), mask=mask.cuda(), return_lse=True)
    keep = [t for t in range(T) if t != 2]                     # (the draft itself: a softmax of one key, or of all but it)
    check_by_key(c, table, n, q, out.cpu(), lse.cpu(), mask)
    only = torch.ones(T, n, dtype=torch.bool)
    only[:, n - T:] = mask
    k, v = (P.values(P.gather(getattr(c, x), table[0], n), P.gather(getattr(c, x + "_scale"), table[0], n), elem) for x in ("k", "v"))
    o, _, a, mag, big = P.attention(q[0].double(), k, v, only, D ** -0.5)
    tol = half_step(BF16) * o.abs() * 1.01 + (2 * ((D + 8) * 2.0 ** -23 * mag.unsqueeze(-1) + 2.0 ** -22) + 2.0 ** -11 + 2.0 ** -16) * a + n * 2.0 ** -31 * big.unsqueeze(-1) + 2.0 ** -24
    assert bool(((out[0].cpu().double() - o).abs() <= tol)[:, keep].all())


@pytest.mark.parametrize("octaves", [12, 26, 60])
@pytest.mark.parametrize("place", [3, 700])
@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_large_keys_without_weight(elem, T, place, octaves):
    """A key that is larger than the others by far, against the queries: its weight is nothing, and the others' scores are their own."""
    import mpsa
    g = torch.Generator().manual_seed(place)
    n, D, Hq = 1000, 64, 4
    k, v = rnd(g, 1, 1, n, D), rnd(g, 1, 1, n, D)
    k[..., 0] = 0.0
    k[:, :, place] = 0.0
    k[:, :, place, 0] = -2.0 ** octaves
    q = rnd(g, 1, Hq, T, D)
    q[..., 0] = 4.0
    c, table = cache_of_rows(g, k, v, elem)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), return_lse=True)
    assert check_by_key(c, table, n, q, out.cpu(), lse.cpu()) > 0.99


@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_keys_and_values_of_all_sizes(elem, T):
    """Keys from 2^-40 to 2^8 and values from 2^-30 to 2^30 of the usual, side by side; drafts that see few of them among them."""
    import mpsa
    g = torch.Generator().manual_seed(T)
    D, Hq, n = 128, 2, 900
    k = rnd(g, 1, 1, n, D, dtype=FP32) * torch.exp2(torch.randint(-40, 9, (1, 1, n, 1), generator=g).float()) * 2.0 ** -6
    v = rnd(g, 1, 1, n, D, dtype=FP32) * torch.exp2(torch.randint(-30, 31, (1, 1, n, 1), generator=g).float())
    c, table = cache_of_rows(g, k, v, elem)
    q = rnd(g, 1, Hq, T, D)
    out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), return_lse=True)
    check_by_key(c, table, n, q, out.cpu(), lse.cpu())


@pytest.mark.parametrize("place", [2, 250, 19000])
@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_keys_without_values_beside_one_with_large_ones(elem, T, place):
    """All values are zero but those of one key, which are 2^60: every key has its weight, where a warp, a CTA or a part of the keys has seen nothing but
    zeros, too."""
    import mpsa
    g = torch.Generator().manual_seed(place)
    D, Hq = 64, 2
    for n in (300, 20000):
        if place >= n - T:
            continue
        k, v = rnd(g, 1, 1, n, D), torch.zeros(1, 1, n, D, dtype=BF16)
        v[0, 0, place] = 2.0 ** 60
        c, table = cache_of_rows(g, k, v, elem)
        q = rnd(g, 1, Hq, T, D, amp=0.5)
        out, lse = mpsa.kv_cache_attention(q.cuda(), c, table.cuda(), i32(n), return_lse=True)
        check_attention(c, table, [n], q, out.cpu(), lse.cpu())
