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
