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
