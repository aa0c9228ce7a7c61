"""A prompt in chunks: append a chunk, read the whole prefix back, and the mixed-precision prefill over it (attention_forward)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import serving_plain as P  # noqa: E402
from test_gpu_serving import BF16, rnd, table_of  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("chunks", [[(300, 300), (17, 17), (200, 200)], [(300, 120), (64, 200)]], ids=["one length", "ragged"])
def test_prefill_over_the_cached_prefix(chunks, elem):
    """The result is the prefill's over the values that the cache stands for, exactly: in one call where all sequences have one length, and for a ragged
    batch a sequence at a time over its own length.  And it is attention over them, as near as the prefill's formats are."""
    import mpsa
    g = torch.Generator().manual_seed(41)
    B, Hq, Hkv, D, page = 2, 4, 2, 128, 32
    m = 20
    c = mpsa.kv_cache(B * m, Hkv, D, page_size=page, elem=elem)
    table = table_of(g, B, m, B * m)
    held = [0] * B
    for counts in chunks:
        T = max(counts)
        q, k, v = rnd(g, B, Hq, T, D), rnd(g, B, Hkv, T, D), rnd(g, B, Hkv, T, D)
        mpsa.kv_cache_append(c, k.cuda(), v.cuda(), table.cuda(), torch.tensor(held, dtype=torch.int32).cuda(), counts=torch.tensor(counts, dtype=torch.int32).cuda())
        held = [h + n for h, n in zip(held, counts)]
        lengths = torch.tensor(held, dtype=torch.int32).cuda()
        keys, values = mpsa.kv_cache_read(c, table.cuda(), lengths, max_len=max(held))
        if len(set(held)) == 1:
            got = mpsa.attention_forward(q.cuda(), keys, values, causal=True, uniform="fp8")
        for b, (n, t) in enumerate(zip(held, counts)):
            x, y = (P.values(P.gather(getattr(c, s), table[b], n), P.gather(getattr(c, s + "_scale"), table[b], n), elem) for s in ("k", "v"))
            ref = mpsa.attention_forward(q[b:b + 1, :, :t].contiguous().cuda(), x.to(BF16)[None].cuda(), y.to(BF16)[None].cuda(), causal=True, uniform="fp8")
            own = mpsa.attention_forward(q[b:b + 1, :, :t].cuda(), keys[b:b + 1, :, :n], values[b:b + 1, :, :n], causal=True, uniform="fp8")
            assert torch.equal(own, ref)
            if len(set(held)) == 1:
                assert torch.equal(got[b:b + 1], ref)
            seen = torch.ones(t, n, dtype=torch.bool)
            seen[:, n - t:] = torch.ones(t, t).tril().bool()
            o = P.attention(q[b, :, :t].double(), x, y, seen, D ** -0.5)[0]
            assert float(torch.nn.functional.cosine_similarity(own[0].cpu().double().flatten(), o.flatten(), dim=0)) > 0.99
