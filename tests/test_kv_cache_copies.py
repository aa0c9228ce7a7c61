"""A cache's calls work on the buffers that it has: copies of a cache have their own, and buffers that a program exchanges are followed."""
import copy
import io
import os
import pickle
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

NAMES = ("k", "k_scale", "v", "v_scale")


@pytest.fixture
def host_cache(monkeypatch):
    """A cache of host buffers: only its argument block is looked at."""
    from mpsa import _lib, serving
    monkeypatch.setattr(_lib, "_native", _lib._LongWay)
    monkeypatch.setattr(serving, "_require_cuda", lambda *_: None)
    return serving.kv_cache(3, 2, 64, page_size=16, elem="e2m1", device="cpu")


def names_its_own(c):
    b = c._block()
    return all(getattr(b, n) == getattr(c, n).data_ptr() for n in NAMES) and (b.num_pages, b.page_size, b.Hkv, b.D, b.elem) == (
        c.k.shape[0], c.page_size, c.num_kv_heads, c.head_dim, {"e4m3": 0, "e5m2": 1, "e2m1": 2}[c.elem])


def by_torch(c):
    f = io.BytesIO()
    torch.save(c, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c)), by_torch, lambda c: copy.deepcopy([c])[0]],
                         ids=["deepcopy", "pickle", "torch.save", "deepcopy of a list"])
def test_copies_name_their_own_buffers(host_cache, how):
    host_cache.k.fill_(7)
    d = how(host_cache)
    assert type(d) is type(host_cache) and d.elem == "e2m1" and torch.equal(d.k, host_cache.k)
    assert all(getattr(d, n).data_ptr() != getattr(host_cache, n).data_ptr() for n in NAMES)
    assert names_its_own(d) and names_its_own(host_cache)


def test_a_shallow_copy_shares_the_buffers(host_cache):
    d = copy.copy(host_cache)
    assert all(getattr(d, n) is getattr(host_cache, n) for n in NAMES) and names_its_own(d)


def test_exchanged_buffers_are_followed_or_refused(host_cache):
    c = host_cache
    old = c.k.data
    c.k.data = torch.zeros_like(c.k)
    assert c.k.data_ptr() != old.data_ptr() and names_its_own(c)
    c.v_scale.set_(torch.zeros_like(c.v_scale))
    assert names_its_own(c)
    for n in NAMES:                                            # (a smaller buffer, and one of another shape, in the same place)
        t, shape = getattr(c, n), getattr(c, n).shape
        t.resize_(2, *shape[1:])
        with pytest.raises(ValueError):
            c._block()
        t.resize_(shape[0], shape[1] // 2, shape[2] * 2, shape[3])
        with pytest.raises(ValueError):
            c._block()
        t.resize_(shape)
        assert names_its_own(c)


@pytest.mark.gpu
@pytest.mark.parametrize("long_way", [False, True])
def test_calls_on_copies_and_exchanged_buffers(long_way, monkeypatch):
    import mpsa
    from mpsa import _lib
    from test_gpu_serving import BF16, filled, rnd
    if long_way:
        monkeypatch.setattr(_lib, "_native", _lib._LongWay)
    g = torch.Generator().manual_seed(31)
    c = filled(g, 8, 2, 16, 64, "e4m3")
    table = torch.tensor([[1, 4, 2], [7, 0, 3]], dtype=torch.int32, device="cuda")
    start = torch.tensor([5, 30], dtype=torch.int32, device="cuda")
    k, v, q = rnd(g, 2, 2, 3, 64).cuda(), rnd(g, 2, 2, 3, 64).cuda(), rnd(g, 2, 4, 3, 64).cuda()

    def everything(cache):
        mpsa.kv_cache_append(cache, k, v, table, start)
        return (*mpsa.kv_cache_read(cache, table, start + 3, max_len=40), mpsa.kv_cache_attention(q, cache, table, start + 3))

    before = [getattr(c, n).clone() for n in NAMES]
    d = copy.deepcopy(c)
    got = everything(d)
    assert all(torch.equal(getattr(c, n), b) for n, b in zip(NAMES, before)) and not torch.equal(d.k, before[0])
    e = pickle.loads(pickle.dumps(c))
    assert all(torch.equal(a, b) for a, b in zip(got, everything(e)))
    # another program's buffers come into the place of the cache's own, which stay as they are
    old = [getattr(c, n).data for n in NAMES]
    for n, b in zip(NAMES, before):
        getattr(c, n).data = b.clone()
    assert all(torch.equal(a, b) for a, b in zip(got, everything(c))) and torch.equal(c.k, d.k)
    assert all(torch.equal(a, b) for a, b in zip(old, before))
    assert all(torch.equal(a, b) for a, b in zip(got, everything(c)))
    c.k.resize_(4, 2, 16, 64)
    for call in (lambda: mpsa.kv_cache_append(c, k, v, table, start), lambda: mpsa.kv_cache_read(c, table, start, max_len=40),
                 lambda: mpsa.kv_cache_attention(q, c, table, start)):
        with pytest.raises(ValueError):
            call()
