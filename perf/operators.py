"""The calls that serve a model token by token beside the mixed-precision prefill, with their inputs, least work and exact values.

`listed()` are fixed cases, `draw(rng)` gives more of the same ranges; `prepare` makes what a program has in hand before the call, `run` is
one pass.  With `own` set, `run` goes through the framework's entry points; otherwise it computes the same in elementary torch operations.

  rope    queries and keys of one layer: RMS norm of each head (or across the heads) and rotary positions with one or several axes
  append  keys and values of new tokens quantised into a paged MX cache
  refill  the same, and the whole cached sequences read back in 16 bits, as a prompt processed in chunks does it
  read    cached sequences read back in 16 bits
  attend  queries of one token, of a chunk or of a tree of drafted tokens against the cache

The cache's numbers: blocks of 32 along the depth share a power of two, the smallest one at which no element of the block exceeds the
element type's largest value; elements are rounded to nearest, ties to even.  A block that holds a NaN or an infinity has the scale code
255 (NaN) and zero element codes.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = {"e4m3": (8, 1.75), "e5m2": (15, 1.75), "e2m1": (2, 1.5)}          # exponent and significand of the largest element
FLOAT8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


# ---------------------------------------------------------------------------------------------------------------- cases
def _rope(B, L, Hq, Hkv, D, dtype="bf16", layout="HND", norm="head", axes=1, rot=0, interleaved=False, **name):
    return dict(name, kind="rope", B=B, L=L, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, layout=layout, norm=norm, axes=axes, rot=rot or D,
                interleaved=interleaved)


def _append(kind, B, T, held, Hkv, D, elem, page, dtype="bf16", layout="HND", **name):
    return dict(name, kind=kind, B=B, T=T, held=held, Hkv=Hkv, D=D, elem=elem, page=page, dtype=dtype, layout=layout)


def _read(B, L, Hkv, D, elem, page, dtype="bf16", **name):
    return dict(name, kind="read", B=B, L=L, Hkv=Hkv, D=D, elem=elem, page=page, dtype=dtype)


def _attend(B, T, L, Hq, Hkv, D, elem, page, dtype="bf16", layout="HND", tree=False, ragged=True, **name):
    return dict(name, kind="attend", B=B, T=T, L=L, Hq=Hq, Hkv=Hkv, D=D, elem=elem, page=page, dtype=dtype, layout=layout, tree=tree,
                ragged=ragged)


def listed():
    return [
        # one decoding step of 32 sequences in a grouped-query layer: the smallest call, latency
        _rope(32, 1, 32, 8, 128, name="rope_decode_32"),
        # a prompt of the benchmark's length
        _rope(1, 32768, 32, 8, 128, name="rope_prefill_32k"),
        # video latents, 21 x 39 x 40 tokens first, norm across the heads, three axes, neighbouring pairs
        _rope(1, 32760, 40, 40, 128, layout="NHD", norm="across", axes=3, interleaved=True, name="rope_video_32760"),
        # one token of 32 sequences goes into the cache in each decoding step
        _append("append", 32, 1, 4096, 8, 128, "e4m3", 64, name="append_decode_32"),
        # a prompt goes into the cache, tokens first as the projection leaves them; an odd count in odd places
        _append("append", 2, 4099, 777, 8, 128, "e4m3", 64, layout="NHD", name="append_prompt_4099"),
        # a chunk of a prompt goes into the 4-bit cache, whose whole prefix comes back for the prefill of that chunk
        _append("refill", 1, 512, 7680, 8, 128, "e2m1", 64, name="refill_chunk_512"),
        # prefixes kept in the cache come back in 16 bits
        _read(4, 8192, 8, 128, "e4m3", 64, name="read_prefix_8k"),
        # one token of one sequence
        _attend(1, 1, 4096, 32, 8, 128, "e4m3", 64, ragged=False, name="decode_1_of_4k"),
        # one token of each of a ragged batch
        _attend(32, 1, 16384, 32, 8, 128, "e4m3", 64, name="decode_32_ragged_16k"),
        # four long contexts held in 4 bits
        _attend(4, 1, 131072, 32, 8, 128, "e2m1", 128, ragged=False, name="decode_4_of_128k_fp4"),
        # fp16, depth 64, a few heads of their own keys, odd lengths in short pages
        _attend(7, 1, 3001, 12, 12, 64, "e5m2", 16, "fp16", "NHD", name="decode_7_of_3001_d64"),
        # trees of 32 drafted tokens verified at once
        _attend(8, 32, 32768, 32, 8, 128, "e4m3", 64, tree=True, name="tree_32_of_32k"),
    ]


def _size(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["rope", "rope", "append", "refill", "read", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    layout = rng.choice(["HND", "NHD"])
    D = rng.choice([64, 128, 128])
    if kind == "rope":
        Hkv = rng.choice([1, 2, 4, 8, 12, 16])
        Hq = Hkv * rng.choice([1, 2, 3, 4])
        B = rng.choice([1, 1, 2, 5, 32])
        axes = rng.choice([1, 1, 2, 3])
        return _rope(B, _size(rng, 1, 65536 // B), Hq, Hkv, D, dtype, layout, rng.choice(["head", "head", "across", "none"]), axes,
                     D if axes > 1 else rng.choice([D, D, D // 2]), rng.random() < 0.5)
    elem = rng.choice(["e4m3", "e4m3", "e5m2", "e2m1"])
    page = rng.choice([16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    if kind in ("append", "refill"):
        B = rng.choice([1, 2, 7, 32])
        T, held = _size(rng, 1, 8192 // B), rng.choice([0, _size(rng, 1, 16384 // B)])
        return _append(kind, B, T, held, Hkv, D, elem, page, dtype, layout)
    if kind == "read":
        B = rng.choice([1, 2, 7])
        return _read(B, _size(rng, 1, 32768 // B), Hkv, D, elem, page, dtype)
    B = _size(rng, 1, 64)
    G = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    L = _size(rng, 1, min(131072, 4 * 131072 * 8 // (B * Hkv)))
    T, tree = 1, False
    if rng.random() < 0.5:
        T, tree = _size(rng, 2, 64), rng.random() < 0.7
        L = max(L, T)
        while B * L * T * G * Hkv > 8 * 32768 * 32 * 32 and B > 1:
            B = B // 2
        L = max(T, min(L, 8 * 32768 * 32 * 32 // (B * T * G * Hkv)))
    return _attend(B, T, L, G * Hkv, Hkv, D, elem, page, dtype, layout, tree)


# ----------------------------------------------------------------------------------------- the cache's numbers, plain form
def _quantise(x, elem):
    """x fp32 [..., D] -> element codes uint8 ([..., D], or [..., D/2] with two 4-bit codes a byte, the lower depth in the low half) and
    scale codes uint8 [..., D/32]."""
    D = x.shape[-1]
    b = x.reshape(*x.shape[:-1], D // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)                       # (a NaN is the largest)
    fine = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(fine, amax, 0.0))            # amax = m 2^e, m in [0.5, 1)
    top, largest = LARGEST[elem]
    e = (e - 1 - top + (2.0 * m > largest)).clamp(-126, 127)
    e = torch.where(amax > 0, e, -126)
    y = torch.where(fine, b, 0.0) * torch.exp2(-e.double()).float()
    if elem == "e2m1":
        a = y.abs()
        a = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
        code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)      # 0 .5 1 1.5 2 3 4 6 -> 0 .. 7
        code = (code + torch.signbit(y).to(torch.uint8) * 8).reshape(*x.shape[:-1], D // 2, 2)
        code = code[..., 0] + code[..., 1] * 16
    else:
        code = y.to(FLOAT8[elem]).view(torch.uint8).reshape(x.shape)
    return code, torch.where(fine, e + 127, 255).to(torch.uint8).squeeze(-1)


def _values(code, scale, elem):
    """What codes and scale codes stand for, fp32 [..., D]."""
    if elem == "e2m1":
        code = torch.stack((code & 15, code >> 4), -1).flatten(-2)
        n = (code & 7).float()
        v = torch.where(n < 4, n / 2, torch.where(n < 6, n - 2, 2 * n - 8)) * (1.0 - 2.0 * (code >> 3).float())
    else:
        v = code.view(FLOAT8[elem]).float()
    s = torch.exp2(scale.double() - 127).float()
    s = torch.where(scale == 255, float("nan"), s)
    return (v.reshape(*scale.shape, 32) * s.unsqueeze(-1)).flatten(-2)


def _pages(buf, table):
    """[pages, Hkv, page, n] seen through a page table [B, m]: [B, Hkv, m * page, n]."""
    return buf[table.long()].transpose(1, 2).flatten(2, 3)


# --------------------------------------------------------------------------------------------------------------- inputs
def _tensor(g, shape, dtype, layout):
    """Logical [B,H,L,D], in memory as the layout says; a few channels are larger than the others, as keys have them."""
    B, H, L, D = shape
    x = torch.randn(B, L, H, D, generator=g, device="cuda", dtype=torch.float32)
    x = x * (1.0 + 3.0 * (torch.rand(1, 1, H, D, generator=g, device="cuda") > 0.95).float())
    x = x.to(dtype)
    return x if layout == "NHD" else x.transpose(1, 2).contiguous()


def _table(g, B, tokens, page):
    """Pages scattered over a pool that is a little larger than the batch needs."""
    m = max(1, -(-tokens // page))
    n = B * m + 3
    return n, torch.randperm(n, generator=g, device="cuda")[: B * m].to(torch.int32).reshape(B, m).contiguous()


def _cache(g, n, Hkv, page, D, elem):
    """A pool of pages with the codes that earlier requests left."""
    out = {}
    for name in ("k", "v"):
        code = torch.empty(n, Hkv, page, D // 2 if elem == "e2m1" else D, dtype=torch.uint8, device="cuda")
        scale = torch.empty(n, Hkv, page, D // 32, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (Hkv * page * D))
        wide = 1.0 + 3.0 * (torch.rand(1, Hkv, 1, D, generator=g, device="cuda") > 0.95).float()
        for i in range(0, n, step):
            x = torch.randn(min(step, n - i), Hkv, page, D, generator=g, device="cuda") * (wide if name == "k" else 1.0)
            code[i:i + step], scale[i:i + step] = _quantise(x, elem)
        out[name], out[name + "_scale"] = code, scale
    return out


def _sections(case):
    h = case["rot"] // 2
    a = case["axes"]
    rest = h // 3 if a == 3 else h // a
    return (h - (a - 1) * rest,) + (rest,) * (a - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    c, dev = case, "cuda"
    B, D, dt = c["B"], c["D"], DTYPE[c["dtype"]]
    s = {"case": case}
    if c["kind"] == "rope":
        L, layout = c["L"], c["layout"]
        s["q"], s["k"] = _tensor(g, (B, c["Hq"], L, D), dt, layout), _tensor(g, (B, c["Hkv"], L, D), dt, layout)
        for n, H in (("q", c["Hq"]), ("k", c["Hkv"])):
            size = {"head": (D,), "across": (H, D), "none": None}[c["norm"]]
            s[n + "_weight"] = None if size is None else (1.0 + 0.2 * torch.randn(size, generator=g, device=dev)).to(dt)
        sec = _sections(c)
        if c["axes"] == 1:
            start = torch.randint(0, 4096, (B, 1), generator=g, device=dev)
            pos = start + torch.arange(L, device=dev)
            rows = 4096 + L
        else:                                    # a grid whose later axes are short, walked in rows
            side = max(1, int(round((L * 0.6) ** (1.0 / c["axes"]))))
            i = torch.arange(L, device=dev)
            pos = [i // side ** (c["axes"] - 1)] + [(i // side ** (c["axes"] - 1 - a)) % side for a in range(1, c["axes"])]
            pos = torch.stack(pos, -1).expand(B, L, c["axes"])
            rows = int(pos.max()) + 1
        s["positions"] = pos.to(torch.int32).contiguous()
        inv = torch.cat([10000.0 ** (-torch.arange(n, device=dev, dtype=torch.float64) / n) for n in sec])
        ang = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        return s
    Hkv, elem, page = c["Hkv"], c["elem"], c["page"]
    if c["kind"] in ("append", "refill"):
        T = c["T"]
        held = torch.randint(c["held"] // 2, c["held"] + 1, (B,), generator=g, device=dev)
        held[0] = c["held"]
        n, s["table"] = _table(g, B, c["held"] + T, page)
        s["cache"] = _cache(g, n, Hkv, page, D, elem)
        s["held"] = held.to(torch.int32)
        s["lengths"] = s["held"] + T
        s["k"], s["v"] = _tensor(g, (B, Hkv, T, D), dt, c["layout"]), _tensor(g, (B, Hkv, T, D), dt, c["layout"])
        return s
    L = c["L"]
    n, s["table"] = _table(g, B, L, page)
    s["cache"] = _cache(g, n, Hkv, page, D, elem)
    if c["kind"] == "read":
        lens = torch.randint(L // 2, L + 1, (B,), generator=g, device=dev)
        lens[0] = L
        s["lengths"] = lens.to(torch.int32)
        return s
    T, Hq = c["T"], c["Hq"]
    qlens = torch.full((B,), T, device=dev)
    lens = torch.full((B,), L, device=dev)
    if c["ragged"]:
        if T > 1:
            qlens = torch.randint(1, T + 1, (B,), generator=g, device=dev)
        lens = qlens + torch.randint(0, L - T + 1, (B,), generator=g, device=dev)
        qlens[0], lens[0] = T, L
    s["lengths"], s["q_lens"] = lens.to(torch.int32), qlens.to(torch.int32) if T > 1 else None
    s["q"] = _tensor(g, (B, Hq, T, D), dt, c["layout"])
    s["mask"] = None
    if c["tree"]:                                # every drafted token sees its ancestors and itself
        r = np.random.RandomState(int(seed) % (1 << 31))
        m = np.zeros((B, T, T), dtype=bool)
        for b in range(B):
            for i in range(T):
                if i:
                    m[b, i] = m[b, r.randint(max(0, i - 8), i)]
                m[b, i, i] = True
        s["mask"] = torch.from_numpy(m).to(dev)
    return s


# ------------------------------------------------------------------------------------------------------------- one pass
def _mpsa():
    pkg = os.path.abspath("mp-sparse-attn_b200")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import mpsa
    return mpsa


def _run_own(s):
    mpsa, c = _mpsa(), s["case"]
    kind = c["kind"]
    if kind == "rope":
        return mpsa.norm_rope(s["q"], s["k"], q_weight=s["q_weight"], k_weight=s["k_weight"], norm=c["norm"] != "none",
                              across_heads=c["norm"] == "across", rope=(s["cos"], s["sin"]), positions=s["positions"],
                              sections=_sections(c) if c["axes"] > 1 else None, interleaved=c["interleaved"], tensor_layout=c["layout"])
    d = s["cache"]
    cache = mpsa.KVCache(d["k"], d["k_scale"], d["v"], d["v_scale"], c["elem"])
    if kind == "attend":
        return mpsa.kv_cache_attention(s["q"], cache, s["table"], s["lengths"], q_lens=s["q_lens"], mask=s["mask"], return_lse=True,
                                       tensor_layout=c["layout"])
    if kind != "read":
        mpsa.kv_cache_append(cache, s["k"], s["v"], s["table"], s["held"], tensor_layout=c["layout"])
        if kind == "append":
            return _held(d, c["elem"])
    return mpsa.kv_cache_read(cache, s["table"], s["lengths"], max_len=_longest(c), out_dtype=DTYPE[c["dtype"]])


def _longest(c):
    return c["L"] if c["kind"] == "read" else c["held"] + c["T"]


def _held(d, elem):
    """The cache's own buffers; 8-bit elements as the values they stand for (scale codes are exponents, and 4-bit codes stay packed)."""
    if elem == "e2m1":
        return dict(d)
    return {n: t.view(FLOAT8[elem]) if n in ("k", "v") else t for n, t in d.items()}


def _heads_first(x, layout):
    return x if layout == "HND" else x.transpose(1, 2)


def _rope_plain(x, w, s, c):
    y = _heads_first(x, c["layout"]).float()
    if c["norm"] != "none":
        ms = y.square().mean((1, 3) if c["norm"] == "across" else (3,), keepdim=True)
        w = w.float().reshape(1, -1, 1, c["D"]) if c["norm"] == "across" else w.float()
        y = y * (1.0 / torch.sqrt(ms + 1e-6)) * w
    h = c["rot"] // 2
    pos = s["positions"].long()
    if c["axes"] > 1:
        axis = torch.repeat_interleave(torch.arange(c["axes"], device=y.device), torch.tensor(_sections(c), device=y.device))
        pos = pos[..., axis]
        cos, sin = (t[pos, torch.arange(h, device=y.device)].unsqueeze(1) for t in (s["cos"], s["sin"]))
    else:
        cos, sin = (t[pos].unsqueeze(1) for t in (s["cos"], s["sin"]))
    a, b = (y[..., 0:2 * h:2], y[..., 1:2 * h:2]) if c["interleaved"] else (y[..., :h], y[..., h:2 * h])
    u, v = a * cos - b * sin, b * cos + a * sin
    y = torch.cat((torch.stack((u, v), -1).flatten(-2) if c["interleaved"] else torch.cat((u, v), -1), y[..., 2 * h:]), -1)
    return _heads_first(y, c["layout"]).to(x.dtype).contiguous()


def _append_plain(s, c):
    d, page, T = s["cache"], c["page"], c["T"]
    at = s["held"].long()[:, None] + torch.arange(T, device="cuda")                     # [B, T]
    slot = s["table"].long().gather(1, at // page)
    for n in ("k", "v"):
        x = s[n] if c["layout"] == "NHD" else s[n].transpose(1, 2)                      # [B, T, Hkv, D]
        code, scale = _quantise(x.float(), c["elem"])
        d[n][slot, :, at % page] = code
        d[n + "_scale"][slot, :, at % page] = scale


def _read_plain(s, c):
    L, out = _longest(c), []
    there = (torch.arange(L, device="cuda") < s["lengths"][:, None])[:, None, :, None]
    for n in ("k", "v"):
        x = _values(_pages(s["cache"][n], s["table"]), _pages(s["cache"][n + "_scale"], s["table"]), c["elem"])[:, :, :L]
        out.append(torch.where(there, x, 0.0).to(DTYPE[c["dtype"]]))
    return tuple(out)


def _attend_plain(s, c):
    B, T, Hq, Hkv, D = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"]
    d, table = s["cache"], s["table"]
    n = table.shape[1] * c["page"]
    at = torch.arange(n, device="cuda")
    lens = s["lengths"].long()[:, None]
    qlens = s["q_lens"].long()[:, None] if s["q_lens"] is not None else torch.full_like(lens, T)
    there = (at < lens)[:, None, :, None]
    q = _heads_first(s["q"], c["layout"]).float().reshape(B, Hkv, (Hq // Hkv) * T, D)
    k = torch.where(there, _values(_pages(d["k"], table), _pages(d["k_scale"], table), c["elem"]), 0.0)
    sc = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    del k
    i = torch.arange(T, device="cuda")[None, :, None]
    j = (at - (lens - qlens))[:, None, :]                                                # [B, 1, n]: which of the call's tokens a key is
    if s["mask"] is not None:
        seen = s["mask"].gather(2, j.clamp(0, T - 1).expand(B, T, n)) | (j < 0)
    else:
        seen = j <= i
    seen = seen & (at < lens)[:, None, :] & (i < qlens[:, :, None])                      # [B, T, n]
    sc = torch.where(seen[:, None, None], sc.reshape(B, Hkv, Hq // Hkv, T, n), float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(sc - m)
    del sc
    l = p.sum(-1, keepdim=True)
    v = torch.where(there, _values(_pages(d["v"], table), _pages(d["v_scale"], table), c["elem"]), 0.0)
    o = torch.matmul(p.reshape(B, Hkv, -1, n), v).reshape(B, Hq, T, D)
    l, m = l.reshape(B, Hq, T, 1), m.reshape(B, Hq, T, 1)
    o = torch.where(l > 0, o / l, 0.0).to(s["q"].dtype)
    lse = torch.where(l > 0, (m + torch.log(l)) * math.log2(math.e), float("-inf")).squeeze(-1)
    return _heads_first(o, c["layout"]).contiguous(), lse


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["kind"] == "rope":
        return tuple(_rope_plain(state[n], state[n + "_weight"], state, c) for n in ("q", "k"))
    if c["kind"] == "attend":
        return _attend_plain(state, c)
    if c["kind"] != "read":
        _append_plain(state, c)
        if c["kind"] == "append":
            return _held(state["cache"], c["elem"])
    return _read_plain(state, c)


# ------------------------------------------------------------------------------------------------------------ least work
def _row_bytes(D, elem):
    return (D // 2 if elem == "e2m1" else D) + D // 32


def work(case):
    c = case
    B, D = c["B"], c["D"]
    w = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "rope":
        rows = B * c["L"] * (c["Hq"] + c["Hkv"])
        table = min(B * c["L"], 4096 + c["L"]) * (c["rot"] // 2) * 8 if c["axes"] == 1 else 0
        return {"bytes": 2 * rows * D * w + table + B * c["L"] * c["axes"] * 4, "flops": rows * (4 * D + 3 * c["rot"])}
    row = 2 * c["Hkv"] * _row_bytes(D, c["elem"])                      # one token's keys and values in the cache
    wide = 2 * c["Hkv"] * D * w
    if c["kind"] == "append":
        return {"bytes": B * c["T"] * (row + wide), "flops": B * c["T"] * c["Hkv"] * D * 6}
    if c["kind"] == "refill":
        n = B * (c["held"] + c["T"]) if B == 1 else int(B * (0.75 * c["held"] + c["T"]))
        return {"bytes": B * c["T"] * (row + wide) + (n * row + B * (c["held"] + c["T"]) * wide), "flops": n * c["Hkv"] * D * 4}
    n = B * c["L"] if B == 1 or not c.get("ragged", True) else int(c["L"] + (B - 1) * (0.75 if c["kind"] == "read" else 0.5) * c["L"])
    if c["kind"] == "read":
        return {"bytes": n * row + B * c["L"] * wide, "flops": n * c["Hkv"] * D * 4}
    t = c["T"] if c["T"] == 1 or not c["ragged"] else (c["T"] + 1) / 2
    return {"bytes": n * row + 2 * B * c["T"] * c["Hq"] * D * w + B * c["T"] * c["Hq"] * 4, "flops": 4 * n * t * c["Hq"] * D}


# --------------------------------------------------------------------------------------- the definition, in 64 bits
def _two_to(e):
    """2^e for whole e (a power of two to 32 bits is exact; a double's exp2 need not be)."""
    return torch.exp2(e).float().double()


def _exact_values(code, scale, elem):
    """Codes looked up in a table of what they stand for (float64)."""
    bits, bias, man = {"e4m3": (8, 7, 3), "e5m2": (8, 15, 2), "e2m1": (4, 1, 1)}[elem]
    t = []
    for n in range(1 << bits):
        e, m, sg = (n >> man) & ((1 << (bits - 1 - man)) - 1), n & ((1 << man) - 1), -1.0 if n >> (bits - 1) else 1.0
        v = m * 2.0 ** (1 - bias - man) if e == 0 else (1 + m / (1 << man)) * 2.0 ** (e - bias)
        if (elem == "e4m3" and n & 127 == 127) or (elem == "e5m2" and e == 31 and m):
            v = float("nan")
        if elem == "e5m2" and e == 31 and not m:
            v = float("inf")
        t.append(sg * v)
    t = torch.tensor(t, dtype=torch.float64, device=code.device)
    if elem == "e2m1":
        v = torch.empty(*code.shape, 2, dtype=torch.float64, device=code.device)
        v[..., 0], v[..., 1] = t[(code % 16).long()], t[torch.div(code, 16, rounding_mode="floor").long()]
        v = v.reshape(*code.shape[:-1], -1)
    else:
        v = t[code.long()]
    z = _two_to(scale.double() - 127)
    z[scale == 255] = float("nan")
    return v * z.repeat_interleave(32, -1)


def _exact_round(x, elem):
    """fp64 [..., D] -> the nearest representable values in units of the block's scale, and the scale's exponent."""
    man, low, big = {"e4m3": (3, -6, 448.0), "e5m2": (2, -14, 57344.0), "e2m1": (1, 0, 6.0)}[elem]
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((amax / big).clamp(min=2.0 ** -140))).clamp(-126, 127)
    e = torch.where(amax > big * _two_to(e), e + 1, torch.where((amax <= big * _two_to(e - 1)) & (e > -126), e - 1, e))
    y = b / _two_to(e)
    p = torch.round(torch.log2(y.abs().clamp(min=2.0 ** low)))
    step = _two_to(torch.where(y.abs() < _two_to(p), p - 1, p).clamp(min=low) - man)      # distance of neighbours at y
    return torch.round(y / step) * step, e


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    B, D = c["B"], c["D"]
    if c["kind"] == "rope":
        if B * c["L"] * (c["Hq"] + c["Hkv"]) * D > 1 << 29:
            return None
        out = []
        for n in ("q", "k"):
            x = _heads_first(s[n], c["layout"]).double()
            if c["norm"] == "head":
                x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s[n + "_weight"].double()
            elif c["norm"] == "across":
                x = x / (x.pow(2).mean(dim=(1, 3), keepdim=True) + 1e-6).sqrt() * s[n + "_weight"].double()[None, :, None, :]
            r, h = c["rot"], c["rot"] // 2
            pos = s["positions"].long()
            pos = pos.unsqueeze(-1).expand(*pos.shape, h) if c["axes"] == 1 else torch.cat(
                [pos[..., a:a + 1].expand(*pos.shape[:-1], w) for a, w in enumerate(_sections(c))], -1)
            turn = torch.complex(s["cos"].double().gather(0, pos.reshape(-1, h)), s["sin"].double().gather(0, pos.reshape(-1, h)))
            turn = turn.reshape(B, 1, c["L"], h)
            if c["interleaved"]:
                z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], h, 2).contiguous()) * turn
                x[..., :r] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(x[..., :h], x[..., h:r]) * turn
                x[..., :h], x[..., h:r] = z.real, z.imag
            out.append(_heads_first(x, c["layout"]).contiguous())
        return tuple(out)
    d, page, table = s["cache"], c["page"], s["table"]
    if c["kind"] in ("append", "refill"):
        new = {}
        for n in ("k", "v"):
            new[n] = _exact_round(_heads_first(s[n], c["layout"]).double(), c["elem"])
    if c["kind"] == "append":
        if c["elem"] == "e2m1":
            return {n: None for n in d}
        got = {}
        for n in ("k", "v"):
            got[n] = d[n].view(FLOAT8[c["elem"]]).double()
            for b in range(B):
                at = int(s["held"][b]) + torch.arange(c["T"], device="cuda")
                got[n][table[b].long()[at // page], :, at % page] = new[n][0][b].flatten(-2).transpose(0, 1)
            got[n + "_scale"] = None
        return got
    if c["kind"] in ("refill", "read"):
        L, out = _longest(c), []
        for n in ("k", "v"):
            x = torch.zeros(B, c["Hkv"], L, D, dtype=torch.float64, device="cuda")
            for b in range(B):
                m = int(s["lengths"][b])
                pages = table[b].long()[: -(-m // page)]
                x[b, :, :m] = _exact_values(torch.cat(list(d[n][pages]), 1)[:, :m], torch.cat(list(d[n + "_scale"][pages]), 1)[:, :m], c["elem"])
                if c["kind"] == "refill":
                    w, e = new[n][0][b], new[n][1][b]
                    x[b, :, m - c["T"]:m] = (w * _two_to(e)).flatten(-2)
            out.append(x)
        return tuple(out)
    T, Hq, Hkv = c["T"], c["Hq"], c["Hkv"]
    if B * c["L"] * Hq * T > 1 << 31:
        return None
    q = _heads_first(s["q"], c["layout"]).double()
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, T), float("-inf"), dtype=torch.float64, device="cuda")
    for b in range(B):
        m = int(s["lengths"][b])
        t = T if s["q_lens"] is None else int(s["q_lens"][b])
        if m == 0 or t == 0:
            continue
        pages = table[b].long()[: -(-m // page)]
        seen = torch.ones(t, m, dtype=torch.bool, device="cuda")
        seen[:, m - t:] = torch.ones(t, t, dtype=torch.bool, device="cuda").tril() if s["mask"] is None else s["mask"][b, :t, :t]
        for h in range(Hkv):
            k, v = (_exact_values(d[n][pages, h].flatten(0, 1)[:m], d[n + "_scale"][pages, h].flatten(0, 1)[:m], c["elem"]) for n in ("k", "v"))
            own_rows = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            sc = (q[b, own_rows, :t] @ k.t() / math.sqrt(D)).masked_fill(~seen, float("-inf"))
            o[b, own_rows, :t] = torch.softmax(sc, -1) @ v
            lse[b, own_rows, :t] = torch.logsumexp(sc, -1) / math.log(2.0)
    return _heads_first(o, c["layout"]).contiguous(), lse
