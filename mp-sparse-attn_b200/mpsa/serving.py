"""Serving token by token: normed and rotated queries and keys, a paged MX cache that is quantised as it is written, and attention of single
tokens, chunks or trees of drafted tokens over it.  The reference has none of these: it sees whole sequences in 16 bits on every call
(ours/mxfp_attn_kernel.py:19-74), and evaluate/llama decodes through the model's own 16-bit cache.

    cache = mpsa.kv_cache(num_pages=4096, num_kv_heads=8, head_dim=128, elem="e4m3", device="cuda")
    q, k = mpsa.norm_rope(q, k, q_weight=wq, k_weight=wk, rope=(cos, sin), positions=positions)
    mpsa.kv_cache_append(cache, k, v, page_table, lengths)              # tokens lengths[b] .. lengths[b] + T - 1
    o = mpsa.kv_cache_attention(q, cache, page_table, lengths + T)      # the last T tokens of each sequence

No gradients: these are inference operations, and operands that ask for one, or have tangents of forward mode, are refused.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _IN_DTYPE, _OUT_DTYPE, _bhld, _on_device, _ptr, _raise_if_failed, _require_cuda, _state

_ELEM = {"e4m3": 0, "e5m2": 1, "e2m1": 2}
_c_int, _c_ll, _c_p = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p


class _NormRopeArgs(ctypes.Structure):
    _fields_ = [("x", _c_p * 2), ("y", _c_p * 2), ("weight", _c_p * 2)] + \
        [(n, _c_ll * 2) for n in ("x_sb", "x_sh", "x_sl", "y_sb", "y_sh", "y_sl")] + \
        [("cos", _c_p), ("sin", _c_p), ("positions", _c_p), ("pos_sb", _c_ll), ("table_rows", _c_ll),
         ("H", _c_int * 2), ("w_dtype", _c_int * 2), ("section_end", _c_int * 4)] + \
        [(n, _c_int) for n in ("in_dtype", "B", "L", "D", "rot", "norm", "axes", "interleaved", "pos64")] + [("eps", ctypes.c_float)]


class _Cache(ctypes.Structure):
    _fields_ = [(n, _c_p) for n in ("k", "v", "k_scale", "v_scale")] + [(n, _c_int) for n in ("num_pages", "page_size", "Hkv", "D", "elem")]


class _AppendArgs(ctypes.Structure):
    _fields_ = [("cache", _Cache), ("k", _c_p), ("v", _c_p)] + \
        [(n, _c_ll) for n in ("k_sb", "k_sh", "k_sl", "v_sb", "v_sh", "v_sl", "table_sb")] + \
        [(n, _c_p) for n in ("page_table", "start", "counts")] + [(n, _c_int) for n in ("in_dtype", "B", "T", "max_pages")]


class _ReadArgs(ctypes.Structure):
    _fields_ = [("cache", _Cache), ("k_out", _c_p), ("v_out", _c_p), ("table_sb", _c_ll), ("page_table", _c_p), ("lengths", _c_p)] + \
        [(n, _c_int) for n in ("out_dtype", "B", "max_len", "max_pages")]


class _AttentionArgs(ctypes.Structure):
    _fields_ = [("cache", _Cache), ("q", _c_p), ("out", _c_p), ("lse", _c_p), ("workspace", _c_p), ("workspace_bytes", _c_ll)] + \
        [(n, _c_ll) for n in ("q_sb", "q_sh", "q_sl", "o_sb", "o_sh", "o_sl", "table_sb", "mask_sb")] + \
        [(n, _c_p) for n in ("page_table", "lengths", "q_lens", "mask", "status")] + \
        [(n, _c_int) for n in ("dtype", "B", "T", "Hq", "max_pages")] + [("sm_scale", ctypes.c_float)]


def _aligned(x: torch.Tensor, tensor_layout: str, elements: int):
    """x, its logical (B,H,L,D) and strides, with bases and strides of the operand that are multiples of `elements` (a copy where they are not)."""
    x, size, st = _bhld(x, tensor_layout)
    if (st[0] | st[1] | st[2]) % elements or x.data_ptr() % min(16, elements * x.element_size()):
        x, size, st = _bhld(x.clone(memory_format=torch.contiguous_format), tensor_layout)
    return x, size, st


def _no_gradient(*ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError("no gradient is computed here: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):       # (no_grad() leaves these on)
        raise ValueError("no derivative is computed here: operands have tangents")


def norm_rope(q: torch.Tensor, k: Optional[torch.Tensor] = None, *, q_weight: Optional[torch.Tensor] = None,
              k_weight: Optional[torch.Tensor] = None, norm: bool = True, across_heads: bool = False, eps: float = 1e-6, rope=None,
              positions: Optional[torch.Tensor] = None, sections: Optional[Tuple[int, ...]] = None, interleaved: bool = False,
              tensor_layout: str = "HND"):
    """RMS norm of queries and keys and their rotation by position, in one pass over both; new tensors like q and k.

    q [B,Hq,L,D], k [B,Hkv,L,D] (or [B,L,H,D] with tensor_layout "NHD"); bf16, fp16 or fp32, D 64 or 128; k None: q alone, and one tensor.
    norm: divide each head's row by the root of its mean square (plus eps) and multiply by the weight [D]; across_heads: the mean over all
    heads of the token, weight [H, D] (or [H * D]).  norm=False: the rotation alone.
    rope: (cos, sin), fp32 [P, R/2]: row p holds the angles of position p; the first R elements of a row are rotated (R <= D, a multiple of
    8), pairs (i, i + R/2), or neighbours with interleaved=True.
    positions: int32 or int64, [L] or [B,L]; None: token l has position l.  With `sections` (R/2 split among up to four axes, in pairs)
    positions are [L,A] or [B,L,A], and pair i goes by the axis that its section belongs to.  A token with a position outside the table
    gets NaN in its rotated elements."""
    r = None
    if tensor_layout in ("HND", "NHD") and (rope is None or len(rope) == 2):
        r = _lib.native().norm_rope(q, k, q_weight, k_weight, (2 if across_heads else 1) if norm else 0, eps, *((None, None) if rope is None else rope), positions, sections,
                                    interleaved, tensor_layout == "HND")
    if r is not None:
        if r.__class__ is int:
            _lib.check(r)
        return r
    _require_cuda(q, k, q_weight, k_weight, positions)
    _no_gradient(q, k, q_weight, k_weight, *(() if rope is None else rope))
    if q.dtype not in _IN_DTYPE:
        raise ValueError(f"unsupported input dtype {q.dtype}")
    a = _NormRopeArgs()
    outs, keep = [], []
    shape = None
    if not norm and (q_weight is not None or k_weight is not None):
        raise ValueError("weights go with a norm")
    for i, (x, w) in enumerate(((q, q_weight), (k, k_weight))):
        if x is None:
            if w is not None:
                raise ValueError("k_weight without k")
            continue
        if x.device != q.device or x.dtype != q.dtype:
            raise ValueError("q and k must have one type and one device")
        x, (B, H, L, D), st = _aligned(x, tensor_layout, 4)
        if shape is None:
            shape = (B, L, D)
        elif shape != (B, L, D):
            raise ValueError("q and k must agree in batch, length and depth")
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _, _, yt = _bhld(y, tensor_layout)
        a.x[i], a.y[i], a.H[i] = x.data_ptr(), y.data_ptr(), H
        a.x_sb[i], a.x_sh[i], a.x_sl[i] = st
        a.y_sb[i], a.y_sh[i], a.y_sl[i] = yt
        if w is not None:
            if w.device != q.device or w.dtype not in _IN_DTYPE or w.numel() != (H * D if across_heads else D) or \
                    tuple(w.shape) not in ((D,), (H, D), (H * D,)) or not w.is_contiguous():
                raise ValueError("weights must be contiguous [D], or [H, D] or [H * D] across heads, on q's device")
            if any(u is not None and u.dtype != q.dtype for u in (q_weight, k_weight)):
                w = w.float()                          # (the kernels take the weights of a call in q's type or in fp32)
            if w.data_ptr() % 16:
                w = w.clone()
            keep.append(w)
            a.weight[i], a.w_dtype[i] = w.data_ptr(), _IN_DTYPE[w.dtype]
        outs.append(y)
        keep.append(x)
    B, L, D = shape
    if D not in (64, 128):
        raise ValueError("headdim should be in [64, 128].")
    a.in_dtype, a.B, a.L, a.D, a.norm, a.eps = _IN_DTYPE[q.dtype], B, L, D, (2 if across_heads else 1) if norm else 0, eps
    a.axes, a.interleaved = 1, int(interleaved)
    if rope is not None:
        cos, sin = rope
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape != cos.shape or t.device != q.device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("rope = (cos, sin): contiguous fp32 [P, R/2] on q's device")
        P, half = cos.shape
        if half == 0 or half % 4 or 2 * half > D:
            raise ValueError("the rotated width must be a multiple of 8, at most the depth")
        a.cos, a.sin, a.rot, a.table_rows = cos.data_ptr(), sin.data_ptr(), 2 * half, P
        if sections is not None:
            if not 1 <= len(sections) <= 4 or any(n < 0 for n in sections) or sum(sections) != half:
                raise ValueError("sections must be one to four numbers of pairs that add up to R/2")
            if positions is None:
                raise ValueError("sections need positions")
            a.axes = len(sections)
            end = 0
            for i, n in enumerate(sections):
                end += n
                a.section_end[i] = end
        if positions is not None:
            want = (L,) if sections is None else (L, a.axes)
            if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device or \
                    tuple(positions.shape) not in (want, (B, *want)):
                raise ValueError("positions must be int32 or int64 [L] or [B, L] (with sections [L, A] or [B, L, A]) on q's device")
            positions = positions.contiguous()
            a.positions, a.pos64 = positions.data_ptr(), int(positions.dtype == torch.int64)
            a.pos_sb = 0 if positions.dim() == len(want) else L * a.axes
        elif L > P:
            raise ValueError("the rotary table has fewer rows than there are tokens")
    elif positions is not None or sections is not None:
        raise ValueError("positions and sections go with rope")
    _lib.check(_on_device(q.get_device(), _lib.load().mpsa_norm_rope, ctypes.byref(a)))
    return tuple(outs) if k is not None else outs[0]


@dataclass(frozen=True, eq=False)
class KVCache:
    """A paged cache of keys and values in MX blocks of 32 along the depth, quantised token by token: what kv_cache() makes, or a program's own buffers.

    k, v uint8 [pages, Hkv, page_size, D] (elem "e4m3" or "e5m2") or [pages, Hkv, page_size, D/2] ("e2m1": two codes a byte, the lower depth
    in the low half); k_scale, v_scale uint8 [pages, Hkv, page_size, D/32]: an element stands for code * 2^(scale - 127), and a block with
    the scale 255 for NaN (element codes are finite numbers).  A sequence's tokens lie in the pages that its row of a page table names; which pages it gets is the program's affair."""
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor
    elem: str = "e4m3"

    def __post_init__(self):
        """The argument block of the buffers as they are now, beside them.  The short way compares the two at every call and leaves it to the long
        way, which comes here again, where they differ: a program may have exchanged a buffer's memory."""
        if self.elem not in _ELEM:
            raise ValueError(f"unknown cache element {self.elem!r}")
        block = _lib.native().kv_cache(k := self.k, ks := self.k_scale, v := self.v, vs := self.v_scale, e := _ELEM[self.elem])         # as bytes
        if block is None:
            _require_cuda(k, v, ks, vs)
            if k.dim() != 4:
                raise ValueError("cache codes must be [pages, heads, page size, bytes]")
            pages, heads, page, row = k.shape
            D = row * 2 if self.elem == "e2m1" else row
            for t, n in ((k, row), (v, row), (ks, D // 32), (vs, D // 32)):
                if t.dtype is not torch.uint8 or t.shape != (pages, heads, page, n) or not t.is_contiguous() or t.device != k.device:
                    raise ValueError("cache buffers must be contiguous uint8 [pages, heads, page size, ...] on one device")
            block = bytes(_Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, heads, D, e))
        object.__setattr__(self, "_c", (block, k, ks, v, vs))

    def __reduce__(self):                              # (a copy, or a cache that comes out of a file, has other buffers and needs a block of its own)
        return type(self), (self.k, self.k_scale, self.v, self.v_scale, self.elem)

    @property
    def num_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3] * (2 if self.elem == "e2m1" else 1)

    def _block(self) -> _Cache:
        self.__post_init__()
        return _Cache.from_buffer_copy(self._c[0])


def kv_cache(num_pages: int, num_kv_heads: int, head_dim: int, *, page_size: int = 64, elem: str = "e4m3", device="cuda") -> KVCache:
    """An empty cache: num_pages pages of page_size tokens (a power of two from 16 to 1024) for num_kv_heads heads of depth 64 or 128."""
    if elem not in _ELEM:
        raise ValueError(f"unknown cache element {elem!r}")
    if head_dim not in (64, 128):
        raise ValueError("headdim should be in [64, 128].")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1) or num_pages <= 0 or num_kv_heads <= 0:
        raise ValueError("a cache needs pages, heads and a page size that is a power of two from 16 to 1024")
    lead = (num_pages, num_kv_heads, page_size)
    row = head_dim // 2 if elem == "e2m1" else head_dim
    k, ks, v, vs = (torch.zeros((*lead, n), dtype=torch.uint8, device=device) for n in (row, head_dim // 32, row, head_dim // 32))
    return KVCache(k, ks, v, vs, elem)


def _index(t, name, shape, device, optional=False):
    if t is None and optional:
        return
    if t is None or t.dtype is not torch.int32 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)} on the cache's device")


def _table(page_table, B, device):
    if page_table is None or page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B or page_table.shape[1] == 0 or \
            page_table.device != device or page_table.stride(1) != 1:
        raise ValueError("page_table must be an int32 tensor [B, pages] on the cache's device")


def kv_cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor, *,
                    counts: Optional[torch.Tensor] = None, tensor_layout: str = "HND") -> None:
    """Quantises new tokens into the cache: token t of k, v [B,Hkv,T,D] (bf16, fp16, fp32) becomes token start[b] + t of sequence b.

    page_table int32 [B, pages]: the pages of each sequence in order; entries outside the cache stand for no page, and what would go there
    is left out.  counts int32 [B]: only the first counts[b] tokens are written (a padded batch).  start int32 [B].
    A block's scale is the smallest power of two at which no element exceeds the type's largest value; a block with a NaN or an infinity
    reads back as NaN.  Pages written by one call must not be shared between its sequences."""
    if tensor_layout in ("HND", "NHD"):
        r = _lib.native().kv_append(cache._c, k, v, page_table, start, counts, tensor_layout == "HND")
        if r is not None:
            return _lib.check(r)
    _require_cuda(k, v, page_table, start, counts)
    _no_gradient(k, v)
    if k.dtype not in _IN_DTYPE or v.dtype != k.dtype:
        raise ValueError(f"unsupported input dtypes {k.dtype}, {v.dtype}")
    dev = cache.k.device
    if k.device != dev or v.device != dev:
        raise ValueError("k and v must be on the cache's device")
    k, (B, H, T, D), ks = _aligned(k, tensor_layout, 8)
    v, vsize, vs = _aligned(v, tensor_layout, 8)
    if vsize != (B, H, T, D) or H != cache.num_kv_heads or D != cache.head_dim:
        raise ValueError("k and v must be [B, Hkv, T, D] with the cache's heads and depth")
    _table(page_table, B, dev)
    _index(start, "start", (B,), dev)
    _index(counts, "counts", (B,), dev, True)
    a = _AppendArgs(cache._block(), k.data_ptr(), v.data_ptr(), *ks, *vs, page_table.stride(0), page_table.data_ptr(), start.data_ptr(), _ptr(counts),
                    _IN_DTYPE[k.dtype], B, T, page_table.shape[1])
    _lib.check(_on_device(dev.index, _lib.load().mpsa_kv_append, ctypes.byref(a)))


def kv_cache_read(cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, *, max_len: Optional[int] = None,
                  out_dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of whole sequences in out_dtype (bf16, fp16, fp32): two tensors [B, Hkv, max_len, D], zero from lengths[b]
    on and where the table names no page.  max_len: all that the table can hold unless given.

    For a prefill over a cached prefix, attention_forward takes them as k and v.  It knows no lengths (a zero row is a key like any other, and
    causality is counted from the end): in one call with max_len the length that all sequences have, and for a ragged batch a sequence at a time,
    k[b:b+1, :, :n], v[b:b+1, :, :n] with n = lengths[b].  kv_cache_attention takes ragged batches as they are."""
    if max_len is not None and out_dtype in _OUT_DTYPE:
        r = _lib.native().kv_read(cache._c, page_table, lengths, max_len, _OUT_DTYPE[out_dtype])
        if r is not None:
            if r.__class__ is int:
                _lib.check(r)
            return r
    _require_cuda(page_table, lengths)
    dev = cache.k.device
    B = page_table.shape[0]
    _table(page_table, B, dev)
    _index(lengths, "lengths", (B,), dev)
    if out_dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"Unsupported dtype: {out_dtype}")
    n = page_table.shape[1] * cache.page_size if max_len is None else max_len
    if n <= 0:
        raise ValueError("max_len must be positive")
    k, v = (torch.empty((B, cache.num_kv_heads, n, cache.head_dim), dtype=out_dtype, device=dev) for _ in range(2))
    a = _ReadArgs(cache._block(), k.data_ptr(), v.data_ptr(), page_table.stride(0), page_table.data_ptr(), lengths.data_ptr(), _OUT_DTYPE[out_dtype], B, n,
                  page_table.shape[1])
    _lib.check(_on_device(dev.index, _lib.load().mpsa_kv_read, ctypes.byref(a)))
    return k, v


def kv_cache_attention(q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                       q_lens: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                       return_lse: bool = False, tensor_layout: str = "HND"):
    """Attention of each sequence's last T tokens over its cached keys and values: a decoding step (T = 1), a short chunk, or drafted tokens.

    q [B,Hq,T,D] (or NHD), bf16 or fp16, T up to 1024; Hq a multiple of the cache's heads; the result has q's shape and type.
    lengths int32 [B]: tokens in the cache, the query tokens among them (append them first).  q_lens int32 [B]: how many of the T are real
    (the first ones; the rows behind them come back as zero); None: all, or lengths[b] where that is fewer.
    mask: bool [T,T] or [B,T,T], True where query token i sees query token j - a tree of drafted tokens; None: every token sees those before
    it and itself.  Cached tokens before the query tokens are seen by all.  A row that sees nothing is zero.
    return_lse: also fp32 [B,Hq,T], log2 of the softmax denominators (-inf for a row that sees nothing), as attention_merge takes it.
    Scores, weights and sums are fp32; a weight times its key's scale of v is rounded to fp16, relative to the largest one of the row.  What a key
    does to a row goes by its own weight and size there, however large the keys beside it are."""
    dev = cache.k.device
    st = _state(dev.index)
    if st.word.value:
        _raise_if_failed(dev)
    if tensor_layout in ("HND", "NHD"):
        r = _lib.native().kv_attention(cache._c, q, page_table, lengths, q_lens, mask, st.status_ptr,
                                       cache.head_dim ** -0.5 if sm_scale is None else sm_scale, return_lse, tensor_layout == "HND")
        if r is not None:
            if r.__class__ is int:
                _lib.check(r)
            return r
    _require_cuda(q, page_table, lengths, q_lens, mask)
    _no_gradient(q)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported query dtype {q.dtype}")
    if q.device != dev:
        raise ValueError("q must be on the cache's device")
    q, (B, Hq, T, D), qs = _aligned(q, tensor_layout, 8)
    if D != cache.head_dim or Hq % cache.num_kv_heads or Hq == 0:
        raise ValueError("q must have the cache's depth and a multiple of its heads")
    if not 0 < T <= 1024:
        raise ValueError("between 1 and 1024 query tokens (longer prompts: kv_cache_read and attention_forward)")
    _table(page_table, B, dev)
    _index(lengths, "lengths", (B,), dev)
    _index(q_lens, "q_lens", (B,), dev, True)
    if mask is not None:
        if mask.dtype is not torch.bool or tuple(mask.shape) not in ((T, T), (B, T, T)) or mask.device != dev:
            raise ValueError("mask must be bool [T, T] or [B, T, T] on the cache's device")
        mask = mask.contiguous()
    sm = D ** -0.5 if sm_scale is None else float(sm_scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _, _, os = _bhld(out, tensor_layout)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=dev) if return_lse else None
    a = _AttentionArgs(cache._block(), q.data_ptr(), out.data_ptr(), _ptr(lse), None, 0, *qs, *os, page_table.stride(0),
                       0 if mask is None or mask.dim() == 2 else T * T, page_table.data_ptr(), lengths.data_ptr(), _ptr(q_lens), _ptr(mask), st.status_ptr,
                       _IN_DTYPE[q.dtype], B, T, Hq, page_table.shape[1], sm)
    lib = _lib.load()
    need = lib.mpsa_kv_attention_workspace(ctypes.byref(a))
    if need < 0:
        _lib.check(need)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _lib.check(_on_device(dev.index, lib.mpsa_kv_attention, ctypes.byref(a)))
    return (out, lse) if return_lse else out
