"""A paged key-value cache: keys and values of sequences in pages, in 16 bits or in 8 with a scale per token and head.

A cache's k and v (D, Page, KV_Heads, Pages) are torch [Pages, KV_Heads, Page, D] in f16, bf16, float8_e4m3fn or int8; the scales
(Page, KV_Heads, Pages) are torch [Pages, KV_Heads, Page] f32.  Pages are named by 1-based numbers, 0 is none: a page table is [Batch, Width]
int32, and a token's slot is (page - 1) * Page + place in the page + 1.  `fmha.fmha_paged` is the attention that reads it.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _host, _lib
from ._util import dense, dtype_code, handles, ids_bits, ptr

_STORES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float8_e4m3fn: _lib.E4M3, torch.int8: _lib.I8}


class KvCache(NamedTuple):
    """Arrays of a cache; they may be views whose pages lie apart (k and v of one allocation)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None  # with 8 bits
    v_scale: Optional[torch.Tensor] = None


def kv_cache(pages, kv_heads, page_size, head_dim, dtype, device="cuda"):
    """An empty cache (all zeros)."""
    if dtype not in _STORES:
        raise _lib.CtbError(_lib.BAD_ARG, f"a cache has elements of f16, bf16, float8_e4m3fn or int8, not {dtype}")
    shape = (int(pages), int(kv_heads), int(page_size), int(head_dim))
    if min(shape) <= 0:
        raise _lib.CtbError(_lib.BAD_ARG, f"non-positive dimension of the cache: {shape}")
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype in (torch.float16, torch.bfloat16):
        return KvCache(k, v)
    return KvCache(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def cache_struct(cache, like):
    """The checked cache as the C structure."""
    k, v, ks, vs = cache
    for t, what in ((k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor) or t.device != like.device:
            raise _lib.CtbError(_lib.BAD_ARG, f"cache.{what}: expected a tensor on {like.device}")
        if t.dim() != 4 or t.shape != k.shape or t.dtype != k.dtype:
            raise _lib.CtbError(_lib.BAD_ARG, f"cache.{what}: expected [Pages, KV_Heads, Page, D], k and v alike")
        if not t[:1].is_contiguous():
            raise _lib.CtbError(_lib.BAD_ARG, f"cache.{what}: a page must be dense")
    if k.dtype not in _STORES:
        raise _lib.CtbError(_lib.BAD_ARG, f"a cache has elements of f16, bf16, float8_e4m3fn or int8, not {k.dtype}")
    bytes_ = k.element_size() == 1
    for t, what in ((ks, "k_scale"), (vs, "v_scale")):
        if not bytes_:
            if t is not None:
                raise _lib.CtbError(_lib.BAD_ARG, f"cache.{what}: a cache of 16-bit elements has no scales")
            continue
        if not isinstance(t, torch.Tensor) or t.device != like.device or t.dtype != torch.float32:
            raise _lib.CtbError(_lib.BAD_ARG, f"cache.{what}: expected an f32 tensor on {like.device}")
        if t.shape != k.shape[:3] or not t[:1].is_contiguous():
            raise _lib.CtbError(_lib.BAD_ARG, f"cache.{what}: expected [Pages, KV_Heads, Page] with dense pages")
    s = _lib.KvCacheArrays()
    s.k, s.v = k.data_ptr(), v.data_ptr()
    s.pages, s.kv_heads, s.page_size, s.head_dim = k.shape
    s.k_page_stride, s.v_page_stride = k.stride(0), v.stride(0)
    if bytes_:
        s.k_scale, s.v_scale, s.k_scale_page_stride, s.v_scale_page_stride = ks.data_ptr(), vs.data_ptr(), ks.stride(0), vs.stride(0)
    s.dtype = _STORES[k.dtype]
    return s


def _rows_of(t, heads, D, T, what, like):
    if not isinstance(t, torch.Tensor) or t.device != like.device:
        raise _lib.CtbError(_lib.BAD_ARG, f"{what}: expected a tensor on {like.device}")
    if t.dim() != 3 or t.shape[0] != T or t.shape[2] != D or (heads is not None and t.shape[1] != heads) or t.stride(2) != 1:
        raise _lib.CtbError(_lib.BAD_ARG, f"{what}: expected [tokens, heads, D] with contiguous heads, got {tuple(t.shape)}")
    if t.dtype != like.dtype:
        raise _lib.CtbError(_lib.BAD_ARG, f"{what}: expected {like.dtype}, got {t.dtype}")
    return t


_LEFT_OUT = object()


def kv_write(cache, slots, k, v, q=None, positions=None, frequencies=_LEFT_OUT, interleaved=False, scale=1.0, out_q=None, **hints):
    """Writes k and v [tokens, KV_Heads, D] (f16 or bf16, any strides but contiguous heads) to slots [tokens] (int32 or int64; 0 writes
    nothing, the others must differ).  With positions [tokens] and frequencies, keys are turned as by `rope.rope_fwd` before they are stored,
    and so are the queries q [tokens, Heads, D], if given: returns them turned (in out_q, which may be q), else None.  Frequencies of None, said
    in so many words, turn nothing, whatever the positions (a model without rotary positions); positions whose frequencies are left
    out are refused."""
    forgotten = frequencies is _LEFT_OUT and positions is not None
    if frequencies is _LEFT_OUT:
        frequencies = None
    if not hints and not forgotten:
        r = _host.kv_write(cache, slots, k, v, q, positions, frequencies, interleaved, scale, out_q)
        if r is not None:
            return r[0]
    ctx, stream = handles(k, hints)
    s = cache_struct(cache, k)
    T, D, KVH = k.shape[0], s.head_dim, s.kv_heads
    _rows_of(k, KVH, D, T, "k", k)
    _rows_of(v, KVH, D, T, "v", k)
    bits = ids_bits(dense(slots, (T,), "slots", k), "slots")
    if forgotten or (positions is None and frequencies is not None):
        raise _lib.CtbError(_lib.BAD_ARG, "kv_write: positions and frequencies come together")
    if frequencies is None and q is not None:
        raise _lib.CtbError(_lib.BAD_ARG, "kv_write: queries come with positions and frequencies")
    if q is None and out_q is not None:
        raise _lib.CtbError(_lib.BAD_ARG, "kv_write: out_q comes with q")
    position_bits, rotary, strides, heads = 32, 0, [0] * 4, 0
    if positions is not None:
        position_bits = ids_bits(dense(positions, (T,), "positions", k), "positions")
    if frequencies is not None:
        if not isinstance(frequencies, torch.Tensor) or frequencies.dim() != 1:
            raise _lib.CtbError(_lib.BAD_ARG, "frequencies: expected a tensor of one dimension")
        rotary = 2 * dense(frequencies, frequencies.shape, "frequencies", k, torch.float64).shape[0]
        if rotary == 0:
            raise _lib.CtbError(_lib.BAD_ARG, "kv_write: frequencies of no pairs (rotary is 0); None turns nothing")
    if q is not None:
        _rows_of(q, None, D, T, "q", k)
        heads = q.shape[1]
        out_q = torch.empty_like(q) if out_q is None else _rows_of(out_q, heads, D, T, "out_q", k)
        strides = [out_q.stride(0), out_q.stride(1), q.stride(0), q.stride(1)]
    strides += [k.stride(0), k.stride(1), v.stride(0), v.stride(1)]
    _lib.check(_lib.lib.ctb_kv_write(ctx, stream, C.byref(s), ptr(slots), bits, ptr(out_q), ptr(q), ptr(k), ptr(v), (C.c_int64 * 8)(*strides),
                                     ptr(None if frequencies is None else positions), position_bits, ptr(frequencies), T, heads, rotary, int(bool(interleaved)),
                                     float(scale), dtype_code(k)))
    return out_q


def page_table_of(page_table, lengths, like):
    """(batch, width, stride) of a checked page table with its lengths."""
    if not isinstance(page_table, torch.Tensor) or page_table.device != like.device or page_table.dtype != torch.int32:
        raise _lib.CtbError(_lib.BAD_ARG, f"page_table: expected an int32 tensor on {like.device}")
    if page_table.dim() != 2 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise _lib.CtbError(_lib.BAD_ARG, "page_table: expected [Batch, Width] with contiguous rows")
    B, W = page_table.shape
    dense(lengths, (B,), "lengths", like, torch.int32)
    return B, W, page_table.stride(0) if B > 1 else max(W, page_table.stride(0))


def kv_read(cache, page_table, lengths, max_length, dtype=None, **hints):
    """The first lengths[b] tokens (int32) of every sequence's pages as dense K and V [Batch, KV_Heads, max_length, D], zeros behind them:
    the layout of `fmha.cutile_fmha`, which takes heads of 64 and sequences of one length (the zeros behind a shorter one would count).  dtype f16
    or bf16, for a 16-bit cache its own."""
    if not hints:
        r = _host.kv_read(cache, page_table, lengths, max_length, dtype)
        if r is not None:
            return r
    ctx, stream = handles(page_table, hints)
    s = cache_struct(cache, page_table)
    B, W, ld = page_table_of(page_table, lengths, page_table)
    if dtype is None:
        if cache.k.element_size() == 1:
            raise _lib.CtbError(_lib.BAD_ARG, "kv_read: what is read from 8 bits needs a dtype")
        dtype = cache.k.dtype
    if int(max_length) < 0:
        raise _lib.CtbError(_lib.BAD_ARG, "kv_read: negative max_length")
    K, V = (torch.empty((B, s.kv_heads, int(max_length), s.head_dim), dtype=dtype, device=page_table.device) for _ in range(2))
    _lib.check(_lib.lib.ctb_kv_read(ctx, stream, ptr(K), ptr(V), C.byref(s), ptr(page_table), ptr(lengths), B, int(max_length), W, ld,
                                    dtype_code(K)))
    return K, V
