"""Keys and values in pages: a cache written as tokens arrive, read back, and attended to by new tokens.

The reference's K/V are contiguous shards of one length; this is what serving needs beside them.  The results of
attn_fwd_paged (o, lse) merge with those of the block ops (ops.update_out_and_lse), and kv_cache_read gives the
packed [2, batch, seq, heads, head_dim] buffer that RingAttention and the generated programs take.

One batch is described the same way to all three calls:

  page_table  int32 [batch, max_pages]: key j of sequence b lies in slot j % page_size of page
              page_table[b, j // page_size]; entries behind a sequence's last page are not read
  seq_lens    int32 [batch]: keys of every sequence, the call's new tokens included
  cu_seqlens  int32 [batch + 1] or None.  Given: the new tokens of sequence b are rows
              [cu_seqlens[b], cu_seqlens[b + 1]) of [tokens, heads, head_dim] tensors; rows behind the last
              sequence are left alone.  None: every sequence has n of them, tensors are [batch, n, heads, head_dim].

The last new token of a sequence is its last key.  All three live on the device and are read there, so that a captured
graph can be replayed with other contents; what does not fit the tables or tensors is skipped there, reported as
status 110, and raised by PagedKV.check().  Sequences may share pages that are only read.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .attention import _on, _stream_ptr

HEAD_DIM = 128
SCALE_BLOCK = 32  # values along head_dim that share a power of two
_DTYPES = {torch.bfloat16: _lib.MB_DTYPE_BF16, torch.float8_e4m3fn: _lib.MB_DTYPE_E4M3}


class PagedKV:
    """A cache of keys and values in pages.

    k, v: [pages, page_size, heads, 128], views are fine (a cache laid out [pages, heads, page_size, 128] goes in
    transposed) as long as head_dim is contiguous, k and v share their strides, and these are multiples of 16 bytes.
    bfloat16, or float8_e4m3fn with k_scale, v_scale: contiguous uint8 [pages, heads, page_size, 4].  Byte x is the power
    of two 2^(x - 127) that 32 values share: a code times its power of two is exact in bfloat16 from byte 3 on (below, the
    least codes fall under bfloat16's least value, 2^-133, and are rounded to it or zero when they are read).  A write chooses
    77 .. 191; bytes from 192 on make their values NaN, and so do e4m3's NaN codes (0x7f, 0xff), which no write makes.  The
    calls go to the memory that these tensors have when the cache is made.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        if k.dim() != 4:
            raise ValueError(f"k must be [pages, page_size, heads, head_dim], got {tuple(k.shape)}")
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise TypeError(f"k and v must both be bfloat16 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
        if k.shape != v.shape or k.stride() != v.stride():
            raise ValueError("k and v must share shape and strides")
        pages, page_size, heads, d = k.shape
        if d != HEAD_DIM:
            raise NotImplementedError(f"head_dim must be {HEAD_DIM}, got {d}")
        if page_size < 1 or heads < 1:
            raise ValueError("pages need at least one slot and one head")
        if k.stride(3) != 1:
            raise ValueError("k, v: head_dim must be contiguous")
        size = k.element_size()
        if pages and any(x % 16 for x in (k.data_ptr(), v.data_ptr(), *(s * size for s in k.stride()[:3]))):
            raise ValueError("k, v: addresses and strides must be multiples of 16 bytes")
        if k.dtype == torch.float8_e4m3fn:
            shape = (pages, heads, page_size, d // SCALE_BLOCK)
            for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
                if s is None or s.dtype != torch.uint8 or tuple(s.shape) != shape or not s.is_contiguous():
                    raise ValueError(f"{name} must be contiguous uint8 {shape}")
                if pages and s.data_ptr() % 4:
                    raise ValueError(f"{name}: the address must be a multiple of 4 bytes")
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales go with float8_e4m3fn")
        for t in (k, v, k_scale, v_scale):
            if t is not None and (not t.is_cuda or t.device != k.device):
                raise ValueError("the cache must be CUDA tensors of one device (there is no CPU path)")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.dtype = k.device, k.dtype
        self.pages, self.page_size, self.heads = pages, page_size, heads
        # the first fields of the calls' argument block
        self._head = (k.data_ptr(), v.data_ptr(), *k.stride()[:3], k_scale.data_ptr() if k_scale is not None else 0,
                      v_scale.data_ptr() if v_scale is not None else 0)
        self._tail = (pages, page_size)
        self._kind = (heads, d, _DTYPES[k.dtype], 0)

    @classmethod
    def empty(cls, pages: int, page_size: int, heads: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "PagedKV":
        """A cache with memory of its own, [pages, page_size, heads, 128] (contents arbitrary)."""
        kv = torch.empty((2, pages, page_size, heads, HEAD_DIM), dtype=dtype, device=device)
        if dtype != torch.float8_e4m3fn:
            return cls(kv[0], kv[1])
        s = torch.empty((2, pages, heads, page_size, HEAD_DIM // SCALE_BLOCK), dtype=torch.uint8, device=device)
        return cls(kv[0], kv[1], s[0], s[1])

    def memory_bytes(self) -> int:
        """Bytes of keys, values and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def check(self) -> None:
        """Synchronise the current stream and raise if a call found a page number, length or offset out of bounds."""
        with _on(self.device):
            _lib.raise_on_status(_stream_ptr())

    def _batch(self, page_table, seq_lens, cu_seqlens, tokens: int) -> tuple:
        """The argument block of a call on this batch (_lib.PagedKVArgs), as values to pack."""
        dev = self.device
        shape = page_table.shape
        if len(shape) != 2 or page_table.dtype != torch.int32 or (shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be int32 [batch, max_pages] with contiguous rows")
        b, columns = shape
        if seq_lens.dtype != torch.int32 or seq_lens.shape != (b,) or not seq_lens.is_contiguous():
            raise ValueError(f"seq_lens must be contiguous int32 [{b}]")
        if page_table.device != dev or seq_lens.device != dev:
            raise ValueError(f"page_table and seq_lens must be on {dev}, where the cache is")
        cu = 0
        if cu_seqlens is not None:
            if cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (b + 1,) or not cu_seqlens.is_contiguous():
                raise ValueError(f"cu_seqlens must be contiguous int32 [{b + 1}]")
            if cu_seqlens.device != dev:
                raise ValueError(f"cu_seqlens must be on {dev}, where the cache is")
            cu = cu_seqlens.data_ptr()
        if columns * self.page_size > 0x7fffff00:
            raise ValueError("a page table may cover at most 2147483392 keys")
        if tokens > 0x7fffff00:
            raise ValueError("at most 2147483392 new tokens per call")
        return (*self._head, page_table.data_ptr(), page_table.stride(0), seq_lens.data_ptr(), cu, b, tokens, *self._tail,
                columns, *self._kind)


def _rows(t: torch.Tensor, name: str, cache: PagedKV, dims: int) -> tuple:
    """(address, batch stride, token stride, head stride) of [(batch,) tokens, heads, head_dim] rows, checked."""
    shape, stride, ptr = t.shape, t.stride(), t.data_ptr()
    if len(shape) != dims:
        want = "[tokens, heads, head_dim]" if dims == 3 else "[batch, tokens, heads, head_dim]"
        raise ValueError(f"{name} must be {want}, got {tuple(shape)}")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on {cache.device}, where the cache is")
    if shape[-1] != HEAD_DIM or stride[-1] != 1:
        raise ValueError(f"{name}: head_dim must be {HEAD_DIM} and contiguous")
    # (the stride of a dimension of one entry is never used)
    sh = stride[-2] if shape[-2] > 1 else 0
    st = stride[-3] if shape[-3] > 1 else 0
    sb = stride[0] if dims == 4 and shape[0] > 1 else 0
    if (ptr | sb * 2 | st * 2 | sh * 2) & 15:
        raise ValueError(f"{name}: address and strides must be multiples of 16 bytes")
    return ptr, sb, st, sh


def kv_cache_write(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                   cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Stores the new tokens' keys and values in their pages, rounded to e4m3 under a power of two per 32 values where
    the cache is float8_e4m3fn: the least 2^e, -50 <= e <= 64, with max|x| <= 448 * 2^e.  Values are rounded to nearest
    even; beyond 448 * 2^64 they become that.  32 values with an infinity or a NaN among them read as NaN.

    k, v: bfloat16 [batch, n, heads, 128], or [tokens, heads, 128] with cu_seqlens.  The new tokens are the
    last ones of the seq_lens[b] keys; where a sequence has more of them than keys, the first ones are not stored.  No
    two new tokens may lie in the same slot.  Nothing is stored under offsets that do not ascend within [0, tokens]."""
    dims = 3 if cu_seqlens is not None else 4
    shape = k.shape
    k_ptr, *strides = _rows(k, "k", cache, dims)
    v_ptr, *v_strides = _rows(v, "v", cache, dims)
    if shape != v.shape or strides != v_strides:
        raise ValueError("k and v must share shape and strides")
    if shape[-2] != cache.heads:
        raise ValueError(f"k, v have {shape[-2]} heads, the cache {cache.heads}")
    if dims == 4 and shape[0] != page_table.shape[0]:
        raise ValueError(f"k, v have batch {shape[0]}, page_table {page_table.shape[0]}")
    args = _lib.PAGED_KV.pack(*cache._batch(page_table, seq_lens, cu_seqlens, shape[0] if dims == 3 else shape[0] * shape[1]))
    with _on(cache.device):
        _lib.check(_lib.lib.mb_kv_cache_write(args, k_ptr, v_ptr, *strides, _stream_ptr()), "mb_kv_cache_write")


def kv_cache_read(cache: PagedKV, page_table: torch.Tensor, seq_lens: torch.Tensor, out: Optional[torch.Tensor] = None,
                  max_keys: Optional[int] = None) -> torch.Tensor:
    """The first keys and values of every sequence, in bfloat16, as one packed [2, batch, rows, heads, 128] buffer.

    out: the buffer to write to; rows behind a sequence's last key are left as they are, keys beyond its rows are left out.
    Without it a zero-filled one of max_keys rows is made (default: what the page table covers).  Values of a
    float8_e4m3fn cache are the code times its power of two, exact from scale byte 3 on."""
    args = cache._batch(page_table, seq_lens, None, 0)
    b, columns = page_table.shape
    if out is None:
        rows = columns * cache.page_size if max_keys is None else int(max_keys)
        if rows < 0:
            raise ValueError("max_keys must not be negative")
        out = torch.zeros((2, b, rows, cache.heads, HEAD_DIM), dtype=torch.bfloat16, device=cache.device)
    shape = out.shape
    if len(shape) != 5 or shape[0] != 2 or shape[1] != b or shape[3] != cache.heads:
        raise ValueError(f"out must be [2, {b}, rows, {cache.heads}, {HEAD_DIM}], got {tuple(shape)}")
    if max_keys is not None and shape[2] != max_keys:
        raise ValueError("out must have max_keys rows")
    ptr, *strides = _rows(out[0], "out", cache, 4)
    half = out.stride(0) * 2
    if half % 16:
        raise ValueError("out: address and strides must be multiples of 16 bytes")
    with _on(cache.device):
        _lib.check(_lib.lib.mb_kv_cache_read(_lib.PAGED_KV.pack(*args), ptr, ptr + half, *strides, shape[2], _stream_ptr()),
                   "mb_kv_cache_read")
    return out


def attn_fwd_paged(
    q: torch.Tensor,
    cache: PagedKV,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    softmax_scale: float,
    causal: bool = True,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_queries: Optional[int] = None,
    max_keys: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """softmax(scale * q k^T) v of every sequence's new tokens over its cached keys (written before, the new tokens' own
    among them).

    q: bfloat16 [batch, n, hq, 128], or [tokens, hq, 128] with cu_seqlens; hq a multiple of the cache's heads.
    causal: new token i of n sees keys j <= seq_lens[b] - n + i (the last one sees all); causal=False: every key, as in
    cross attention to states of another length.  max_queries, max_keys: upper bounds on a sequence's new tokens
    (with cu_seqlens; default: all tokens) and keys (default: what the page table covers), by which the launch is cut, and
    scratch: where a float8_e4m3fn sequence may have more than 32 rows (new tokens x heads of a group), sequences of many rows
    are computed from a bfloat16 copy, 512 bytes per key and K/V head of max_keys, as many at once as take 1 GiB, or one.
    Returns (o like q, lse fp32 [batch, hq, n] or [hq, tokens]).  A row that sees no key gets o = 0, lse = -inf;
    rows behind the last sequence are left as they are.  out must not overlap q.

    Slots behind a sequence's last key are not read, whatever they hold.  A NaN or an infinity in a key or value reaches every
    row that a tile computes it with, also rows before it: probabilities of hidden keys are zeros, not gaps.

    Rows of a sequence may be split over several SMs: the same call repeats bit for bit, but a row's bits may
    differ between calls of other shapes."""
    dims = 3 if cu_seqlens is not None else 4
    q_rows = _rows(q, "q", cache, dims)
    shape = q.shape
    hq = shape[-2]
    if hq == 0 or hq % cache.heads:
        raise ValueError(f"q has {hq} heads, not a multiple of the cache's {cache.heads}")
    if not 0 < softmax_scale < float("inf"):
        raise ValueError(f"softmax_scale must be positive and finite, got {softmax_scale}")
    covered = page_table.shape[-1] * cache.page_size
    max_keys = covered if max_keys is None else min(int(max_keys), covered)
    if dims == 4:
        n = shape[1]
        tokens = shape[0] * n
        if shape[0] != page_table.shape[0]:
            raise ValueError(f"q has batch {shape[0]}, page_table {page_table.shape[0]}")
        if max_queries is not None and max_queries < n:
            raise ValueError(f"max_queries is {max_queries}, q has {n} tokens per sequence")
        max_queries = n
        lse_shape = (shape[0], hq, n)
    else:
        tokens = shape[0]
        max_queries = tokens if max_queries is None else min(int(max_queries), tokens)
        if max_queries == 0 and tokens > 0:  # no sequence has new tokens, or the bound is wrong and the device says so
            max_queries = 1
        lse_shape = (hq, tokens)
    if max_queries < 0 or max_keys < 0:
        raise ValueError("max_queries and max_keys must not be negative")
    batch = cache._batch(page_table, seq_lens, cu_seqlens, tokens)
    checked = False
    if out is None:
        out = torch.empty_like(q)
        checked = out.stride() == q.stride()
    elif out.shape != shape:
        raise ValueError(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    out_rows = (out.data_ptr(), *q_rows[1:]) if checked else _rows(out, "out", cache, dims)
    if lse is None:
        lse = q.new_empty(lse_shape, dtype=torch.float32)
    elif (lse.dtype != torch.float32 or lse.shape != lse_shape or lse.device != cache.device
          or (lse_shape[-1] > 1 and lse.stride(-1) != 1)):
        raise ValueError(f"lse must be fp32 {lse_shape} with contiguous rows on {cache.device}")
    lse_strides = lse.stride()
    args = _lib.ATTN_PAGED.pack(*batch, *q_rows, *out_rows, lse.data_ptr(),
                                lse_strides[0] if dims == 4 else 0, lse_strides[-2], hq, max_queries, max_keys,
                                1 if causal else 0, softmax_scale)
    with _on(cache.device):
        # scratch of units that several SMs share; freed in stream order by the caching allocator
        need = _lib.lib.mb_attn_paged_workspace(args)
        ws = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
        _lib.check(_lib.lib.mb_attn_paged(args, ws.data_ptr() if need > 0 else None, need, _stream_ptr()), "mb_attn_paged")
    return out, lse
