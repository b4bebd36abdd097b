"""A paged cache of keys and values in 8 bits, and attention over it (no counterpart in the reference, which is one product).

A page holds ``page_size`` tokens of every head as int8 codes, with one float32 scale per page, head and side (keys, values). Three tensors:

    k       [pages, kv_heads, page_size, head_dim]  int8
    v       [pages, kv_heads, head_dim, page_size]  int8 -- the tokens of a channel together, as attention reads them
    scales  [pages, kv_heads, 2]                    float32

and, per call, where the tokens of each sequence are: ``block_table`` [sequences, width] int32 (an entry that is no page number, -1 say, is no
page: nothing is stored there, and attention passes over its tokens), ``lengths`` [sequences] int32 with the new tokens counted in,
``query_start`` [sequences + 1] int32 for new tokens packed one sequence after the other (None: the same number each).

:func:`append` stores, :func:`attend` reads, :func:`read` gives pages back as floats; :class:`PagedKVCache` holds the three tensors. All of
them are asynchronous, on the current stream, and may be captured into a HIP graph; none is differentiable. Exact definitions: ``include/qm_abi.h``.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import KvCache, KvNew, QuadmulError, _check, _has_extension, _native, _stream_ptr, library

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 96, 128, 192, 256)

_KINDS = {torch.float16: 1, torch.bfloat16: 2}
_INT_MAX = 2 ** 31 - 1


def _cache(what, k, v, scales) -> KvCache:
    if not (k.is_cuda and k.device == v.device == scales.device and k.dim() == 4 and k.dtype == v.dtype == torch.int8 and k.is_contiguous() and v.is_contiguous()):
        raise QuadmulError(f"{what}: the codes must be contiguous 4-D int8 tensors on one GPU")
    pages, heads, page, dim = k.shape
    if not 1 <= heads <= 4096 or pages > _INT_MAX:
        raise QuadmulError(f"{what}: 1 to 4096 heads, and less than 2^31 pages")
    if page not in PAGE_SIZES or dim not in HEAD_DIMS or v.shape != (pages, heads, dim, page):
        raise QuadmulError(f"{what}: pages of {PAGE_SIZES} tokens, heads of {HEAD_DIMS}; the values' codes are [pages, kv_heads, head_dim, page_size]")
    if scales.shape != (pages, heads, 2) or scales.dtype != torch.float32 or not scales.is_contiguous():
        raise QuadmulError(f"{what}: the scales must be a contiguous float32 tensor [pages, kv_heads, 2]")
    return KvCache(k.data_ptr(), v.data_ptr(), scales.data_ptr(), pages, heads, page, dim)


def _sequences(what, c, device, block_table, lengths, query_start, tokens):
    for t, dims in ((block_table, 2), (lengths, 1), (query_start, 1)):
        if t is not None and not (t.device == device and t.dtype == torch.int32 and t.dim() == dims and t.is_contiguous()):
            raise QuadmulError(f"{what}: block_table, lengths and query_start must be contiguous int32 tensors on the cache's device")
    count = lengths.shape[0]
    if block_table.shape[0] != count or (query_start is not None and query_start.shape[0] != count + 1):
        raise QuadmulError(f"{what}: block_table [sequences, width], lengths [sequences], query_start [sequences + 1]")
    if max(tokens, count, block_table.shape[1]) > _INT_MAX:
        raise QuadmulError(f"{what}: sizes must fit in int32")
    if tokens and (not count or (query_start is None and tokens % count)):
        raise QuadmulError(f"{what}: {tokens} tokens of {count} sequences need a query_start")
    c.block_table, c.lengths = block_table.data_ptr(), lengths.data_ptr()
    c.query_start = None if query_start is None else query_start.data_ptr()
    c.sequences, c.table_width = count, block_table.shape[1]


def _rows(what, t, c, device, dtype):
    if not (t.device == device and t.dtype == dtype and t.dim() == 3 and t.shape[2] == c.head_dim and (t.stride(2) == 1 or t.numel() == 0)):
        raise QuadmulError(f"{what}: queries, keys and values must be [tokens, heads, {c.head_dim}] of one 16-bit type on the cache's device, the last dimension contiguous")


def append(k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
           lengths: torch.Tensor, query_start: Optional[torch.Tensor] = None, *, q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
           sin: Optional[torch.Tensor] = None, interleaved: bool = False, max_query: int = 0) -> Optional[torch.Tensor]:
    """New keys and values ``[tokens, kv_heads, head_dim]`` (float16 or bfloat16, views of a projection's rows as they are) into the cache, the keys rotated to
    their positions; with ``q`` [tokens, heads, head_dim] returns the queries rotated too, else None.

    ``cos`` and ``sin`` [positions, pairs] float32, ``2 * pairs <= head_dim``: pairs of elements ``i`` and ``i + pairs``, or with ``interleaved`` ``2i`` and
    ``2i + 1``; without them nothing is rotated. A page that new tokens begin at its start begins anew; in one that held tokens the scale grows
    with the largest value and the codes that are there are rounded again. ``max_query``: the most new tokens of a sequence, if known (only a
    matter of speed; 0: one, if there are no more tokens than sequences, else what the shapes allow). No two sequences may write to one page in one call."""
    interleaved, max_query = bool(interleaved), int(max_query)
    if _has_extension():
        return _native("kv_append", k, v, cache_k, cache_v, scales, block_table, lengths, query_start, q, cos, sin, interleaved, max_query)
    c = _cache("append", cache_k, cache_v, scales)
    if k.dtype not in _KINDS or k.shape != v.shape or k.dim() != 3 or k.shape[1] != c.kv_heads:
        raise QuadmulError(f"append: keys and values must be [tokens, {c.kv_heads}, {c.head_dim}], float16 or bfloat16")
    for t in (k, v) if q is None else (k, v, q):
        _rows("append", t, c, cache_k.device, k.dtype)
    tokens = k.shape[0]
    _sequences("append", c, cache_k.device, block_table, lengths, query_start, tokens)
    if q is not None and (q.shape[0] != tokens or not 1 <= q.shape[1] <= _INT_MAX):
        raise QuadmulError("append: as many queries as keys")
    if (cos is None) != (sin is None):
        raise QuadmulError("append: cos and sin go together")
    for t in () if cos is None else (cos, sin):
        if not (t.device == cache_k.device and t.dtype == torch.float32 and t.dim() == 2 and t.is_contiguous() and t.shape == cos.shape and t.shape[0] >= 1 and 2 * t.shape[1] <= c.head_dim):
            raise QuadmulError(f"append: cos and sin must be contiguous float32 tensors [positions, at most {c.head_dim // 2}] on the cache's device")
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    n = KvNew(k.data_ptr(), v.data_ptr(), None if q is None else q.data_ptr(), None if q is None else out.data_ptr(), k.stride(0), k.stride(1), v.stride(0),
              v.stride(1), 0 if q is None else q.stride(0), 0 if q is None else q.stride(1), None if cos is None else cos.data_ptr(),
              None if sin is None else sin.data_ptr(), tokens, 0 if q is None else q.shape[1], _KINDS[k.dtype], 0 if cos is None else cos.shape[1],
              0 if cos is None else cos.shape[0], int(interleaved), min(max(max_query, 0), _INT_MAX))
    with torch.cuda.device(cache_k.device):
        _check(library().qm_kv_append_i8(ctypes.byref(c), ctypes.byref(n), _stream_ptr(cache_k)), "qm_kv_append_i8")
    return out


def attend(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
           query_start: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, causal: bool = True, window: int = 0, max_query: int = 0,
           max_length: int = 0) -> torch.Tensor:
    """Attention of the last tokens of each sequence over the cache: ``q`` [tokens, heads, head_dim] float16 or bfloat16 -> the same shape and type.

    ``heads`` is a multiple of the cache's; each of those serves as many in turn. ``scale``: 1 / sqrt(head_dim) by default. ``causal``: a token sees those up to its own
    position, else all of its sequence; ``window`` > 0: only the last ``window`` of them. A row that sees nothing is 0. Scores, softmax and sums are in
    float32; a weight, times its value's scale, enters the product with the values as a float16 of 11 bits, or, below 2^-20 of the row's largest, to 2^-31 of that.
    ``max_query``, ``max_length``: the most new tokens, and the most tokens, of a sequence, if known (only a matter of speed; 0: what the
    shapes allow, and for ``max_query`` one, if there are no more tokens than sequences)."""
    causal, window, max_query, max_length = bool(causal), int(window), int(max_query), int(max_length)
    out = _native("kv_attend", q, cache_k, cache_v, scales, block_table, lengths, query_start, scale, causal, window, max_query, max_length)
    if out is not None:
        return out
    c = _cache("attend", cache_k, cache_v, scales)
    if q.dtype not in _KINDS:
        raise QuadmulError("attend: the queries must be float16 or bfloat16")
    _rows("attend", q, c, cache_k.device, q.dtype)
    tokens, heads = q.shape[:2]
    _sequences("attend", c, cache_k.device, block_table, lengths, query_start, tokens)
    if heads < 1 or heads > 65535 or heads % c.kv_heads or window < 0:
        raise QuadmulError(f"attend: the heads of the queries must be a multiple of the cache's {c.kv_heads}, the window 0 or more tokens")
    max_query, max_length, window = (min(max(i, 0), _INT_MAX) for i in (max_query, max_length, window))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    need = library().qm_kv_attend_workspace_bytes(ctypes.byref(c), tokens, heads, window, max_query, max_length)
    scratch = torch.empty((need,), dtype=torch.uint8, device=q.device) if need else None
    with torch.cuda.device(q.device):
        st = library().qm_kv_attend_i8(ctypes.byref(c), q.data_ptr(), _KINDS[q.dtype], q.stride(0), q.stride(1), out.data_ptr(), tokens, heads,
                                       1.0 / math.sqrt(c.head_dim) if scale is None else scale, int(causal), window, max_query, max_length, _stream_ptr(q),
                                       scratch.data_ptr() if need else None, need)
    _check(st, "qm_kv_attend_i8")
    return out


def read(cache_k: torch.Tensor, cache_v: torch.Tensor, scales: torch.Tensor, pages: torch.Tensor, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages of ``pages`` ([count] int32) as values: keys and values, both ``[count, kv_heads, page_size, head_dim]``, float16 or bfloat16. Places that no
    token was stored in hold whatever codes are there."""
    if dtype not in _KINDS:
        raise QuadmulError("read: float16 or bfloat16")
    found = _native("kv_read", cache_k, cache_v, scales, pages, dtype == torch.bfloat16)
    if found is not None:
        return found
    c = _cache("read", cache_k, cache_v, scales)
    if not (pages.device == cache_k.device and pages.dtype == torch.int32 and pages.dim() == 1 and pages.is_contiguous()):
        raise QuadmulError("read: the pages must be a contiguous int32 vector on the cache's device")
    k = torch.empty((pages.shape[0], c.kv_heads, c.page_size, c.head_dim), dtype=dtype, device=cache_k.device)
    v = torch.empty_like(k)
    with torch.cuda.device(cache_k.device):
        st = library().qm_kv_read_i8(ctypes.byref(c), pages.data_ptr(), pages.shape[0], _KINDS[dtype], k.data_ptr(), v.data_ptr(), _stream_ptr(cache_k))
    _check(st, "qm_kv_read_i8")
    return k, v


class PagedKVCache:
    """The three tensors of a cache and the calls on them: ``append``, ``attend`` and ``read`` as the functions of this module, without the tensors. Which
    page belongs to which sequence is the caller's to decide."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 16, device="cuda"):
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS or pages < 0 or kv_heads < 1:
            raise QuadmulError(f"PagedKVCache: pages of {PAGE_SIZES} tokens, heads of {HEAD_DIMS}")
        self.k = torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.int8, device=device)
        self.v = torch.zeros((pages, kv_heads, head_dim, page_size), dtype=torch.int8, device=device)
        self.scales = torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=device)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def append(self, k, v, block_table, lengths, query_start=None, **options):
        return append(k, v, self.k, self.v, self.scales, block_table, lengths, query_start, **options)

    def attend(self, q, block_table, lengths, query_start=None, **options):
        return attend(q, self.k, self.v, self.scales, block_table, lengths, query_start, **options)

    def read(self, pages, dtype=torch.float16):
        return read(self.k, self.v, self.scales, pages, dtype)
