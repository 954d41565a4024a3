"""A paged key/value cache, and attention over it: what the indexer selects for.

The reference scores the cached keys (sidecar.py:89-107), selects each query's
top-k (metrics.py:9-22) and hands the positions back to the model's own
attention.  Here the cache and that attention are operators of the library:

  PagedCache          the cache: pages of key and value rows, bf16, fp16, fp8
                      e4m3 with one fp32 scale per row and head, or fp4 e2m1
                      with a power of two (e8m0) per 32 dims
  new_cache           an empty one
  cache_rows          the cache rows of positions, through a page table
  append              new tokens' keys and values, rotated to their positions,
                      into cache rows (``dsa_paged_append``)
  read                what cache rows stand for (``dsa_paged_read``)
  attention           each sequence's newest tokens, one or a chunk, over its
                      whole cache (``dsa_paged_attention``)
  selected_attention  each token over the positions its index list names, as
                      ``decode.indexer_topk`` and ``sidecar.score_encoded_topk``
                      give them (``dsa_paged_selected_attention``)

Query heads share kv heads in equal groups: head h reads kv head
h * kv_heads // heads.  Inference only: no autograd graph is kept.

Every call may be captured in a HIP graph.  Attention calls on one stream share its
workspace (:func:`dsa_amd._lib.workspace`), and so do graphs that were captured on
it: replay them one after the other, not side by side on several streams.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

HEAD_DIMS = (64, 128, 256)
POWER_DIMS = 32  # dims of an fp4 head that share a power of two
FP4 = getattr(torch, "float4_e2m1fn_x2", None)  # None: a torch without it, which has the other caches
_CACHE_DTYPES = tuple(t for t in (torch.bfloat16, torch.float16, torch.float8_e4m3fn, FP4) if t is not None)


class PagedCache:
    """Keys and values ``[pages, page_size, kv_heads, head_dim]``, of any page,
    slot and head strides (16-byte aligned heads of contiguous dims), with
    ``key_scales`` / ``value_scales`` ``[pages, page_size, kv_heads]`` fp32 when
    they are fp8 e4m3fn.  Of fp4 e2m1 (``torch.float4_e2m1fn_x2``, two codes an
    element, the first in the low half) they are ``[pages, page_size, kv_heads,
    head_dim / 2]``, and the scales e8m0 (``torch.float8_e8m0fnu``) ``[pages, kv_heads,
    page_size, head_dim / 32]``.  The tensors are the caller's and are written in place;
    cache row r is slot ``r % page_size`` of page ``r // page_size``."""

    __slots__ = ("keys", "values", "key_scales", "value_scales", "pages", "page_size", "kv_heads", "head_dim", "dtype",
                 "row_dtype", "device", "_index", "_code", "_struct", "_address", "_needs")

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor | None = None,
                 value_scales: torch.Tensor | None = None) -> None:
        if keys.ndim != 4 or values.shape != keys.shape:
            raise ValueError("keys and values must both be [pages,page_size,kv_heads,head_dim]")
        if keys.dtype not in _CACHE_DTYPES or values.dtype != keys.dtype:
            raise ValueError("a paged cache is BF16, FP16 or FP8 e4m3fn, or FP4 e2m1fn_x2")
        if not (keys.is_cuda and values.is_cuda) or keys.device != values.device:
            raise ValueError("HIP kernels require GPU tensors")
        pages, page_size, kv_heads, head_dim = keys.shape
        fp4 = keys.dtype == FP4
        if fp4:
            head_dim *= 2
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if head_dim not in HEAD_DIMS:
            raise ValueError("head_dim must be 64, 128 or 256")
        if pages < 1 or kv_heads < 1:
            raise ValueError("need at least one page and one kv head")
        for t in (keys, values):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(s * t.element_size() % 16 for s in t.stride()[:3]):
                raise ValueError("cache heads must be contiguous and 16-byte aligned")
        fp8 = keys.dtype == torch.float8_e4m3fn
        for t in (key_scales, value_scales):
            if fp8 and (t is None or t.shape != keys.shape[:3] or t.dtype != torch.float32 or not t.is_contiguous()
                        or t.device != keys.device):
                raise ValueError("an fp8 cache needs contiguous fp32 scales [pages,page_size,kv_heads]")
            if fp4 and (t is None or t.shape != (pages, kv_heads, page_size, head_dim // POWER_DIMS)
                        or t.dtype != torch.float8_e8m0fnu or not t.is_contiguous() or t.data_ptr() % 16
                        or t.device != keys.device):
                raise ValueError("an fp4 cache needs contiguous, 16-byte aligned e8m0 scales "
                                 "[pages,kv_heads,page_size,head_dim/32]")
            if not (fp8 or fp4) and t is not None:
                raise ValueError("only an fp8 or fp4 cache has scales")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self.dtype = keys.dtype
        self.row_dtype = torch.bfloat16 if fp8 or fp4 else keys.dtype  # of the queries and of appended rows
        self.device = keys.device
        self._index = keys.get_device()
        self._code = _lib.dtype_code(self.row_dtype)
        self._needs: dict[tuple, int] = {}
        self._struct = _lib.PagedCacheC(
            _lib.ptr(keys), _lib.ptr(values), _lib.ptr(key_scales), _lib.ptr(value_scales), pages, *keys.stride()[:3],
            *values.stride()[:3], page_size, kv_heads, head_dim, _lib.dtype_code(keys.dtype))
        self._address = ctypes.addressof(self._struct)

    @property
    def rows(self) -> int:
        return self.pages * self.page_size

    def _workspace(self, stream: int, entry: str, *sizes: int, kind: str = "paged_attention",
                   zeroed_rows: int | None = 0) -> tuple[int | None, int]:
        """Address and size of the workspace that ``entry`` asks for at these sizes;
        ``zeroed_rows`` as :func:`dsa_amd._lib.workspace`'s rows, None if it needs no zeros."""

        need = self._needs.get((entry, sizes))
        if need is None:
            if len(self._needs) >= 256:  # a serving loop's sizes; a prompt's do not pile up
                self._needs.clear()
            need = self._needs[entry, sizes] = _lib.query(entry, self._address, *sizes)
        if need <= 0:
            return None, 0
        return _lib.workspace(kind, self.device, stream, need, zeroed=zeroed_rows is not None,
                              rows=zeroed_rows or 0).data_ptr(), need


def new_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> PagedCache:
    """An empty cache.  Its rows are uninitialised: attention reads none that
    was not appended.  In an fp4 one a page's rows of one head lie together: a row
    of its own is 64 bytes at head_dim 128, half of what memory serves well."""

    if FP4 is not None and dtype == FP4:
        if head_dim not in HEAD_DIMS:
            raise ValueError("head_dim must be 64, 128 or 256")
        parts = [torch.empty((pages, kv_heads, page_size, n), dtype=torch.uint8, device=device)
                 for n in (head_dim // 2, head_dim // 2, head_dim // POWER_DIMS, head_dim // POWER_DIMS)]
        return PagedCache(*(x.transpose(1, 2).view(FP4) for x in parts[:2]),
                          *(x.view(torch.float8_e8m0fnu) for x in parts[2:]))
    shape = (pages, page_size, kv_heads, head_dim)
    keys, values = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype != torch.float8_e4m3fn:
        return PagedCache(keys, values)
    key_scales, value_scales = (torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
    return PagedCache(keys, values, key_scales, value_scales)


def cache_rows(cache: PagedCache, page_table: torch.Tensor, positions: torch.Tensor,
               sequences: torch.Tensor | None = None) -> torch.Tensor:
    """int64 cache rows of ``positions`` ``[T]``; token t belongs to sequence
    ``sequences[t]`` (default: token t to sequence t).  Padding, which is any token
    whose position or sequence is not in the page table (-1), has row -1."""

    if page_table.ndim != 2 or positions.ndim != 1:
        raise ValueError("page_table must be [sequences,columns] and positions [tokens]")
    size = cache.page_size
    count, columns = page_table.shape
    positions = positions.long()
    if page_table.numel() == 0:
        return torch.full_like(positions, -1)
    inside = positions.clamp(0, columns * size - 1)
    column = inside >> (size.bit_length() - 1)
    padding = inside != positions
    if sequences is None:
        if positions.shape[0] != count:
            raise ValueError("without sequences there is one token per sequence")
        page = page_table.gather(1, column.unsqueeze(1)).squeeze(1)
    else:
        sequences = sequences.to(positions.device, torch.int64)
        at = sequences.clamp(0, count - 1)
        padding = padding.logical_or_(at != sequences)
        page = page_table.take(torch.add(column, at, alpha=columns))
    return torch.add(inside & (size - 1), page, alpha=size).masked_fill_(padding, -1)


# A short call is bound by the host, so its checks are the cheap ones where they
# pass: sizes are unpacked once, devices compared by index, and only tensors that
# are not as the kernels read them take another look.


def _rows(x: torch.Tensor, heads: int, dim: int) -> tuple[torch.Tensor, int]:
    """``x`` ``[T, heads, dim]`` as rows the kernels read (heads packed, tokens
    16-byte aligned at any stride), and its token stride."""

    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, heads * dim
    stride, head, unit = x.stride()
    packed = unit == 1 and (head == dim or heads == 1)
    if x.shape[0] == 1 and packed:
        stride = heads * dim
    if not packed or stride % 8 or stride < heads * dim or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        stride = heads * dim
    return x, stride


def _like(x: torch.Tensor, stride: int, heads: int, dim: int) -> torch.Tensor:
    """An uninitialised dense tensor like the rows ``x`` (empty_like is the
    cheaper call by 0.6 us, a twentieth of a short call's host time)."""

    return torch.empty_like(x) if stride == heads * dim else torch.empty(x.shape, device=x.device, dtype=x.dtype)


def _queries(queries: torch.Tensor, cache: PagedCache) -> tuple[torch.Tensor, int, int, int]:
    """Checked queries, their token stride, tokens and heads."""

    if queries.ndim != 3:
        raise ValueError("queries must be [tokens,heads,head_dim]")
    tokens, heads, dim = queries.shape
    if dim != cache.head_dim:
        raise ValueError("queries must be [tokens,heads,head_dim]")
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError("heads must be a multiple of the cache's kv_heads")
    if queries.dtype is not cache.row_dtype:
        raise ValueError("queries must have the cache's dtype (BF16 for an FP8 or FP4 cache)")
    if queries.get_device() != cache._index:
        raise ValueError("queries and cache must be on one GPU")
    queries, stride = _rows(queries, heads, dim)
    return queries, stride, tokens, heads


def _integers(x: torch.Tensor, dtype: torch.dtype, name: str, cache: PagedCache) -> torch.Tensor:
    """``x`` as contiguous ``dtype`` on the cache's GPU."""

    if x.dtype is dtype and x.get_device() == cache._index and x.is_contiguous():
        return x
    if x.is_floating_point() or x.is_complex():
        raise ValueError(f"{name} must be integers")
    return x.to(device=cache.device, dtype=dtype).contiguous()


def append(
    cache: PagedCache,
    keys: torch.Tensor,
    values: torch.Tensor,
    rows: torch.Tensor,
    positions: torch.Tensor,
    *,
    queries: torch.Tensor | None = None,
    rope_dim: int | None = None,
    theta: float = 10_000.0,
) -> torch.Tensor | None:
    """Writes tokens' ``keys`` and ``values`` ``[T, kv_heads, head_dim]`` into
    cache rows ``rows`` ``[T]``, the keys rotated to ``positions`` ``[T]`` by the
    non-interleaved RoPE of their first ``rope_dim`` dims (default: all; 0: none).

    With ``queries`` ``[T, heads, head_dim]`` the rotated queries are returned.
    Tokens whose row is outside the cache (-1: padding) are not written; no two
    tokens may have the same row.  An fp8 cache scales each head by its largest
    magnitude, an fp4 one each 32 dims by the least power of two, 2^125 at most, under
    which theirs is 7 or less: no value up to 7 * 2^125 (2.98e38; larger ones become 6 *
    2^125) is then off by more than half a step of the codes, and what is not finite
    makes its 32 dims NaN.  The angles are exact to fp32 at any position; taken as an fp32
    product, as the sidecar's encoders and many models take theirs, they are 0.0006
    rad off at position 65535, so keys and queries are best rotated by one of the two.
    """

    dim, kv_heads = cache.head_dim, cache.kv_heads
    if keys.ndim != 3 or values.shape != keys.shape:
        raise ValueError("keys and values must both be [tokens,kv_heads,head_dim]")
    tokens, rows_heads, rows_dim = keys.shape
    if rows_heads != kv_heads or rows_dim != dim:
        raise ValueError("keys and values must both be [tokens,kv_heads,head_dim]")
    if keys.dtype is not cache.row_dtype or values.dtype is not cache.row_dtype:
        raise ValueError("appended rows must have the cache's dtype (BF16 for an FP8 or FP4 cache)")
    if keys.get_device() != cache._index or values.get_device() != cache._index:
        raise ValueError("appended rows and cache must be on one GPU")
    if rows.ndim != 1 or len(rows) != tokens or positions.shape != rows.shape:
        raise ValueError("rows and positions must be [tokens]")
    if rope_dim is None:
        rope_dim = dim
    if rope_dim % 16 or not 0 <= rope_dim <= dim:
        raise ValueError("rope_dim must be a multiple of 16 no larger than head_dim")
    if not 0 < theta < math.inf:
        raise ValueError("theta must be positive")
    rows = _integers(rows, torch.int64, "rows", cache)
    positions = _integers(positions, torch.int64, "positions", cache)
    out = None
    heads = query_stride = 0
    if queries is not None:
        queries, query_stride, query_tokens, heads = _queries(queries, cache)
        if query_tokens != tokens:
            raise ValueError("queries must be [tokens,heads,head_dim]")
        out = _like(queries, query_stride, heads, dim)
    if tokens == 0:
        return out
    keys, key_stride = _rows(keys, kv_heads, dim)
    values, value_stride = _rows(values, kv_heads, dim)
    _lib.call("dsa_paged_append", cache._address, keys.data_ptr(), key_stride, values.data_ptr(), value_stride,
              _lib.ptr(queries), query_stride, _lib.ptr(out), heads, cache._code, rows.data_ptr(),
              positions.data_ptr(), tokens, rope_dim, theta, _lib.stream_of(keys))
    return out


def read(cache: PagedCache, rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and the values ``[n, kv_heads, head_dim]`` that cache rows ``rows``
    ``[n]`` stand for, in the type that rows are appended in: the rows themselves
    of a 16-bit cache, bf16 for fp8 (rounded) and fp4 (exact, infinite from 2^128
    on).  Rows outside the cache (-1: padding) give zeros."""

    if rows.ndim != 1:
        raise ValueError("rows must be [n]")
    rows = _integers(rows, torch.int64, "rows", cache)
    count = len(rows)
    keys = torch.empty((count, cache.kv_heads, cache.head_dim), dtype=cache.row_dtype, device=cache.device)
    values = torch.empty_like(keys)
    if count:
        _lib.call("dsa_paged_read", cache._address, rows.data_ptr(), count, keys.data_ptr(), values.data_ptr(),
                  _lib.stream_of(keys))
    return keys, values


def _batch(tokens: int, cache: PagedCache, page_table, lengths, starts):
    """Checked page table with its sizes and row stride, lengths and starts."""

    if page_table.ndim != 2 or 0 in page_table.shape:
        raise ValueError("page_table must be [sequences,columns]")
    sequences, columns = page_table.shape
    if lengths.ndim != 1 or len(lengths) != sequences:
        raise ValueError("lengths must be [sequences]")
    stride, unit = page_table.stride()
    if (page_table.dtype is not torch.int32 or page_table.get_device() != cache._index or unit != 1
            or (stride < columns and sequences > 1)):
        page_table = _integers(page_table, torch.int32, "page_table", cache)
        stride = columns
    if sequences == 1:
        stride = columns
    if starts is None:
        if tokens % sequences:
            raise ValueError("without starts every sequence has the same number of tokens")
    elif starts.ndim != 1 or len(starts) != sequences + 1:
        raise ValueError("starts must be [sequences + 1]")
    else:
        starts = _integers(starts, torch.int32, "starts", cache)
    return page_table, sequences, columns, stride, _integers(lengths, torch.int32, "lengths", cache), starts


def attention(
    queries: torch.Tensor,
    cache: PagedCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    starts: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    causal: bool = True,
    return_lse: bool = False,
):
    """Softmax attention of each sequence's newest tokens over its cached keys.

    queries ``[T, heads, head_dim]`` of the cache's dtype (bf16 for fp8 and fp4), already
    rotated; ``page_table`` ``[B, columns]`` int32 page ids; ``lengths`` ``[B]``
    int32 keys of each sequence, the new tokens' own included.  Sequence b's
    tokens are ``starts[b] .. starts[b + 1]`` (``[B + 1]`` int32, ascending, within
    0 .. T; tokens outside ``starts[0] .. starts[B]`` are padding, which sees no key);
    without ``starts`` every sequence has T / B.  ``causal``: the i-th of n new tokens
    sees keys ``j <= lengths[b] - n + i``.  ``scale`` defaults to head_dim^-0.5.

    Returns ``[T, heads, head_dim]`` in the queries' dtype, and with
    ``return_lse`` the natural log of each row's softmax denominator, fp32
    ``[T, heads]``.  A row that sees no key gets zeros and -inf; what a row does
    not see does not reach it, whatever it holds.
    """

    queries, query_stride, tokens, heads = _queries(queries, cache)
    page_table, sequences, columns, table_stride, lengths, starts = _batch(tokens, cache, page_table, lengths, starts)
    dim = cache.head_dim
    out = _like(queries, query_stride, heads, dim)
    lse = torch.empty((tokens, heads), device=cache.device, dtype=torch.float32) if return_lse else None
    if tokens:
        stream = _lib.stream_of(queries)
        ws, need = cache._workspace(stream, "dsa_paged_attention_workspace_bytes", sequences, tokens, heads, columns,
                                    starts is None)
        _lib.call("dsa_paged_attention", cache._address, queries.data_ptr(), query_stride, page_table.data_ptr(),
                  table_stride, columns, lengths.data_ptr(), _lib.ptr(starts), sequences, tokens, heads, cache._code,
                  dim**-0.5 if scale is None else scale, causal, out.data_ptr(), _lib.ptr(lse), ws, need, stream)
    return (out, lse) if return_lse else out


def selected_attention(
    queries: torch.Tensor,
    cache: PagedCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    indices: torch.Tensor,
    starts: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    return_lse: bool = False,
):
    """``attention`` of each token over the positions that its row of ``indices``
    ``[T, k]`` names, for all of its heads: positions in the token's sequence in
    any order; entries below 0 or at or past the sequence's length are padding.
    The lists of ``indexer_topk`` and ``score_encoded_topk`` fit as they are (int64
    with contiguous entries is read in place).
    """

    queries, query_stride, tokens, heads = _queries(queries, cache)
    page_table, sequences, columns, table_stride, lengths, starts = _batch(tokens, cache, page_table, lengths, starts)
    dim = cache.head_dim
    if indices.ndim != 2 or indices.shape[0] != tokens:
        raise ValueError("indices must be [tokens,k]")
    k = indices.shape[1]
    index_stride, unit = indices.stride()
    if indices.dtype is not torch.int64 or indices.get_device() != cache._index or (k > 1 and unit != 1) or index_stride < k:
        indices = _integers(indices, torch.int64, "indices", cache)
        index_stride = k
    out = _like(queries, query_stride, heads, dim)
    lse = torch.empty((tokens, heads), device=cache.device, dtype=torch.float32) if return_lse else None
    if tokens:
        stream = _lib.stream_of(queries)
        ws, need = cache._workspace(stream, "dsa_paged_selected_workspace_bytes", tokens, heads, k)
        _lib.call("dsa_paged_selected_attention", cache._address, queries.data_ptr(), query_stride,
                  page_table.data_ptr(), table_stride, columns, lengths.data_ptr(), _lib.ptr(starts), sequences, tokens,
                  heads, cache._code, indices.data_ptr(), index_stride, k, dim**-0.5 if scale is None else scale,
                  out.data_ptr(), _lib.ptr(lse), ws, need, stream)
    return (out, lse) if return_lse else out
