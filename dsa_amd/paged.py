"""A paged key/value cache, and attention over it: what the indexer selects for.

The reference scores the cached keys (sidecar.py:89-107), selects each query's
top-k (metrics.py:9-22) and hands the positions back to the model's own
attention.  Here the cache and that attention are operators of the library:

  PagedCache          the cache: pages of key and value rows, bf16, fp16 or fp8
                      e4m3 with one fp32 scale per row and head
  new_cache           an empty one
  cache_rows          the cache rows of positions, through a page table
  append              new tokens' keys and values, rotated to their positions,
                      into cache rows (``dsa_paged_append``)
  attention           each sequence's newest tokens, one or a chunk, over its
                      whole cache (``dsa_paged_attention``)
  selected_attention  each token over the positions its index list names, as
                      ``decode.indexer_topk`` and ``sidecar.score_encoded_topk``
                      give them (``dsa_paged_selected_attention``)

Query heads share kv heads in equal groups: head h reads kv head
h * kv_heads // heads.  Inference only: no autograd graph is kept.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

HEAD_DIMS = (64, 128, 256)
_CACHE_DTYPES = (torch.bfloat16, torch.float16, torch.float8_e4m3fn)


class PagedCache:
    """Keys and values ``[pages, page_size, kv_heads, head_dim]``, of any page,
    slot and head strides (16-byte aligned heads of contiguous dims), with
    ``key_scales`` / ``value_scales`` ``[pages, page_size, kv_heads]`` fp32 when
    they are fp8 e4m3fn.  The tensors are the caller's and are written in place;
    cache row r is slot ``r % page_size`` of page ``r // page_size``."""

    __slots__ = ("keys", "values", "key_scales", "value_scales", "pages", "page_size", "kv_heads", "head_dim", "dtype",
                 "row_dtype", "_struct", "_address")

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor | None = None,
                 value_scales: torch.Tensor | None = None) -> None:
        if keys.ndim != 4 or values.shape != keys.shape:
            raise ValueError("keys and values must both be [pages,page_size,kv_heads,head_dim]")
        if keys.dtype not in _CACHE_DTYPES or values.dtype != keys.dtype:
            raise ValueError("a paged cache is BF16, FP16 or FP8 e4m3fn")
        if not (keys.is_cuda and values.is_cuda) or keys.device != values.device:
            raise ValueError("HIP kernels require GPU tensors")
        pages, page_size, kv_heads, head_dim = keys.shape
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
            if not fp8 and t is not None:
                raise ValueError("only an fp8 cache has scales")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self.dtype = keys.dtype
        self.row_dtype = torch.bfloat16 if fp8 else keys.dtype  # of the queries and of appended rows
        self._struct = _lib.PagedCacheC(
            _lib.ptr(keys), _lib.ptr(values), _lib.ptr(key_scales), _lib.ptr(value_scales), pages, *keys.stride()[:3],
            *values.stride()[:3], page_size, kv_heads, head_dim, _lib.dtype_code(keys.dtype))
        self._address = ctypes.addressof(self._struct)

    @property
    def rows(self) -> int:
        return self.pages * self.page_size


def new_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> PagedCache:
    """An empty cache.  Its rows are uninitialised: attention reads none that
    was not appended."""

    shape = (pages, page_size, kv_heads, head_dim)
    keys, values = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype != torch.float8_e4m3fn:
        return PagedCache(keys, values)
    key_scales, value_scales = (torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
    return PagedCache(keys, values, key_scales, value_scales)


def cache_rows(cache: PagedCache, page_table: torch.Tensor, positions: torch.Tensor,
               sequences: torch.Tensor | None = None) -> torch.Tensor:
    """int64 cache rows of ``positions`` ``[T]``; token t belongs to sequence
    ``sequences[t]`` (default: token t to sequence t)."""

    if page_table.ndim != 2 or positions.ndim != 1:
        raise ValueError("page_table must be [sequences,columns] and positions [tokens]")
    if sequences is None:
        if positions.shape[0] != page_table.shape[0]:
            raise ValueError("without sequences there is one token per sequence")
        sequences = torch.arange(positions.shape[0], device=positions.device)
    size = cache.page_size
    positions = positions.long()
    page = page_table[sequences.long(), torch.div(positions, size, rounding_mode="floor")]
    return page.long() * size + positions % size


def _rows(x: torch.Tensor, dim: int) -> tuple[torch.Tensor, int]:
    """``x`` ``[T, heads, dim]`` as rows the kernels read (heads packed, tokens
    16-byte aligned at any stride), and its token stride."""

    heads = x.shape[1]
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


def _dense_like(x: torch.Tensor, stride: int) -> torch.Tensor:
    """An uninitialised dense tensor like the rows ``x`` (empty_like is the
    cheaper call by 0.6 us, a twentieth of a short call's host time)."""

    return torch.empty_like(x) if stride == x.shape[1] * x.shape[2] else torch.empty(x.shape, device=x.device, dtype=x.dtype)


def _queries(queries: torch.Tensor, cache: PagedCache) -> tuple[torch.Tensor, int]:
    if queries.ndim != 3 or queries.shape[2] != cache.head_dim:
        raise ValueError("queries must be [tokens,heads,head_dim]")
    if queries.shape[1] == 0 or queries.shape[1] % cache.kv_heads:
        raise ValueError("heads must be a multiple of the cache's kv_heads")
    if queries.dtype != cache.row_dtype:
        raise ValueError("queries must have the cache's dtype (BF16 for an FP8 cache)")
    if queries.device != cache.keys.device:
        raise ValueError("queries and cache must be on one GPU")
    return _rows(queries, cache.head_dim)


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
    Tokens whose row is outside the cache (-1: padding) are not written.  An fp8
    cache scales each head by its largest magnitude.
    """

    dim = cache.head_dim
    tokens = keys.shape[0]
    if keys.ndim != 3 or keys.shape[1:] != (cache.kv_heads, dim) or values.shape != keys.shape:
        raise ValueError("keys and values must both be [tokens,kv_heads,head_dim]")
    if keys.dtype != cache.row_dtype or values.dtype != keys.dtype:
        raise ValueError("appended rows must have the cache's dtype (BF16 for an FP8 cache)")
    if keys.device != cache.keys.device or values.device != keys.device:
        raise ValueError("appended rows and cache must be on one GPU")
    if rows.shape != (tokens,) or positions.shape != (tokens,):
        raise ValueError("rows and positions must be [tokens]")
    rope_dim = dim if rope_dim is None else rope_dim
    if rope_dim % 16 or not 0 <= rope_dim <= dim:
        raise ValueError("rope_dim must be a multiple of 16 no larger than head_dim")
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError("theta must be positive")
    rows, positions = _tokens(rows, keys.device), _tokens(positions, keys.device)
    out = None
    heads = query_stride = 0
    if queries is not None:
        if queries.shape[0] != tokens:
            raise ValueError("queries must be [tokens,heads,head_dim]")
        queries, query_stride = _queries(queries, cache)
        heads = queries.shape[1]
        out = _dense_like(queries, query_stride)
    if tokens == 0:
        return out
    keys, key_stride = _rows(keys, dim)
    values, value_stride = _rows(values, dim)
    _lib.call("dsa_paged_append", cache._address, keys.data_ptr(), key_stride, values.data_ptr(), value_stride,
              _lib.ptr(queries), query_stride, _lib.ptr(out), heads, _lib.dtype_code(keys.dtype), rows.data_ptr(),
              positions.data_ptr(), tokens, rope_dim, theta, _lib.stream_of(keys))
    return out


def _tokens(x: torch.Tensor, device: torch.device) -> torch.Tensor:
    if x.dtype == torch.int64 and x.device == device and x.is_contiguous():
        return x
    if x.is_floating_point() or x.is_complex():
        raise ValueError("rows and positions must be integers")
    return x.to(device=device, dtype=torch.int64).contiguous()


def _int32(x: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if x.dtype == torch.int32 and x.device == device and x.is_contiguous():
        return x
    if x.is_floating_point() or x.is_complex():
        raise ValueError(f"{name} must be integers")
    return x.to(device=device, dtype=torch.int32).contiguous()


def _batch(queries, cache, page_table, lengths, starts):
    """Checked page table, lengths and starts of a call's sequences."""

    device = cache.keys.device
    if page_table.ndim != 2 or page_table.shape[1] == 0 or page_table.shape[0] == 0:
        raise ValueError("page_table must be [sequences,columns]")
    sequences = page_table.shape[0]
    if lengths.shape != (sequences,):
        raise ValueError("lengths must be [sequences]")
    if page_table.dtype != torch.int32 or page_table.device != device or page_table.stride(1) != 1:
        page_table = _int32(page_table, "page_table", device)
    if starts is None:
        if queries.shape[0] % sequences:
            raise ValueError("without starts every sequence has the same number of tokens")
    elif starts.shape != (sequences + 1,):
        raise ValueError("starts must be [sequences + 1]")
    else:
        starts = _int32(starts, "starts", device)
    stride = page_table.stride(0) if sequences > 1 else page_table.shape[1]
    if stride < page_table.shape[1]:
        page_table = page_table.contiguous()
        stride = page_table.shape[1]
    return page_table, stride, _int32(lengths, "lengths", device), starts


def _workspace(cache: PagedCache, stream: int, need: int) -> torch.Tensor | None:
    if need <= 0:
        return None
    return _lib.workspace("paged_attention", cache.keys.device, stream, need, zeroed=True)


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

    queries ``[T, heads, head_dim]`` of the cache's dtype (bf16 for fp8), already
    rotated; ``page_table`` ``[B, columns]`` int32 page ids; ``lengths`` ``[B]``
    int32 keys of each sequence, the new tokens' own included.  Sequence b's
    tokens are ``starts[b] .. starts[b + 1]`` (``[B + 1]`` int32); without
    ``starts`` every sequence has T / B.  ``causal``: the i-th of n new tokens
    sees keys ``j <= lengths[b] - n + i``.  ``scale`` defaults to head_dim^-0.5.

    Returns ``[T, heads, head_dim]`` in the queries' dtype, and with
    ``return_lse`` the natural log of each row's softmax denominator, fp32
    ``[T, heads]``.  A row that sees no key gets zeros and -inf.
    """

    queries, query_stride = _queries(queries, cache)
    page_table, table_stride, lengths, starts = _batch(queries, cache, page_table, lengths, starts)
    tokens, heads, dim = queries.shape
    device = queries.device
    out = _dense_like(queries, query_stride)
    lse = torch.empty((tokens, heads), device=device, dtype=torch.float32) if return_lse else None
    if tokens:
        sequences, columns = page_table.shape
        stream = _lib.stream_of(queries)
        need = _lib.query("dsa_paged_attention_workspace_bytes", cache._address, sequences, tokens, heads, columns,
                          starts is None)
        ws = _workspace(cache, stream, need)
        _lib.call("dsa_paged_attention", cache._address, queries.data_ptr(), query_stride, page_table.data_ptr(),
                  table_stride, columns, lengths.data_ptr(), _lib.ptr(starts), sequences, tokens, heads,
                  _lib.dtype_code(queries.dtype), dim**-0.5 if scale is None else scale, causal, out.data_ptr(),
                  _lib.ptr(lse), _lib.ptr(ws), need, stream)
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

    queries, query_stride = _queries(queries, cache)
    page_table, table_stride, lengths, starts = _batch(queries, cache, page_table, lengths, starts)
    tokens, heads, dim = queries.shape
    device = queries.device
    if indices.ndim != 2 or indices.shape[0] != tokens:
        raise ValueError("indices must be [tokens,k]")
    if indices.is_floating_point() or indices.is_complex():
        raise ValueError("indices must be integers")
    k = indices.shape[1]
    index_stride = indices.stride(0)
    if indices.dtype != torch.int64 or indices.device != device or (k > 1 and indices.stride(1) != 1) or index_stride < k:
        indices = indices.to(device=device, dtype=torch.int64).contiguous()
        index_stride = k
    out = _dense_like(queries, query_stride)
    lse = torch.empty((tokens, heads), device=device, dtype=torch.float32) if return_lse else None
    if tokens:
        sequences, columns = page_table.shape
        stream = _lib.stream_of(queries)
        need = _lib.query("dsa_paged_selected_workspace_bytes", cache._address, tokens, heads, k)
        ws = _workspace(cache, stream, need)
        _lib.call("dsa_paged_selected_attention", cache._address, queries.data_ptr(), query_stride,
                  page_table.data_ptr(), table_stride, columns, lengths.data_ptr(), _lib.ptr(starts), sequences, tokens,
                  heads, _lib.dtype_code(queries.dtype), indices.data_ptr(), index_stride, k,
                  dim**-0.5 if scale is None else scale, out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), need, stream)
    return (out, lse) if return_lse else out
