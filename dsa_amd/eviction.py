"""Eviction from a paged cache by accumulated attention weight.

The reference keeps every key and selects among them (metrics.py:9-22); a cache
that does not fit is cut instead.  What a key has had of the softmax weights of the
queries so far says what it is worth, and a sequence is cut to its newest keys and
those of largest weight:

  new_weights          no key has had any: fp32 ``[kv_heads, cache.rows]``
  accumulate_weights   adds what an attention's rows gave each key
                       (``dsa_paged_weights``)
  evict                cuts each sequence, in place (``dsa_paged_evict``)

A program calls ``paged.attention(..., return_lse=True)``, then ``accumulate_weights``
with the same arguments and the log sums, and ``evict`` when a sequence has outgrown
its budget; it goes on appending at the new length.  Positions then no longer count
tokens: rotate by the token's own position, and where an indexer's keys lie beside the
cache, move them by the list that ``evict`` returns.  Weights belong to cache rows: those
of pages that go to another sequence have to be zeroed (``weights[:, rows] = 0``).

Every call may be captured in a HIP graph, under the conditions of :mod:`dsa_amd.paged`.
"""

from __future__ import annotations

import torch

from . import _lib
from .paged import PagedCache, _batch, _integers, _queries


def new_weights(cache: PagedCache) -> torch.Tensor:
    """Zeros ``[kv_heads, cache.rows]``: the weight of each kv head's key in each
    cache row."""

    return torch.zeros((cache.kv_heads, cache.rows), dtype=torch.float32, device=cache.device)


def _weights(weights: torch.Tensor, cache: PagedCache) -> torch.Tensor:
    if weights.dtype is not torch.float32 or weights.shape != (cache.kv_heads, cache.rows) or not weights.is_contiguous():
        raise ValueError("weights must be contiguous FP32 [kv_heads,cache.rows]")
    if weights.get_device() != cache._index:
        raise ValueError("weights and cache must be on one GPU")
    return weights


def accumulate_weights(
    weights: torch.Tensor,
    queries: torch.Tensor,
    cache: PagedCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    lse: torch.Tensor,
    starts: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    causal: bool = True,
) -> None:
    """Adds to ``weights`` ``[kv_heads, cache.rows]``, in place, what each cached key
    has of the softmax weights of the tokens ``queries``: over the rows (tokens and
    heads of the key's kv head) that see it, the sum of exp(scale q.k - lse).

    The other arguments are those of :func:`dsa_amd.paged.attention`, and ``lse``
    ``[T, heads]`` fp32 what it returned for them; a row whose log sum is -inf adds
    nothing.  Some of a prompt's tokens, its last ones say, may be given alone.  Sums
    are fp32; the same call gives the same bits, unless sequences share pages, whose keys
    get the sums of all of them.  A sequence batched with others may get other last bits:
    the order of its sums follows the whole call.
    """

    weights = _weights(weights, cache)
    queries, query_stride, tokens, heads = _queries(queries, cache)
    page_table, sequences, columns, table_stride, lengths, starts = _batch(tokens, cache, page_table, lengths, starts)
    if lse.shape != (tokens, heads) or lse.dtype is not torch.float32 or lse.get_device() != cache._index:
        raise ValueError("lse must be FP32 [tokens,heads] on the cache's GPU")
    if tokens == 0:
        return
    lse = lse.contiguous()
    stream = _lib.stream_of(queries)
    ws, need = cache._workspace(stream, "dsa_paged_weights_workspace_bytes", sequences, tokens, heads, columns,
                                starts is None, kind="paged_weights", zeroed_rows=None)
    _lib.call("dsa_paged_weights", cache._address, queries.data_ptr(), query_stride, page_table.data_ptr(), table_stride,
              columns, lengths.data_ptr(), _lib.ptr(starts), sequences, tokens, heads, cache._code,
              cache.head_dim**-0.5 if scale is None else scale, causal, lse.data_ptr(), weights.data_ptr(), ws, need,
              stream)


def evict(
    cache: PagedCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    weights: torch.Tensor,
    keep: int,
    *,
    recent: int = 0,
    per_head: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cuts each sequence of ``lengths`` ``[B]`` keys to at most ``keep``, in place:
    its newest ``recent`` ones and those of largest weight among the others (ties: the
    lowest position; NaN counts as the least).  Shorter sequences stay as they are.

    All heads keep the same keys, by the sum of their weights, or with ``per_head``
    each kv head its own by its own: positions are then no longer one token's, and
    :func:`dsa_amd.paged.selected_attention` no longer fits.  Kept keys below the new
    length stay where they lie, those past it fill the freed positions in order; the
    weights move with them, and those past the new lengths become 0.  No page may be
    of two sequences.

    Returns the new lengths, int32 ``[B]``, and int64 ``[B, keep]`` (``per_head``:
    ``[B, kv_heads, keep]``) the former position of the key now at each position, -1
    past the new length.  The page ids past the new lengths are free again.
    """

    weights = _weights(weights, cache)
    page_table, sequences, columns, table_stride, lengths, _ = _batch(0, cache, page_table, lengths, None)
    if isinstance(keep, bool) or not isinstance(keep, int) or not 0 < keep <= 1 << 30:
        raise ValueError("keep must be a positive integer")
    if isinstance(recent, bool) or not isinstance(recent, int) or not 0 <= recent <= keep:
        raise ValueError("recent must be an integer from 0 to keep")
    out = torch.empty_like(lengths)
    kept = torch.empty((sequences, cache.kv_heads, keep) if per_head else (sequences, keep), dtype=torch.int64,
                       device=cache.device)
    stream = _lib.stream_of(weights)
    ws, need = cache._workspace(stream, "dsa_paged_evict_workspace_bytes", sequences, columns, keep, bool(per_head),
                                kind="paged_evict", zeroed_rows=None)
    _lib.call("dsa_paged_evict", cache._address, page_table.data_ptr(), table_stride, columns, lengths.data_ptr(),
              sequences, weights.data_ptr(), keep, recent, bool(per_head), out.data_ptr(), kept.data_ptr(), ws, need,
              stream)
    return out, kept
