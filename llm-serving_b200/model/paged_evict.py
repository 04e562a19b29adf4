"""Eviction from a paged KV cache by accumulated attention weight.

A row that reached its budget gives up the tokens that its queries have looked at least: a decode that
adds up every cached token's attention weights, and the eviction that keeps the heaviest tokens of each (layer,
row, kv head), next to the first and the last ones, and closes the ranks. Keys are cached rotated, so a kept
token keeps its meaning wherever it moves; only the cache's length shrinks, not the position of the next token.
The reference never evicts, so there is no counterpart there.

* :func:`paged_decode_weights` -- ``paged_decode`` that adds attention weights to running sums;
* :func:`evict_tokens` -- every layer's tokens cut down to a budget, in place or into other pages.

Tensors on CUDA, the current stream, no host synchronisation. There is no CPU path and no fallback.
"""

from __future__ import annotations

from model import _native

__all__ = ["evict_tokens", "paged_decode_weights"]


def paged_decode_weights(q, k_cache, v_cache, block_table, seqlen, weights, *, scale: float | None = None, out=None,
                         workspace=None):
    """Decode one query token per row (``paged_decode``), and add to ``weights[b, g, j]``, for every token ``j``
    below ``seqlen[b]``, its attention weight summed over the query heads of kv head ``g`` (one kernel launch for few
    rows, else one for every 4096 rows and one for the sums).

    ``weights`` is float32 ``(B, H_kv, W)``, ``W`` at least the table's capacity, updated in place; what lies at
    or past a row's length is left as it is. A row's weights of one step sum to the number of query heads per
    kv head. ``workspace`` as in :func:`model.paged_window.paged_decode_window`; a call of more than a few rows
    also takes 4 bytes per query head and token of the table from the allocator while it runs. Other arguments and
    types as there.
    """
    ops = _native.ops or _native.require_ops()
    return ops.decode_weights(q, k_cache, v_cache, block_table, seqlen, weights, scale, out, workspace)


def evict_tokens(k_caches, v_caches, block_table, seqlen, weights, keep: int, *, recent: int = 0, sinks: int = 0,
                 new_table=None, seqlen_out=None, weights_out=None):
    """Cut every row above ``keep`` tokens down to ``keep``, in every layer (two kernel launches for 64 layers).

    Per layer, row and kv head of ``n > keep`` tokens, the first ``sinks`` and the last ``recent`` stay
    (``sinks + recent <= keep``); of the others those with the largest ``weights[layer, b, g, j]``: a tie
    keeps the lower ``j``, NaN counts as the smallest. The kept tokens' K and V move, in their order, to
    positions ``0 .. keep - 1`` of the row's pages, so heads of one row may hold different tokens there.

    ``k_caches`` / ``v_caches``: one pool per layer, of one layout, each named once; up to 131,071 (row, kv head) pairs. ``weights`` float32
    ``(n_layer, B, H_kv, W)``, ``W`` at least the table's capacity. With ``new_table`` (int32 ``(B, max_blocks)``) the kept tokens go
    to its pages instead, shorter rows are copied there whole, and the old pages keep what they hold: that is
    for rows whose pages others share. A block that is written for one row must be read or written
    for no other: without ``new_table`` rows share no blocks, and its blocks are distinct and in no old table
    (nothing on the host can check that without waiting for the device; ``block_table`` itself is refused).

    Returns ``(seqlen, weights)``: int32 ``min(n, keep)`` and the kept tokens' weights in their new places,
    zeros behind them; new tensors, or ``seqlen_out`` / ``weights_out``, which may be the inputs themselves.
    A block id outside the pool is skipped and sets ``_native.DEVERR_COPY_RANGE`` in the device error word.
    """
    ops = _native.ops or _native.require_ops()
    k_caches = k_caches if isinstance(k_caches, list) else list(k_caches)
    v_caches = v_caches if isinstance(v_caches, list) else list(v_caches)
    return ops.evict(k_caches, v_caches, block_table, seqlen, weights, keep, recent, sinks, new_table, seqlen_out,
                     weights_out)
