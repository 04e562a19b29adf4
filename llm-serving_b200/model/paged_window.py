"""Attention over a paged KV cache that sees a window: the last ``window`` tokens and the first ``sinks``.

Key ``j`` is visible to the query at position ``i`` if ``j <= i`` and (``i - j < window`` or ``j < sinks``). A
row's step then costs its window, not its length, and what a table names for pages that hold no
visible token does not matter: their blocks may be given back (``model.paged.PagedKV(window=, sinks=)`` says which). The
reference has no windowed attention to mirror.

* :func:`paged_decode_window` -- one query token per row (``paged_decode``'s contract);
* :func:`paged_prefill_window` -- a chunk of query tokens per row (``paged_prefill``'s contract).

Tensors on CUDA, the current stream, no host synchronisation: ``seqlen`` is never read on the host, lengths (int32, or
int64 that fit it) are clamped to the table's capacity on the device. Rows of length 0 give zeros; a block id outside the pool reads
zeros. Pools need a unit head_dim stride and strides of 16-byte multiples (any contiguous pool has them). There
is no CPU path and no fallback.
"""

from __future__ import annotations

import torch

from model import _native

__all__ = ["decode_workspace", "paged_decode_window", "paged_prefill_window"]


def decode_workspace(rows: int, n_head: int, n_kv_head: int, head_dim: int, like: torch.Tensor) -> torch.Tensor:
    """A workspace of its own for decode calls of :mod:`model.paged_window` and :mod:`model.paged_evict` that
    may run beside others: up to ``rows`` rows of these heads, in ``like``'s dtype and on its device."""
    return _native.require_ops().decode_window_workspace(rows, n_head, n_kv_head, head_dim, like)


def paged_decode_window(q, k_cache, v_cache, block_table, seqlen, window: int, *, sinks: int = 0,
                        scale: float | None = None, out=None, workspace=None):
    """Decode one query token per row, at position ``seqlen[b] - 1``, against its window of a paged pool (one
    kernel launch for every 4096 rows).

    ``q`` ``(B, H, D)`` in the pools' dtype (fp16, bf16 or fp32); head_dim a power of two in 8..256; any number
    of query heads per kv head. ``window`` is at least 1, ``sinks`` at least 0; either may exceed the rows.
    Of row ``b``'s table only the entries of pages with a visible token matter. ``workspace`` (optional) is a
    tensor of :func:`decode_workspace` that no concurrent launch uses; without it the eager calls of one stream
    share one, and those of a graph's capture another that is the graph's own.
    """
    ops = _native.ops or _native.require_ops()
    return ops.decode_window(q, k_cache, v_cache, block_table, seqlen, window, sinks, scale, out, workspace)


def paged_prefill_window(q, k_cache, v_cache, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q: int, window: int, *,
                         sinks: int = 0, scale: float | None = None, out=None):
    """Attention of a chunk of query tokens per row, each against its window of a paged pool (one kernel launch).

    ``paged_prefill``'s contract: ``q`` is the packed ``(total_q, H, D)``, row ``b`` owning
    ``q[cu_seqlens_q[b]:cu_seqlens_q[b + 1]]``; the chunk's K/V are already in the pools, and its token ``i`` of
    ``Sq`` sits at position ``seqlen_k[b] - Sq + i``. ``max_seqlen_q`` must be at least the longest chunk;
    tokens of a longer one past it, and those of no row, are left unwritten. It changes no result but sizes the launch: a loose
    bound costs time (16 chunks of 1 to 8 tokens 17.4 us with 8, 23.2 with 81), and so does one long chunk beside many
    short ones, which are better attended in a call of their own. A token that sees no key gives zeros.

    fp16 or bf16, head_dim 64, 128 or 256, block_size at least 8, any number of query heads per kv head. Scores
    and sums are fp32; the weights enter the second product in two 16-bit parts.
    """
    ops = _native.ops or _native.require_ops()
    return ops.prefill_window(q, k_cache, v_cache, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q, window, sinks, scale,
                              out)
