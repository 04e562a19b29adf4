"""Pages copied between blocks of a pool, in every layer, in one launch.

What block sharing (``serve.block_sharing``) needs of the device: a fork copies its last, partly
filled page; a write to a shared page first copies it; a compaction moves pages down and renumbers
the block tables. The reference's pools are never rearranged, so there is no counterpart there.
"""

from __future__ import annotations

import torch

from model import _native

__all__ = ["copy_blocks"]


def _checked(name: str, ids, pool: torch.Tensor) -> list[int]:
    """Block ids given as Python ints."""
    ids = list(ids)
    for i in ids:
        if isinstance(i, bool) or not isinstance(i, int):
            raise ValueError(f"{name} must hold ints, got {i!r}")
        if not 0 <= i < pool.shape[0]:
            raise IndexError(f"{name}: block id {i} outside the pool's {pool.shape[0]} blocks")
    if name == "dst" and len(set(ids)) != len(ids):
        raise ValueError("dst holds a block id twice")
    return ids


def copy_blocks(pools, src, dst, *, block_table=None, remap=None) -> None:
    """Block ``dst[i]`` of every pool takes the bytes of block ``src[i]``, in place.

    ``pools`` is a ``PagedPool`` / ``Fp4Pool``, or tensors whose first dimension is the blocks, all
    with one shape and type, contiguous, on one CUDA device. ``src`` and ``dst`` are device vectors
    (int32 or int64; ids outside the pool are skipped and set ``_native.DEVERR_COPY_RANGE`` in the
    device error word) or Python ints (checked here: ValueError). Destinations must be distinct and none
    may be the source of another copy: the copies run side by side. One plan of the block manager
    keeps to that; plans joined into one call do only if none was made from a block that another has
    yet to fill (a fork of a fork: copy before the second). Nothing on the host can check device vectors
    without waiting for them. With ``block_table`` (int32 ``(B, max_blocks)``) and
    ``remap`` (int32 ``(n_blocks,)``), every table entry ``e`` inside the pool becomes ``remap[e]``
    in the same launch; that is for tables of the caller's own and for ``Fp4KV.move_blocks``, not for the
    table of a live ``PagedKV``, which is fixed: after moving a ``PagedPool``'s blocks, build its
    containers and captured steps anew over renumbered tables. Runs on the current stream.
    """
    ops = _native.ops or _native.require_ops()
    if hasattr(pools, "block_tensors"):
        pools = pools.block_tensors()
    elif not isinstance(pools, list):
        pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    if not isinstance(src, torch.Tensor) or not isinstance(dst, torch.Tensor):
        if not pools or not isinstance(pools[0], torch.Tensor) or pools[0].dim() == 0:
            raise ValueError("copy_blocks needs at least one pool of (n_blocks, ...) elements")
        src, dst = (ids if isinstance(ids, torch.Tensor) else _checked(name, ids, pools[0])
                    for name, ids in (("src", src), ("dst", dst)))
        if isinstance(src, list) and isinstance(dst, list):
            sources = set(src)
            for a, b in zip(src, dst):
                if b in sources and a != b:
                    raise ValueError(f"block {b} is the destination of one copy and the source of another")
        src, dst = (ids if isinstance(ids, torch.Tensor) else torch.tensor(ids, dtype=torch.int64, device=pools[0].device)
                    for ids in (src, dst))
    ops.block_copy(pools, src, dst, block_table, remap)
