"""Pages copied between blocks of a pool, in every layer, in one launch.

What block sharing (``serve.block_sharing``) needs of the device: a fork copies its last, partly
filled page; a write to a shared page first copies it; a compaction moves pages down and renumbers
the block tables. The reference's pools are never rearranged, so there is no counterpart there.
"""

from __future__ import annotations

import torch

from model import _native

__all__ = ["copy_blocks"]


def _ids(name: str, ids, pool: torch.Tensor) -> torch.Tensor:
    """A device vector of block ids from Python ints (a tensor passes as it is)."""
    if isinstance(ids, torch.Tensor):
        return ids
    ids = list(ids)
    for i in ids:
        if isinstance(i, bool) or not isinstance(i, int):
            raise ValueError(f"{name} must hold ints, got {i!r}")
        if not 0 <= i < pool.shape[0]:
            raise IndexError(f"{name}: block id {i} outside the pool's {pool.shape[0]} blocks")
    if name == "dst" and len(set(ids)) != len(ids):
        raise ValueError("dst holds a block id twice")
    return torch.tensor(ids, dtype=torch.int64, device=pool.device)


def copy_blocks(pools, src, dst, *, block_table=None, remap=None) -> None:
    """Block ``dst[i]`` of every pool takes the bytes of block ``src[i]``, in place.

    ``pools`` is a ``PagedPool`` / ``Fp4Pool``, or tensors whose first dimension is the blocks, all
    with one shape and type, contiguous, on one CUDA device. ``src`` and ``dst`` are device vectors
    (int32 or int64; ids outside the pool are skipped and set ``_native.DEVERR_COPY_RANGE`` in the
    device error word) or Python ints (checked here). Destinations must be distinct and none may
    also be a source, as the block manager's plans guarantee; nothing on the host can check device
    vectors without waiting for them. With ``block_table`` (int32 ``(B, max_blocks)``) and
    ``remap`` (int32 ``(n_blocks,)``), every table entry ``e`` inside the pool becomes ``remap[e]``
    in the same launch. Runs on the current stream.
    """
    ops = _native.ops or _native.require_ops()
    if hasattr(pools, "block_tensors"):
        pools = pools.block_tensors()
    elif not isinstance(pools, list):
        pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    if not isinstance(src, torch.Tensor) or not isinstance(dst, torch.Tensor):
        if not pools or not isinstance(pools[0], torch.Tensor) or pools[0].dim() == 0:
            raise ValueError("copy_blocks needs at least one pool of (n_blocks, ...) elements")
        src, dst = _ids("src", src, pools[0]), _ids("dst", dst, pools[0])
    ops.block_copy(pools, src, dst, block_table, remap)
