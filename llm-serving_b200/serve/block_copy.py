"""Pages copied between blocks of a pool, in every layer, in one launch.

What block sharing (``serve.block_sharing``) needs of the device: a fork copies its last, partly
filled page; a write to a shared page first copies it; a compaction moves pages down and renumbers
the block tables. The reference's pools are never rearranged, so there is no counterpart there.
"""

from __future__ import annotations

import torch

from model import _native
from model.triton_decode import _require_backend

__all__ = ["copy_blocks"]


def _ids(name: str, ids, device, n_blocks: int) -> torch.Tensor:
    if isinstance(ids, torch.Tensor):
        if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be a 1-D int32 or int64 tensor, got {tuple(ids.shape)} {ids.dtype}")
        if ids.device != device:
            raise ValueError(f"{name} is on {ids.device} but the pools are on {device}")
        return ids.contiguous()
    ids = list(ids)
    for i in ids:
        if isinstance(i, bool) or not isinstance(i, int):
            raise ValueError(f"{name} must hold ints, got {i!r}")
        if not 0 <= i < n_blocks:
            raise IndexError(f"{name}: block id {i} outside the pool's {n_blocks} blocks")
    if name == "dst" and len(set(ids)) != len(ids):
        raise ValueError("dst holds a block id twice")
    return torch.tensor(ids, dtype=torch.int64, device=device)


def _tensors(pools) -> list[torch.Tensor]:
    if hasattr(pools, "block_tensors"):
        return pools.block_tensors()
    return [pools] if isinstance(pools, torch.Tensor) else list(pools)


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
    _require_backend()
    tensors = _tensors(pools)
    if not tensors:
        raise ValueError("copy_blocks needs at least one pool")
    first = tensors[0]
    shape, dtype, device = first.shape, first.dtype, first.device
    if not first.is_cuda:
        raise RuntimeError(f"copy_blocks requires CUDA pools, got {device}; there is no CPU path.")
    if first.dim() < 2 or first.numel() == 0:
        raise ValueError(f"a pool needs (n_blocks, ...) elements, got {tuple(shape)}")
    for t in tensors:
        if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
            raise ValueError(f"every pool must be a contiguous {tuple(shape)} {dtype} tensor on {device}")
    n_blocks = shape[0]
    src, dst = _ids("src", src, device, n_blocks), _ids("dst", dst, device, n_blocks)
    if src.shape != dst.shape:
        raise ValueError(f"src has {src.numel()} blocks and dst {dst.numel()}")
    if src.dtype != dst.dtype:
        src, dst = src.long(), dst.long()
    if (block_table is None) != (remap is None):
        raise ValueError("block_table and remap go together")
    if block_table is not None:
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != device:
            raise ValueError(f"block_table must be an int32 (B, max_blocks) tensor on {device}")
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("block_table needs a unit column stride (it is renumbered in place)")
        if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
            raise ValueError("block_table rows must not overlap (it is renumbered in place)")
        if remap.dtype != torch.int32 or tuple(remap.shape) != (n_blocks,) or remap.device != device:
            raise ValueError(f"remap must be an int32 ({n_blocks},) tensor on {device}")
        remap = remap.contiguous()
    with _native.device_guard(device):
        _native.block_copy(tensors, src, dst, block_table, remap)
