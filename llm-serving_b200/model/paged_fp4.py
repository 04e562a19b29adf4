"""A paged KV cache held in 4 bits: write, read back, decode and chunked prefill over its pages.

The same protocol as :mod:`model.paged` with pools a quarter to a third of the size: an element is
an e2m1 code (0 .5 1 1.5 2 3 4 6 and a sign), 16 neighbours share one e4m3 scale, 4.5 bits in all,
and a power-of-two unit per (K or V, head) places a head's range. A layer's pool is one uint8 tensor
``(n_blocks, n_kv_head, block_size / 16, 18 * head_dim)``; the record layout is in
``include/paged_decode.h``. The reference has no quantised cache to mirror.

Functions (tensors on CUDA, the current stream, no host synchronisation):

* :func:`fp4_pages` -- an empty pool tensor;
* :func:`write_slots_fp4` / :func:`read_slots_fp4` -- tokens into and out of flat slots;
* :func:`paged_decode_fp4` -- one query token per row (``paged_decode``'s contract);
* :func:`paged_prefill_fp4` -- a causal chunk per row (``paged_prefill``'s contract).

Containers: :class:`Fp4Pool` (``PagedPool``) and :class:`Fp4KV` (``PagedKV``), which the serving
loop and ``serve.graph`` drive unchanged.

Contract: fp16 or bf16 queries; head_dim 64, 128 or 256; block_size a power of two >= 16; any number
of query heads per kv head. Rows of length 0 give zeros; lengths are clamped to the table's
capacity on the device (``seqlen`` is never read on the host); a block id outside the pool reads
zeros. There is no CPU path and no fallback.
"""

from __future__ import annotations

import math

import torch

from model import _native
from model.paged import PagedKV, PagedPool, _positive
from model.triton_decode import _pow2, _raise_first
from serve.block_copy import copy_blocks

__all__ = ["Fp4KV", "Fp4Pool", "fp4_pages", "fp4_workspace", "paged_decode_fp4", "paged_prefill_fp4", "read_slots_fp4",
           "write_slots_fp4"]

_HEAD_DIMS = (64, 128, 256)
_QUERY_DTYPES = (torch.float16, torch.bfloat16)


def _pool_rules(block_size, head_dim):
    yield not _pow2(block_size) or block_size < 16, lambda: (
        f"block_size must be a power of two of at least 16, got {block_size}")
    yield head_dim not in _HEAD_DIMS, lambda: f"head_dim must be 64, 128 or 256 for 4-bit pages, got {head_dim}"


def fp4_pages(n_blocks: int, block_size: int, n_kv_head: int, head_dim: int, *, device="cuda") -> torch.Tensor:
    """A zeroed pool tensor of 4-bit pages (every element stands for 0)."""
    for name, value in (("n_blocks", n_blocks), ("block_size", block_size), ("n_kv_head", n_kv_head),
                        ("head_dim", head_dim)):
        _positive(name, value)
    _raise_first(_pool_rules(block_size, head_dim))
    return torch.zeros(n_blocks, n_kv_head, block_size // 16, 18 * head_dim, dtype=torch.uint8, device=device)


def fp4_workspace(like: torch.Tensor) -> torch.Tensor:
    """A workspace of its own for attention calls that may run beside others, on ``like``'s device:
    zero-filled once, and left at zero by every call."""
    return _native.require_ops().fp4_workspace(like)


def write_slots_fp4(pages, slot_ids, k, v, *, units=None) -> None:
    """Quantise token ``i`` of k/v ``(n, H_kv, D)`` (fp32, fp16 or bf16) into flat slot ``slot_ids[i]``
    (``block * block_size + offset``) of ``pages``, one launch.

    Slots must be distinct; one outside the pool is skipped and sets
    ``_native.DEVERR_APPEND_RANGE`` in the device error word. ``units`` float32 ``(2, H_kv)`` holds
    the powers of two that K's and V's elements are counted in (``None``: 1). Values beyond
    ``6 * 448`` units saturate and NaN counts as zero.
    """
    (_native.ops or _native.require_ops()).fp4_write_slots(pages, slot_ids, k, v, units)


def read_slots_fp4(pages, slot_ids, dtype=torch.bfloat16, *, units=None):
    """``(k, v)``, each ``(n, H_kv, D)`` in ``dtype``: the values that flat slots ``slot_ids`` hold, one
    launch. A slot outside the pool reads zeros and sets ``_native.DEVERR_APPEND_RANGE``."""
    return (_native.ops or _native.require_ops()).fp4_read_slots(pages, slot_ids, dtype, units)


def paged_decode_fp4(q, pages, block_table, seqlen, *, units=None, scale: float | None = None, out=None,
                     workspace=None):
    """Decode one query token per row against 4-bit pages (one kernel launch for every 896 rows).

    ``q`` ``(B, H, D)`` fp16 or bf16; ``block_table`` int32 ``(B, max_blocks)``, of whose row ``b`` only
    the first ``ceil(seqlen[b] / block_size)`` entries matter; ``seqlen`` ``(B,)`` int32 (int64 is
    cast). Returns ``(B, H, D)`` in ``q.dtype``. ``workspace`` (optional) is a tensor of
    :func:`fp4_workspace` that no concurrent launch uses; without it the eager calls of one stream
    share one, and those of a graph's capture another that is the graph's own.
    """
    ops = _native.ops or _native.require_ops()
    return ops.fp4_decode(q, pages, block_table, seqlen, units, scale, out, workspace)


def paged_prefill_fp4(q, pages, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q: int, *, units=None,
                      scale: float | None = None, out=None, workspace=None):
    """Causal attention of a chunk of query tokens per row over 4-bit pages (one kernel launch for every
    896 rows).

    ``paged_prefill``'s contract: ``q`` is the packed ``(total_q, H, D)``, row ``b`` owning
    ``q[cu_seqlens_q[b]:cu_seqlens_q[b + 1]]``; the chunk's K/V are already in the pages, and its token
    ``i`` of ``Sq`` sees keys ``0 .. seqlen_k[b] - Sq + i``. ``max_seqlen_q`` must be at least the longest
    chunk (a loose bound costs nothing); tokens of a longer one past it are left unwritten. ``workspace``
    as in :func:`paged_decode_fp4`.
    """
    ops = _native.ops or _native.require_ops()
    return ops.fp4_prefill(q, pages, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q, units, scale, out, workspace)


class Fp4Pool(PagedPool):
    """Physical KV blocks in 4 bits: one :func:`fp4_pages` tensor per layer, in :attr:`pages`.

    ``dtype`` is the type of the activations that are written and attend (fp16 or bf16). ``k_unit`` /
    ``v_unit`` are the powers of two that elements are counted in, one number or
    ``(n_layer, n_kv_head)`` nested lists: about the size of a head's typical absolute value.
    A group's scale is at least ``2**-9`` and at most 448 units per code step, so values from about
    ``0.01`` to ``2688`` units keep their accuracy.
    """

    def __init__(self, n_layer: int, n_blocks: int, block_size: int, n_kv_head: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cpu", n_head: int | None = None, k_unit=1.0,
                 v_unit=1.0):
        self.n_layer = _positive("n_layer", n_layer)
        self.n_blocks = _positive("n_blocks", n_blocks)
        self.block_size = _positive("block_size", block_size)
        self.n_kv_head = _positive("n_kv_head", n_kv_head)
        self.head_dim = _positive("head_dim", head_dim)
        _raise_first(_pool_rules(block_size, head_dim))
        n_head = self.n_kv_head if n_head is None else int(n_head)
        if n_head % self.n_kv_head != 0:
            raise ValueError(f"n_head ({n_head}) must be a multiple of n_kv_head ({self.n_kv_head})")
        if dtype not in _QUERY_DTYPES:
            raise ValueError(f"Fp4Pool dtype must be fp16 or bf16, got {dtype}")
        self.n_head = n_head
        self.n_group = n_head // self.n_kv_head
        self.dtype = dtype
        self.device = torch.device(device)
        self.pages = [fp4_pages(n_blocks, block_size, n_kv_head, head_dim, device=self.device)
                      for _ in range(self.n_layer)]
        units = torch.empty(self.n_layer, 2, self.n_kv_head)
        for i, (name, unit) in enumerate((("k_unit", k_unit), ("v_unit", v_unit))):
            unit = torch.as_tensor(unit, dtype=torch.float32)
            if unit.dim() and tuple(unit.shape) != (self.n_layer, self.n_kv_head):
                raise ValueError(f"{name} must be a number or ({self.n_layer}, {self.n_kv_head}), got {tuple(unit.shape)}")
            if not bool(((unit >= 2.0 ** -60) & (unit <= 2.0 ** 60) & (torch.frexp(unit)[0] == 0.5)).all()):
                raise ValueError(f"{name} must hold powers of two between 2**-60 and 2**60")
            units[:, i] = unit
        #: (n_layer, 2, n_kv_head) float32: the units of K and V.
        self.units = units.to(self.device)
        self._pending = None
        self._prefill_key: tuple | None = None
        self._prefill_slots: torch.Tensor | None = None

    @property
    def keys(self):
        raise AttributeError("a 4-bit pool has no K tensors: use pages, or read_slots for values")

    @property
    def values(self):
        raise AttributeError("a 4-bit pool has no V tensors: use pages, or read_slots for values")

    def block_tensors(self) -> list[torch.Tensor]:
        """Every tensor that holds blocks of the pool."""
        return list(self.pages)

    def write_slots(self, layer: int, slot_ids: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantise token ``i`` of k/v ``(n, n_kv_head, head_dim)`` into flat slot ``slot_ids[i]``."""
        layer = self._check_layer(layer)
        self._check_rows("write_slots", k, v)
        self._require_cuda("write_slots")
        write_slots_fp4(self.pages[layer], slot_ids, k, v.to(k.dtype), units=self.units[layer])

    def read_slots(self, layer: int, slot_ids: torch.Tensor, dtype: torch.dtype | None = None):
        """``(k, v)`` values of flat slots, in ``dtype`` (default: the pool's)."""
        layer = self._check_layer(layer)
        self._require_cuda("read_slots")
        return read_slots_fp4(self.pages[layer], slot_ids, self.dtype if dtype is None else dtype,
                              units=self.units[layer])

    def prefill(self, layer: int, q, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q: int, *, scale=None,
                workspace=None):
        """:func:`paged_prefill_fp4` over one layer's pages."""
        layer = self._check_layer(layer)
        return paged_prefill_fp4(q, self.pages[layer], block_table, cu_seqlens_q, seqlen_k, max_seqlen_q,
                                 units=self.units[layer], scale=scale, workspace=workspace)

    def bytes(self) -> int:
        """Physical bytes of the pool: 9/16 of a byte per element of K and V."""
        return sum(t.numel() for t in self.pages)


class Fp4KV(PagedKV):
    """Decode-time container over an :class:`Fp4Pool`: ``PagedKV``'s step protocol, with the step's
    token quantised by ``write`` (one launch) and read by ``attend`` (one launch for every 896 rows).

    K comes rotated (``qk_norm_rope`` rotates q and k together); ``write(rope=...)`` is refused.
    """

    def __init__(self, pool: Fp4Pool, block_tables, lengths, *, rope_len: int, seats=None,
                 n_head: int | None = None, check_bounds: bool = True) -> None:
        if not isinstance(pool, Fp4Pool):
            raise TypeError(f"Fp4KV needs an Fp4Pool, got {type(pool).__name__}")
        super().__init__(pool, block_tables, lengths, rope_len=rope_len, seats=seats, n_head=n_head,
                         check_bounds=check_bounds, fuse_append=False)
        self._fp4_workspace = fp4_workspace(pool.pages[0])
        self._scale = 1.0 / math.sqrt(self.head_dim)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, *, rope=None) -> None:
        if rope is not None:
            raise ValueError("Fp4KV.write takes K already rotated (model.qk_norm.qk_norm_rope), not rope tables")
        super().write(layer, k, v)

    def _append_now(self, layer: int, k3: torch.Tensor, v3: torch.Tensor, rope=None) -> None:
        _native.require_ops().fp4_write_table(self.pool.pages[layer], self._block_table_tensor, self.pos, k3,
                                              v3.to(k3.dtype), self.pool.units[layer])

    def attend(self, layer: int, q: torch.Tensor, *, dropout_p: float = 0.0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """4-bit block-table decode for one layer; ``q`` is ``(B, H, 1, D)``, output the same."""
        expected = (self.batch, self.n_head, 1, self.head_dim)
        for violated, error, message in (
                (not self._seqlen_ready, RuntimeError, "Fp4KV.attend() before build_mask(): seqlen is stale"),
                (not self._step_written, RuntimeError, "Fp4KV.attend() before write(): this step has no token yet"),
                (bool(dropout_p), ValueError, "paged decode is inference-only; dropout_p must be 0"),
                (tuple(q.shape) != expected, ValueError, f"attend needs q {expected}, got {tuple(q.shape)}")):
            if violated:
                raise error(message)
        return self._decode(layer, q, out)

    def move_blocks(self, src, dst, remap) -> None:
        """Carry out a compaction plan (``SharedBlockManager.compact()``) on the pool and on this
        container's block table, in one launch; a captured step stays valid. Other holders of the
        pool's blocks renumber theirs by ``remap``."""
        if len(remap) != self.pool.n_blocks:
            raise ValueError(f"remap must have one entry per block ({self.pool.n_blocks}), got {len(remap)}")
        copy_blocks(self.pool, src, dst, block_table=self._block_table_tensor,
                    remap=torch.tensor(remap, dtype=torch.int32, device=self.device))
        self.block_tables = [[remap[i] for i in table] for table in self.block_tables]
        self._slot_cache = None

    def _decode(self, layer: int, q: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        layer = self.pool._check_layer(layer)
        out3 = None if out is None else out[:, :, 0, :]
        return paged_decode_fp4(q[:, :, 0, :], self.pool.pages[layer], self._block_table_tensor, self._seqlen,
                                units=self.pool.units[layer], scale=self._scale, out=out3,
                                workspace=self._fp4_workspace).unsqueeze(2)

    def prepare(self, q: torch.Tensor) -> None:
        """Load the decode kernel (one decode into a scratch output) before a capture."""
        expected = (self.batch, self.n_head, 1, self.head_dim)
        if tuple(q.shape) != expected:
            raise ValueError(f"prepare needs q {expected}, got {tuple(q.shape)}")
        self._decode(0, q)
