"""Blocks shared between requests: forks, copies on write, and compaction (host side).

The reference's allocator gives every request its own blocks for its whole life. Sampling several
continuations of one prompt, or reusing a cached prefix, wants the prompt's pages once:
:class:`SharedBlockManager` counts a block's holders. Its plans are lists of block ids;
``serve.block_copy.copy_blocks`` carries them out on the device.
"""

from __future__ import annotations

from typing import Sequence

from serve.block_manager import BlockManager, _count

__all__ = ["SharedBlockManager"]


class SharedBlockManager(BlockManager):
    """:class:`BlockManager` whose blocks may have several holders.

    ``reserve`` gives blocks with one holder; ``free`` gives one hold back and returns a block to
    the free list with its last. Ids still come out smallest first.
    """

    def __init__(self, n_blocks: int, block_size: int) -> None:
        super().__init__(n_blocks, block_size)
        self._holders: dict[int, int] = {}

    def reserve(self, n: int) -> list[int] | None:
        ids = super().reserve(n)
        if ids:
            self._holders.update((i, 1) for i in ids)
        return ids

    def holders(self, block_id: int) -> int:
        """How many requests hold the block (0: free)."""
        return self._holders.get(block_id, 0)

    def _check_held(self, ids: Sequence[int]) -> list[int]:
        ids = list(ids)
        seen: set[int] = set()
        for i in ids:
            if isinstance(i, bool) or not isinstance(i, int):
                raise ValueError(f"block ids must be ints, got {i!r}")
            if i in seen:
                raise ValueError(f"duplicate block id {i} in one call")
            if i not in self._allocated:
                raise ValueError(f"block {i} is not allocated")
            seen.add(i)
        return ids

    def free(self, ids: Sequence[int]) -> None:
        """Give one hold of every id back; the whole call is validated before anything changes."""
        ids = self._check_held(ids)
        last = [i for i in ids if self._holders[i] == 1]
        for i in ids:
            self._holders[i] -= 1
        for i in last:
            del self._holders[i]
        super().free(last)

    def share(self, ids: Sequence[int]) -> None:
        """Take one more hold of every id (a cached prefix used by another request)."""
        for i in self._check_held(ids):
            self._holders[i] += 1

    def fork(self, table: Sequence[int], length: int) -> tuple[list[int], list[tuple[int, int]]] | None:
        """A continuation of the first ``length`` tokens of ``table``: its own block table of the
        same width and the ``(from, to)`` copies it needs before either writes on, and before the new
        table is forked, copied or compacted itself. Blocks that the ``length`` tokens fill are
        shared; the rest are reserved, and a partly filled last one is copied. ``None`` (nothing
        changed) when the free blocks do not suffice."""
        table = self._check_held(table)
        length = _count("length", length, allow_zero=True)
        if length > len(table) * self.block_size:
            raise ValueError(f"length {length} exceeds the table's {len(table) * self.block_size} tokens")
        full = length // self.block_size
        own = self.reserve(len(table) - full)
        if own is None:
            return None
        self.share(table[:full])
        copies = [(table[full], own[0])] if length % self.block_size else []
        return table[:full] + own, copies

    def make_writable(self, table: list[int], index: int) -> list[tuple[int, int]] | None:
        """Before a write into block ``table[index]``: when others hold it too, puts a block of its
        own in its place in ``table`` and returns the copy that fills it (``[]`` when it is already
        its own, ``None`` when no block is free). Carry the copy out before the block is forked or
        copied again."""
        if not 0 <= index < len(table):
            raise IndexError(f"index {index} outside a table of {len(table)} blocks")
        self._check_held([table[index]])
        old = table[index]
        if self._holders[old] == 1:
            return []
        new = self.reserve(1)
        if new is None:
            return None
        self._holders[old] -= 1
        table[index] = new[0]
        return [(old, new[0])]

    def compact(self) -> tuple[list[int], list[int], list[int]]:
        """Moves the blocks in use down to ids ``0 .. in_use - 1``: ``(src, dst, remap)``. The highest
        go to the lowest holes, so as few as possible move, and no destination is a source.
        ``remap[id]`` is every block's id afterwards (its own where it stays, and for free ones).
        The manager's state is already the one after the move."""
        n = len(self._allocated)
        dst = [i for i in self._free if i < n]
        src = sorted((i for i in self._allocated if i >= n), reverse=True)
        remap = list(range(self.n_blocks))
        for a, b in zip(src, dst):
            remap[a] = b
            self._holders[b] = self._holders.pop(a)
        self._allocated = set(range(n))
        self._free = list(range(n, self.n_blocks))
        return src, dst, remap
