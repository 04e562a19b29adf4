"""Host side of shared blocks: holders, forks, copies on write, compaction."""

from __future__ import annotations

import random

import pytest

from serve.block_manager import BlockManager
from serve.block_sharing import SharedBlockManager


def test_without_sharing_it_is_the_block_manager():
    rng = random.Random(0)
    a, b = BlockManager(64, 16), SharedBlockManager(64, 16)
    live = []
    for _ in range(300):
        n = rng.randint(0, 9)
        x, y = a.reserve(n), b.reserve(n)
        assert x == y
        if x:
            live.append(x)
        if live and rng.random() < 0.5:
            ids = live.pop(rng.randrange(len(live)))
            a.free(ids)
            b.free(ids)
        assert a.stats() == b.stats()


def test_fork_shares_full_blocks_and_copies_the_partial_one():
    m = SharedBlockManager(10, 16)
    table = m.reserve(4)
    for length, shared, copies in ((0, 0, False), (16, 1, False), (40, 2, True), (64, 4, False)):
        new, plan = m.fork(table, length)
        assert new[:shared] == table[:shared] and not set(new[shared:]) & set(table) and len(new) == 4
        assert plan == ([(table[shared], new[shared])] if copies else [])
        assert all(m.holders(i) == 2 for i in table[:shared]) and all(m.holders(i) == 1 for i in table[shared:])
        m.free(new)
        assert all(m.holders(i) == 1 for i in table) and m.in_use == 4
    assert m.fork(table, 3) is not None  # 4 more
    before = m.stats()
    assert m.fork(table, 3) is None and m.stats() == before, "no room: nothing changes"
    with pytest.raises(ValueError, match="exceeds"):
        m.fork(table, 65)
    with pytest.raises(ValueError, match="not allocated"):
        m.fork([9], 1)


def test_free_gives_back_one_hold():
    m = SharedBlockManager(4, 16)
    a = m.reserve(2)
    m.share(a)
    m.free(a)
    assert m.in_use == 2 and m.stats()["free"] == 2
    m.free(a)
    assert m.in_use == 0 and m.holders(0) == 0
    for bad in ([0], [5], [True]):
        with pytest.raises(ValueError):
            m.free(bad)
    b = m.reserve(1)
    with pytest.raises(ValueError, match="duplicate"):
        m.free([b[0], b[0]])
    assert m.holders(b[0]) == 1


def test_make_writable_copies_a_shared_block_once():
    m = SharedBlockManager(4, 16)
    a = m.reserve(2)
    b, _ = m.fork(a, 32)
    assert b == a
    assert m.make_writable(b, 1) == [(a[1], 2)] and b == [a[0], 2] and m.holders(a[1]) == 1
    assert m.make_writable(b, 1) == [] and m.make_writable(a, 1) == []
    m.reserve(1)
    assert m.make_writable(b, 0) is None and b[0] == a[0] and m.holders(a[0]) == 2
    with pytest.raises(IndexError):
        m.make_writable(b, 2)


def test_compact_fills_the_holes_from_the_top():
    rng = random.Random(3)
    for _ in range(50):
        m = SharedBlockManager(40, 16)
        tables = [t for t in (m.reserve(rng.randint(1, 6)) for _ in range(9)) if t]
        for t in [t for t in tables if rng.random() < 0.5]:
            m.free(t)
            tables.remove(t)
        if tables:
            f = m.fork(tables[0], 16)
            if f:
                tables.append(f[0])
        held = {i: m.holders(i) for t in tables for i in t}
        n = m.in_use
        src, dst, remap = m.compact()
        assert len(src) == len(dst) == len(set(dst)) and not set(src) & set(dst)
        assert all(s >= n for s in src) and all(d < n for d in dst)
        assert sorted({remap[i] for i in held}) == list(range(n)) and m.in_use == n
        assert all(m.holders(remap[i]) == c for i, c in held.items())
        assert m.reserve(40 - n) == (list(range(n, 40)) or [])
        assert m.compact() == ([], [], list(range(40)))
