"""Plans of block copies joined into one call (host side)."""

from __future__ import annotations

import pytest
import torch

from serve.block_copy import copy_blocks
from serve.block_sharing import SharedBlockManager

POOL = torch.zeros(8, 4)  # ids are checked before the pool's device is


def test_a_fork_of_a_fork_cannot_be_copied_together_with_it():
    m = SharedBlockManager(8, 16)
    table = m.reserve(2)
    first, plan = m.fork(table, 20)
    _, second = m.fork(first, 20)
    assert plan[0][1] == second[0][0], "the first copy fills what the second reads"
    joined = plan + second
    with pytest.raises(ValueError, match="destination of one copy and the source of another"):
        copy_blocks(POOL, [a for a, _ in joined], [b for _, b in joined])


@pytest.mark.parametrize("src,dst", [([0, 1], [1, 2]), ([3, 5], [4, 3]), ([1, 2], [2, 1]), ([0, 2, 4], [1, 3, 0])])
def test_overlapping_ids_are_refused(src, dst):
    for make in (list, tuple, iter):
        with pytest.raises(ValueError, match="destination of one copy"):
            copy_blocks(POOL, make(src), make(dst))


@pytest.mark.parametrize("src,dst", [([0, 0, 1], [2, 3, 4]), ([], []), ([5], [5]), ([7, 6], [0, 1])])
def test_independent_ids_pass_the_check(src, dst):
    with pytest.raises(RuntimeError, match="CUDA"):  # the next check
        copy_blocks(POOL, src, dst)


def test_forks_of_one_table_may_be_joined():
    m = SharedBlockManager(16, 16)
    table, copies = m.reserve(3), []
    for _ in range(3):
        copies += m.fork(table, 20)[1]
    with pytest.raises(RuntimeError, match="CUDA"):
        copy_blocks(torch.zeros(16, 4), [a for a, _ in copies], [b for _, b in copies])
