"""Compaction of a 16-bit pool: blocks moved, containers built anew over the renumbered tables."""

from __future__ import annotations

import pytest
import torch

from model.paged import PagedKV, PagedPool
from serve.block_copy import copy_blocks
from serve.block_sharing import SharedBlockManager

pytestmark = pytest.mark.gpu


def test_a_paged_pool_is_compacted_between_containers(cuda_device):
    g = torch.Generator().manual_seed(0)
    pool = PagedPool(2, 40, 16, 2, 64, dtype=torch.bfloat16, device=cuda_device, n_head=4)
    for t in pool.block_tensors():
        t.copy_(torch.randn(t.shape, generator=g).to(torch.bfloat16))
    m = SharedBlockManager(40, 16)
    tables = [m.reserve(n) for n in (5, 9, 3, 8, 6)]
    m.free(tables[0])
    m.free(tables[2])
    tables, lengths = [tables[i] for i in (1, 3, 4)], [130, 100, 80]
    q, k, v = (torch.randn(3, h, 1, 64, generator=g).to(torch.bfloat16).to(cuda_device) for h in (4, 2, 2))

    def step(tables):
        kv = PagedKV(pool, tables, lengths, rope_len=200, n_head=4)
        kv.build_mask(next_token=True)
        out = []
        for layer in range(2):
            kv.write(layer, k, v)
            out.append(kv.attend(layer, q).clone())
        return kv, torch.stack(out)

    kv, before = step(tables)
    src, dst, remap = m.compact()
    assert src and m.in_use == 23
    with pytest.raises(RuntimeError, match="build a new container"):
        kv.move_blocks(src, dst, remap)
    copy_blocks(pool, src, dst)
    assert torch.equal(step([[remap[i] for i in t] for t in tables])[1], before)
