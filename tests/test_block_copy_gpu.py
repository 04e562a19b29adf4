"""Page copies and table renumbering on a B200: bytes equal to the plain indexing."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,shape", [
    (torch.bfloat16, (12, 16, 2, 64)), (torch.uint8, (12, 2, 1, 18 * 128)), (torch.float32, (12, 7, 3, 5)),
    (torch.uint8, (12, 13)), (torch.float16, (12, 16, 8, 128)), (torch.uint8, (12, 40001)),
])
@pytest.mark.parametrize("n_pools", [1, 3, 130])
@pytest.mark.parametrize("ids", ["int32", "int64", "list"])
def test_copies_are_byte_exact(cuda_device, dtype, shape, n_pools, ids):
    from serve.block_copy import copy_blocks

    g = torch.Generator().manual_seed(0)
    es = torch.empty(0, dtype=dtype).element_size()
    n = torch.Size(shape).numel() * es
    pools = [torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8).view(dtype).view(shape) for _ in range(n_pools)]
    src, dst = [7, 0, 7, 11, 4], [1, 2, 3, 9, 10]  # one source twice
    want = [p.clone() for p in pools]
    for p in want:
        p[dst] = p[src]
    dev = [p.to(cuda_device) for p in pools]
    s, d = (src, dst) if ids == "list" else (torch.tensor(x, dtype=getattr(torch, ids), device=cuda_device) for x in (src, dst))
    copy_blocks(dev, s, d)
    for a, b in zip(dev, want):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


def test_unaligned_pools(cuda_device):
    from serve.block_copy import copy_blocks

    base = torch.arange(1 + 6 * 32, dtype=torch.uint8, device=cuda_device)
    pool = base[1:].view(6, 32)
    want = pool.clone()
    want[[0, 5]] = want[[3, 2]]
    copy_blocks([pool], [3, 2], [0, 5])
    assert torch.equal(pool, want) and base[0] == 0


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (3, 0)])
def test_tables_are_renumbered_in_the_same_call(cuda_device, rows, cols):
    from serve.block_copy import copy_blocks

    g = torch.Generator().manual_seed(1)
    n = 40
    pool = torch.randn(n, 16, 2, 64, generator=g).to(cuda_device)
    wide = torch.randint(-3, n + 4, (rows, cols + 3), generator=g, dtype=torch.int32).to(cuda_device)
    remap = torch.randperm(n, generator=g).to(torch.int32).to(cuda_device)
    table = wide[:, 1:cols + 1]
    inside = (table >= 0) & (table < n)
    want_wide = wide.clone()
    want_wide[:, 1:cols + 1] = torch.where(inside, remap[table.clamp(0, n - 1).long()], table)
    want = pool.clone()
    want[[1, 2]] = want[[30, 31]]
    copy_blocks(pool, [30, 31], [1, 2], block_table=table, remap=remap)
    assert torch.equal(wide, want_wide) and torch.equal(pool, want)
    copy_blocks(pool, [], [], block_table=table, remap=torch.arange(n, dtype=torch.int32, device=cuda_device))
    assert torch.equal(wide, want_wide) and torch.equal(pool, want)


def test_ids_outside_the_pool_are_skipped_and_flagged(cuda_device):
    from model import _native
    from serve.block_copy import copy_blocks

    pool = torch.arange(8, device=cuda_device)[:, None].expand(8, 100).contiguous()
    assert _native.device_error() == 0
    copy_blocks(pool, torch.tensor([5, 8, -1, 6], device=cuda_device), torch.tensor([0, 1, 2, 1 << 40], device=cuda_device))
    assert _native.device_error() == _native.DEVERR_COPY_RANGE
    assert pool[:, 0].tolist() == [5, 1, 2, 3, 4, 5, 6, 7]


def test_a_pool_object_moves_every_layer(cuda_device):
    from model.paged import PagedKV, PagedPool
    from model.paged_fp4 import Fp4Pool
    from serve.block_copy import copy_blocks

    pool = PagedPool(2, 4, 16, 2, 64, dtype=torch.bfloat16, device=cuda_device, n_head=4)
    kv = PagedKV(pool, [[2]], [0], rope_len=16, n_head=4)
    kv.build_mask(next_token=True)
    kv.write(0, torch.ones(1, 2, 1, 64, dtype=torch.bfloat16, device=cuda_device),
             torch.ones(1, 2, 1, 64, dtype=torch.bfloat16, device=cuda_device))  # recorded, not yet in the pool
    copy_blocks(pool, [2], [0])
    assert (pool.keys[0][0, 0] == 1).all() and (pool.values[0][0, 0] == 1).all() and (pool.keys[1][0] == 0).all()
    four = Fp4Pool(2, 4, 16, 2, 64, device=cuda_device, n_head=4)
    four.pages[1][3] = 9
    copy_blocks(four, [3], [1])
    assert (four.pages[1][1] == 9).all() and (four.pages[0] == 0).all()


def test_refusals(cuda_device):
    from serve.block_copy import copy_blocks

    pool = torch.zeros(4, 8, device=cuda_device)
    for args, kw, error, match in (
            (([], [0], [1]), {}, ValueError, "at least one pool"),
            ((pool, [0], [1, 2]), {}, ValueError, "src has"),
            ((pool, [4], [1]), {}, IndexError, "outside the pool"),
            ((pool, [0, 1], [2, 2]), {}, ValueError, "twice"),
            ((pool, [0.5], [1]), {}, ValueError, "ints"),
            ((pool.t(), [0], [1]), {}, ValueError, "contiguous"),
            (([pool, pool[:2]], [0], [1]), {}, ValueError, "every pool"),
            ((pool, torch.zeros(1, device=cuda_device), [1]), {}, ValueError, "int32 or int64"),
            ((pool, torch.zeros(1, dtype=torch.int32), [1]), {}, ValueError, "is on cpu"),
            ((pool, [0], [1]), dict(remap=torch.zeros(4, dtype=torch.int32, device=cuda_device)), ValueError, "go together"),
            ((pool, [0], [1]), dict(block_table=torch.zeros(1, 1, dtype=torch.int32, device=cuda_device),
                                    remap=torch.zeros(3, dtype=torch.int32, device=cuda_device)), ValueError, "remap must be"),
            ((pool, [0], [1]), dict(block_table=torch.zeros(1, 3, dtype=torch.int32, device=cuda_device).expand(2, 3),
                                    remap=torch.zeros(4, dtype=torch.int32, device=cuda_device)), ValueError, "overlap"),
            ((pool.cpu(), [0], [1]), {}, RuntimeError, "CUDA"),
    ):
        with pytest.raises(error, match=match):
            copy_blocks(*args, **kw)
