"""Chunks of the 4-bit prefill whose query tokens see no key, or only the last ones do: zeros there, whatever
the output's memory held before."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[1, 2], ids=["warps", "tiles"])
def kernel(request):
    from model import _native

    _native.set_fp4_prefill_mode(request.param)
    yield request.param
    _native.set_fp4_prefill_mode(0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,hkv,d", [(48, 4, 64), (8, 8, 64), (36, 4, 128), (16, 8, 128), (16, 2, 256), (5, 1, 256)])
def test_blocks_of_tokens_that_see_nothing(cuda_device, kernel, dtype, heads, hkv, d):
    from model.paged_fp4 import paged_prefill_fp4

    rows = [(300, 0), (300, 1), (257, 0), (1, 0), (120, 40), (300, 17), (0, 3), (64, 0)]
    g = torch.Generator().manual_seed(d)
    chunks, lengths = [c for c, _ in rows], [n for _, n in rows]
    pages = torch.randint(0, 256, (4, hkv, 1, 18 * d), generator=g, dtype=torch.uint8)
    _, ks, _, vs = ref.places(d)
    for at in (ks, vs):
        pages[..., at.flatten()] = torch.randint(0x20, 0x34, (4, hkv, 1, at.numel()), generator=g, dtype=torch.uint8)
    table = torch.arange(4, dtype=torch.int32).repeat(len(rows), 1)
    cu = torch.tensor([sum(chunks[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
    q = torch.randn(sum(chunks), heads, d, generator=g).to(dtype)
    seen = torch.cat([n - c + torch.arange(c) >= 0 for c, n in rows])
    dev = [t.to(cuda_device) for t in (q, pages, table, cu, torch.tensor(lengths, dtype=torch.int32))]
    first = None
    for _ in range(20):
        out = torch.full_like(dev[0], 7)
        paged_prefill_fp4(*dev, 300, out=out)
        assert (out[~seen.to(cuda_device)] == 0).all()
        first = out if first is None else first
        assert torch.equal(out, first)
    assert (first[seen.to(cuda_device)] != 0).any()
