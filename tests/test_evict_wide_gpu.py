"""``pd_evict`` over rows that its Python binding does not pass: up to 4096 bytes, and of an odd number of 16-byte units."""

from __future__ import annotations

import ctypes

import pytest
import torch

from bounded_reference import evict_reference, make_pools
from model import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("d,dtype", [(2048, torch.float16), (1024, torch.float32), (1032, torch.bfloat16), (24, torch.bfloat16),
                                     (20, torch.float32)])
def test_wide_rows(d, dtype, rows, fresh):
    hkv, bs, keep, recent, sinks = 2, 16, 30, 5, 2
    lens = [(37 * b) % 90 for b in range(rows)]
    k, v, table, free = make_pools(lens, hkv, d, bs, dtype, gen=torch.Generator().manual_seed(d), spare=2 * rows)
    old, width = (k.clone(), v.clone()), table.shape[1]
    w = torch.rand(1, rows, hkv, width * bs, generator=torch.Generator().manual_seed(1)).cuda()
    new = torch.cat([free[:2 * rows].view(rows, 2), torch.zeros(rows, width - 2, dtype=torch.int32, device="cuda")], 1)
    target = new if fresh else table
    seqlen, n = torch.tensor(lens, dtype=torch.int32).cuda(), torch.empty(rows, dtype=torch.int32, device="cuda")
    sums = torch.empty_like(w)
    size = _native.lib.pd_evict_scratch_bytes(1, rows, hkv, keep)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    pools = [(ctypes.c_void_p * 1)(x.data_ptr()) for x in (k, v)]
    strides = _native.strides3(k)
    w_strides = (ctypes.c_int64 * 3)(*w.stride()[:3])
    stream = torch.cuda.current_stream().cuda_stream
    status = _native.lib.pd_evict(
        *pools, 1, k.shape[0], bs, hkv, d, _native.dtype_code(dtype), strides, strides, table.data_ptr(), width, width,
        new.data_ptr() if fresh else None, width if fresh else 0, width if fresh else 0, seqlen.data_ptr(), n.data_ptr(),
        w.data_ptr(), w_strides, sums.data_ptr(), w_strides, width * bs, rows, keep, recent, sinks, scratch.data_ptr(), size, stream)
    assert status == _native.PD_OK
    assert n.tolist() == [min(x, keep) for x in lens]
    for got, x in zip((k, v), old):
        want = x.clone()
        for (_, b, h), tokens in evict_reference(w, lens, keep, recent, sinks).items():
            src, dst = torch.tensor(tokens, dtype=torch.long).cuda(), torch.arange(len(tokens)).cuda()
            want[target[b].long()[dst // bs], dst % bs, h] = x[table[b].long()[src // bs], src % bs, h]
        assert torch.equal(got, want)
    assert _native.device_error() == 0
