"""The announced longest chunk of a 4-bit prefill is a bound: a loose one changes neither the kernel that
runs nor the result."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fp4_reference as ref
from model import _native

PTR = ctypes.c_void_p(256)  # never dereferenced: the calls on the CPU are refused before a launch


def _prefill(total_q, heads, longest=4, hkv=2, d=128):
    return _native.lib.pd_fp4_prefill(PTR, total_q, 1024, 128, PTR, 4, 16, None, PTR, 4, 4, PTR, PTR, PTR, 1024, 128, 2,
                                      longest, heads, hkv, d, _native.PD_BF16, 1.0, PTR, 0, None)


def test_more_query_rows_than_32_bits_index_are_refused():
    assert _prefill(1 << 30, 4) == _native.PD_ERR_UNSUPPORTED
    assert _prefill((1 << 28) + 1, 4) == _native.PD_ERR_UNSUPPORTED
    assert _prefill(0x7fffffff, 2) == _native.PD_ERR_UNSUPPORTED
    assert _prefill(1 << 28, 4) != _native.PD_ERR_UNSUPPORTED


def _case(device, rows, heads, hkv, d):
    g = torch.Generator().manual_seed(0)
    chunks, lengths = [c for c, _ in rows], [n for _, n in rows]
    need = [-(-n // 16) for n in lengths]
    pages = torch.randint(0, 256, (sum(need), hkv, 1, 18 * d), generator=g, dtype=torch.uint8)
    _, ks, _, vs = ref.places(d)
    for at in (ks, vs):
        pages[..., at.flatten()] = torch.randint(0x20, 0x34, (sum(need), hkv, 1, at.numel()), generator=g, dtype=torch.uint8)
    table = torch.zeros(len(rows), max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(n) + sum(need[:b])
    q = torch.randn(sum(chunks), heads, d, generator=g).to(torch.bfloat16)
    cu = torch.tensor([sum(chunks[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
    return [t.to(device) for t in (q, pages, table, cu, torch.tensor(lengths, dtype=torch.int32))]


@pytest.mark.gpu
def test_a_loose_bound_runs_the_same_kernel(cuda_device):
    from model.paged_fp4 import paged_prefill_fp4

    assert _native.get_fp4_prefill_mode() == 0
    args = _case(cuda_device, [(1024, 2048)], 16, 8, 128)
    tight = paged_prefill_fp4(*args, 1024)
    for loose in (1025, 16384, 0x7fffffff):
        assert torch.equal(paged_prefill_fp4(*args, loose), tight), loose


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("heads,hkv,d", [(8, 1, 128), (16, 8, 64), (2, 2, 256)])
def test_the_largest_bound_on_each_kernel(cuda_device, mode, heads, hkv, d):
    """2^31 - 1 tokens announced: rows times heads would pass 32 bits."""
    from model.paged_fp4 import paged_prefill_fp4

    args = _case(cuda_device, [(70, 200), (0, 33), (5, 5)], heads, hkv, d)
    try:
        _native.set_fp4_prefill_mode(mode)
        assert torch.equal(paged_prefill_fp4(*args, 0x7fffffff), paged_prefill_fp4(*args, 70))
    finally:
        _native.set_fp4_prefill_mode(0)
