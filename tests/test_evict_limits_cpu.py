"""``pd_evict``'s refusals beyond those of its Python binding, before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest

from model import _native

S3 = (ctypes.c_int64 * 3)(1 << 20, 1 << 16, 1 << 12)
F32, F16, BF16 = _native.PD_F32, _native.PD_F16, _native.PD_BF16


def _evict(d, dtype, layers=1, batch=1, table=1 << 20, stride=4, new=None, new_stride=0, new_blocks=0):
    """Every other argument but the scratch is one that the call takes; no address of it is one."""
    at = 1 << 20
    pools = [(ctypes.c_void_p * 1)(at + (i << 30)) for i in range(2)]
    here = ctypes.c_void_p(at)
    return _native.lib.pd_evict(pools[0], pools[1], layers, 8, 16, 2, d, dtype, S3, S3, ctypes.c_void_p(table), stride, 4,
                                new, new_stride, new_blocks, here, here, here, S3, here, S3, 64, batch, 8, 2, 1, None, 0, None)


@pytest.mark.parametrize("d,dtype", [(1028, F32), (1032, F32), (2048, F32), (2056, F16), (2056, BF16), (4096, BF16),
                                     *((d, t) for d in (1 << 20, 0x40000000, 0x7ffffff0) for t in (F32, F16, BF16))])
def test_rows_wider_than_the_move(d, dtype):
    """The move gives every 16-byte unit of a row a thread of its CTA: 4096 bytes."""
    assert _evict(d, dtype) == _native.PD_ERR_UNSUPPORTED
    assert _evict(d, dtype, layers=0) == _native.PD_ERR_UNSUPPORTED


@pytest.mark.parametrize("d,dtype", [(256, F32), (1024, F32), (2048, F16), (2048, BF16), (24, BF16)])
def test_rows_that_it_takes(d, dtype):
    assert _evict(d, dtype) == _native.PD_ERR_WORKSPACE  # taken but for the scratch
    assert _evict(d, dtype, batch=0) == _native.PD_OK


@pytest.mark.parametrize("batch,new,stride,new_stride,new_blocks", [
    (1, 0, 4, 4, 4), (3, 0, 4, 4, 4), (3, 0, 9, 9, 9), (3, 3, 9, 9, 4), (3, -8, 9, 9, 9), (5, 0, 4, 8, 4), (5, 4, 9, 8, 4),
    (5, -11, 8, 9, 8)])
def test_a_rows_own_pages_as_its_new_ones(batch, new, stride, new_stride, new_blocks):
    """New pages are filled by several CTAs in no order: block_table itself, whole or in part, as new_table is refused."""
    at = 1 << 20
    status = _evict(64, BF16, batch=batch, table=at, stride=stride, new=at + 4 * new, new_stride=new_stride, new_blocks=new_blocks)
    assert status == _native.PD_ERR_INVALID and b"own block_table" in _native.lib.pd_last_error_string()


@pytest.mark.parametrize("batch,new,stride,new_stride,new_blocks", [
    (1, 4, 4, 4, 4), (3, 4, 8, 8, 4), (3, -4, 8, 8, 4), (3, 12, 4, 4, 4), (5, 20, 4, 8, 4), (5, 4, 9, 9, 4)])
def test_two_tables_in_one_tensor(batch, new, stride, new_stride, new_blocks):
    at = 1 << 20
    assert _evict(64, BF16, batch=batch, table=at, stride=stride, new=at + 4 * new, new_stride=new_stride,
                  new_blocks=new_blocks) == _native.PD_ERR_WORKSPACE  # taken but for the scratch
