"""Blocks too small for the decode kernel's copies are refused: a tile takes its boxes (one block of one
head each) side by side in shared memory, where a TMA copy has to start on 128 bytes."""

from __future__ import annotations

import ctypes

import pytest
import torch

from model import _native
from model.triton_decode import _contract, _raise_first

SMALL = [(8, 4, torch.bfloat16), (8, 1, torch.float16), (16, 2, torch.bfloat16), (32, 1, torch.float16), (8, 2, torch.float32),
         (16, 1, torch.float32)]
ENOUGH = [(8, 8, torch.bfloat16), (16, 4, torch.float16), (32, 2, torch.bfloat16), (64, 1, torch.float16), (8, 4, torch.float32),
          (32, 1, torch.float32)]


def _args(d, bs, dtype):
    pool = torch.zeros(4, bs, 2, d, dtype=dtype)
    return torch.zeros(1, 4, d, dtype=dtype), pool, pool, torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)


@pytest.mark.parametrize("d,bs,dtype", SMALL)
def test_refused(d, bs, dtype):
    with pytest.raises(ValueError, match="multiple of 128 bytes"):
        _raise_first(_contract(*_args(d, bs, dtype)))
    s3 = (ctypes.c_int64 * 3)(bs * 2 * d, 2 * d, d)
    status = _native.lib.pd_decode(None, 0, 0, None, None, 4, bs, s3, s3, None, 2, 2, None, None, 0, 0, 1, 4, 2, d,
                                   _native.dtype_code(dtype), 1.0, None, 0, None)
    assert status == _native.PD_ERR_UNSUPPORTED


@pytest.mark.parametrize("d,bs,dtype", ENOUGH)
def test_taken(d, bs, dtype):
    _raise_first(_contract(*_args(d, bs, dtype)))
