"""``pd_prefill_window`` refuses what no launch holds before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest

from model import _native

S3 = (ctypes.c_int64 * 3)(2048, 128, 64)


def _prefill(batch, longest, heads, hkv, total):
    here = ctypes.c_void_p(1 << 20)
    return _native.lib.pd_prefill_window(here, total, heads * 64, 64, here, here, 8, 16, S3, S3, here, 4, 4, here, here, 5, 2, here,
                                         heads * 64, 64, batch, longest, heads, hkv, 64, _native.PD_BF16, 1.0, None)


@pytest.mark.parametrize("batch,longest,heads,hkv,total", [
    (1 << 18, 1 << 18, 16, 8, 1 << 18), (0x7fffffff, 129, 1, 1, 1 << 20), (1 << 20, 1 << 20, 512, 512, 1 << 20),
    (0x40000000, 1, 2, 2, 1 << 20)])
def test_more_ctas_than_a_launch(batch, longest, heads, hkv, total):
    assert _prefill(batch, longest, heads, hkv, total) == _native.PD_ERR_UNSUPPORTED
    assert b"tighter bound" in _native.lib.pd_last_error_string()
