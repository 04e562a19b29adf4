"""The cache of bounded length on a host without a GPU: what its C entries refuse before any CUDA call, what its
Python functions refuse, and the host side of its containers."""

from __future__ import annotations

import ctypes

import pytest
import torch

from bounded_reference import evict_reference, window_mask
from model import _native
from model.triton_decode import _raise_first, window_rules

INVALID, UNSUPPORTED = _native.PD_ERR_INVALID, _native.PD_ERR_UNSUPPORTED
S3 = (ctypes.c_int64 * 3)(2048, 128, 64)


def _decode(**over):
    a = dict(n_blocks=8, bs=16, st=S3, bt=4, blocks=4, window=5, sinks=2, batch=1, h=4, hkv=2, d=64, dtype=_native.PD_BF16)
    a.update(over)
    return _native.lib.pd_decode_window(None, 0, 0, None, None, a["n_blocks"], a["bs"], a["st"], a["st"], None, a["bt"],
                                        a["blocks"], None, a["window"], a["sinks"], None, 0, 0, a["batch"], a["h"], a["hkv"],
                                        a["d"], a["dtype"], 1.0, None, 0, None)


@pytest.mark.parametrize("over,status", [
    (dict(window=0), INVALID), (dict(window=-3), INVALID), (dict(sinks=-1), INVALID), (dict(bs=12), INVALID), (dict(d=96), INVALID),
    (dict(d=512), UNSUPPORTED), (dict(h=3), INVALID), (dict(dtype=9), INVALID), (dict(batch=-1), INVALID),
    (dict(n_blocks=0), INVALID), (dict(st=None), INVALID), (dict(d=8, bs=4), UNSUPPORTED)])
def test_decode_window_refuses(over, status):
    assert _decode(**over) == status


def _prefill(**over):
    a = dict(total=10, n_blocks=8, bs=16, st=S3, bt=4, blocks=4, window=5, sinks=2, batch=1, longest=5, h=4, hkv=2, d=64,
             dtype=_native.PD_BF16)
    a.update(over)
    return _native.lib.pd_prefill_window(None, a["total"], 0, 0, None, None, a["n_blocks"], a["bs"], a["st"], a["st"], None,
                                         a["bt"], a["blocks"], None, None, a["window"], a["sinks"], None, 0, 0, a["batch"],
                                         a["longest"], a["h"], a["hkv"], a["d"], a["dtype"], 1.0, None)


@pytest.mark.parametrize("over,status", [
    (dict(window=0), INVALID), (dict(sinks=-1), INVALID), (dict(bs=12), INVALID), (dict(bs=4), UNSUPPORTED),
    (dict(d=32), UNSUPPORTED), (dict(dtype=_native.PD_F32), UNSUPPORTED), (dict(h=3), INVALID), (dict(total=-1), INVALID),
    (dict(longest=-1), INVALID), (dict(bt=3), INVALID), (dict(st=None), INVALID), (dict(total=1 << 30), UNSUPPORTED),
    (dict(), INVALID), (dict(batch=0), _native.PD_OK), (dict(total=0), _native.PD_OK), (dict(longest=0), _native.PD_OK)])
def test_prefill_window_refuses(over, status):
    assert _prefill(**over) == status


def _evict(**over):
    a = dict(layers=1, n_blocks=8, bs=16, hkv=2, d=64, dtype=_native.PD_BF16, blocks=4, bt=4, wlen=64, batch=1, keep=8, recent=2,
             sinks=1, fresh=None, new_blocks=0, ks=None)
    a.update(over)
    return _native.lib.pd_evict(a["ks"], None, a["layers"], a["n_blocks"], a["bs"], a["hkv"], a["d"], a["dtype"], S3, S3, None,
                                a["bt"], a["blocks"], a["fresh"], 0, a["new_blocks"], None, None, None, S3, None, S3, a["wlen"],
                                a["batch"], a["keep"], a["recent"], a["sinks"], None, 0, None)


@pytest.mark.parametrize("over,status", [
    (dict(keep=0), INVALID), (dict(recent=-1), INVALID), (dict(recent=5, sinks=4), INVALID), (dict(wlen=63), INVALID),
    (dict(bs=12), INVALID), (dict(bt=3), INVALID), (dict(dtype=7), INVALID), (dict(d=4), UNSUPPORTED), (dict(layers=-1), INVALID),
    (dict(n_blocks=0), INVALID), (dict(), INVALID), (dict(layers=0), _native.PD_OK), (dict(batch=0), _native.PD_OK),
    (dict(recent=0x7fffffff, sinks=0x7fffffff, keep=0x7fffffff), INVALID)])
def test_evict_refuses(over, status):
    assert _evict(**over) == status


def test_evict_refuses_a_pool_named_twice():
    at = 1 << 20  # any aligned address: it is refused before anything is read
    pools = [(ctypes.c_void_p * 2)(at, at + (1 << 16)), (ctypes.c_void_p * 2)(at + (2 << 16), at)]
    table = ctypes.c_void_p(at)
    status = _native.lib.pd_evict(pools[0], pools[1], 2, 8, 16, 2, 64, _native.PD_BF16, S3, S3, table, 4, 4, None, 0, 0, table,
                                  table, table, S3, table, S3, 64, 1, 8, 2, 1, table, 1 << 20, None)
    assert status == INVALID and b"named twice" in _native.lib.pd_last_error_string()


def test_weights_refuse():
    f = _native.lib.pd_decode_weights
    args = lambda wlen, hkv=2: (None, 0, 0, None, None, 8, 16, S3, S3, None, 4, 4, None, None, 0, 0, wlen, None, 0, 0, 1, 2 * hkv,  # noqa: E731
                                hkv, 64, _native.PD_BF16, 1.0, None, 0, None, 0, None)
    assert f(*args(63)) == INVALID  # shorter than the table
    assert f(*args(64)) == INVALID  # no weights
    assert f(*args(64, 65536)) == UNSUPPORTED


def test_functions_need_cuda():
    pytest.importorskip("torch")
    if _native.ops is None:
        pytest.skip("the operators' binding is not built here")
    from model.paged_evict import evict_tokens, paged_decode_weights
    from model.paged_window import paged_decode_window, paged_prefill_window

    pool, q = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    w = torch.zeros(1, 1, 2, 32)
    for call in (lambda: paged_decode_window(q, pool, pool, table, lens, 8),
                 lambda: paged_prefill_window(q, pool, pool, table, torch.tensor([0, 1]), lens, 1, 8),
                 lambda: paged_decode_weights(q, pool, pool, table, lens, w[0]),
                 lambda: evict_tokens([pool], [pool], table, lens, w, 4)):
        with pytest.raises(RuntimeError, match="requires CUDA"):
            call()
    with pytest.raises(TypeError):
        paged_decode_window(None, pool, pool, table, lens, 8)


def test_window_rules():
    for window, sinks in ((None, 0), (1, 0), (7, 3), (1 << 50, 1 << 50)):
        _raise_first(window_rules(window, sinks))
    for window, sinks in ((0, 0), (-1, 0), (3, -1), (None, 1), (2.0, 0), (True, 0), (3, None), (3, "1")):
        with pytest.raises(ValueError):
            _raise_first(window_rules(window, sinks))


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (16, 16), (100, 33)])
def test_the_references_agree_with_the_definition(window, sinks):
    n = 90
    mask = window_mask(0, n, n, window, sinks, "cpu")
    for i in range(n):
        for j in range(n):
            assert bool(mask[i, j]) == (j <= i and (i - j < window or j < sinks))


def test_the_eviction_reference():
    w = torch.tensor([[[[5.0, 1.0, 3.0, 3.0, float("nan"), 3.0, 0.0, 9.0]]]])
    assert evict_reference(w, [8], 4, 1, 1)[0, 0, 0] == [0, 2, 3, 7]
    assert evict_reference(w, [8], 7, 0, 0)[0, 0, 0] == [0, 1, 2, 3, 5, 6, 7]
    assert evict_reference(w, [3], 4, 1, 1)[0, 0, 0] == [0, 1, 2]
