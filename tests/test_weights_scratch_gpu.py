"""``pd_decode_weights`` decides once whether its rows are few: with too little scratch it runs in one launch or not at all."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import check, make_pools, weights_reference
from model import _native

pytestmark = pytest.mark.gpu


def _call(lens, scratch_bytes, null=False):
    """(status, launches, out, sums, the case) of a call with that much scratch."""
    hkv, group, d, bs = 8, 2, 128, 16
    gen = torch.Generator().manual_seed(0)
    k, v, table, _ = make_pools(lens, hkv, d, bs, torch.bfloat16, gen=gen)
    q = torch.randn(len(lens), hkv * group, d, generator=gen).to(torch.bfloat16).cuda()
    seqlen = torch.tensor(lens, dtype=torch.int32).cuda()
    w = torch.zeros(len(lens), hkv, table.shape[1] * bs, device="cuda")
    out = torch.full_like(q, 7.0)
    lib, code = _native.lib, _native.dtype_code(q.dtype)
    ws = torch.empty(_native.workspace_bytes(len(lens), hkv * group, hkv, d, q.dtype, window=True), dtype=torch.uint8, device="cuda")
    need = lib.pd_decode_weights_scratch_bytes(len(lens), hkv * group, table.shape[1], bs)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    size = need if scratch_bytes is None else scratch_bytes
    before = _native.launch_count()
    status = lib.pd_decode_weights(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), k.shape[0], bs, _native.strides3(k), _native.strides3(v),
        table.data_ptr(), table.stride(0), table.shape[1], seqlen.data_ptr(), w.data_ptr(), w.stride(0), w.stride(1), w.shape[2],
        out.data_ptr(), out.stride(0), out.stride(1), len(lens), hkv * group, hkv, d, code, _native.log2e_scale(d ** -0.5),
        ws.data_ptr(), ws.numel(), None if null else scratch.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    launches = _native.launch_count() - before
    return status, launches, out, w, weights_reference(q, k, v, table, lens, torch.zeros_like(w))


MANY, FEW = [500, 33, 1] * 40, [300, 33]


@pytest.mark.parametrize("size,null", [(0, True), (0, False), (100, False), (1 << 16, False)])
def test_too_little(size, null):
    status, launches, out, w, _ = _call(MANY, size, null)
    assert status == _native.PD_ERR_WORKSPACE and launches == 0 and b"scratch" in _native.lib.pd_last_error_string()
    assert bool((out == 7).all()) and bool((w == 0).all())
    status, launches, out, w, (want, bound, sums, off) = _call(FEW, size, null)
    assert status == _native.PD_OK and launches == 1
    check(out, want, bound)
    check(w, sums, off)
    assert _native.device_error() == 0


def test_enough():
    for lens in (MANY, FEW):
        status, _, out, w, (want, bound, sums, off) = _call(lens, None)
        assert status == _native.PD_OK
        check(out, want, bound)
        check(w, sums, off)


def test_the_decode_mode_of_another_thread():
    """Calls beside a thread that switches the decode mode to and fro: each is whole in one mode or the other."""
    import threading

    from model.paged_evict import paged_decode_weights
    from model.paged_window import paged_decode_window

    hkv, group, d, bs = 8, 2, 128, 16
    gen = torch.Generator().manual_seed(1)
    k, v, table, _ = make_pools(FEW, hkv, d, bs, torch.bfloat16, gen=gen)
    q = torch.randn(2, hkv * group, d, generator=gen).to(torch.bfloat16).cuda()
    seqlen = torch.tensor(FEW, dtype=torch.int32).cuda()
    w = torch.zeros(2, hkv, table.shape[1] * bs, device="cuda")
    want, bound, sums, off = weights_reference(q, k, v, table, FEW, w)
    mode, done = _native.get_decode_mode(), threading.Event()

    def switch():
        while not done.is_set():
            for m in (2, 0):
                _native.set_decode_mode(m)

    thread = threading.Thread(target=switch)
    thread.start()
    try:
        whole = 0
        for _ in range(400):
            w.zero_()
            try:
                out = paged_decode_weights(q, k, v, table, seqlen, w)
                again = paged_decode_window(q, k, v, table, seqlen, 1 << 20)
            except ValueError:  # sized for few rows, and called in the mode that has no kernel of few rows
                continue
            check(out, want, bound)
            check(w, sums, off)
            check(again, want, bound)
            whole += 1
        assert whole > 0
    finally:
        done.set()
        thread.join()
        _native.set_decode_mode(*(mode if isinstance(mode, tuple) else (mode,)))
    assert _native.device_error() == 0
