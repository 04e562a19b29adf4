"""The 4-bit operators on a host without a GPU: argument checks of the C ABI and the Python surface."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fp4_reference as ref
from model import _native

LIB = _native.lib
PTR = ctypes.c_void_p(256)  # never dereferenced: every call below is refused before a launch
TWO = (ctypes.c_int64 * 2)(1024, 128)


def test_the_binding_loads_without_a_gpu():
    assert _native.ops is not None, _native.OPS_ERROR


def _norm(**o):
    a = dict(d=128, rotary=128, n=4, dtype=_native.PD_BF16, pos=_native.PD_SLOT_I64, heads=2)
    a.update(o)
    return LIB.pd_qk_norm_rope(None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, None, None, None, 0, 0, 8, None,
                               a["pos"], a["n"], a["heads"], 1, a["d"], a["rotary"], 1e-6, a["dtype"], None)


@pytest.mark.parametrize("over,status", [
    (dict(), _native.PD_ERR_INVALID),  # no pointers
    (dict(n=0), _native.PD_OK), (dict(n=-1), _native.PD_ERR_INVALID), (dict(d=512), _native.PD_ERR_UNSUPPORTED),
    (dict(d=1, rotary=0), _native.PD_ERR_INVALID), (dict(rotary=3), _native.PD_ERR_INVALID),
    (dict(rotary=130), _native.PD_ERR_INVALID), (dict(dtype=9), _native.PD_ERR_INVALID),
    (dict(pos=5), _native.PD_ERR_INVALID), (dict(heads=0), _native.PD_ERR_INVALID),
])
def test_norm_arguments(over, status):
    assert _norm(**over) == status


def _write(**o):
    a = dict(pages=PTR, blocks=4, bs=16, slots=PTR, st=_native.PD_SLOT_I64, k=PTR, dtype=_native.PD_BF16, n=3, hkv=2, d=128)
    a.update(o)
    return LIB.pd_fp4_write_slots(a["pages"], a["blocks"], a["bs"], a["slots"], a["st"], a["k"], TWO, PTR, TWO, None,
                                  a["dtype"], a["n"], a["hkv"], a["d"], None)


@pytest.mark.parametrize("over,status", [
    (dict(bs=8), _native.PD_ERR_UNSUPPORTED), (dict(bs=24), _native.PD_ERR_INVALID), (dict(d=32), _native.PD_ERR_UNSUPPORTED),
    (dict(d=96), _native.PD_ERR_UNSUPPORTED), (dict(pages=None), _native.PD_ERR_INVALID),
    (dict(pages=ctypes.c_void_p(264)), _native.PD_ERR_INVALID), (dict(slots=None), _native.PD_ERR_INVALID),
    (dict(st=7), _native.PD_ERR_INVALID), (dict(k=None), _native.PD_ERR_INVALID), (dict(dtype=7), _native.PD_ERR_INVALID),
    (dict(n=-1), _native.PD_ERR_INVALID), (dict(n=0), _native.PD_OK), (dict(blocks=0), _native.PD_ERR_INVALID),
    (dict(hkv=0), _native.PD_ERR_INVALID),
])
def test_write_arguments(over, status):
    assert _write(**over) == status


def _decode(**o):
    a = dict(q=PTR, st=1024, blocks=4, bs=16, bt=4, maxb=4, seqlen=PTR, B=2, H=4, hkv=2, d=128, dtype=_native.PD_BF16,
             ws=PTR)
    a.update(o)
    return LIB.pd_fp4_decode(a["q"], a["st"], 128, PTR, a["blocks"], a["bs"], None, PTR, a["bt"], a["maxb"], a["seqlen"],
                             PTR, 1024, 128, a["B"], a["H"], a["hkv"], a["d"], a["dtype"], 1.0, a["ws"], 0, None)


@pytest.mark.parametrize("over,status", [
    (dict(H=3), _native.PD_ERR_INVALID), (dict(dtype=_native.PD_F32), _native.PD_ERR_UNSUPPORTED),
    (dict(dtype=8), _native.PD_ERR_INVALID), (dict(d=32), _native.PD_ERR_UNSUPPORTED), (dict(bt=2), _native.PD_ERR_INVALID),
    (dict(maxb=1 << 27, bt=1 << 27), _native.PD_ERR_INVALID), (dict(B=0), _native.PD_OK), (dict(B=-1), _native.PD_ERR_INVALID),
    (dict(q=None), _native.PD_ERR_INVALID), (dict(st=1020), _native.PD_ERR_INVALID), (dict(seqlen=None), _native.PD_ERR_INVALID),
])
def test_decode_arguments(over, status):
    assert _decode(**over) == status


@pytest.mark.parametrize("bs,hkv,d,status", [
    (1 << 23, 1, 128, _native.PD_OK), (1 << 24, 1, 128, _native.PD_ERR_UNSUPPORTED), (1 << 20, 16, 128, _native.PD_ERR_UNSUPPORTED),
    (1 << 22, 2, 256, _native.PD_ERR_UNSUPPORTED), (1 << 30, 4, 64, _native.PD_ERR_UNSUPPORTED),
])
def test_a_block_is_below_two_gib(bs, hkv, d, status):
    assert _write(bs=bs, hkv=hkv, d=d, n=0) == status
    assert _decode(bs=bs, hkv=hkv, H=hkv, d=d, maxb=1, B=0) == status


def test_prefill_and_copy_arguments():
    args = [PTR, 4, 1024, 128, PTR, 4, 16, None, PTR, 4, 4, None, PTR, PTR, 1024, 128, 2, 2, 4, 2, 128, _native.PD_BF16,
            1.0, PTR, 0, None]
    assert LIB.pd_fp4_prefill(*args) == _native.PD_ERR_INVALID  # no offsets
    args[17] = 0
    assert LIB.pd_fp4_prefill(*args) == _native.PD_OK  # no query tokens announced
    pools = (ctypes.c_void_p * 1)(256)
    ok = [pools, 1, 4, 64, PTR, PTR, _native.PD_SLOT_I64, 1, None, 0, 0, 0, None, None]
    for i, bad in ((1, -1), (2, 0), (3, 0), (4, None), (6, 9), (7, -1), (8, PTR)):
        a = list(ok)
        a[i] = bad
        assert LIB.pd_block_copy(*a) == _native.PD_ERR_INVALID, i


def test_python_surface_refuses_cpu_tensors():
    from model.paged_fp4 import fp4_pages, paged_decode_fp4, read_slots_fp4, write_slots_fp4
    from model.qk_norm import qk_norm_rope
    from serve.block_copy import copy_blocks

    pages = fp4_pages(2, 16, 1, 64, device="cpu")
    assert pages.shape == (2, 1, 1, 18 * 64) and not pages.any()
    x = torch.zeros(1, 1, 64)
    for call in (lambda: write_slots_fp4(pages, torch.zeros(1, dtype=torch.long), x, x),
                 lambda: read_slots_fp4(pages, torch.zeros(1, dtype=torch.long)),
                 lambda: paged_decode_fp4(x.half(), pages, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)),
                 lambda: qk_norm_rope(x, x, x[0, 0], x[0, 0], x[0], x[0]),
                 lambda: copy_blocks(pages, [0], [1])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_pool_arguments():
    from model.paged_fp4 import Fp4KV, Fp4Pool, fp4_pages

    for bad in (dict(block_size=8), dict(block_size=24), dict(head_dim=32), dict(n_blocks=0), dict(n_head=3),
                dict(dtype=torch.float32), dict(k_unit=3.0), dict(v_unit=0.0), dict(v_unit=[[1.0, 2.0, 4.0]]),
                dict(k_unit=-1.0), dict(k_unit=float("nan"))):
        a = dict(n_layer=2, n_blocks=4, block_size=16, n_kv_head=2, head_dim=64) | bad
        with pytest.raises(ValueError):
            Fp4Pool(**a)
    pool = Fp4Pool(2, 4, 32, 2, 64, n_head=6, k_unit=0.5, v_unit=[[1.0, 2.0], [0.25, 4.0]])
    assert pool.bytes() == 2 * 4 * 2 * 2 * 18 * 64 and pool.units[1].tolist() == [[0.5, 0.5], [0.25, 4.0]]
    assert len(pool.block_tensors()) == 2
    k = torch.zeros(1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        pool.write_slots(0, torch.zeros(1, dtype=torch.long), k, k)
    with pytest.raises(IndexError):
        pool.write_prefill(0, [0], 0, torch.zeros(33, 2, 64), torch.zeros(33, 2, 64))
    with pytest.raises(AttributeError, match="4-bit"):
        pool.keys
    with pytest.raises(TypeError, match="Fp4Pool"):
        Fp4KV(None, [[0]], [0], rope_len=4)
    with pytest.raises(ValueError, match="CUDA"):
        Fp4KV(pool, [[0]], [0], rope_len=4, n_head=6)
    with pytest.raises(ValueError):
        fp4_pages(1, 16, 1, 63)


def test_the_reference_round_trips_its_own_values():
    """The tests' 64-bit form: a value that a page can hold comes back unchanged; the relative error of
    the others is at most half a step, a sixth of the group's maximum."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 2, 64, generator=g)
    unit = torch.tensor([1.0, 0.25])
    y = ref.values(*ref.quantise(x, unit), unit)
    assert torch.equal(ref.values(*ref.quantise(y, unit), unit), y)
    top = x.unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True)
    assert ((x.double() - y).unflatten(-1, (-1, 16)).abs() <= top.double() * (1 / 6 + 1 / 16)).all()
    pages = torch.zeros(2, 2, 1, 18 * 64, dtype=torch.uint8)
    units = torch.stack((unit, unit))
    slots = torch.tensor([3, 17, 0, 31, 8])
    ref.write(pages, slots, x, x, units)
    k, v = ref.read(pages, slots, units)
    assert torch.equal(k, y) and torch.equal(v, y)
