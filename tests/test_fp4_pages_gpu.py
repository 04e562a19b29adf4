"""4-bit pages on a B200: quantised writes and reads, byte for byte against the 64-bit definition."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu


def _units(hkv, seed=0):
    g = torch.Generator().manual_seed(seed)
    return 2.0 ** torch.randint(-6, 4, (2, hkv), generator=g).float()


def _rows(n, hkv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    # magnitudes over the whole range of the scales, exact ties, zeros and saturating rows among them
    k = torch.randn(n, hkv, d, generator=g) * 2.0 ** torch.randint(-14, 12, (n, hkv, 1), generator=g)
    v = torch.randint(-24, 25, (n, hkv, d), generator=g) * 0.25
    v[::3] *= 2.0 ** -3
    k[n // 2, 0] = 0
    return k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,hkv,d,bs", [(1, 1, 64, 16), (37, 3, 128, 16), (70, 2, 256, 32), (129, 8, 64, 64), (5, 2, 128, 128)])
def test_write_and_read_are_exact(cuda_device, dtype, n, hkv, d, bs):
    from model.paged_fp4 import fp4_pages, read_slots_fp4, write_slots_fp4

    n_blocks = -(-n // bs) + 2
    units = _units(hkv, seed=n)
    k, v = _rows(n, hkv, d, dtype, seed=d)
    slots = torch.randperm(n_blocks * bs, generator=torch.Generator().manual_seed(1))[:n]
    want = torch.zeros(n_blocks, hkv, bs // 16, 18 * d, dtype=torch.uint8)
    ref.write(want, slots, k, v, units)
    pages = fp4_pages(n_blocks, bs, hkv, d, device=cuda_device)
    ud = units.to(cuda_device)
    for ids in (slots.to(cuda_device), slots.to(torch.int32).to(cuda_device)):
        pages.zero_()
        write_slots_fp4(pages, ids, k.to(cuda_device), v.to(cuda_device), units=ud)
        got = pages.cpu()
        # a negative zero code stands for zero as well
        for a, b in zip(ref.read(got, slots, units), ref.read(want, slots, units)):
            assert torch.equal(a, b)
        kc, ks, vc, vs = ref.places(d)
        for at in (ks, vs):  # every scale byte, written or not
            assert torch.equal(got[..., at.flatten()], want[..., at.flatten()])
    kk, vv = read_slots_fp4(pages, slots.to(cuda_device), torch.float32, units=ud)
    for a, b in zip((kk, vv), ref.read(want, slots, units)):
        assert torch.equal(a.cpu().double(), b)
    kk, _ = read_slots_fp4(pages, slots.to(cuda_device), torch.bfloat16, units=ud)
    assert torch.equal(kk.cpu().double(), ref.read(want, slots, units)[0])


def test_every_rounding_boundary(cuda_device):
    """For every scale, the values on, just under and just over each tie between two codes."""
    from model.paged_fp4 import fp4_pages, read_slots_fp4, write_slots_fp4

    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    scales = ref.SCALES[1:].float()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        rows = []
        for eps in (0.0, 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -7, -(2.0 ** -23 if dtype == torch.float32 else 2.0 ** -7)):
            x = torch.zeros(len(scales), 16)
            x[:, 0] = 6 * scales  # fixes the scale
            x[:, 1:8] = ties * scales[:, None] * (1 + eps)
            x[:, 8:15] = -x[:, 1:8]
            rows.append(x)
        x = torch.cat(rows).to(dtype)
        x = x[torch.isfinite(x.float()).all(-1)]
        x = torch.nn.functional.pad(x, (0, 0, 0, -len(x) % 4)).view(-1, 1, 64)
        n = len(x)
        pages = fp4_pages(-(-n // 16), 16, 1, 64, device=cuda_device)
        slots = torch.arange(n, device=cuda_device)
        write_slots_fp4(pages, slots, x.to(cuda_device), x.to(cuda_device))
        unit = torch.ones(1)
        want = ref.values(*ref.quantise(x, unit), unit)
        for got in read_slots_fp4(pages, slots, torch.float32):
            assert torch.equal(got.cpu().double(), want)


def test_scale_rounding_boundaries(cuda_device):
    """Group maxima on, just under and just over six times each tie between two scales."""
    from model.paged_fp4 import fp4_pages, read_slots_fp4, write_slots_fp4

    mid = ((ref.SCALES[1:] + ref.SCALES[:-1]) * 3).float()  # exact: six times the middle
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        rel = 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -7
        m = torch.cat([mid, mid * (1 + rel), mid * (1 - rel)]).to(dtype)
        x = (m[:, None] * torch.linspace(0, 1, 16)).to(dtype)
        x[:, -1] = m
        x = torch.nn.functional.pad(x, (0, 0, 0, -len(x) % 4)).view(-1, 1, 64)
        n = len(x)
        pages = fp4_pages(-(-n // 16), 16, 1, 64, device=cuda_device)
        slots = torch.arange(n, device=cuda_device)
        write_slots_fp4(pages, slots, x.to(cuda_device), x.to(cuda_device))
        unit = torch.ones(1)
        want = ref.values(*ref.quantise(x, unit), unit)
        assert torch.equal(read_slots_fp4(pages, slots, torch.float32)[0].cpu().double(), want)


def test_non_finite_values_and_saturation(cuda_device):
    from model.paged_fp4 import fp4_pages, read_slots_fp4, write_slots_fp4

    x = torch.zeros(1, 1, 64)
    x[0, 0, :16] = torch.tensor([float("nan"), 1.0, -3.0, 6.0] * 4)
    x[0, 0, 16] = float("inf")
    x[0, 0, 17] = -float("inf")
    x[0, 0, 18:20] = torch.tensor([1e5, -100.0])
    x[0, 0, 32] = -1e9
    for dtype in (torch.float32, torch.bfloat16):
        pages = fp4_pages(1, 16, 1, 64, device=cuda_device)
        slots = torch.zeros(1, dtype=torch.long, device=cuda_device)
        xd = x.to(dtype)
        write_slots_fp4(pages, slots, xd.to(cuda_device), xd.to(cuda_device))
        unit = torch.ones(1)
        want = ref.values(*ref.quantise(xd, unit), unit)
        got = read_slots_fp4(pages, slots, torch.float32)[0].cpu().double()
        assert torch.equal(got, want) and got[0, 0, 16] == 2688 and got[0, 0, 17] == -2688 and got[0, 0, 0] == 0


def test_strided_sources_other_slots_stay_and_slots_outside_the_pool(cuda_device):
    from model import _native
    from model.paged_fp4 import fp4_pages, read_slots_fp4, write_slots_fp4

    hkv, d, bs, n = 2, 128, 16, 6
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(n, 5 * d + 1, generator=g).to(torch.bfloat16)
    pages = torch.randint(0, 100, (4, hkv, 1, 18 * d), generator=g, dtype=torch.uint8)
    units = _units(hkv)
    for off in (0, 1):  # aligned rows, and rows one element off
        k, v = qkv[:, off:off + 2 * d].view(n, hkv, d), qkv[:, off + 2 * d:off + 4 * d].view(n, hkv, d)
        slots = torch.tensor([3, 64, 17, -1, 63, 1 << 40])
        keep = torch.tensor([True, False, True, False, True, False])
        want = pages.clone()
        ref.write(want, slots[keep], k[keep], v[keep], units)
        dev = pages.to(cuda_device)
        base = qkv.to(cuda_device)
        assert _native.device_error() == 0
        write_slots_fp4(dev, slots.to(cuda_device), base[:, off:off + 2 * d].view(n, hkv, d),
                        base[:, off + 2 * d:off + 4 * d].view(n, hkv, d), units=units.to(cuda_device))
        assert _native.device_error() == _native.DEVERR_APPEND_RANGE
        assert torch.equal(dev.cpu(), want)
        kk, _ = read_slots_fp4(dev, slots.to(cuda_device), torch.float32, units=units.to(cuda_device))
        assert (kk[~keep] == 0).all() and _native.device_error() == _native.DEVERR_APPEND_RANGE
    write_slots_fp4(dev, slots[:0].to(cuda_device), base[:0, :2 * d].view(0, hkv, d), base[:0, :2 * d].view(0, hkv, d))
    assert read_slots_fp4(dev, slots[:0].to(cuda_device))[0].shape == (0, hkv, d)


@pytest.mark.parametrize("change,match", [
    (dict(pages=lambda t: t.float()), "uint8"), (dict(pages=lambda t: t[..., :-1]), "not 4-bit pages"),
    (dict(pages=lambda t: t[:, ::2]), "contiguous"), (dict(k=lambda t: t[..., :64]), "k/v must be"),
    (dict(v=lambda t: t[:-1]), "shapes differ"), (dict(k=lambda t: t.double(), v=lambda t: t.double()), "one dtype"),
    (dict(v=lambda t: t.half()), "one dtype"), (dict(slots=lambda t: t.float()), "integer tensor"),
    (dict(slots=lambda t: t[:-1]), "one entry per token"), (dict(units=lambda t: t[:1]), "units must be"),
    (dict(units=lambda t: t.half()), "units must be"), (dict(k=lambda t: t.cpu()), "is on cpu"),
])
def test_refusals(cuda_device, change, match):
    from model.paged_fp4 import write_slots_fp4

    a = dict(pages=torch.zeros(2, 2, 2, 18 * 128, dtype=torch.uint8, device=cuda_device),
             slots=torch.arange(3, device=cuda_device), k=torch.zeros(3, 2, 128, device=cuda_device),
             v=torch.zeros(3, 2, 128, device=cuda_device), units=torch.ones(2, 2, device=cuda_device))
    for name, f in change.items():
        a[name] = f(a[name])
    with pytest.raises(ValueError, match=match):
        write_slots_fp4(a["pages"], a["slots"], a["k"], a["v"], units=a["units"])
