"""Head norm with rotation on a B200 against the 64-bit formula.

Tolerance: the result is one rounding (half an ulp of the output type, relative) of an fp32
evaluation. Its sum of D squares, square root, division and five products and sums lose at most
some D / 8 + 12 roundings of 2^-24 of the magnitudes that are added, under 2^-18 of them.
fp16 outputs below the normal range round to multiples of 2^-24, so half of that is added.
"""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu


def _case(tokens, heads, hkv, d, rotary, dtype, seed=0, fused=True, n_pos=97):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, (heads + 2 * hkv) * d, generator=g).to(dtype)
    q = qkv[:, :heads * d].view(tokens, heads, d)
    k = qkv[:, heads * d:(heads + hkv) * d].view(tokens, hkv, d)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g)).to(dtype)
    ang = torch.rand(n_pos, max(rotary // 2, 1), generator=g) * 6.3
    pos = torch.randint(0, n_pos, (tokens,), generator=g)
    return qkv, q, k, wq, wk, ang.cos().to(dtype), ang.sin().to(dtype), pos


def _check(got, x, w, cos, sin, pos, eps, rotary):
    want, size = ref.norm_rope(x, w, cos, sin, pos, eps, rotary)
    bound = ref.HALF_ULP[got.dtype] * want.abs() + 2.0 ** -18 * size + 2.0 ** -25
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,hkv,d,rotary", [
    (1, 16, 8, 128, 128), (3, 16, 8, 128, 64), (33, 8, 2, 256, 64), (7, 3, 1, 64, 64), (5, 5, 5, 64, 16),
    (2, 40, 8, 128, 0), (4, 2, 2, 80, 20), (3, 2, 1, 96, 96), (2, 1, 1, 10, 6), (1, 1, 1, 2, 2), (2, 2, 2, 250, 250),
])
def test_matches_the_formula(cuda_device, dtype, tokens, heads, hkv, d, rotary):
    from model.qk_norm import qk_norm_rope

    qkv, q, k, wq, wk, cos, sin, pos = _case(tokens, heads, hkv, d, rotary, dtype)
    dev = qkv.to(cuda_device)
    qd = dev[:, :heads * d].view(tokens, heads, d)
    kd = dev[:, heads * d:(heads + hkv) * d].view(tokens, hkv, d)
    args = [t.to(cuda_device) for t in (wq, wk, cos, sin)]
    qo, ko = qk_norm_rope(qd, kd, *args, pos.to(cuda_device), eps=1e-6, rotary_dim=rotary)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.is_contiguous() and ko.is_contiguous()
    _check(qo, q, wq, cos, sin, pos, 1e-6, rotary)
    _check(ko, k, wk, cos, sin, pos, 1e-6, rotary)
    assert torch.equal(dev.cpu(), qkv), "inputs are left alone"


@pytest.mark.parametrize("aligned", [True, False])
def test_strides_positions_and_in_place(cuda_device, aligned):
    from model.qk_norm import qk_norm_rope

    tokens, h, hkv, d, rotary = 9, 4, 2, 128, 128
    _, q, k, wq, wk, cos, sin, pos = _case(tokens, h, hkv, d, rotary, torch.bfloat16, seed=3, fused=False)
    # heads-major storage, and (unaligned) rows that start one element off any vector boundary
    base = torch.zeros(h, tokens, d + 3, dtype=torch.bfloat16, device=cuda_device)
    view = (base[:, :, 1:d + 1] if not aligned else base[:, :, :d]).transpose(0, 1)
    view.copy_(q)
    args = [t.to(cuda_device) for t in (wq, wk, cos, sin)]
    pd = pos.to(cuda_device)
    kd = k.to(cuda_device)
    qo, ko = qk_norm_rope(view, kd, *args, pd.to(torch.int32))
    _check(qo, q, wq, cos, sin, pos, 1e-6, rotary)
    # wide tables (both halves stored), an expanded weight, in place
    wide = [torch.cat((t, t), 1) for t in args[2:]]
    q2, k2 = q.to(cuda_device), k.to(cuda_device)
    r = qk_norm_rope(q2, k2, args[0], args[1], *wide, pd, rotary_dim=rotary, q_out=q2, k_out=k2)
    assert r[0] is q2 or r[0].data_ptr() == q2.data_ptr()
    _check(q2, q, wq, cos, sin, pos, 1e-6, rotary)
    _check(k2, k, wk, cos, sin, pos, 1e-6, rotary)
    apart = qk_norm_rope(q.to(cuda_device), k.to(cuda_device), *args, pd)
    assert torch.equal(q2, apart[0]) and torch.equal(k2, apart[1]), "in place changes no bit"
    # no positions: token t at position t
    r = qk_norm_rope(q.to(cuda_device), kd, *args)
    _check(r[0], q, wq, cos, sin, torch.arange(tokens), 1e-6, rotary)


def test_extremes_and_positions_outside_the_tables(cuda_device):
    from model import _native
    from model.qk_norm import qk_norm_rope

    q = torch.zeros(4, 2, 64, dtype=torch.float32)
    q[0] = 1e18  # the squares' sum stays finite in fp32
    q[1, 0, 5] = 3.0
    k = q[:, :1].clone()
    w = torch.ones(64)
    cos, sin = torch.ones(8, 32), torch.zeros(8, 32)
    dev = [t.to(cuda_device) for t in (q, k, w, w, cos, sin)]
    assert _native.device_error() == 0
    qo, _ = qk_norm_rope(*dev, torch.tensor([0, 7, 2, 3], device=cuda_device))
    _check(qo, q, w, cos, sin, torch.tensor([0, 7, 2, 3]), 1e-6, 64)
    assert (qo[2:] == 0).all(), "a zero row stays zero"
    assert _native.device_error() == 0
    qo, ko = qk_norm_rope(*dev, torch.tensor([0, 8, -1, 3], device=cuda_device))
    assert (qo[1:3] == 0).all() and (ko[1:3] == 0).all() and (qo[0] != 0).any()
    assert _native.device_error() == _native.DEVERR_ROPE_RANGE
    empty = qk_norm_rope(dev[0][:0], dev[1][:0], *dev[2:])
    assert empty[0].shape == (0, 2, 64) and empty[1].shape == (0, 1, 64)


@pytest.mark.parametrize("change,match", [
    (dict(q=lambda t: t[0]), "must be"), (dict(k=lambda t: t[:1]), "share their tokens"),
    (dict(k=lambda t: t.float()), "like q"), (dict(wq=lambda t: t[:-1]), "q_weight must be"),
    (dict(cos=lambda t: t[:, :-1]), "cos and sin"), (dict(pos=lambda t: t.float()), "int32 or int64"),
    (dict(pos=lambda t: t[:-1]), "positions must be"), (dict(sin=lambda t: t.cpu()), "is on cpu"),
    (dict(rotary=lambda t: 7), "even"), (dict(rotary=lambda t: 256), "rotary_dim"),
])
def test_refusals(cuda_device, change, match):
    from model.qk_norm import qk_norm_rope

    _, q, k, wq, wk, cos, sin, pos = _case(3, 2, 1, 64, 64, torch.bfloat16, fused=False)
    a = dict(zip(("q", "k", "wq", "wk", "cos", "sin", "pos"), (t.to(cuda_device) for t in (q, k, wq, wk, cos, sin, pos))))
    a["rotary"] = None
    for name, f in change.items():
        a[name] = f(a[name])
    rotary = a.pop("rotary")
    with pytest.raises(ValueError, match=match):
        qk_norm_rope(*a.values(), rotary_dim=rotary)
