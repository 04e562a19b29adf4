"""How exactly the attention weights of the 4-bit cache enter the products, against a 64-bit softmax.

The inputs are such that everything but the weights' rounding is small: queries are multiples of 1/8
and cached values multiples of 1/4, so scores are sums without rounding. What is left is, relative to
the weighted mean of |v|:
* the exponent: scale, product and difference in fp32, scores below 32 in log2 units, under 2^-18;
* exp2 (2 ulp) and the fp32 sums over the few hundred keys here, under 2^-17; both together under 2^-16;
* the weights' rounding: 2^-11 of each for bf16 outputs (fp16, 11 significant bits), 2^-22 for fp16
  outputs (two fp16 parts);
and, where a weight is too small for fp16's exponents, 2^-32 of the largest weight for each key.
To that comes the output's rounding, half an ulp.
"""

from __future__ import annotations

import math

import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu

WEIGHT = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -22}


@pytest.fixture(params=[1, 2], ids=["warps", "tiles"])
def kernel(request):
    from model import _native

    _native.set_fp4_prefill_mode(request.param)
    yield request.param
    _native.set_fp4_prefill_mode(0)


def _check(got, want, mean, keys, largest):
    bound = (ref.HALF_ULP[got.dtype] * want.abs() + (WEIGHT[got.dtype] + 2.0 ** -16) * mean + keys * 2.0 ** -32 * largest
             + 2.0 ** -25)
    err = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound).max()):.3g} times the bound"


def _sink(n, hkv, d, bs=16):
    """Pages whose key 0 has element 0 at 6 and values 0; every other key is 0 with positive values."""
    g = torch.Generator().manual_seed(d)
    blocks = -(-n // bs)
    codes = torch.randint(1, 8, (blocks * bs, hkv, d), generator=g)
    kc, ks, vc, vs = ref.places(d)
    pages = torch.zeros(blocks, hkv, bs // 16, 18 * d, dtype=torch.uint8)
    for t in range(blocks * bs):
        rec = pages[t // bs, :, t % bs // 16]
        rec[:, ks[t % 16]] = rec[:, vs[t % 16]] = 0x38  # a scale of 1
        if t:
            rec[:, vc[t % 16]] = (codes[t, :, 0::2] | (codes[t, :, 1::2] << 4)).to(torch.uint8)
        else:
            rec[:, kc[0][0]] = 7  # 6 in element 0
    return pages, torch.arange(blocks, dtype=torch.int32)[None]


# The other keys' weight is 37.45 * 2^-24 of the sink's: between two of fp16's numbers, were the sink's 1.
GAP = 24 - math.log2(37.45)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_weights_beside_a_large_one_decode(cuda_device, dtype, d):
    from model.paged_fp4 import paged_decode_fp4

    n, rows, hkv, heads = 320, 300, 8, 16
    pages, table = _sink(n, hkv, d)
    q = torch.zeros(1, heads, d, dtype=dtype)
    q[..., 0] = 1
    scale = GAP * math.log(2) / 6
    want, mean = ref.attention(q, pages, table, [n], [1], torch.ones(2, hkv), scale)
    got = paged_decode_fp4(q.to(cuda_device).expand(rows, heads, d), pages.to(cuda_device),
                           table.to(cuda_device).expand(rows, -1),
                           torch.full((rows,), n, dtype=torch.int32, device=cuda_device), scale=scale)
    _check(got, want.expand(rows, heads, d), mean.expand(rows, heads, d), n, 6.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_weights_beside_a_large_one_chunks(cuda_device, kernel, dtype, d):
    from model.paged_fp4 import paged_prefill_fp4

    n, rows, hkv, heads, chunk = 320, 4, 8, 16, 300
    pages, table = _sink(n, hkv, d)
    q = torch.zeros(chunk, heads, d, dtype=dtype)
    q[..., 0] = 1
    scale = GAP * math.log(2) / 6
    want, mean = ref.attention(q, pages, table, [n], [chunk], torch.ones(2, hkv), scale)
    got = paged_prefill_fp4(q.to(cuda_device).repeat(rows, 1, 1), pages.to(cuda_device),
                            table.to(cuda_device).expand(rows, -1),
                            torch.arange(rows + 1, dtype=torch.int32, device=cuda_device) * chunk,
                            torch.full((rows,), n, dtype=torch.int32, device=cuda_device), chunk, scale=scale)
    _check(got, want.repeat(rows, 1, 1), mean.repeat(rows, 1, 1), n, 6.0)


def _exact_scores(rows, heads, hkv, d, seed):
    """q (total, heads, d) in eighths, and pages of scales 1/2 and 1 with both signs of values, so that
    results are far smaller than the mean of |v|."""
    g = torch.Generator().manual_seed(seed)
    chunks, lengths = [c for c, _ in rows], [n for _, n in rows]
    need = [-(-n // 16) for n in lengths]
    pages = torch.randint(0, 256, (sum(need) + 1, hkv, 1, 18 * d), generator=g, dtype=torch.uint8)
    _, ks, _, vs = ref.places(d)
    for at in (ks, vs):
        pick = torch.randint(0, 2, (sum(need) + 1, hkv, 1, at.numel()), generator=g)
        pages[..., at.flatten()] = (0x30 + 8 * pick).to(torch.uint8)
    table = torch.full((len(rows), max(need) + 1), sum(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    q = torch.randint(-8, 9, (sum(chunks), heads, d), generator=g) / 8
    return q, pages, table, chunks, lengths


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,heads,hkv,d", [
    ([(200, 200)], 4, 2, 64), ([(130, 150), (3, 40)], 4, 2, 128), ([(150, 190)], 2, 1, 256), ([(1, 2), (7, 90)], 6, 2, 128),
])
def test_values_that_cancel_chunks(cuda_device, kernel, dtype, rows, heads, hkv, d):
    from model.paged_fp4 import paged_prefill_fp4

    q, pages, table, chunks, lengths = _exact_scores(rows, heads, hkv, d, seed=d)
    scale = 0.7 / d ** 0.5
    want, mean = ref.attention(q, pages, table, lengths, chunks, torch.ones(2, hkv), scale)
    cu = torch.tensor([sum(chunks[:i]) for i in range(len(chunks) + 1)], dtype=torch.int32)
    got = paged_prefill_fp4(*(t.to(cuda_device) for t in (q.to(dtype), pages, table, cu,
                                                          torch.tensor(lengths, dtype=torch.int32))), max(chunks),
                            scale=scale)
    _check(got, want, mean, max(lengths), 6.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_values_that_cancel_decode(cuda_device, dtype, d):
    from model.paged_fp4 import paged_decode_fp4

    q, pages, table, _, lengths = _exact_scores([(1, n) for n in (2, 3, 17, 90, 200, 5, 33)], 6, 2, d, seed=d + 1)
    scale = 0.7 / d ** 0.5
    want, mean = ref.attention(q, pages, table, lengths, [1] * len(lengths), torch.ones(2, 2), scale)
    got = paged_decode_fp4(*(t.to(cuda_device) for t in (q.to(dtype), pages, table, torch.tensor(lengths, dtype=torch.int32))),
                           scale=scale)
    _check(got, want, mean, max(lengths), 6.0)


@pytest.mark.parametrize("exponent", [-122, -101, 100, 118])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_queries_over_the_range_of_bf16(cuda_device, kernel, d, exponent):
    """Queries as large and as small as bf16 holds them, with a scale that brings the scores back."""
    from model.paged_fp4 import paged_decode_fp4, paged_prefill_fp4

    q, pages, table, chunks, lengths = _exact_scores([(40, 70), (5, 5)], 4, 2, d, seed=d + 2)
    q = (q * 2.0 ** exponent).to(torch.bfloat16)
    scale = 0.7 / d ** 0.5 * 2.0 ** -exponent
    want, mean = ref.attention(q, pages, table, lengths, chunks, torch.ones(2, 2), scale)
    cu = torch.tensor([0, 40, 45], dtype=torch.int32)
    dev = [t.to(cuda_device) for t in (q, pages, table, cu, torch.tensor(lengths, dtype=torch.int32))]
    _check(paged_prefill_fp4(*dev, 40, scale=scale), want, mean, 70, 6.0)
    want, mean = ref.attention(q[:2], pages, table, lengths, [1, 1], torch.ones(2, 2), scale)
    _check(paged_decode_fp4(dev[0][:2], *dev[1:3], dev[4], scale=scale), want, mean, 70, 6.0)
