"""NaN and infinite scores of visible keys in the paged decodes: a softmax that holds a NaN is NaN, a score of -inf has
weight 0, and both stay in the (row, head) that they belong to, whichever kernel and split a call takes."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import attend, check, make_pools, row_of, window_mask
from model import _native
from model.paged_evict import paged_decode_weights
from model.paged_window import paged_decode_window
from model.triton_decode import paged_decode, paged_decode_plan

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")
ALL = 1 << 20  # a window over every row

# (lengths, kv heads, group, head_dim, block, dtype): few rows, one tile a warp and several; many rows, split and whole;
# CUDA-core tiles; fp32
SHAPES = [
    ([33, 17, 1, 65], 8, 2, 128, 16, BF16), ([700], 8, 2, 128, 16, BF16), ([257, 33], 2, 4, 256, 32, F16),
    ([400, 9], 4, 2, 128, 16, F32), ([65], 3, 5, 64, 64, F16), ([3000] + [41, 900] * 25, 8, 2, 128, 16, BF16),
    ([5000, 0, 33, 1200] * 16, 2, 4, 256, 32, F16), ([20, 33] * 150, 8, 1, 64, 16, BF16), ([900, 33], 4, 2, 32, 16, BF16),
    ([2100] + [300, 9] * 30, 8, 2, 128, 16, F32), ([40, 17] * 120, 4, 3, 16, 16, F32)]
CALLS = ["plain", "window", "narrow", "weights", "plan"]
NARROW = 100, 5


def _call(kind, q, k, v, table, seqlen):
    """(out, sums or None) of one decode."""
    if kind == "plain":
        return paged_decode(q, k, v, table, seqlen), None
    if kind == "plan":
        return paged_decode_plan(q, [k], [v], table, seqlen, window=ALL).run(0, q), None
    if kind == "weights":
        w = torch.zeros(q.shape[0], k.shape[2], table.shape[1] * k.shape[1], device="cuda")
        return paged_decode_weights(q, k, v, table, seqlen, w), w
    window, sinks = (ALL, 0) if kind == "window" else NARROW
    return paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks), None


def _case(shape, seed=0):
    lens, hkv, group, d, bs, dtype = shape
    gen = torch.Generator().manual_seed(seed)
    k, v, table, _ = make_pools(lens, hkv, d, bs, dtype, gen=gen)
    q = torch.randn(len(lens), hkv * group, d, generator=gen).to(dtype).cuda()
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda()


def _same_elsewhere(got, clean, touched):
    """NaN in every touched (row, head), the clean call's bits in every other."""
    assert bool(got[touched].isnan().all())
    assert torch.equal(got[~touched], clean[~touched])


@pytest.mark.parametrize("kind", CALLS)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_nan_query_head(shape, kind):
    lens, hkv, group = shape[:3]
    q, k, v, table, seqlen = _case(shape)
    clean, clean_sums = _call(kind, q, k, v, table, seqlen)
    touched = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        if n and b % 3 == 0:
            touched[b, (b + group - 1) % (hkv * group)] = True
    q[touched.nonzero(as_tuple=True)[0], touched.nonzero(as_tuple=True)[1], 1] = NAN
    got, sums = _call(kind, q, k, v, table, seqlen)
    _same_elsewhere(got, clean, touched)
    if sums is not None:
        j = torch.arange(sums.shape[2], device="cuda")
        hit = touched.view(len(lens), hkv, group).any(2)[..., None] & (j < seqlen[:, None, None])
        _same_elsewhere(sums, clean_sums, hit)
    assert _native.device_error() == 0


@pytest.mark.parametrize("kind", CALLS)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_nan_key(shape, kind):
    """The last token's, so that it is alone in the last tile of many rows, and a middle one's."""
    lens, hkv, group, _, bs = shape[:5]
    q, k, v, table, seqlen = _case(shape, seed=1)
    clean, clean_sums = _call(kind, q, k, v, table, seqlen)
    heads = torch.zeros(len(lens), hkv, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        if n and b % 4 != 3:
            j = n - 1 if b % 2 == 0 else n - 1 - min(n - 1, 60)
            k[table[b, j // bs], j % bs, b % hkv, 0] = NAN
            heads[b, b % hkv] = True
    got, sums = _call(kind, q, k, v, table, seqlen)
    _same_elsewhere(got, clean, heads.repeat_interleave(group, 1))
    if sums is not None:
        j = torch.arange(sums.shape[2], device="cuda")
        _same_elsewhere(sums, clean_sums, heads[..., None] & (j < seqlen[:, None, None]))
    assert _native.device_error() == 0


def _without(q, k, v, table, lens, gone, window, sinks):
    """(out, bound, sums, their bound) where the keys `gone` (row -> tokens) have no weight."""
    heads, d, hkv = q.shape[1], q.shape[2], k.shape[2]
    out, bound = (torch.zeros_like(q, dtype=torch.float64) for _ in range(2))
    sums, off = (torch.zeros(len(lens), hkv, table.shape[1] * k.shape[1], dtype=torch.float64, device="cuda") for _ in range(2))
    for b, n in enumerate(lens):
        if not n:
            continue
        seen = window_mask(n - 1, 1, n, window, sinks, "cuda")
        seen[:, gone[b]] = False
        x = q[b].double().view(hkv, heads // hkv, 1, d)
        o, p, e, rel = attend(x, row_of(k, table, b, n), row_of(v, table, b, n), seen, d ** -0.5)
        out[b], bound[b] = o.reshape(heads, d), e.reshape(heads, d)
        sums[b, :, :n], off[b, :, :n] = p[:, :, 0].sum(1), rel * p[:, :, 0].sum(1)
    return out, bound, sums, off


@pytest.mark.parametrize("kind", CALLS)
@pytest.mark.parametrize("shape", SHAPES)
def test_scores_of_minus_infinity(shape, kind):
    """Keys with scores of -inf, whole tiles of them at a row's start and end: weight 0, whatever else a warp has."""
    lens, hkv, group, d, bs, dtype = shape
    q, k, v, table, seqlen = _case(shape, seed=2)
    q[..., 0] = 1.0
    gone = []
    for b, n in enumerate(lens):
        left = n // 3  # stays, in the middle
        tokens = [j for j in range(n) if j != left and (j < 70 or j >= n - 40 or j % 5 == 0)]
        gone.append(tokens)
        at = torch.tensor(tokens, dtype=torch.long, device="cuda")
        k[table[b].long()[at // bs], at % bs, :, 0] = -INF
    window, sinks = NARROW if kind == "narrow" else (ALL, 0)
    blind = []  # rows whose visible keys are all gone
    for b, n in enumerate(lens):
        dead = set(gone[b])
        blind.append(n > 0 and all(j in dead for j in range(n) if j < sinks or n - 1 - j < window))
    blind = torch.tensor(blind, device="cuda")
    got, sums = _call(kind, q, k, v, table, seqlen)
    out, bound, want_sums, off = _without(q, k, v, table, lens, gone, window, sinks)
    assert bool(got[blind].isnan().all())  # nothing but -inf: 0 / 0, as the softmax has it
    check(got[~blind], out[~blind], bound[~blind])
    if sums is not None:
        check(sums, want_sums, off)
    assert _native.device_error() == 0


@pytest.mark.parametrize("shape", [([700], 8, 2, 128, 16, BF16), ([33, 0], 2, 4, 256, 32, F16), ([300] * 90, 8, 1, 64, 16, BF16),
                                   ([100, 9], 4, 2, 64, 16, F32), ([900, 1], 4, 2, 32, 16, BF16)])
def test_rows_of_nothing_but_minus_infinity(shape):
    """As the softmax has it, 0 / 0; a row without tokens gives zeros."""
    lens = shape[0]
    q, k, v, table, seqlen = _case(shape, seed=3)
    q[..., 0] = 1.0
    k[..., 0] = -INF
    empty = torch.tensor([n == 0 for n in lens], device="cuda")
    for kind in CALLS:
        got, sums = _call(kind, q, k, v, table, seqlen)
        assert bool(got[~empty].isnan().all()) and bool((got[empty] == 0).all())
        if sums is not None:
            assert all(bool(sums[b, :, :n].isnan().all()) and bool((sums[b, :, n:] == 0).all()) for b, n in enumerate(lens))


@pytest.mark.parametrize("shape", SHAPES[1:4] + SHAPES[8:10])
def test_partials_of_two_ranks(shape):
    """Partials of the rows' first and second halves, merged: every score of the first half is -inf."""
    q, k, v, table, seqlen = _case(shape, seed=4)
    lens, hkv, group, d, bs, _ = shape
    pages = table.shape[1] // 2
    q[..., 0] = 1.0
    gone = [list(range(min(n, pages * bs))) for n in lens]
    for b, n in enumerate(lens):
        k[table[b, :pages][:-(-n // bs)].long(), :, :, 0] = -INF
    heads = hkv * group
    m, l = (torch.empty(2, len(lens), heads, device="cuda") for _ in range(2))
    acc = torch.empty(2, len(lens), heads, d, device="cuda")
    ws = torch.empty(_native.workspace_bytes(len(lens), heads, hkv, d, q.dtype), dtype=torch.uint8, device="cuda")
    for half in (0, 1):
        t = (table[:, :pages], table[:, pages:])[half].contiguous()
        n = (seqlen - half * pages * bs).clamp(min=0, max=(pages if half == 0 else 1 << 20) * bs).to(torch.int32)
        _native.decode_partials(q, k, v, t, n, m[half], l[half], acc[half], _native.log2e_scale(d ** -0.5), ws)
    got = torch.empty_like(q)
    _native.lse_merge(m, l, acc, got)
    out, bound, _, _ = _without(q, k, v, table, lens, gone, ALL, 0)
    dead = torch.tensor([0 < n <= pages * bs for n in lens], device="cuda")
    assert bool(got[dead].isnan().all())
    check(got[~dead], out[~dead], bound[~dead])
