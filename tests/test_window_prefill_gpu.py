"""Chunks of queries over a sliding window with sinks against their definition in 64 bits (tolerances:
bounded_reference.attend)."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import check, chunk_reference, make_pools
from model import _native
from model.paged_window import paged_decode_window, paged_prefill_window

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _case(rows, hkv, group, d, bs, dtype, seed=0):
    """rows: (query tokens, cached tokens with them)."""
    gen = torch.Generator().manual_seed(seed)
    lens = [n for _, n in rows]
    k, v, table, _ = make_pools(lens, hkv, d, bs, dtype, gen=gen)
    cu = [0]
    for c, _ in rows:
        cu.append(cu[-1] + c)
    q = torch.randn(cu[-1], hkv * group, d, generator=gen).to(dtype).cuda()
    return q, k, v, table, cu, lens


def _run(case, window, sinks, longest=None, **more):
    q, k, v, table, cu, lens = case
    return paged_prefill_window(q, k, v, table, torch.tensor(cu, dtype=torch.int32).cuda(),
                                torch.tensor(lens, dtype=torch.int32).cuda(),
                                max(b - a for a, b in zip(cu, cu[1:])) if longest is None else longest, window, sinks=sinks, **more)


def _check(rows, hkv, group, d, bs, dtype, window, sinks, seed=0, scale=None):
    case = _case(rows, hkv, group, d, bs, dtype, seed)
    got = _run(case, window, sinks, scale=scale)
    want, bound = chunk_reference(*case, window, sinks, scale)
    check(got, want, bound)
    assert _native.device_error() == 0


ROWS = [(1, 1), (5, 5), (0, 40), (64, 64), (65, 200), (3, 700), (130, 130), (200, 333), (17, 16 * 30)]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (16, 0), (16, 16), (17, 15), (33, 4), (64, 32), (100, 0),
                                          (129, 130), (255, 1), (500, 100), (5000, 0), (1 << 40, 1 << 40), (7, 2000)])
def test_windows(window, sinks):
    _check(ROWS, 4, 2, 128, 16, BF16, window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hkv,group,d,bs", [(2, 4, 256, 32), (4, 1, 64, 16), (1, 8, 128, 16), (3, 5, 64, 64), (4, 3, 128, 8),
                                            (2, 6, 256, 8), (1, 16, 64, 128), (2, 7, 128, 256), (1, 1, 256, 16), (8, 2, 128, 16)])
def test_heads_and_blocks(dtype, hkv, group, d, bs):
    _check(ROWS, hkv, group, d, bs, dtype, 37, 5, seed=1)
    _check([(300, 900), (7, 7)], hkv, group, d, bs, dtype, 250, 20, seed=2)


@pytest.mark.parametrize("rows,window,sinks", [([(1500, 1500)], 400, 4), ([(700, 4000), (1, 4000), (129, 150)], 1024, 64),
                                               ([(2049, 2100)], 100, 0), ([(1, 3)] * 200, 2, 1)])
def test_long_and_many(rows, window, sinks):
    _check(rows, 4, 2, 128, 16, BF16, window, sinks, seed=3)
    _check(rows, 2, 4, 256, 32, F16, window, sinks, seed=4)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 1e-30])
def test_scales(scale):
    _check(ROWS, 2, 2, 64, 16, F16, 50, 3, scale=scale)
    _check(ROWS, 2, 2, 128, 16, BF16, 50, 3, scale=scale)


def test_queries_before_their_row():
    """Tokens of a chunk longer than its row sit before the row's first token and see nothing."""
    rows = [(40, 10), (5, 0), (200, 130), (3, 3)]
    case = _case(rows, 4, 2, 128, 16, BF16)
    got = _run(case, 20, 2)
    want, bound = chunk_reference(*case, 20, 2)
    check(got, want, bound)
    assert got[:30].abs().max() == 0 and got[40:45].abs().max() == 0


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 256), (BF16, 64)])
def test_hidden_tokens_may_hold_anything(dtype, d):
    """NaN in tokens that no query of the chunk sees, past the row, and in unused blocks leave no trace."""
    rows, window, sinks = [(20, 400), (1, 33), (50, 90), (7, 7)], 50, 6
    case = _case(rows, 4, 2, d, 16, dtype)
    q, k, v, table, cu, lens = case
    want, bound = chunk_reference(*case, window, sinks)
    bad = torch.full(k.shape[:2], True, device="cuda")
    for b, (c, n) in enumerate(rows):
        for j in range(n):
            if j < sinks or j > n - c - window:
                bad[table[b, j // 16], j % 16] = False
    for value in (float("nan"), float("inf")):
        k[bad] = value
        v[bad] = value
        check(_run(case, window, sinks), want, bound)


def test_hidden_pages_are_not_looked_up():
    rows, window, sinks = [(30, 2000), (100, 1500)], 100, 5
    case = _case(rows, 8, 2, 128, 16, BF16)
    want = _run(case, window, sinks)
    table = case[3]
    for b, (c, n) in enumerate(rows):
        table[b, 1:(n - c - window + 1) // 16] = 0x7fffffff
        table[b, -(-n // 16):] = -5
    assert torch.equal(_run(case, window, sinks), want)


def test_blocks_outside_the_pool_read_zeros():
    case = _case([(10, 64)], 2, 2, 128, 16, BF16)
    q, k, v, table, cu, lens = case
    spare = 0 if int(table[0, 1]) != 0 else 1
    good = table.clone()
    k[good[0, 1].long()] = 0
    v[good[0, 1].long()] = 0
    want = _run(case, 60, 0)
    for wrong in (-1, k.shape[0], 0x10000000, 0x7fffffff):
        table[0, 1] = wrong
        assert torch.equal(_run(case, 60, 0), want)


def test_single_tokens_match_the_decode():
    lens = [1, 40, 700, 1500]
    case = _case([(1, n) for n in lens], 8, 2, 128, 16, BF16)
    q, k, v, table, cu, _ = case
    want, bound = chunk_reference(*case, 256, 4)
    check(_run(case, 256, 4), want, bound)
    check(paged_decode_window(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), 256, sinks=4), want, bound)


def test_strides_and_what_is_left_alone():
    rows, window, sinks = [(30, 100), (64, 70), (5, 300)], 64, 3
    case = _case(rows, 4, 2, 128, 16, BF16)
    q, k, v, table, cu, lens = case
    want = _run(case, window, sinks)
    fused = torch.zeros(q.shape[0], 20, 128, dtype=BF16, device="cuda")
    fused[:, 5:13] = q
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    for x in (fused[:, 5:13], odd, q.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        assert torch.equal(_run((x, *case[1:]), window, sinks), want)
    # pools inside one tensor; every other block of a larger pool (its blocks are not evenly spaced in tokens)
    big = torch.stack((k, v), 3)
    assert torch.equal(_run((q, big[..., 0, :], big[..., 1, :], table, cu, lens), window, sinks), want)
    two = torch.stack((k, v), 1)
    assert torch.equal(_run((q, two[:, 0], two[:, 1], table, cu, lens), window, sinks), want)
    wide = torch.full((3, 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    out = torch.full((q.shape[0] + 9, 8, 128), 5.0, dtype=BF16, device="cuda")
    more = torch.cat((q, q[:9]))  # tokens behind the last row
    _run((more, k, v, wide[:, ::2], cu, lens), window, sinks, longest=10 ** 9, out=out)
    assert torch.equal(out[:q.shape[0]], want) and bool((out[q.shape[0]:] == 5).all())
    # a chunk's tokens past the announced longest stay as they were
    out.fill_(5.0)
    _run((more, k, v, table, cu, lens), window, sinks, longest=32, out=out)
    assert torch.equal(out[:62], want[:62]) and bool((out[62:94] == 5).all()) and torch.equal(out[94:99], want[94:])
    got = paged_prefill_window(q, k, v, table, torch.tensor(cu).cuda(), torch.tensor(lens).cuda(), 64, window, sinks=sinks)
    assert torch.equal(got, want)


def test_streams_and_graphs():
    cases = [_case([(40, 900 + 40 * i), (17, 17), (300, 1000)], 4, 2, 128, 16, BF16, seed=i) for i in range(2)]
    want = [_run(c, 512, 4) for c in cases]
    q, k, v, table, cu, lens = cases[0]
    cu_t, lens_t = torch.tensor(cu, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = paged_prefill_window(q, k, v, table, cu_t, lens_t, 300, 512, sinks=4)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(side):
            g.replay()
        with torch.cuda.stream(other):
            eager = _run(cases[1], 512, 4)
    torch.cuda.synchronize()
    assert torch.equal(captured, want[0]) and torch.equal(eager, want[1])


def test_empty_calls():
    case = _case([(4, 10)], 2, 2, 64, 16, BF16)
    q, k, v, table, cu, lens = case
    assert _run(case, 8, 0, longest=0).shape == q.shape
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged_prefill_window(q[:0], k, v, table[:0], torch.zeros(1, dtype=torch.int32, device="cuda"), none, 5, 8).shape[0] == 0
    assert _run((q, k, v, table[:, :0], cu, lens), 8, 0).abs().max() == 0


@pytest.mark.parametrize("rows,hkv,group,d,dtype", [([(300, 900)], 4, 2, 128, BF16), ([(8, 900)], 1, 4, 64, F16),
                                                    ([(600, 900)] * 20, 4, 4, 128, F16), ([(40, 700)], 2, 2, 256, BF16)])
def test_a_wait_that_runs_out_is_reported(rows, hkv, group, d, dtype):
    """Under the test limit every wait gives up at once: the flag is set, the kernel returns, the next call is right."""
    case = _case(rows, hkv, group, d, 16, dtype)
    want = _run(case, 200, 4)
    limit = _native.lib.pd_get_wait_limit()
    try:
        _native.lib.pd_set_wait_limit(10)
        _run(case, 200, 4)
        torch.cuda.synchronize()
        assert _native.device_error(clear=True) & _native.DEVERR_WAIT_TIMEOUT
    finally:
        _native.lib.pd_set_wait_limit(limit)
    assert torch.equal(_run(case, 200, 4), want)
    assert _native.device_error() == 0


def test_refusals():
    case = _case([(10, 100), (4, 40)], 4, 2, 128, 16, BF16)
    q, k, v, table, cu, lens = case
    cu_t, lens_t = torch.tensor(cu, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()

    def refused(error=ValueError, match=None, **change):
        args = dict(q=q, k_cache=k, v_cache=v, block_table=table, cu_seqlens_q=cu_t, seqlen_k=lens_t, max_seqlen_q=10, window=8)
        args.update(change)
        with pytest.raises(error, match=match):
            paged_prefill_window(**args)

    refused(match="window must be", window=0)
    refused(match="sinks must be", sinks=-1)
    refused(match="needs fp16 or bf16", q=q.float(), k_cache=k.float(), v_cache=v.float())
    refused(match="head_dim must be 64", q=q[..., :32], k_cache=k[..., :32].contiguous(), v_cache=v[..., :32].contiguous())
    refused(match="block_size must be at least 8", k_cache=k[:, :4].contiguous(), v_cache=v[:, :4].contiguous())
    refused(match="share one dtype", q=q.half())
    refused(match="cu_seqlens_q must be", cu_seqlens_q=cu_t[:2])
    refused(match="cu_seqlens_q must be int32", cu_seqlens_q=cu_t.float())
    refused(match="block_table must be", block_table=table[:1])
    refused(match="seqlen_k must be 1-D", seqlen_k=lens_t[None])
    refused(match="multiple of n_kv_head", q=q[:, :6])
    refused(match="out must be", out=torch.empty_like(q)[:5])
    refused(match="share memory with q", out=q)
    refused(match="seqlen_k is on", seqlen_k=lens_t.cpu())
    refused(RuntimeError, "requires CUDA", q=q.cpu())
    refused(TypeError, max_seqlen_q="10")


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("rows,hkv,group,d,dtype", [([(300, 400), (5, 90)], 2, 2, 128, BF16), ([(260, 260)], 3, 5, 64, F16),
                                                    ([(70, 200)], 2, 4, 256, BF16), ([(9, 300)], 8, 2, 128, F16),
                                                    ([(700, 1700)] * 5, 4, 2, 128, BF16)])
def test_a_value_that_is_not_finite_reaches_its_viewers_only(value, rows, hkv, group, d, dtype):
    """V of a few tokens is not finite: queries that see one of them are not either, the others as if it were 0."""
    window, sinks = 40, 3
    case = _case(rows, hkv, group, d, 16, dtype)
    q, k, v, table, cu, lens = case
    bad = [(b, j) for b, n in enumerate(lens) for j in (10, n // 2, n - 44)]  # the last is in sight of the first queries only
    clean = v.clone()
    for b, j in bad:
        clean[table[b, j // 16], j % 16] = 0
        v[table[b, j // 16], j % 16] = value
    want, bound = chunk_reference(q, k, clean, table, cu, lens, window, sinks)
    got = _run(case, window, sinks)
    sees = torch.zeros(q.shape[0], dtype=torch.bool)
    for b, j in bad:
        for t in range(cu[b], cu[b + 1]):
            i = lens[b] - (cu[b + 1] - t)
            sees[t] |= j <= i and (i - j < window or j < sinks)
    sees = sees.cuda()
    assert 0 < int(sees.sum())
    assert not bool(got[sees].isfinite().any())
    check(got[~sees], want[~sees], bound[~sees])


def test_only_blind_rows_beside_a_value_that_is_not_finite():
    case = _case([(40, 10)], 2, 2, 128, 16, BF16)
    case[2][:] = float("nan")
    assert _run(case, 20, 2)[:30].abs().max() == 0
