"""Decode with a sliding window and sinks against its definition in 64 bits (tolerances: bounded_reference.attend)."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import check, chunk_reference, make_pools
from model import _native
from model.paged_window import decode_workspace, paged_decode_window, paged_prefill_window
from model.triton_decode import paged_decode_plan

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _case(lens, hkv, group, d, bs, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    k, v, table, _ = make_pools(lens, hkv, d, bs, dtype, gen=gen)
    q = torch.randn(len(lens), hkv * group, d, generator=gen).to(dtype).cuda()
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda()


def _check(lens, hkv, group, d, bs, dtype, window, sinks, seed=0):
    q, k, v, table, seqlen = _case(lens, hkv, group, d, bs, dtype, seed)
    got = paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks)
    want, bound = chunk_reference(q, k, v, table, list(range(len(lens) + 1)), lens, window, sinks)
    check(got, want, bound)
    assert _native.device_error() == 0


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 257, 500, 1023]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (16, 0), (16, 16), (17, 15), (33, 4), (64, 32), (100, 0),
                                          (255, 1), (1000, 100), (5000, 0), (1 << 40, 1 << 40), (7, 2000)])
def test_windows(window, sinks):
    _check(LENS, 8, 2, 128, 16, BF16, window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hkv,group,d,bs", [(2, 4, 256, 32), (4, 1, 64, 16), (1, 8, 128, 16), (3, 5, 64, 64), (4, 3, 128, 8),
                                            (2, 6, 128, 16), (1, 7, 256, 16), (2, 9, 64, 16), (8, 2, 16, 16), (2, 3, 8, 8),
                                            (1, 16, 64, 1), (5, 2, 128, 4), (2, 12, 128, 128)])
def test_heads_and_blocks(dtype, hkv, group, d, bs):
    _check(LENS, hkv, group, d, bs, dtype, 37, 5, seed=1)
    _check([0, 700, 3], hkv, group, d, bs, dtype, 300, 0, seed=2)


@pytest.mark.parametrize("rows,length,window,sinks", [(1, 5000, 1024, 4), (1, 5000, 3, 0), (40, 3000, 700, 9), (150, 300, 64, 1),
                                                       (12, 1000, 500, 4), (24, 400, 1 << 20, 0), (33, 700, 400, 20)])
def test_long_and_many(rows, length, window, sinks):
    gen = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, length + 1, (rows,), generator=gen).tolist()
    lens[0] = length
    _check(lens, 8, 2, 128, 16, BF16, window, sinks, seed=3)
    _check(lens[:20], 2, 4, 256, 32, F16, window, sinks, seed=4)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 256), (F32, 64), (BF16, 32)])
def test_hidden_tokens_may_hold_anything(dtype, d):
    """NaN and infinities in hidden tokens, in tokens past the row and in unused blocks leave no trace."""
    lens, window, sinks = [400, 33, 90, 7], 50, 6
    q, k, v, table, seqlen = _case(lens, 4, 2, d, 16, dtype)
    want, bound = chunk_reference(q, k, v, table, list(range(5)), lens, window, sinks)
    bad = torch.full((2, *k.shape[:2]), True, device="cuda")
    for b, n in enumerate(lens):
        for j in range(n):
            if j < sinks or n - 1 - j < window:
                bad[:, table[b, j // 16], j % 16] = False
    k[bad[0]] = float("nan")
    v[bad[1]] = float("nan")
    v[bad[1].nonzero(as_tuple=True)[0][:1]] = v[bad[1].nonzero(as_tuple=True)[0][:1]].clone()
    got = paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks)
    check(got, want, bound)
    v[bad[1]] = float("inf")
    check(paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks), want, bound)


def test_hidden_pages_are_not_looked_up():
    """Entries of pages without a visible token may be anything, ids outside the pool among them."""
    lens, window, sinks = [2000, 1500], 100, 5
    q, k, v, table, seqlen = _case(lens, 8, 2, 128, 16, BF16)
    want = paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks)
    for b, n in enumerate(lens):
        table[b, 1:(n - window) // 16] = 0x7fffffff
        table[b, -(-n // 16):] = -5
    assert torch.equal(paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks), want)


def test_a_window_over_the_row_is_paged_decode():
    """Both are within the bound of the definition; their sums are split differently, so not bit for bit."""
    from model.triton_decode import paged_decode

    q, k, v, table, seqlen = _case(LENS, 8, 2, 128, 16, BF16)
    want, bound = chunk_reference(q, k, v, table, list(range(len(LENS) + 1)), LENS, 1023, 0)
    check(paged_decode_window(q, k, v, table, seqlen, 1023), want, bound)
    check(paged_decode(q, k, v, table, seqlen), want, bound)


def test_strides_types_and_outputs():
    lens, window, sinks = [100, 40, 0, 333], 64, 3
    q, k, v, table, seqlen = _case(lens, 4, 2, 128, 16, BF16)
    want = paged_decode_window(q, k, v, table, seqlen, window, sinks=sinks, scale=0.2)
    ref, bound = chunk_reference(q, k, v, table, list(range(5)), lens, window, sinks, 0.2)
    check(want, ref, bound)
    # a view of a fused projection, an unaligned copy, a transposed one
    fused = torch.zeros(4, 16, 128, dtype=BF16, device="cuda")
    fused[:, 3:11] = q
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    turned = q.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for x in (fused[:, 3:11], odd, turned):
        assert torch.equal(paged_decode_window(x, k, v, table, seqlen, window, sinks=sinks, scale=0.2), want)
    # int64 lengths, a table with other strides, pools inside a larger tensor
    wide = torch.full((4, 3 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::3] = table
    big = torch.stack((k, v), 3)  # (n, bs, h, 2, d)
    out = torch.empty_like(q)
    got = paged_decode_window(q, big[..., 0, :], big[..., 1, :], wide[:, ::3], seqlen.long(), window, sinks=sinks, scale=0.2,
                              out=out, workspace=decode_workspace(4, 8, 4, 128, q))
    assert got is out or got.data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    # lengths beyond the table are cut to it, negative ones are empty
    full = torch.tensor([10 ** 6, -3, 0, 333], dtype=torch.int32, device="cuda")
    ref, bound = chunk_reference(q, k, v, table, list(range(5)), [table.shape[1] * 16, 0, 0, 333], window, sinks)
    check(paged_decode_window(q, k, v, table, full, window, sinks=sinks), ref, bound)


def test_streams_and_graphs():
    """Calls on two streams, two captured graphs replayed side by side with eager calls: one result."""
    cases = [_case([900 + 40 * i, 17, 3000], 8, 2, 128, 16, BF16, seed=i) for i in range(3)]
    want = [paged_decode_window(*c, 512, sinks=4) for c in cases]
    graphs, outs = [], []
    for c in cases[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged_decode_window(*c, 512, sinks=4))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = paged_decode_window(*cases[2], 512, sinks=4)
    torch.cuda.synchronize()
    for got, ref in zip([*outs, eager], want):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("lens,hkv,group,d,dtype", [([900], 8, 2, 128, BF16), ([300] * 9, 2, 4, 64, F16), ([300, 0] * 12, 8, 2, 128, BF16),
                                                    ([900, 5, 300] * 20, 8, 2, 128, BF16)])
def test_a_wait_that_runs_out_is_reported(lens, hkv, group, d, dtype):
    """Under the test limit every wait gives up at once: the flag is set, the kernel returns, the next call is right."""
    case = _case(lens, hkv, group, d, 16, dtype)
    want = paged_decode_window(*case, 700, sinks=4)
    limit = _native.get_wait_limit()
    try:
        _native.set_wait_limit(10)
        paged_decode_window(*case, 700, sinks=4)
        torch.cuda.synchronize()
        assert _native.device_error(clear=True) & _native.DEVERR_WAIT_TIMEOUT
    finally:
        _native.set_wait_limit(limit)
    for _ in range(2):  # the workspace that the call left
        assert torch.equal(paged_decode_window(*case, 700, sinks=4), want)
    assert _native.device_error() == 0


@pytest.mark.parametrize("rows", [1, 40])
def test_what_a_kernel_two_back_wrote(rows):
    """A plan whose launches overlap reads lengths and pools early: the call between it and the kernel that wrote
    them lets it in only when that kernel is through."""
    q, k, v, table, seqlen = _case([900] * rows, 8, 2, 128, 16, BF16)
    other = _case([60], 8, 2, 128, 16, BF16, seed=9)
    plan = paged_decode_plan(q, [k], [v], table, seqlen, window=300, sinks=4)
    values = [torch.randn(v.shape, dtype=BF16, device="cuda") for _ in range(4)]
    lens = [torch.full_like(seqlen, n) for n in (900, 333, 1, 600)]
    want = [chunk_reference(q, k, x, table, list(range(rows + 1)), n.tolist(), 300, 4) for x, n in zip(values, lens)]
    cu, mid = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), []
    between = [lambda: paged_decode_window(*other, 20),
               lambda: paged_prefill_window(other[0], *other[1:4], cu, other[4], 1, 20),
               lambda: paged_decode_window(q, k, v, table, seqlen, 300, sinks=4)]
    for call in between:
        for x, n, ref in zip(values, lens, want):  # nothing waits in here for the device
            v.copy_(x)
            seqlen.copy_(n)
            call()
            mid.append((plan.run(0, q, overlap=True), ref))
    for got, ref in mid:
        check(got, *ref)


def test_empty_batch_and_table():
    q = torch.zeros(0, 16, 128, dtype=BF16, device="cuda")
    k = torch.zeros(4, 16, 8, 128, dtype=BF16, device="cuda")
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    assert paged_decode_window(q, k, k, none, none[:, 0], 8).shape == (0, 16, 128)
    q = torch.ones(2, 16, 128, dtype=BF16, device="cuda")
    table = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    lens = torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    assert paged_decode_window(q, k, k, table, lens, 8).abs().max() == 0


def test_refusals():
    q, k, v, table, seqlen = _case([100, 40], 4, 2, 128, 16, BF16)

    def refused(error=ValueError, match=None, **change):
        args = dict(q=q, k_cache=k, v_cache=v, block_table=table, seqlen=seqlen, window=8)
        args.update(change)
        with pytest.raises(error, match=match):
            paged_decode_window(**args)

    refused(match="window must be", window=0)
    refused(match="sinks must be", sinks=-1)
    refused(match="q must be", q=q[0])
    refused(match="share one dtype", q=q.half())
    refused(match="share one dtype", v_cache=v.half())
    refused(match="head_dim", q=q[..., :64])
    refused(match="multiple of n_kv_head", q=q[:, :6])
    refused(match="shapes differ", v_cache=v[:-1])
    refused(match="block_table must be int32", block_table=table.long())
    refused(match="block_table must be", block_table=table[:1])
    refused(match="seqlen must be", seqlen=seqlen[:1])
    refused(match="seqlen must be int32", seqlen=seqlen.float())
    refused(match="power of two", k_cache=k[:, :12], v_cache=v[:, :12])
    refused(match="multiple of 128 bytes", q=q[..., :8], k_cache=torch.zeros(9, 4, 4, 8, dtype=BF16, device="cuda"),
            v_cache=torch.zeros(9, 4, 4, 8, dtype=BF16, device="cuda"))
    refused(match="unit head_dim stride", k_cache=k.transpose(1, 3).contiguous().transpose(1, 3))
    refused(match="out must be", out=torch.empty_like(q).half())
    refused(match="workspace must be", workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    refused(RuntimeError, "requires CUDA", q=q.cpu())
    refused(RuntimeError, "requires CUDA", k_cache=k.cpu())
    refused(match="seqlen is on", seqlen=seqlen.cpu())
    refused(match="block_table is on", block_table=table.cpu())
    refused(TypeError, window="8")
