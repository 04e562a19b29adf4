"""Attention over 4-bit pages on a B200 (one token per row, and chunks) against a 64-bit softmax.

Tolerance. The cached values enter exactly and so does q (a power of two per column), so what is
lost is: the output's rounding, half an ulp relative; P's rounding to fp16, 2^-11 of each weight;
fp32 scores, whose D products of sum S = sum |q k| scale lose at most D 2^-24 S, here S < 40 and
D <= 256, under 6.2e-4 in the exponent; exp2 and the sums, under 2^-18. The last three change a
result by their total, below 1.2e-3, of the weighted mean of |v|.
"""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu


def _pool(lengths, hkv, d, bs, seed=0, extra=3):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lengths]
    n_blocks = sum(need) + extra
    ids = torch.randperm(n_blocks, generator=g)
    table = torch.zeros(len(lengths), max(max(need, default=0), 1) + 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        table[b, n:] = ids[-1]
        at += n
    # random codes, scales between 2^-3 and 2 (e4m3 bytes 0x20 .. 0x40), NaN scales in unused tokens
    pages = torch.randint(0, 256, (n_blocks, hkv, bs // 16, 18 * d), generator=g, dtype=torch.uint8)
    _, ks, _, vs = ref.places(d)
    for at in (ks, vs):
        shape = (n_blocks, hkv, bs // 16, at.numel())
        pages[..., at.flatten()] = torch.randint(0x20, 0x34, shape, generator=g, dtype=torch.uint8)
    return pages, table


def _poison(pages, table, lengths, bs):
    """NaN scales in every token past its row's end, and in blocks no row uses."""
    d = pages.shape[3] // 18
    _, ks, _, vs = ref.places(d)
    used = torch.zeros(pages.shape[0], bs, dtype=torch.bool)
    for b, n in enumerate(lengths):
        t = torch.arange(n)
        used[table[b].long()[t // bs], t % bs] = True
    for blk, off in (~used).nonzero().tolist():
        pages[blk, :, off // 16, ks[off % 16]] = 0x7f
        pages[blk, :, off // 16, vs[off % 16]] = 0x7f


def _check(got, want, mean):
    err = (got.cpu().double() - want).abs()
    bound = ref.HALF_ULP[got.dtype] * want.abs() + 1.2e-3 * mean + 2.0 ** -25
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound.clamp(min=1e-30)).max()):.3g} times the bound"


def _units(hkv):
    u = torch.ones(2, hkv)
    u[0] = 0.25
    u[1, ::2] = 2.0 ** -5
    return u


@pytest.fixture(params=[1, 2], ids=["warps", "tiles"])
def kernel(request):
    """Runs the test on each chunk kernel, whatever the rule on the counts would choose."""
    from model import _native

    before = _native.get_fp4_prefill_mode()
    _native.set_fp4_prefill_mode(request.param)
    yield request.param
    _native.set_fp4_prefill_mode(before)


DECODE = [
    # lengths, H, H_kv, D, block_size
    ([1], 1, 1, 64, 16),
    ([0, 1, 16, 17, 33], 4, 2, 64, 16),
    ([700], 16, 8, 128, 16),
    ([31, 32, 33, 0, 64, 65, 4], 10, 2, 128, 32),
    ([257, 5, 1030], 8, 2, 256, 16),
    ([100, 200], 24, 1, 128, 64),          # three column blocks
    ([3] * 40 + [0] * 5 + [97] * 20, 3, 1, 64, 16),
    ([2000, 1, 900, 0, 3001], 16, 8, 128, 16),
    ([513], 7, 1, 256, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,heads,hkv,d,bs", DECODE)
def test_decode_matches_the_softmax(cuda_device, dtype, lengths, heads, hkv, d, bs):
    from model.paged_fp4 import paged_decode_fp4

    pages, table = _pool(lengths, hkv, d, bs, seed=len(lengths))
    _poison(pages, table, lengths, bs)
    q = torch.randn(len(lengths), heads, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    units = _units(hkv)
    want, mean = ref.attention(q, pages, table, lengths, [1] * len(lengths), units, d ** -0.5)
    dev = [t.to(cuda_device) for t in (q, pages, table, torch.tensor(lengths, dtype=torch.int32))]
    got = paged_decode_fp4(*dev, units=units.to(cuda_device))
    _check(got, want, mean)
    again = paged_decode_fp4(*dev[:3], dev[3].long(), units=units.to(cuda_device))
    assert torch.equal(got, again), "the same call gives the same bits"


PREFILL = [
    # (chunk, length) per row, H, H_kv, D, block_size
    ([(1, 1)], 1, 1, 64, 16),
    ([(3, 3), (0, 9), (1, 40), (8, 8)], 4, 2, 128, 16),
    ([(5, 300), (2, 2), (7, 64)], 16, 8, 128, 16),
    ([(200, 200), (33, 150), (0, 5), (64, 1000)], 8, 4, 128, 32),
    ([(130, 400), (257, 257)], 6, 2, 64, 16),
    ([(140, 333), (1, 70)], 8, 2, 256, 16),
    ([(90, 513)], 10, 2, 128, 64),
    ([(300, 310)], 1, 1, 256, 32),
    ([(12, 5), (40, 25)], 4, 1, 128, 16),  # queries before the first key see none
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,heads,hkv,d,bs", PREFILL)
def test_chunks_match_the_softmax(cuda_device, kernel, dtype, rows, heads, hkv, d, bs):
    from model.paged_fp4 import paged_prefill_fp4

    chunks, lengths = [c for c, _ in rows], [n for _, n in rows]
    pages, table = _pool(lengths, hkv, d, bs, seed=sum(lengths))
    _poison(pages, table, lengths, bs)
    total = sum(chunks)
    q = torch.randn(total, heads, d, generator=torch.Generator().manual_seed(5)).to(dtype)
    units = _units(hkv)
    want, mean = ref.attention(q, pages, table, lengths, chunks, units, d ** -0.5)
    cu = torch.tensor([sum(chunks[:i]) for i in range(len(chunks) + 1)], dtype=torch.int32)
    dev = [t.to(cuda_device) for t in (q, pages, table, cu, torch.tensor(lengths, dtype=torch.int32))]
    got = paged_prefill_fp4(*dev, max(chunks), units=units.to(cuda_device))
    _check(got, want, mean)
    # a larger announced maximum changes the launch, not the function
    again = paged_prefill_fp4(*dev, max(chunks) + 300, units=units.to(cuda_device))
    _check(again, want, mean)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_rows_and_scales(cuda_device, kernel, d):
    """Scores far apart (one key dominates), a negative and a zero scale, large and tiny q."""
    from model.paged_fp4 import paged_decode_fp4, paged_prefill_fp4

    lengths, heads, hkv, bs = [1500, 40], 4, 2, 16
    pages, table = _pool(lengths, hkv, d, bs, seed=9)
    units = torch.ones(2, hkv)
    g = torch.Generator().manual_seed(1)
    chunks = [150, 40]
    cu = torch.tensor([0, 150, 190], dtype=torch.int32, device=cuda_device)
    seqlen = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    pd, td = pages.to(cuda_device), table.to(cuda_device)
    for factor, scale in ((1.0, -0.02), (1.0, 0.0), (1e4, 1e-5), (2.0 ** -60, 2.0 ** 55), (2.0, 0.02)):
        q = (torch.randn(190, heads, d, generator=g) * factor).to(torch.bfloat16)
        want, mean = ref.attention(q, pages, table, lengths, chunks, units, scale)
        _check(paged_prefill_fp4(q.to(cuda_device), pd, td, cu, seqlen, 150, scale=scale), want, mean)
        want, mean = ref.attention(q[:2], pages, table, lengths, [1, 1], units, scale)
        _check(paged_decode_fp4(q[:2].to(cuda_device), pd, td, seqlen, scale=scale), want, mean)


def test_blocks_outside_the_pool_read_zeros_and_lengths_are_clamped(cuda_device, kernel):
    from model.paged_fp4 import paged_decode_fp4, paged_prefill_fp4

    hkv, d, bs, heads = 2, 128, 16, 4
    pages, table = _pool([96, 96], hkv, d, bs, seed=3)
    clean = torch.cat((pages, torch.zeros_like(pages[:1])))  # a block of zeros stands for the outside ones
    t = table[:, :6].clone()
    bad = t.clone()
    bad[0, 1], bad[0, 4], bad[1, 0] = -1, pages.shape[0], 2 ** 30
    t[0, 1] = t[0, 4] = t[1, 0] = pages.shape[0]
    q = torch.randn(2, heads, d, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    units = torch.ones(2, hkv)
    want, mean = ref.attention(q, clean, t, [96, 96], [1, 1], units, d ** -0.5)
    dev = [x.to(cuda_device) for x in (q, pages, bad)]
    over = torch.tensor([1000, 96], dtype=torch.int32, device=cuda_device)  # capacity is 96
    _check(paged_decode_fp4(*dev, over), want, mean)
    chunk = torch.randn(200, heads, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    want, mean = ref.attention(chunk[:180], clean, t, [96, 96], [90, 90], units, d ** -0.5)
    cu = torch.tensor([0, 90, 180], dtype=torch.int32, device=cuda_device)
    _check(paged_prefill_fp4(chunk[:180].to(cuda_device), dev[1], dev[2], cu, over, 90), want, mean)
    negative = torch.tensor([-5, 0], dtype=torch.int32, device=cuda_device)
    assert (paged_decode_fp4(*dev, negative) == 0).all()


def test_views_streams_workspaces_and_graphs(cuda_device):
    from model.paged_fp4 import fp4_workspace, paged_decode_fp4

    lengths, heads, hkv, d, bs = [1200, 77, 640], 16, 8, 128, 16
    pages, table = _pool(lengths, hkv, d, bs, seed=6)
    units = _units(hkv)
    q = torch.randn(3, heads, d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    want, mean = ref.attention(q, pages, table, lengths, [1] * 3, units, d ** -0.5)
    pd, td, ud = pages.to(cuda_device), table.to(cuda_device), units.to(cuda_device)
    sl = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    wide = torch.zeros(3, heads + 2, d + 8, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 1:-1, :d] = q.to(cuda_device)
    base = paged_decode_fp4(wide[:, 1:-1, :d], pd, td, sl, units=ud)
    _check(base, want, mean)
    off = torch.zeros(3 * heads * d + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(3, heads, d)
    off.copy_(q)  # rows off any 16-byte boundary
    assert torch.equal(paged_decode_fp4(off, pd, td, sl, units=ud), base)
    wide_table = torch.cat((td, td), 1)[:, :td.shape[1]]  # a row stride wider than the table
    strided = torch.stack((sl, sl), 1)[:, 0]
    assert torch.equal(paged_decode_fp4(q.to(cuda_device), pd, wide_table, strided, units=ud), base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_decode_fp4(q.to(cuda_device), pd, td, sl, units=ud)
    side.synchronize()
    assert torch.equal(other, base)
    ws = fp4_workspace(pd)
    out = torch.empty_like(base)
    assert paged_decode_fp4(q.to(cuda_device), pd, td, sl, units=ud, out=out, workspace=ws).data_ptr() == out.data_ptr()
    assert torch.equal(out, base)
    qd = q.to(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = paged_decode_fp4(qd, pd, td, sl, units=ud)
    for _ in range(3):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, base)
    assert torch.equal(paged_decode_fp4(qd, pd, td, sl, units=ud), base)


def test_many_rows_in_one_call(cuda_device, kernel):
    """More rows than one launch takes: row 1100 of 1300 equals the same row alone."""
    from model.paged_fp4 import paged_decode_fp4, paged_prefill_fp4

    n, heads, hkv, d, bs = 1300, 2, 1, 64, 16
    g = torch.Generator().manual_seed(0)
    lengths = torch.randint(0, 60, (n,), generator=g)
    pages, _ = _pool([16 * 64], hkv, d, bs, seed=2)
    table = torch.randint(0, 64, (n, 4), generator=g, dtype=torch.int32)
    q = torch.randn(n, heads, d, generator=g).to(torch.bfloat16)
    dev = [t.to(cuda_device) for t in (q, pages, table, lengths.to(torch.int32))]
    got = paged_decode_fp4(*dev)
    cu = torch.arange(n + 1, dtype=torch.int32, device=cuda_device)
    chunk = paged_prefill_fp4(dev[0], dev[1], dev[2], cu, dev[3], 1)
    pick = [0, 511, 1023, 1024, 1100, 1299]
    want, mean = ref.attention(q[pick], pages, table[pick], lengths[pick].tolist(), [1] * len(pick), torch.ones(2, hkv),
                               d ** -0.5)
    _check(got[pick], want, mean)
    _check(chunk[pick], want, mean)


@pytest.mark.parametrize("n,heads,d", [(897, 8, 128), (1000, 8, 128), (1024, 8, 64), (1024, 8, 256), (2100, 3, 128)])
def test_many_rows_of_wide_groups(cuda_device, n, heads, d):
    """As many rows as a launch takes, or more, at the widest unit (eight columns)."""
    from model.paged_fp4 import paged_decode_fp4

    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 60, (n,), generator=g)
    pages, _ = _pool([16 * 64], 1, d, 16, seed=2)
    table = torch.randint(0, 64, (n, 4), generator=g, dtype=torch.int32)
    q = torch.randn(n, heads, d, generator=g).to(torch.bfloat16)
    got = paged_decode_fp4(*(t.to(cuda_device) for t in (q, pages, table, lengths.to(torch.int32))))
    pick = [0, 600, 895, 896, n - 1]
    want, mean = ref.attention(q[pick], pages, table[pick], lengths[pick].tolist(), [1] * len(pick), torch.ones(2, 1),
                               d ** -0.5)
    _check(got[pick], want, mean)


def test_wait_limit_sets_the_error_word_and_the_next_call_is_right(cuda_device, kernel):
    from model import _native
    from model.paged_fp4 import paged_decode_fp4, paged_prefill_fp4

    lengths, heads, hkv, d, bs = [900, 350], 8, 4, 128, 16
    pages, table = _pool(lengths, hkv, d, bs, seed=8)
    q = torch.randn(400, heads, d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    dev = [t.to(cuda_device) for t in (pages, table, torch.tensor(lengths, dtype=torch.int32))]
    cu = torch.tensor([0, 200, 400], dtype=torch.int32, device=cuda_device)
    qd = q.to(cuda_device)
    units = torch.ones(2, hkv)
    before = _native.get_wait_limit()
    try:
        assert _native.device_error() == 0
        for call in (lambda: paged_decode_fp4(qd[:2], *dev),
                     lambda: paged_prefill_fp4(qd, dev[0], dev[1], cu, dev[2], 200)):
            _native.set_wait_limit(1)  # every wait gives up at once
            call()
            assert _native.device_error() == _native.DEVERR_WAIT_TIMEOUT
            _native.set_wait_limit(0)
            call()
            assert _native.device_error() == 0
    finally:
        _native.set_wait_limit(before)
    want, mean = ref.attention(q[:2], pages, table, lengths, [1, 1], units, d ** -0.5)
    _check(paged_decode_fp4(qd[:2], *dev), want, mean)


def test_the_rule_keeps_short_chunks_on_warps_and_long_ones_on_tiles(cuda_device):
    """Both forms agree within rounding where the default switches, and the default equals one of them."""
    from model import _native
    from model.paged_fp4 import paged_prefill_fp4

    assert _native.get_fp4_prefill_mode() == 0
    hkv, d, bs, heads = 8, 128, 16, 16
    for chunk, expect in ((2, 1), (900, 2)):
        lengths = [chunk + 200] * 4
        pages, table = _pool(lengths, hkv, d, bs, seed=1)
        q = torch.randn(4 * chunk, heads, d, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(cuda_device)
        cu = torch.arange(5, dtype=torch.int32, device=cuda_device) * chunk
        args = (q, pages.to(cuda_device), table.to(cuda_device), cu,
                torch.tensor(lengths, dtype=torch.int32, device=cuda_device), chunk)
        default = paged_prefill_fp4(*args)
        try:
            out = {}
            for mode in (1, 2):
                _native.set_fp4_prefill_mode(mode)
                out[mode] = paged_prefill_fp4(*args)
        finally:
            _native.set_fp4_prefill_mode(0)
        assert torch.equal(default, out[expect]) and not torch.equal(out[1], out[2])
        # two roundings of the output and two of P, of values below four times the mean of |v| here
        assert (out[1].float() - out[2].float()).abs().max() <= 2 * (2.0 ** -8 + 1.2e-3) * float(out[1].float().abs().max() * 4)


@pytest.mark.parametrize("change,match", [
    (dict(q=lambda t: t[0]), "must be"), (dict(q=lambda t: t.float()), "fp16 or bf16"),
    (dict(q=lambda t: t[..., :64]), "head_dim"), (dict(q=lambda t: t[:, :3]), "multiple of n_kv_head"),
    (dict(table=lambda t: t.long()), "int32"), (dict(table=lambda t: t[:1]), "block_table must be"),
    (dict(seqlen=lambda t: t.float()), "int32 or int64"), (dict(seqlen=lambda t: t[:1]), "entries for a batch|block_table"),
    (dict(table=lambda t: t.cpu()), "is on cpu"), (dict(units=lambda t: t[:, :1]), "units must be"),
    (dict(out=lambda t: torch.empty(2, 4, 64)), "out must be"),
    (dict(ws=lambda t: torch.zeros(16, dtype=torch.uint8, device="cuda")), "workspace"),
])
def test_refusals(cuda_device, change, match):
    from model.paged_fp4 import paged_decode_fp4

    a = dict(q=torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=cuda_device),
             pages=torch.zeros(3, 2, 1, 18 * 128, dtype=torch.uint8, device=cuda_device),
             table=torch.zeros(2, 2, dtype=torch.int32, device=cuda_device),
             seqlen=torch.ones(2, dtype=torch.int32, device=cuda_device),
             units=torch.ones(2, 2, device=cuda_device), out=None, ws=None)
    for name, f in change.items():
        a[name] = f(a[name])
    with pytest.raises(ValueError, match=match):
        paged_decode_fp4(a["q"], a["pages"], a["table"], a["seqlen"], units=a["units"], out=a["out"], workspace=a["ws"])
