"""Attention weight sums and the eviction by them against their definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import check, evict_reference, make_pools, weights_reference
from model import _native
from model.paged_evict import evict_tokens, paged_decode_weights
from model.paged_window import paged_decode_window

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LENS = [0, 1, 2, 15, 16, 17, 33, 64, 100, 257, 500, 1023]


def _weights_case(lens, hkv, group, d, bs, dtype, seed=0, extra=0):
    gen = torch.Generator().manual_seed(seed)
    k, v, table, _ = make_pools(lens, hkv, d, bs, dtype, gen=gen)
    q = torch.randn(len(lens), hkv * group, d, generator=gen).to(dtype).cuda()
    w = torch.rand(len(lens), hkv, table.shape[1] * bs + extra, generator=gen).cuda()
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), w


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hkv,group,d,bs", [(8, 2, 128, 16), (2, 4, 256, 32), (4, 1, 64, 16), (1, 8, 128, 16), (3, 5, 64, 64),
                                            (4, 3, 128, 8), (2, 16, 64, 16), (2, 9, 64, 16), (8, 2, 16, 16), (2, 3, 8, 8)])
def test_weights(dtype, hkv, group, d, bs):
    q, k, v, table, seqlen, w = _weights_case(LENS, hkv, group, d, bs, dtype, extra=3)
    out, bound, sums, off = weights_reference(q, k, v, table, LENS, w)
    got = paged_decode_weights(q, k, v, table, seqlen, w)
    check(got, out, bound)
    check(w, sums, off)
    assert _native.device_error() == 0


@pytest.mark.parametrize("rows,length", [(1, 5000), (40, 3000), (150, 300), (12, 900), (24, 400), (35, 700)])
def test_weights_of_many_and_long_rows(rows, length):
    gen = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, length + 1, (rows,), generator=gen).tolist()
    lens[0] = length
    q, k, v, table, seqlen, w = _weights_case(lens, 8, 2, 128, 16, BF16, seed=1)
    before = w.clone()
    for _ in range(2):
        w.copy_(before)
        out, bound, sums, off = weights_reference(q, k, v, table, lens, w)
        check(paged_decode_weights(q, k, v, table, seqlen, w), out, bound)
        check(w, sums, off)


@pytest.mark.parametrize("rows", [9000, 70000])
def test_more_rows_than_a_launch_takes(rows):
    """One block a row: decode over a window and with weights in several launches, and eviction of every row."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    d, bs, group, blocks = 64, 16, 2, 300
    k, v = (torch.randn(blocks, bs, 1, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
    table = torch.randint(0, blocks, (rows, 1), generator=gen, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, bs + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    q = torch.randn(rows, group, d, generator=gen, device="cuda").to(BF16)
    w = torch.zeros(rows, 1, bs, device="cuda")
    j = torch.arange(bs, device="cuda")
    s = torch.einsum("bhd,bjd->bhj", q.double(), k[table[:, 0].long(), :, 0].double()) * d ** -0.5
    vv = v[table[:, 0].long(), :, 0].double()
    size = float(torch.einsum("bhd,bjd->bhj", q.abs().double(), k[table[:, 0].long(), :, 0].abs().double()).max()) * d ** -0.5
    rel = 2.0 ** -16 + 2.0 ** -20 + 2 * (d + 4) * 2.0 ** -24 * size + 2 * bs * 2.0 ** -24
    for window in (None, 5):
        seen = (j < lens[:, None]) & (j >= (lens[:, None] - window if window else 0))
        p = s.masked_fill(~seen[:, None], float("-inf")).softmax(-1).nan_to_num(0.0)
        out = paged_decode_weights(q, k, v, table, lens, w) if window is None else paged_decode_window(q, k, v, table, lens, 5)
        check(out, torch.einsum("bhj,bjd->bhd", p, vv), rel * torch.einsum("bhj,bjd->bhd", p, vv.abs()))
        if window is None:
            check(w[:, 0], p.sum(1), rel * p.sum(1))
    # every row its own block
    own = torch.arange(rows, device="cuda", dtype=torch.int32)[:, None]
    kk, vv = (torch.randn(rows, bs, 1, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
    sums = torch.rand(1, rows, 1, bs, generator=gen, device="cuda")
    old = kk.clone()
    left, kept = evict_tokens([kk], [vv], own, lens, sums, 6, recent=1, sinks=1)
    assert torch.equal(left, lens.clamp(max=6))
    cut = lens > 6
    middle = sums[0, :, 0].masked_fill((j < 1) | (j >= lens[:, None] - 1), -1.0)
    places = middle[cut].topk(4, -1).indices.sort(-1).values
    places = torch.cat((torch.zeros_like(places[:, :1]), places, lens[cut, None].long() - 1), 1)
    assert torch.equal(kept[0, cut, 0, :6], sums[0, cut, 0].gather(1, places))
    assert torch.equal(kk[cut, :6, 0], old[cut, :, 0].gather(1, places[..., None].expand(-1, -1, d)))
    assert torch.equal(kk[~cut], old[~cut]) and _native.device_error() == 0


def test_weights_beside_others():
    """A step's weights sum to the group; what lies past a row stays; strided sums; graphs and streams."""
    lens = [300, 0, 1, 77]
    q, k, v, table, seqlen, w = _weights_case(lens, 4, 2, 128, 16, BF16)
    store = torch.full((4, 2, 4, w.shape[2]), 7.0, device="cuda")
    mine = store[:, 1]
    mine.zero_()
    out = paged_decode_weights(q, k, v, table, seqlen, mine)
    assert bool((store[:, 0] == 7).all())
    for b, n in enumerate(lens):
        assert bool((mine[b, :, n:] == 0).all())
        if n:  # n terms, each off by 2^-20 of itself at most
            assert (mine[b].double().sum(-1) - 2).abs().max().item() <= 2 * 2.0 ** -14
    g = torch.cuda.CUDAGraph()
    again = torch.zeros_like(w)
    with torch.cuda.graph(g):
        captured = paged_decode_weights(q, k, v, table, seqlen, again)
    again.zero_()
    for _ in range(3):
        g.replay()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    third = torch.zeros_like(w)
    with torch.cuda.stream(other):
        for _ in range(3):
            paged_decode_weights(q, k, v, table, seqlen, third)
    torch.cuda.synchronize()
    assert torch.equal(captured, out) and torch.equal(again, third)


@pytest.mark.parametrize("lens", [[900], [300, 0] * 12, [700, 0, 33] * 30])
def test_a_wait_that_runs_out_is_reported(lens):
    """Under the test limit every wait gives up at once: the flag is set, the kernels return, the next call is right."""
    q, k, v, table, seqlen, w = _weights_case(lens, 8, 2, 128, 16, BF16)
    before = w.clone()
    limit = _native.get_wait_limit()
    try:
        _native.set_wait_limit(10)
        paged_decode_weights(q, k, v, table, seqlen, w)
        torch.cuda.synchronize()
        assert _native.device_error(clear=True) & _native.DEVERR_WAIT_TIMEOUT
    finally:
        _native.set_wait_limit(limit)
    w.copy_(before)
    out, bound, sums, off = weights_reference(q, k, v, table, lens, w)
    check(paged_decode_weights(q, k, v, table, seqlen, w), out, bound)
    check(w, sums, off)
    assert _native.device_error() == 0


def test_weights_of_nan_past_the_row():
    lens = [100, 3]
    q, k, v, table, seqlen, w = _weights_case(lens, 4, 2, 128, 16, BF16)
    out, bound, sums, off = weights_reference(q, k, v, table, lens, w)
    for b, n in enumerate(lens):
        k[table[b, n // 16], n % 16:] = float("nan")
        v[table[b, n // 16], n % 16:] = float("nan")
    check(paged_decode_weights(q, k, v, table, seqlen, w), out, bound)
    check(w, sums, off)


# --------------------------------------------------------------------------- eviction


def _evict_case(lens, layers, hkv, d, bs, dtype, seed=0, ties=False, keep=8):
    gen = torch.Generator().manual_seed(seed)
    width = max(1, -(-min(keep, max(lens)) // bs))
    made = [make_pools(lens, hkv, d, bs, dtype, gen=torch.Generator().manual_seed(seed), spare=width * len(lens) + 3)
            for _ in range(layers)]
    table, free = made[0][2], made[0][3]
    ks = [(torch.randn(m[0].shape, generator=gen)).to(dtype).cuda() for m in made]
    vs = [(torch.randn(m[1].shape, generator=gen)).to(dtype).cuda() for m in made]
    w = torch.rand(layers, len(lens), hkv, table.shape[1] * bs, generator=gen)
    if ties:
        w = torch.randint(0, 3, w.shape, generator=gen).float()
    new = free[:width * len(lens)].view(len(lens), width).contiguous()
    return ks, vs, table, torch.tensor(lens, dtype=torch.int32).cuda(), w.cuda(), new


def _check_evicted(case, lens, keep, recent, sinks, fresh=False, in_place=False):
    ks, vs, table, seqlen, w, new = case
    kept = evict_reference(w, lens, keep, recent, sinks)
    old_k, old_v, old_w = [x.clone() for x in ks], [x.clone() for x in vs], w.clone()
    more = dict(seqlen_out=seqlen, weights_out=w) if in_place else {}
    n, sums = evict_tokens(ks, vs, table, seqlen, w, keep, recent=recent, sinks=sinks, new_table=new if fresh else None, **more)
    if in_place:
        assert n.data_ptr() == seqlen.data_ptr() and sums.data_ptr() == w.data_ptr()
    else:
        assert torch.equal(w, old_w) or bool(w.isnan().any())
    assert n.tolist() == [min(x, keep) for x in lens]
    bs = ks[0].shape[1]
    target = new if fresh else table
    for x, old in ((ks, old_k), (vs, old_v)):
        for layer in range(len(x)):
            want = old[layer].clone()
            for (la, b, h), tokens in kept.items():
                if la == layer and tokens:
                    src = torch.tensor(tokens, device="cuda")
                    dst = torch.arange(len(tokens), device="cuda")
                    want[target[b].long()[dst // bs], dst % bs, h] = old[layer][table[b].long()[src // bs], src % bs, h]
            assert torch.equal(x[layer].view(torch.uint8), want.view(torch.uint8))
    want = torch.zeros_like(old_w)
    for (layer, b, h), tokens in kept.items():
        want[layer, b, h, :len(tokens)] = old_w[layer, b, h, tokens]
    assert torch.equal(sums.view(torch.int32), want.view(torch.int32))
    assert _native.device_error() == 0


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (16, 4, 2), (33, 0, 0), (33, 33, 0), (33, 0, 33),
                                               (64, 30, 34), (100, 10, 4), (500, 100, 1), (5000, 10, 10)])
def test_budgets(fresh, keep, recent, sinks):
    _check_evicted(_evict_case(LENS, 2, 4, 64, 16, BF16, keep=keep), LENS, keep, recent, sinks, fresh)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layers,hkv,d,bs,dtype", [(1, 8, 128, 16, BF16), (3, 2, 256, 32, F16), (2, 3, 64, 64, F32),
                                                   (2, 5, 8, 8, BF16), (1, 1, 256, 1, F32), (65, 2, 16, 16, F16)])
def test_heads_and_layers(in_place, layers, hkv, d, bs, dtype):
    lens = [0, 40, 41, 200, 999] if layers < 10 else [5, 60]
    _check_evicted(_evict_case(lens, layers, hkv, d, bs, dtype, seed=2, keep=40), lens, 40, 7, 3, in_place=in_place)


@pytest.mark.parametrize("length", [3000, 9000, 40000])
def test_long_rows(length):
    lens = [length, length // 2, 10]
    for fresh in (False, True):
        _check_evicted(_evict_case(lens, 1, 2, 64, 32, F16, seed=3, keep=1001), lens, 1001, 32, 16, fresh)


def test_ties_keep_the_lower_index():
    lens = [50, 300, 3000]
    _check_evicted(_evict_case(lens, 2, 2, 64, 16, BF16, seed=4, ties=True, keep=37), lens, 37, 5, 2)
    case = _evict_case(lens, 1, 2, 64, 16, BF16, seed=5, keep=37)
    case[4].zero_()
    _check_evicted(case, lens, 37, 5, 2)


def test_odd_weights():
    """Infinities, NaN, negative values and both zeros have their place in the order."""
    lens = [64, 200]
    case = _evict_case(lens, 1, 2, 64, 16, BF16, seed=6, keep=30)
    w = case[4]
    odd = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38], device="cuda")
    w.copy_(odd[torch.randint(0, 9, w.shape, generator=torch.Generator().manual_seed(1)).cuda()])
    _check_evicted(case, lens, 30, 2, 1)
    w.fill_(float("nan"))
    case[3].copy_(torch.tensor(lens, dtype=torch.int32))
    _check_evicted(case, lens, 30, 2, 1)


def test_pools_in_one_tensor_other_types_and_graphs():
    lens, keep = [100, 20, 300], 32
    ks, vs, table, seqlen, w, new = _evict_case(lens, 2, 2, 64, 16, BF16, seed=7, keep=keep)
    both = torch.stack([torch.stack((k, v), 3) for k, v in zip(ks, vs)])  # (layer, n, bs, h, 2, d)
    first = both.clone()
    views = [x[..., 0, :] for x in both], [x[..., 1, :] for x in both]
    wide = torch.full((3, 2 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    _check_evicted((*views, wide[:, ::2], seqlen, w, new), lens, keep, 4, 1)
    done = both.clone()
    # a captured eviction, replayed on the same state
    n, sums = torch.empty_like(seqlen), torch.empty_like(w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        evict_tokens(*views, table, seqlen.long(), w, keep, recent=4, sinks=1, seqlen_out=n, weights_out=sums)
    both.copy_(first)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(both, done) and n.tolist() == [32, 20, 32]


def test_bad_blocks_are_skipped_and_reported():
    lens = [60, 60]
    ks, vs, table, seqlen, w, new = _evict_case(lens, 1, 2, 64, 16, BF16, seed=8, keep=20)
    kept = evict_reference(w, lens, 20, 0, 0)
    before = ks[0].clone()
    good = table.clone()
    table[0, 3], table[1, 1] = 10 ** 6, -1
    evict_tokens(ks, vs, table, seqlen, w, 20)
    assert _native.device_error(clear=True) == _native.DEVERR_COPY_RANGE
    want = before.clone()
    for (_, b, h), tokens in kept.items():
        for r, t in enumerate(tokens):
            if (b, t // 16) not in ((0, 3), (1, 1)) and (b, r // 16) not in ((0, 3), (1, 1)):
                want[good[b, r // 16], r % 16, h] = before[good[b, t // 16], t % 16, h]
    assert torch.equal(ks[0], want)
    assert _native.device_error() == 0


def test_steps_of_a_bounded_row():
    """Decode steps with sums, evicted whenever the row passes its budget: the cache holds the tokens that a
    host model of it holds, and attends over exactly those."""
    gen = torch.Generator().manual_seed(9)
    hkv, group, d, bs, keep, recent, sinks = 2, 2, 64, 16, 40, 8, 2
    blocks, width = 12, 4
    k = torch.zeros(blocks, bs, hkv, d, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.randperm(blocks, generator=gen)[:width].view(1, width).to(torch.int32).cuda()
    w = torch.zeros(1, 1, hkv, width * bs, device="cuda")
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    length = 0
    rows = {h: [] for h in range(hkv)}  # (key, value) of the host model
    for step in range(150):
        kn, vn = (torch.randn(hkv, d, generator=gen).to(BF16) for _ in range(2))
        at = int(table[0, length // bs])
        k[at, length % bs], v[at, length % bs] = kn.cuda(), vn.cuda()
        for h in range(hkv):
            rows[h].append((kn[h].double(), vn[h].double()))
        length += 1
        n.fill_(length)
        q = torch.randn(1, hkv * group, d, generator=gen).to(BF16)
        out, bound, sums, off = weights_reference(q.cuda(), k, v, table, [length], w[0])
        got = paged_decode_weights(q.cuda(), k, v, table, n, w[0])
        check(got, out, bound)
        check(w[0], sums, off)
        for h in range(hkv):
            kk, vv = (torch.stack([r[i] for r in rows[h]]) for i in (0, 1))
            p = (q[0, h * group:(h + 1) * group].double() @ kk.T / d ** 0.5).softmax(-1)
            # half a step of results below 4, and the weights' error of at most 2^-9 of values below 4
            assert (got[0, h * group:(h + 1) * group].cpu().double() - p @ vv).abs().max().item() <= 2.0 ** -8 * 4
        if length == width * bs:
            exact = w.clone()
            evict_tokens([k], [v], table, n, w, keep, recent=recent, sinks=sinks, seqlen_out=n, weights_out=w)
            kept = evict_reference(exact, [length], keep, recent, sinks)
            for h in range(hkv):
                rows[h] = [rows[h][j] for j in kept[0, 0, h]]
            length = keep
            assert n.item() == keep
    assert length < width * bs


def test_refusals():
    lens = [100, 40]
    ks, vs, table, seqlen, w, new = _evict_case(lens, 2, 2, 64, 16, BF16, keep=32)
    q = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")

    def refused(error=ValueError, match=None, **change):
        args = dict(k_caches=ks, v_caches=vs, block_table=table, seqlen=seqlen, weights=w, keep=32)
        args.update(change)
        with pytest.raises(error, match=match):
            evict_tokens(**args)

    refused(match="keep must be", keep=0)
    refused(match="fit into keep", recent=20, sinks=13)
    refused(match="at least 0", recent=-1)
    refused(match="per layer", k_caches=ks[:1])
    refused(match="one k_cache", k_caches=[], v_caches=[])
    refused(match="one shape", k_caches=[ks[0], ks[1][:-1]], v_caches=vs)
    refused(match="weights must be", weights=w[:1])
    refused(match="weights must be", weights=w[..., :8])
    refused(match="weights must be", weights=w.double())
    refused(match="unit last stride", weights=w.transpose(2, 3).contiguous().transpose(2, 3))
    refused(match="new_table holds", new_table=new[:, :1])
    refused(match="new_table must be", new_table=new[:1])
    refused(match="seqlen_out", seqlen_out=seqlen.long())
    refused(match="weights_out must be", weights_out=w[..., :-1])
    refused(match="must not overlap", weights=w[:1].expand(2, -1, -1, -1), weights_out=w[:1].expand(2, -1, -1, -1))
    room = torch.zeros(w.numel() + 4, device="cuda")
    refused(match="not as weights itself", weights=room[:w.numel()].view(w.shape), weights_out=room[4:].view(w.shape))
    refused(match="named twice", k_caches=[ks[0], ks[0]])
    refused(match="named twice", v_caches=[vs[0], ks[1]])
    refused(match="int32", block_table=table.long())
    refused(RuntimeError, "requires CUDA", k_caches=[x.cpu() for x in ks], v_caches=vs)
    refused(match="seqlen is on", seqlen=seqlen.cpu())

    def refused_step(error=ValueError, match=None, **change):
        args = dict(q=q, k_cache=ks[0], v_cache=vs[0], block_table=table, seqlen=seqlen, weights=w[0])
        args.update(change)
        with pytest.raises(error, match=match):
            paged_decode_weights(**args)

    refused_step(match="weights must be", weights=w)
    refused_step(match="weights must be", weights=w[0, :, :, :10])
    refused_step(match="weights must be", weights=w[0].half())
    refused_step(match="must not overlap", weights=w[0, :1].expand(2, -1, -1))
    refused_step(match="unit last stride", weights=w[0].transpose(1, 2).contiguous().transpose(1, 2))
    refused_step(match="weights is on", weights=w[0].cpu())
    refused_step(match="q must be", q=q[0])
