"""The containers of a cache of bounded length, as a serving loop uses them: prompts in chunks, captured steps with a
window, steps that keep attention weights with evictions between them. Tolerances: bounded_reference.attend."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import check, chunk_reference, evict_reference, weights_reference
from model import _native
from model.paged import PagedKV, PagedPool
from model.paged_evict import evict_tokens, paged_decode_weights
from model.paged_window import paged_decode_window, paged_prefill_window
from serve.block_manager import BlockManager
from serve.graph import PagedStepGraph

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _pool(n_layer, blocks, hkv, d, n_head, bs=16):
    return PagedPool(n_layer, blocks, bs, hkv, d, dtype=BF16, device="cuda", n_head=n_head)


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen).to(BF16).cuda()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("hkv,group,d", [(8, 2, 128), (2, 5, 64), (2, 4, 256)])
def test_windowed_prompts_and_steps(captured, hkv, group, d):
    """Prompts written and attended in chunks, then steps through the container, eager with overlapped layers or
    replayed: every output against its definition over what was written."""
    gen = torch.Generator().manual_seed(1)
    layers, bs, window, sinks, steps = 3, 16, 50, 5, 40
    heads, prompts = hkv * group, [130, 3, 60]
    pool = _pool(layers, 64, hkv, d, heads)
    manager = BlockManager(64, bs)
    tables = [manager.reserve(-(-(n + steps) // bs)) for n in prompts]
    width = max(len(t) for t in tables)
    table = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32).cuda()
    # prompts in chunks of at most 48 tokens
    for start in range(0, max(prompts), 48):
        ends = [min(n, start + 48) for n in prompts]
        counts = [max(e - start, 0) for e in ends]
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        slots = torch.tensor([tables[b][t // bs] * bs + t % bs for b, e in enumerate(ends) for t in range(start, e)]).cuda()
        for layer in range(layers):
            pool.write_slots(layer, slots, _rand(gen, cu[-1], hkv, d), _rand(gen, cu[-1], hkv, d))
            q = _rand(gen, cu[-1], heads, d)
            lens = [e if c else 0 for e, c in zip(ends, counts)]
            got = paged_prefill_window(q, pool.keys[layer], pool.values[layer], table, torch.tensor(cu).cuda(),
                                       torch.tensor(lens).cuda(), 48, window, sinks=sinks)
            want, bound = chunk_reference(q, pool.keys[layer], pool.values[layer], table, cu, lens, window, sinks)
            check(got, want, bound)
    kv = PagedKV(pool, tables, prompts, rope_len=1000, n_head=heads, window=window, sinks=sinks)
    shape = (layers, len(prompts), hkv, 1, d)
    q, k, v = _rand(gen, layers, len(prompts), heads, 1, d), _rand(gen, *shape), _rand(gen, *shape)
    graph = PagedStepGraph(kv, q, k, v) if captured else None
    for step in range(steps):
        q.copy_(_rand(gen, *q.shape))
        k.copy_(_rand(gen, *shape))
        v.copy_(_rand(gen, *shape))
        if captured:
            out = graph.replay()
        else:
            kv.build_mask(next_token=True)
            out = []
            for layer in range(layers):
                kv.write(layer, k[layer], v[layer])
                out.append(kv.attend(layer, q[layer]))
            kv.advance()
        lens = [n + step + 1 for n in prompts]
        if step % 13 and step != steps - 1:
            continue
        for layer in range(layers):
            want, bound = chunk_reference(q[layer, :, :, 0], pool.keys[layer], pool.values[layer], table,
                                          list(range(len(prompts) + 1)), lens, window, sinks)
            check(out[layer][:, :, 0], want, bound)
    # the blocks that the container calls hidden may hold anything from now on
    hidden = kv.hidden_blocks()
    first = [n + steps + 1 - window for n in prompts]
    assert [len(h) for h in hidden] == [max(0, f // bs - 1) for f in first] and sum(map(len, hidden)) > 0
    for row, blocks in enumerate(hidden):
        assert blocks == tables[row][1:1 + len(blocks)]
        for layer in range(layers):
            pool.keys[layer][blocks] = float("nan")
            pool.values[layer][blocks] = float("nan")
    kv.build_mask(next_token=True)
    kv.write(0, k[0], v[0])
    out = kv.attend(0, q[0])
    assert bool(out.isfinite().all())
    assert _native.device_error() == 0


@pytest.mark.parametrize("seed", range(6))
def test_captured_layers_that_overlap(seed):
    """Every step of overlapped captured layers, each of which may read the split that the layer before it is still
    recording."""
    gen = torch.Generator().manual_seed(seed)
    layers, bs, hkv, heads, d, window, sinks, steps = 3, 16, 2, 8, 256, 50, 5, 40
    prompts = [130, 3, 60]
    pool = _pool(layers, 64, hkv, d, heads)
    manager = BlockManager(64, bs)
    tables = [manager.reserve(-(-(n + steps) // bs)) for n in prompts]
    width = max(len(t) for t in tables)
    table = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32).cuda()
    slots = torch.tensor([tables[b][t // bs] * bs + t % bs for b, n in enumerate(prompts) for t in range(n)]).cuda()
    for layer in range(layers):
        pool.write_slots(layer, slots, _rand(gen, len(slots), hkv, d), _rand(gen, len(slots), hkv, d))
    kv = PagedKV(pool, tables, prompts, rope_len=1000, n_head=heads, window=window, sinks=sinks)
    shape = (layers, len(prompts), hkv, 1, d)
    q, k, v = _rand(gen, layers, len(prompts), heads, 1, d), _rand(gen, *shape), _rand(gen, *shape)
    graph = PagedStepGraph(kv, q, k, v)
    for step in range(steps):
        for x in (q, k, v):
            x.copy_(_rand(gen, *x.shape))
        out = graph.replay()
        lens = [n + step + 1 for n in prompts]
        for layer in range(layers):
            want, bound = chunk_reference(q[layer, :, :, 0], pool.keys[layer], pool.values[layer], table,
                                          list(range(len(prompts) + 1)), lens, window, sinks)
            check(out[layer][:, :, 0], want, bound)
    assert _native.device_error() == 0


@pytest.mark.parametrize("captured", [False, True])
def test_steps_with_weights_and_evictions(captured):
    """Rows of different lengths, several layers, a budget that they pass again and again: cache, weights and
    outputs follow a host model that drops the same tokens."""
    gen = torch.Generator().manual_seed(2)
    layers, bs, hkv, group, d = 2, 16, 2, 2, 64
    keep, recent, sinks, limit, steps = 40, 9, 3, 64, 90
    heads, prompts = hkv * group, [50, 7, 20]
    pool = _pool(layers, 12, hkv, d, heads)
    tables = [list(range(4 * b, 4 * b + 4)) for b in range(3)]
    for layer in range(layers):
        slots = torch.tensor([tables[b][t // bs] * bs + t % bs for b, n in enumerate(prompts) for t in range(n)]).cuda()
        pool.write_slots(layer, slots, _rand(gen, len(slots), hkv, d), _rand(gen, len(slots), hkv, d))
    kv = PagedKV(pool, tables, prompts, rope_len=200, n_head=heads, track_weights=True)
    table = kv._block_table_tensor
    shape = (layers, 3, hkv, 1, d)
    q, k, v = _rand(gen, layers, 3, heads, 1, d), _rand(gen, *shape), _rand(gen, *shape)
    graph = PagedStepGraph(kv, q, k, v) if captured else None
    kv.weights.zero_()
    lens = list(prompts)
    evictions = 0
    for step in range(steps):
        q.copy_(_rand(gen, *q.shape))
        k.copy_(_rand(gen, *shape))
        v.copy_(_rand(gen, *shape))
        before = kv.weights.clone()
        assert kv.position.tolist() == [n + step for n in prompts]
        if captured:
            out = graph.replay()
        else:
            kv.build_mask(next_token=True)
            out = []
            for layer in range(layers):
                kv.write(layer, k[layer], v[layer])
                out.append(kv.attend(layer, q[layer]))
            kv.advance()
        lens = [n + 1 for n in lens]
        assert kv.pos.tolist() == lens == kv._host_pos
        for layer in range(layers):
            want, bound, sums, off = weights_reference(q[layer, :, :, 0], pool.keys[layer], pool.values[layer], table, lens,
                                                       before[layer])
            check(out[layer][:, :, 0], want, bound)
            check(kv.weights[layer], sums, off)
            for b, n in enumerate(lens):
                at = tables[b][(n - 1) // bs]
                assert torch.equal(pool.keys[layer][at, (n - 1) % bs], k[layer, b, :, 0])
        if max(lens) == limit:
            evictions += 1
            kept = evict_reference(kv.weights, lens, keep, recent, sinks)
            old = [x.clone() for x in (*pool.keys, *pool.values)], kv.weights.clone()
            kv.evict(keep, recent=recent, sinks=sinks)
            for (layer, b, h), tokens in kept.items():
                src = torch.tensor(tokens).cuda()
                dst = torch.arange(len(tokens)).cuda()
                for x, y in ((pool.keys[layer], old[0][layer]), (pool.values[layer], old[0][layers + layer])):
                    assert torch.equal(x[table[b].long()[dst // bs], dst % bs, h], y[table[b].long()[src // bs], src % bs, h])
                assert torch.equal(kv.weights[layer, b, h, :len(tokens)], old[1][layer, b, h, src])
                assert bool((kv.weights[layer, b, h, len(tokens):] == 0).all())
            lens = [min(n, keep) for n in lens]
            assert kv.pos.tolist() == lens == kv._host_pos
    assert evictions >= 3 and kv.evicted.tolist() == kv._host_evicted
    assert _native.device_error() == 0


def test_blocks_past_32_bit_offsets():
    """Pools of more than 2^31 elements give what small ones with the same blocks give, bit for bit."""
    gen = torch.Generator().manual_seed(4)
    hkv, group, d, bs, few, many = 8, 2, 128, 16, 96, (1 << 17) + 1000  # 16,384 elements a block
    lens = [700, 1, 333]
    small = [_rand(gen, few, bs, hkv, d) for _ in range(2)]
    big = [torch.empty(many, bs, hkv, d, dtype=small[0].dtype, device="cuda") for _ in range(2)]
    at = many - few
    for x, y in zip(big, small):
        x[at:].copy_(y)
    ids = torch.randperm(few, generator=gen)
    width, tables, cursor = -(-max(lens) // bs), torch.zeros(len(lens), -(-max(lens) // bs), dtype=torch.int32), 0
    for row, n in enumerate(lens):
        pages = -(-n // bs)
        tables[row, :pages] = ids[cursor:cursor + pages]
        cursor += pages
    tables = tables.cuda()
    seqlen = torch.tensor(lens, dtype=torch.int32).cuda()
    q = _rand(gen, 40, hkv * group, d)
    cu = torch.tensor([0, 30, 31, 40], dtype=torch.int32).cuda()
    weights = torch.rand(1, len(lens), hkv, width * bs, generator=gen).cuda()
    results = []
    for (k, v), table in ((small, tables), (big, tables + at)):
        w = weights[0].clone()
        results.append([paged_decode_window(q[:3], k, v, table, seqlen, 200, sinks=4),
                        paged_prefill_window(q, k, v, table, cu, seqlen, 30, 200, sinks=4),
                        paged_decode_weights(q[:3], k, v, table, seqlen, w), w,
                        *evict_tokens([k], [v], table, seqlen, weights, 128, recent=16, sinks=4)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    for x, y in zip(big, small):
        assert torch.equal(x[at:], y)
    assert _native.device_error() == 0


def test_a_decoder_over_bounded_containers():
    """The decoder runs over a windowed and a weight-keeping container: with bounds that no row reaches it computes
    what it computes without them, and past them it goes on at the sequence's positions."""
    from decode_model import PagedDecoder

    def tokens(steps, evict=None, **bound):
        pool = _pool(2, 40, 2, 64, 4)
        kv = PagedKV(pool, [list(range(0, 10)), list(range(10, 20))], [1, 1], rope_len=400, n_head=4, **bound)
        model = PagedDecoder(kv, n_layer=2, n_head=4, n_kv_head=2, head_dim=64, rotary=64, max_pos=400)
        model.tok.copy_(torch.tensor([5, 900]))
        out = []
        for _ in range(steps):
            kv.build_mask(next_token=True)
            model.step()
            kv.advance()
            out.append(model.next.tolist())
            if evict and max(kv._host_pos) >= 100:
                kv.evict(evict, recent=16, sinks=2)
        return out, kv

    plain, _ = tokens(60)
    windowed, _ = tokens(60, window=1000, sinks=4)
    tracked, kv = tokens(60, track_weights=True)
    # greedy tokens of random weights: near ties may fall otherwise, so the first ones
    for got in (windowed, tracked):
        assert got[:2] == plain[:2]
    assert kv.position.tolist() == [61, 61]
    _, kv = tokens(250, evict=64, track_weights=True)
    assert kv.position.tolist() == [251, 251] and max(kv.pos.tolist()) < 100


def test_refusals():
    pool = _pool(1, 8, 2, 64, 4)
    make = lambda tables=([0, 1], [2, 3]), **more: PagedKV(pool, list(tables), [1, 1], rope_len=64, n_head=4, **more)  # noqa: E731
    for more, match in ((dict(window=0), "at least 1"), (dict(window=4, sinks=-1), "at least 0"), (dict(sinks=2), "need a window"),
                        (dict(window=2.5), "must be an int"), (dict(window=True), "must be an int"),
                        (dict(window=3, track_weights=True), "not both")):
        with pytest.raises(ValueError, match=match):
            make(**more)
    with pytest.raises(RuntimeError, match="track_weights"):
        make().evict(4)
    kv = make(track_weights=True)
    for args, match in (((0,), "fit into keep"), ((4, 3, 2), "fit into keep"), ((4, -1), "at least 0"), ((2.0,), "ints")):
        with pytest.raises(ValueError, match=match):
            kv.evict(args[0], recent=args[1] if len(args) > 1 else 0, sinks=args[2] if len(args) > 2 else 0)
    kv.build_mask(next_token=True)
    with pytest.raises(RuntimeError, match="inside a step"):
        kv.evict(1)
    shared = make(([0, 1], [0, 2]), track_weights=True)
    with pytest.raises(ValueError, match="share blocks"):
        shared.evict(1)
