"""The operators of a KV cache of bounded length, measured over the range a serving engine calls them in.

Four operators over 16- and 32-bit paged pools ``(n_blocks, block_size, H_kv, D)``:

* ``window_decode``: one query token per row, which sees the last ``window`` tokens of its row and the
  first ``sinks`` (``model.paged_window.paged_decode_window``);
* ``window_prefill``: the same for a chunk of query tokens per row
  (``model.paged_window.paged_prefill_window``);
* ``weights``: a decode that also adds every cached token's attention weight, summed over the query
  heads of its key head, to running sums (``model.paged_evict.paged_decode_weights``);
* ``evict``: per layer, row and key head the tokens with the largest sums are kept, with the first and the
  last ones, and their keys and values close ranks, in place or in new pages
  (``model.paged_evict.evict_tokens``).

Key ``j`` is visible to the query at position ``i`` if ``j <= i`` and (``i - j < window`` or ``j < sinks``).
The plain forms below are the definitions in elementary operations in 32 bits; ``exact`` is the same in 64 bits.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------- cases


def listed():
    return [
        # one long conversation at the engine's main head shape: latency of a step
        dict(name="window_decode_one_row", op="window_decode", rows=1, low=5000, high=5000, window=1024, sinks=4, heads=16,
             kv_heads=8, dim=128, block=16, dtype="bf16", lens=1),
        # the ordinary step: 32 conversations past their window
        dict(name="window_decode_batch", op="window_decode", rows=32, low=1500, high=8192, window=2048, sinks=16, heads=16,
             kv_heads=8, dim=128, block=16, dtype="bf16", lens=2),
        # wide heads, an odd window, rows shorter than it and empty ones among long ones
        dict(name="window_decode_skewed", op="window_decode", rows=61, low=0, high=8192, window=777, sinks=3, heads=8,
             kv_heads=2, dim=256, block=32, dtype="f16", lens=3),
        # a few drafted tokens of each row checked at once
        dict(name="window_prefill_draft", op="window_prefill", rows=16, chunk_low=1, chunk_high=8, low=64, high=4096,
             window=1024, sinks=4, heads=16, kv_heads=8, dim=128, block=16, dtype="bf16", lens=4),
        # long prompts from their first token
        dict(name="window_prefill_prompt", op="window_prefill", rows=4, chunk_low=4001, chunk_high=4096, low=0, high=0,
             window=1024, sinks=4, heads=16, kv_heads=8, dim=128, block=16, dtype="bf16", lens=5),
        # later chunks of prompts, narrow heads in an odd group
        dict(name="window_prefill_chunk", op="window_prefill", rows=7, chunk_low=250, chunk_high=512, low=500, high=3000,
             window=333, sinks=1, heads=15, kv_heads=3, dim=64, block=32, dtype="f16", lens=6),
        # one row below its budget: latency of a step that keeps sums
        dict(name="weights_one_row", op="weights", rows=1, low=700, high=700, heads=16, kv_heads=8, dim=128, block=16,
             dtype="bf16", lens=7),
        # the ordinary step, 32 rows at their budget
        dict(name="weights_batch", op="weights", rows=32, low=1800, high=2048, heads=16, kv_heads=8, dim=128, block=16,
             dtype="bf16", lens=8),
        # long contexts before their first eviction, wide heads
        dict(name="weights_long", op="weights", rows=24, low=4000, high=8192, heads=8, kv_heads=2, dim=256, block=32,
             dtype="f16", lens=9),
        # one conversation brought back to its budget in every layer
        dict(name="evict_one_row", op="evict", rows=1, low=700, high=700, keep=512, recent=64, sinks=4, fresh=False, layers=28,
             kv_heads=8, dim=128, block=16, dtype="bf16", lens=10),
        # 32 rows give back a page each, in place
        dict(name="evict_page", op="evict", rows=32, low=1040, high=1040, keep=1024, recent=128, sinks=4, fresh=False, layers=8,
             kv_heads=8, dim=128, block=16, dtype="bf16", lens=11),
        # prompts cut down to a budget into pages of their own, some already below it
        dict(name="evict_prompt", op="evict", rows=9, low=800, high=8000, keep=1001, recent=32, sinks=16, fresh=True, layers=4,
             kv_heads=2, dim=256, block=32, dtype="f16", lens=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_HEADS = [(8, 2, 128), (2, 4, 256), (4, 1, 64), (8, 4, 128), (1, 8, 128), (3, 5, 64), (4, 3, 128)]


def draw(rng):
    op = rng.choice(["window_decode", "window_prefill", "weights", "evict"])
    kv_heads, group, dim = rng.choice(_HEADS)
    block, lens = rng.choice([16, 16, 32, 64]), rng.randint(20, 1 << 20)
    case = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, block=block,
                dtype=rng.choice(["bf16", "bf16", "f16"]), lens=lens)
    if op == "window_prefill":
        # at most the listed prompts' pairs before masking
        chunk = _log(rng, 1, 2048)
        before = rng.choice([0, _log(rng, 1, 4096)])
        rows = _log(rng, 1, 16)
        most = 4 * 4096 * 4096 * 16 * 128
        while rows > 1 and rows * chunk * (chunk + before) * kv_heads * group * dim > most:
            rows -= 1
        return dict(case, rows=rows, chunk_low=rng.choice([0, 1, chunk]), chunk_high=chunk, low=rng.choice([0, before // 2, before]),
                    high=before, window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 16, 100]))
    if rng.random() < 0.15:
        case["dtype"] = "f32"
    size = 4 if case["dtype"] == "f32" else 2
    if op == "evict":
        high = _log(rng, 8, 8192)
        layers = rng.randint(1, 12)
        # at most the listed page case's pools
        rows = _log(rng, 1, max(1, min(64, 8 * 32 * 1040 * 8 * 128 * 2 // (layers * high * kv_heads * dim * size))))
        keep = max(1, min(high, _log(rng, max(1, high // 16), high)))
        sinks = min(rng.choice([0, 1, 4, 16]), keep)
        return dict(case, rows=rows, low=rng.choice([0, high // 2, high]), high=high, keep=keep,
                    recent=rng.randint(0, (keep - sinks) // 2), sinks=sinks, fresh=rng.random() < 0.5, layers=layers)
    # at most the listed long case's cache
    high = _log(rng, 1, 16384)
    most = 24 * 8192 * 2 * 256 * 2 // (kv_heads * dim * size) // high
    rows = _log(rng, 1, max(1, min(128, most)))
    case.update(rows=rows, low=rng.choice([0, 1, max(1, high // 4), high]), high=high)
    if op == "window_decode":
        case.update(window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 16, 100]))
    return case


def _lengths(case):
    """Per row (query tokens, cached tokens, those of the queries included) of a case, from the case alone."""
    rng = random.Random(case["lens"])
    rows = []
    for i in range(case["rows"]):
        if case["op"] == "window_prefill":
            chunk = rng.randint(case["chunk_low"], case["chunk_high"]) if i else case["chunk_high"]
            rows.append((chunk, chunk + rng.randint(case["low"], max(case["low"], case["high"]))))
        elif i == 0:  # one row of the longest, so that no case is empty
            rows.append((1, case["high"]))
        else:
            rows.append((1, rng.randint(case["low"], case["high"])))
    return rows


# --------------------------------------------------------------------------- inputs


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _tables(rng, lengths, block, spare=7):
    """Block tables through a shuffled pool, and the pool's block count."""
    need = [-(-n // block) for n in lengths]
    blocks = sum(need) + spare
    ids = list(range(blocks))
    rng.shuffle(ids)
    width = max(max(need), 1)
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [0] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), blocks, ids[at:]


def _sums(gen, *shape):
    """Running sums of attention weights: most tokens near nothing, a few heavy, some never seen (ties at zero)."""
    x = torch.exp(2.0 * _normal(gen, *shape) - 3.0)
    return x * (torch.rand(shape, generator=gen, device="cuda") > 0.1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    h, d, bs = case["kv_heads"], case["dim"], case["block"]
    rows = _lengths(case)
    lens = [n for _, n in rows]
    s = dict(op=op, dtype=dtype, seqlen=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if op == "evict":
        s.update({k: case[k] for k in ("keep", "recent", "sinks")})
        new_width = max(1, -(-min(case["keep"], max(lens)) // bs))
        spare = new_width * case["rows"] if case["fresh"] else 3
        s["table"], blocks, free = _tables(random.Random(seed), lens, bs, spare)
        s["new_table"] = None
        if case["fresh"]:
            s["new_table"] = torch.tensor(free, dtype=torch.int32, device="cuda").view(case["rows"], new_width)
        shape = (case["layers"], blocks, bs, h, d)
        # values that follow from their place, with few bits: quick to make, and every row differs
        n = math.prod(shape)
        s["pools"] = []
        for _ in range(2):
            x = torch.randint(-2 ** 15, 2 ** 15, (n // 8,), generator=gen, device="cuda", dtype=torch.int16).repeat(9)
            x = x[n // 8 // 2:n // 8 // 2 + n]
            s["pools"].append((x.float() / 256).to(dtype).view(shape))
        s["ks"], s["vs"] = list(s["pools"][0].unbind(0)), list(s["pools"][1].unbind(0))
        s["weights"] = _sums(gen, case["layers"], case["rows"], h, s["table"].shape[1] * bs)
        return s
    s["table"], blocks, _ = _tables(random.Random(seed), lens, bs)
    # keys with a few loud channels, as after a norm's weight, and quieter values
    loud = 1.0 + 3.0 * (torch.rand(h, d, generator=gen, device="cuda") > 0.95)
    s["k"] = (_normal(gen, blocks, bs, h, d) * loud).to(dtype)
    s["v"] = (_normal(gen, blocks, bs, h, d) * 0.3).to(dtype)
    s["q"] = _normal(gen, sum(c for c, _ in rows), case["heads"], d).to(dtype)
    if op == "weights":
        s["weights"] = _sums(gen, case["rows"], h, s["table"].shape[1] * bs)
        return s
    s.update(window=case["window"], sinks=case["sinks"])
    if op == "window_prefill":
        ends = [0]
        for c, _ in rows:
            ends.append(ends[-1] + c)
        s["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["longest"] = max(c for c, _ in rows)
    return s


# --------------------------------------------------------------------------- the plain forms


def _context(s):
    """K and V (rows, heads, capacity, dim) in 32 bits of every row through its block table."""
    at = s["table"].long()
    return [x[at].flatten(1, 2).transpose(1, 2).float() for x in (s["k"], s["v"])]


def _softmax(scores, seen):
    """Weights of the scores over the keys that are seen; a query that sees none has zeros."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _plain_decode(s):
    q = s["q"]
    rows, heads, d = q.shape
    k, v = _context(s)
    hkv = k.shape[1]
    key, n = torch.arange(k.shape[2], device=q.device), s["seqlen"][:, None]
    seen = key < n
    if s["op"] == "window_decode":
        seen = seen & ((n - 1 - key < s["window"]) | (key < s["sinks"]))
    scores = torch.matmul(q.float().view(rows, hkv, heads // hkv, d), k.transpose(-1, -2)) / math.sqrt(d)
    p = _softmax(scores, seen[:, None, None])
    out = torch.matmul(p, v).reshape(rows, heads, d).to(s["dtype"])
    if s["op"] == "window_decode":
        return out
    s["weights"].add_(p.sum(2))
    return [out, s["weights"]]


def _plain_prefill(s):
    q, cu = s["q"], s["cu"].long()
    total, heads, d = q.shape
    k, v = _context(s)
    hkv = k.shape[1]
    group, rows, longest = heads // hkv, cu.numel() - 1, s["longest"]
    token = torch.arange(total, device=q.device)
    row = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    index = token - cu[row]
    padded = torch.zeros(rows, longest, heads, d, device=q.device)
    padded[row, index] = q.float()
    x = padded.view(rows, longest, hkv, group, d).permute(0, 2, 3, 1, 4)
    at = s["seqlen"].long()[:, None] - (cu[1:] - cu[:-1])[:, None] + torch.arange(longest, device=q.device)
    key = torch.arange(k.shape[2], device=q.device)
    seen = (key <= at[..., None]) & ((at[..., None] - key < s["window"]) | (key < s["sinks"]))
    p = _softmax(torch.matmul(x, k.transpose(-1, -2)[:, :, None]) / math.sqrt(d), seen[:, None, None])
    o = torch.matmul(p, v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(rows, longest, heads, d)
    return o[row, index].to(s["dtype"])


def _plain_evict(s):
    w, n, keep = s["weights"], s["seqlen"].long(), s["keep"]
    layers, rows, hkv, cap = w.shape
    k, v = s["pools"]
    bs = k.shape[2]
    key = torch.arange(cap, device=w.device)
    live = key < n[:, None]
    always = live & ((n[:, None] <= keep) | (key < s["sinks"]) | (key >= n[:, None] - s["recent"]))
    # first the tokens that always stay, then by their sums; a stable order keeps the lowest index of a tie
    rank = torch.where(always[:, None], torch.inf, w)
    rank = torch.where(live[:, None], rank, -torch.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    new = n.clamp(max=keep)
    chosen = torch.zeros(w.shape, dtype=torch.bool, device=w.device)
    chosen.scatter_(-1, order, (key < new[:, None])[None, :, None].expand(w.shape))
    # the kept tokens in their order, then the others
    most = min(keep, cap)
    source = torch.sort((~chosen).to(torch.uint8), dim=-1, stable=True).indices[..., :most]
    stays = torch.arange(most, device=w.device) < new[:, None]
    table, target = s["table"].long(), (s["table"] if s["new_table"] is None else s["new_table"]).long()
    slots = table.repeat_interleave(bs, 1) * bs + key % bs  # (rows, cap)
    where = torch.gather(slots[None, :, None].expand(w.shape), -1, source)  # (layers, rows, heads, most)
    head = torch.arange(hkv, device=w.device)[:, None]
    layer = torch.arange(layers, device=w.device)[:, None, None, None]
    to = (target.repeat_interleave(bs, 1) * bs + torch.arange(target.shape[1] * bs, device=w.device) % bs)[:, :most]
    valid = stays[None, :, None].expand(where.shape)
    dst = (layer.expand(where.shape)[valid], to[None, :, None].expand(where.shape)[valid], head.expand(where.shape)[valid])
    src = (dst[0], where[valid], dst[2])
    for x in (k.flatten(1, 2), v.flatten(1, 2)):
        x[dst] = x[src]
    sums = torch.zeros_like(w)
    sums[..., :most] = torch.gather(w, -1, source) * stays[None, :, None]
    return [k, v, sums, new.to(torch.int32)]


def run(state):
    op = state["op"]
    if own:
        return _own(op)(state)
    return {"window_decode": _plain_decode, "window_prefill": _plain_prefill, "weights": _plain_decode,
            "evict": _plain_evict}[op](state)


# --------------------------------------------------------------------------- the framework's calls

_calls = {}


def _own(op):
    if not _calls:
        path = str(Path(__file__).resolve().parent.parent / "llm-serving_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from model.paged_evict import evict_tokens, paged_decode_weights
        from model.paged_window import paged_decode_window, paged_prefill_window

        def weights(s):
            return [paged_decode_weights(s["q"], s["k"], s["v"], s["table"], s["seqlen"], s["weights"]), s["weights"]]

        def evict(s):
            n, sums = evict_tokens(s["ks"], s["vs"], s["table"], s["seqlen"], s["weights"], s["keep"], recent=s["recent"],
                                   sinks=s["sinks"], new_table=s["new_table"])
            return [s["pools"][0], s["pools"][1], sums, n]

        _calls.update(
            window_decode=lambda s: paged_decode_window(s["q"], s["k"], s["v"], s["table"], s["seqlen"], s["window"],
                                                        sinks=s["sinks"]),
            window_prefill=lambda s: paged_prefill_window(s["q"], s["k"], s["v"], s["table"], s["cu"], s["seqlen"],
                                                          s["longest"], s["window"], sinks=s["sinks"]),
            weights=weights,
            evict=evict)
    return _calls[op]


# --------------------------------------------------------------------------- what a pass cannot do without


def _visible(i, window, sinks):
    """Keys that the query at position i sees."""
    return min(window, i + 1) + min(sinks, max(0, i + 1 - window)) if i >= 0 else 0


def work(case):
    op = case["op"]
    es = 4 if case["dtype"] == "f32" else 2
    rows, token = _lengths(case), case["kv_heads"] * case["dim"] * es
    if op == "evict":
        # a row above its budget moves what lies behind the first sinks; one below it only into new pages
        moved = sum((case["keep"] - (0 if case["fresh"] else case["sinks"])) if n > case["keep"] else (n if case["fresh"] else 0)
                    for _, n in rows)
        cap = -(-max(n for _, n in rows) // case["block"]) * case["block"]
        sums = 4 * case["kv_heads"] * (sum(n for _, n in rows) + case["rows"] * cap)
        return {"bytes": case["layers"] * (2 * 2 * moved * token + sums), "flops": 0}
    if op == "weights":
        cached = seen = sum(n for _, n in rows)
        extra = 8 * case["kv_heads"] * seen
    elif op == "window_decode":
        cached = seen = sum(_visible(n - 1, case["window"], case["sinks"]) for _, n in rows)
        extra = 0
    else:
        # a row's keys are read once, whatever the number of its queries
        cached = seen = extra = 0
        for c, n in rows:
            if c:
                first = max(0, n - c - case["window"] + 1)
                cached += n - first + min(case["sinks"], first)
                seen += sum(_visible(i, case["window"], case["sinks"]) for i in range(n - c, n))
    queries = sum(c for c, _ in rows)
    return {"bytes": 2 * cached * token + 2 * queries * case["heads"] * case["dim"] * es + 4 * (cached // case["block"]) + extra,
            "flops": 4 * seen * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------- the same in 64 bits


def _row(s, b, n):
    """K and V (heads, n, dim) in 64 bits of row b's first n tokens."""
    bs = s["k"].shape[1]
    t = torch.arange(n, device=s["q"].device)
    block = s["table"][b].long()[t // bs]
    return [x[block, t % bs].double().permute(1, 0, 2) for x in (s["k"], s["v"])]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(case, s)
    q, hkv, d = s["q"].double(), case["kv_heads"], case["dim"]
    heads = case["heads"]
    out = torch.zeros_like(q)
    sums = s["weights"].double() if case["op"] == "weights" else None
    at = 0
    for b, (count, n) in enumerate(_lengths(case)):
        if count and n:
            k, v = _row(s, b, n)
            # a stretch of queries at a time, so that long prompts' scores stay small
            for first in range(0, count, 512):
                x = q[at + first:at + min(count, first + 512)]
                x = x.view(-1, hkv, heads // hkv, d).permute(1, 2, 0, 3)
                scores = torch.einsum("hgid,hjd->hgij", x, k) * d ** -0.5
                if case["op"] != "weights":
                    i = n - count + first + torch.arange(x.shape[2], device=q.device)[:, None]
                    j = torch.arange(n, device=q.device)
                    hidden = (j > i) | ((j <= i - case["window"]) & (j >= case["sinks"]))
                    scores = scores.masked_fill(hidden, -math.inf)
                p = torch.softmax(scores, -1)
                out[at + first:at + first + x.shape[2]] = torch.einsum("hgij,hjd->ihgd", p, v).reshape(-1, heads, d)
            if sums is not None:
                sums[b, :, :n] += p[:, :, 0].sum(1)
        at += count
    return out if sums is None else [out, sums]


def _exact_evict(case, s):
    keep, bs = case["keep"], case["block"]
    k, v = (x.double() for x in s["pools"])
    old_k, old_v = k.clone(), v.clone()
    w = s["weights"].double()
    sums = torch.zeros_like(w)
    target = s["table"] if s["new_table"] is None else s["new_table"]
    new = []
    for b, (_, n) in enumerate(_lengths(case)):
        m = min(n, keep)
        new.append(m)
        kept = torch.arange(n, device=w.device).expand(*w.shape[:1], w.shape[2], n)
        if n > keep:
            lo, hi = case["sinks"], n - case["recent"]
            middle = w[:, b, :, lo:hi]
            # a token's place: how many have a larger sum, or the same and a lower index
            value, _ = torch.unique(middle, return_inverse=True)
            dense = torch.searchsorted(value, middle.contiguous())
            index = torch.arange(hi - lo, device=w.device)
            best = (dense * (hi - lo) + (hi - lo - 1 - index)).topk(keep - lo - case["recent"], -1).indices.sort(-1).values + lo
            ends = [torch.arange(x, y, device=w.device).expand(*best.shape[:2], y - x) for x, y in ((0, lo), (hi, n))]
            kept = torch.cat((ends[0], best, ends[1]), -1)
        sums[:, b, :, :m] = torch.gather(w[:, b], -1, kept)
        place = torch.arange(m, device=w.device)
        to = target[b].long()[place // bs]
        layer = torch.arange(w.shape[0], device=w.device)[:, None, None]
        head = torch.arange(w.shape[2], device=w.device)[:, None]
        source = s["table"][b].long()[kept // bs]
        for x, old in ((k, old_k), (v, old_v)):
            x[layer, to, place % bs, head] = old[layer, source, kept % bs, head]
    return [k, v, sums, torch.tensor(new, dtype=torch.int32, device=w.device)]
