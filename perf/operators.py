"""The operators around a KV cache held in 4 bits, measured over the range a serving engine calls them in.

Five operators, in the order a decode step or a prompt chunk runs them:

* ``norm_rope``: RMS norm of each query and key head with the rotary rotation, in one pass
  (``model.qk_norm.qk_norm_rope``);
* ``write``: keys and values quantised into 4-bit pages, and read back through the same slots
  (``model.paged_fp4.write_slots_fp4`` / ``read_slots_fp4``);
* ``decode``: attention of one query token per row over 4-bit pages
  (``model.paged_fp4.paged_decode_fp4``);
* ``prefill``: causal attention of a chunk of query tokens per row over 4-bit pages
  (``model.paged_fp4.paged_prefill_fp4``);
* ``copy``: pages copied from block to block in every layer's pools, with the block tables
  renumbered when a pool is compacted (``serve.block_copy.copy_blocks``).

A 4-bit page. ``pages`` is uint8 ``(n_blocks, n_kv_head, block_size / 16, 18 * head_dim)``: the last
dimension is one head's record of 16 consecutive tokens,

  K codes   8 D bytes  [D / W blocks][16 tokens][W / 2 bytes], W = min(D, 128)
  K scales    D bytes  [D / W blocks][16 tokens][W / 16]
  V codes   8 D bytes  [2 halves][D / 16 groups][8 tokens][8 bytes]
  V scales    D bytes  [2 halves][D / 16 groups][8 tokens]

A byte holds elements 2 j (low nibble) and 2 j + 1 (high). A nibble is sign, two exponent bits, one
mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6. A scale is one e4m3 byte for 16 neighbouring elements. An
element stands for nibble * scale * unit[head], the units being powers of two that the pool keeps
per (K or V, head). Quantising: scale = e4m3(max|x / unit| / 6), code = the nearest nibble of
x / unit / scale, both to nearest, ties to even, both saturating.

The plain forms below are the definitions in elementary operations in 32 bits; ``exact`` is the
same in 64 bits.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6


# --------------------------------------------------------------------------- cases


def listed():
    return [
        # one row's single token at the engine's main head shape: pure latency
        dict(name="norm_rope_token", op="norm_rope", tokens=1, heads=16, kv_heads=8, dim=128, rotary=128, dtype="bf16",
             fused=True, positions=4096),
        # a packed prompt batch of odd length, wide heads with a partly rotated head_dim
        dict(name="norm_rope_prompt", op="norm_rope", tokens=6001, heads=8, kv_heads=2, dim=256, rotary=64, dtype="f16",
             fused=True, positions=8192),
        # a decode step's write: one token of each of 32 rows
        dict(name="write_step", op="write", tokens=32, kv_heads=8, dim=128, block=16, blocks=4224, dtype="bf16"),
        # a packed prompt batch written at once
        dict(name="write_prompt", op="write", tokens=7001, kv_heads=8, dim=128, block=16, blocks=1024, dtype="bf16"),
        # one row of a short conversation: latency of the decode itself
        dict(name="decode_one_row", op="decode", rows=1, low=700, high=700, spread="even", heads=16, kv_heads=8, dim=128,
             block=16, dtype="bf16", lens=1),
        # the ordinary step: 32 rows at context 2048
        dict(name="decode_batch", op="decode", rows=32, low=2048, high=2048, spread="even", heads=16, kv_heads=8, dim=128,
             block=16, dtype="bf16", lens=2),
        # skewed lengths, some rows empty, wide heads with four query heads to a key head
        dict(name="decode_skewed", op="decode", rows=61, low=0, high=8192, spread="skewed", heads=8, kv_heads=2, dim=256,
             block=32, dtype="f16", lens=3),
        # long contexts, a cache well past the L2
        dict(name="decode_long", op="decode", rows=32, low=8192, high=8192, spread="even", heads=16, kv_heads=8, dim=128,
             block=16, dtype="bf16", lens=4),
        # a few drafted tokens of each row checked at once
        dict(name="prefill_draft", op="prefill", rows=16, chunk_low=1, chunk_high=8, low=64, high=2048, heads=16, kv_heads=8,
             dim=128, block=16, dtype="bf16", lens=5),
        # long prompt chunks behind an earlier context
        dict(name="prefill_chunk", op="prefill", rows=4, chunk_low=1001, chunk_high=1024, low=1900, high=2048, heads=16,
             kv_heads=8, dim=128, block=16, dtype="bf16", lens=6),
        # a fork: the last, partly filled page of four continuations, in every layer
        dict(name="copy_fork", op="copy", pairs=4, layers=28, blocks=512, block=16, kv_heads=8, dim=128, dtype="bf16",
             rows=0, width=0),
        # compaction of a fragmented pool: pages moved down, the tables of 32 rows renumbered
        dict(name="copy_compact", op="copy", pairs=701, layers=12, blocks=2048, block=16, kv_heads=8, dim=128, dtype="bf16",
             rows=32, width=33),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm_rope", "write", "decode", "decode", "prefill", "prefill", "copy"])
    kv_heads, group, dim = rng.choice([(8, 2, 128), (2, 4, 256), (4, 1, 64), (8, 4, 128), (1, 8, 128), (3, 5, 64), (4, 3, 128)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm_rope":
        return dict(op=op, tokens=_log(rng, 1, 8192), heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([dim, dim // 2, dim // 4]), dtype=rng.choice(["bf16", "f16", "f32"]),
                    fused=rng.random() < 0.7, positions=rng.randint(1024, 16384))
    if op == "write":
        block = rng.choice([16, 32])
        tokens = _log(rng, 1, 8192)
        return dict(op=op, tokens=tokens, kv_heads=kv_heads, dim=dim, block=block,
                    blocks=-(-tokens // block) + rng.randint(1, 400), dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "decode":
        # at most the long case's cache: 32 x 8192 tokens of 8 heads of 128
        high = _log(rng, 16, 16384)
        most = 32 * 8192 * 8 * 128 // (kv_heads * dim) // high
        rows = _log(rng, 1, max(1, min(128, most)))
        return dict(op=op, rows=rows, low=rng.choice([0, 1, max(1, high // 4), high]), high=high,
                    spread=rng.choice(["even", "skewed"]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    block=rng.choice([16, 32, 64]), dtype=dtype, lens=rng.randint(10, 1 << 20))
    if op == "prefill":
        # at most the listed chunk case's products
        high = _log(rng, 1, 2048)
        chunk = _log(rng, 1, 1024)
        rows = rng.randint(1, 16)
        heads = kv_heads * group
        most = 4 * 1001 * (1900 + 500) * 16 * 128
        while rows > 1 and rows * chunk * (high + chunk) * heads * dim > most:
            rows -= 1
        while rows * chunk * (high + chunk) * heads * dim > most:
            chunk = max(1, chunk // 2)
        return dict(op=op, rows=rows, chunk_low=rng.choice([0, 1, chunk]), chunk_high=chunk, low=rng.choice([0, high // 2, high]),
                    high=high, heads=heads, kv_heads=kv_heads, dim=dim, block=rng.choice([16, 32, 64]), dtype=dtype,
                    lens=rng.randint(10, 1 << 20))
    layers = rng.randint(1, 28)
    pairs = _log(rng, 1, max(1, 8000 // layers))
    rows = rng.choice([0, 0, 1, 7, 32])
    return dict(op=op, pairs=pairs, layers=layers, blocks=2 * pairs + rng.randint(1, 64), block=rng.choice([16, 32]),
                kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "f16"]), rows=rows,
                width=rng.randint(1, 128) if rows else 0)


def _lengths(case):
    """Per row (query tokens, cached tokens the queries see) of a case, from the case alone."""
    rng = random.Random(case["lens"])
    rows = []
    for i in range(case["rows"]):
        if case["op"] == "prefill":
            chunk = rng.randint(case["chunk_low"], case["chunk_high"]) if i else case["chunk_high"]
            rows.append((chunk, chunk + rng.randint(case["low"], max(case["low"], case["high"]))))
        elif i == 0:  # one row of the longest, so that no case is empty
            rows.append((1, case["high"]))
        elif case["spread"] == "even":
            rows.append((1, rng.randint(case["low"], case["high"])))
        else:  # lognormal around an eighth of the longest, a few rows at the lower end
            n = int(case["high"] / 8 * math.exp(rng.gauss(0, 1)))
            rows.append((1, case["low"] if rng.random() < 0.05 else max(case["low"], min(case["high"], n))))
    return rows


# --------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _units(kv_heads):
    """The pool's power-of-two units per (K or V, head): values are small, keys about one."""
    u = torch.ones(2, kv_heads, device="cuda")
    u[1] = 2.0 ** -4
    u[0, ::3] = 2.0 ** -2
    return u


def _kv(gen, tokens, kv_heads, dim, dtype):
    """Keys with a few loud channels, as after the norm's weight, and quieter values."""
    loud = 1.0 + 3.0 * (torch.rand(kv_heads, dim, generator=gen, device="cuda") > 0.95)
    k = (_normal(gen, tokens, kv_heads, dim) * loud).to(dtype)
    v = (_normal(gen, tokens, kv_heads, dim) * 0.3).to(dtype)
    return k, v


def _tables(rng, lengths, block):
    """Block tables through a shuffled pool, and the pool's block count."""
    need = [-(-n // block) for n in lengths]
    blocks = sum(need) + 7
    ids = list(range(blocks))
    rng.shuffle(ids)
    width = max(max(need), 1)
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [0] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), blocks


def prepare(case, seed):
    gen = _gen(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    s = dict(op=op, dtype=dtype)
    if op == "norm_rope":
        t, h, hkv, d, r = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rotary"))
        # q and k are views of the fused projection's output, or tensors of their own
        qkv = _normal(gen, t, (h + 2 * hkv) * d) * 0.8
        qkv = qkv.to(dtype)
        q, k = qkv[:, :h * d].view(t, h, d), qkv[:, h * d:(h + hkv) * d].view(t, hkv, d)
        if not case["fused"]:
            q, k = q.contiguous(), k.contiguous()
        inv = 1e6 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float32) / r)
        angle = torch.arange(case["positions"], device="cuda", dtype=torch.float32)[:, None] * inv
        s.update(q=q, k=k, wq=(1 + 0.1 * _normal(gen, d)).to(dtype), wk=(1 + 0.1 * _normal(gen, d)).to(dtype),
                 cos=angle.cos().to(dtype), sin=angle.sin().to(dtype),
                 pos=torch.randint(0, case["positions"], (t,), generator=gen, device="cuda"))
        return s
    if op == "copy":
        es = 2
        shape = (case["blocks"], case["block"], case["kv_heads"], case["dim"])
        n = case["blocks"] * case["block"] * case["kv_heads"] * case["dim"] * es
        pools = []
        for _ in range(2 * case["layers"]):
            # random finite 16-bit patterns: the exponent's top bit is cleared
            raw = torch.randint(0, 256, (n,), generator=gen, device="cuda", dtype=torch.uint8).view(torch.int16)
            pools.append((raw & -16385).view(dtype).view(shape))
        perm = torch.randperm(case["blocks"], generator=gen, device="cuda").to(torch.int32)
        src, dst = perm[:case["pairs"]].contiguous(), perm[case["pairs"]:2 * case["pairs"]].contiguous()
        s.update(pools=pools, src=src, dst=dst, table=None, remap=None)
        if case["rows"]:
            s["table"] = torch.randint(0, case["blocks"], (case["rows"], case["width"]), generator=gen, device="cuda",
                                       dtype=torch.int32)
            s["remap"] = torch.arange(case["blocks"], device="cuda", dtype=torch.int32)
            s["remap"][src.long()] = dst
        return s
    hkv, d, bs = case["kv_heads"], case["dim"], case["block"]
    s["units"] = _units(hkv)
    if op == "write":
        t = case["tokens"]
        s["pages"] = torch.zeros(case["blocks"], hkv, bs // 16, 18 * d, dtype=torch.uint8, device="cuda")
        s["slots"] = torch.randperm(case["blocks"] * bs, generator=gen, device="cuda")[:t].contiguous()
        s["k"], s["v"] = _kv(gen, t, hkv, d, dtype)
        return s
    rows = _lengths(case)
    table, blocks = _tables(random.Random(seed), [n for _, n in rows], bs)
    k, v = _kv(gen, blocks * bs, hkv, d, torch.bfloat16)
    s["pages"] = _encode(k, v, s["units"], blocks, bs)
    s["table"] = table
    s["seqlen"] = torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda")
    total = sum(c for c, _ in rows)
    s["q"] = _normal(gen, total, case["heads"], d).to(dtype)
    if op == "prefill":
        ends = [0]
        for c, _ in rows:
            ends.append(ends[-1] + c)
        s["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["longest"] = max(c for c, _ in rows)
    return s


# --------------------------------------------------------------------------- the plain forms


def _quantise(x, unit):
    """(codes, scales) of x (tokens, heads, dim): codes uint8 of the same shape, scales (.., dim / 16) e4m3."""
    t, h, d = x.shape
    x = (x.float() / unit[:, None]).view(t, h, d // 16, 16)
    six = torch.full((1,), 6.0, device=x.device)
    scale = (x.abs().amax(-1) / six).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float()[..., None]
    y = torch.where(s > 0, x.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = code.to(torch.uint8) + 8 * (x < 0).to(torch.uint8)
    return code.view(t, h, d), scale.view(torch.uint8)


def _encode(k, v, units, blocks, bs):
    """Pages (blocks, heads, bs / 16, 18 dim) of the tokens k, v (blocks * bs, heads, dim) in slot order."""
    h, d = k.shape[1], k.shape[2]
    w = min(d, 128)
    parts = []
    for x, unit, is_k in ((k, units[0], True), (v, units[1], False)):
        code, scale = _quantise(x, unit)
        byte = code[..., 0::2] | (code[..., 1::2] << 4)
        if is_k:  # (tile, 16 tokens, head, block, bytes) -> (tile, head, block, token, bytes)
            byte = byte.view(-1, 16, h, d // w, w // 2).permute(0, 2, 3, 1, 4)
            scale = scale.view(-1, 16, h, d // w, w // 16).permute(0, 2, 3, 1, 4)
        else:  # (tile, half, 8 tokens, head, group, bytes) -> (tile, head, half, group, token, bytes)
            byte = byte.view(-1, 2, 8, h, d // 16, 8).permute(0, 3, 1, 4, 2, 5)
            scale = scale.view(-1, 2, 8, h, d // 16).permute(0, 3, 1, 4, 2)
        parts += [byte.reshape(-1, h, 8 * d), scale.reshape(-1, h, d)]
    tiles = torch.cat(parts, -1)
    return tiles.view(blocks, bs // 16, h, 18 * d).permute(0, 2, 1, 3).contiguous()


def _codes(tiles, d):
    """K and V codes (.., 16, d) and e4m3 scale bytes (.., 16, d / 16) of records (.., 18 d)."""
    lead, w = tiles.shape[:-1], min(d, 128)
    n = len(lead)
    head = list(range(n))

    def nibbles(b):
        return torch.stack((b & 15, b >> 4), -1).flatten(-2)

    kc = tiles[..., :8 * d].reshape(*lead, d // w, 16, w // 2).permute(*head, n + 1, n, n + 2).reshape(*lead, 16, d // 2)
    ks = tiles[..., 8 * d:9 * d].reshape(*lead, d // w, 16, w // 16).permute(*head, n + 1, n, n + 2).reshape(*lead, 16, d // 16)
    vc = tiles[..., 9 * d:17 * d].reshape(*lead, 2, d // 16, 8, 8).permute(*head, n, n + 2, n + 1, n + 3)
    vs = tiles[..., 17 * d:].reshape(*lead, 2, d // 16, 8).permute(*head, n, n + 2, n + 1)
    return nibbles(kc), ks, nibbles(vc.reshape(*lead, 16, d // 2)), vs.reshape(*lead, 16, d // 16)


def _values(code, scale, unit):
    """What codes and scale bytes stand for, in 32 bits; unit broadcasts over (.., tokens, dim)."""
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    s = scale.view(torch.float8_e4m3fn).float()
    return (lut[code.int()].unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2) * unit


def _context(s):
    """K and V (rows, heads, capacity, dim) of every row through its block table."""
    pages, d = s["pages"], s["pages"].shape[-1] // 18
    rows, width = s["table"].shape
    tiles = pages[s["table"].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)  # (rows, heads, tiles, 18 d)
    kc, ks, vc, vs = _codes(tiles, d)
    unit = s["units"][:, None, :, None, None]
    k = _values(kc.flatten(2, 3), ks.flatten(2, 3), unit[0])
    return k, _values(vc.flatten(2, 3), vs.flatten(2, 3), unit[1])


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(dim)) v with key j of query i visible where seen; a query with none gives zeros."""
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_norm_rope(s):
    out = []
    cos, sin = s["cos"][s["pos"]].float()[:, None], s["sin"][s["pos"]].float()[:, None]
    half = cos.shape[-1]
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * w.float()
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        out.append(torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1).to(s["dtype"]))
    return out


def _plain_write(s):
    k, v, units, pages = s["k"], s["v"], s["units"], s["pages"]
    blocks, h, nt, rec = pages.shape
    d, t = rec // 18, k.shape[0]
    # a token's bytes of a record: its own offsets, gathered from the record of a tile full of tokens
    one = torch.arange(rec, device=k.device).view(1, 1, 1, rec)
    kc, ks, vc, vs = (x.reshape(16, -1) for x in _places(one, d))
    slot = s["slots"]
    tile = slot // 16
    base = (((tile // nt)[:, None] * h + torch.arange(h, device=k.device)) * nt + (tile % nt)[:, None]) * rec
    flat, at = pages.view(-1), slot % 16
    places = [base[..., None] + p[at][:, None] for p in (kc, ks, vc, vs)]
    codes = []
    for x, unit in ((k, units[0]), (v, units[1])):
        code, scale = _quantise(x, unit)
        codes += [code[..., 0::2] | (code[..., 1::2] << 4), scale]
    for p, c in zip(places, codes):
        flat[p] = c
    got = [flat[p] for p in places]
    out = []
    for c, sc, unit in ((got[0], got[1], units[0]), (got[2], got[3], units[1])):
        code = torch.stack((c & 15, c >> 4), -1).flatten(-2)
        out.append(_values(code, sc, unit[:, None]).to(s["dtype"]))
    return out


def _places(one, d):
    """Byte offsets inside a record, per token: K codes (16, d / 2), K scales (16, d / 16), and V's."""
    w = min(d, 128)
    kc = one[..., :8 * d].reshape(d // w, 16, w // 2).permute(1, 0, 2)
    ks = one[..., 8 * d:9 * d].reshape(d // w, 16, w // 16).permute(1, 0, 2)
    vc = one[..., 9 * d:17 * d].reshape(2, d // 16, 8, 8).permute(0, 2, 1, 3)
    vs = one[..., 17 * d:].reshape(2, d // 16, 8).permute(0, 2, 1)
    return kc, ks, vc, vs


def _plain_decode(s):
    q, pages = s["q"], s["pages"]
    rows, heads, d = q.shape
    hkv = pages.shape[1]
    k, v = _context(s)
    seen = torch.arange(k.shape[2], device=q.device) < s["seqlen"][:, None]
    o = _attend(q.float().view(rows, hkv, heads // hkv, d), k, v, seen[:, None, None])
    return o.reshape(rows, heads, d).to(s["dtype"])


def _plain_prefill(s):
    q, pages, cu = s["q"], s["pages"], s["cu"].long()
    total, heads, d = q.shape
    hkv = pages.shape[1]
    group, rows, longest = heads // hkv, cu.numel() - 1, s["longest"]
    k, v = _context(s)
    token = torch.arange(total, device=q.device)
    row = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    index = token - cu[row]
    padded = torch.zeros(rows, longest, heads, d, device=q.device)
    padded[row, index] = q.float()
    x = padded.view(rows, longest, hkv, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    last = s["seqlen"].long()[:, None] - (cu[1:] - cu[:-1])[:, None] + torch.arange(longest, device=q.device)
    seen = torch.arange(k.shape[2], device=q.device) <= last[..., None]
    o = _attend(x, k, v, seen[:, None].repeat(1, 1, group, 1))
    o = o.view(rows, hkv, group, longest, d).permute(0, 3, 1, 2, 4).reshape(rows, longest, heads, d)
    return o[row, index].to(s["dtype"])


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for pool in s["pools"]:
        pool[dst] = pool[src]
    if s["table"] is None:
        return s["pools"]
    s["table"].copy_(s["remap"][s["table"].long()])
    return s["pools"] + [s["table"]]


def run(state):
    op = state["op"]
    if own:
        return _own(op)(state)
    return {"norm_rope": _plain_norm_rope, "write": _plain_write, "decode": _plain_decode, "prefill": _plain_prefill,
            "copy": _plain_copy}[op](state)


# --------------------------------------------------------------------------- the framework's calls

_calls = {}


def _own(op):
    if not _calls:
        path = str(Path(__file__).resolve().parent.parent / "llm-serving_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from model.paged_fp4 import paged_decode_fp4, paged_prefill_fp4, read_slots_fp4, write_slots_fp4
        from model.qk_norm import qk_norm_rope
        from serve.block_copy import copy_blocks

        def write(s):
            write_slots_fp4(s["pages"], s["slots"], s["k"], s["v"], units=s["units"])
            return list(read_slots_fp4(s["pages"], s["slots"], s["dtype"], units=s["units"]))

        def copy(s):
            copy_blocks(s["pools"], s["src"], s["dst"], block_table=s["table"], remap=s["remap"])
            return s["pools"] if s["table"] is None else s["pools"] + [s["table"]]

        _calls.update(
            norm_rope=lambda s: list(qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["pos"], eps=_EPS)),
            write=write,
            decode=lambda s: paged_decode_fp4(s["q"], s["pages"], s["table"], s["seqlen"], units=s["units"]),
            prefill=lambda s: paged_prefill_fp4(s["q"], s["pages"], s["table"], s["cu"], s["seqlen"], s["longest"],
                                                units=s["units"]),
            copy=copy)
    return _calls[op]


# --------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    es = 4 if case["dtype"] == "f32" else 2
    if op == "norm_rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        side = case["tokens"] * (case["rotary"] * es + 8) + 2 * case["dim"] * es
        return {"bytes": 2 * n * es + side, "flops": 7 * n}
    if op == "write":
        n = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * n * es + 2 * n * 9 // 16 + 16 * case["tokens"], "flops": 4 * n}
    if op == "copy":
        page = case["block"] * case["kv_heads"] * case["dim"] * es
        table = 8 * case["rows"] * case["width"] + (4 * case["blocks"] if case["rows"] else 0)
        return {"bytes": 2 * 2 * case["layers"] * case["pairs"] * page + 8 * case["pairs"] + table, "flops": 0}
    rows = _lengths(case)
    queries = sum(c for c, _ in rows)
    # a row's keys are read once, whatever the number of its queries
    cache = sum(n for c, n in rows if c) * case["kv_heads"] * case["dim"] * 2 * 9 // 16
    pages = sum(-(-n // case["block"]) for c, n in rows if c)
    seen = sum(c * (n - c) + c * (c + 1) // 2 for c, n in rows) if op == "prefill" else sum(n for _, n in rows)
    return {"bytes": cache + 2 * queries * case["heads"] * case["dim"] * es + 4 * pages + 4 * len(rows),
            "flops": 4 * seen * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------- the same in 64 bits


def _e4m3_table():
    """The 127 non-negative e4m3 values by their code, in 64 bits."""
    values = []
    for c in range(127):
        e, m = c >> 3, c & 7
        values.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return torch.tensor(values, dtype=torch.float64, device="cuda")


def _nearest(x, values):
    """Index of the value nearest to x >= 0 (values ascending), ties to the even index."""
    low = (torch.searchsorted(values, x.contiguous(), right=True) - 1).clamp(0, values.numel() - 1)
    high = (low + 1).clamp(max=values.numel() - 1)
    a, b = x - values[low], values[high] - x
    return torch.where((b < a) | ((b == a) & (low % 2 == 1)), high, low)


def _exact_values(x, unit):
    """What x (tokens, heads, dim) stands for after quantising, in 64 bits."""
    steps = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    scales = _e4m3_table()
    y = x.double().unflatten(-1, (-1, 16)) / unit.double()[:, None, None]
    scale = scales[_nearest(y.abs().amax(-1) / 6, scales)][..., None]
    ratio = torch.where(scale > 0, y.abs() / scale.clamp(min=1e-300), torch.zeros_like(y))
    return (torch.sign(y) * steps[_nearest(ratio, steps)] * scale * unit.double()[:, None, None]).flatten(-2)


def _exact_row(s, row, n):
    """K and V (heads, n, dim) of one row's first n tokens in 64 bits, from the bytes of its pages."""
    pages = s["pages"]
    h, nt, d = pages.shape[1], pages.shape[2], pages.shape[3] // 18
    w = min(d, 128)
    tok = torch.arange(n, device=pages.device)
    block = s["table"][row].long()[tok // (16 * nt)]
    rec = pages[block, :, (tok // 16) % nt].permute(1, 0, 2).long()  # (heads, n, 18 d)
    at = (tok % 16)[:, None]
    el = torch.arange(d, device=pages.device)
    places = (
        (el // w) * 8 * w + at * (w // 2) + (el % w) // 2,
        8 * d + (el // w) * w + at * (w // 16) + (el % w) // 16,
        9 * d + (at // 8) * 4 * d + (el // 16) * 64 + (at % 8) * 8 + (el % 16) // 2,
        17 * d + (at // 8) * (d // 2) + (el // 16) * 8 + at % 8,
    )
    kc, ks, vc, vs = (torch.gather(rec, 2, p[None].expand(h, -1, -1)) for p in places)
    steps = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=pages.device)
    scales = _e4m3_table()
    out = []
    for c, sc, unit in ((kc, ks, s["units"][0]), (vc, vs, s["units"][1])):
        nib = (c >> (4 * (el % 2))) & 15
        out.append(steps[nib & 7] * (1.0 - 2.0 * (nib >> 3)) * scales[sc] * unit.double()[:, None, None])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm_rope":
        out = []
        cos, sin = s["cos"].double()[s["pos"]].unsqueeze(1), s["sin"].double()[s["pos"]].unsqueeze(1)
        half = cos.shape[-1]
        for x, w in ((s["q"].double(), s["wq"].double()), (s["k"].double(), s["wk"].double())):
            y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w
            z = y.clone()
            z[..., :half] = y[..., :half] * cos - y[..., half:2 * half] * sin
            z[..., half:2 * half] = y[..., half:2 * half] * cos + y[..., :half] * sin
            out.append(z)
        return out
    if op == "write":
        return [_exact_values(s["k"], s["units"][0]), _exact_values(s["v"], s["units"][1])]
    if op == "copy":
        for pool in s["pools"]:
            pool.index_copy_(0, s["dst"].long(), pool.index_select(0, s["src"].long()))
        got = [p.double() for p in s["pools"]]
        return got if s["table"] is None else got + [None]
    q, hkv = s["q"].double(), s["pages"].shape[1]
    heads, d = q.shape[1], q.shape[2]
    out = torch.zeros_like(q)
    at = 0
    for row, (count, n) in enumerate(_lengths(case)):
        if count and n:
            k, v = _exact_row(s, row, n)
            x = q[at:at + count].view(count, hkv, heads // hkv, d).permute(1, 2, 0, 3)
            scores = torch.einsum("hgid,hjd->hgij", x, k) * d ** -0.5
            hidden = torch.arange(n, device=q.device) > n - count + torch.arange(count, device=q.device)[:, None]
            p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            out[at:at + count] = torch.einsum("hgij,hjd->ihgd", p, v).reshape(count, heads, d)
        at += count
    return out
