"""64-bit forms of the operators of a cache of bounded length, and how far the kernels may be from them."""

from __future__ import annotations

import math

import torch


def row_of(pool, table, row, n):
    """The first n tokens (heads, n, D) of one row of a pool, in 64 bits."""
    bs = pool.shape[1]
    t = torch.arange(n, device=pool.device)
    return pool[table[row].long()[t // bs], t % bs].double().permute(1, 0, 2)


def attend(q, k, v, seen, scale):
    """(out, weights, bound, rel) of queries (Hkv, G, S, D) over k, v (Hkv, n, D) with keys seen (S, n).

    ``bound`` is how far fp32 scores, softmax and sums may be off, before the result's own rounding: a score is
    a sum of D products, each rounded to 2^-24 of the running sum of |q k| (D + 4 roundings with the scale and the
    subtraction of the maximum); a weight's relative error is twice that (its own and the normaliser's), 2^-16 for
    P's two 16-bit parts and 2^-20 for the exponential's approximation; the sums over n tokens add 2^-24 each.
    The result is off by that much of the weighted mean of |v|. Unseen keys' values count as absent, NaN or not.
    """
    n = k.shape[1]
    any_seen = seen.any(0)
    k = torch.where(any_seen[None, :, None], k, 0.0)
    v = torch.where(any_seen[None, :, None], v, 0.0)
    s = torch.einsum("hgid,hjd->hgij", q, k) * scale
    size = (torch.einsum("hgid,hjd->hgij", q.abs(), k.abs()) * abs(scale)).masked_fill(~seen, 0).amax()
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    rel = 2.0 ** -16 + 2.0 ** -20 + 2 * (q.shape[-1] + 4) * 2.0 ** -24 * float(size) + 2 * n * 2.0 ** -24
    # a weight of the unseen is 0 and times a NaN must stay 0
    return (torch.einsum("hgij,hjd->hgid", p, v), p, rel * torch.einsum("hgij,hjd->hgid", p, v.abs()), rel)


def window_mask(first, count, n, window, sinks, device):
    """Keys 0..n-1 that queries at positions first .. first + count - 1 see."""
    i = first + torch.arange(count, device=device)[:, None]
    j = torch.arange(n, device=device)
    return (j <= i) & ((i - j < window) | (j < sinks))


def check(got, want, bound):
    """Off by at most ``bound`` and half a step of got's type."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny
    err = (got.double() - want).abs()
    allowed = bound * (1 + half) + half * want.abs() + tiny
    worst = (err - allowed).max().item()
    assert bool((err <= allowed).all()), f"off by {err.max().item():.3e}, {worst:.3e} more than allowed"


def chunk_reference(q, k_pool, v_pool, table, cu, lens, window, sinks, scale=None):
    """(out, bound) (tokens, H, D) of packed chunks; decode is chunks of one token."""
    heads, d = q.shape[1], q.shape[2]
    hkv = k_pool.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for b, n in enumerate(lens):
        at, end = cu[b], cu[b + 1]
        count = end - at
        if not count or not n:
            continue
        k, v = row_of(k_pool, table, b, n), row_of(v_pool, table, b, n)
        x = q[at:end].double().view(count, hkv, heads // hkv, d).permute(1, 2, 0, 3)
        seen = window_mask(n - count, count, n, window, sinks, q.device)
        o, _, e, _ = attend(x, k, v, seen, scale)
        out[at:end] = o.permute(2, 0, 1, 3).reshape(count, heads, d)
        bound[at:end] = e.permute(2, 0, 1, 3).reshape(count, heads, d)
    return out, bound


def weights_reference(q, k_pool, v_pool, table, lens, before):
    """(out, bound, sums, bound of the sums) of one decode step."""
    heads, d = q.shape[1], q.shape[2]
    hkv = k_pool.shape[2]
    out, bound = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    sums, off = before.double(), torch.zeros_like(before, dtype=torch.float64)
    for b, n in enumerate(lens):
        if not n:
            continue
        k, v = row_of(k_pool, table, b, n), row_of(v_pool, table, b, n)
        x = q[b].double().view(hkv, heads // hkv, 1, d)
        o, p, e, rel = attend(x, k, v, torch.ones(1, n, dtype=torch.bool, device=q.device), d ** -0.5)
        out[b], bound[b] = o.reshape(heads, d), e.reshape(heads, d)
        step = p[:, :, 0].sum(1)
        sums[b, :, :n] += step
        off[b, :, :n] = rel * step
    return out, bound, sums, off


def evict_reference(weights, lens, keep, recent, sinks):
    """Kept tokens: {(layer, row, head): list} by a stable sort on the host."""
    kept = {}
    w = weights.cpu().double()
    for layer in range(w.shape[0]):
        for b, n in enumerate(lens):
            for h in range(w.shape[2]):
                if n <= keep:
                    kept[layer, b, h] = list(range(n))
                    continue
                row = w[layer, b, h].tolist()
                middle = sorted(range(sinks, n - recent),
                                key=lambda j: (row[j] == row[j], row[j] if row[j] == row[j] else 0.0, -j), reverse=True)
                kept[layer, b, h] = sorted([*range(sinks), *middle[:keep - sinks - recent], *range(n - recent, n)])
    return kept


def make_pools(lens, hkv, d, bs, dtype, *, gen, spare=5, scale=(1.0, 0.5)):
    """Random K and V pools, a shuffled table of every row's pages, on cuda."""
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), max(max(need), 1), dtype=torch.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = perm[at:at + c]
        at += c
    k, v = ((torch.randn(blocks, bs, hkv, d, generator=gen) * f).to(dtype).cuda() for f in scale)
    return k, v, table.cuda(), perm[at:].cuda()
