"""Plain 64-bit forms of the 4-bit page operators and the head norm, for the parity tests.

Written from the definitions, with no code of the library: pages are read and written byte by byte
from the documented record layout, quantising searches the nearest representable value, attention
is one softmax per query. Everything runs on the CPU in float64 (or exact integers).
"""

from __future__ import annotations

import torch

STEPS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
SCALES = torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)
                       if (e, m) != (15, 7)], dtype=torch.float64)


def nearest(x, values):
    """Index of the value nearest to x >= 0, ties to the even index, saturating."""
    hi = torch.searchsorted(values, x.contiguous()).clamp(max=len(values) - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = x - values[lo], values[hi] - x
    take_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    return torch.where(take_lo & (x < values[hi]), lo, hi)


def quantise(x, unit):
    """(codes, scale bytes) of x (n, heads, d): codes (n, heads, d) and scales (n, heads, d / 16)."""
    y = x.double().nan_to_num(nan=0.0, posinf=1e30, neginf=-1e30).unflatten(-1, (-1, 16)) / unit.double()[:, None, None]
    sb = nearest(y.abs().amax(-1) / 6, SCALES)
    s = SCALES[sb][..., None]
    ratio = torch.where(s > 0, y.abs() / s.clamp(min=2.0 ** -9), torch.zeros_like(y))
    code = nearest(ratio, STEPS) + 8 * (y < 0)
    return code.flatten(-2), sb


def values(codes, scales, unit):
    v = STEPS[codes & 7] * (1.0 - 2.0 * (codes >> 3))
    return (v.unflatten(-1, (-1, 16)) * SCALES[scales][..., None]).flatten(-2) * unit.double()[:, None]


def places(d):
    """Byte offsets in a record: K codes (16, d / 2), K scales (16, d / 16), V codes, V scales."""
    w = min(d, 128)
    kc = torch.tensor([[(j // (w // 2)) * 8 * w + t * (w // 2) + j % (w // 2) for j in range(d // 2)] for t in range(16)])
    ks = torch.tensor([[8 * d + (g // (w // 16)) * w + t * (w // 16) + g % (w // 16) for g in range(d // 16)]
                       for t in range(16)])
    vc = torch.tensor([[9 * d + (t // 8) * 4 * d + (j // 8) * 64 + (t % 8) * 8 + j % 8 for j in range(d // 2)]
                       for t in range(16)])
    vs = torch.tensor([[17 * d + (t // 8) * (d // 2) + g * 8 + t % 8 for g in range(d // 16)] for t in range(16)])
    return kc, ks, vc, vs


def write(pages, slots, k, v, units):
    """Quantise tokens into a CPU pages tensor (n_blocks, heads, tpb, 18 d) in place."""
    _, _, tpb, rec = pages.shape
    d = rec // 18
    kc, ks, vc, vs = places(d)
    for i, slot in enumerate(slots.tolist()):
        blk, off = divmod(slot, 16 * tpb)
        r = pages[blk, :, off // 16]
        for x, unit, c_at, s_at in ((k, units[0], kc, ks), (v, units[1], vc, vs)):
            code, scale = quantise(x[i:i + 1], unit)
            r[:, c_at[off % 16]] = (code[0, :, 0::2] | (code[0, :, 1::2] << 4)).to(torch.uint8)
            r[:, s_at[off % 16]] = scale[0].to(torch.uint8)


def read(pages, slots, units):
    """(k, v) float64 (n, heads, d) of flat slots of a CPU pages tensor."""
    _, h, tpb, rec = pages.shape
    d = rec // 18
    blk, off = slots // (16 * tpb), slots % (16 * tpb)
    r = pages[blk, :, off // 16].long()  # (n, heads, rec)
    kc, ks, vc, vs = places(d)
    out = []
    for unit, c_at, s_at in ((units[0], kc, ks), (units[1], vc, vs)):
        b = r.gather(2, c_at[off % 16][:, None].expand(-1, h, -1))
        s = r.gather(2, s_at[off % 16][:, None].expand(-1, h, -1))
        codes = torch.stack((b & 15, b >> 4), -1).flatten(-2)
        out.append(values(codes, s, unit))
    return out


def attention(q, pages, table, lengths, chunks, units, scale):
    """(out, weighted mean |v|), float64 (total_q, H, D): row b's chunk of chunks[b] queries over its
    lengths[b] keys, causal and bottom-right aligned; no visible key gives zeros."""
    h, tpb = pages.shape[1], pages.shape[2]
    heads, d = q.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mean = torch.zeros_like(out)
    at = 0
    for b, (n, count) in enumerate(zip(lengths, chunks)):
        if n and count:
            t = torch.arange(n)
            k, v = read(pages, table[b].long()[t // (16 * tpb)] * 16 * tpb + t % (16 * tpb), units)
            x = q[at:at + count].double().view(count, h, heads // h, d)
            s = torch.einsum("ihgd,jhd->hgij", x, k) * scale
            hidden = t[None] > (n - count + torch.arange(count))[:, None]
            p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)
            out[at:at + count] = torch.einsum("hgij,jhd->ihgd", p, v).reshape(count, heads, d)
            mean[at:at + count] = torch.einsum("hgij,jhd->ihgd", p, v.abs()).reshape(count, heads, d)
        at += count
    return out, mean


def norm_rope(x, w, cos, sin, pos, eps, rotary):
    """RMS norm of each head row and its rotation, float64; also the magnitudes that were summed."""
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    half = rotary // 2
    c, s = cos.double()[pos][:, None, :half], sin.double()[pos][:, None, :half]
    out, size = y.clone(), y.abs().clone()
    a, b = y[..., :half], y[..., half:rotary]
    out[..., :half], out[..., half:rotary] = a * c - b * s, a * s + b * c
    size[..., :half] = (a * c).abs() + (b * s).abs()
    size[..., half:rotary] = (a * s).abs() + (b * c).abs()
    return out, size


#: Half an ulp relative to a value, at most: 2^-8 for bf16 (8 significant bits), 2^-11 for fp16, 2^-24.
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
