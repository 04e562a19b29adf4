"""``PagedDecoder`` over bounded containers, step by step: where its queries and keys are rotated, and what its attention
returns, past evictions and windows."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import check, chunk_reference, weights_reference
from decode_model import PagedDecoder
from model import _native
from model.paged import PagedKV, PagedPool

pytestmark = pytest.mark.gpu

LAYERS, HEADS, HKV, DIM, BS = 2, 4, 2, 64, 16


def _rotated(x, model, position):
    """(value, bound) of x (B, heads, D), each row rotated to its position: two products and their sum, each rounded."""
    cos, sin = (t[position].double()[:, None] for t in (model.cos, model.sin))
    x = x.double()
    half = DIM // 2
    a, b = x * cos, torch.cat([-x[..., half:], x[..., :half]], -1) * sin
    return a + b, 2.0 ** -8 * (a.abs() + b.abs() + (a + b).abs()) * (1 + 2.0 ** -7)


@pytest.mark.parametrize("bound", [dict(), dict(window=24, sinks=3), dict(window=1000), dict(track_weights=True)])
def test_steps(bound):
    pool = PagedPool(LAYERS, 24, BS, HKV, DIM, dtype=torch.bfloat16, device="cuda", n_head=HEADS)
    tables = [list(range(0, 6)), list(range(8, 14))]
    kv = PagedKV(pool, tables, [1, 1], rope_len=400, n_head=HEADS, **bound)
    model = PagedDecoder(kv, n_layer=LAYERS, n_head=HEADS, n_kv_head=HKV, head_dim=DIM, rotary=DIM, max_pos=400)
    model.tok.copy_(torch.tensor([5, 900]))
    seen, attend = [], kv.attend

    def spy(layer, q, **more):
        out = attend(layer, q, **more)
        seen.append((layer, q[:, :, 0].clone(), out[:, :, 0].clone()))
        return out

    kv.attend = spy
    evict = "track_weights" in bound
    evictions = moved = 0
    for step in range(150 if evict else 90):
        seen.clear()
        n, position = kv.pos.clone(), kv.position.clone()
        assert position.tolist() == [1 + step] * 2
        x, before = model.embed[model.tok], kv.weights.clone() if evict else None
        kv.build_mask(next_token=True)
        model.step()
        kv.advance()
        # layer 0's query and key: the normed projections of the input token, at its place in the sequence
        qkv = model._rms(x, model.layers[0]["ln1"]) @ model.layers[0]["wqkv"].T
        q = model._rms(qkv[:, :HEADS * DIM].view(2, HEADS, DIM), model.layers[0]["qn"])
        k = model._rms(qkv[:, HEADS * DIM:(HEADS + HKV) * DIM].view(2, HKV, DIM), model.layers[0]["kn"])
        at = torch.arange(2, device="cuda")
        written = pool.keys[0][kv._block_table_tensor[at, n // BS].long(), n % BS]
        for got, x0 in ((seen[0][1], q), (written, k)):
            check(got.double(), *_rotated(x0, model, position))
            if evictions:
                here, allowed = _rotated(x0, model, n)
                moved += int(((got.double() - here).abs() > allowed).any())
        # every layer's attention over what the cache holds now
        lens = (n + 1).tolist()
        for layer, q, out in seen:
            args = q, pool.keys[layer], pool.values[layer], kv._block_table_tensor
            if evict:
                want, off, sums, sums_off = weights_reference(*args, lens, before[layer])
                check(kv.weights[layer], sums, sums_off)
            else:
                want, off = chunk_reference(*args, [0, 1, 2], lens, bound.get("window", 1000), bound.get("sinks", 0))
            check(out, want, off)
        if evict and max(kv._host_pos) >= 90:
            kv.evict(64, recent=16, sinks=2)
            evictions += 1
    if evict:
        assert evictions >= 2 and moved == 2 * (150 - 89)  # at the cache's positions the angles would be others
    assert _native.device_error() == 0
