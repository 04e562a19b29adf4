"""A weight-keeping container that is built anew between steps: positions, sums and outputs go on as in one that is not."""

from __future__ import annotations

import pytest
import torch

from model import _native
from model.paged import PagedKV, PagedPool

pytestmark = pytest.mark.gpu

LAYERS, HEADS, HKV, DIM, BS = 2, 4, 2, 64, 16
TABLES = [[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]]


def _make(seed=0):
    gen = torch.Generator().manual_seed(seed)
    pool = PagedPool(LAYERS, 16, BS, HKV, DIM, dtype=torch.bfloat16, device="cuda", n_head=HEADS)
    for layer in range(LAYERS):
        for x in (pool.keys[layer], pool.values[layer]):
            x.copy_(torch.randn(x.shape, generator=gen))
    return pool, PagedKV(pool, TABLES, [40, 3, 20], rope_len=300, n_head=HEADS, track_weights=True)


def _step(kv, rows, step):
    gen = torch.Generator().manual_seed(1000 + step)
    q, k, v = (torch.randn(LAYERS, 3, h, 1, DIM, generator=gen).to(torch.bfloat16).cuda()[:, rows] for h in (HEADS, HKV, HKV))
    kv.build_mask(next_token=True)
    out = []
    for layer in range(LAYERS):
        kv.write(layer, k[layer], v[layer])
        out.append(kv.attend(layer, q[layer]).clone())
    kv.advance()
    if max(kv._host_pos) >= 60:
        kv.evict(30, recent=6, sinks=2)
    return torch.stack(out)


def test_it_goes_on():
    """Row 1 leaves and rows 2, 0 go on in another order, in tables that grew."""
    _, whole = _make()
    pool, kv = _make()
    for step in range(50):
        assert torch.equal(_step(whole, [0, 1, 2], step), _step(kv, [0, 1, 2], step))
    assert max(kv._host_evicted) > 0
    rows = [2, 0]
    new = PagedKV(pool, [TABLES[2] + [12], TABLES[0] + [13]], kv.pos[rows].tolist(), rope_len=300, n_head=HEADS, track_weights=True,
                  evicted=kv.evicted[rows].tolist())
    new.weights[..., :kv.weights.shape[3]] = kv.weights[:, rows]
    for step in range(50, 120):
        assert new.position.tolist() == whole.position[rows].tolist() == [70 + step - 50, 90 + step - 50]
        want = _step(whole, [0, 1, 2], step)
        assert torch.equal(_step(new, rows, step), want[:, rows])
        assert torch.equal(new.weights[..., :64], whole.weights[:, rows])
    assert new.evicted.tolist() == new._host_evicted == whole.evicted[rows].tolist()
    assert _native.device_error() == 0


def test_the_position_bound_counts_evicted_tokens():
    pool, _ = _make()
    kv = PagedKV(pool, TABLES, [10, 3, 20], rope_len=61, n_head=HEADS, track_weights=True, evicted=[50, 0, 1])
    _step(kv, [0, 1, 2], 0)
    kv.build_mask()
    with pytest.raises(IndexError, match="overflow"):
        kv.build_mask(next_token=True)


def test_refusals():
    pool, _ = _make()
    make = lambda **more: PagedKV(pool, TABLES, [10, 3, 20], rope_len=60, n_head=HEADS, **more)  # noqa: E731
    for evicted in ([0, 0], [0, 0, 0, 0], [0, -1, 0], []):
        with pytest.raises(ValueError, match="one count"):
            make(track_weights=True, evicted=evicted)
    with pytest.raises(IndexError, match="position bound"):
        make(track_weights=True, evicted=[0, 0, 41])
    for more in (dict(), dict(window=5)):
        with pytest.raises(ValueError, match="track_weights"):
            make(evicted=[0, 0, 0], **more)
