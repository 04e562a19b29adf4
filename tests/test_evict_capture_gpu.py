"""``PagedKV.evict`` moves tokens and the container's host positions together, so a graph may not record it."""

from __future__ import annotations

import pytest
import torch

from model.paged import PagedKV, PagedPool

pytestmark = pytest.mark.gpu


def test_refused_inside_a_capture():
    pool = PagedPool(2, 8, 16, 2, 64, dtype=torch.bfloat16, device="cuda", n_head=4)
    kv = PagedKV(pool, [[0, 1, 2], [3, 4, 5]], [40, 30], rope_len=100, n_head=4, track_weights=True)
    kv.evict(45)  # nothing to do; and loaded
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph):
        x.add_(1.0)
        for keep in (32, 45):
            with pytest.raises(RuntimeError, match="inside a capture"):
                kv.evict(keep)
    assert kv._host_pos == [40, 30] == kv.pos.tolist()
    graph.replay()
    kv.evict(32)
    torch.cuda.synchronize()
    assert kv._host_pos == [32, 30] == kv.pos.tolist() and kv.position.tolist() == [40, 30] and bool((x == 1).all())
