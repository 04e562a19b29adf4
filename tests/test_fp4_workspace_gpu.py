"""The workspace of 4-bit attention calls that are given none, on streams that are also captured."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu


def _case(device, lengths=(1200, 77, 640)):
    g = torch.Generator().manual_seed(0)
    hkv, d, heads = 8, 128, 16
    need = [-(-n // 16) for n in lengths]
    pages = torch.randint(0, 256, (sum(need), hkv, 1, 18 * d), generator=g, dtype=torch.uint8)
    _, ks, _, vs = ref.places(d)
    for at in (ks, vs):
        pages[..., at.flatten()] = torch.randint(0x20, 0x34, (sum(need), hkv, 1, at.numel()), generator=g, dtype=torch.uint8)
    table = torch.zeros(len(lengths), max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(n) + sum(need[:b])
    q = torch.randn(len(lengths), heads, d, generator=g).to(torch.bfloat16)
    return [t.to(device) for t in (q, pages, table, torch.tensor(lengths, dtype=torch.int32))]


def _allocated():
    return torch.cuda.memory_stats()["allocated_bytes.all.allocated"]


def test_a_capture_has_a_workspace_of_its_own(cuda_device):
    """Also on a stream whose eager calls have one already: the graph may be replayed beside them."""
    from model.paged_fp4 import fp4_workspace, paged_decode_fp4

    args = _case(cuda_device)
    size = fp4_workspace(args[1]).numel()
    out = torch.empty_like(args[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_decode_fp4(*args, out=out)
        base = out.clone()
    side.synchronize()
    taken = []
    for _ in range(2):
        graph, captured = torch.cuda.CUDAGraph(), torch.zeros_like(out)
        with torch.cuda.graph(graph, stream=side):
            before = _allocated()
            paged_decode_fp4(*args, out=captured)
            first = _allocated() - before
            paged_decode_fp4(*args, out=captured)
            taken.append((first, _allocated() - before - first))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, base)
    assert all(first >= size and second == 0 for first, second in taken), taken
    with torch.cuda.stream(side):
        before = _allocated()
        paged_decode_fp4(*args, out=out)
        assert _allocated() == before, "eager calls keep theirs"
    side.synchronize()
    assert torch.equal(out, base)


def test_a_graph_beside_eager_calls_and_another_graph(cuda_device):
    """Two graphs captured on a stream that is used eagerly too, replayed on streams of their own beside
    eager calls on the first: every result is the one that a call alone gives."""
    from model.paged_fp4 import paged_decode_fp4

    cases = [_case(cuda_device, lengths) for lengths in ((3000, 77, 640), (2500,), (1800, 1900))]
    alone = [paged_decode_fp4(*args) for args in cases]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        paged_decode_fp4(*cases[0])
    torch.cuda.synchronize()
    graphs, outs = [], [[torch.zeros_like(a) for _ in range(20)] for a in alone]
    for i in (1, 2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            for out in outs[i]:
                paged_decode_fp4(*cases[i], out=out)
        graphs.append(graph)
    for _ in range(20):
        for graph, stream in zip(graphs, streams[1:]):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[0]):
            for out in outs[0]:
                paged_decode_fp4(*cases[0], out=out)
        torch.cuda.synchronize()
        for out, want in zip(outs, alone):
            assert all(torch.equal(o, want) for o in out)
            for o in out:
                o.zero_()


def test_a_pool_takes_a_workspace(cuda_device):
    from model.paged_fp4 import Fp4Pool, fp4_workspace

    q, pages, table, seqlen = _case(cuda_device)
    pool = Fp4Pool(1, pages.shape[0], 16, 8, 128, device=cuda_device, n_head=16)
    pool.pages[0].copy_(pages)
    cu = torch.arange(4, dtype=torch.int32, device=cuda_device)
    want = pool.prefill(0, q, table, cu, seqlen, 1)
    ws = fp4_workspace(pages)
    assert torch.equal(pool.prefill(0, q, table, cu, seqlen, 1, workspace=ws), want)
    with pytest.raises(ValueError, match="workspace"):
        pool.prefill(0, q, table, cu, seqlen, 1, workspace=ws[:256])
