"""The 4-bit cache's operators together, as ``sample_fp4.py`` runs them.

Tolerances. Against the 64-bit model the kernels' path rounds some ten times per layer to bf16 (2^-9
each, about 1 % together after two layers). That moves some 4 % of the cached elements across a code
boundary, a step of about a quarter: 0.25 sqrt(0.04) = 5 % of the cache's norm, hence logits with a cosine
above 1 - 0.06^2 / 2 = 0.998; the test asks for 0.99. Two paths that round the same model differently
have caches that differ by the same 5 %; the test asks for 15 %.
"""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
from decode_model import EPS, INTER, VOCAB, PagedDecoder
from model.paged_fp4 import Fp4KV, Fp4Pool
from sample_fp4 import sample_continuations
from serve.block_sharing import SharedBlockManager

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, LAYERS, BS = 4, 2, 128, 2, 16


def _model(rotary=DIM):
    return PagedDecoder(None, n_layer=LAYERS, n_head=HEADS, n_kv_head=KV_HEADS, head_dim=DIM, rotary=rotary, max_pos=256)


def _pool(blocks=64):
    return Fp4Pool(LAYERS, blocks, BS, KV_HEADS, DIM, device="cuda", n_head=HEADS)


def _prompts(lengths):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in lengths]


def _cached(pool, table, n):
    slots = torch.tensor([table[p // BS] * BS + p % BS for p in range(n)], device="cuda")
    return [torch.stack(pool.read_slots(layer, slots, torch.float32)) for layer in range(LAYERS)]


def _plain_logits(model, prompt):
    """float64, the whole prompt at once, K and V through the 64-bit quantiser."""
    n, r = len(prompt), model.rotary
    unit = torch.ones(KV_HEADS)

    def rms(x, w):
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()

    def rope(x):
        cos, sin = model.cos[:n, None].double(), model.sin[:n, None].double()
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat((x[..., :r] * cos + torch.cat((-b, a), -1) * sin, x[..., r:]), -1)

    def cache(x):
        return ref.values(*ref.quantise(x.cpu(), unit), unit).to(x.device)

    x = model.embed[torch.tensor(prompt, device="cuda")].double()
    for L in model.layers:
        qkv = (rms(x, L["ln1"]) @ L["wqkv"].T.double()).view(n, -1, DIM)
        q, k, v = qkv.split((HEADS, KV_HEADS, KV_HEADS), 1)
        q, k, v = rope(rms(q, L["qn"])), cache(rope(rms(k, L["kn"]))), cache(v)
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / DIM ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        x = x + torch.einsum("hqk,khd->qhd", s.softmax(-1), v).flatten(1) @ L["wo"].T.double()
        gu = rms(x, L["ln2"]) @ L["wgu"].T.double()
        x = x + (torch.nn.functional.silu(gu[:, :INTER]) * gu[:, INTER:]) @ L["wd"].T.double()
    return rms(x[-1], model.norm) @ model.embed.T.double()


@pytest.mark.parametrize("rotary", [DIM, 64])
def test_prompt_logits(cuda_device, rotary):
    model, pool = _model(rotary), _pool()
    prompts = _prompts([1, 9, 40])
    tables = [[5, 0, 1], [2, 9, 8], [7, 3, 6]]
    got = model.prefill(pool, prompts, tables, [0, 0, 0])
    for row, prompt in zip(got, prompts):
        want = _plain_logits(model, prompt)
        assert torch.cosine_similarity(row.double(), want, 0) > 0.99


@pytest.mark.parametrize("lengths", [[1], [16, 33, 50]])
def test_continuations(cuda_device, lengths):
    """Captured steps and a compaction under them give the tokens and cache of eager steps without;
    and the cache that decode steps wrote is the one that a prompt of the same tokens writes."""
    model, prompts, new = _model(), _prompts(lengths), 12
    runs = []
    for compact, graph in ((True, True), (False, False)):
        pool, manager = _pool(), SharedBlockManager(64, BS)
        held = manager.reserve(3)  # another request's blocks, freed before the winners decode on
        manager.free(held[:2])
        tokens, tables = sample_continuations(model, pool, manager, prompts, continuations=3, new_tokens=new,
                                              chunk=20, compact=compact, graph=graph)
        runs.append((tokens, [_cached(pool, t, n + new) for t, n in zip(tables, lengths)]))
        assert all(manager.holders(b) == 1 for t in tables for b in t)
        if compact:
            assert max(b for t in tables for b in t) < manager.in_use == 1 + sum(len(t) for t in tables)
    assert runs[0][0] == runs[1][0]
    for a, b in zip(runs[0][1], runs[1][1]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for prompt, continuations, cached in zip(prompts, *runs[0]):
        assert [len(t) for t in continuations] == [new + 1, new // 2 + 1, new // 2 + 1]
        assert len({t[0] for t in continuations}) == 3
        pool, seen = _pool(), prompt + continuations[0][:new]
        table = list(range(8))
        model.prefill(pool, [seen], [table], [0])
        for x, y in zip(_cached(pool, table, len(seen)), cached):
            assert (x - y).norm() < 0.15 * y.norm()


def test_container_protocol(cuda_device):
    pool = _pool()
    kv = Fp4KV(pool, [[3, 1], [0]], [17, 4], rope_len=20, n_head=HEADS)
    q = torch.zeros(2, HEADS, 1, DIM, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(2, KV_HEADS, 1, DIM, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="build_mask"):
        kv.attend(0, q)
    kv.build_mask(next_token=True)
    with pytest.raises(RuntimeError, match="write"):
        kv.attend(0, q)
    with pytest.raises(ValueError, match="already rotated"):
        kv.write(0, k, k, rope=(k, k))
    with pytest.raises(ValueError, match="write needs"):
        kv.write(0, q, k)
    kv.write(0, k, k)
    with pytest.raises(ValueError, match="dropout"):
        kv.attend(0, q, dropout_p=0.1)
    with pytest.raises(ValueError, match="attend needs"):
        kv.attend(0, k)
    out = torch.empty_like(q)
    assert kv.attend(0, q, out=out).data_ptr() == out.data_ptr() and not out.any()
    with pytest.raises(ValueError, match="remap"):
        kv.move_blocks([3], [2], [0, 1])
    for _ in range(3):
        kv.advance()
    with pytest.raises(IndexError, match="position bound"):
        kv.build_mask(next_token=True)
    with pytest.raises(IndexError, match="max_len"):
        kv.write(0, k, k)
