"""Several continuations per prompt over a 4-bit KV cache: the cache's operators as a server uses them.

Prompts are run in chunks (``qk_norm_rope``, the 4-bit write, the chunk attention); each prompt's pages are
then shared by its continuations, which copy only the partly filled page (``SharedBlockManager.fork``,
``copy_blocks``); all decode together in a captured step; half-way the losers leave, the pool is
compacted in place, and the winners decode on. Random weights (``decode_model.PagedDecoder``).

    python sample_fp4.py --prompts 4 --continuations 4 --prompt-tokens 1000 --new-tokens 64
"""

from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "llm-serving_b200"))

import torch

from decode_model import VOCAB, PagedDecoder
from model.paged_fp4 import Fp4KV, Fp4Pool
from serve.block_copy import copy_blocks
from serve.block_sharing import SharedBlockManager
from serve.graph import DecodeStepGraph


def prefill_prompts(model, pool, prompts, tables, chunk):
    """Prompts in chunks of up to ``chunk`` tokens, all rows together; logits after each prompt."""
    logits = torch.empty(len(prompts), VOCAB, dtype=torch.bfloat16, device=pool.device)
    for start in range(0, max(len(p) for p in prompts), chunk):
        rows = [i for i, p in enumerate(prompts) if len(p) > start]
        logits[rows] = model.prefill(pool, [prompts[i][start:start + chunk] for i in rows], [tables[i] for i in rows],
                                     [start] * len(rows))
    return logits


def decode(model, kv, first, steps, *, before=None, graph=True):
    """``steps`` greedy tokens after ``first`` of every row of ``kv``: ``(rows, steps)`` on the host.
    ``before`` runs between the capture and the first step."""
    model.attach(kv)
    captured = DecodeStepGraph(kv, model.step, model.prepare_q) if graph else None
    if before is not None:
        before()
    model.tok.copy_(first)
    out = torch.empty(steps, kv.batch, dtype=torch.long, device=model.tok.device)
    for i in range(steps):
        if captured is not None:
            captured.replay()
        else:
            kv.build_mask(next_token=True)
            model.step()
            kv.advance()
        out[i] = model.next
    return out.T.tolist()


def sample_continuations(model, pool, manager, prompts, *, continuations, new_tokens, chunk=512, compact=True,
                         graph=True):
    """Greedy continuations of each prompt from its ``continuations`` most likely first tokens.

    Half of ``new_tokens`` are decoded for all of them, the rest for each prompt's first.
    Returns ``(tokens, tables)``: a list per prompt of the continuations' tokens, and the winners' block
    tables. The blocks stay held by the winners.
    """
    bs, half = pool.block_size, new_tokens // 2
    tables = []
    for p in prompts:
        table = manager.reserve(-(-(len(p) + new_tokens) // bs))
        if table is None:
            raise RuntimeError("the pool has too few blocks for the prompts")
        tables.append(table)
    logits = prefill_prompts(model, pool, prompts, tables, chunk)

    rows, copies = [], []
    for table, p in zip(tables, prompts):
        rows.append(table)
        for _ in range(continuations - 1):
            forked = manager.fork(table, len(p))
            if forked is None:
                raise RuntimeError("the pool has too few blocks for the continuations")
            rows.append(forked[0])
            copies += forked[1]
    copy_blocks(pool, [a for a, _ in copies], [b for _, b in copies])

    first = logits.float().topk(continuations, dim=-1).indices.flatten()
    lengths = [len(p) for p in prompts for _ in range(continuations)]
    bound = max(lengths) + new_tokens
    tokens = [[t] for t in first.tolist()]
    new = decode(model, Fp4KV(pool, rows, lengths, rope_len=bound, n_head=pool.n_head), first, half, graph=graph)
    tokens = [t + n for t, n in zip(tokens, new)]

    winners = range(0, len(rows), continuations)
    for i, table in enumerate(rows):
        if i not in winners:
            manager.free(table)
    kv = Fp4KV(pool, [rows[i] for i in winners], [lengths[i] + half for i in winners], rope_len=bound, n_head=pool.n_head)
    last = torch.tensor([tokens[i][-1] for i in winners], device=pool.device)
    new = decode(model, kv, last, new_tokens - half, graph=graph,
                 before=(lambda: kv.move_blocks(*manager.compact())) if compact else None)
    for i, n in zip(winners, new):
        tokens[i] += n
    return [tokens[i:i + continuations] for i in winners], kv.block_tables


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--prompts", type=int, default=4)
    ap.add_argument("--continuations", type=int, default=4)
    ap.add_argument("--prompt-tokens", type=int, default=1000)
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--layers", type=int, default=28)
    a = ap.parse_args()
    heads, kv_heads, dim, bs = 16, 8, 128, 16
    per_row = -(-(a.prompt_tokens + a.new_tokens) // bs) + 1
    pool = Fp4Pool(a.layers, a.prompts * a.continuations * per_row, bs, kv_heads, dim, device="cuda", n_head=heads)
    manager = SharedBlockManager(pool.n_blocks, bs)
    model = PagedDecoder(None, n_layer=a.layers, n_head=heads, n_kv_head=kv_heads, head_dim=dim, rotary=dim,
                         max_pos=a.prompt_tokens + a.new_tokens)
    gen = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, VOCAB, (a.prompt_tokens,), generator=gen).tolist() for _ in range(a.prompts)]
    t0 = time.perf_counter()
    tokens, tables = sample_continuations(model, pool, manager, prompts, continuations=a.continuations,
                                          new_tokens=a.new_tokens)
    torch.cuda.synchronize()
    print(f"{sum(len(t) for c in tokens for t in c)} tokens of {len(prompts)} x {a.continuations} continuations in "
          f"{time.perf_counter() - t0:.2f} s; pool {pool.bytes() / 2 ** 20:.0f} MiB, {manager.in_use} of {pool.n_blocks} "
          f"blocks in use, the highest {max(b for t in tables for b in t)}")


if __name__ == "__main__":
    main()
