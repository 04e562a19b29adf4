"""Windowed chunks whose scores are not finite, with and without rows that the kernel computes again."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import attend, check, make_pools, row_of, window_mask
from model import _native
from model.paged_window import paged_prefill_window

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("lens,counts,window", [([400, 90], [3, 90], 150), ([3000, 700], [700, 64], 1 << 20), ([100] * 40, [5] * 40, 60)])
@pytest.mark.parametrize("hidden", [0.0, INF])
def test_scores_of_minus_infinity_and_a_nan_query(lens, counts, window, hidden):
    """Keys of -inf scores have weight 0, also in rows that meet an infinity in a hidden value; a query that sees nothing
    else gives 0 / 0; a NaN query head is NaN and no other is."""
    hkv, group, d, bs = 4, 2, 128, 16
    gen = torch.Generator().manual_seed(5)
    k, v, table, _ = make_pools(lens, hkv, d, bs, BF16, gen=gen)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    q = torch.randn(cu[-1], hkv * group, d, generator=gen).to(BF16).cuda()
    q[..., 0] = 1.0
    gone = []
    for b, n in enumerate(lens):
        first = max(n - counts[b] - window + 1, 0)
        gone.append([j for j in range(n) if j < first + 80 and j % 90 != 45])
        at = torch.tensor(gone[b], device="cuda")
        k[table[b].long()[at // bs], at % bs, :, 0] = -INF
        at = torch.arange(first, device="cuda")  # what no query sees
        v[table[b].long()[at // bs], at % bs] = hidden
        if counts[b] > 1:  # what only the chunk's last query sees
            v[table[b, (n - 1) // bs], (n - 1) % bs] = hidden
    args = (k, v, table, torch.tensor(cu).cuda(), torch.tensor(lens).cuda(), max(counts), window)
    got = paged_prefill_window(q, *args)
    broken = q.clone()
    broken[:, 3, 7] = NAN
    hurt = paged_prefill_window(broken, *args)
    for b, n in enumerate(lens):
        seen = window_mask(n - counts[b], counts[b], n, window, 0, "cuda")
        seen[:, gone[b]] = False
        some = seen.any(1)
        x = q[cu[b]:cu[b + 1]].double().view(counts[b], hkv, group, d).permute(1, 2, 0, 3)
        vv = row_of(v, table, b, n)
        out, _, bound, _ = attend(x, row_of(k, table, b, n), vv, seen, d ** -0.5)
        out, bound = (t.permute(2, 0, 1, 3).reshape(counts[b], hkv * group, d) for t in (out, bound))
        mine = got[cu[b]:cu[b + 1]]
        assert bool(mine[~some].isnan().all())
        if hidden and counts[b] > 1:
            assert bool((~mine[-1].isfinite()).all())
            some[-1] = False
            out[some], bound[some] = _finite(x, k, v, table, b, n, seen, some)
        check(mine[some], out[some], bound[some])
    assert bool(hurt[:, 3].isnan().all())
    others = [h for h in range(hkv * group) if h != 3]
    assert torch.equal(hurt[:, others].nan_to_num(7.0), got[:, others].nan_to_num(7.0))
    assert _native.device_error() == 0


def _finite(x, k, v, table, b, n, seen, some):
    """The reference of the queries `some` alone, which do not see what the last one sees."""
    out, _, bound, _ = attend(x[:, :, some], row_of(k, table, b, n), row_of(v, table, b, n), seen[some], x.shape[-1] ** -0.5)
    return tuple(t.permute(2, 0, 1, 3).reshape(int(some.sum()), -1, x.shape[-1]) for t in (out, bound))
