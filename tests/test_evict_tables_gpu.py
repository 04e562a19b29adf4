"""Block tables that ``evict_tokens`` refuses as new ones, and views of one tensor that it takes."""

from __future__ import annotations

import pytest
import torch

from bounded_reference import evict_reference, make_pools
from model import _native
from model.paged_evict import evict_tokens

pytestmark = pytest.mark.gpu


def _case():
    lens = [100, 20, 70]
    k, v, table, free = make_pools(lens, 2, 64, 16, torch.bfloat16, gen=torch.Generator().manual_seed(0), spare=6)
    w = torch.rand(1, 3, 2, table.shape[1] * 16, generator=torch.Generator().manual_seed(1)).cuda()
    return lens, k, v, table, free.view(3, 2), torch.tensor(lens, dtype=torch.int32).cuda(), w


def test_the_rows_own_table():
    lens, k, v, table, _, seqlen, w = _case()
    wide = torch.zeros(3, 2 * table.shape[1], dtype=torch.int32, device="cuda")
    wide[:, ::2] = table
    before = k.clone(), v.clone()
    for old, new in ((table, table), (table, table[:, :4]), (table[:, :7], table.view(3, -1)), (wide[:, ::2], wide[:, ::2]),
                     (table, table[:, 1:])):
        with pytest.raises(ValueError, match="new_table|pd_evict"):
            evict_tokens([k], [v], old, seqlen, w, 30, new_table=new)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def test_two_tables_in_one_tensor():
    lens, k, v, table, free, seqlen, w = _case()
    both = torch.cat([table, free], 1)
    old, new = both[:, :table.shape[1]], both[:, table.shape[1]:]
    want = k.clone()
    for (_, b, h), tokens in evict_reference(w, lens, 30, 4, 1).items():
        src, dst = torch.tensor(tokens).cuda(), torch.arange(len(tokens)).cuda()
        want[new[b].long()[dst // 16], dst % 16, h] = k[old[b].long()[src // 16], src % 16, h]
    n, _ = evict_tokens([k], [v], old, seqlen, w, 30, recent=4, sinks=1, new_table=new)
    assert n.tolist() == [30, 20, 30] and torch.equal(k, want)
    assert _native.device_error() == 0
