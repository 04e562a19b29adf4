"""What the workspaces of the bounded cache's decodes have to hold."""

from __future__ import annotations

import pytest
import torch

from model import _native
from model.paged_window import decode_workspace, paged_decode_window

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("heads,hkv,d,dtype", [(16, 8, 128, BF16), (4, 1, 64, torch.float16), (8, 2, 256, torch.float32)])
def test_a_workspace_serves_fewer_rows(heads, hkv, d, dtype):
    """``decode_workspace(rows, ...)`` is for up to that many rows, also where more rows go in several launches of fewer."""
    like = torch.empty(0, dtype=dtype, device="cuda")
    sizes = [decode_workspace(r, heads, hkv, d, like).numel() for r in [*range(0, 4097, 128), 4500, 6000, 8192, 20000]]
    assert sizes == sorted(sizes)


def test_a_call_in_a_workspace_of_more_rows():
    gen = torch.Generator(device="cuda").manual_seed(0)
    heads, hkv, d, bs, most = 4, 2, 64, 16, 4000
    k, v = (torch.randn(300, bs, hkv, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
    ws = decode_workspace(most, heads, hkv, d, k)
    for rows in (1, 2000, 2700, 2900, 3500, most):
        table = torch.randint(0, 300, (rows, 2), generator=gen, device="cuda", dtype=torch.int32)
        lens = torch.randint(0, 2 * bs + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        q = torch.randn(rows, heads, d, generator=gen, device="cuda").to(BF16)
        want = paged_decode_window(q, k, v, table, lens, 20, sinks=1)
        assert torch.equal(paged_decode_window(q, k, v, table, lens, 20, sinks=1, workspace=ws), want)
    assert _native.device_error() == 0
