"""Head norm with rotation: rows normalised in place by the kernel for any head_dim and alignment, and rows
at positions outside the tables."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(tokens, heads, hkv, d, rotary, dtype, device, offset):
    """q and k as views of one projection, `offset` elements off its start, and their weights and tables."""
    g = torch.Generator().manual_seed(d + rotary)
    qkv = torch.randn(tokens, (heads + 2 * hkv) * d + offset, generator=g).to(dtype).to(device)
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g)).to(dtype).to(device)
    angle = torch.rand(50, max(rotary // 2, 1), generator=g) * 6.3
    pos = torch.randint(0, 50, (tokens,), generator=g).to(device)

    def views(base):
        return (base[:, offset:offset + heads * d].view(tokens, heads, d),
                base[:, offset + heads * d:offset + (heads + hkv) * d].view(tokens, hkv, d))

    return qkv, views, (wq, wk, angle.cos().to(dtype).to(device), angle.sin().to(dtype).to(device), pos)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rotary,offset", [(80, 80, 0), (96, 64, 0), (250, 250, 0), (128, 128, 1), (64, 64, 3), (256, 256, 1),
                                             (256, 20, 0), (2, 2, 0)])
def test_in_place_changes_no_bit_at_any_head_dim_and_alignment(cuda_device, dtype, d, rotary, offset):
    from model.qk_norm import qk_norm_rope

    qkv, views, args = _case(301, 5, 2, d, rotary, dtype, cuda_device, offset)
    q, k = views(qkv)
    want = qk_norm_rope(q, k, *args, rotary_dim=rotary)
    for _ in range(3):
        work = qkv.clone()
        qi, ki = views(work)
        got = qk_norm_rope(qi, ki, *args, rotary_dim=rotary, q_out=qi, k_out=ki)
        assert got[0].data_ptr() == qi.data_ptr()
        assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])
        rest = (5 + 2) * d + offset
        assert torch.equal(work[:, rest:], qkv[:, rest:]) and torch.equal(work[:, :offset], qkv[:, :offset])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rotary", [(128, 128), (64, 32), (256, 0), (80, 20)])
def test_a_position_outside_the_tables_gives_zeros_whatever_the_row_holds(cuda_device, dtype, d, rotary):
    from model import _native
    from model.qk_norm import qk_norm_rope

    q = torch.ones(4, 3, d, dtype=dtype, device=cuda_device)
    q[1, 0, 0], q[1, 1, 1], q[1, 2, d - 1] = float("inf"), -float("inf"), float("nan")
    k = q[:, :1].clone()
    w = torch.ones(d, dtype=dtype, device=cuda_device)
    w[0] = float("inf")
    tables = torch.ones(8, max(rotary // 2, 1), dtype=dtype, device=cuda_device)
    assert _native.device_error() == 0
    qo, ko = qk_norm_rope(q, k, w, w, tables, tables, torch.tensor([0, 8, -1, 7], device=cuda_device), rotary_dim=rotary)
    assert _native.device_error() == _native.DEVERR_ROPE_RANGE
    assert (qo[1:3] == 0).all() and (ko[1:3] == 0).all()
