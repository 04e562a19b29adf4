"""What ``pd_decode_noalloc`` needs of its built-in scratch."""

from __future__ import annotations

import pytest
import torch

from model import _native
from model.triton_decode import paged_decode

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_noalloc_takes_what_its_scratch_holds():
    """The step records of plans are no part of what ``pd_decode_noalloc`` needs of its 8 MiB."""
    rows, group, d, bs = 1450, 4, 128, 16
    hkv = next(n for n in range(200, 400) if _native.workspace_bytes(rows, n * group, n, d, BF16) > 8 << 20)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(4, bs, hkv, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
    table = torch.tensor([[1, 3]], dtype=torch.int32, device="cuda").repeat(rows, 1)
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lens[::97] = 25
    q = torch.randn(rows, 1, d, generator=gen, device="cuda").to(BF16).repeat(1, hkv * group, 1)
    want = paged_decode(q, k, v, table, lens)
    got = torch.full_like(q, float("nan"))
    _native.decode_noalloc(q, k, v, table, lens, got, _native.log2e_scale(d ** -0.5))
    assert torch.equal(got, want)
    assert _native.device_error() == 0
