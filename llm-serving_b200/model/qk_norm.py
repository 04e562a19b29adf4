"""RMS norm of each query and key head with its rotary rotation, in one launch.

The reference's attention layers normalise every head of q and k and rotate them in separate
elementwise steps (``model/layers.py:200-211``, ``apply_rotary_emb_partial`` 59-117): some ten
passes over the same rows. :func:`qk_norm_rope` reads each element once and writes it once, with
everything in between in fp32 and a single rounding at the end. Its results therefore differ from
the stepwise torch form, which rounds after every step, by up to a few ulp; callers that need the
reference's bits keep the stepwise form (``decode_model.PagedDecoder`` does by default).
"""

from __future__ import annotations

import torch

from model import _native
from model.triton_decode import _require_backend, _require_cuda_tensors

__all__ = ["qk_norm_rope"]

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _contract(q, k, q_weight, k_weight, cos, sin, positions, rotary_dim):
    """The call's contract as (violated, message) rules in the order they are checked; a later rule
    may rely on the earlier ones."""
    yield q.dim() != 3 or k.dim() != 3, lambda: (
        f"q must be (T, H, D) and k (T, H_kv, D), got {tuple(q.shape)} / {tuple(k.shape)}")
    tokens, _, d = q.shape
    yield k.shape[0] != tokens or k.shape[2] != d, lambda: (
        f"q {tuple(q.shape)} and k {tuple(k.shape)} must share their tokens and head_dim")
    yield q.shape[1] < 1 or k.shape[1] < 1, lambda: "q and k need at least one head each"
    yield not 2 <= d <= 256, lambda: f"head_dim {d} is outside the kernel's range 2..256"
    yield q.dtype not in _DTYPES, lambda: f"q dtype must be fp16, bf16 or fp32, got {q.dtype}"
    for name, t in (("k", k), ("q_weight", q_weight), ("k_weight", k_weight), ("cos", cos), ("sin", sin)):
        yield t.dtype != q.dtype, lambda name=name, t=t: f"{name} must be {q.dtype} like q, got {t.dtype}"
        yield t.device != q.device, lambda name=name, t=t: f"{name} is on {t.device} but q is on {q.device}"
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        yield tuple(t.shape) != (d,), lambda name=name, t=t: f"{name} must be ({d},), got {tuple(t.shape)}"
    yield cos.dim() != 2 or cos.shape != sin.shape, lambda: (
        f"cos and sin must be (positions, rotary_dim / 2), got {tuple(cos.shape)} / {tuple(sin.shape)}")
    yield rotary_dim < 0 or rotary_dim % 2 != 0 or rotary_dim > d, lambda: (
        f"rotary_dim must be even and in [0, {d}], got {rotary_dim}")
    yield rotary_dim > 2 * cos.shape[1], lambda: (
        f"rotary_dim {rotary_dim} needs {rotary_dim // 2} table columns, got {cos.shape[1]}")
    if positions is not None:
        yield positions.dtype not in (torch.int32, torch.int64), lambda: (
            f"positions must be int32 or int64, got {positions.dtype}")
        yield tuple(positions.shape) != (tokens,), lambda: (
            f"positions must be ({tokens},), got {tuple(positions.shape)}")
        yield positions.device != q.device, lambda: f"positions is on {positions.device} but q is on {q.device}"


def _output(name, like, out):
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or out.stride(-1) != 1:
        raise ValueError(f"{name} must be a {tuple(like.shape)} {like.dtype} tensor on {like.device} with a unit last stride")
    return out


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, *, eps: float = 1e-6,
                 rotary_dim: int | None = None, q_out=None, k_out=None):
    """Normalised and rotated ``(q, k)``.

    ``q`` ``(T, H, D)`` and ``k`` ``(T, H_kv, D)`` may be views of one fused projection (any token
    and head strides). Row ``t`` is rotated by row ``positions[t]`` (``t`` without ``positions``) of
    ``cos`` / ``sin`` ``(n_pos, >= rotary_dim / 2)``: GPT-NeoX pairs ``(i, i + rotary_dim / 2)`` over
    the first ``rotary_dim`` elements (default ``2 * cos.shape[1]``), the rest passing through.
    All tensors share one dtype: fp16, bf16 or fp32. ``q_out`` / ``k_out`` (optional) receive the
    result and may be ``q`` / ``k`` themselves. A position outside the tables gives a row of zeros
    and sets ``_native.DEVERR_ROPE_RANGE`` in the device error word.
    """
    _require_backend()
    _require_cuda_tensors((("q", q), ("k", k)))
    rotary_dim = 2 * cos.shape[-1] if rotary_dim is None else int(rotary_dim)
    for violated, message in _contract(q, k, q_weight, k_weight, cos, sin, positions, rotary_dim):
        if violated:
            raise ValueError(message())
    if q.stride(2) != 1:
        q = q.contiguous()
    if k.stride(2) != 1:
        k = k.contiguous()
    if rotary_dim and cos.stride(1) != 1:
        cos = cos.contiguous()
    if rotary_dim and sin.stride(1) != 1:
        sin = sin.contiguous()
    if positions is not None:
        positions = positions.contiguous()
    q_out, k_out = _output("q_out", q, q_out), _output("k_out", k, k_out)
    with _native.device_guard(q.device):
        _native.qk_norm_rope(q, k, q_out, k_out, q_weight.contiguous(), k_weight.contiguous(), cos, sin, positions,
                             rotary_dim, float(eps))
    return q_out, k_out
