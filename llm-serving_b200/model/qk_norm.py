"""RMS norm of each query and key head with its rotary rotation, in one launch.

The reference's attention layers normalise every head of q and k and rotate them in separate
elementwise steps (``model/layers.py:200-211``, ``apply_rotary_emb_partial`` 59-117): some ten
passes over the same rows. :func:`qk_norm_rope` reads each element once and writes it once, with
everything in between in fp32 and a single rounding at the end. Its results therefore differ from
the stepwise torch form, which rounds after every step, by up to a few ulp; callers that need the
reference's bits keep the stepwise form (``decode_model.PagedDecoder`` does by default).
"""

from __future__ import annotations

from model import _native

__all__ = ["qk_norm_rope"]


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
    ops = _native.ops or _native.require_ops()
    return ops.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, rotary_dim, eps, q_out, k_out)
