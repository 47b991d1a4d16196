"""Norm of queries and keys per head with the position rotation (libmuon_amd
``muon_qk_norm_rope``). No counterpart in the reference."""

from __future__ import annotations

import torch
from torch import Tensor

from .. import _row_ops

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check_on(device: torch.device, *tensors: Tensor | None) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise RuntimeError(f"tensors on two devices: {device} and {t.device}")


def _weight(w: Tensor | None, dim: int) -> Tensor | None:
    if w is None:
        return None
    if w.dim() != 1 or w.size(0) != dim:
        raise ValueError(f"weights are ({dim},); got {tuple(w.shape)}")
    if w.dtype not in _FLOATS:
        raise TypeError(f"weights are fp32, bf16 or fp16; got {w.dtype}")
    return w.contiguous()


def qk_norm_rope(
    q: Tensor,
    k: Tensor,
    q_weight: Tensor | None = None,
    k_weight: Tensor | None = None,
    cos: Tensor | None = None,
    sin: Tensor | None = None,
    positions: Tensor | None = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[Tensor, Tensor]:
    """The RMS norm of every query and key head, then the rotation by the token's position, in
    one pass: ``n = x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, and
    ``(a, b) -> (a cos - b sin, b cos + a sin)`` for the pairs of its first ``rotary`` values.

    Args:
        q, k: ``(batch, tokens, heads, dim)`` or ``(tokens, heads, dim)``, fp32, bf16 or fp16,
            ``dim`` at most 1024; any strides (slices of a fused projection are read in
            place) with a contiguous last dimension (others are copied first). k may have fewer
            heads.
        q_weight, k_weight: ``(dim,)`` gains of one floating type, or None for ones.
        cos, sin: ``(length, rotary / 2)`` fp32 tables, or None for no rotation. ``rotary`` may be
            less than ``dim``: the rest passes unturned.
        positions: int32 or int64 rows of the tables, ``(tokens,)`` or ``(batch, tokens)``;
            None: token t is at position t. A position outside the table makes its token NaN.
        interleaved: pairs are (2i, 2i + 1) instead of (i, i + rotary / 2).

    Returns the new queries and keys, contiguous, in their input's type. Differentiable in q, k
    and the weights; computed in fp32 and rounded once."""
    shape, other, device = q.shape, k.shape, q.device
    dim = shape[-1]
    if len(shape) not in (3, 4) or len(other) != len(shape):
        raise ValueError(f"q and k are (batch, tokens, heads, dim) or (tokens, heads, dim); got "
                         f"{tuple(shape)} and {tuple(other)}")
    lead = shape[:-2]
    if lead != other[:-2] or dim != other[-1]:
        raise ValueError(f"q and k differ in batch, tokens or dim: {tuple(shape)} and "
                         f"{tuple(other)}")
    if q.dtype not in _FLOATS or k.dtype != q.dtype:
        raise TypeError(f"q and k are both fp32, bf16 or fp16; got {q.dtype} and {k.dtype}")
    if not 1 <= dim <= 1024:
        raise ValueError(f"dim is 1 to 1024; got {dim}")
    _check_on(device, k, q_weight, k_weight, cos, sin, positions)
    q_weight, k_weight = _weight(q_weight, dim), _weight(k_weight, dim)
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"weights of two types: {q_weight.dtype} and {k_weight.dtype}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.size(1) > dim:
            raise ValueError(f"cos and sin are (length, rotary / 2) with rotary at most {dim}; got "
                             f"{tuple(cos.shape)} and {tuple(sin.shape)}")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise TypeError(f"cos and sin are fp32; got {cos.dtype} and {sin.dtype}")
        if cos.requires_grad or sin.requires_grad:
            raise ValueError("cos and sin are tables: no gradient is made for them")
        cos, sin = cos.contiguous(), sin.contiguous()
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions are int32 or int64; got {positions.dtype}")
        if positions.shape != lead and positions.shape != lead[-1:]:
            raise ValueError(f"positions are ({lead[-1]},) or {tuple(lead)}; got "
                             f"{tuple(positions.shape)}")
        positions = _row_ops.unit_last(positions)
    elif cos is not None and lead[-1] > cos.size(0):
        raise ValueError(f"{lead[-1]} tokens, but the tables have {cos.size(0)} positions")
    _row_ops.check_device(device)
    return _row_ops.qk_norm_rope(_row_ops.unit_last(q), _row_ops.unit_last(k), q_weight, k_weight,
                                 cos, sin, positions, eps, interleaved)
