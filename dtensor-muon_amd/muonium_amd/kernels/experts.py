"""Routed tokens to their experts, the experts' products, and back (libmuon_amd
``muon_expert_order``, ``muon_dispatch``, ``muon_expert_linear``, ``muon_combine``). No counterpart in
the reference."""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .. import _row_ops
from .heads import _FLOATS, _check_on


class ExpertOrder(NamedTuple):
    """What :func:`sort_by_expert` returns: where each choice's row stands among all of them."""

    slots: Tensor  #: (..., k) int32: the choice's row; -1 - row for an empty choice
    offsets: Tensor  #: (experts + 1,) int32: the experts' first rows, and the end of the last one's


def sort_by_expert(experts: Tensor, num_experts: int) -> ExpertOrder:
    """The order of all tokens' choices by expert, tokens in their own order within one.

    Args:
        experts: ``(..., k)`` int64, the experts of each token as :func:`route` gives them. A number
            outside ``0 .. num_experts - 1`` (an empty slot's -1) names none: its choice gets no
            expert, and one of the rows behind the last expert's.
        num_experts: at most 1024.

    There are as many rows as choices, ``tokens * k`` (below 2^31), whatever the experts are: nothing is
    copied to the host."""
    if experts.dim() < 1:
        raise ValueError("experts are (..., k)")
    if experts.dtype != torch.int64:
        raise TypeError(f"experts are int64; got {experts.dtype}")
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"1 to 1024 experts; got {num_experts}")
    if experts.numel() >= 2**31:
        raise ValueError(f"below 2^31 choices; got {experts.numel()}")
    _row_ops.check_device(experts.device)
    return ExpertOrder(*_row_ops.sort_by_expert(experts.contiguous(), num_experts))


def _slots(order: ExpertOrder, like: Tensor) -> Tensor:
    slots = order.slots
    if slots.dim() < 1 or slots.shape[-1] < 1:
        raise ValueError(f"slots are (..., k); got {tuple(slots.shape)}")
    if slots.dtype != torch.int32:
        raise TypeError(f"slots are int32; got {slots.dtype}")
    if slots.numel() >= 2**31:
        raise ValueError(f"below 2^31 choices; got {slots.numel()}")
    _check_on(like.device, slots)
    return slots if slots.dim() == 2 else slots.reshape(-1, slots.shape[-1])


def _check_floats(name: str, t: Tensor) -> None:
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name} are fp32, bf16 or fp16; got {t.dtype}")
    if t.shape[-1] > 2**30:
        raise ValueError(f"{name} have at most 2^30 columns; got {t.shape[-1]}")


def dispatch(x: Tensor, order: ExpertOrder) -> Tensor:
    """Every token's row at the places of its choices: ``(tokens * k, width)``, sorted by expert. The
    rows behind the last expert's (``order.offsets[-1]`` on) are zeros.

    Args:
        x: ``(..., width)``, fp32, bf16 or fp16; rows may be strided.
        order: of :func:`sort_by_expert`, with x's leading dimensions.

    Differentiable in x: a token's gradient is the sum of its choices' rows, in fp32, rounded once; what
    comes back for the rows behind the last expert's reaches nothing."""
    if x.dim() < 1 or x.shape[:-1] != order.slots.shape[:-1]:
        raise ValueError(f"x is {(*order.slots.shape[:-1], 'width')}; got {tuple(x.shape)}")
    _check_floats("rows", x)
    slots = _slots(order, x)
    _row_ops.check_device(x.device)
    return _row_ops.dispatch(x if x.dim() == 2 else x.reshape(slots.shape[0], x.shape[-1]), slots)


def combine(rows: Tensor, order: ExpertOrder, gates: Tensor | None = None) -> Tensor:
    """Each token's sum of its choices' rows times their gates: ``(..., width)``.

    Args:
        rows: ``(tokens * k, width)`` in the order's order, fp32, bf16 or fp16; rows may be strided.
        order: of :func:`sort_by_expert`.
        gates: ``(..., k)`` fp32, as :func:`route` gives them, or None for ones. Those of empty choices
            and the rows behind the last expert's reach nothing.

    Differentiable in rows and gates (zeros for what reaches nothing); sums in fp32, rounded once."""
    slots = _slots(order, rows)
    if rows.dim() != 2 or rows.shape[0] != slots.numel():
        raise ValueError(f"rows are ({slots.numel()}, width); got {tuple(rows.shape)}")
    _check_floats("rows", rows)
    if gates is not None:
        _check_on(rows.device, gates)
        if gates.dtype != torch.float32:
            raise TypeError(f"gates are fp32; got {gates.dtype}")
        if gates.shape != order.slots.shape:
            raise ValueError(f"gates are {tuple(order.slots.shape)}; got {tuple(gates.shape)}")
        gates = gates if gates.dim() == 2 else gates.reshape(slots.shape)
    _row_ops.check_device(rows.device)
    y = _row_ops.combine(rows, slots, gates)
    return y if order.slots.dim() == 2 else y.view(*order.slots.shape[:-1], rows.shape[1])


def expert_linear(rows: Tensor, weight: Tensor, offsets: Tensor) -> Tensor:
    """Every expert's matrix on its own rows: ``rows[a:b] @ weight[e].T`` for
    ``a, b = offsets[e], offsets[e + 1]``; zeros behind the last expert's rows.

    Args:
        rows: ``(rows, in)``, fp32, bf16 or fp16, as :func:`dispatch` gives them; rows may be strided.
        weight: ``(experts, out, in)`` of the same type, at most 1024 experts (copied if not
            contiguous).
        offsets: ``(experts + 1,)`` int32, rising from 0, as :func:`sort_by_expert` gives them.

    Differentiable in rows and weight (zeros for the rows behind the last expert's, which reach no
    weight, and for the weight of an expert without rows). 16-bit products are summed in fp32 and
    rounded once. Nothing is copied to the host; the work goes by the experts' rows."""
    if rows.dim() != 2 or weight.dim() != 3 or rows.shape[1] != weight.shape[2]:
        raise ValueError(f"rows are (rows, in), weight is (experts, out, in); got {tuple(rows.shape)} "
                         f"and {tuple(weight.shape)}")
    if rows.dtype not in _FLOATS or weight.dtype != rows.dtype:
        raise TypeError(f"rows and weight are both fp32, bf16 or fp16; got {rows.dtype} and "
                        f"{weight.dtype}")
    experts, out, width = weight.shape
    if not 1 <= experts <= 1024:
        raise ValueError(f"1 to 1024 experts; got {experts}")
    if rows.shape[0] >= 2**31 or max(out, width) > 2**24:
        raise ValueError(f"below 2^31 rows and extents to 2^24; got {tuple(rows.shape)} and "
                         f"{tuple(weight.shape)}")
    _check_on(rows.device, weight, offsets)
    if offsets.dtype != torch.int32:
        raise TypeError(f"offsets are int32; got {offsets.dtype}")
    if offsets.shape != (experts + 1,):
        raise ValueError(f"offsets are ({experts + 1},); got {tuple(offsets.shape)}")
    _row_ops.check_device(rows.device)
    return _row_ops.expert_linear(rows, weight, offsets)
