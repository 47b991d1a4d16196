"""Top-k expert routing with its counts and losses (libmuon_amd ``muon_route``). No counterpart
in the reference."""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .. import _row_ops
from .heads import _FLOATS, _check_on


class Routing(NamedTuple):
    """What :func:`route` returns; leading dimensions are those of its logits."""

    gates: Tensor  #: (..., k) fp32: the chosen experts' shares
    experts: Tensor  #: (..., k) int64: the chosen experts, best first; -1 for an empty slot
    counts: Tensor  #: (experts,) int64: the tokens that chose each expert
    balance_loss: Tensor  #: fp32 scalar: E sum_e counts_e / (k N) * mean_t p_te
    z_loss: Tensor  #: fp32 scalar: mean_t logsumexp_t^2


def route(logits: Tensor, k: int, *, token_mask: Tensor | None = None, normalize: bool = True
          ) -> Routing:
    """Each token's ``k`` best experts by its router logits, with the losses that keep the
    experts' load even and the logits small.

    Args:
        logits: ``(..., experts)``, fp32, bf16 or fp16, at most 1024 experts. An expert at -inf is
            never chosen (a token with fewer than ``k`` others gets empty slots: expert -1, gate 0).
        k: experts per token, at most 64.
        token_mask: ``(...)`` bool, False for tokens (padding) that are sent nowhere and count in
            neither counts nor losses; as do tokens with all logits -inf.
        normalize: gates are the softmax values over the chosen ones' sum, else the values.

    Ties go to the lower index; a NaN logit counts as the largest and makes its token's gates and
    the losses NaN. gates, balance_loss and z_loss are differentiable in the logits (the counts
    in the balance loss are constants); the losses over no token at all are 0."""
    if logits.dim() < 1:
        raise ValueError("logits are (..., experts)")
    experts = logits.shape[-1]
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits are fp32, bf16 or fp16; got {logits.dtype}")
    if not 1 <= experts <= 1024:
        raise ValueError(f"1 to 1024 experts; got {experts}")
    if not 1 <= k <= min(experts, 64):
        raise ValueError(f"k is 1 to {min(experts, 64)} for {experts} experts; got {k}")
    if token_mask is not None:
        _check_on(logits.device, token_mask)
        if token_mask.dtype != torch.bool:
            raise TypeError(f"token_mask is bool; got {token_mask.dtype}")
        if token_mask.shape != logits.shape[:-1]:
            raise ValueError(f"token_mask is {tuple(logits.shape[:-1])}; got "
                             f"{tuple(token_mask.shape)}")
        token_mask = token_mask.reshape(-1).contiguous()
    flat = logits if logits.dim() == 2 else logits.reshape(-1, experts)
    _row_ops.check_device(logits.device)
    gates, chosen, counts, balance, zloss, _ = _row_ops.route(_row_ops.unit_last(flat), k,
                                                              token_mask, normalize)
    if logits.dim() != 2:
        gates, chosen = (t.view(*logits.shape[:-1], k) for t in (gates, chosen))
    return Routing(gates, chosen, counts, balance, zloss)
