"""Log probabilities of tokens and the clipped policy loss on them (libmuon_amd
``muon_token_logprobs``, ``muon_policy_loss``). No counterpart in the reference."""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .. import _row_ops
from .heads import _FLOATS, _check_on


class PolicyLoss(NamedTuple):
    """What :func:`policy_loss` returns."""

    loss: Tensor  #: fp32 scalar, differentiable in the logits
    logprobs: Tensor  #: fp32, the tokens' log probabilities (0 where left out), not differentiable


def _check(logits: Tensor, tokens: Tensor, temperature: float) -> None:
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits are (..., vocabulary); got {tuple(logits.shape)}")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits are fp32, bf16 or fp16; got {logits.dtype}")
    _check_on(logits.device, tokens)
    if tokens.dtype != torch.int64:
        raise TypeError(f"tokens are int64; got {tokens.dtype}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens are {tuple(logits.shape[:-1])}; got {tuple(tokens.shape)}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature is 1e-30 to 1e30; got {temperature}")


def _rows(logits: Tensor) -> Tensor:
    flat = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return _row_ops.unit_last(flat)


def _flat(t: Tensor) -> Tensor:
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


def _keeps(logits: Tensor) -> bool:
    """Whether a backward pass may ask for what the forward pass knows of each row."""
    return logits.requires_grad and torch.is_grad_enabled()


def token_logprobs(logits: Tensor, tokens: Tensor, *, temperature: float = 1.0) -> Tensor:
    """``log softmax(logits / temperature)`` at each position's token, in fp32.

    Args:
        logits: ``(..., vocabulary)``, fp32, bf16 or fp16; rows may be strided.
        tokens: ``(...)`` int64. A negative one leaves its position out: 0, with no gradient.
            One outside the vocabulary gives NaN.

    Differentiable in the logits (the negative sum is the cross entropy). One pass over the
    logits; the backward pass reads them once more and keeps two floats a row besides. Positions
    whose incoming gradient is 0 get zeros, whatever their logits hold."""
    _check(logits, tokens, temperature)
    _row_ops.check_device(logits.device)
    out = _row_ops.token_logprobs(_rows(logits), _flat(tokens), temperature, _keeps(logits))[0]
    return out if logits.dim() == 2 else out.view(tokens.shape)


def policy_loss(
    logits: Tensor,
    tokens: Tensor,
    old_logprobs: Tensor,
    advantages: Tensor,
    weights: Tensor,
    ref_logprobs: Tensor | None = None,
    *,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_coef: float = 0.0,
    temperature: float = 1.0,
) -> PolicyLoss:
    """The clipped policy loss over sampled tokens, with a KL term to a reference policy.

    With ``logp`` the tokens' log probabilities and ``r = exp(logp - old_logprobs)``::

        term = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
               + kl_coef (exp(ref - logp) - (ref - logp) - 1)
        loss = sum(weights * term)

    Args:
        logits, tokens, temperature: as for :func:`token_logprobs`.
        old_logprobs, advantages, weights: fp32, shaped like the tokens. Weights carry masks and
            whatever mean is wanted (1 / tokens, 1 / (sequences * length), ...); a position of
            weight 0 (prompt, padding) is not read at all and contributes exactly nothing.
        ref_logprobs: the reference's log probabilities, or None for no KL term.

    Differentiable in the logits alone. In bf16 and fp32, for rows that fit a workgroup's registers
    (163840 and 81920 values), the gradient is made in the forward pass, from one reading of the
    logits, for a loss gradient of 1; for any other one the backward pass makes it again from
    the logits, so that each value is rounded once. fp16, whose unscaled gradient would underflow,
    and longer rows read the logits again in the backward pass."""
    _check(logits, tokens, temperature)
    _check_on(logits.device, old_logprobs, advantages, weights, ref_logprobs)
    shape = tokens.shape
    for name, t in (("old_logprobs", old_logprobs), ("advantages", advantages),
                    ("weights", weights), ("ref_logprobs", ref_logprobs)):
        if t is None:
            continue
        if t.dtype != torch.float32:
            raise TypeError(f"{name} is fp32; got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name} is {tuple(shape)}; got {tuple(t.shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: policy_loss makes one for the logits "
                             "alone (detach it)")
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"the clip range is not negative; got {clip_low}, {clip_high}")
    _row_ops.check_device(logits.device)
    loss, logp, _, _ = _row_ops.policy_loss(
        _rows(logits), _flat(tokens), _flat(old_logprobs), _flat(advantages), _flat(weights),
        None if ref_logprobs is None else _flat(ref_logprobs), clip_low, clip_high, kl_coef,
        temperature, _keeps(logits), False)
    return PolicyLoss(loss, logp if logits.dim() == 2 else logp.view(tokens.shape))
