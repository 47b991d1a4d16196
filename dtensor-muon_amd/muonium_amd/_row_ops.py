"""The training step's row operators (include/muon_amd.h, "Row operators") as torch operators of
namespace ``muonium_amd``: query and key norm with rotation, expert routing, token log
probabilities, policy loss.

Schemas, device implementations and gradients are in csrc/row_ops.cpp
(``libmuon_amd_torch.so``, built beside ``libmuon_amd.so``); the fake implementations here let an
outer torch.compile trace them. The arguments are checked in ``muonium_amd.kernels``; here they
are taken as they are.
"""

from __future__ import annotations

import os

import torch
from torch import Tensor

from . import _lib

_TORCH_LIB_PATH = os.path.join(os.path.dirname(_lib.library_path()), "libmuon_amd_torch.so")


def _load() -> None:
    if not os.path.exists(_TORCH_LIB_PATH):
        raise ImportError(
            f"muonium_amd: {_TORCH_LIB_PATH} is missing; build it with "
            "`python -c 'import __graft_entry__ as g; g.build()'` "
            "or `make -C dtensor-muon_amd/csrc`"
        )
    _lib.load()  # the library it binds, from the place this package looks in
    torch.ops.load_library(_TORCH_LIB_PATH)


_load()
_ops = torch.ops.muonium_amd
qk_norm_rope = _ops.qk_norm_rope.default
route = _ops.route.default
token_logprobs = _ops.token_logprobs.default
policy_loss = _ops.policy_loss.default


def unit_last(t: Tensor) -> Tensor:
    """t with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.size(-1) <= 1 else t.contiguous()


def check_device(device: torch.device) -> None:
    """A gfx950 whose code objects load (looked at once per device)."""
    if not torch.compiler.is_compiling():
        _lib.ensure_device(device)


# ---------------------------------------------------------------------------------
# fake implementations


def _fake(name):
    return torch.library.register_fake(f"muonium_amd::{name}")


def _like(t: Tensor) -> Tensor:
    return t.new_empty(t.shape)


@_fake("qk_norm_rope")
def _(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    return _like(q), _like(k)


@_fake("qk_norm_rope_backward")
def _(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    return (_like(q), _like(k), q.new_empty(0) if q_weight is None else _like(q_weight),
            k.new_empty(0) if k_weight is None else _like(k_weight))


@_fake("route")
def _(logits, top, token_mask, normalize):
    n, e = logits.shape
    f32, i64 = torch.float32, torch.int64
    return (logits.new_empty((n, top), dtype=f32), logits.new_empty((n, top), dtype=i64),
            logits.new_empty(e, dtype=i64), logits.new_empty((), dtype=f32),
            logits.new_empty((), dtype=f32), logits.new_empty((), dtype=f32))


@_fake("route_backward")
def _(dgates, dbalance, dzloss, logits, token_mask, experts, counts, kept, normalize):
    return _like(logits)


@_fake("token_logprobs")
def _(logits, tokens, temperature, keep):
    n = logits.size(0)
    return (logits.new_empty(n, dtype=torch.float32),
            logits.new_empty(2 * n if keep else 0, dtype=torch.float32))


@_fake("token_logprobs_backward")
def _(dlogp, logits, tokens, stats, temperature):
    return _like(logits)


@_fake("policy_loss")
def _(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef, temperature,
      keep, one_pass):
    n = logits.size(0)
    return (logits.new_empty((), dtype=torch.float32), logits.new_empty(n, dtype=torch.float32),
            logits.new_empty((4 if keep else 1, n), dtype=torch.float32),
            _like(logits) if one_pass else logits.new_empty(0))


@_fake("policy_loss_backward")
def _(dloss, logits, tokens, rows, temperature):
    return _like(logits)


@_fake("policy_loss_rescale_")
def _(dlogits, dloss, logits, tokens, rows, temperature):
    return None
