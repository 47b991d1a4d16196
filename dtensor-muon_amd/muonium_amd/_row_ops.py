"""The training step's row operators (include/muon_amd.h, "Row operators", "Experts" and "AdamW") as
torch operators of namespace ``muonium_amd``: query and key norm with rotation, expert routing,
token log probabilities, policy loss; tokens to their experts and back, the experts' products, and
the AdamW step.

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
_PYTHON_LIB_PATH = os.path.join(os.path.dirname(_lib.library_path()), "libmuon_amd_python.so")


def _load() -> None:
    if not os.path.exists(_TORCH_LIB_PATH):
        raise ImportError(
            f"muonium_amd: {_TORCH_LIB_PATH} is missing; build it with "
            "`python -c 'import __graft_entry__ as g; g.build()'` "
            "or `make -C dtensor-muon_amd/csrc`"
        )
    _lib.load()  # the library it binds, from the place this package looks in
    torch.ops.load_library(_TORCH_LIB_PATH)


def _module():
    """The module that walks an optimizer's parameters; None where it was built without Python's headers."""
    import importlib.machinery
    import importlib.util

    if not os.path.exists(_PYTHON_LIB_PATH):
        return None
    loader = importlib.machinery.ExtensionFileLoader("libmuon_amd_python", _PYTHON_LIB_PATH)
    return importlib.util.module_from_spec(
        importlib.util.spec_from_loader("libmuon_amd_python", loader))


_load()
module = _module()
_ops = torch.ops.muonium_amd
qk_norm_rope = _ops.qk_norm_rope.default
route = _ops.route.default
token_logprobs = _ops.token_logprobs.default
policy_loss = _ops.policy_loss.default
sort_by_expert = _ops.sort_by_expert.default
dispatch = _ops.dispatch.default
combine = _ops.combine.default
expert_linear = _ops.expert_linear.default
adamw_ = _ops.adamw_.default


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


@_fake("sort_by_expert")
def _(experts, num_experts):
    return (experts.new_empty(experts.shape, dtype=torch.int32),
            experts.new_empty(num_experts + 1, dtype=torch.int32))


@_fake("dispatch")
def _(x, slots):
    return x.new_empty((slots.size(0) * slots.size(1), x.size(1)))


@_fake("combine")
def _(rows, slots, gates):
    return rows.new_empty((slots.size(0), rows.size(1)))


@_fake("combine_backward")
def _(dy, rows, slots, gates, rows_wanted, gates_wanted):
    return (dy.new_empty((slots.size(0) * slots.size(1), dy.size(1)) if rows_wanted else 0),
            gates.new_empty(slots.shape if gates_wanted else 0))


@_fake("expert_linear")
def _(rows, weight, offsets):
    return rows.new_empty((rows.size(0), weight.size(1)))


@_fake("expert_linear_backward_rows")
def _(dy, weight, offsets):
    return dy.new_empty((dy.size(0), weight.size(2)))


@_fake("expert_linear_backward_weight")
def _(dy, rows, offsets):
    return rows.new_empty((offsets.size(0) - 1, dy.size(1), rows.size(1)))


@_fake("adamw_")
def _(params, grads, exp_avgs, exp_avg_sqs, avg_scales, sq_scales, steps, block, lr, beta1, beta2,
      eps, weight_decay, maximize):
    return None
