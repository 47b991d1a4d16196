"""Device operations of the training step's row operators (include/muon_amd.h, "Row operators"):
query and key norm with rotation, expert routing, token log probabilities, policy loss.

Each is an implementation on plain tensors (``_*_impl``: outputs and scratch from torch's
allocator on the current stream, so they may be reused there as soon as the launches are
enqueued), an ``autograd.Function`` around it for eager calls that need gradients, and a
``torch.library`` op of namespace ``muonium_amd`` with a fake implementation and the same
gradient, which calls take while an outer torch.compile traces them.

The arguments are checked in ``muonium_amd.kernels``; here they are taken as they are.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib

_i64x6 = ctypes.c_int64 * 6
_i64x12 = ctypes.c_int64 * 12


def _ptr(t: Tensor | None):
    return None if t is None else t.data_ptr()


def _call(what: str, device: torch.device, *args) -> None:
    """One library call on ``device``'s current stream (appended to ``args``)."""
    _lib.ensure_device(device)
    fn = getattr(_lib.load(), what)
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(*args, _lib.stream(device))
    else:  # launches go to the current device
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream(device))
    _lib.check(rc, what)


def _scratch(nbytes: int, device: torch.device) -> Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ---------------------------------------------------------------------------------
# queries and keys


def _unit_last(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.size(-1) <= 1 else t.contiguous()


def _strides(t: Tensor) -> tuple[int, int, int]:
    """(batch, token, head) strides of a (batch, tokens, heads, dim) or (tokens, heads, dim)
    tensor."""
    s = t.stride()
    return (s[0], s[1], s[2]) if len(s) == 4 else (0, s[0], s[1])


def _qk_args(q: Tensor, k: Tensor, q_weight, k_weight, cos, sin, positions):
    """The arguments that both directions take, by the ABI's names."""
    batch = q.size(0) if q.dim() == 4 else 1
    w = q_weight if q_weight is not None else k_weight
    if positions is None:
        pos = (None, 64, 0)
    else:
        pos = (positions.data_ptr(), 64 if positions.dtype == torch.int64 else 32,
               positions.stride(0) if positions.dim() == 2 else 0)
    front = (_ptr(q_weight), _ptr(k_weight), 0 if w is None else _lib.dtype_code(w.dtype),
             _ptr(cos), _ptr(sin), 0 if cos is None else cos.size(0), *pos)
    extents = (_lib.dtype_code(q.dtype), batch, q.size(-3), q.size(-2), k.size(-2), q.size(-1),
               0 if cos is None else 2 * cos.size(1))
    return front, extents


def _qk_impl(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
             cos: Optional[Tensor], sin: Optional[Tensor], positions: Optional[Tensor],
             eps: float, interleaved: bool) -> tuple[Tensor, Tensor]:
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    front, extents = _qk_args(q, k, q_weight, k_weight, cos, sin, positions)
    _call("muon_qk_norm_rope", q.device, q.data_ptr(), k.data_ptr(),
          _i64x6(*_strides(q), *_strides(k)), *front, q_out.data_ptr(), k_out.data_ptr(), *extents,
          interleaved, eps)
    return q_out, k_out


def _qk_backward_impl(dq_out: Tensor, dk_out: Tensor, q: Tensor, k: Tensor,
                      q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                      cos: Optional[Tensor], sin: Optional[Tensor], positions: Optional[Tensor],
                      eps: float, interleaved: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dq_out, dk_out = _unit_last(dq_out), _unit_last(dk_out)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dqw = q.new_empty(0) if q_weight is None else torch.empty_like(q_weight)
    dkw = q.new_empty(0) if k_weight is None else torch.empty_like(k_weight)
    weights = q_weight is not None or k_weight is not None
    ws = None
    if weights:
        ws = _scratch(_lib.load().muon_qk_norm_rope_workspace_bytes(q.size(-1)), q.device)
    front, extents = _qk_args(q, k, q_weight, k_weight, cos, sin, positions)
    _call("muon_qk_norm_rope_backward", q.device, q.data_ptr(), k.data_ptr(), dq_out.data_ptr(),
          dk_out.data_ptr(), _i64x12(*_strides(q), *_strides(k), *_strides(dq_out),
                                     *_strides(dk_out)),
          *front, dq.data_ptr(), dk.data_ptr(), None if q_weight is None else dqw.data_ptr(),
          None if k_weight is None else dkw.data_ptr(), _ptr(ws), *extents, interleaved, eps)
    return dq, dk, dqw, dkw


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.rest = (eps, interleaved)
        return _qk_impl(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        saved = ctx.saved_tensors
        grads = _qk_backward_impl(dq_out, dk_out, *saved, *ctx.rest)
        return (grads[0], grads[1], None if saved[2] is None else grads[2],
                None if saved[3] is None else grads[3], None, None, None, None, None)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    args = (q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if torch.compiler.is_compiling():
        return torch.ops.muonium_amd.qk_norm_rope(*args)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRope.apply(*args)
    return _qk_impl(*args)


# ---------------------------------------------------------------------------------
# routing


def _route_impl(logits: Tensor, top: int, token_mask: Optional[Tensor], normalize: bool
                ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    n, e = logits.shape
    device = logits.device
    gates = torch.empty((n, top), dtype=torch.float32, device=device)
    experts = torch.empty((n, top), dtype=torch.int64, device=device)
    counts = torch.empty(e, dtype=torch.int64, device=device)
    balance, zloss, kept = (torch.empty((), dtype=torch.float32, device=device) for _ in range(3))
    ws = _scratch(_lib.load().muon_route_workspace_bytes(n, e), device)
    _call("muon_route", device, logits.data_ptr(), _lib.dtype_code(logits.dtype),
          logits.stride(0), n, e, top, normalize, _ptr(token_mask), gates.data_ptr(),
          experts.data_ptr(), counts.data_ptr(), balance.data_ptr(), zloss.data_ptr(),
          kept.data_ptr(), ws.data_ptr())
    return gates, experts, counts, balance, zloss, kept


def _route_backward_impl(dgates: Optional[Tensor], dbalance: Optional[Tensor],
                         dzloss: Optional[Tensor], logits: Tensor, token_mask: Optional[Tensor],
                         experts: Tensor, counts: Tensor, kept: Tensor, normalize: bool) -> Tensor:
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if dgates is not None:
        dgates = dgates.contiguous()
    n, e = logits.shape
    _call("muon_route_backward", logits.device, logits.data_ptr(), _lib.dtype_code(logits.dtype),
          logits.stride(0), n, e, experts.size(1), normalize, _ptr(token_mask),
          experts.data_ptr(), counts.data_ptr(), kept.data_ptr(), _ptr(dgates), _ptr(dbalance),
          _ptr(dzloss), dlogits.data_ptr())
    return dlogits


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top, token_mask, normalize):
        gates, experts, counts, balance, zloss, kept = _route_impl(logits, top, token_mask,
                                                                   normalize)
        ctx.save_for_backward(logits, token_mask, experts, counts, kept)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(experts, counts, kept)
        ctx.set_materialize_grads(False)
        return gates, experts, counts, balance, zloss, kept

    @staticmethod
    @once_differentiable
    def backward(ctx, dgates, _experts, _counts, dbalance, dzloss, _kept):
        return (_route_backward_impl(dgates, dbalance, dzloss, *ctx.saved_tensors, ctx.normalize),
                None, None, None)


def route(logits, top, token_mask, normalize):
    args = (logits, top, token_mask, normalize)
    if torch.compiler.is_compiling():
        return torch.ops.muonium_amd.route(*args)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(*args)
    return _route_impl(*args)


# ---------------------------------------------------------------------------------
# token log probabilities and the policy loss


def _logp_workspace(logits: Tensor) -> Tensor | None:
    n, v = logits.shape
    return _scratch(_lib.load().muon_token_logprobs_workspace_bytes(
        _lib.dtype_code(logits.dtype), n, v), logits.device)


def _logp_impl(logits: Tensor, tokens: Tensor, temperature: float, keep: bool
               ) -> tuple[Tensor, Tensor]:
    n, v = logits.shape
    logp = torch.empty(n, dtype=torch.float32, device=logits.device)
    stats = torch.empty(2 * n if keep else 0, dtype=torch.float32, device=logits.device)
    ws = _logp_workspace(logits)
    _call("muon_token_logprobs", logits.device, logits.data_ptr(),
          _lib.dtype_code(logits.dtype), logits.stride(0), n, v, tokens.data_ptr(), temperature,
          logp.data_ptr(), stats.data_ptr() if keep else None, _ptr(ws))
    return logp, stats


def _logp_backward_impl(dlogp: Tensor, scale: Optional[Tensor], logits: Tensor, tokens: Tensor,
                        stats: Tensor, temperature: float) -> Tensor:
    n, v = logits.shape
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    dlogp = dlogp.contiguous()
    _call("muon_token_logprobs_backward", logits.device, logits.data_ptr(),
          _lib.dtype_code(logits.dtype), logits.stride(0), n, v, tokens.data_ptr(), temperature,
          stats.data_ptr(), dlogp.data_ptr(), _ptr(scale), dlogits.data_ptr())
    return dlogits


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        logp, stats = _logp_impl(logits, tokens, temperature, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.temperature = temperature
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        return _logp_backward_impl(dlogp, None, *ctx.saved_tensors, ctx.temperature), None, None


def token_logprobs(logits, tokens, temperature):
    grad = logits.requires_grad and torch.is_grad_enabled()
    if torch.compiler.is_compiling():
        return torch.ops.muonium_amd.token_logprobs(logits, tokens, temperature, grad)[0]
    if grad:
        return _TokenLogprobs.apply(logits, tokens, temperature)
    return _logp_impl(logits, tokens, temperature, False)[0]


def _policy(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
            temperature, keep, dlogits):
    n, v = logits.shape
    device = logits.device
    # the rows' terms and, for a later gradient, their slopes
    # and statistics, in one allocation
    rows = torch.empty((4 if keep else 1, n), dtype=torch.float32, device=device)
    loss = torch.empty((), dtype=torch.float32, device=device)
    logp = torch.empty(n, dtype=torch.float32, device=device)
    at = rows.data_ptr()
    ws = None if dlogits is not None else _logp_workspace(logits)
    _call("muon_policy_loss", device, logits.data_ptr(), _lib.dtype_code(logits.dtype),
          logits.stride(0), n, v, tokens.data_ptr(), old.data_ptr(), advantages.data_ptr(),
          weights.data_ptr(), _ptr(ref), clip_low, clip_high, kl_coef, temperature,
          loss.data_ptr(), logp.data_ptr(), at, at + 8 * n if keep else None,
          at + 4 * n if keep else None, _ptr(dlogits), _ptr(ws))
    return loss, logp, rows


def _policy_impl(logits: Tensor, tokens: Tensor, old: Tensor, advantages: Tensor, weights: Tensor,
                 ref: Optional[Tensor], clip_low: float, clip_high: float, kl_coef: float,
                 temperature: float, keep: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _policy(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
                   temperature, keep, None)


def _policy_backward_impl(dloss: Tensor, logits: Tensor, tokens: Tensor, rows: Tensor,
                          temperature: float) -> Tensor:
    return _logp_backward_impl(rows[1], dloss, logits, tokens, rows[2:4].view(-1), temperature)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
                temperature):
        dlogits = None
        if _lib.load().muon_policy_loss_one_pass(_lib.dtype_code(logits.dtype), logits.size(1)):
            dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        loss, logp, rows = _policy(logits, tokens, old, advantages, weights, ref, clip_low,
                                   clip_high, kl_coef, temperature, True, dlogits)
        ctx.save_for_backward(logits, tokens, rows)
        ctx.temperature, ctx.dlogits = temperature, dlogits
        ctx.mark_non_differentiable(logp)
        ctx.set_materialize_grads(False)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _logp):
        if dloss is None:
            return (None,) * 10
        # The gradient of the forward pass is handed over once; a second backward pass through
        # the same graph makes its own from the logits.
        dlogits, ctx.dlogits = ctx.dlogits, None
        logits, tokens, rows = ctx.saved_tensors
        if dlogits is None:
            dlogits = _policy_backward_impl(dloss, logits, tokens, rows, ctx.temperature)
        elif dlogits.numel():
            _call("muon_scale_gradient", dlogits.device, dlogits.data_ptr(),
                  _lib.dtype_code(dlogits.dtype), dlogits.numel(), dloss.data_ptr())
        return dlogits, *(None,) * 9


def policy_loss(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
                temperature):
    args = (logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
            temperature)
    grad = logits.requires_grad and torch.is_grad_enabled()
    if torch.compiler.is_compiling():
        return torch.ops.muonium_amd.policy_loss(*args, grad)[:2]
    if grad:
        return _PolicyLoss.apply(*args)
    return _policy_impl(*args, False)[:2]


# ---------------------------------------------------------------------------------
# torch.library registration


def _register_ops() -> None:
    def op(name, impl, fake):
        o = torch.library.custom_op(f"muonium_amd::{name}", impl, mutates_args=())
        o.register_fake(fake)
        return o

    def like(t):
        return t.new_empty(t.shape)

    def weight_like(w, q):
        return q.new_empty(0) if w is None else w.new_empty(w.shape)

    # queries and keys
    forward = op("qk_norm_rope", _qk_impl, lambda q, k, *rest: (like(q), like(k)))
    op("qk_norm_rope_backward", _qk_backward_impl,
       lambda dq_out, dk_out, q, k, qw, kw, *rest: (like(q), like(k), weight_like(qw, q),
                                                     weight_like(kw, q)))

    def qk_setup(ctx, inputs, output):
        ctx.save_for_backward(*inputs[:7])
        ctx.rest = inputs[7:]

    def qk_backward(ctx, dq_out, dk_out):
        saved = ctx.saved_tensors
        g = torch.ops.muonium_amd.qk_norm_rope_backward(dq_out, dk_out, *saved, *ctx.rest)
        return (g[0], g[1], None if saved[2] is None else g[2], None if saved[3] is None else g[3],
                None, None, None, None, None)

    forward.register_autograd(qk_backward, setup_context=qk_setup)

    # routing
    def route_fake(logits, top, token_mask, normalize):
        n, e = logits.shape
        f32 = torch.float32
        return (logits.new_empty((n, top), dtype=f32),
                logits.new_empty((n, top), dtype=torch.int64),
                logits.new_empty(e, dtype=torch.int64), logits.new_empty((), dtype=f32),
                logits.new_empty((), dtype=f32), logits.new_empty((), dtype=f32))

    forward = op("route", _route_impl, route_fake)
    op("route_backward", _route_backward_impl,
       lambda dgates, dbalance, dzloss, logits, *rest: like(logits))

    def route_setup(ctx, inputs, output):
        logits, _, token_mask, ctx.normalize = inputs
        ctx.save_for_backward(logits, token_mask, output[1], output[2], output[5])

    def route_backward(ctx, dgates, _experts, _counts, dbalance, dzloss, _kept):
        return (torch.ops.muonium_amd.route_backward(dgates, dbalance, dzloss, *ctx.saved_tensors,
                                                     ctx.normalize), None, None, None)

    forward.register_autograd(route_backward, setup_context=route_setup)

    # log probabilities and the policy loss
    def logp_fake(logits, tokens, temperature, keep):
        n = logits.size(0)
        return (logits.new_empty(n, dtype=torch.float32),
                logits.new_empty(2 * n if keep else 0, dtype=torch.float32))

    forward = op("token_logprobs", _logp_impl, logp_fake)
    op("token_logprobs_backward", _logp_backward_impl,
       lambda dlogp, scale, logits, *rest: like(logits))

    def logp_setup(ctx, inputs, output):
        ctx.save_for_backward(inputs[0], inputs[1], output[1])
        ctx.temperature = inputs[2]

    def logp_backward(ctx, dlogp, _stats):
        return (torch.ops.muonium_amd.token_logprobs_backward(
            dlogp, None, *ctx.saved_tensors, ctx.temperature), None, None, None)

    forward.register_autograd(logp_backward, setup_context=logp_setup)

    def policy_fake(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
                    temperature, keep):
        n = logits.size(0)
        return (logits.new_empty((), dtype=torch.float32),
                logits.new_empty(n, dtype=torch.float32),
                logits.new_empty((4 if keep else 1, n), dtype=torch.float32))

    forward = op("policy_loss", _policy_impl, policy_fake)
    op("policy_loss_backward", _policy_backward_impl, lambda dloss, logits, *rest: like(logits))

    def policy_setup(ctx, inputs, output):
        ctx.save_for_backward(inputs[0], inputs[1], output[2])
        ctx.temperature = inputs[9]

    def policy_backward(ctx, dloss, _logp, _rows):
        return (torch.ops.muonium_amd.policy_loss_backward(dloss, *ctx.saved_tensors,
                                                           ctx.temperature), *(None,) * 10)

    forward.register_autograd(policy_backward, setup_context=policy_setup)


_register_ops()
