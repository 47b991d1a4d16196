"""The training step's row operators without a device: what their entry points refuse, what the C
ABI refuses before any launch, the torch.library registrations, and the oracle of the device
tests against torch's own autograd in float64."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from muonium_amd import _lib
from muonium_amd.kernels import policy_loss, qk_norm_rope, route, token_logprobs
from oracle import row_ops_ref as ref

F32 = torch.float32


def t(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call, error, match", [
    (lambda: qk_norm_rope(t(2, 4), t(2, 4)), ValueError, "batch, tokens"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(3, 4, 8)), ValueError, "batch, tokens"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 2, 4, 8)), ValueError, "differ"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 6)), ValueError, "differ"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8, dtype=torch.bfloat16)), TypeError, "both"),
    (lambda: qk_norm_rope(*(t(2, 3, 4, 8, dtype=torch.float64),) * 2), TypeError, "both"),
    (lambda: qk_norm_rope(t(1, 1, 1, 1025), t(1, 1, 1, 1025)), ValueError, "1024"),
    (lambda: qk_norm_rope(t(1, 1, 1, 0), t(1, 1, 1, 0)), ValueError, "1024"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), t(4)), ValueError, "weights"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), t(8), t(8, dtype=torch.float16)), TypeError, "two types"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), t(8, dtype=torch.int32)), TypeError, "weights"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), cos=t(9, 4)), ValueError, "together"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), cos=t(9, 5), sin=t(9, 5)), ValueError, "rotary"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), cos=t(9, 4), sin=t(8, 4)), ValueError, "rotary"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), None, None, *(t(9, 4, dtype=torch.bfloat16),) * 2), TypeError, "fp32"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), None, None, *(t(9, 4).requires_grad_(),) * 2), ValueError, "gradient"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), None, None, t(2, 4), t(2, 4)), ValueError, "2 positions"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), None, None, t(9, 4), t(9, 4), t(3)), TypeError, "int32"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8), None, None, t(9, 4), t(9, 4), t(2, dtype=torch.int64)), ValueError, "positions"),
    (lambda: qk_norm_rope(t(2, 3, 4, 8), t(2, 3, 4, 8)), RuntimeError, "HIP device"),
    (lambda: route(t(3, 4), 0), ValueError, "k is 1"),
    (lambda: route(t(3, 4), 5), ValueError, "k is 1"),
    (lambda: route(t(3, 100), 65), ValueError, "k is 1"),
    (lambda: route(t(3, 1025), 2), ValueError, "1024"),
    (lambda: route(t(3, 4, dtype=torch.int32), 2), TypeError, "logits"),
    (lambda: route(t(3, 4), 2, token_mask=t(3)), TypeError, "bool"),
    (lambda: route(t(3, 4), 2, token_mask=t(4, dtype=torch.bool)), ValueError, "token_mask"),
    (lambda: route(t(3, 4), 2), RuntimeError, "HIP device"),
    (lambda: token_logprobs(t(3, 0), t(3, dtype=torch.int64)), ValueError, "vocabulary"),
    (lambda: token_logprobs(t(3, 4, dtype=torch.float64), t(3, dtype=torch.int64)), TypeError, "logits"),
    (lambda: token_logprobs(t(3, 4), t(3, dtype=torch.int32)), TypeError, "int64"),
    (lambda: token_logprobs(t(3, 4), t(4, dtype=torch.int64)), ValueError, "tokens"),
    (lambda: token_logprobs(t(3, 4), t(3, dtype=torch.int64), temperature=0.0), ValueError, "temperature"),
    (lambda: token_logprobs(t(3, 4), t(3, dtype=torch.int64), temperature=math.nan), ValueError, "temperature"),
    (lambda: token_logprobs(t(3, 4), t(3, dtype=torch.int64), temperature=math.inf), ValueError, "temperature"),
    (lambda: token_logprobs(t(3, 4), t(3, dtype=torch.int64)), RuntimeError, "HIP device"),
    (lambda: policy_loss(t(3, 4), t(3, dtype=torch.int64), t(3), t(3), t(2)), ValueError, "weights"),
    (lambda: policy_loss(t(3, 4), t(3, dtype=torch.int64), t(3), t(3, dtype=torch.bfloat16), t(3)), TypeError, "advantages"),
    (lambda: policy_loss(t(3, 4), t(3, dtype=torch.int64), t(3).requires_grad_(), t(3), t(3)), ValueError, "detach"),
    (lambda: policy_loss(t(3, 4), t(3, dtype=torch.int64), t(3), t(3), t(3), clip_low=-0.1), ValueError, "clip"),
    (lambda: policy_loss(t(3, 4), t(3, dtype=torch.int64), t(3), t(3), t(3), clip_high=math.nan), ValueError, "clip"),
    (lambda: policy_loss(t(3, 4), t(3, dtype=torch.int64), t(3), t(3), t(3)), RuntimeError, "HIP device"),
])
def test_entry_points_refuse(call, error, match):
    with pytest.raises(error, match=match):
        call()


@pytest.mark.parametrize("call, code", [
    (lambda L, s: L.muon_qk_norm_rope(1, 1, None, None, None, 0, None, None, 0, None, 64, 0, 1, 1, 1, 1, 1, 1, 1, 8, 0, 0, 1e-6, None), 5),
    (lambda L, s: L.muon_qk_norm_rope(1, 1, s, None, None, 0, None, None, 0, None, 64, 0, 1, 1, 7, 1, 1, 1, 1, 8, 0, 0, 1e-6, None), 2),
    (lambda L, s: L.muon_qk_norm_rope(1, 1, s, None, None, 0, None, None, 0, None, 64, 0, 1, 1, 1, 1, 1, 1, 1, 1025, 0, 0, 1e-6, None), 1),
    (lambda L, s: L.muon_qk_norm_rope(1, 1, s, None, None, 0, None, None, 0, None, 64, 0, 1, 1, 1, 1, 1, 1, 1, 8, 3, 0, 1e-6, None), 1),
    (lambda L, s: L.muon_qk_norm_rope(1, 1, s, None, None, 0, None, None, 0, None, 64, 0, 1, 1, 1, 1 << 31, 1, 1, 1, 8, 0, 0, 1e-6, None), 1),
    (lambda L, s: L.muon_qk_norm_rope(1, 1, s, None, None, 0, None, None, 9, None, 64, 0, 1, 1, 1, 1, 1, 1, 1, 8, 8, 0, 1e-6, None), 5),
    (lambda L, s: L.muon_qk_norm_rope_backward(1, 1, 1, 1, s, 1, None, 0, None, None, 0, None, 64, 0, 1, 1, 1, None, None, 1, 1, 1, 1, 1, 8, 0, 0, 1e-6, None), 5),
    (lambda L, s: L.muon_route(1, 9, 4, 3, 4, 2, 1, None, 1, 1, 1, 1, 1, 1, 1, None), 2),
    (lambda L, s: L.muon_route(1, 0, 4, 3, 4, 5, 1, None, 1, 1, 1, 1, 1, 1, 1, None), 1),
    (lambda L, s: L.muon_route(1, 0, 4, 3, 4, 2, 1, None, 1, 1, 1, 1, 1, 1, None, None), 5),
    (lambda L, s: L.muon_route_backward(1, 0, 4, 3, 4, 2, 1, None, 1, 1, 1, None, None, None, None, None), 5),
    (lambda L, s: L.muon_token_logprobs(1, 3, 4, 3, 4, 1, 1.0, 1, None, 1, None), 2),
    (lambda L, s: L.muon_token_logprobs(1, 0, 4, 3, 0, 1, 1.0, 1, None, 1, None), 1),
    (lambda L, s: L.muon_token_logprobs(1, 0, 4, 3, 4, 1, -1.0, 1, None, 1, None), 5),
    (lambda L, s: L.muon_token_logprobs(1, 0, 4, 1, 1 << 20, 1, 1.0, 1, None, None, None), 5),
    (lambda L, s: L.muon_token_logprobs_backward(1, 0, 4, 3, 4, 1, 1.0, None, 1, None, 1, None), 5),
    (lambda L, s: L.muon_policy_loss(1, 2, 4, 3, 4, 1, 1, 1, 1, None, 0.2, 0.2, 0.0, 1.0, 1, 1, 1, None, None, 1, None, None), 5),
    (lambda L, s: L.muon_policy_loss(1, 1, 4, 3, 4, 1, 1, 1, 1, None, -0.2, 0.2, 0.0, 1.0, 1, 1, 1, None, None, None, None, None), 5),
    (lambda L, s: L.muon_policy_loss(1, 1, 4, 3, 4, 1, 1, 1, None, None, 0.2, 0.2, 0.0, 1.0, 1, 1, 1, None, None, None, None, None), 5),
    (lambda L, s: L.muon_scale_gradient(1, 5, 4, 1, None), 2),
    (lambda L, s: L.muon_scale_gradient(1, 0, 4, None, None), 5),
])
def test_abi_refuses_without_launching(call, code):
    lib = _lib.load()
    assert call(lib, _lib.i64_array([8] * 12)) == code
    assert _lib.last_error() != ""


def test_abi_calls_with_nothing_to_do_return_ok():
    lib = _lib.load()
    s = _lib.i64_array([8] * 12)
    assert lib.muon_qk_norm_rope(None, None, s, None, None, 0, None, None, 0, None, 64, 0, None, None,
                                 1, 0, 5, 1, 1, 8, 0, 0, 1e-6, None) == 0
    assert lib.muon_route_backward(None, 0, 4, 0, 4, 2, 1, None, None, None, None, None, None, None,
                                   None, None) == 0
    assert lib.muon_token_logprobs(None, 0, 4, 0, 4, None, 1.0, None, None, None, None) == 0
    assert lib.muon_scale_gradient(None, 0, 0, None, None) == 0
    assert lib.muon_policy_loss_one_pass(_lib.DT_BF16, 163840) == 1
    assert lib.muon_policy_loss_one_pass(_lib.DT_BF16, 163841) == 0
    assert lib.muon_policy_loss_one_pass(_lib.DT_F32, 81920) == 1
    assert lib.muon_policy_loss_one_pass(_lib.DT_F16, 100) == 0
    assert lib.muon_route_workspace_bytes(0, 1025) == -1
    assert lib.muon_qk_norm_rope_workspace_bytes(0) == -1
    assert lib.muon_token_logprobs_workspace_bytes(1, 100000, 32000) == 0


def test_registered_ops_run_on_fake_tensors():
    ops = torch.ops.muonium_amd
    with FakeTensorMode():
        q, k = (torch.empty(2, 3, h, 16, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
        w = torch.empty(16, device="cuda")
        cos = torch.empty(9, 8, device="cuda")
        a, b = ops.qk_norm_rope(q, k, w, None, cos, cos, None, 1e-6, False)
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == q.dtype
        g = ops.qk_norm_rope_backward(a, b, q, k, w, None, cos, cos, None, 1e-6, False)
        assert [x.shape for x in g] == [q.shape, k.shape, w.shape, (0,)] and g[2].dtype == F32
        z = torch.empty(5, 8, device="cuda", dtype=torch.float16)
        r = ops.route(z, 2, None, True)
        assert [tuple(x.shape) for x in r] == [(5, 2), (5, 2), (8,), (), (), ()]
        assert ops.route_backward(r[0], None, r[4], z, None, r[1], r[2], r[5], True).dtype == z.dtype
        tok = torch.empty(5, device="cuda", dtype=torch.int64)
        lp, st = ops.token_logprobs(z, tok, 1.0, True)
        assert lp.shape == (5,) and st.shape == (10,)
        assert ops.token_logprobs_backward(lp, z, tok, st, 1.0).shape == z.shape
        loss, _, rows, d = ops.policy_loss(z, tok, lp, lp, lp, None, 0.2, 0.2, 0.0, 1.0, True, False)
        assert d.numel() == 0
        assert loss.shape == () and ops.policy_loss_backward(loss, z, tok, rows, 1.0).shape == z.shape


# ---- the oracle against torch in float64 ------------------------------------------------------


def close(a, b):
    torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-13)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 6, 10])
def test_oracle_norm_rope(interleaved, rotary):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 4, 10, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(10, generator=g, dtype=torch.float64, requires_grad=True)
    angle = torch.rand(3, rotary // 2, generator=g, dtype=torch.float64)
    y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    if rotary:
        head = y[..., :rotary]
        pair = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        pair = torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
        pair = torch.view_as_real(pair)
        pair = pair if interleaved else pair.transpose(-1, -2)
        y = torch.cat([pair.flatten(-2), y[..., rotary:]], -1)
    turned = ref.angles(x, angle.cos(), angle.sin(), None) if rotary else None
    close(ref.norm_rope(x.detach(), w.detach(), turned, 1e-6, interleaved)[0], y.detach())
    dy = torch.randn(y.shape, generator=g, dtype=torch.float64)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    got = ref.norm_rope_grad(x.detach(), w.detach(), dy, turned, 1e-6, interleaved)
    close(got[0], dx)
    close(got[2], dw)


@pytest.mark.parametrize("normalize", [False, True])
def test_oracle_route(normalize):
    g = torch.Generator().manual_seed(2)
    z = torch.randn(20, 9, generator=g, dtype=torch.float64, requires_grad=True)
    mask = torch.rand(20, generator=g) > 0.3
    p = z.softmax(1)
    top = z.topk(3, 1).indices
    gates = p.gather(1, top)
    gates = gates / gates.sum(1, keepdim=True) if normalize else gates
    gates = gates * mask[:, None]
    n = int(mask.sum())
    counts = torch.bincount(top[mask].flatten(), minlength=9)
    balance = 9 * (counts.double() / (3 * n) * p[mask].sum(0) / n).sum()
    zl = z.logsumexp(1)[mask].square().sum() / n
    r = ref.route(z.detach(), 3, mask, normalize)
    close(r["gates"], gates.detach())
    close(r["balance"], balance.detach())
    close(r["z"], zl.detach())
    assert torch.equal(r["counts"], counts) and torch.equal(r["experts"][mask], top[mask])
    grads = [torch.randn(20, 3, generator=g, dtype=torch.float64), torch.tensor(0.7), torch.tensor(0.3)]
    d, = torch.autograd.grad((gates, balance, zl), (z,), [grads[0], *(x.double() for x in grads[1:])])
    close(ref.route_grad(r, grads[0], grads[1].double(), grads[2].double())[0], d)


def test_oracle_policy():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, 30, generator=g, dtype=torch.float64, requires_grad=True)
    tok = torch.randint(0, 30, (12,), generator=g)
    lp = (x / 0.7).log_softmax(1).gather(1, tok[:, None])[:, 0]
    old, adv, w, rf = (torch.randn(12, generator=g, dtype=torch.float64) * s for s in (0.3, 1, 1, 0.3))
    old, rf, w = lp.detach() + old, lp.detach() + rf, w.abs()
    w[::4] = 0
    r = (lp - old).exp()
    loss = (w * (-torch.minimum(r * adv, r.clamp(0.8, 1.3) * adv) + 0.1 * ((rf - lp).exp() - (rf - lp) - 1))).sum()
    d, = torch.autograd.grad(loss, (x,))
    logp, p = ref.logprobs(x.detach(), tok, 0.7)
    close(logp, lp.detach())
    got, slope, _, _ = ref.policy(logp, old, adv, w, rf, 0.2, 0.3, 0.1)
    close(got, loss.detach())
    close(ref.logprobs_grad(p, tok, slope, 0.7)[0], d)
