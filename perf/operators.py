"""Performance cases of the training step's row operators: what a program that trains (or samples
from) a decoder calls of this package besides the optimizer's step.

Four operators, each through its public entry point:

* ``qk``: ``qk_norm_rope``, the per-head norm of queries and keys with the position rotation. The
  queries and keys are slices of one fused projection's output, ``batch x tokens x heads x dim``.
* ``route``: ``route``, the top-k choice of experts with the per-expert counts, the balance loss
  and the z loss.
* ``logp``: ``token_logprobs``, the log probability of each position's token over a vocabulary.
* ``policy``: ``policy_loss``, the clipped policy loss with a KL term on such a vocabulary.

``mode`` is ``forward`` (inference: no gradient is asked for) or ``train`` (outputs and the
gradients of every differentiable input, as a backward pass asks for them).
"""

import functools
import importlib
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "dtensor-muon_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
EPS = 1e-6
BALANCE_COEF, Z_COEF = 1e-2, 1e-3


def _qk(**kw):
    return {"kind": "qk", "mode": "train", "dtype": "bf16", "batch": 1, "tokens": 1, "q_heads": 32,
            "k_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, **kw}


def _route(**kw):
    return {"kind": "route", "mode": "train", "dtype": "fp32", "tokens": 1, "experts": 64, "top": 8,
            "normalize": True, "masked": 0.0, **kw}


def _logp(**kw):
    return {"kind": "logp", "mode": "train", "dtype": "bf16", "rows": 1, "vocab": 32000,
            "temperature": 1.0, **kw}


def _policy(**kw):
    return {"kind": "policy", "mode": "train", "dtype": "bf16", "rows": 1, "vocab": 32000,
            "temperature": 1.0, "masked": 0.0, "reference": True, **kw}


def listed():
    return [
        # one new token of 16 sequences, each at its own position: nothing but latency
        _qk(name="qk decode", mode="forward", batch=16),
        # one layer's pass over a training batch of the Llama-3-8B-shaped heads
        _qk(name="qk train", batch=4, tokens=8192),
        # 12 heads of 64 (the small model's), fp32, a quarter rotated in pairs, a ragged length
        _qk(name="qk train fp32 ragged", dtype="fp32", batch=3, tokens=1021, q_heads=12, k_heads=12,
            dim=64, rotary=16, interleaved=True),
        # the router of 64 experts for a few sequences' new tokens
        _route(name="route decode", mode="forward", tokens=48),
        # the same router over a training batch, padding masked out
        _route(name="route train", tokens=32768, masked=0.1),
        # many experts and tokens in half precision, gates as they are
        _route(name="route train wide", dtype="bf16", tokens=131071, experts=256, normalize=False),
        # the tokens that eight sequences just sampled
        _logp(name="logp decode", mode="forward", dtype="fp32", rows=8, vocab=128000),
        # old and reference values of a batch of samples
        _logp(name="logp score", mode="forward", rows=8192, vocab=128000, temperature=0.7),
        # cross entropy's gradient on a vocabulary of odd size
        _logp(name="logp train odd", rows=2047, vocab=50257),
        # a short answer's update
        _policy(name="policy small", rows=61, vocab=32000, reference=False),
        # a batch of long answers behind their prompts, whose positions weigh nothing
        _policy(name="policy train", rows=6144, vocab=128000, masked=0.25, temperature=0.7),
        # an odd vocabulary in fp32
        _policy(name="policy fp32 odd", dtype="fp32", rows=1500, vocab=50257, masked=0.1),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    largest = {kind: max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
               for kind in ("qk", "route", "logp", "policy")}
    while True:
        kind = rng.choice(("qk", "route", "logp", "policy"))
        mode = rng.choice(("forward", "train", "train"))
        if kind == "qk":
            dim = rng.choice((64, 96, 128, 128, 160, 256, 8 * rng.randint(4, 32) + 2))
            rotary = rng.choice((dim, dim, 2 * (dim // 4)))
            k_heads = _log_uniform(rng, 1, 16)
            case = _qk(mode=mode, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                       batch=_log_uniform(rng, 1, 64),
                       tokens=1 if rng.random() < 0.15 else _log_uniform(rng, 1, 16384),
                       k_heads=k_heads, q_heads=k_heads * rng.choice((1, 2, 4, 7, 8)), dim=dim,
                       rotary=rotary, interleaved=rng.random() < 0.3)
        elif kind == "route":
            experts = rng.choice((8, 16, 64, 128, 256, _log_uniform(rng, 4, 512)))
            case = _route(mode=mode, dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")),
                          tokens=_log_uniform(rng, 1, 131072), experts=experts,
                          top=rng.randint(1, min(experts, 10)), normalize=rng.random() < 0.6,
                          masked=rng.choice((0.0, 0.0, 0.1, 0.5)))
        else:
            rows, vocab = _log_uniform(rng, 1, 8192), _log_uniform(rng, 1000, 160000)
            if rng.random() < 0.5:
                vocab = max(8, vocab // 128 * 128)
            dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
            temperature = rng.choice((1.0, 1.0, 0.7))
            if kind == "logp":
                case = _logp(mode=mode, dtype=dtype, rows=rows, vocab=vocab,
                             temperature=temperature)
            else:
                case = _policy(mode="train", dtype=dtype, rows=rows, vocab=vocab,
                               temperature=temperature, masked=rng.choice((0.0, 0.25, 0.6)),
                               reference=rng.random() < 0.7)
        if work(case)["bytes"] <= largest[kind]:
            return case


def _masked_rows(case, n):
    return int(n * case["masked"])


def _loss_scale(case):
    """What a half-precision run multiplies its loss by, so that the smallest slopes stay above
    the type's least value (a mean over n positions divides them by n)."""
    n = case["rows" if "rows" in case else "tokens"]
    return 1.0 if case["dtype"] != "fp16" else n * (64.0 if case["kind"] == "route" else 2048.0)


def work(case):
    """Each input read once and each output written once; the tables, tokens and per-row values
    are counted where they are not lost in the rounding."""
    es, train = BYTES[case["dtype"]], case["mode"] == "train"
    if case["kind"] == "qk":
        heads = case["q_heads"] + case["k_heads"]
        n = case["batch"] * case["tokens"] * heads * case["dim"]
        tables = case["batch"] * case["tokens"] * (8 + case["rotary"] * 4)
        return {"bytes": n * es * (4 if train else 2) + tables, "flops": n * (20 if train else 7)}
    if case["kind"] == "route":
        n = case["tokens"] * case["experts"]
        rows = case["tokens"] * (12 * case["top"] + 1)
        return {"bytes": n * es * (2 if train else 1) + rows * (2 if train else 1) + 8 * case["experts"],
                "flops": n * (15 if train else 5)}
    rows = case["rows"]
    read = rows - (_masked_rows(case, rows) if case["kind"] == "policy" else 0)
    per_row = 12 if case["kind"] == "logp" else 28
    return {"bytes": (read + (rows if train else 0)) * case["vocab"] * es + rows * per_row,
            "flops": read * case["vocab"] * (8 if train else 4)}


# ---- inputs ------------------------------------------------------------------------------


def _chunks(rows, vocab):
    """Row ranges of about 2^27 values, for what is made in 32 or 64 bits beside large logits."""
    step = max(1, (1 << 27) // vocab)
    return [slice(r, min(rows, r + step)) for r in range(0, rows, step)]


def _logits_and_tokens(case, g):
    """Logits as a head leaves them (spread 2 to 3, a few tokens far ahead of the rest) and one
    token a row, drawn from the distribution itself, with its log probability."""
    rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    logits = torch.empty(rows, vocab, dtype=dt, device="cuda")
    tokens = torch.empty(rows, dtype=torch.int64, device="cuda")
    logp = torch.empty(rows, dtype=torch.float32, device="cuda")
    for r in _chunks(rows, vocab):
        x = torch.randn(r.stop - r.start, vocab, generator=g, device="cuda")
        logits[r] = x.mul_(2.2).add_(x.pow(3), alpha=0.01)
        x = logits[r].float().div_(case["temperature"])
        noise = torch.rand(x.shape, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
        tokens[r] = (x - noise.log_().neg_().log_()).argmax(1)
        x -= x.amax(1, keepdim=True)
        picked = x.gather(1, tokens[r, None])[:, 0]
        logp[r] = picked - x.exp_().sum(1).log_()
    return logits, tokens, logp


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    if case["kind"] == "qk":
        b, t, hq, hk, d = (case[k] for k in ("batch", "tokens", "q_heads", "k_heads", "dim"))
        qkv = randn(b, t, hq + 2 * hk, d, dtype=dt)
        qkv.mul_(torch.exp(0.3 * randn(1, 1, hq + 2 * hk, 1)).to(dt))
        weights = [(1 + 0.2 * randn(d)).to(dt) for _ in range(2)]
        half = case["rotary"] // 2
        length = max(4096, t) + 1000
        angle = torch.arange(length, device="cuda")[:, None] * torch.exp(
            torch.arange(half, device="cuda") * (-math.log(500000.0) / half))
        # one new token of each sequence at its own place, or whole sequences that start anywhere
        start = torch.randint(0, length - t + 1, (b, 1), generator=g, device="cuda")
        state = {"q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk], "weights": weights,
                 "cos": angle.cos(), "sin": angle.sin(),
                 "positions": start + torch.arange(t, device="cuda")}
        if train:
            state["grads"] = [randn(b, t, h, d, dtype=dt) for h in (hq, hk)]
            state["q"] = state["q"].detach().requires_grad_()
            state["k"] = state["k"].detach().requires_grad_()
            state["weights"] = [w.requires_grad_() for w in weights]
    elif case["kind"] == "route":
        n, e, k = case["tokens"], case["experts"], case["top"]
        # some experts are liked more than others
        logits = (randn(n, e) * 1.5 + 0.7 * randn(1, e)).to(dt)
        mask = None
        if case["masked"]:
            mask = torch.ones(n, dtype=torch.bool, device="cuda")
            mask[torch.randperm(n, generator=g, device="cuda")[:_masked_rows(case, n)]] = False
        state = {"logits": logits.requires_grad_(train), "mask": mask}
        if train:
            scale = _loss_scale(case)
            state["grads"] = [randn(n, k) * (scale / n),
                              torch.full((), BALANCE_COEF * scale, device="cuda"),
                              torch.full((), Z_COEF * scale, device="cuda")]
    else:
        n = case["rows"]
        logits, tokens, logp = _logits_and_tokens(case, g)
        state = {"logits": logits.requires_grad_(train), "tokens": tokens}
        if case["kind"] == "logp":
            if train:
                state["grads"] = -(0.5 + torch.rand(n, generator=g, device="cuda")) * (
                    _loss_scale(case) / n)
        else:
            # the policy has moved a little from the one that sampled, and further from the
            # reference. A ratio at the clip's very edge would have its gradient decided by the
            # last bit of a logarithm: those are moved off it
            moved = 0.15 * randn(n)
            for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
                moved = torch.where((moved - edge).abs() < 1e-3, moved + 2e-3, moved)
            weights = torch.full((n,), 1.0 / n, device="cuda") * (
                0.5 + torch.rand(n, generator=g, device="cuda"))
            order = torch.randperm(n, generator=g, device="cuda")
            weights[order[:_masked_rows(case, n)]] = 0.0
            state |= {"old": logp - moved, "advantages": 0.75 + randn(n), "weights": weights,
                      "ref": logp + 0.3 * randn(n) if case["reference"] else None,
                      "grads": torch.full((), _loss_scale(case), device="cuda")}
    return {"case": case, **state}


# ---- one pass ----------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return globals()["_plain_" + state["case"]["kind"]](state)


@functools.cache
def _kernels():
    return importlib.import_module("muonium_amd.kernels")


def _run_own(state):
    K, case = _kernels(), state["case"]
    train = case["mode"] == "train"
    if case["kind"] == "qk":
        wq, wk = state["weights"]
        outs = K.qk_norm_rope(state["q"], state["k"], wq, wk, state["cos"], state["sin"],
                              state["positions"], eps=EPS, interleaved=case["interleaved"])
        if not train:
            return list(outs)
        return [*outs, *torch.autograd.grad(outs, (state["q"], state["k"], wq, wk), state["grads"])]
    if case["kind"] == "route":
        r = K.route(state["logits"], case["top"], token_mask=state["mask"],
                    normalize=case["normalize"])
        outs = [r.gates, r.experts, r.counts, r.balance_loss, r.z_loss]
        if train:
            outs += torch.autograd.grad((r.gates, r.balance_loss, r.z_loss), (state["logits"],),
                                        state["grads"])
        return outs
    if case["kind"] == "logp":
        logp = K.token_logprobs(state["logits"], state["tokens"], temperature=case["temperature"])
        if not train:
            return [logp]
        return [logp, *torch.autograd.grad((logp,), (state["logits"],), (state["grads"],))]
    r = K.policy_loss(state["logits"], state["tokens"], state["old"], state["advantages"],
                      state["weights"], state["ref"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                      kl_coef=KL_COEF, temperature=case["temperature"])
    return [r.loss, r.logprobs,
            *torch.autograd.grad((r.loss,), (state["logits"],), (state["grads"],))]


# ---- the plain forms: elementary torch operations in 32 bits -------------------------------


def _turn(x, c, s, case):
    """The rotation of the first ``rotary`` components by the angles of cosine c and sine s."""
    n = case["rotary"]
    head, rest = x[..., :n], x[..., n:]
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)
    a, b = head[..., :n // 2], head[..., n // 2:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def _plain_qk(state):
    case = state["case"]
    c = state["cos"][state["positions"]][:, :, None]
    s = state["sin"][state["positions"]][:, :, None]
    outs, dx, dw = [], [], []
    for i, name in enumerate("qk"):
        x, w = state[name].float(), state["weights"][i].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xhat = x * r
        outs.append(_turn(xhat * w, c, s, case).to(state[name].dtype))
        if case["mode"] == "train":
            u = _turn(state["grads"][i].float(), c, -s, case)
            dw.append((u * xhat).sum((0, 1, 2)).to(state["weights"][i].dtype))
            u *= w
            dx.append((r * (u - xhat * (u * xhat).mean(-1, keepdim=True))).to(state[name].dtype))
    return outs + dx + dw


def _plain_route(state):
    case, mask = state["case"], state["mask"]
    n, e, k = case["tokens"], case["experts"], case["top"]
    z = state["logits"].float()
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    p = p / total
    lse = (top + torch.log(total))[:, 0]
    experts = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    gates = p.gather(1, experts)
    held = gates.sum(1, keepdim=True) if case["normalize"] else torch.ones_like(total)
    gates = gates / held
    tokens = torch.full((), n, device=z.device)
    if mask is not None:
        tokens = mask.sum()
        p, lse = p * mask[:, None], lse * mask
        gates = gates * mask[:, None]
        experts = torch.where(mask[:, None], experts, -1)
    at = experts % (e + 1)  # a masked token's -1 goes to a place of its own, past the last expert
    counts = at.new_zeros(e + 1).scatter_add_(0, at.flatten(), torch.ones_like(at).flatten())[:e]
    share = counts.float() / (k * tokens)
    balance = e * (share * p.sum(0) / tokens).sum()
    z_loss = (lse * lse).sum() / tokens
    outs = [gates, experts, counts, balance, z_loss]
    if case["mode"] == "train":
        dgates, dbalance, dz = state["grads"]
        a = dbalance * e * share / tokens
        dlogits = p * (a - (p * a).sum(1, keepdim=True)) + p * (2 * dz / tokens * lse)[:, None]
        part = gates * dgates
        inner = part.sum(1, keepdim=True)
        if case["normalize"]:
            part = part - gates * inner
        else:
            dlogits -= p * inner
        dlogits = torch.cat([dlogits, torch.zeros_like(total)], 1)
        dlogits.scatter_add_(1, at, part)
        outs.append(dlogits[:, :e].to(state["logits"].dtype).contiguous())
    return outs


def _plain_logp(state):
    case = state["case"]
    x = state["logits"].float() / case["temperature"]
    x = x - x.amax(1, keepdim=True)
    x -= torch.log(torch.exp(x).sum(1, keepdim=True))
    at = state["tokens"][:, None]
    logp = x.gather(1, at)[:, 0]
    if case["mode"] == "forward":
        return [logp]
    slope = (state["grads"] / case["temperature"])[:, None]
    d = torch.exp_(x).mul_(-slope).scatter_add_(1, at, slope)
    return [logp, d.to(state["logits"].dtype)]


def _plain_policy(state):
    case, w = state["case"], state["weights"]
    x = state["logits"].float() / case["temperature"]
    x = x - x.amax(1, keepdim=True)
    x -= torch.log(torch.exp(x).sum(1, keepdim=True))
    at = state["tokens"][:, None]
    logp = x.gather(1, at)[:, 0]
    ratio, adv = torch.exp(logp - state["old"]), state["advantages"]
    term = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    inside = torch.where(adv >= 0, ratio <= 1 + CLIP_HIGH, ratio >= 1 - CLIP_LOW)
    slope = -ratio * adv * inside
    if state["ref"] is not None:
        ahead = state["ref"] - logp
        term = term + KL_COEF * (torch.exp(ahead) - ahead - 1)
        slope = slope + KL_COEF * (1 - torch.exp(ahead))
    loss = (w * term)[w != 0].sum()
    slope = torch.where(w != 0, w * slope, 0) * (state["grads"] / case["temperature"])
    slope = slope[:, None]
    d = torch.exp_(x).mul_(-slope).scatter_add_(1, at, slope)
    return [loss, torch.where(w != 0, logp, 0), d.to(state["logits"].dtype)]


# ---- the definitions in 64 bits: the gradients are autograd's -------------------------------


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))


def _leaf(x):
    return x.detach().double().requires_grad_()


def _exact_qk(case, state):
    cos, sin = (state[n].double()[state["positions"]].unsqueeze(2) for n in ("cos", "sin"))
    half = case["rotary"] // 2
    turn = torch.complex(cos, sin)
    outs, dx, dw = [], [], []
    for i, name in enumerate("qk"):
        x, w = state[name].detach(), _leaf(state["weights"][i])
        out, slope = torch.empty(x.shape, dtype=torch.float64, device="cuda"), None
        if case["mode"] == "train":
            slope, total = torch.empty_like(out), torch.zeros_like(w)
        for h in range(x.shape[2]):  # a head at a time: 64 bits take room
            one = _leaf(x[:, :, h:h + 1])
            y = one / torch.sqrt(one.square().mean(-1, keepdim=True) + EPS) * w
            first, rest = y[..., :2 * half], y[..., 2 * half:]
            if case["interleaved"]:
                pair = first.unflatten(-1, (half, 2))
            else:
                pair = first.unflatten(-1, (2, half)).transpose(-1, -2)
            pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            pair = pair if case["interleaved"] else pair.transpose(-1, -2)
            y = torch.cat([pair.flatten(-2), rest], -1)
            out[:, :, h:h + 1] = y.detach()
            if slope is not None:
                gx, gw = torch.autograd.grad(y, (one, w), state["grads"][i][:, :, h:h + 1].double())
                slope[:, :, h:h + 1] = gx
                total += gw
        outs.append(out)
        if slope is not None:
            dx.append(slope)
            dw.append(total)
    return outs + dx + dw


def _exact_route(case, state):
    z = _leaf(state["logits"])
    n, e, k = case["tokens"], case["experts"], case["top"]
    keep = torch.ones(n, dtype=torch.bool, device="cuda") if state["mask"] is None else state["mask"]
    p = torch.softmax(z, 1)
    experts = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :k]
    gates = p.gather(1, experts)
    if case["normalize"]:
        gates = gates / gates.sum(1, keepdim=True)
    gates = torch.where(keep[:, None], gates, 0.0)
    counts = torch.bincount(experts[keep].flatten(), minlength=e)
    kept = keep.sum().double()
    balance = e * (counts.double() / (k * kept) * p[keep].sum(0) / kept).sum()
    z_loss = torch.logsumexp(z, 1)[keep].square().sum() / kept
    outs = [gates.detach(), torch.where(keep[:, None], experts, -1), counts, balance.detach(),
            z_loss.detach()]
    if case["mode"] == "train":
        outs += torch.autograd.grad((gates, balance, z_loss), (z,),
                                    [d.double() for d in state["grads"]])
    return outs


def _exact_logp(case, state):
    logp = torch.empty(case["rows"], dtype=torch.float64, device="cuda")
    slopes = []
    for r in _chunks(case["rows"], case["vocab"]):
        z = _leaf(state["logits"][r])
        y = torch.log_softmax(z / case["temperature"], 1).gather(1, state["tokens"][r, None])[:, 0]
        logp[r] = y.detach()
        if case["mode"] == "train":
            slopes += torch.autograd.grad(y, (z,), state["grads"][r].double())
    return [logp, torch.cat(slopes)] if slopes else [logp]


def _exact_policy(case, state):
    rows = case["rows"]
    logp = torch.zeros(rows, dtype=torch.float64, device="cuda")
    loss, slopes = 0.0, []
    for r in _chunks(rows, case["vocab"]):
        z = _leaf(state["logits"][r])
        w = state["weights"][r].double()
        y = torch.log_softmax(z / case["temperature"], 1).gather(1, state["tokens"][r, None])[:, 0]
        ratio, adv = (y - state["old"][r].double()).exp(), state["advantages"][r].double()
        term = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
        if state["ref"] is not None:
            ahead = state["ref"][r].double() - y
            term = term + KL_COEF * (ahead.exp() - ahead - 1)
        part = (w * term).sum()
        slopes += torch.autograd.grad((part,), (z,), (state["grads"].double(),))
        loss = loss + part.detach()
        logp[r] = torch.where(w != 0, y.detach(), 0.0)
    return [loss, logp, torch.cat(slopes)]
