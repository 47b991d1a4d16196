"""Performance cases of what a decoder with experts trains and answers with around ``route`` and the
``Muon`` step: the routed tokens brought to their experts and back, the experts' products, and the
step of the parameters that are no matrices.

Four operators, each through its public entry point:

* ``dispatch``: ``sort_by_expert`` and ``dispatch``, the order of the routed tokens by expert and their
  rows in that order.
* ``combine``: ``combine``, each token's sum of its experts' rows with its gates.
* ``product``: ``expert_linear``, every expert's matrix on its own rows.
* ``adamw``: ``AdamW`` and ``AdamWFp8``, one step over all tensors of a group.

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
KINDS = ("dispatch", "combine", "product", "adamw")
LR, WD, BETAS, EPS, STEPS = 3e-4, 0.1, (0.9, 0.95), 1e-8, 100
BLOCK = 256  # values that share a scale in fp8 state


def _dispatch(**kw):
    return {"kind": "dispatch", "mode": "train", "dtype": "bf16", "tokens": 1, "experts": 64,
            "top": 8, "width": 2048, "masked": 0.0, **kw}


def _combine(**kw):
    return {**_dispatch(**kw), "kind": "combine"}


def _product(**kw):
    return {"kind": "product", "mode": "train", "dtype": "bf16", "tokens": 1, "experts": 64,
            "top": 8, "width": 2048, "out": 1408, **kw}


def _adamw(**kw):
    return {"kind": "adamw", "mode": "train", "dtype": "bf16", "state": "fp32", **kw}


def listed():
    return [
        # the new tokens of 16 sequences, each with 8 of 64 experts: nothing but latency
        _dispatch(name="dispatch decode", mode="forward", tokens=16),
        # one layer's pass over a training batch, a tenth of it padding that is sent nowhere
        _dispatch(name="dispatch train", tokens=32768, masked=0.1),
        # two experts each, fp32, odd numbers of tokens and columns
        _dispatch(name="dispatch train fp32 odd", dtype="fp32", tokens=8191, experts=8, top=2,
                  width=1001),
        # the same tokens' way back
        _combine(name="combine decode", mode="forward", tokens=16),
        _combine(name="combine train", tokens=32768, masked=0.1),
        # a ragged width in fp16, as many experts as one token takes in a wide model
        _combine(name="combine train fp16 odd", dtype="fp16", tokens=5001, experts=60, top=6,
                 width=1411),
        # the first product of the stacked experts (1408 x 2048) on those 16 tokens: every
        # weight that is met has to be read
        _product(name="product decode", mode="forward", tokens=16),
        # the same on a training batch, with the gradients of rows and weights
        _product(name="product train", tokens=32768),
        # a small model's experts in fp32 at odd widths
        _product(name="product train fp32 odd", dtype="fp32", tokens=2047, experts=8, top=2,
                 width=769, out=1001),
        # the gains of 32 layers' norms and heads: many small tensors
        _adamw(name="adamw gains", sizes="4096*65 128*64"),
        # the small model's embeddings, biases and gains, in fp32
        _adamw(name="adamw fp32 odd", dtype="fp32", sizes="50257x768 1024x768 2304*12 768*49"),
        # embedding and head of a large vocabulary, with the moments in 8 bits
        _adamw(name="adamw fp8 embeddings", state="fp8", sizes="64000x4096*2"),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    largest = {kind: max(_cost(c) for c in listed() if c["kind"] == kind) for kind in KINDS}
    while True:
        kind, dtype = rng.choice(KINDS), rng.choice(("bf16", "bf16", "fp16", "fp32"))
        if kind == "adamw":
            state = rng.choice(("fp32", "fp32", "fp8"))
            sizes = []
            for _ in range(rng.randint(1, 4)):
                n = _log_uniform(rng, 1, 1 << 27)
                if state == "fp8":  # smaller tensors and ragged ones keep their moments in fp32
                    n = BLOCK * max(4096 // BLOCK, n // BLOCK)
                sizes.append(f"{n}*{_log_uniform(rng, 1, 60)}")
            case = _adamw(dtype=dtype, state=state, sizes=" ".join(sizes))
        else:
            experts = rng.choice((8, 64, 128, _log_uniform(rng, 2, 256)))
            case = {"mode": rng.choice(("forward", "train", "train")), "dtype": dtype,
                    "tokens": _log_uniform(rng, 1, 32768), "experts": experts,
                    "top": rng.randint(1, min(experts, 8))}
            width, out = (_log_uniform(rng, 16, 4096) for _ in range(2))
            if rng.random() < 0.7:
                width, out = (64 * max(1, n // 64) for n in (width, out))
            if kind == "product":
                case = _product(**case, width=width, out=out)
            else:
                case = (_dispatch if kind == "dispatch" else _combine)(
                    **case, width=width, masked=rng.choice((0.0, 0.0, 0.1, 0.5)))
        if _cost(case) <= largest[kind]:
            return case


def _sizes(case):
    """The shapes of a text such as "50257x768 128*3"."""
    shapes = []
    for part in case["sizes"].split():
        shape, _, times = part.partition("*")
        shapes += [tuple(int(n) for n in shape.split("x"))] * int(times or 1)
    return shapes


def _kept(case):
    """Tokens that are sent to experts, and their rows."""
    tokens = case["tokens"] - int(case["tokens"] * case.get("masked", 0.0))
    return tokens, tokens * case["top"]


def work(case):
    """Each input read once and each output written once, rows of padding aside: the order's
    numbers are 8 bytes an expert id read and 4 a slot written; of an expert's weights, as many as
    its rows can meet."""
    es, train = BYTES[case["dtype"]], case["mode"] == "train"
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _sizes(case))
        return {"bytes": n * (3 * es + (16 if case["state"] == "fp32" else 4)), "flops": 15 * n}
    tokens, rows = _kept(case)
    w = case["width"]
    if case["kind"] == "product":
        o, met = case["out"], min(case["experts"], rows)
        once = rows * (w + o) + met * w * o
        return {"bytes": es * once * (2 if train else 1), "flops": 2 * rows * w * o * (3 if train else 1)}
    there = (rows + tokens) * w * es
    if case["kind"] == "dispatch":
        return {"bytes": there * (2 if train else 1) + 12 * case["tokens"] * case["top"],
                "flops": rows * w if train else 0}
    # the rows and the outputs' gradient are each read once and their gradient written
    return {"bytes": there * (2 if train else 1) + 8 * rows * (2 if train else 1),
            "flops": rows * w * (5 if train else 2)}


def _cost(case):
    """What a case takes of the card in its plain form: bytes, or for products what 32 bits cost."""
    w = work(case)
    return max(w["bytes"], w["flops"] / 20)


# ---- inputs ------------------------------------------------------------------------------


def _routed(case, g):
    """Experts of each token, best first, as a router chooses them: some are liked more than
    others; -1 for padding."""
    t, e = case["tokens"], case["experts"]
    liked = torch.randn(1, e, generator=g, device="cuda")
    scores = 1.5 * torch.randn(t, e, generator=g, device="cuda") + 0.7 * liked
    top = scores.topk(case["top"], 1)
    experts, gates = top.indices, torch.exp(top.values - top.values[:, :1])
    gates /= gates.sum(1, keepdim=True)
    out = torch.randperm(t, generator=g, device="cuda")[:t - _kept(case)[0]]
    if "masked" in case and len(out):
        experts[out], gates[out] = -1, 0.0
    return experts, gates


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["mode"] == "train"

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    if case["kind"] == "adamw":
        return {"case": case, **_parameters(case, g)}
    experts, gates = _routed(case, g)
    rows, w = case["tokens"] * case["top"], case["width"]
    state = {"case": case}
    if case["kind"] == "dispatch":
        state |= {"experts": experts, "x": randn(case["tokens"], w).requires_grad_(train)}
        if train:
            state["grad"] = randn(rows, w)
        return state
    slots, offsets = _order(experts, case["experts"])
    state["offsets"] = offsets
    if case["kind"] == "combine":
        state |= {"slots": slots, "gates": gates.requires_grad_(train),
                  "rows": randn(rows, w).requires_grad_(train)}
        if train:
            state["grad"] = randn(case["tokens"], w)
        return state
    # the plain form's loop over experts needs the bounds on the host; they stand there beforehand
    state["bounds"] = offsets.tolist()
    state["rows"] = randn(rows, w).requires_grad_(train)
    state["weight"] = randn(case["experts"], case["out"], w, scale=w**-0.5).requires_grad_(train)
    if train:
        state["grad"] = randn(rows, case["out"])
    return state


def _parameters(case, g):
    """Parameters, gradients and moments as some steps have left them, each kind in one buffer
    whose tensors start at multiples of 256 values (the gaps are zeros and stay so)."""
    dt, shapes = DTYPES[case["dtype"]], _sizes(case)
    starts, n = [], 0
    for s in shapes:
        starts.append(n)
        n += -(-math.prod(s) // BLOCK) * BLOCK

    def views(flat):
        return [flat[a:a + math.prod(s)].view(s) for a, s in zip(starts, shapes)]

    def filled(dtype, make):
        """A buffer of zeros with make(count) in each tensor's place, 2^27 values at a time."""
        flat = torch.zeros(n, dtype=dtype, device="cuda")
        if all(math.prod(s) % BLOCK == 0 for s in shapes):
            parts = [(0, n)]
        else:
            parts = [(a, a + math.prod(s)) for a, s in zip(starts, shapes)]
        for a, b in parts:
            for c in range(a, b, 1 << 27):
                flat[c:min(b, c + (1 << 27))] = make(min(b - c, 1 << 27))
        return flat

    def randn(k):
        return torch.randn(k, generator=g, device="cuda")

    state = {"param": filled(dt, lambda k: 0.1 * randn(k)),
             "grad": filled(dt, lambda k: 1e-3 * randn(k) * torch.exp(randn(k)))}
    m = filled(torch.float32, lambda k: 2e-4 * randn(k) * torch.exp(randn(k)))
    # the mean square is at least about the mean's square
    v = filled(torch.float32, lambda k: 1e-6 * torch.exp(2 * randn(k)))
    v += 2 * m * m
    if case["state"] == "fp32":
        state |= {"m": m, "v": v}
    else:  # fp8 codes of the mean and of the mean square's root, and the blocks' scales
        for name, x in (("m", m), ("r", v.sqrt_())):
            scale = x.view(-1, BLOCK).abs().amax(1) / torch.full((), 448.0, device="cuda")
            codes = (x.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn)
            state |= {name: codes.view(-1), name + "_scale": scale}
    state["steps"] = torch.full((len(shapes),), float(STEPS), device="cuda")
    state["params"] = [p.detach().requires_grad_() for p in views(state["param"])]
    for p, d in zip(state["params"], views(state["grad"])):
        p.grad = d
    state["starts"] = starts
    return state


# ---- one pass ----------------------------------------------------------------------------


def run(state):
    if own:
        return globals()["_own_" + state["case"]["kind"]](state)
    with torch.no_grad():
        return globals()["_plain_" + state["case"]["kind"]](state)


@functools.cache
def _kernels():
    return importlib.import_module("muonium_amd.kernels")


def _own_dispatch(state):
    K, case = _kernels(), state["case"]
    order = K.sort_by_expert(state["experts"], case["experts"])
    rows = K.dispatch(state["x"], order)
    outs = [order.slots, order.offsets, rows]
    if case["mode"] == "train":
        outs += torch.autograd.grad((rows,), (state["x"],), (state["grad"],))
    return outs


def _own_combine(state):
    K = _kernels()
    order = K.ExpertOrder(state["slots"], state["offsets"])
    y = K.combine(state["rows"], order, state["gates"])
    if state["case"]["mode"] == "forward":
        return [y]
    return [y, *torch.autograd.grad((y,), (state["rows"], state["gates"]), (state["grad"],))]


def _own_product(state):
    y = _kernels().expert_linear(state["rows"], state["weight"], state["offsets"])
    if state["case"]["mode"] == "forward":
        return [y]
    return [y, *torch.autograd.grad((y,), (state["rows"], state["weight"]), (state["grad"],))]


def _moments(state):
    names = ("m", "v") if state["case"]["state"] == "fp32" else ("m", "m_scale", "r", "r_scale")
    return [state[n] for n in names]


def _optimizer(state):
    """The optimizer that a program keeps, on this state's buffers."""
    O = importlib.import_module("muonium_amd.optim")
    fp8 = state["case"]["state"] == "fp8"
    kw = {"lr": LR, "wd": WD, "betas": BETAS, "eps": EPS}
    made = O.AdamWFp8(state["params"], block_size=BLOCK, **kw) if fp8 else O.AdamW(state["params"], **kw)
    for i, (p, a) in enumerate(zip(state["params"], state["starts"])):
        n = p.numel()

        def quantized(name):
            codes = state[name].view(torch.uint8)[a:a + n]
            return O.OptimStateFp8(codes, state[name + "_scale"][a // BLOCK:(a + n) // BLOCK], None,
                                   True, p.shape, BLOCK)

        made.state[p] = {"step": state["steps"][i]}
        if fp8:
            made.state[p] |= {"exp_avg": quantized("m"), "exp_avg_sq_root": quantized("r")}
        else:
            made.state[p] |= {"exp_avg": state["m"][a:a + n].view(p.shape),
                              "exp_avg_sq": state["v"][a:a + n].view(p.shape)}
    return made


def _own_adamw(state):
    if "optimizer" not in state:
        state["optimizer"] = _optimizer(state)
    state["optimizer"].step()
    return [state["param"], *_moments(state), state["steps"]]


# ---- the plain forms: elementary torch operations in 32 bits -------------------------------


def _order(experts, e):
    """slots: each choice's row among all sorted by expert, in the order of tokens within one;
    for an empty one -1 - the row behind the experts' that it leaves. offsets: the experts' first
    rows, and the end of the last one's."""
    flat = experts.flatten()
    key = torch.where((flat >= 0) & (flat < e), flat, e)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(len(flat), device=flat.device)
    slots = torch.where(key < e, place, -1 - place).int().view(experts.shape)
    counts = key.new_zeros(e + 1).scatter_add_(0, key, torch.ones_like(key))
    return slots, torch.cat([counts.new_zeros(1), counts[:e].cumsum(0)]).int()


def _plain_dispatch(state):
    case, x = state["case"], state["x"]
    slots, offsets = _order(state["experts"], case["experts"])
    flat = slots.flatten().long()
    kept = flat >= 0
    at = torch.where(kept, flat, -1 - flat)
    source = torch.arange(case["tokens"], device=x.device).repeat_interleave(case["top"])
    rows = x.new_zeros(len(flat), case["width"])
    rows[at] = x[source] * kept[:, None]
    if case["mode"] == "forward":
        return [slots, offsets, rows]
    back = (state["grad"].float()[at] * kept[:, None]).view(*slots.shape, -1)
    return [slots, offsets, rows, back.sum(1).to(x.dtype)]


def _plain_combine(state):
    case, rows, gates = state["case"], state["rows"].float(), state["gates"]
    flat = state["slots"].flatten().long()
    kept = flat >= 0
    at = torch.where(kept, flat, -1 - flat)
    met = (rows[at] * kept[:, None]).view(*gates.shape, -1)
    y = (gates[..., None] * met).sum(1).to(state["rows"].dtype)
    if case["mode"] == "forward":
        return [y]
    d = state["grad"].float()
    drows = torch.zeros_like(rows)
    drows[at] = (gates[..., None] * d[:, None]).flatten(0, 1) * kept[:, None]
    return [y, drows.to(state["rows"].dtype), (met * d[:, None]).sum(-1)]


def _plain_product(state):
    case, bounds, dt = state["case"], state["bounds"], state["rows"].dtype
    rows, weight = state["rows"].float(), state["weight"].float()
    spans = list(zip(bounds, bounds[1:]))
    rest = [rows.new_zeros(len(rows) - bounds[-1], case["out"])]
    y = torch.cat([rows[a:b] @ w.T for (a, b), w in zip(spans, weight)] + rest).to(dt)
    if case["mode"] == "forward":
        return [y]
    d = state["grad"].float()
    drows = torch.cat([d[a:b] @ w for (a, b), w in zip(spans, weight)] + [torch.zeros_like(rows[bounds[-1]:])])
    dweight = torch.stack([d[a:b].T @ rows[a:b] for a, b in spans])
    return [y, drows.to(dt), dweight.to(dt)]


def _plain_adamw(state):
    case, p, d = state["case"], state["param"], state["grad"].float()
    state["steps"] += 1
    t = state["steps"][0].double()
    size = (LR / (1 - BETAS[0] ** t)).float()
    scale = (1 / (1 - BETAS[1] ** t).sqrt()).float()
    fp8 = case["state"] == "fp8"
    if fp8:
        m, r = ((state[n].view(-1, BLOCK).float() * state[n + "_scale"][:, None]).view(-1) for n in "mr")
        v = r * r
    else:
        m, v = state["m"], state["v"]
    m = m * BETAS[0] + d * (1 - BETAS[0])
    v = v * BETAS[1] + (d * d) * (1 - BETAS[1])
    root = v.sqrt()
    p.copy_(p.float() * (1 - LR * WD) - size * (m / (root * scale + EPS)))
    if fp8:
        for name, x in (("m", m), ("r", root)):
            x = x.view(-1, BLOCK)
            s = x.abs().amax(1).clamp(min=1e-12) / torch.full((), 448.0, device=x.device)
            state[name].copy_((x / s[:, None]).to(torch.float8_e4m3fn).view(-1))
            state[name + "_scale"].copy_(s)
    else:
        state["m"].copy_(m)
        state["v"].copy_(v)
    return [p, *_moments(state), state["steps"]]


# ---- the definitions in 64 bits --------------------------------------------------------------


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))


def _rank(experts, e):
    """Each choice's row: the choices of lower experts, and those of its own before it."""
    flat = [n if 0 <= n < e else e for n in experts.flatten().tolist()]
    starts, total = [0] * (e + 2), 0
    for n in flat:
        starts[n + 1] += 1
    for n in range(e + 1):
        starts[n + 1] += starts[n]
    free, slots = list(starts), []
    for n in flat:
        slots.append(free[n] if n < e else -1 - free[n])
        free[n] += 1
    slots = torch.tensor(slots, dtype=torch.int32, device="cuda").view(experts.shape)
    return slots, torch.tensor(starts[:e + 1], dtype=torch.int32, device="cuda")


def _token_by_choice(case):
    return torch.arange(case["tokens"], device="cuda")[:, None].expand(-1, case["top"])


def _exact_dispatch(case, state):
    x = state["x"].detach().double()
    slots, offsets = _rank(state["experts"], case["experts"])
    sent = slots >= 0
    rows = torch.zeros(slots.numel(), case["width"], dtype=torch.float64, device="cuda")
    rows[slots[sent].long()] = x[_token_by_choice(case)[sent]]
    if case["mode"] == "forward":
        return [slots, offsets, rows]
    dx = torch.zeros_like(x)
    for j in range(case["top"]):
        at = sent[:, j]
        dx[at] += state["grad"][slots[at, j].long()]
    return [slots, offsets, rows, dx]


def _exact_combine(case, state):
    slots, gates = state["slots"], state["gates"].detach().double()
    y = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
    drows, dgates = torch.zeros_like(state["rows"], dtype=torch.float64), torch.zeros_like(gates)
    for j in range(case["top"]):
        tokens = (slots[:, j] >= 0).nonzero()[:, 0]
        at = slots[tokens, j].long()
        row, gate = state["rows"].detach()[at].double(), gates[tokens, j, None]
        y.index_add_(0, tokens, gate * row)
        if case["mode"] == "train":
            d = state["grad"][tokens].double()
            drows[at] = gate * d
            dgates[tokens, j] = (d * row).sum(1)
    return [y, drows, dgates] if case["mode"] == "train" else [y]


def _exact_product(case, state):
    y = torch.zeros(len(state["rows"]), case["out"], dtype=torch.float64, device="cuda")
    train = case["mode"] == "train"
    if train:
        drows = torch.zeros_like(state["rows"], dtype=torch.float64)
        dweight = torch.zeros_like(state["weight"], dtype=torch.float64)
    for e in range(case["experts"]):
        at = slice(state["bounds"][e], state["bounds"][e + 1])
        row, w = state["rows"].detach()[at].double(), state["weight"].detach()[e].double()
        y[at] = torch.mm(row, w.t())
        if train:
            d = state["grad"][at].double()
            drows[at], dweight[e] = torch.mm(d, w), torch.mm(d.t(), row)
    return [y, drows, dweight] if train else [y]


def _exact_adamw(case, state):
    """A part at a time: 64 bits take room. What is held in fp8 has no exact value; its scales
    have one."""
    n, (b1, b2) = len(state["param"]), BETAS
    t = STEPS + 1
    fp8 = case["state"] == "fp8"
    p = torch.empty(n, dtype=torch.float64, device="cuda")
    m_new, v_new = ((None, None) if fp8 else (torch.empty_like(p), torch.empty_like(p)))
    tops = [torch.empty(n // BLOCK, dtype=torch.float64, device="cuda") for _ in range(2)]
    for a in range(0, n, 1 << 26):
        at = slice(a, min(n, a + (1 << 26)))
        blocks = slice(at.start // BLOCK, at.stop // BLOCK)
        old, d = state["param"][at].double(), state["grad"][at].double()
        if fp8:
            def value(name):
                scale = state[name + "_scale"][blocks].double()
                return state[name][at].double() * scale.repeat_interleave(BLOCK)
            m, v = value("m"), value("r").square()
        else:
            m, v = state["m"][at].double(), state["v"][at].double()
        m = b1 * m + (1 - b1) * d
        v = b2 * v + (1 - b2) * d.square()
        hat = torch.sqrt(v / (1 - b2**t))
        p[at] = old - LR * WD * old - LR * (m / (1 - b1**t)) / (hat + EPS)
        if fp8:
            for top, x in zip(tops, (m, v.sqrt())):
                top[blocks] = x.abs().unflatten(0, (-1, BLOCK)).amax(1).clamp(min=1e-12) / 448
        else:
            m_new[at], v_new[at] = m, v
    steps = torch.full((len(state["steps"]),), float(t), dtype=torch.float64, device="cuda")
    return [p, None, tops[0], None, tops[1], steps] if fp8 else [p, m_new, v_new, steps]
