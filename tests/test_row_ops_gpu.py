"""The training step's row operators (qk_norm_rope, route, token_logprobs, policy_loss) against
their definitions in float64 (oracle/row_ops_ref.py).

Tolerances. U is half a unit in the last place of the output's type (2^-8 bf16, 2^-11 fp16,
2^-24 fp32): the one rounding at the end. Inside, everything is fp32: each result carries at most K
roundings of 2^-24 of the magnitudes that meet in it (the oracle's `scale`). K counts the longest
chain: a row sum of up to 1024 values is at most 18 additions in a lane and 6 between lanes, twice
(square sum and dot product), and about 20 products, quotients and roots around them: 96. An
exponential's argument of size a is off by 2 a 2^-24 and its result by 2 more, sums of exponentials
over a vocabulary are at most 64 additions deep in a thread and 15 across: 256 for arguments
up to 80. A gradient by `dw` adds its rows one after the other in a lane: below 128 here."""

import math

import pytest
import torch

from muonium_amd.kernels import policy_loss, qk_norm_rope, route, token_logprobs
from oracle import row_ops_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
E = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def bound(want, scale, k, dtype):
    return U[dtype] * want.abs() * (1 + k * E) + k * E * scale + TINY[dtype]


def check(got, want, scale, k, dtype=None, what=""):
    dtype = dtype or got.dtype
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), (what, int(got.isnan().sum()), int(nan.sum()))
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    ok = ~nan & ~inf
    off = ((got - want).abs() - bound(want, scale.expand_as(want), k, dtype))[ok]
    assert off.numel() == 0 or off.max() <= 0, (what, off.max().item())


def gen(seed):
    return torch.Generator().manual_seed(seed)


def leaf(t):
    return t.cuda().requires_grad_()


# ---- queries and keys ---------------------------------------------------------------------

QK = [
    # lead shape, q heads, k heads, dim, rotary, interleaved, positions
    ((2, 5), 4, 2, 128, 128, False, None),
    ((3, 1), 32, 8, 128, 128, False, "batch"),       # single tokens at their own places
    ((2, 7), 5, 1, 64, 32, False, "shared"),         # head counts of no whole group, part rotated
    ((1, 9), 3, 3, 64, 16, True, "batch32"),
    ((4,), 6, 2, 256, 256, True, None),              # no batch
    ((2, 3), 2, 1, 96, 96, False, "shared"),         # lanes without a share
    ((2, 3), 9, 1, 160, 96, True, None),
    ((1, 2), 2, 2, 512, 512, False, None),
    ((1, 2), 2, 1, 1024, 64, False, None),
    ((2, 3), 3, 2, 80, 40, False, "shared"),         # rotary no multiple of 16: single values
    ((2, 3), 3, 2, 34, 34, False, "batch"),
    ((2, 3), 2, 1, 162, 80, True, None),
    ((2, 3), 2, 1, 7, 4, False, None),
    ((2, 3), 2, 1, 1, 0, False, None),
    ((1, 3), 2, 1, 301, 0, False, None),
    ((1, 2), 2, 1, 1022, 1022, True, None),
    ((1, 2), 1, 1, 1023, 2, False, None),
    ((70, 11), 7, 3, 48, 48, False, "batch"),        # several workgroups a side
]


def qk_case(lead, hq, hk, dim, rotary, positions, dtype, seed, weights=True):
    g = gen(seed)
    q = (torch.randn(*lead, hq, dim, generator=g) * 1.7).to(dtype)
    k = (torch.randn(*lead, hk, dim, generator=g) * 0.4).to(dtype)
    ws = [None, None]
    if weights:
        ws = [(1 + 0.3 * torch.randn(dim, generator=g)) for _ in range(2)]
    cos = sin = None
    if rotary:
        angle = torch.rand(40, rotary // 2, generator=g) * 6.3
        cos, sin = angle.cos(), angle.sin()
    pos = None
    if positions:
        shape = lead[-1:] if positions == "shared" else lead
        pos = torch.randint(0, 40, shape, generator=g)
        pos = pos.int() if positions == "batch32" else pos
    return q, k, ws, cos, sin, pos, g


def cuda(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(QK)))
def test_qk_norm_rope_and_its_gradient(case, dtype):
    lead, hq, hk, dim, rotary, inter, positions = QK[case]
    q, k, ws, cos, sin, pos, g = qk_case(lead, hq, hk, dim, rotary, positions, dtype, case)
    wdt = torch.float32 if case % 2 else dtype
    ws = [w.to(wdt) for w in ws]
    grads = [torch.randn(t.shape, generator=g).to(dtype) for t in (q, k)]
    ql, kl, wl = leaf(q), leaf(k), [leaf(w) for w in ws]
    args = (cuda(cos), cuda(sin), cuda(pos))
    outs = qk_norm_rope(ql, kl, *wl, *args, eps=1e-5, interleaved=inter)
    plain = qk_norm_rope(q.cuda(), k.cuda(), *(w.cuda() for w in ws), *args, eps=1e-5,
                         interleaved=inter)
    got = torch.autograd.grad(outs, (ql, kl, *wl), [t.cuda() for t in grads])
    turned = ref.angles(q, cos, sin, pos)
    for i, x in enumerate((q, k)):
        y, scale = ref.norm_rope(x, ws[i], turned, 1e-5, inter)
        assert torch.equal(outs[i], plain[i]) and outs[i].is_contiguous()
        check(outs[i], y, scale, 96, dtype, "out")
        dx, sx, dw, sw = ref.norm_rope_grad(x, ws[i], grads[i], turned, 1e-5, inter)
        check(got[i], dx, sx, 96, dtype, "dx")
        check(got[2 + i], dw, sw, 128 + 96, wdt, "dw")
        # against differences of the definition along a direction
        d = torch.randn(x.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = (ref.norm_rope(x.double() + s * h * d, ws[i], turned, 1e-5, inter)[0]
                    for s in (1, -1))
        slope = (grads[i].double() * (up - down)).sum() / (2 * h)
        room = (bound(dx, sx, 96, dtype) * d.abs()).sum() + 1e-6 * (dx * d).abs().sum() + 1e-6
        assert abs((got[i].double().cpu() * d).sum() - slope) <= room


def test_qk_strided_inputs_and_gradients_match_contiguous_ones():
    """Slices of a fused projection, head-major tensors, expanded heads, misaligned bases and
    strided incoming gradients give what contiguous copies give."""
    g = gen(3)
    qkv = torch.randn(2, 6, 10, 64, generator=g).bfloat16().cuda()
    cos, sin = (torch.rand(8, 32, generator=g).cuda() for _ in range(2))
    w = torch.randn(64, generator=g).cuda()
    wide = torch.randn(2, 6, 4 * 64 + 1, generator=g).bfloat16().cuda()
    pairs = [
        (qkv[:, :, :6], qkv[:, :, 6:8]),
        (qkv.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :4], qkv[:, :, 4:5].expand(2, 6, 3, 64)),
        (wide[..., 1:].unflatten(-1, (4, 64)), qkv[:, 0:1, :2].expand(2, 6, 2, 64)),
        (qkv.transpose(0, 1)[:2].transpose(2, 3).contiguous().transpose(2, 3), qkv.transpose(0, 1)[:2, :, 3:4]),
    ]
    for q, k in pairs:
        res = []
        for make in (lambda t: t.detach(), lambda t: t.detach().contiguous()):
            a, b = make(q).requires_grad_(), make(k).requires_grad_()
            ww = [w.clone().requires_grad_() for _ in range(2)]
            o = qk_norm_rope(a, b, *ww, cos, sin)
            gr = [torch.randn(t.transpose(1, 2).shape, generator=gen(5)).bfloat16().cuda().transpose(1, 2)
                  for t in o]
            if make(q).is_contiguous():
                gr = [t.contiguous() for t in gr]
            res.append([*o, *torch.autograd.grad(o, (a, b, *ww), gr)])
        for x, y in zip(*res):
            torch.testing.assert_close(x, y, rtol=2.0**-7, atol=1e-5)


def test_qk_gradients_of_shared_and_partial_inputs():
    """A leaf behind expanded heads and a fused projection collects the sum of its uses; a single
    output's gradient, or no weights, works alone."""
    g = gen(4)
    one = leaf(torch.randn(2, 3, 1, 32, generator=g))
    q = torch.randn(2, 3, 4, 32, generator=g)
    _, k_out = qk_norm_rope(q.cuda(), one.expand(2, 3, 5, 32))
    dy = torch.randn(2, 3, 5, 32, generator=g)
    k_out.backward(dy.cuda())
    dx, sx, _, _ = ref.norm_rope_grad(one.detach().cpu().expand(2, 3, 5, 32), None, dy, None, 1e-6, False)
    # five fp32 gradients summed by torch
    check(one.grad, dx.sum(2, keepdim=True), sx.sum(2, keepdim=True), 104, torch.float32)
    w = leaf(torch.randn(32, generator=g))
    q_out, _ = qk_norm_rope(q.cuda(), q.cuda(), w, None)
    q_out.backward(q_out.detach())
    y, _ = ref.norm_rope(q, w.detach().cpu(), None, 1e-6, False)
    _, _, dw, sw = ref.norm_rope_grad(q, w.detach().cpu(), q_out.detach().cpu(), None, 1e-6, False)
    check(w.grad, dw, sw, 224, torch.float32)


def test_qk_positions_outside_the_table_are_nan_and_empty_calls_return():
    x = torch.randn(1, 4, 2, 32).cuda()
    cos = sin = torch.ones(3, 16, device="cuda")
    q, k = qk_norm_rope(x, x, None, None, cos, sin, torch.tensor([0, -1, 3, 2], device="cuda"))
    for t in (q, k):
        assert torch.equal(t.isnan().flatten(2).all(-1).cpu(), torch.tensor([[False, True, True, False]]))
        assert torch.equal(t.isnan().flatten(2).any(-1).cpu(), torch.tensor([[False, True, True, False]]))
    for lead, hq, hk in (((0, 3), 2, 1), ((2, 0), 2, 1), ((2, 3), 0, 1), ((2, 3), 2, 0), ((2, 3), 0, 0)):
        a, b = (leaf(torch.randn(*lead, h, 32)) for h in (hq, hk))
        w = leaf(torch.ones(32))
        o = qk_norm_rope(a, b, w, w, cos, sin)
        gr = torch.autograd.grad(o, (a, b, w), [torch.ones_like(t) for t in o])
        assert [t.shape for t in o] == [a.shape, b.shape] and gr[0].shape == a.shape
        if 0 in lead or hq + hk == 0:
            assert torch.count_nonzero(gr[2]) == 0


def test_qk_rows_of_extreme_size():
    """A zero row stays zero with a finite gradient; an infinity or NaN stays in its own row."""
    x = torch.randn(1, 5, 2, 64)
    x[0, 0] = 0
    x[0, 1, 0, 3] = math.inf
    x[0, 2, 1, 60] = math.nan
    x[0, 3] *= 1e-18
    w = torch.ones(64)
    dy = torch.randn(1, 5, 2, 64)
    a = leaf(x)
    o, _ = qk_norm_rope(a, x.cuda(), w.cuda(), None)
    o.backward(dy.cuda())
    y, scale = ref.norm_rope(x, w, None, 1e-6, False)
    check(o, y, scale.nan_to_num(0.0), 96, torch.float32)
    dx, sx, _, _ = ref.norm_rope_grad(x, w, dy, None, 1e-6, False)
    fine = torch.ones(1, 5, 2, dtype=torch.bool)
    fine[0, 1, 0] = fine[0, 2, 1] = False
    check(a.grad.cpu()[fine], dx[fine], sx[fine], 96, torch.float32)


# ---- routing ------------------------------------------------------------------------------


def route_case(n, e, dtype, seed, masked=0.0):
    g = gen(seed)
    z = torch.randn(n, e, generator=g) * 2
    z = (z * 4).round() / 4 if seed % 2 else z  # many equal logits
    mask = None
    if masked:
        mask = torch.rand(n, generator=g) >= masked
    return z.to(dtype), mask, g


ROUTE = [(1, 1, 1), (5, 3, 2), (7, 8, 8), (33, 9, 3), (64, 16, 16), (50, 31, 4), (48, 64, 8),
         (300, 64, 6), (5, 65, 3), (130, 128, 8), (9, 200, 10), (600, 256, 8), (3, 257, 40), (17, 512, 9),
         (4, 700, 64), (5, 1024, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(ROUTE)))
def test_route_and_its_gradient(case, dtype):
    n, e, k = ROUTE[case]
    normalize, masked = bool(case % 3), (0.0, 0.4)[case % 2]
    z, mask, g = route_case(n, e, dtype, case, masked)
    x = leaf(z)
    got = route(x, k, token_mask=cuda(mask), normalize=normalize)
    want = ref.route(z, k, mask, normalize)
    assert torch.equal(got.experts.cpu(), want["experts"])
    assert torch.equal(got.counts.cpu(), want["counts"])
    check(got.gates, want["gates"], want["gates"], 256, torch.float32, "gates")
    check(got.balance_loss, want["balance"], want["balance"], 512, torch.float32, "balance")
    size = (1 + z.double().abs().max()) * 2 * (want["z"].sqrt() + 1)
    check(got.z_loss, want["z"], size, 256, torch.float32, "z")
    scale = 256.0 if dtype == torch.float16 else 1.0  # a loss scale, as half-precision runs use
    grads = [torch.randn(n, k, generator=g) * scale, torch.tensor(1.3 * n * scale),
             torch.tensor(0.2 * n * scale)]
    dz, = torch.autograd.grad((got.gates, got.balance_loss, got.z_loss), (x,),
                              [t.cuda() for t in grads])
    d, sd = ref.route_grad(want, *grads)
    check(dz, d, sd, 320, dtype, "dlogits")
    # against differences of the definition, where a small step changes no choice
    if case % 2 == 0 and want["kept"]:
        step = torch.randn(n, e, generator=g, dtype=torch.float64) * 1e-6
        both = [ref.route(z.double() + s * step, k, mask, normalize) for s in (1, -1)]
        if all(torch.equal(b["experts"], want["experts"]) for b in both):
            value = [(b["gates"] * grads[0]).sum() + b["balance"] * grads[1] + b["z"] * grads[2]
                     for b in both]
            room = (bound(d, sd, 320, dtype) * step.abs()).sum() + 1e-3 * (d * step).abs().sum() + 1e-12 * scale * n
            assert abs((dz.double().cpu() * step).sum() - (value[0] - value[1]) / 2) <= room


@pytest.mark.parametrize("dtype", TYPES)
def test_route_masked_experts_rows_and_values(dtype):
    """Experts at -inf are never chosen and leave empty slots, rows without any other expert count
    nowhere, the type's lowest value is a value, -0 equals 0, and what stands in masked rows
    (infinities, NaN) reaches nothing."""
    low = torch.finfo(dtype).min
    z = torch.randn(9, 12, generator=gen(1)).to(dtype)
    z[0] = -math.inf
    z[1, 2:] = -math.inf
    z[2] = low
    z[3, ::2] = low
    z[4] = 0.0
    z[4, 5:] = -0.0
    z[5] = math.nan
    z[6, 3] = math.inf
    z[7, :] = -math.inf
    z[7, 11] = low
    mask = torch.ones(9, dtype=torch.bool)
    mask[5] = mask[6] = False
    x = leaf(z)
    got = route(x, 4, token_mask=mask.cuda())
    want = ref.route(z, 4, mask)
    assert torch.equal(got.experts.cpu(), want["experts"])
    assert torch.equal(got.counts.cpu(), want["counts"])
    assert got.experts[0].tolist() == [-1] * 4 and got.experts[1].tolist()[2:] == [-1, -1]
    check(got.gates, want["gates"], want["gates"], 256)
    check(got.balance_loss, want["balance"], want["balance"], 512)
    dg = torch.randn(9, 4, generator=gen(2))
    dz, = torch.autograd.grad((got.gates, got.balance_loss), (x,), [dg.cuda(), torch.ones((), device="cuda")])
    d, sd = ref.route_grad(want, dg, torch.tensor(1.0), torch.tensor(0.0))
    check(dz, d, sd, 320, dtype)


def test_route_nan_and_infinity_stay_in_their_rows():
    z = torch.randn(6, 10, generator=gen(1))
    z[1, 4] = math.nan
    z[2, 7] = math.inf
    z[3] = math.nan
    got = route(z.cuda(), 3)
    want = ref.route(z, 3)
    assert got.experts[1, 0] == 4 and got.experts[2, 0] == 7 and got.experts[3].tolist() == [0, 1, 2]
    assert torch.equal(got.experts.cpu(), want["experts"])
    assert torch.equal(got.counts.cpu(), want["counts"])
    assert torch.equal(got.gates.isnan().any(1).cpu(), torch.tensor([False, True, True, True, False, False]))
    assert got.balance_loss.isnan() and got.z_loss.isnan()


def test_route_of_nothing_and_partial_gradients():
    """No tokens, or none that counts: losses 0, no gradient; and gradients of single outputs."""
    for z, mask in ((torch.zeros(0, 8), None), (torch.randn(5, 8), torch.zeros(5, dtype=torch.bool)),
                    (torch.full((5, 8), -math.inf), None)):
        x = leaf(z)
        r = route(x, 2, token_mask=cuda(mask))
        assert r.balance_loss == 0 and r.z_loss == 0 and torch.count_nonzero(r.counts) == 0
        assert (r.experts == -1).all() and torch.count_nonzero(r.gates) == 0
        (r.balance_loss + r.z_loss + r.gates.sum()).backward()
        assert torch.count_nonzero(x.grad) == 0 and x.grad.shape == z.shape
    z, _, g = route_case(40, 24, torch.float32, 2)
    want = ref.route(z, 3)
    zero = torch.zeros(())
    dg = torch.randn(40, 3, generator=g)
    for pick, grads in (("gates", (dg, zero, zero)), ("balance_loss", (dg * 0, zero + 1, zero)),
                        ("z_loss", (dg * 0, zero, zero + 1))):
        x = leaf(z)
        out = getattr(route(x, 3), pick)
        d, = torch.autograd.grad((out,), (x,), (dg.cuda() if pick == "gates" else torch.ones((), device="cuda"),))
        check(d, *ref.route_grad(want, *grads), 320, torch.float32, pick)


def test_route_leading_dimensions_strides_and_determinism():
    z = torch.randn(3, 7, 40, generator=gen(6)).cuda()
    a = route(z[..., 3:35], 5)
    b = route(z[..., 3:35].reshape(21, 32).contiguous(), 5)
    assert a.gates.shape == (3, 7, 5) and torch.equal(a.experts.view(21, 5), b.experts)
    assert torch.equal(a.gates.view(21, 5), b.gates) and torch.equal(a.balance_loss, b.balance_loss)
    assert route(z[0, 0, :32], 5).gates.shape == (5,)
    t = torch.randn(40, 21, generator=gen(7)).cuda().t()  # last dimension not contiguous
    assert torch.equal(route(t, 3).experts, route(t.contiguous(), 3).experts)
    big = torch.randn(40000, 64, generator=gen(8)).cuda()
    x, y = route(big, 8), route(big, 8)
    assert all(torch.equal(p, q) for p, q in zip(x, y))
    assert int(x.counts.sum()) == 40000 * 8
    want = torch.softmax(big.double(), 1).mean(0) @ x.counts.double() * 64 / (8 * 40000)
    check(x.balance_loss, want.cpu(), want.cpu(), 512)


# ---- token log probabilities ----------------------------------------------------------------


def logits_case(n, v, dtype, seed, spread=3.0):
    g = gen(seed)
    x = (torch.randn(n, v, generator=g) * spread).to(dtype)
    tokens = torch.randint(0, v, (n,), generator=g)
    tokens[::2] = x[::2].float().argmax(1)  # half of them likely ones
    return x, tokens, g


LOGP = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 9), (3, 63), (7, 1000), (2, 4097), (70, 515), (1100, 40),
        (3, 40000), (1, 131073), (2, 170001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(LOGP)))
def test_token_logprobs_and_its_gradient(case, dtype):
    n, v = LOGP[case]
    temperature = (1.0, 0.7, 2.5)[case % 3]
    x, tokens, g = logits_case(n, v, dtype, case)
    xl = leaf(x)
    got = token_logprobs(xl, tokens.cuda(), temperature=temperature)
    assert torch.equal(got, token_logprobs(x.cuda(), tokens.cuda(), temperature=temperature))
    logp, p = ref.logprobs(x, tokens, temperature)
    check(got, logp, torch.ones(n, dtype=torch.float64), 256, torch.float32, "logp")
    grad = torch.randn(n, generator=g)
    d, = torch.autograd.grad((got,), (xl,), (grad.cuda(),))
    want, scale = ref.logprobs_grad(p, tokens, grad, temperature)
    check(d, want, scale, 256, dtype, "dlogits")
    step = torch.randn(n, v, generator=g, dtype=torch.float64) * 1e-5
    up, down = (ref.logprobs(x.double() + s * step, tokens, temperature)[0] for s in (1, -1))
    slope = (grad.double() * (up - down)).sum() / 2
    room = (bound(want, scale, 256, dtype) * step.abs()).sum() + 1e-5 * (want * step).abs().sum() + 1e-10
    assert abs((d.double().cpu() * step).sum() - slope) <= room


@pytest.mark.parametrize("v", [50, 40000, 140000])
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_special_rows(dtype, v):
    """Left-out and impossible tokens, masked vocabularies, rows of the lowest value, of infinities
    and of NaN."""
    low = torch.finfo(dtype).min
    x = (torch.randn(10, v, generator=gen(1)) * 2).to(dtype)
    tokens = torch.randint(0, v, (10,), generator=gen(2))
    tokens[0], x[0] = -100, math.nan            # left out: nothing of its row is seen
    tokens[1] = v                               # not in the vocabulary
    x[2, : v // 2], tokens[2] = -math.inf, v - 1
    x[3, 1:], tokens[3] = -math.inf, 0          # one possible token: 0
    x[4], tokens[4] = low, 5
    x[5, 1:], tokens[5] = low, 7
    x[6], tokens[6] = -math.inf, 3              # nothing possible
    x[7, 2], tokens[7] = math.nan, 1
    x[8, 4], tokens[8] = math.inf, 0
    x[9, 6], tokens[9] = -math.inf, 6           # an impossible token of a fine row: -inf
    xl = leaf(x)
    got = token_logprobs(xl, tokens.cuda())
    logp, p = ref.logprobs(x, tokens)
    check(got, logp, torch.ones(10, dtype=torch.float64), 256, torch.float32)
    assert got[0] == 0 and got[1].isnan() and got[3] == 0 and got[6].isnan() and got[9] == -math.inf
    grad = torch.linspace(-1, 1, 10)
    d, = torch.autograd.grad((got,), (xl,), (grad.cuda(),))
    want, scale = ref.logprobs_grad(p, tokens, grad)
    check(d, want, scale.nan_to_num(0.0), 256, dtype)
    assert torch.count_nonzero(d[0]) == 0
    zero, = torch.autograd.grad((token_logprobs(xl, tokens.cuda()),), (xl,), (torch.zeros(10, device="cuda"),))
    assert torch.count_nonzero(zero) == 0


def test_logprobs_shapes_strides_and_broadcast():
    x, tokens, _ = logits_case(12, 301, torch.bfloat16, 1)
    x, tokens = x.cuda(), tokens.cuda()
    want = token_logprobs(x, tokens)
    got = token_logprobs(x.view(3, 4, 301), tokens.view(3, 4))
    assert got.shape == (3, 4) and torch.equal(got.flatten(), want)
    assert token_logprobs(x[0], tokens[0]).shape == ()
    wide = torch.randn(12, 400, device="cuda").bfloat16()
    wide[:, 50:351] = x
    view = wide[:, 50:351].detach().requires_grad_()  # rows neither 16-byte aligned nor adjacent
    d, = torch.autograd.grad((token_logprobs(view, tokens),), (view,), (torch.ones(12, device="cuda"),))
    y = x.clone().requires_grad_()
    e, = torch.autograd.grad((token_logprobs(y, tokens),), (y,), (torch.ones(12, device="cuda"),))
    assert torch.equal(token_logprobs(view, tokens), want) and torch.equal(d, e)
    t = x.t().contiguous().t()
    assert torch.equal(token_logprobs(t, tokens), want)
    one = x[:1].clone().requires_grad_()  # one row for all tokens: its gradient is the sum
    many = token_logprobs(one.expand(12, 301), tokens)
    many.sum().backward()
    logp, p = ref.logprobs(x[:1].cpu().expand(12, 301), tokens.cpu())
    check(many, logp, torch.ones(12, dtype=torch.float64), 256, torch.float32)
    full, scale = ref.logprobs_grad(p, tokens.cpu(), torch.ones(12))
    # twelve bf16 gradients, each rounded, then summed in bf16 by torch
    room = 14 * U[torch.bfloat16] * scale.sum(0)
    assert ((one.grad[0].double().cpu() - full.sum(0)).abs() <= room).all()
    empty = token_logprobs(torch.empty(0, 9, device="cuda").requires_grad_(), torch.empty(0, dtype=torch.int64, device="cuda"))
    assert empty.shape == (0,)
    empty.sum().backward()


# ---- the policy loss ------------------------------------------------------------------------


def policy_case(n, v, dtype, seed, reference, temperature):
    x, tokens, g = logits_case(n, v, dtype, seed)
    logp, p = ref.logprobs(x, tokens, temperature)
    moved = 0.2 * torch.randn(n, generator=g).double()
    for edge in (math.log(0.8), math.log(1.3)):  # a ratio at the edge has two gradients
        moved = torch.where((moved - edge).abs() < 1e-3, moved + 2e-3, moved)
    old = (logp - moved).float()
    adv = torch.randn(n, generator=g)
    w = torch.rand(n, generator=g) / n
    w[1::3] = 0
    r = (logp + 0.3 * torch.randn(n, generator=g)).float() if reference else None
    return x, tokens, old, adv, w, r, logp, p


POLICY = [(1, 1), (4, 5), (9, 64), (6, 1001), (50, 2048), (5, 4100), (3, 8192), (4, 16385), (3, 32768),
          (3, 50257), (2, 70000), (2, 81920), (2, 81921), (2, 98305), (2, 131072), (2, 163840), (2, 163841)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(POLICY)))
def test_policy_loss_and_its_gradient(case, dtype):
    n, v = POLICY[case]
    temperature, reference = (1.0, 0.7)[case % 2], case % 3 != 0
    x, tokens, old, adv, w, r, logp, p = policy_case(n, v, dtype, case, reference, temperature)
    kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05, temperature=temperature)
    xl = leaf(x)
    args = [t.cuda() for t in (tokens, old, adv, w)] + [cuda(r)]
    got = policy_loss(xl, *args, **kw)
    plain = policy_loss(x.cuda(), *args, **kw)
    loss, slope, size, sizes = ref.policy(logp, old, adv, w, r, 0.2, 0.3, 0.05)
    on = w != 0
    check(got.logprobs, torch.where(on, logp, 0.0), torch.ones(n, dtype=torch.float64), 256, torch.float32)
    # logp's own error, 256 2^-24, moves the loss by that much of its slope
    check(got.loss, loss, size, 2 * 256, torch.float32, "loss")
    # the two forms of the forward pass add a row in different orders
    check(plain.loss, loss, size, 2 * 256, torch.float32, "loss without gradient")
    check(plain.logprobs, torch.where(on, logp, 0.0), torch.ones(n, dtype=torch.float64), 256, torch.float32)
    scale = 1024.0 * n if dtype == torch.float16 else 1.0
    d, = torch.autograd.grad((got.loss,), (xl,), (torch.tensor(scale, device="cuda"),))
    want, ds = ref.logprobs_grad(p, tokens, slope, temperature)
    _, room = ref.logprobs_grad(p, tokens, sizes, temperature)  # the slope's own error
    check(d, want * scale, (ds + 2 * room) * scale, 256, dtype, "dlogits")
    assert torch.count_nonzero(d[(~on).cuda()]) == 0
    # against differences of the definition
    g = gen(case + 100)
    step = torch.randn(n, v, generator=g, dtype=torch.float64) * 1e-6
    up, down = (ref.policy(ref.logprobs(x.double() + s * step, tokens, temperature)[0], old, adv, w,
                           r, 0.2, 0.3, 0.05)[0] for s in (1, -1))
    off = (bound(want * scale, (ds + 2 * room) * scale, 256, dtype) * step.abs()).sum()
    assert abs((d.double().cpu() * step).sum() - scale * (up - down) / 2) <= \
        off + scale * (1e-4 * (want * step).abs().sum() + 1e-12)


@pytest.mark.parametrize("dtype", TYPES)
def test_policy_gradient_scales_and_repeats(dtype):
    """A loss gradient of any value, a second backward pass through the same graph, and a
    gradient that arrives beside another loss's."""
    x, tokens, old, adv, w, r, logp, p = policy_case(6, 1500, dtype, 3, True, 1.0)
    args = [t.cuda() for t in (tokens, old, adv, w, r)]
    _, slope, _, sizes = ref.policy(logp, old, adv, w, r, 0.2, 0.2, 0.1)
    want, ds = ref.logprobs_grad(p, tokens, slope)
    _, room = ref.logprobs_grad(p, tokens, sizes)
    xl = leaf(x)
    out = policy_loss(xl, *args, kl_coef=0.1)
    for scale in (3.0, 0.0, 1.0, 4096.0):
        d, = torch.autograd.grad((out.loss,), (xl,), (torch.tensor(scale, device="cuda"),), retain_graph=True)
        # the first pass scales the rounded gradient: two roundings
        want_s = want * scale
        got = d.double().cpu()
        tol = 2 * bound(want_s, (ds + 2 * room) * scale, 256, dtype)
        assert ((got - want_s).abs() <= tol).all(), scale
    # beside another loss: exactly the sum of the two gradients
    part, = torch.autograd.grad((policy_loss(xl, *args, kl_coef=0.1).loss,), (xl,),
                                (torch.tensor(2.0, device="cuda"),))
    other, = torch.autograd.grad((token_logprobs(xl, args[0]),), (xl,),
                                 (torch.full((6,), 0.5, device="cuda"),))
    both = policy_loss(xl, *args, kl_coef=0.1).loss * 2 + token_logprobs(xl, args[0]).sum() * 0.5
    both.backward()
    assert torch.equal(xl.grad, part + other)


@pytest.mark.parametrize("dtype", TYPES)
def test_policy_loss_sees_nothing_of_rows_left_out(dtype):
    x, tokens, old, adv, w, r, logp, p = policy_case(9, 700, dtype, 4, True, 1.0)
    w[5], tokens[2] = 0.0, -100
    on = (w != 0) & (tokens >= 0)
    x2, bad = x.clone(), [t.clone() for t in (old, adv, r)]
    x2[~on] = math.nan
    for t in bad:
        t[~on] = math.inf
    tokens2 = torch.where(w == 0, 10**9, tokens)
    res = []
    for a, t, (o, ad, rr) in ((x, tokens, (old, adv, r)), (x2, tokens2, bad)):
        xl = leaf(a)
        out = policy_loss(xl, t.cuda(), o.cuda(), ad.cuda(), w.cuda(), rr.cuda(), kl_coef=0.1)
        res.append((out.loss, out.logprobs, *torch.autograd.grad((out.loss,), (xl,))))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert torch.count_nonzero(res[0][2][(~on).cuda()]) == 0
    assert torch.count_nonzero(res[0][1][(~on).cuda()]) == 0
    none = policy_loss(leaf(x), tokens.cuda(), old.cuda(), adv.cuda(), torch.zeros(9, device="cuda"))
    assert none.loss == 0
    empty = policy_loss(leaf(x[:0]), *(t[:0].cuda() for t in (tokens, old, adv, w)))
    assert empty.loss == 0
    empty.loss.backward()
    wrong = tokens.clone()
    wrong[0] = 700  # not in the vocabulary, and weighed
    xl = leaf(x)
    out = policy_loss(xl, wrong.cuda(), old.cuda(), adv.cuda(), w.cuda())
    d, = torch.autograd.grad((out.loss,), (xl,))
    assert out.loss.isnan() and d[0].isnan().all() and not d[1:].isnan().any()


def test_policy_loss_strided_rows():
    x, tokens, old, adv, w, r, logp, p = policy_case(8, 301, torch.bfloat16, 5, True, 1.0)
    wide = torch.randn(8, 333).bfloat16()
    wide[:, 7:308] = x
    args = [t.cuda() for t in (tokens, old, adv, w, r)]
    res = []
    for a in (x.cuda(), wide.cuda()[:, 7:308], x.cuda().t().contiguous().t()):
        a = a.detach().requires_grad_()
        out = policy_loss(a, *args, kl_coef=0.1)
        res.append((out.loss, out.logprobs, *torch.autograd.grad((out.loss,), (a,))))
    three = x.cuda().view(2, 4, 301).requires_grad_()
    out = policy_loss(three, *(t.view(2, 4) for t in args), kl_coef=0.1)
    assert out.logprobs.shape == (2, 4)
    res.append((out.loss, out.logprobs.flatten(), torch.autograd.grad((out.loss,), (three,))[0].view(8, 301)))
    for other in res[1:]:
        for a, b in zip(res[0], other):
            assert torch.equal(a, b)


# ---- tensors of more than 2^31 values ---------------------------------------------------------


def test_rows_past_32_bit_offsets():
    """The last rows of tensors of more than 2^31 values come out as they do alone, forward and
    backward, in every operator."""
    bf16, n = torch.bfloat16, 3
    x = torch.randn(17000, 128000, device="cuda", dtype=bf16)
    assert x.numel() > 2**31
    tokens = torch.randint(0, 128000, (17000,), device="cuda")
    f = torch.rand(17000, device="cuda")

    def logits_calls(x, tokens, f):
        x = x.detach().requires_grad_()
        lp = token_logprobs(x, tokens)
        d, = torch.autograd.grad((lp,), (x,), (f,))
        keep = [lp[-n:].detach().clone(), d[-n:].clone()]
        del d
        out = policy_loss(x, tokens, lp.detach() - 0.1, f, f)
        d, = torch.autograd.grad((out.loss,), (x,))
        return keep + [out.logprobs[-n:].clone(), d[-n:].clone()]

    big, small = logits_calls(x, tokens, f), logits_calls(x[-n:], tokens[-n:], f[-n:])
    for a, b in zip(big, small):
        # a few rows alone take another number of threads: sums in another order
        torch.testing.assert_close(a, b, rtol=2.0**-7, atol=1e-5)
    del x, big, small
    torch.cuda.empty_cache()

    z = torch.randn(9_000_000, 256, device="cuda", dtype=bf16).requires_grad_()
    assert z.numel() > 2**31
    r = route(z, 8)
    few = route(z[-n:].detach(), 8)
    assert torch.equal(r.experts[-n:], few.experts) and torch.equal(r.gates[-n:], few.gates)
    assert int(r.counts.sum()) == 8 * 9_000_000
    g = torch.zeros_like(r.gates)
    g[-n:] = torch.rand(n, 8, device="cuda")
    d, = torch.autograd.grad((r.gates,), (z,), (g,))
    y = z[-n:].detach().requires_grad_()
    e, = torch.autograd.grad((route(y, 8).gates,), (y,), (g[-n:],))
    assert torch.equal(d[-n:], e) and torch.count_nonzero(d[:-n]) == 0
    del z, r, d, g
    torch.cuda.empty_cache()

    q = torch.randn(560_000, 32, 128, device="cuda", dtype=bf16)
    assert q.numel() > 2**31
    angle = torch.rand(560_000, 64, device="cuda")
    w = torch.rand(128, device="cuda")

    def heads_calls(q, positions):
        q = q.detach().requires_grad_()
        a, b = qk_norm_rope(q, q[:, :1], w, w, angle, angle, positions)
        d, = torch.autograd.grad((a,), (q,), (a.detach(),))
        return a[-n:].detach().clone(), b[-n:].detach().clone(), d[-n:].clone()

    positions = torch.arange(560_000, device="cuda")
    for a, b in zip(heads_calls(q, positions), heads_calls(q[-n:], positions[-n:])):
        assert torch.equal(a, b)


# ---- streams, determinism, graphs, torch.compile ----------------------------------------------


def _all_calls(seed=0):
    """Leaves and a closure that runs all four operators with their gradients."""
    g = gen(seed)
    q, k = leaf(torch.randn(2, 33, 8, 64, generator=g)), leaf(torch.randn(2, 33, 2, 64, generator=g))
    w = leaf(torch.randn(64, generator=g))
    angle = torch.rand(64, 32, generator=g).cuda()
    z = leaf(torch.randn(5000, 64, generator=g))
    x, tokens, old, adv, wt, r, _, _ = policy_case(40, 3001, torch.bfloat16, seed, True, 1.0)
    x = leaf(x)
    args = [t.cuda() for t in (tokens, old, adv, wt, r)]

    def run():
        a, b = qk_norm_rope(q, k, w, w, angle, angle)
        rt = route(z, 6)
        lp = token_logprobs(x, args[0])
        out = policy_loss(x, *args, kl_coef=0.1)
        loss = (a * a.detach()).sum() + b.sum() + rt.balance_loss + rt.gates[:, 0].sum() + lp.sum() + out.loss
        return [a, b, rt.gates, rt.experts, rt.counts, lp, out.loss,
                *torch.autograd.grad((loss,), (q, k, w, z, x))]

    return run


def test_row_operators_repeat_bit_for_bit_and_on_side_streams():
    run = _all_calls()
    first = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    third = run()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_row_operators_in_a_captured_graph():
    """Forward calls in a captured graph: every replay gives the eager result of its inputs."""
    g = gen(9)
    q = torch.randn(3, 1, 8, 64, generator=g).cuda()
    z = torch.randn(3000, 64, generator=g).cuda()
    x, tokens, old, adv, wt, r, _, _ = policy_case(12, 9000, torch.bfloat16, 2, True, 1.0)
    x, args = x.cuda(), [t.cuda() for t in (tokens, old, adv, wt, r)]

    def run():
        rt = route(z, 6)
        return [*qk_norm_rope(q, q), rt.gates, rt.counts, rt.balance_loss, rt.z_loss,
                token_logprobs(x, args[0]), *policy_loss(x, *args, kl_coef=0.1)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        for t in (q, z, x):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, run()):
            assert torch.equal(a, b), i


def test_registered_ops_refuse_what_their_kernels_could_not_read():
    """The torch operators behind the entry points check what the kernels take by pointer."""
    ops = torch.ops.muonium_amd
    z = torch.randn(6, 8, device="cuda")
    tok = torch.zeros(6, dtype=torch.int64, device="cuda")
    f = torch.zeros(6, device="cuda")
    q = torch.randn(1, 3, 2, 16, device="cuda")
    for call in (lambda: ops.token_logprobs(z, tok.int(), 1.0, False),
                 lambda: ops.token_logprobs(z, tok[:5], 1.0, False),
                 lambda: ops.token_logprobs(z, tok.cpu(), 1.0, False),
                 lambda: ops.token_logprobs(z.double(), tok, 1.0, False),
                 lambda: ops.token_logprobs_backward(f, z, tok, f, 1.0),
                 lambda: ops.route(z, 2, torch.ones(5, dtype=torch.bool, device="cuda"), True),
                 lambda: ops.route(z, 9, None, True),
                 lambda: ops.route(z[0], 2, None, True),
                 lambda: ops.policy_loss(z, tok, f.double(), f, f, None, 0.2, 0.2, 0.0, 1.0, False, False),
                 lambda: ops.policy_loss(z.half(), tok, f, f, f, None, 0.2, 0.2, 0.0, 1.0, True, True),
                 lambda: ops.policy_loss_backward(f[0], z, tok, f, 1.0),
                 lambda: ops.qk_norm_rope(q, q[:, :2], None, None, None, None, None, 1e-6, False),
                 lambda: ops.qk_norm_rope(q, q, f, None, None, None, None, 1e-6, False),
                 lambda: ops.qk_norm_rope(q, q, None, None, z[:, :5], z[:, :5], tok[:2], 1e-6, False),
                 lambda: ops.qk_norm_rope(q, q, None, None, torch.ones(4, 9, device="cuda"),
                                          torch.ones(4, 9, device="cuda"), None, 1e-6, False)):
        with pytest.raises((RuntimeError, TypeError)):
            call()
    torch.cuda.synchronize()


def test_row_operators_have_no_second_derivative():
    x = leaf(torch.randn(4, 50, generator=gen(1)))
    y = token_logprobs(x, torch.zeros(4, dtype=torch.int64, device="cuda"))
    d, = torch.autograd.grad((y.sum(),), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        d.sum().backward()


def test_row_operators_are_well_behaved_torch_operators():
    """Schemas, autograd registration, fake implementations and ahead-of-time tracing."""
    ops = torch.ops.muonium_amd
    q, k = leaf(torch.randn(2, 3, 4, 32)), leaf(torch.randn(2, 3, 2, 32))
    w, cos = leaf(torch.ones(32)), torch.rand(9, 16, device="cuda")
    z = leaf(torch.randn(20, 16))
    tokens, f = torch.randint(0, 16, (20,), device="cuda"), torch.rand(20, device="cuda")
    torch.library.opcheck(ops.qk_norm_rope.default, (q, k, w, None, cos, cos, None, 1e-6, False))
    torch.library.opcheck(ops.route.default, (z, 2, f > 0.2, True))
    torch.library.opcheck(ops.token_logprobs.default, (z, tokens, 1.0, True))
    torch.library.opcheck(ops.policy_loss.default,
                          (z, tokens, f, f, f, None, 0.2, 0.2, 0.1, 1.0, True, False))


def test_row_operators_under_an_outer_compile():
    run = _all_calls(1)
    want = run()
    torch._dynamo.reset()
    got = torch.compile(run, backend="aot_eager")()
    torch._dynamo.reset()
    for i, (a, b) in enumerate(zip(got, want)):
        # the policy gradient takes its two-pass form there: one bf16 rounding apart
        torch.testing.assert_close(a, b, rtol=2.0**-7, atol=1e-6, msg=lambda m: f"{i}: {m}")
