"""AdamWFp8's state over one step and over many: its codes are those of the definition, bit for bit, and
what they stand for follows AdamW."""

import pytest
import torch

from muonium_amd import AdamWFp8

pytestmark = pytest.mark.gpu

ARGS = {"lr": 3e-3, "wd": 0.1, "betas": (0.9, 0.95), "eps": 1e-8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def decoded(q):
    """The values that codes and scales stand for, in fp32 as the step takes them, on the CPU."""
    return (q.codes.view(torch.float8_e4m3fn).cpu().float().view(-1, q.block_size) * q.scale.cpu()[:, None]).flatten()


def quantized(x, block):
    """(codes, scales) of x by the definition: x over absmax / 448 of its block, to nearest even."""
    x = x.view(-1, block)
    top = x.abs().amax(1)
    scale = torch.where(top < 1e-12, 1e-12, top) / torch.full((), 448.0)
    return (x / scale[:, None]).to(torch.float8_e4m3fn).flatten(), scale


def least(roots, means):
    """The roots' codes where a mean's code is not 0: the least one in place of 0."""
    return torch.where((roots.float() == 0) & (means.float() != 0), 2.0**-9, roots.float())


@pytest.mark.parametrize("block", [64, 256, 512, 2048])
def test_codes_are_the_quotients_by_the_scale(block):
    """Four million codes, whose moments take the same fp32 operations on the CPU: a product with the
    scale's inverse, an ulp off the quotient, falls on the other side of a code's border in some of them."""
    g = gen(1)
    n = 1 << 20
    p = torch.zeros(n).cuda().requires_grad_()
    opt = AdamWFp8([p], block_size=block, **ARGS)
    b1, b2 = ARGS["betas"]
    m, root = torch.zeros(n), torch.zeros(n)
    for _ in range(4):
        d = torch.randn(n, generator=g) * torch.exp(3 * torch.randn(n // 64, 1, generator=g)).expand(-1, 64).flatten()
        d[:64], d[-64:] = 0, d[-64:] * 1e-14  # a scale at its least
        p.grad = d.cuda()
        opt.step()
        m = m * b1 + d * (1 - b1)
        # a root through float64 is the correctly rounded one; torch's own in fp32 on the CPU is an ulp off at times
        root = (root * root * b2 + (d * d) * (1 - b2)).double().sqrt().float()
        (cm, sm), (cr, sr) = quantized(m, block), quantized(root, block)
        for name, codes, scale in (("exp_avg", cm.float(), sm), ("exp_avg_sq_root", least(cr, cm), sr)):
            q = opt.state[p][name]
            assert torch.equal(q.scale.cpu(), scale), name
            assert torch.equal(q.codes.view(torch.float8_e4m3fn).cpu().float(), codes), name
        m, root = (decoded(opt.state[p][name]) for name in ("exp_avg", "exp_avg_sq_root"))


# What happens beside a block's large value: its gradient at each step, and the small ones' size.
BESIDE = {
    "alternating": (lambda i: 1.0 if i % 2 else -1.0, 1.5e-6),
    "past": (lambda i: 100.0 if i == 0 else 0.0, 1e-5),
}


@pytest.mark.parametrize("name", BESIDE)
def test_a_small_mean_does_not_lose_its_root(name):
    """Small constant gradients g beside a large one, whose mean is soon far below its root, then none: AdamW in 64
    bits moves them by at most 1 lr, a root of 0 beside a mean moved them by 128 and 813. A root r at the least
    code stays there while the next one, sqrt(0.95 r^2 + 0.05 g^2), is below 1.5 codes, so g / r is below
    sqrt((1.5^2 - 0.95) / 0.05) = 5.1. A mean is g at most, and half a step of its code, 2^-4, more; without a
    gradient the step is 0.9 of the mean over 0.975 of the root, 5.0 lr, and smaller with one."""
    large, small = BESIDE[name]
    block = 256
    p = torch.zeros(4096).cuda().requires_grad_()
    opt = AdamWFp8([p], lr=1.0, wd=0.0, betas=(0.9, 0.95), eps=1e-8, block_size=block)
    worst = torch.zeros(4096)
    for i in range(160):
        d = torch.full((4096,), small if i % 40 < 39 else 0.0)  # a row that is not met every fortieth step
        d[::block] = large(i)
        p.grad = d.cuda()
        before = p.detach().cpu()
        opt.step()
        worst = torch.maximum(worst, (p.detach().cpu() - before).abs())
    inner = torch.ones(4096, dtype=torch.bool)
    inner[::block] = False
    assert worst[inner].max() <= 5.2
    m, root = (opt.state[p][n].codes.view(torch.float8_e4m3fn).float() for n in ("exp_avg", "exp_avg_sq_root"))
    assert not ((m != 0) & (root == 0)).any()


def test_a_root_without_a_mean_may_fall_out():
    """Every code is the nearest one, but for roots of 0 beside a mean's code that is not: then it is the least."""
    g = gen(2)
    n, block = 1 << 18, 256
    p = torch.zeros(n).cuda().requires_grad_()
    opt = AdamWFp8([p], block_size=block, **ARGS)
    b1, b2 = ARGS["betas"]
    m, root, raised, fallen = torch.zeros(n), torch.zeros(n), 0, 0
    for i in range(4):
        d = torch.randn(n, generator=g) * torch.exp(-5 * torch.rand(n, generator=g) ** 2 - 9)
        d[::block] = (-1.0) ** i
        p.grad = d.cuda()
        opt.step()
        m = m * b1 + d * (1 - b1)
        root = (root * root * b2 + (d * d) * (1 - b2)).double().sqrt().float()
        (cm, _), (cr, _) = quantized(m, block), quantized(root, block)
        lost = (cr.float() == 0) & (cm.float() != 0)
        raised, fallen = raised + int(lost.sum()), fallen + int(((cr.float() == 0) & ~lost).sum())
        assert torch.equal(opt.state[p]["exp_avg"].codes.view(torch.float8_e4m3fn).cpu().float(), cm.float())
        assert torch.equal(opt.state[p]["exp_avg_sq_root"].codes.view(torch.float8_e4m3fn).cpu().float(), least(cr, cm))
        m, root = (decoded(opt.state[p][name]) for name in ("exp_avg", "exp_avg_sq_root"))
    assert raised > 100 and fallen > 100


def run_of(betas, size, steps, varying, seed=5):
    """(root, its exact value, mean, its exact value) of the small values of a parameter whose gradients have
    size(i) at step i, beside one of size 1 in every block, after so many steps; exact: in float64."""
    n, block = 4096, 256
    g = torch.Generator("cuda").manual_seed(seed)
    p = torch.zeros(n, device="cuda", requires_grad=True)
    opt = AdamWFp8([p], lr=1e-3, betas=betas, block_size=block)
    p.grad = torch.zeros_like(p)
    sizes = torch.ones(n, device="cuda")
    inner = torch.arange(n, device="cuda") % block != 0
    m, v = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(steps):
        sizes.masked_fill_(inner, size(i))
        torch.mul(torch.randn(n, generator=g, device="cuda") if varying else 1.0, sizes, out=p.grad)
        opt.step()
        d = p.grad.double()
        m = m * betas[0] + d * (1 - betas[0])
        v = v * betas[1] + d * d * (1 - betas[1])
    held = [decoded(opt.state[p][name]).double()[inner.cpu()] for name in ("exp_avg_sq_root", "exp_avg")]
    return held[0], v.sqrt()[inner].cpu(), held[1], m[inner].cpu()


@pytest.mark.parametrize("varying", [True, False])
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("beta2, steps", [(0.99, 2500), (0.999, 4000)])
def test_roots_follow_gradients_whose_size_changes(beta2, steps, rising, varying):
    """A hundred times smaller or larger gradients after 300 steps, beside others that stay. A code rounded at
    random has the right mean, and a variance of at most step times move, where a step is 1/16 to 1/8 of a root
    and moves it by (1 - b2) / 2 of it for each size of its relative change, 1 on the average: 6% of v at most
    once it is steady, 3% of the root. Each of 4080 values is off by some ten percent, while it falls by
    fifty: 4 deviations of the mean are 3%. (Rounded to nearest the roots were 32 to 100 times too large after a
    fall, and half to a fifth of what they should be after a rise.) The mean, without varying gradients, is a
    linear recursion: no bias."""
    low, high = (0.5, 0.005) if rising else (0.005, 0.5)
    root, root64, mean, mean64 = run_of((0.9, beta2), lambda i: high if i < 300 else low, steps, varying)
    assert 0.97 <= (root.mean() / root64.mean()).item() <= 1.09
    if not varying:
        assert 0.97 <= (mean.mean() / mean64.mean()).item() <= 1.03


@pytest.mark.parametrize("rising", [False, True])
def test_roots_follow_varying_gradients_with_the_nearest_codes(rising):
    """At beta2 = 0.95 the scale, which moves by 2.5% or more a step, moves the codes: within a code's step, 1/8."""
    low, high = (0.5, 0.005) if rising else (0.005, 0.5)
    root, root64, *_ = run_of((0.9, 0.95), lambda i: high if i < 300 else low, 1000, True)
    assert 7 / 8 <= (root.mean() / root64.mean()).item() <= 9 / 8


def test_a_mean_decays_at_any_beta1():
    """Without further gradients, beside one of 1 that goes on. 0.3 for 30 steps leaves 0.14, which 512 steps bring to
    the least code, 2^-9 / 448; from there on it is lost with a chance of 1 in 50 a step, and kept over 1058
    with one of 5e-10. (The nearest codes are kept for good.)"""
    *_, mean, mean64 = run_of((0.98, 0.95), lambda i: 0.3 if i < 30 else 0.0, 1600, False)
    assert mean.abs().max() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_random_codes_are_the_neighbours_in_the_right_share(dtype):
    """Each is one of the two codes around the quotient, up by its distance from the lower one: the mean of a
    million differences, each within a step and at most half a step's deviation, is within 5 / 2048 steps of 0.
    The same step of the same values gives the same bits."""
    g = gen(3)
    n, block = 1 << 20, 256
    start, d = torch.randn(n, generator=g).to(dtype), torch.randn(n, generator=g).to(dtype)
    states = []
    for _ in range(2):
        p = start.cuda().requires_grad_()
        opt = AdamWFp8([p], block_size=block, lr=1e-3, betas=(0.9, 0.999))
        p.grad = d.cuda()
        opt.step()
        states.append(opt.state[p])
    x = d.float()
    for name, value in (("exp_avg", x * (1 - 0.9)), ("exp_avg_sq_root", ((x * x) * (1 - 0.999)).double().sqrt().float())):
        a, b = (s[name] for s in states)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)
        nearest, scale = quantized(value, block)
        assert torch.equal(a.scale.cpu(), scale)
        y = (value.view(-1, block) / scale[:, None]).flatten().double()
        got = a.codes.view(torch.float8_e4m3fn).cpu().double()
        step = torch.exp2(torch.log2(y.abs().clamp(min=2.0**-6)).floor() - 3)
        off = (got - y) / step
        assert off.abs().max() <= 1.0
        assert off.mean().abs() <= 5 / 2048 and (off * y.sign()).mean().abs() <= 5 / 2048
        assert (got != nearest.double()).float().mean() > 0.1


def test_captured_random_codes_are_those_of_the_steps():
    g = gen(4)
    values, grads = torch.randn(8192, generator=g), [torch.randn(8192, generator=g).cuda() for _ in range(5)]
    both = [values.cuda().requires_grad_() for _ in range(2)]
    opts = [AdamWFp8([p], betas=(0.9, 0.999)) for p in both]
    for p, o in zip(both, opts):
        p.grad = grads[0].clone()
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[1].step()
    for d in grads[1:]:
        for p in both:
            p.grad.copy_(d)
        opts[0].step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(*both)
        for name in ("exp_avg", "exp_avg_sq_root"):
            assert torch.equal(*(o.state[p][name].codes for p, o in zip(both, opts)))


def test_a_first_step_is_not_captured():
    """Its state would be zeros again in every replay. The optimizer is as it was, and steps on."""
    made = [AdamWFp8([torch.ones(8192, device="cuda").requires_grad_()]) for _ in range(2)]
    for opt in made:
        p = opt.param_groups[0]["params"][0]
        p.grad = torch.ones_like(p)
    made[0].step()
    p = made[1].param_groups[0]["params"][0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="no state while a graph is captured"):
        with torch.cuda.graph(graph):
            made[1].step()
    torch.cuda.synchronize()
    assert (p == 1).all() and not made[1].state[p]
    made[1].step()
    assert torch.equal(p, made[0].param_groups[0]["params"][0])


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.93, 0.9), (0.9, 0.999), (0.95, 0.95)])
def test_a_row_that_is_not_met_comes_to_rest(betas):
    """Rows of 64 values, four to a block, of which one goes on: the others' means lose a code at least a step
    without a gradient (at random one in ten or twenty steps: of 0.9^700 or 0.95^700 none is left), and are at 0
    after at most 130 + 17 codes' steps of them. AdamW in 64 bits moves such a row by under 1e-20 lr then; a
    mean that kept its last code moved it by 0.1 to 0.3 lr."""
    n = 4096
    g = torch.Generator("cuda").manual_seed(7)
    p = torch.zeros(n, device="cuda", requires_grad=True)
    opt = AdamWFp8([p], lr=1e-3, wd=0.0, betas=betas, block_size=256)
    met = torch.arange(n, device="cuda") // 64 % 4 == 0
    p.grad = torch.zeros_like(p)
    for i in range(2000):
        p.grad.normal_(generator=g)
        if i >= 50:
            p.grad.masked_fill_(~met, 0.0)
        if i == 1000:
            at_rest = p.detach().clone()
        opt.step()
    assert torch.equal(p.detach()[~met], at_rest[~met])
    assert not torch.equal(p.detach()[met], at_rest[met])
    codes = opt.state[p]["exp_avg"].codes.view(torch.float8_e4m3fn).float()
    assert (codes[~met] == 0).all() and (codes[met] != 0).any()
