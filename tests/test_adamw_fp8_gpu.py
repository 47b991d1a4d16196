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
