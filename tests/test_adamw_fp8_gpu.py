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
        for name, x in (("exp_avg", m), ("exp_avg_sq_root", root)):
            codes, scale = quantized(x, block)
            q = opt.state[p][name]
            assert torch.equal(q.scale.cpu(), scale), name
            assert torch.equal(q.codes.view(torch.float8_e4m3fn).cpu().float(), codes.float()), name
        m, root = (decoded(opt.state[p][name]) for name in ("exp_avg", "exp_avg_sq_root"))
