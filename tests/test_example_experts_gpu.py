"""The experts of examples/policy_experts.py, forward and gradients, against every expert on every token
in float64."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "policy_experts.py")


def test_experts_of_the_example():
    """In fp32 the longest chain is a router's product of 128 terms with its softmax, and two products of
    128 terms with a square between, forward and back: about 4 * 2 * 128 roundings of 2^-24 of the largest
    magnitudes that meet, at most 16 times the result's largest value."""
    spec = importlib.util.spec_from_file_location("policy_experts", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(3)
    layer = example.Layer()
    x, dy, dz = torch.randn(2, 9, example.WIDTH), torch.randn(2, 9, example.WIDTH), 0.3
    names = ("router", "up", "down")
    exact = [t.detach().double().requires_grad_() for t in (x, *(getattr(layer, n) for n in names))]
    fx, router, up, down = exact
    z = fx @ router.T
    p = z.softmax(-1)
    top = p.topk(example.TOP, -1)
    share = torch.zeros_like(p).scatter(-1, top.indices, top.values / top.values.sum(-1, keepdim=True))
    hidden = torch.einsum("btw,ehw->bteh", fx, up).relu().square()
    want = torch.einsum("bte,bteh,ewh->btw", share, hidden, down)
    zloss = z.logsumexp(-1).square().mean()
    grads = torch.autograd.grad([want, zloss], exact, [dy.double(), torch.tensor(dz, dtype=torch.float64)])

    layer = layer.cuda()
    leaf = x.cuda().requires_grad_()
    y, r = layer.experts(leaf)
    assert torch.equal(r.experts.cpu(), top.indices)
    got = torch.autograd.grad([y, r.z_loss], [leaf, *(getattr(layer, n) for n in names)],
                              [dy.cuda(), torch.tensor(dz).cuda()])
    for a, b in zip((y, *got), (want, *grads)):
        assert (a.detach().double().cpu() - b).abs().max() <= 1024 * 2.0**-24 * 16 * b.abs().max()
