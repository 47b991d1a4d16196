"""The experts' products where much is summed: long gradients of small matrices and of ragged ones, against
float64."""

import math

import pytest
import torch

from muonium_amd.kernels import expert_linear
from oracle import experts_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
E = 2.0**-24
HALVES = [torch.bfloat16, torch.float16]


def check(got, want, scale, k, what=""):
    """got within one rounding of its type and 2 k + 2 of fp32 at the result's scale."""
    dtype = got.dtype
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    off = (got - want).abs() - (U[dtype] * want.abs() + (2 * k + 2) * E * (1 + U[dtype]) * scale + TINY[dtype])
    assert off.max() <= 0, (what, off.max().item())  # a NaN is not


def made(counts, rest, out, width, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    n = int(offsets[-1]) + rest
    rows, dy = torch.randn(n, width, generator=g).to(dtype), torch.randn(n, out, generator=g).to(dtype)
    return rows, torch.randn(len(counts), out, width, generator=g).to(dtype), offsets, dy


LONG = [
    ([32768, 32768], 0, 64, 64),      # a tile or two for all rows
    ([16384], 7, 512, 512),
    ([65521, 15], 0, 24, 136),
    ([9000, 0, 4100, 1], 3, 1001, 777),  # no whole 16-byte runs, several hundred tiles
    ([8200, 8200], 0, 2050, 65),
]


@pytest.mark.parametrize("dtype", [*HALVES, torch.float32])
@pytest.mark.parametrize("counts, rest, out, width", LONG)
def test_long_gradients(counts, rest, out, width, dtype):
    rows, weight, offsets, dy = made(counts, rest, out, width, dtype)
    end = int(offsets[-1])
    rows[end:], dy[end:] = math.nan, math.inf
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y = expert_linear(x, w, offsets.cuda())
    dx, dw = torch.autograd.grad(y, (x, w), dy.cuda())
    check(y, *ref.linear(rows, weight, offsets), width, "y")
    want_x, scale_x, want_w, scale_w = ref.linear_grad(rows, weight, offsets, dy)
    check(dx, want_x, scale_x, out, "dx")
    check(dw, want_w, scale_w, max(counts), "dw")
