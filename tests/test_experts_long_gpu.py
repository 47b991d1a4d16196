"""The experts' products where much is summed or many tiles are walked: long gradients of small matrices and of
ragged ones, offsets of any value in the 256-row tiles, and the size of fp32's errors, against float64."""

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


@pytest.mark.parametrize("dtype", HALVES)
def test_offsets_of_any_value_in_tiles_of_256(dtype):
    """4 experts of 2048 x 2048 and 4000 rows: outputs and both gradients walk tiles of 256. Falling, negative and
    too large offsets are taken into the rows; experts 0 and 2, which meet in some, have one weight."""
    rows, weight, _, dy = made([1000] * 4, 0, 2048, 2048, dtype)
    weight[2] = weight[0]
    given = torch.tensor([99, 1300, -2**31, 2600, 2**31 - 1], dtype=torch.int32)
    meant = [(0, 1300), (1300, 1300), (0, 2600), (2600, 4000)]
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y = expert_linear(x, w, given.cuda())
    dx, dw = torch.autograd.grad(y, (x, w), dy.cuda())
    bounds = torch.tensor([0, 2600, 4000])
    check(y, *ref.linear(rows, weight[2:], bounds), 2048, "y")
    want_x, scale_x, *_ = ref.linear_grad(rows, weight[2:], bounds, dy)
    check(dx, want_x, scale_x, 2048, "dx")
    for e, (a, b) in enumerate(meant):
        _, _, want, scale = ref.linear_grad(rows[a:b], weight[:1], torch.tensor([0, b - a]), dy[a:b])
        check(dw[e:e + 1], want, scale, 4000, e)


@pytest.mark.parametrize("form", ["y", "dx", "dw"])
def test_fp32_sums_are_added_in_parts(form):
    """Sums of 4096 random products in parts of 256. A running sum of j products has the size sqrt(j), and each addition
    an error of U / sqrt(3) of it: a part's are 104 U, sixteen parts' 416, their own additions' 108: 430 U beside a
    sum of size 64, or 6.7 U of it. One sum over all 4096 has 26 U, a product of fewer bits more than 100."""
    k, other = 4096, 300
    n, out, width = {"y": (other, 200, k), "dx": (other, k, 200), "dw": (k, 200, other)}[form]
    rows, weight, offsets, dy = made([n], 0, out, width, torch.float32)
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y = expert_linear(x, w, offsets.cuda())
    if form == "y":
        got, (want, _) = y.detach(), ref.linear(rows, weight, offsets)
    else:
        dx, dw = torch.autograd.grad(y, (x, w), dy.cuda())
        want_x, _, want_w, _ = ref.linear_grad(rows, weight, offsets, dy)
        got, want = (dx, want_x) if form == "dx" else (dw, want_w)
    off = got.double().cpu() - want
    assert off.square().mean().sqrt() / want.square().mean().sqrt() <= 8.4 * U[torch.float32]  # a quarter more
