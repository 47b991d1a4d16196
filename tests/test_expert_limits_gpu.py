"""The experts' products at the ends of what they take: nearly 2^31 rows, all of one expert or behind the last
one. Weights permute the columns and double them, so that every result is exact."""

import gc

import pytest
import torch

from muonium_amd.kernels import expert_linear

pytestmark = pytest.mark.gpu

MOST = 2**31 - 1  # rows


@pytest.fixture(autouse=True)
def memory():
    """Up to 140 GB, given back."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


def made(rows, width, dtype, seed):
    """Values from -1 to 1, two million rows over and over."""
    g = torch.Generator("cuda").manual_seed(seed)
    part = (torch.rand(1 << 21, width, generator=g, device="cuda") * 2 - 1).to(dtype)
    x = torch.empty(rows, width, dtype=dtype, device="cuda")
    for a in range(0, rows, 1 << 21):
        x[a:a + (1 << 21)] = part[:rows - a]
    return x, part


def check(got, part, factor):
    """got is the part's rows, over and over, rolled by a column, times the factor."""
    want = part.roll(1, 1) * factor
    bad = torch.zeros((), dtype=torch.int64, device="cuda")
    for a in range(0, len(got), len(part)):
        piece = got[a:a + len(part)]
        bad += (piece != want[:len(piece)]).sum()
    assert int(bad) == 0


def rolled(width, dtype):
    """(1, width, width): y = 2 x rolled by a column; the gradient's way rolls back."""
    return (2 * torch.eye(width, dtype=dtype, device="cuda")).roll(1, 0)[None].contiguous()


def run(width, dtype):
    w = rolled(width, dtype)
    x, part = made(MOST, width, dtype, 1)
    for offsets, factor in (((0, MOST), 2), ((0, 0), 0)):
        offsets = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        y = expert_linear(x, w, offsets)
        check(y, part, factor)
        # the rows' gradient of the transposed weight is the same product
        drows = torch.ops.muonium_amd.expert_linear_backward_rows(x, w.mT.contiguous(), offsets)
        del y
        check(drows, part, factor)
        del drows


def test_most_rows_of_direct_loads():
    run(8, torch.bfloat16)


@pytest.mark.parametrize("width, dtype", [(7, torch.bfloat16), (3, torch.float32)])
def test_most_rows_of_small_tiles(width, dtype):
    """2^24 tiles of 128 rows: as many workgroups of 256 and 512 threads have 2^32 threads and more."""
    run(width, dtype)
