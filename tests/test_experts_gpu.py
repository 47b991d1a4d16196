"""Tokens to their experts and back, and the experts' products, against their definitions in float64
(oracle/experts_ref.py).

Tolerances. U is half a unit in the last place of the output's type, the one rounding at the end. Inside,
everything is fp32, E = 2^-24 a rounding of a result's scale (the sum of the magnitudes that meet in it): a
sum over k choices is at most k + 1 roundings deep (its products and its additions); a gate's gradient
adds the products of a lane's columns, 8 lanes a row at the least and 64 at the most, and joins the lanes
in 6 additions. A product of matrices over K is K products and K additions deep; the products of 16-bit
values are exact in fp32, and the matrix cores' additions are counted as two roundings each."""

import math

import pytest
import torch

from muonium_amd.kernels import (ExpertOrder, combine, dispatch, expert_linear, route,
                                 sort_by_expert)
from oracle import experts_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
E = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(got, want, scale, k, what=""):
    """got within one rounding of its type and k of fp32 at the result's scale."""
    dtype = got.dtype
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    off = (got - want).abs() - (U[dtype] * want.abs() + k * E * (1 + U[dtype]) * scale + TINY[dtype])
    off = off[~want.isnan()]
    assert off.numel() == 0 or off.max() <= 0, (what, off.max().item())


def gen(seed):
    return torch.Generator().manual_seed(seed)


def some_experts(g, tokens, k, n, empty=0.2, kind="random"):
    """Choices with empty ones, numbers that name no expert, and the same expert twice in a token."""
    e = torch.randint(0, n, (tokens, k), generator=g)
    if kind == "one":
        e[:] = n // 2
    if kind == "skewed":
        e = torch.where(torch.rand(tokens, k, generator=g) < 0.7, torch.tensor(n - 1), e)
    away = torch.tensor([-1, n, -2**63, 2**63 - 1, n + 2**32, -5])
    out = torch.rand(tokens, k, generator=g) < empty
    e[out] = away[torch.randint(0, 6, (int(out.sum()),), generator=g)]
    return e


# ---- the order ------------------------------------------------------------------------------

ORDERS = [
    # tokens, k, experts, share of empty choices, kind
    (0, 3, 5, 0.0, "random"),
    (1, 1, 1, 0.0, "random"),
    (1, 8, 64, 0.0, "random"),
    (16, 8, 64, 0.1, "random"),
    (33, 2, 7, 1.0, "random"),       # nothing goes anywhere
    (100, 3, 1024, 0.1, "random"),
    (513, 1, 2, 0.0, "one"),
    (512, 8, 64, 0.1, "skewed"),     # the most that one workgroup orders
    (513, 8, 64, 0.1, "skewed"),     # the least that several do
    (1025, 8, 64, 0.1, "skewed"),
    (4099, 5, 63, 0.3, "random"),
    (3001, 4, 255, 0.2, "random"),
    (30011, 1, 1024, 0.05, "random"),
]


@pytest.mark.parametrize("tokens, k, n, empty, kind", ORDERS)
def test_order(tokens, k, n, empty, kind):
    e = some_experts(gen(1), tokens, k, n, empty, kind)
    got = sort_by_expert(e.cuda(), n)
    slots, offsets = ref.order(e, n)
    assert got.slots.dtype == got.offsets.dtype == torch.int32
    assert torch.equal(got.offsets.cpu(), offsets)
    assert torch.equal(got.slots.cpu(), slots)


def test_order_of_many_choices():
    """Chunks of more than the least size: 256 workgroups of 4608 choices."""
    e = torch.randint(-1, 200, (1 << 17, 9), generator=gen(2)).cuda()
    got = sort_by_expert(e, 200)
    key = torch.where(e < 0, 200, e).flatten()
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order).scatter_(0, order, torch.arange(len(order), device="cuda"))
    want = torch.where(key < 200, place, -1 - place).view(e.shape)
    assert torch.equal(got.slots.long(), want)
    counts = torch.bincount(key, minlength=201)[:200]
    assert torch.equal(got.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))


def test_order_of_shapes_and_strides():
    e = some_experts(gen(3), 24, 6, 9)
    whole = sort_by_expert(e.view(2, 3, 4, 6).cuda(), 9)
    assert whole.slots.shape == (2, 3, 4, 6)
    flat = sort_by_expert(e.cuda(), 9)
    assert torch.equal(whole.slots.view(24, 6), flat.slots)
    strided = sort_by_expert(e.cuda().t().contiguous().t(), 9)
    assert torch.equal(strided.slots, flat.slots) and torch.equal(strided.offsets, flat.offsets)


# ---- rows -----------------------------------------------------------------------------------

ROWS = [
    # tokens, k, width, experts
    (1, 1, 1, 1),
    (1, 8, 2048, 64),
    (5, 3, 7, 4),
    (17, 8, 64, 16),
    (130, 2, 1001, 8),
    (31, 9, 515, 5),      # more choices than are in flight together
    (9, 64, 40, 70),
    (3, 17, 4100, 6),     # more columns than a workgroup's lanes
    (257, 4, 24, 3),
    (64, 1, 8, 64),
]


def rows_case(tokens, k, width, n, dtype, seed=5):
    g = gen(seed)
    e = some_experts(g, tokens, k, n)
    slots, offsets = ref.order(e, n)
    x = torch.randn(tokens, width, generator=g).to(dtype)
    rows = torch.randn(tokens * k, width, generator=g).to(dtype)
    gates = torch.rand(tokens, k, generator=g)
    dy = torch.randn(tokens, width, generator=g).to(dtype)
    return e, slots, offsets, x, rows, gates, dy


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, k, width, n", ROWS)
def test_dispatch(tokens, k, width, n, dtype):
    e, slots, _, x, drows, _, _ = rows_case(tokens, k, width, n, dtype)
    order = sort_by_expert(e.cuda(), n)
    leaf = x.cuda().requires_grad_()
    rows = dispatch(leaf, order)
    assert torch.equal(rows.detach().cpu().double(), ref.dispatch(x, slots))
    # what comes back for the rows behind the last expert's reaches nothing
    d = drows.clone()
    d[int(order.offsets[-1]):] = math.nan
    dx, = torch.autograd.grad(rows, leaf, d.cuda())
    want, scale = ref.combine(drows, slots, None)
    check(dx, want, scale, k, "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, k, width, n", ROWS)
def test_combine(tokens, k, width, n, dtype):
    e, slots, offsets, _, rows, gates, dy = rows_case(tokens, k, width, n, dtype)
    order = sort_by_expert(e.cuda(), n)
    # nothing of what is empty is read: not its gates, not the rows behind the last expert's
    rows[int(offsets[-1]):] = math.nan
    gates[slots < 0] = math.inf
    leaf, g = rows.cuda().requires_grad_(), gates.cuda().requires_grad_()
    y = combine(leaf, order, g)
    want, scale = ref.combine(rows, slots, gates)
    check(y, want, scale, k + 1, "y")
    drows, dgates = torch.autograd.grad(y, (leaf, g), dy.cuda())
    want_rows, want_gates, scale = ref.combine_grad(rows, slots, gates, dy)
    check(drows, want_rows, want_rows.abs(), 1, "drows")
    runs = -(-width // (4 if dtype == torch.float32 else 8))
    lanes = min(64, max(8, 1 << (runs - 1).bit_length()))
    lane = -(-runs // lanes) * (4 if dtype == torch.float32 else 8)
    check(dgates, want_gates, scale, 2 * lane + 6, "dgates")
    # ones for gates
    y = combine(leaf, order)
    want, scale = ref.combine(rows, slots, None)
    check(y, want, scale, k, "sum")
    drows, = torch.autograd.grad(y, leaf, dy.cuda())
    assert torch.equal(drows.cpu().double(), ref.dispatch(dy, slots))


@pytest.mark.parametrize("wanted", ["rows", "gates"])
def test_one_gradient_of_combine_alone(wanted):
    e, slots, _, _, rows, gates, dy = rows_case(33, 3, 72, 6, torch.bfloat16)
    order = sort_by_expert(e.cuda(), 6)
    both = rows.cuda().requires_grad_(), gates.cuda().requires_grad_()
    whole = torch.autograd.grad(combine(both[0], order, both[1]), both, dy.cuda())
    one = [t.detach().requires_grad_(wanted == name) for t, name in zip(both, ("rows", "gates"))]
    y = combine(one[0], order, one[1])
    i = 0 if wanted == "rows" else 1
    assert torch.equal(torch.autograd.grad(y, one[i], dy.cuda())[0], whole[i])
    # and one of two that both may
    y = combine(both[0], order, both[1])
    assert torch.equal(torch.autograd.grad(y, both[i], dy.cuda())[0], whole[i])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_other_strides(dtype):
    """Slices of wider rows, columns that are not contiguous, a gradient that is one value expanded."""
    e, slots, _, x, rows, gates, _ = rows_case(21, 4, 40, 5, dtype)
    order = sort_by_expert(e.cuda(), 5)
    wide = torch.zeros(21, 99, dtype=dtype)
    wide[:, 3:43] = x
    flipped = x.t().contiguous().cuda().t()
    for one in (wide.cuda()[:, 3:43], flipped, x.cuda()[:, :1].expand(-1, 40)):
        assert torch.equal(dispatch(one, order).cpu().double(), ref.dispatch(one.cpu(), slots))
    tall = torch.zeros(84, 77, dtype=dtype)
    tall[:, 5:45] = rows
    for one in (tall.cuda()[:, 5:45], rows.t().contiguous().cuda().t(), rows.cuda()[:1].expand(84, -1)):
        leaf = one.detach().requires_grad_()
        g = gates.cuda().t().contiguous().t().requires_grad_()
        y = combine(leaf, order, g)
        want, scale = ref.combine(one.cpu(), slots, gates)
        check(y, want, scale, 5, "y")
        y.float().sum().backward()
        ones = torch.ones(21, 40)
        want_rows, want_gates, scale = ref.combine_grad(one.cpu(), slots, gates, ones)
        check(leaf.grad, want_rows, want_rows.abs(), 1, "drows")
        check(g.grad, want_gates, scale, 22, "dgates")


@pytest.mark.parametrize("lead", [(), (3,), (2, 3)])
def test_leading_dimensions(lead):
    n = math.prod(lead)
    e, slots, _, x, rows, gates, _ = rows_case(n, 2, 16, 3, torch.float32)
    order = sort_by_expert(e.view(*lead, 2).cuda(), 3)
    assert order.slots.shape == (*lead, 2)
    assert torch.equal(dispatch(x.view(*lead, 16).cuda(), order).cpu().double(), ref.dispatch(x, slots))
    y = combine(rows.cuda(), order, gates.view(*lead, 2).cuda())
    assert y.shape == (*lead, 16)
    want, scale = ref.combine(rows, slots, gates)
    check(y.view(n, 16), want, scale, 3)


def test_rows_of_nothing():
    order = sort_by_expert(torch.zeros(0, 3, dtype=torch.int64, device="cuda"), 4)
    assert order.offsets.tolist() == [0] * 5
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    rows = dispatch(x, order)
    y = combine(rows, order, torch.zeros(0, 3, device="cuda"))
    assert rows.shape == (0, 8) and y.shape == (0, 8)
    y.sum().backward()
    assert x.grad.shape == (0, 8)
    order = sort_by_expert(torch.zeros(3, 2, dtype=torch.int64, device="cuda"), 4)
    gates = torch.ones(3, 2, device="cuda", requires_grad=True)
    y = combine(dispatch(torch.zeros(3, 0, device="cuda"), order), order, gates)
    assert y.shape == (3, 0)
    y.sum().backward()
    assert torch.equal(gates.grad, torch.zeros(3, 2, device="cuda"))


def test_slots_out_of_range_are_left_out():
    """Slots of somebody's own making: nothing outside the rows is read or written."""
    slots = torch.tensor([[0, 4], [2**31 - 1, -2**31], [3, -3], [1, 8]], dtype=torch.int32)
    order = ExpertOrder(slots.cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"))
    x = torch.arange(1.0, 13).view(4, 3)
    rows = dispatch(x.cuda(), order).cpu()
    for row, token in ((0, 0), (4, 0), (3, 2), (1, 3)):
        assert torch.equal(rows[row], x[token])
    some = torch.arange(24.0).view(8, 3)
    y = combine(some.cuda(), order, torch.ones(4, 2, device="cuda")).cpu()
    assert torch.equal(y, torch.stack([some[0] + some[4], torch.zeros(3), some[3], some[1]]))


def test_infinities_and_nan_go_where_they_belong():
    e = torch.tensor([[0, 1], [1, -1], [0, 0]])
    order = sort_by_expert(e.cuda(), 2)
    x = torch.ones(3, 5)
    x[0, 1], x[2, 3] = math.nan, math.inf
    assert torch.equal(dispatch(x.cuda(), order).cpu().double().nan_to_num(7),
                       ref.dispatch(x, order.slots.cpu()).nan_to_num(7))
    rows = torch.ones(6, 5)
    rows[int(order.slots[0, 1])] = math.nan
    y = combine(rows.cuda(), order, torch.ones(3, 2, device="cuda")).cpu()
    assert y[0].isnan().all() and y[1:].isfinite().all()


def among_nan(t, after=5):
    """t on the GPU, in the middle of rows of NaN."""
    wide = torch.full((t.shape[0], t.shape[1] + 2 + after), math.nan, dtype=t.dtype)
    wide[:, 2:2 + t.shape[1]] = t
    return wide.cuda()[:, 2:2 + t.shape[1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 2, 3, 8])
@pytest.mark.parametrize("width", [3, 4, 5, 8, 9, 13, 15, 31, 517])
def test_ends_of_rows(width, k, dtype):
    """The last columns, which two lanes may have, count once, and what lies beside a row is not read."""
    e, slots, _, x, rows, gates, dy = rows_case(41, k, width, 6, dtype)
    rows[::5, -1], dy[3::7, -2] = math.inf, -math.inf
    rows[2::9, max(0, width - 6)] = math.nan
    order = sort_by_expert(e.cuda(), 6)
    assert torch.equal(dispatch(among_nan(dy), order).cpu().double(), ref.dispatch(dy, slots))
    leaf, g = among_nan(rows).requires_grad_(), gates.cuda().requires_grad_()
    y = combine(leaf, order, g)
    got = (y, *torch.autograd.grad(y, (leaf, g), among_nan(dy)))
    want, scale = ref.combine(rows, slots, gates)
    want_rows, want_gates, scale_gates = ref.combine_grad(rows, slots, gates, dy)
    for a, b, c, n, what in ((got[0], want, scale, k + 1, "y"), (got[1], want_rows, want_rows.abs(), 1, "drows"),
                             (got[2], want_gates, scale_gates, 2 * 16 + 6, "dgates")):
        inf = b.isinf()
        assert torch.equal(a.cpu().double()[inf], b[inf]), what
        check(a.cpu().masked_fill(inf, 0), b.masked_fill(inf, 0), c.masked_fill(inf, 0), n, what)


# ---- products -------------------------------------------------------------------------------

PRODUCTS = [
    # rows of each expert, rows behind them, out, in
    ([1], 0, 1, 1),
    ([0, 3, 0], 2, 8, 8),
    ([5, 0, 70, 1], 9, 24, 40),
    ([300, 17, 0, 256], 0, 264, 72),
    ([64, 65, 63], 1, 128, 64),
    ([2, 1, 3, 0, 2], 0, 1408, 512),       # a few rows each
    ([33, 128, 257], 60, 96, 200),         # no whole K-tile
    ([7, 0, 20], 3, 33, 19),               # odd everywhere
    ([129, 1], 0, 257, 129),
    ([40, 300], 5, 100, 260),
    ([0, 0], 12, 16, 16),                  # nobody's rows
    ([0] * 70 + [3] + [1] * 30 + [0] * 29, 2, 16, 32),  # several experts to a lane
    ([513], 0, 72, 16),
]


def product_case(counts, rest, out, width, dtype, seed=7):
    g = gen(seed)
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    n = int(offsets[-1]) + rest
    rows, dy = torch.randn(n, width, generator=g).to(dtype), torch.randn(n, out, generator=g).to(dtype)
    weight = torch.randn(len(counts), out, width, generator=g).to(dtype)
    return rows, weight, offsets, dy


def depth(k, dtype):
    return 2 * k + 2 if dtype != torch.float32 else 2 * k


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(PRODUCTS)))
def test_expert_linear(case, dtype):
    counts, rest, out, width = PRODUCTS[case]
    rows, weight, offsets, dy = product_case(counts, rest, out, width, dtype)
    end = int(offsets[-1])
    # rows behind the last expert's reach nothing
    rows[end:], dy[end:] = math.nan, math.inf
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y = expert_linear(x, w, offsets.cuda())
    want, scale = ref.linear(rows, weight, offsets)
    check(y, want, scale, depth(width, dtype), "y")
    dx, dw = torch.autograd.grad(y, (x, w), dy.cuda())
    want_x, scale_x, want_w, scale_w = ref.linear_grad(rows, weight, offsets, dy)
    check(dx, want_x, scale_x, depth(out, dtype), "dx")
    check(dw, want_w, scale_w, depth(max(counts), dtype), "dw")
    # the same bits again, and for each gradient alone
    again = expert_linear(x, w, offsets.cuda())
    assert torch.equal(again, y)
    assert torch.equal(torch.autograd.grad(again, x, dy.cuda(), retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(again, w, dy.cuda())[0], dw)


@pytest.mark.parametrize("dtype", TYPES)
def test_products_of_other_strides(dtype):
    rows, weight, offsets, dy = product_case([20, 3, 41], 4, 48, 56, dtype)
    wide = torch.zeros(len(rows), 131, dtype=dtype)
    wide[:, 3:59] = rows
    even = torch.zeros(len(rows), 128, dtype=dtype)
    even[:, 8:64] = rows
    want, scale = ref.linear(rows, weight, offsets)
    _, _, want_w, scale_w = ref.linear_grad(rows, weight, offsets, dy)
    slow = weight.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    odd = torch.zeros(weight.numel() + 1, dtype=dtype).cuda()
    odd[1:] = weight.flatten().cuda()
    for x in (wide.cuda()[:, 3:59], even.cuda()[:, 8:64], rows.t().contiguous().cuda().t()):
        for w in (weight.cuda(), slow, odd[1:].view(weight.shape)):
            leaf = w.detach().requires_grad_()
            y = expert_linear(x, leaf, offsets.cuda())
            check(y, want, scale, depth(56, dtype), "y")
            dw, = torch.autograd.grad(y, leaf, dy.cuda().t().contiguous().t())
            check(dw, want_w, scale_w, depth(41, dtype), "dw")
    # a gradient that is one value expanded
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    expert_linear(x, w, offsets.cuda()).float().sum().backward()
    want_x, scale_x, want_w, scale_w = ref.linear_grad(rows, weight, offsets, torch.ones(dy.shape))
    check(x.grad, want_x, scale_x, depth(48, dtype), "dx")
    check(w.grad, want_w, scale_w, depth(41, dtype), "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out, width", [(1, 7), (7, 8), (8, 9), (9, 15), (15, 65), (65, 71), (72, 127),
                                        (127, 129), (129, 136), (136, 1), (130, 250)])
def test_products_among_nan(out, width, dtype):
    """Runs that end with a matrix's row bring nothing of what lies beside it."""
    rows, weight, offsets, dy = product_case([70, 0, 61, 3], 2, out, width, dtype)
    x, d, w = among_nan(rows), among_nan(dy), weight.cuda().requires_grad_()
    y = expert_linear(x.requires_grad_(), w, offsets.cuda())
    want, scale = ref.linear(rows, weight, offsets)
    check(y, want, scale, depth(width, dtype), "y")
    dx, dw = torch.autograd.grad(y, (x, w), d)
    want_x, scale_x, want_w, scale_w = ref.linear_grad(rows, weight, offsets, dy)
    check(dx, want_x, scale_x, depth(out, dtype), "dx")
    check(dw, want_w, scale_w, depth(70, dtype), "dw")


MANY = [
    # outputs and gradients of so many rows, or of so large weights, that wider tiles are taken
    ([0, 1, 3000, 255, 4001, 257], 30, 1000, 72, TYPES),
    ([0, 1, 3000, 255, 4001, 257], 30, 72, 1000, TYPES),
    ([7400, 300], 0, 1032, 8, TYPES),
    ([3000, 0, 1, 255, 4001, 257], 1, 968, 1032, TYPES),       # whole K-tiles and a part
    ([0, 1, 70, 64, 65, 513, 0, 8] * 8, 3, 520, 512, TYPES),
    ([8200], 0, 264, 40, TYPES),                                # one expert's long gradient
    ([1, 20000, 0, 22000], 5, 1024, 20, [torch.float32]),
    ([1, 20000, 0, 22000], 5, 17, 1027, [torch.float32]),
    ([5, 0, 40, 33] * 2, 2, 2050, 2047, [torch.float32]),
]


@pytest.mark.parametrize("case, dtype", [(i, t) for i, c in enumerate(MANY) for t in c[4]])
def test_many_rows_and_large_weights(case, dtype):
    counts, rest, out, width, _ = MANY[case]
    rows, weight, offsets, dy = product_case(counts, rest, out, width, dtype)
    end = int(offsets[-1])
    rows[end:], dy[end:] = math.nan, math.inf
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y = expert_linear(x, w, offsets.cuda())
    want, scale = ref.linear(rows, weight, offsets)
    check(y, want, scale, depth(width, dtype), "y")
    dx, dw = torch.autograd.grad(y, (x, w), dy.cuda())
    want_x, scale_x, want_w, scale_w = ref.linear_grad(rows, weight, offsets, dy)
    check(dx, want_x, scale_x, depth(out, dtype), "dx")
    check(dw, want_w, scale_w, depth(max(counts), dtype), "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, out, width", [(0, 8, 16), (5, 0, 16), (5, 8, 0)])
def test_products_of_nothing(rows, out, width, dtype):
    x = torch.ones(rows, width, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.ones(2, out, width, dtype=dtype, device="cuda", requires_grad=True)
    y = expert_linear(x, w, torch.tensor([0, min(rows, 2), rows], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, torch.zeros(rows, out, dtype=dtype, device="cuda"))
    y.sum().backward()
    assert torch.equal(x.grad, torch.zeros_like(x)) and torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_of_any_value_read_nothing_out_of_range(dtype):
    """Offsets behind the rows, below 0 and falling ones are taken into the rows; the first counts as 0."""
    rows, weight, _, dy = product_case([40], 0, 16, 24, dtype)
    weight = torch.cat([weight] * 3)
    given = torch.tensor([7, 2**31 - 1, -2**31, 41], dtype=torch.int32)
    meant = [(0, 40), (40, 40), (0, 40)]
    x, w = rows.cuda().requires_grad_(), weight.cuda().requires_grad_()
    y = expert_linear(x, w, given.cuda())
    want, scale = ref.linear(rows, weight[:1], torch.tensor([0, 40]))
    check(y, want, scale, depth(24, dtype), "y")
    dw, = torch.autograd.grad(y, w, dy.cuda())
    for e, (a, b) in enumerate(meant):
        _, _, want, scale = ref.linear_grad(rows[a:b], weight[:1], torch.tensor([0, b - a]), dy[a:b])
        check(dw[e:e + 1], want, scale, depth(40, dtype), e)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite_stays_with_its_rows(dtype):
    rows, weight, offsets, dy = product_case([30, 40], 0, 24, 72, dtype)
    rows[3, 70], weight[1, 5, 1] = math.nan, math.inf
    y = expert_linear(rows.cuda(), weight.cuda(), offsets.cuda()).cpu().double()
    want, _ = ref.linear(rows, weight, offsets)
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.isinf(), want.isinf())


# ---- against differences --------------------------------------------------------------------


def test_gradients_against_differences():
    """All three operators are linear in each input: f(x + d) - f(x) = f(d), and <f(d), g> is <d, the
    gradient>. In fp32 both sums of n products agree within n roundings of their magnitudes."""
    g = gen(11)
    e = some_experts(g, 50, 3, 6)
    order = sort_by_expert(e.cuda(), 6)

    def randn(*shape):
        return torch.randn(*shape, generator=g).cuda()

    def agree(f, x):
        d = randn(*x.shape)
        leaf = x.clone().requires_grad_()
        y = f(leaf)
        dy = randn(*y.shape)
        grad, = torch.autograd.grad(y, leaf, dy)
        change = (f(x + d) - f(x)).double()
        a, b = (change * dy.double()).sum(), (d.double() * grad.double()).sum()
        # every value of f(x + d) and of f(x) is off by at most 200 roundings of its sums' magnitudes
        room = 200 * E * 2 * (f((x.abs() + d.abs())).abs() + 40).double().mul(dy.double().abs()).sum()
        assert (a - b).abs() <= room, (a.item(), b.item(), room.item())

    rows, gates = randn(150, 36), randn(50, 3)
    weight = randn(6, 20, 36)
    agree(lambda x: dispatch(x, order), randn(50, 36))
    agree(lambda x: combine(x, order, gates), rows)
    agree(lambda x: combine(rows, order, x), gates)
    agree(lambda x: expert_linear(x, weight, order.offsets), rows)
    agree(lambda x: expert_linear(rows, x, order.offsets), weight)


# ---- together -------------------------------------------------------------------------------


def layer(x, z, up, down, k, mask=None):
    """A layer of experts on the operators: routed, sent, through two products, and back."""
    r = route(z, k, token_mask=mask)
    order = sort_by_expert(r.experts, z.shape[-1])
    hidden = torch.relu(expert_linear(dispatch(x, order), up, order.offsets)).square()
    return combine(expert_linear(hidden, down, order.offsets), order, r.gates), r


def test_a_layer_of_experts_gives_what_all_experts_on_all_tokens_give():
    """Against every expert on every token in float64, gradients included. In fp32 the longest chain is
    two products of 48 and 64 terms with a square between, about 4 * 112 roundings; 2^-24 of the
    largest magnitudes each, which the bound takes as the result's largest value times 16."""
    g = gen(13)
    t, w, h, n, k = 60, 48, 64, 7, 3
    x, z = torch.randn(2, t // 2, w, generator=g), torch.randn(2, t // 2, n, generator=g)
    up, down = torch.randn(n, h, w, generator=g) * w**-0.5, torch.randn(n, w, h, generator=g) * h**-0.5
    mask = torch.rand(2, t // 2, generator=g) > 0.2
    leaves = [y.cuda().requires_grad_() for y in (x, z, up, down)]
    out, r = layer(*leaves, k, mask.cuda())
    dy = torch.randn(out.shape, generator=g)
    grads = torch.autograd.grad(out, leaves, dy.cuda())

    exact = [y.double().requires_grad_() for y in (x, z, up, down)]
    fx, fz, fup, fdown = exact
    p = fz.softmax(-1)
    top = p.topk(k, -1)
    share = torch.zeros_like(p).scatter(-1, top.indices, top.values / top.values.sum(-1, keepdim=True))
    share = share * mask[..., None]
    hidden = torch.einsum("btw,ehw->bteh", fx, fup).relu().square()
    want = torch.einsum("bte,bteh,ewh->btw", share, hidden, fdown)
    want_grads = torch.autograd.grad(want, exact, dy.double())
    for a, b in zip((out, *grads), (want, *want_grads)):
        assert (a.detach().double().cpu() - b).abs().max() <= 448 * E * 16 * b.abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_layer(dtype):
    """Forward and backward passes in a graph, replayed on other inputs, with eager work between."""
    g = gen(17)
    t, w, h, n, k = 70, 64, 40, 8, 2

    def inputs():
        return [(torch.randn(*s, generator=g) * 0.3).to(dtype).cuda()
                for s in ((t, w), (t, n), (n, h, w), (n, w, h), (t, w))]

    def run(x, z, up, down, dy):
        leaves = [y.detach().requires_grad_() for y in (x, z, up, down)]
        out, _ = layer(*leaves, k)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    held = inputs()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(*held)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = run(*held)
    for _ in range(4):
        for old, new in zip(held, inputs()):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = run(*held)
        for a, b in zip(made, want):
            assert torch.equal(a, b)


def test_captured_products_of_many_rows():
    """Products and gradients in wide tiles, replayed on other rows and other offsets."""
    g = gen(37)
    n, experts, out, width = 7500, 16, 1024, 1032

    def inputs():
        at = torch.randint(0, n, (experts - 1,), generator=g).sort().values
        return (torch.randn(n, width, generator=g).bfloat16(), torch.randn(experts, out, width, generator=g).bfloat16(),
                torch.cat([torch.zeros(1, dtype=torch.int64), at, torch.tensor([n - 3])]).clamp(max=n - 3).int(),
                torch.randn(n, out, generator=g).bfloat16())

    def run(x, w, offsets, dy):
        leaf, wleaf = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = expert_linear(leaf, wleaf, offsets)
        return (y.detach(), *torch.autograd.grad(y, (leaf, wleaf), dy))

    held = [t.cuda() for t in inputs()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*held)
    for _ in range(3):
        for to, t in zip(held, inputs()):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run(*held)):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    g = gen(19)
    cases = []
    for _ in range(2):
        cases.append([torch.randn(*s, generator=g).cuda() for s in ((3000, 64), (3000, 16), (16, 48, 64), (16, 64, 48))])
    want = [layer(*c, 4)[0] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(*cases[i], 4)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_outer_compile_gives_the_same_bits():
    """One operator a graph: what inductor makes of the torch operations around them may round otherwise."""
    g = gen(23)
    z, x = torch.randn(40, 8, generator=g).cuda(), torch.randn(40, 32, generator=g).cuda()
    w = torch.randn(8, 24, 32, generator=g).cuda()
    r = route(z, 2)

    def step(x, gates, w, experts):
        order = sort_by_expert(experts, 8)
        return combine(expert_linear(dispatch(x, order), w, order.offsets), order, gates)

    dy = torch.randn(40, 24, generator=g).cuda()
    both = []
    for f in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        leaves = [y.detach().requires_grad_() for y in (x, r.gates, w)]
        out = f(*leaves, r.experts)
        both.append([out.detach(), *torch.autograd.grad(out, leaves, dy)])
    for a, b in zip(*both):
        assert torch.equal(a, b)


def test_well_behaved_torch_operators():
    ops = torch.ops.muonium_amd
    e = torch.tensor([[0, 1], [2, -1], [1, 1]], device="cuda")
    order = sort_by_expert(e, 3)
    x, rows = (torch.randn(n, 16, device="cuda", requires_grad=True) for n in (3, 6))
    gates = torch.rand(3, 2, device="cuda", requires_grad=True)
    w = torch.randn(3, 8, 16, device="cuda", requires_grad=True)
    torch.library.opcheck(ops.sort_by_expert.default, (e, 3))
    torch.library.opcheck(ops.dispatch.default, (x, order.slots))
    torch.library.opcheck(ops.combine.default, (rows, order.slots, gates))
    torch.library.opcheck(ops.combine.default, (rows, order.slots, None))
    torch.library.opcheck(ops.expert_linear.default, (rows, w, order.offsets))


def test_no_second_and_no_forward_derivative():
    order = sort_by_expert(torch.tensor([[0, 1], [2, -1]], device="cuda"), 3)
    x, rows = (torch.randn(n, 16, device="cuda", requires_grad=True) for n in (2, 4))
    gates = torch.rand(2, 2, device="cuda", requires_grad=True)
    w = torch.randn(3, 8, 16, device="cuda", requires_grad=True)
    calls = [(lambda a: dispatch(a, order), x), (lambda a: combine(a, order, gates), rows),
             (lambda a: combine(rows, order, a), gates), (lambda a: expert_linear(a, w, order.offsets), rows),
             (lambda a: expert_linear(rows, a, order.offsets), w)]
    import torch.autograd.forward_ad as fwad
    for f, a in calls:
        y = f(a)
        d, = torch.autograd.grad(y, a, torch.ones_like(y).requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.sum().backward()
        with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(fwad.make_dual(a.detach(), torch.ones_like(a)))


# ---- offsets past 32 bits ---------------------------------------------------------------------


def test_rows_behind_offsets_past_32_bits():
    """300000 tokens of 8 choices, width 1024: 2.5e9 values of rows."""
    t, k, w, n = 300000, 8, 1024, 16
    e = torch.randint(0, n, (t, k), device="cuda")
    order = sort_by_expert(e, n)
    x = torch.randn(t, w, device="cuda", dtype=torch.bfloat16)
    rows = dispatch(x, order)
    flat = order.slots.view(-1).long()
    last = torch.arange(t * k - 100, t * k, device="cuda")
    source = torch.empty_like(flat).scatter_(0, flat, torch.arange(t * k, device="cuda") // k)
    assert torch.equal(rows[last], x[source[last]])
    back = combine(rows, order)
    assert torch.equal(back[-100:].float(), (x[-100:].float() * k).bfloat16().float())
    weight = torch.randn(n, 8, w, device="cuda", dtype=torch.bfloat16) * 0.03
    y = expert_linear(rows, weight, order.offsets)
    a = int(order.offsets[-2])
    at = torch.arange(max(a, t * k - 50), t * k, device="cuda")
    want = rows[at].double() @ weight[-1].double().T
    scale = rows[at].double().abs() @ weight[-1].double().abs().T
    check(y[at], want.cpu(), scale.cpu(), depth(w, torch.bfloat16), "y")
    dx, = torch.autograd.grad(expert_linear(rows.requires_grad_(), weight, order.offsets), rows, y)
    want = y[at].double() @ weight[-1].double()
    scale = y[at].double().abs() @ weight[-1].double().abs()
    check(dx[at], want.cpu(), scale.cpu(), depth(8, torch.bfloat16), "dx")


@pytest.mark.parametrize("wide", ["out", "stride"])
def test_extents_beyond_what_direct_loads_index(wide):
    """A result of 2^20 + 8 columns; rows 2^20 + 8 values apart: 32 bits would not do for 256 of them."""
    n, far = 300, 2**20 + 8
    g = gen(29)
    rows = torch.randn(n, 16, generator=g).bfloat16().cuda()
    offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    if wide == "out":
        weight = torch.randn(1, far, 16, generator=g).bfloat16().cuda()
    else:
        weight = torch.randn(1, 16384, 16, generator=g).bfloat16().cuda()
        spread = torch.zeros(n, far, dtype=torch.bfloat16, device="cuda")
        rows = spread[:, 8:24].copy_(rows)
    y = expert_linear(rows, weight, offsets)
    at = torch.cat([torch.arange(40), torch.arange(weight.shape[1] - 40, weight.shape[1])]).cuda()
    want = rows.double() @ weight[0, at].double().T
    scale = rows.double().abs() @ weight[0, at].double().abs().T
    check(y[:, at], want.cpu(), scale.cpu(), depth(16, torch.bfloat16))


def test_many_rows_of_many_experts():
    """More row tiles than a wave counts in one go, experts of none to thousands of rows, in whole tiles."""
    g = gen(31)
    counts = torch.randint(0, 40, (200,), generator=g)
    counts[::7] = torch.randint(200, 3000, (29,), generator=g)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int()
    n, out, width = int(offsets[-1]) + 100, 1032, 328
    x, dy = (torch.randn(n, w, generator=g).bfloat16().cuda() for w in (width, out))
    w = torch.randn(200, out, width, generator=g).bfloat16().cuda()
    leaf, wleaf = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = expert_linear(leaf, wleaf, offsets.cuda())
    dx, dw = torch.autograd.grad(y, (leaf, wleaf), dy)
    assert (y[int(offsets[-1]):] == 0).all() and (dx[int(offsets[-1]):] == 0).all()
    for e, (a, b) in enumerate(ref.spans(offsets)):
        xe, de, we = x[a:b].double(), dy[a:b].double(), w[e].double()
        for got, p, q in ((y[a:b], xe, we.T), (dx[a:b], de, we), (dw[e], de.T, xe)):
            check(got, (p @ q).cpu(), (p.abs() @ q.abs()).cpu(), depth(p.shape[1], torch.bfloat16), e)
