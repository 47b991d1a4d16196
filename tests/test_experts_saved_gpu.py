"""What the experts' operators keep for their backward passes: what its gradients read, and nothing else."""

import pytest
import torch

from muonium_amd.kernels import combine, dispatch, expert_linear, sort_by_expert

pytestmark = pytest.mark.gpu

TOKENS, TOP, EXPERTS, WIDTH, OUT = 21, 3, 4, 24, 16


def parts(**needs):
    g = torch.Generator().manual_seed(1)
    made = {"x": torch.randn(TOKENS, WIDTH, generator=g), "rows": torch.randn(TOKENS * TOP, WIDTH, generator=g),
            "gates": torch.rand(TOKENS, TOP, generator=g), "weight": torch.randn(EXPERTS, OUT, WIDTH, generator=g)}
    made = {n: t.cuda().requires_grad_(needs.get(n, False)) for n, t in made.items()}
    experts = torch.randint(-1, EXPERTS, (TOKENS, TOP), generator=g).cuda()
    return made, sort_by_expert(experts, EXPERTS)


def kept(call):
    """(result, the shapes of what it saved)."""
    shapes = []

    def pack(t):
        shapes.append(tuple(t.shape))
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        return call(), sorted(shapes)


SLOTS, ROWS, GATES, WEIGHT, OFFSETS = (TOKENS, TOP), (TOKENS * TOP, WIDTH), (TOKENS, TOP), (EXPERTS, OUT, WIDTH), (EXPERTS + 1,)


@pytest.mark.parametrize("needs, want", [
    ({"rows": True}, [SLOTS, GATES]),
    ({"gates": True}, [SLOTS, GATES, ROWS]),
    ({"rows": True, "gates": True}, [SLOTS, GATES, ROWS]),
])
def test_combine_keeps_the_rows_for_the_gates_alone(needs, want):
    p, order = parts(**needs)
    y, shapes = kept(lambda: combine(p["rows"], order, p["gates"]))
    assert shapes == sorted(want)
    dy = torch.randn_like(y)
    both, _ = parts(rows=True, gates=True)
    want = dict(zip(("rows", "gates"), torch.autograd.grad(combine(both["rows"], order, both["gates"]),
                                                           (both["rows"], both["gates"]), dy)))
    for n, got in zip(needs, torch.autograd.grad(y, [p[n] for n in needs], dy)):
        assert torch.equal(got, want[n])


@pytest.mark.parametrize("needs, want", [
    ({"rows": True}, [WEIGHT, OFFSETS]),
    ({"weight": True}, [ROWS, OFFSETS]),
    ({"rows": True, "weight": True}, [ROWS, WEIGHT, OFFSETS]),
])
def test_products_keep_each_for_the_others_gradient(needs, want):
    p, order = parts(**needs)
    y, shapes = kept(lambda: expert_linear(p["rows"], p["weight"], order.offsets))
    assert shapes == sorted(want)
    dy = torch.randn_like(y)
    both, _ = parts(rows=True, weight=True)
    want = dict(zip(("rows", "weight"), torch.autograd.grad(expert_linear(both["rows"], both["weight"], order.offsets),
                                                            (both["rows"], both["weight"]), dy)))
    for n, got in zip(needs, torch.autograd.grad(y, [p[n] for n in needs], dy)):
        assert torch.equal(got, want[n])


def test_others_keep_the_slots():
    p, order = parts(x=True, rows=True)
    assert kept(lambda: dispatch(p["x"], order))[1] == [SLOTS]
    assert kept(lambda: combine(p["rows"], order))[1] == [SLOTS]


def test_the_gates_gradient_asks_for_the_rows():
    p, order = parts()
    dy = torch.zeros(TOKENS, WIDTH, device="cuda")
    drows, dgates = torch.ops.muonium_amd.combine_backward(dy, None, order.slots, p["gates"], True, False)
    assert drows.shape == ROWS and dgates.shape == (0,)
    with pytest.raises(RuntimeError, match="takes the rows"):
        torch.ops.muonium_amd.combine_backward(dy, None, order.slots, p["gates"], False, True)


@pytest.mark.parametrize("lead", [(), (21,), (3, 7), (0, 7), (3, 0)])
def test_rows_of_no_columns(lead):
    """Of any leading dimensions, with their gradients."""
    order = sort_by_expert(torch.zeros(*lead, TOP, dtype=torch.int64, device="cuda"), EXPERTS)
    x = torch.zeros(*lead, 0, device="cuda", requires_grad=True)
    gates = torch.ones(*lead, TOP, device="cuda", requires_grad=True)
    rows = dispatch(x, order)
    assert rows.shape == (order.slots.numel(), 0)
    y = combine(rows, order, gates)
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape and torch.equal(gates.grad, torch.zeros_like(gates))
