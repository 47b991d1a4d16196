"""Tokens to their experts and back, the experts' products and AdamW without a device: what their
entry points refuse, what the C ABI refuses before any launch, the registrations, and the oracle of the
device tests against torch's own operations and autograd in float64."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from muonium_amd import AdamW, AdamWFp8, _lib
from muonium_amd.kernels import ExpertOrder, combine, dispatch, expert_linear, sort_by_expert
from oracle import experts_ref as ref

F32, I32, I64 = torch.float32, torch.int32, torch.int64


def t(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def order(*shape, n=4, dtype=I32):
    return ExpertOrder(t(*shape, dtype=dtype), t(n + 1, dtype=I32))


@pytest.mark.parametrize("call, error, match", [
    (lambda: sort_by_expert(t(dtype=I64), 4), ValueError, "experts are"),
    (lambda: sort_by_expert(t(3, 2, dtype=I32), 4), TypeError, "int64"),
    (lambda: sort_by_expert(t(3, 2, dtype=I64), 0), ValueError, "1024"),
    (lambda: sort_by_expert(t(3, 2, dtype=I64), 1025), ValueError, "1024"),
    (lambda: sort_by_expert(t(1, 1, dtype=I64).expand(2**16, 2**15), 4), ValueError, "2\\^31"),
    (lambda: sort_by_expert(t(3, 2, dtype=I64), 4), RuntimeError, "HIP device"),
    (lambda: dispatch(t(), order(2)), ValueError, "x is"),
    (lambda: dispatch(t(4, 8), order(3, 2)), ValueError, "x is"),
    (lambda: dispatch(t(2, 3, 8), order(3, 2)), ValueError, "x is"),
    (lambda: dispatch(t(3, 8, dtype=I32), order(3, 2)), TypeError, "fp32"),
    (lambda: dispatch(t(3, 8), order(3, 2, dtype=I64)), TypeError, "int32"),
    (lambda: dispatch(t(3, 8), order(3, 0)), ValueError, "slots are"),
    (lambda: dispatch(t(1, 1).expand(1, 2**30 + 1), order(1, 1)), ValueError, "columns"),
    (lambda: dispatch(t(3, 8), order(3, 2)), RuntimeError, "HIP device"),
    (lambda: combine(t(5, 8), order(3, 2)), ValueError, "rows are"),
    (lambda: combine(t(6), order(3, 2)), ValueError, "rows are"),
    (lambda: combine(t(6, 8, dtype=torch.float64), order(3, 2)), TypeError, "fp32"),
    (lambda: combine(t(6, 8), order(3, 2), t(3, 2, dtype=torch.bfloat16)), TypeError, "gates"),
    (lambda: combine(t(6, 8), order(3, 2), t(2, 3)), ValueError, "gates"),
    (lambda: combine(t(6, 8), order(3, 2), t(3, 2)), RuntimeError, "HIP device"),
    (lambda: expert_linear(t(6), t(4, 5, 6), t(5, dtype=I32)), ValueError, "rows are"),
    (lambda: expert_linear(t(6, 8), t(5, 8), t(5, dtype=I32)), ValueError, "rows are"),
    (lambda: expert_linear(t(6, 8), t(4, 5, 7), t(5, dtype=I32)), ValueError, "rows are"),
    (lambda: expert_linear(t(6, 8), t(4, 5, 8, dtype=torch.bfloat16), t(5, dtype=I32)), TypeError, "both"),
    (lambda: expert_linear(t(6, 8, dtype=I32), t(4, 5, 8, dtype=I32), t(5, dtype=I32)), TypeError, "both"),
    (lambda: expert_linear(t(6, 8), t(0, 5, 8), t(1, dtype=I32)), ValueError, "1024"),
    (lambda: expert_linear(t(6, 8), t(1025, 5, 8), t(1026, dtype=I32)), ValueError, "1024"),
    (lambda: expert_linear(t(6, 8), t(4, 5, 8), t(5, dtype=I64)), TypeError, "int32"),
    (lambda: expert_linear(t(6, 8), t(4, 5, 8), t(4, dtype=I32)), ValueError, "offsets"),
    (lambda: expert_linear(t(6, 1).expand(6, 2**24 + 8), t(1, 1, 1).expand(1, 1, 2**24 + 8), t(2, dtype=I32)), ValueError, "2\\^24"),
    (lambda: expert_linear(t(6, 8), t(4, 5, 8), t(5, dtype=I32)), RuntimeError, "HIP device"),
])
def test_entry_points_refuse(call, error, match):
    with pytest.raises(error, match=match):
        call()


def param(*shape, dtype=F32, grad=True):
    p = torch.nn.Parameter(t(*shape, dtype=dtype), requires_grad=dtype.is_floating_point)
    if grad:
        p.grad = t(*shape, dtype=dtype)
    return p


@pytest.mark.parametrize("kind", [AdamW, AdamWFp8])
@pytest.mark.parametrize("args, match", [
    ({"lr": -1.0}, "learning rate"), ({"lr": float("nan")}, "learning rate"), ({"eps": -1e-8}, "epsilon"),
    ({"wd": -0.1}, "weight decay"), ({"betas": (1.0, 0.9)}, "index 0"), ({"betas": (0.9, -0.1)}, "index 1"),
])
def test_optimizers_refuse_numbers(kind, args, match):
    with pytest.raises(ValueError, match=match):
        kind([param(3)], **args)
    opt = kind([param(3)])
    with pytest.raises(ValueError, match=match):
        opt.add_param_group({"params": [param(4)], **args})
    assert len(opt.param_groups) == 1


def test_optimizers_refuse():
    for size in (0, 32, 100, 4096, None):
        with pytest.raises(ValueError, match="block_size"):
            AdamWFp8([param(3)], block_size=size)
    with pytest.raises(RuntimeError, match="HIP device"):
        AdamW([param(3)]).step()
    with pytest.raises(TypeError, match="bf16"):
        AdamW([param(3, dtype=torch.float64)]).step()
    p = param(3, grad=False)
    AdamW([p]).step()  # nothing to do
    p = param(3, 2, grad=False)
    p.grad = torch.zeros(3, 2).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        AdamW([p]).step()


def tensor(numel, **other):
    """A MuonAdamTensor of plausible pointers."""
    values = {"param": 1, "grad": 1, "m": 1, "v": 1, "ms": 1, "vs": 1, "step": 1, **other}
    return (ctypes.c_int64 * 8)(*(values[n] or 0 for n in ("param", "grad", "m", "v", "ms", "vs", "step")), numel)


@pytest.mark.parametrize("call, code", [
    (lambda L: L.muon_expert_order(1, -1, 4, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_order(1, 1 << 31, 4, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_order(1, 3, 0, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_order(1, 3, 1025, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_order(None, 3, 4, 1, 1, 1, None), 5),
    (lambda L: L.muon_expert_order(1, 3, 4, 1, None, 1, None), 5),
    (lambda L: L.muon_expert_order(1, 100000, 4, 1, 1, None, None), 5),
    (lambda L: L.muon_dispatch(1, 3, 8, 2, 2, 8, 1, 1, None), 2),
    (lambda L: L.muon_dispatch(1, 0, 8, 2, 0, 8, 1, 1, None), 1),
    (lambda L: L.muon_dispatch(1, 0, 8, -1, 2, 8, 1, 1, None), 1),
    (lambda L: L.muon_dispatch(1, 0, 8, 1 << 30, 2, 8, 1, 1, None), 1),
    (lambda L: L.muon_dispatch(1, 0, 8, 2, 2, (1 << 30) + 1, 1, 1, None), 1),
    (lambda L: L.muon_dispatch(1, 0, 8, 2, 2, 8, None, 1, None), 5),
    (lambda L: L.muon_combine(1, 7, 8, 2, 2, 8, 1, 1, 1, None), 2),
    (lambda L: L.muon_combine(1, 0, 8, 2, 2, -1, 1, 1, 1, None), 1),
    (lambda L: L.muon_combine(None, 0, 8, 2, 2, 8, 1, 1, 1, None), 5),
    (lambda L: L.muon_combine_backward(1, 8, 1, 8, 4, 2, 2, 8, 1, 1, 1, 1, None), 2),
    (lambda L: L.muon_combine_backward(1, 8, 1, 8, 0, 2, 2, 8, 1, None, 1, 1, None), 5),
    (lambda L: L.muon_combine_backward(1, 8, None, 8, 0, 2, 2, 8, 1, 1, 1, 1, None), 5),
    (lambda L: L.muon_expert_linear(1, 3, 8, 4, 2, 8, 8, 1, 1, 1, None), 2),
    (lambda L: L.muon_expert_linear(1, 0, 8, 1 << 31, 2, 8, 8, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_linear(1, 0, 8, 4, 0, 8, 8, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_linear(1, 0, 8, 4, 1025, 8, 8, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_linear(1, 0, 8, 4, 2, (1 << 24) + 1, 8, 1, 1, 1, None), 1),
    (lambda L: L.muon_expert_linear(1, 0, 8, 4, 2, 8, 8, None, 1, 1, None), 5),
    (lambda L: L.muon_expert_linear(1, 0, 8, 4, 2, 8, 8, 1, None, 1, None), 5),
    (lambda L: L.muon_expert_linear_backward_rows(1, 3, 8, 4, 2, 8, 8, 1, 1, 1, None), 2),
    (lambda L: L.muon_expert_linear_backward_rows(None, 0, 8, 4, 2, 8, 8, 1, 1, 1, None), 5),
    (lambda L: L.muon_expert_linear_backward_weight(1, 3, 8, 1, 8, 4, 2, 8, 8, 1, 1, None), 2),
    (lambda L: L.muon_expert_linear_backward_weight(1, 0, 8, 1, 8, 4, 2, 8, 8, 1, None, None), 5),
    (lambda L: L.muon_adamw(1, tensor(8), 3, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 2),
    (lambda L: L.muon_adamw(1, tensor(4096), 0, 32, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw(1, tensor(4096), 0, 192, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw(1, tensor(4096), 0, 4096, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw(1, tensor(4100), 0, 256, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw(1, tensor(-1), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw(-1, tensor(8), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw((1 << 20) + 1, tensor(8), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
    (lambda L: L.muon_adamw(1, tensor(8, grad=None), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 5),
    (lambda L: L.muon_adamw(1, tensor(8, step=None), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 5),
    (lambda L: L.muon_adamw(1, tensor(4096, vs=None), 0, 256, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 5),
    (lambda L: L.muon_adamw(1, tensor(8), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, None, None), 5),
    (lambda L: L.muon_adamw(1, tensor(1 << 40), 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 1, None), 1),
])
def test_abi_refuses_without_launching(call, code):
    assert call(_lib.load()) == code
    assert _lib.last_error() != ""


def test_abi_calls_with_nothing_to_do_return_ok():
    lib = _lib.load()
    assert lib.muon_dispatch(None, 0, 8, 0, 2, 8, None, None, None) == 0
    assert lib.muon_combine(None, 0, 8, 0, 2, 8, None, None, None, None) == 0
    assert lib.muon_combine_backward(None, 8, None, 8, 0, 2, 2, 8, None, None, None, None, None) == 0
    assert lib.muon_expert_linear(None, 0, 8, 0, 2, 8, 8, None, None, None, None) == 0
    assert lib.muon_expert_linear_backward_rows(None, 0, 8, 4, 2, 8, 0, None, None, None, None) == 0
    assert lib.muon_expert_linear_backward_weight(None, 0, 8, None, 8, 4, 2, 0, 8, None, None, None) == 0
    assert lib.muon_adamw(0, None, 0, 0, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, None, None) == 0
    assert lib.muon_expert_order_workspace_bytes(100, 64) == 0
    assert lib.muon_expert_order_workspace_bytes(1 << 20, 64) % (65 * 4) == 0
    assert lib.muon_expert_order_workspace_bytes(1 << 20, 64) > 65 * 4
    assert lib.muon_expert_order_workspace_bytes(8193, 1025) == -1
    assert lib.muon_adamw_workspace_bytes(-1) == -1
    assert lib.muon_adamw_workspace_bytes(3) > 3 * 64


def test_registered_ops_run_on_fake_tensors():
    ops = torch.ops.muonium_amd
    with FakeTensorMode():
        e = torch.empty(5, 3, device="cuda", dtype=I64)
        slots, offsets = ops.sort_by_expert(e, 8)
        assert slots.shape == (5, 3) and offsets.shape == (9,) and slots.dtype == offsets.dtype == I32
        x = torch.empty(5, 16, device="cuda", dtype=torch.bfloat16)
        rows = ops.dispatch(x, slots)
        assert rows.shape == (15, 16) and rows.dtype == x.dtype
        gates = torch.empty(5, 3, device="cuda")
        y = ops.combine(rows, slots, gates)
        assert y.shape == x.shape and y.dtype == x.dtype
        a, b = ops.combine_backward(y, rows, slots, gates, True, False)
        assert a.shape == rows.shape and b.shape == (0,)
        a, b = ops.combine_backward(y, rows, slots, gates, False, True)
        assert a.shape == (0,) and b.shape == gates.shape and b.dtype == F32
        w = torch.empty(8, 24, 16, device="cuda", dtype=torch.bfloat16)
        z = ops.expert_linear(rows, w, offsets)
        assert z.shape == (15, 24) and z.dtype == x.dtype
        assert ops.expert_linear_backward_rows(z, w, offsets).shape == rows.shape
        assert ops.expert_linear_backward_weight(z, rows, offsets).shape == w.shape
        p = torch.empty(7, device="cuda")
        s = torch.empty((), device="cuda")
        assert ops.adamw_([p], [p], [p], [p], [], [], [s], 0, 0.1, 0.9, 0.9, 1e-8, 0.0, False) is None


# ---- the oracle against torch in float64 ------------------------------------------------------


def close(a, b):
    torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-13)


def test_oracle_of_the_experts():
    g = torch.Generator().manual_seed(1)
    e = torch.randint(-1, 5, (20, 3), generator=g)
    slots, offsets = ref.order(e, 4)
    # every row once; sorted by expert, tokens in order within one
    rows = torch.where(slots >= 0, slots, -1 - slots).flatten()
    assert torch.equal(rows.sort().values, torch.arange(60, dtype=I32))
    kept = (e >= 0) & (e < 4)
    assert torch.equal(slots >= 0, kept)
    listed = [n for x in range(4) for n in (e.flatten() == x).nonzero()[:, 0].tolist()]
    assert [int(rows[n]) for n in listed] == list(range(int(kept.sum())))
    assert offsets.tolist() == [0, *(int((e[kept] <= x).sum()) for x in range(4))]

    def double(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_()

    x, gates, w = double(20, 6), double(20, 3), double(4, 5, 6)
    one_hot = torch.where(kept[..., None], torch.nn.functional.one_hot(e.clamp(0, 3), 4), 0).double()
    by_hand = torch.einsum("tke,eoi,ti->tko", one_hot, w, x)
    y = (gates[..., None] * by_hand).sum(1)
    dy = torch.randn(20, 5, generator=g, dtype=torch.float64)
    dx, dgates, dw = torch.autograd.grad(y, (x, gates, w), dy)
    sent = ref.dispatch(x.detach(), slots)
    made, _ = ref.linear(sent, w.detach(), offsets)
    close(ref.combine(made, slots, gates.detach())[0], y.detach())
    drows, dg, _ = ref.combine_grad(made, slots, gates.detach(), dy)
    close(dg, dgates)
    dsent, _, dweight, _ = ref.linear_grad(sent, w.detach(), offsets, drows)
    close(dweight, dw)
    close(ref.combine(dsent, slots, None)[0], dx)


@pytest.mark.parametrize("maximize", [False, True])
def test_oracle_of_adamw(maximize):
    g = torch.Generator().manual_seed(2)
    p = torch.randn(30, generator=g, dtype=torch.float64)
    theirs = p.clone().requires_grad_()
    opt = torch.optim.AdamW([theirs], lr=0.01, weight_decay=0.1, betas=(0.8, 0.95), eps=1e-6, maximize=maximize)
    m = v = torch.zeros(30, dtype=torch.float64)
    for step in (1, 2, 3):
        theirs.grad = torch.randn(30, generator=g, dtype=torch.float64)
        p, m, v, root, _ = ref.adamw(p, theirs.grad, m, v, step, 0.01, 0.1, (0.8, 0.95), 1e-6, maximize)
        opt.step()
        close(p, theirs.detach())
        close(root.square(), v)
