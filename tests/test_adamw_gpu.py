"""AdamW and AdamWFp8 against the step's definition in float64 (oracle/experts_ref.py).

Tolerances. U is half a unit in the last place of the parameter's type, E = 2^-24. In fp32 a new moment is
two products, their rounded constants and a sum: 5 roundings of the magnitudes that meet in it. The
change of a parameter is the quotient of such a mean and a root: the mean's 5, half of the square's 6 and 1
of its root, and at most 10 of the constants, products and quotients around them: 20 roundings of its
size; the decayed parameter and the difference add 4 of the parameter's. An fp8 code is half a step of its
scale's units off, 2^-4 of the value or 2^-10 units where values have no exponent left, and its scale 6
roundings."""

import copy

import pytest
import torch

from muonium_amd import AdamW, AdamWFp8, Muon
from muonium_amd.optim import OptimStateFp8
from oracle import experts_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
E = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ARGS = {"lr": 3e-3, "wd": 0.1, "betas": (0.9, 0.95), "eps": 1e-8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def leaf(t):
    return t.cuda().requires_grad_()


def held(state):
    """The moments of a parameter's state, m and v, as float64 on the CPU."""
    if "exp_avg_sq_root" in state:
        decode = [(s.codes.view(torch.float8_e4m3fn).double().view(-1, s.block_size)
                   * s.scale.double()[:, None]).view(s.shape).cpu()
                  for s in (state["exp_avg"], state["exp_avg_sq_root"])]
        return decode[0], decode[1].square()
    return state["exp_avg"].double().cpu(), state["exp_avg_sq"].double().cpu()


def close(got, want, room, what):
    got = got.detach().double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), what
    off = ((got - want).abs() - room)[~want.isnan()]
    assert off.numel() == 0 or off.max() <= 0, (what, off.max().item())


def check_step(p, before, grad, moments, state, number, args, maximize=False):
    """What a step left of a parameter, given what it found."""
    want, m, v, root, change = ref.adamw(before, grad, *moments, number, args["lr"], args["wd"],
                                         args["betas"], args["eps"], maximize)
    b1, b2 = args["betas"]
    size = (b1 * moments[0]).abs() + ((1 - b1) * grad.double()).abs()
    grown = torch.where(m != 0, change.abs() / m.abs() * size, 0.0)
    close(p, want, U[p.dtype] * want.abs() + E * (1 + U[p.dtype]) * (4 * before.double().abs() + 20 * grown)
          + TINY[p.dtype], "p")
    assert state["step"].item() == number
    if "exp_avg_sq_root" not in state:
        close(state["exp_avg"], m, 5 * E * size + TINY[torch.float32], "m")
        close(state["exp_avg_sq"], v, 5 * E * v + TINY[torch.float32], "v")
        return
    for name, x, slack in (("exp_avg", m, 5 * E * size), ("exp_avg_sq_root", root, 5 * E * root)):
        s = state[name]
        top = x.view(-1, s.block_size).abs().amax(1)
        scale = top.clamp(min=1e-12) / 448
        far = slack.view(-1, s.block_size).amax(1) / 448
        close(s.scale, scale, 6 * E * scale + far, name + " scale")
        units = scale[:, None]
        got = (s.codes.view(torch.float8_e4m3fn).double().cpu().view(-1, s.block_size)
               * s.scale.double().cpu()[:, None])
        x = x.view(-1, s.block_size)
        room = torch.maximum(2.0**-4 * x.abs(), 2.0**-10 * units) * (1 + 2.0**-20)
        close(got, x, room + 16 * E * x.abs() + slack.view(x.shape), name)


SHAPES = [(1,), (7,), (64, 64), (2048,), (4099,), (33, 257), (4096, 3), (130, 256), (1, 1), (6, 4096), (0,), (0, 5)]


@pytest.mark.parametrize("maximize", [False, True])
@pytest.mark.parametrize("kind", [AdamW, AdamWFp8])
@pytest.mark.parametrize("dtype", TYPES)
def test_steps(dtype, kind, maximize):
    g = gen(1)
    params = [leaf((torch.randn(s, generator=g)).to(dtype)) for s in SHAPES]
    opt = kind(params, maximize=maximize, **ARGS)
    for number in range(1, 5):
        grads = [(torch.randn(s, generator=g) * 0.01).to(dtype) for s in SHAPES]
        for p, d in zip(params, grads):
            p.grad = d.cuda()
        before = [p.detach().cpu() for p in params]
        moments = [held(opt.state[p]) if opt.state.get(p) else (torch.zeros(p.shape),) * 2 for p in params]
        opt.step()
        for p, old, d, mom in zip(params, before, grads, moments):
            check_step(p, old, d, mom, opt.state[p], number, ARGS, maximize)
    fp8 = [isinstance(opt.state[p]["exp_avg"], OptimStateFp8) for p in params]
    whole = [kind is AdamWFp8 and p.numel() >= 4096 and p.numel() % 256 == 0 for p in params]
    assert fp8 == whole


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [64, 128, 256, 512, 1024, 2048])
def test_blocks(block, dtype):
    """Every block size; numbers of blocks that leave waves and workgroups partly filled."""
    g = gen(2)
    shapes = [(4096,), (block * 67 if block * 67 >= 4096 else block * 131,), (2048 * 9 + block * 3,)]
    params = [leaf((torch.randn(s, generator=g)).to(dtype)) for s in shapes]
    opt = AdamWFp8(params, block_size=block, **ARGS)
    for number in (1, 2, 3):
        # blocks of very different sizes beside each other, one of zeros, one of tiny values
        grads = [(torch.randn(s, generator=g).view(-1, block)
                  * torch.exp(2 * torch.randn(s[0] // block, 1, generator=g))).view(s).to(dtype) for s in shapes]
        for d in grads:
            d.view(-1, block)[1] = 0
            d.view(-1, block)[2:3] *= 1e-6
        for p, d in zip(params, grads):
            p.grad = d.cuda()
        before = [p.detach().cpu() for p in params]
        moments = [held(opt.state[p]) if opt.state.get(p) else (torch.zeros(p.shape),) * 2 for p in params]
        opt.step()
        for p, old, d, mom in zip(params, before, grads, moments):
            assert opt.state[p]["exp_avg"].block_size == block
            check_step(p, old, d, mom, opt.state[p], number, ARGS)


@pytest.mark.parametrize("args", [
    {"lr": 0.0, "wd": 0.0, "betas": (0.0, 0.0), "eps": 1e-8},
    {"lr": 1e-2, "wd": 0.0, "betas": (0.0, 0.999), "eps": 1e-3},
    {"lr": 1e-2, "wd": 1.0, "betas": (0.95, 0.0), "eps": 1e-6},
])
def test_numbers_at_their_ends(args):
    g = gen(3)
    p = leaf(torch.randn(5000, generator=g))
    opt = AdamW([p], **args)
    for number in (1, 2, 3):
        d = torch.randn(5000, generator=g)
        before, mom = p.detach().cpu(), held(opt.state[p]) if opt.state.get(p) else (torch.zeros(5000),) * 2
        p.grad = d.cuda()
        opt.step()
        check_step(p, before, d, mom, opt.state[p], number, args)


def test_against_torch():
    """Twenty steps beside torch's AdamW in fp32. Each step of either is off by at most 24 roundings of
    the change's and the parameter's sizes, at most 1 and 1e-2 here, and what differs goes on: the
    moments of both see the same gradients."""
    g = gen(4)
    values = [torch.randn(s, generator=g).clamp(-1, 1) for s in ((300, 20), (17,))]
    mine, theirs = [leaf(v.clone()) for v in values], [leaf(v.clone()) for v in values]
    opt = AdamW(mine, lr=1e-3, wd=0.05, betas=(0.9, 0.999), eps=1e-8)
    other = torch.optim.AdamW(theirs, lr=1e-3, weight_decay=0.05, betas=(0.9, 0.999), eps=1e-8)
    for _ in range(20):
        for a, b in zip(mine, theirs):
            a.grad = torch.randn(a.shape, generator=g).cuda()
            b.grad = a.grad.clone()
        opt.step()
        other.step()
    for a, b in zip(mine, theirs):
        assert (a - b).abs().max() <= 20 * 2 * 24 * E * (1 + 1e-2)


def test_many_tensors():
    """More than two tables of tensors, empty ones among them, the last piece of work far from the
    first; each as if it were alone."""
    g = gen(5)
    shapes = [(int(n),) for n in torch.randint(0, 300, (131,), generator=g)] + [(70001,), (0,), (5,)]
    values = [torch.randn(s, generator=g) for s in shapes]
    grads = [torch.randn(s, generator=g) for s in shapes]
    together, alone = [leaf(v.clone()) for v in values], [leaf(v.clone()) for v in values]
    opt = AdamW(together, **ARGS)
    single = [AdamW([p], **ARGS) for p in alone]
    for _ in range(2):
        for p, q, d in zip(together, alone, grads):
            p.grad, q.grad = d.cuda(), d.cuda()
        opt.step()
        for o in single:
            o.step()
    for p, q, o in zip(together, alone, single):
        assert torch.equal(p, q)
        for name in ("step", "exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[p][name], o.state[q][name])


@pytest.mark.parametrize("kind", [AdamW, AdamWFp8])
def test_parameters_of_other_layouts(kind):
    """Transposed, sliced and expanded storage, gradients laid out otherwise, starts off 16 bytes."""
    g = gen(6)
    base = torch.randn(64, 128, generator=g)
    grad = torch.randn(64, 128, generator=g)
    flat = torch.zeros(64 * 128 + 1).cuda()
    wide = torch.zeros(64, 300).cuda()
    made = {
        "plain": base.cuda(),
        "transposed": base.t().contiguous().cuda().t(),
        "sliced": wide[:, 7:135].copy_(base),
        "unaligned": flat[1:].view(64, 128).copy_(base),
    }
    left = {}
    for name, t in made.items():
        for turned in (False, True):
            p = t.detach().clone(memory_format=torch.preserve_format) if name != "sliced" else t.detach()
            if name == "unaligned":
                p = t.detach()
            p.copy_(base)
            p = p.requires_grad_()
            opt = kind([p], **ARGS)
            for scale in (1.0, -0.5):
                d = (grad * scale).cuda()
                p.grad = d.t().contiguous().t() if turned else d
                opt.step()
            left[name, turned] = p.detach().contiguous()
    for value in left.values():
        assert torch.equal(value, left["plain", False])
    assert (wide[:, :7] == 0).all() and (wide[:, 135:] == 0).all() and flat[0] == 0


def test_parameters_that_share_memory():
    """A weight and a view of a part of it: one after the other, in their order."""
    g = gen(7)
    base, grad = torch.randn(40, 8, generator=g), torch.randn(40, 8, generator=g)
    whole = base.cuda().requires_grad_()
    part = whole.detach()[:, ::2].requires_grad_()  # not dense either
    opt = AdamW([whole, part], **ARGS)
    whole.grad, part.grad = grad.cuda(), grad[:, ::2].cuda()
    opt.step()
    one, two = base.cuda().requires_grad_(), None
    a = AdamW([one], **ARGS)
    one.grad = grad.cuda()
    a.step()
    two = one.detach()[:, ::2].contiguous().requires_grad_()
    b = AdamW([two], **ARGS)
    two.grad = grad[:, ::2].contiguous().cuda()
    b.step()
    want = one.detach().clone()
    want[:, ::2] = two.detach()
    assert torch.equal(whole.detach(), want)


def test_groups_types_and_missing_gradients():
    g = gen(8)
    a, b, c, d = (leaf(torch.randn(5000, generator=g).to(t)) for t in (*TYPES, torch.float32))
    opt = AdamW([{"params": [a, b]}, {"params": [c, d], "lr": 1e-2, "wd": 0.0, "betas": (0.8, 0.9), "eps": 1e-6}], **ARGS)
    other = {"lr": 1e-2, "wd": 0.0, "betas": (0.8, 0.9), "eps": 1e-6}
    before = [p.detach().cpu() for p in (a, b, c, d)]
    grads = [torch.randn(5000, generator=g).to(p.dtype) for p in (a, b, c, d)]
    for p, x in zip((a, b, c), grads):
        p.grad = x.cuda()
    assert opt.step(lambda: torch.tensor(2.5)).item() == 2.5
    zero = (torch.zeros(5000),) * 2
    for p, old, x, args in zip((a, b, c), before, grads, (ARGS, ARGS, other)):
        check_step(p, old, x, zero, opt.state[p], 1, args)
    assert torch.equal(d.detach().cpu(), before[3]) and d not in opt.state


def test_nan_and_infinite_gradients_stay_in_their_values_or_blocks():
    for kind, reach in ((AdamW, 1), (AdamWFp8, 256)):
        p = leaf(torch.ones(8192))
        opt = kind([p], **ARGS)
        p.grad = torch.full((8192,), 0.5).cuda()
        opt.step()
        p.grad[300], p.grad[5000] = float("nan"), float("inf")
        opt.step()
        assert p[[300, 5000]].isnan().all() and int(p.isnan().sum()) == 2
        p.grad = torch.full((8192,), 0.5).cuda()
        opt.step()
        bad = p.isnan().nonzero()[:, 0].tolist()
        assert bad == [i for at in (300, 5000) for i in range(at // reach * reach, at // reach * reach + reach)]


@pytest.mark.parametrize("kind", [AdamW, AdamWFp8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoint(kind, dtype, tmp_path):
    """A saved and loaded optimizer steps on as the one that was saved, moments in fp32 for 16-bit
    parameters too."""
    g = gen(9)
    shapes = [(64, 64), (130,)]
    first = [leaf(torch.randn(s, generator=g).to(dtype)) for s in shapes]
    opt = kind(first, **ARGS)
    grads = [[torch.randn(s, generator=g).to(dtype).cuda() for s in shapes] for _ in range(3)]

    def step(o, params, ds):
        for p, d in zip(params, ds):
            p.grad = d
        o.step()

    step(opt, first, grads[0])
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    second = [p.detach().clone().requires_grad_() for p in first]
    for where in ("cpu", "cuda"):
        loaded = kind([p.detach().clone().requires_grad_() for p in second], **ARGS)
        loaded.load_state_dict(torch.load(tmp_path / "opt.pt", map_location=where, weights_only=True))
        params = loaded.param_groups[0]["params"]
        mine = copy.deepcopy(opt)
        for ds in grads[1:]:
            step(loaded, params, ds)
            step(mine, mine.param_groups[0]["params"], ds)
        for p, q in zip(params, mine.param_groups[0]["params"]):
            assert torch.equal(p, q)
            assert loaded.state[p]["step"].item() == 3 and loaded.state[p]["step"].device == p.device
            for x, y in zip(held(loaded.state[p]), held(mine.state[q])):
                assert torch.equal(x, y)
            if "exp_avg_sq" in loaded.state[p]:
                assert loaded.state[p]["exp_avg"].dtype == torch.float32


@pytest.mark.parametrize("kind", [AdamW, AdamWFp8])
def test_captured_steps_count_on(kind):
    g = gen(10)
    shapes = [(130,), (64, 64), (3, 4096)]
    values = [torch.randn(s, generator=g).bfloat16() for s in shapes]
    grads = [[torch.randn(s, generator=g).bfloat16().cuda() for s in shapes] for _ in range(6)]
    eager, kept = [leaf(v.clone()) for v in values], [leaf(v.clone()) for v in values]
    a, b = kind(eager, **ARGS), kind(kept, **ARGS)
    for p, q, d in zip(eager, kept, grads[0]):
        p.grad, q.grad = d.clone(), d.clone()
    a.step()
    b.step()  # makes the state
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for p, q in zip(eager, kept):
        assert torch.equal(p, q)  # capturing did nothing
    for ds in grads[1:]:
        for p, q, d in zip(eager, kept, ds):
            p.grad.copy_(d)
            q.grad.copy_(d)
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, kept):
            assert torch.equal(p, q)
            assert a.state[p]["step"].item() == b.state[q]["step"].item()
            for x, y in zip(held(a.state[p]), held(b.state[q])):
                assert torch.equal(x, y)


def test_two_streams_at_once():
    g = gen(11)
    values = [torch.randn(300000, generator=g) for _ in range(2)]
    grads = [torch.randn(300000, generator=g).cuda() for _ in range(2)]
    want = []
    for v, d in zip(values, grads):
        p = leaf(v.clone())
        p.grad = d
        opt = AdamW([p], **ARGS)
        for _ in range(6):
            opt.step()
        want.append(p.detach())
    params = [leaf(v.clone()) for v in values]
    opts = [AdamW([p], **ARGS) for p in params]
    for p, d in zip(params, grads):
        p.grad = d
    streams = [torch.cuda.Stream() for _ in params]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for s, o in zip(streams, opts):
            with torch.cuda.stream(s):
                o.step()
    torch.cuda.synchronize()
    for p, w in zip(params, want):
        assert torch.equal(p, w)


def test_a_saved_parameter_that_was_stepped_is_found_changed():
    p = leaf(torch.ones(8))
    p.grad = torch.ones(8).cuda()
    y = (p * p).sum()
    AdamW([p], **ARGS).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_beside_muon_in_a_training_loop():
    """A small regression: Muon on the matrix, AdamW on the rest; both move their own."""
    g = gen(12)
    w, gain, bias = leaf(torch.randn(16, 32, generator=g)), leaf(torch.ones(32)), leaf(torch.zeros(16))
    x, y = torch.randn(50, 32, generator=g).cuda(), torch.randn(50, 16, generator=g).cuda()
    opts = [Muon([w], lr=0.01), AdamW([gain, bias], lr=0.01, wd=0.0)]
    for _ in range(3):
        loss = (((x * gain) @ w.T + bias - y) ** 2).mean()
        loss.backward()
        old = [t.detach().clone() for t in (w, gain, bias)]
        for o in opts:
            o.step()
            o.zero_grad()
        assert all(not torch.equal(a, b) and b.isfinite().all() for a, b in zip(old, (w, gain, bias)))


def test_outer_compile_gives_the_same_bits():
    g = gen(13)
    values = [torch.randn(s, generator=g) for s in ((64, 64), (7,))]
    grads = [torch.randn(v.shape, generator=g).cuda() for v in values]
    both = []
    for compiled in (False, True):
        params = [leaf(v.clone()) for v in values]
        opt = AdamW(params, **ARGS)
        for p, d in zip(params, grads):
            p.grad = d
        opt.step()
        step = torch.compile(opt.step, backend="aot_eager") if compiled else opt.step
        step()
        step()
        both.append([p.detach() for p in params] + [opt.state[p]["exp_avg"] for p in params])
    for a, b in zip(*both):
        assert torch.equal(a, b)


def test_values_behind_offsets_past_32_bits():
    """One tensor of 2^31 + 2^20 values."""
    n = 2**31 + 2**20
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda").requires_grad_()
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = gen(14)
    ends = torch.tensor([0, 5, 2**31 - 1, 2**31, 2**31 + 777, n - 1])
    d = torch.randn(6, generator=g).bfloat16()
    for kind in (AdamW, AdamWFp8):
        with torch.no_grad():
            p.zero_()
            p[ends.cuda()] = 1.0
            p.grad[ends.cuda()] = d.cuda()
        opt = kind([p], **ARGS)
        opt.step()
        want, *_ = ref.adamw(torch.ones(6), d, torch.zeros(6), torch.zeros(6), 1, **ARGS)
        got = p.detach()[ends.cuda()].double().cpu()
        assert ((got - want).abs() <= 2.0**-8 * want.abs() * (1 + 2.0**-10)).all()
        assert int((p != 0).sum()) == 6
        del opt
