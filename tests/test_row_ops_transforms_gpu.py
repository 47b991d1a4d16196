"""The row operators under torch's transforms of a program: forward mode, torch.func, tracing by a
dispatch mode, saved-tensor hooks, captured graphs with a backward pass, an outer compile; and
gradients that meet what was left out. Tolerances are those of test_row_ops_gpu.py."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

from muonium_amd.kernels import policy_loss, qk_norm_rope, route, token_logprobs
from oracle import row_ops_ref as ref
from test_row_ops_gpu import E, TYPES, _all_calls, check, gen, leaf, policy_case

pytestmark = pytest.mark.gpu


def policy_args(n, v, dtype, seed=3):
    """Logits on the device and the other arguments of a policy loss with a reference."""
    x, tokens, old, adv, w, r, _, _ = policy_case(n, v, dtype, seed, True, 1.0)
    return x.cuda(), [t.cuda() for t in (tokens, old, adv, w, r)]


# ---- forward mode -------------------------------------------------------------------------


def _forward_mode_calls():
    """(name, a call on one input, that input): every floating input of every operator."""
    q, k = torch.randn(2, 3, 4, 16, device="cuda"), torch.randn(2, 3, 2, 16, device="cuda")
    w, cos = torch.ones(16, device="cuda"), torch.rand(9, 8, device="cuda")
    z = torch.randn(6, 8, device="cuda")
    tok, f = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.rand(6, device="cuda")
    return [
        ("q", lambda t: qk_norm_rope(t, k, w, w, cos, cos)[0], q),
        ("k", lambda t: qk_norm_rope(q, t, w, w, cos, cos)[1], k),
        ("q_weight", lambda t: qk_norm_rope(q, k, t, w, cos, cos)[0], w),
        ("k_weight", lambda t: qk_norm_rope(q, k, None, t, cos, cos)[1], w),
        ("cos", lambda t: qk_norm_rope(q, k, w, w, t, cos)[0], cos),
        ("sin", lambda t: qk_norm_rope(q, k, w, w, cos, t)[0], cos),
        ("route", lambda t: route(t, 2).gates, z),
        ("logprobs", lambda t: token_logprobs(t, tok), z),
        ("policy", lambda t: policy_loss(t, tok, f, f, f).loss, z),
        ("old", lambda t: policy_loss(z, tok, t, f, f).loss, f),
        ("advantages", lambda t: policy_loss(z, tok, f, t, f).loss, f),
        ("weights", lambda t: policy_loss(z, tok, f, f, t).loss, f),
        ("ref", lambda t: policy_loss(z, tok, f, f, f, t, kl_coef=0.1).loss, f),
    ]


@pytest.mark.parametrize("case", range(13))
def test_forward_mode_raises(case):
    """There is no forward-mode derivative: a tangent on any input is refused, never dropped."""
    name, call, x = _forward_mode_calls()[case]
    tangent = torch.ones_like(x)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(call, (x,), (tangent,))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jacfwd(call)(x)
    with fwad.dual_level():
        dual = fwad.make_dual(x, tangent)
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
        call(x)  # without a tangent, as ever
    call(x)


# ---- torch.func, tracing by a dispatch mode ----------------------------------------------------


def test_reverse_transforms_of_torch_func_are_refused():
    """torch has no torch.func transforms over C++ autograd functions: they raise."""
    for _, call, x in _forward_mode_calls()[6:9]:
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(x)


@pytest.mark.parametrize("dtype", TYPES)
def test_traced_policy_gradient_keeps_its_scale(dtype):
    """A trace over plain tensors, by a dispatch mode, computes what eager does, whatever the loss
    gradient, also on other inputs than those it was recorded with; as does a trace of the
    backward pass alone."""
    x, args = policy_args(6, 500, dtype)

    def grad_of(t):
        t = t.detach().requires_grad_()
        return torch.autograd.grad((3 * policy_loss(t, *args, kl_coef=0.1).loss,), (t,))[0]

    graph = make_fx(grad_of)(x)
    for t in (x, x.flip(1).contiguous(), x):
        torch.testing.assert_close(graph(t), grad_of(t), rtol=2.0**-7, atol=1e-6)
    a = x.clone().requires_grad_()
    loss = policy_loss(a, *args, kl_coef=0.1).loss

    def back(g):
        return torch.autograd.grad((loss,), (a,), (g,), retain_graph=True)[0]

    graph = make_fx(back)(torch.tensor(3.0, device="cuda"))
    for scale in (3.0, 1.0, 0.5, 3.0):
        got = graph(torch.tensor(scale, device="cuda"))
        torch.testing.assert_close(got, grad_of(x) * (scale / 3), rtol=2.0**-6, atol=1e-6)


def test_rescale_is_a_well_behaved_torch_operator():
    """It says what it changes, and does so in eager and traced programs."""
    ops = torch.ops.muonium_amd
    x, args = policy_args(6, 300, torch.bfloat16)
    _, _, rows, d = ops.policy_loss(x, *args, 0.2, 0.2, 0.1, 1.0, True, True)
    scale = torch.tensor(3.0, device="cuda")
    torch.library.opcheck(ops.policy_loss_rescale_.default, (d.clone(), scale, x, args[0], rows, 1.0))
    want = ops.policy_loss_backward(scale, x, args[0], rows, 1.0)
    got = d.clone()
    ops.policy_loss_rescale_(got, scale, x, args[0], rows, 1.0)
    assert torch.equal(got, want) and not torch.equal(got, d)
    ops.policy_loss_rescale_(d, torch.ones((), device="cuda"), x, args[0], rows, 1.0)
    assert torch.equal(d, ops.policy_loss_backward(scale / 3, x, args[0], rows, 1.0))
    for bad in (d[:5], d.float(), d.t().contiguous().t(), d.cpu()):
        with pytest.raises((RuntimeError, TypeError)):
            ops.policy_loss_rescale_(bad, scale, x, args[0], rows, 1.0)


# ---- the registered operators keep their schemas -------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_registered_results_are_what_was_asked_for(dtype):
    """keep and one_pass decide the shapes with and without a gradient, and a gradient that was asked
    for as a result stays as it is when the backward pass runs."""
    ops = torch.ops.muonium_amd
    x, args = policy_args(6, 300, dtype)
    rest = (0.2, 0.2, 0.1, 1.0)
    for keep in (False, True):
        for one_pass in (False, True):
            a = x.clone().requires_grad_()
            loss, logp, rows, d = ops.policy_loss(a, *args, *rest, keep, one_pass)
            plain = ops.policy_loss(x, *args, *rest, keep, one_pass)
            assert rows.shape == plain[2].shape == (4 if keep else 1, 6)
            assert d.shape == plain[3].shape == (x.shape if one_pass else (0,))
            held = d.clone()
            g, = torch.autograd.grad((loss,), (a,), (torch.tensor(3.0, device="cuda"),))
            assert torch.equal(d, held) and torch.equal(d, plain[3])
            one, = torch.autograd.grad((ops.policy_loss(a, *args, *rest, True, False)[0],), (a,))
            torch.testing.assert_close(g, 3 * one, rtol=2.0**-6, atol=1e-6)
            if one_pass:
                torch.testing.assert_close(d, one, rtol=2.0**-7, atol=1e-6)
        b = x.clone().requires_grad_()
        for t in (x, b):
            assert ops.token_logprobs(t, args[0], 1.0, keep)[1].shape == (12 if keep else 0,)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("one_pass", [False, True])
def test_policy_operators_are_well_behaved_torch_operators(keep, one_pass):
    ops = torch.ops.muonium_amd
    z = leaf(torch.randn(20, 16))
    tokens, f = torch.randint(0, 16, (20,), device="cuda"), torch.rand(20, device="cuda")
    args = (z, tokens, f, f, f, None, 0.2, 0.2, 0.1, 1.0)
    torch.library.opcheck(ops.policy_loss.default, (*args, keep, one_pass))
    torch.library.opcheck(ops.token_logprobs.default, (z, tokens, 1.0, keep))


# ---- saved-tensor hooks --------------------------------------------------------------------


def test_saved_tensor_hooks_see_the_gradient_of_the_forward_pass():
    """What the forward pass keeps of the logits' size is offered to saved-tensor hooks, which may
    move it: to the host and back, or away until a checkpoint is computed again."""
    x, args = policy_args(64, 32000, torch.bfloat16)
    x.requires_grad_()
    scale = torch.tensor(0.3, device="cuda")

    def loss():
        return policy_loss(x, *args, kl_coef=0.1).loss

    want, = torch.autograd.grad((loss(),), (x,), (scale,))
    seen = []

    def pack(t):
        seen.append(t.shape)
        return t.to("cpu")

    size = x.numel() * x.element_size()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to("cuda")):
        before = torch.cuda.memory_allocated()
        out = loss()
        assert torch.cuda.memory_allocated() - before < size
    assert seen.count(x.shape) == 2  # the logits and the gradient made of them
    assert torch.equal(torch.autograd.grad((out,), (x,), (scale,))[0], want)
    before = torch.cuda.memory_allocated()
    out = checkpoint(loss, use_reentrant=False)
    assert torch.cuda.memory_allocated() - before < size
    assert torch.equal(torch.autograd.grad((out,), (x,), (scale,))[0], want)
    # one that keeps the operator's results, by a dispatch mode
    op = torch.ops.muonium_amd.policy_loss.default

    def keep(ctx, func, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if func == op else CheckpointPolicy.PREFER_RECOMPUTE

    out = checkpoint(loss, use_reentrant=False,
                     context_fn=lambda: create_selective_checkpoint_contexts(keep))
    got, = torch.autograd.grad((out,), (x,), (scale,))
    torch.testing.assert_close(got, want, rtol=2.0**-7, atol=1e-9)


def test_a_handed_over_gradient_is_its_takers():
    """What becomes of the first gradient of a graph changes no later one."""
    x, args = policy_args(6, 1500, torch.bfloat16)
    x.requires_grad_()
    loss = policy_loss(x, *args, kl_coef=0.1).loss
    scale = torch.tensor(3.0, device="cuda")
    first, = torch.autograd.grad((loss,), (x,), (scale,), retain_graph=True)
    want = first.clone()
    first.zero_()
    assert torch.equal(torch.autograd.grad((loss,), (x,), (scale,), retain_graph=True)[0], want)
    loss.backward(scale)
    loss = policy_loss(x, *args, kl_coef=0.1).loss
    loss.backward(scale, retain_graph=True)
    loss.backward(scale)
    torch.testing.assert_close(x.grad, 3 * want, rtol=2.0**-6, atol=1e-9)
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward(scale)


# ---- the policy gradient under any loss gradient ------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [70, 1500, 50257])
def test_policy_gradient_is_rounded_once(dtype, v):
    """One rounding whatever the loss gradient, and however many backward passes a graph serves."""
    x, tokens, old, adv, w, r, logp, p = policy_case(6, v, dtype, 3, True, 0.7)
    args = [t.cuda() for t in (tokens, old, adv, w, r)]
    _, slope, _, sizes = ref.policy(logp, old, adv, w, r, 0.2, 0.2, 0.1)
    want, ds = ref.logprobs_grad(p, tokens, slope, 0.7)
    _, room = ref.logprobs_grad(p, tokens, sizes, 0.7)
    xl = leaf(x)
    lift = 1024.0 if dtype == torch.float16 else 1.0
    for scales in ((1 / 3,), (3.0, 0.7), (1.0, 0.1), (0.0, 1.3), (-2.6, 1.0)):
        out = policy_loss(xl, *args, kl_coef=0.1, temperature=0.7)
        for scale in scales:
            s = torch.tensor(scale * lift, device="cuda")
            d, = torch.autograd.grad((out.loss,), (xl,), (s,), retain_graph=True)
            # the slope's product with the loss gradient is one more rounding in fp32
            check(d, want * s.item(), (ds + 2 * room) * abs(s.item()), 257, dtype, scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_left_out_rows_stay_out_of_a_gradient_that_is_not_finite(dtype):
    """A loss gradient of infinity or NaN (a loss scale that overflowed) makes no gradient in rows of
    weight 0 and of negative tokens."""
    x, (tokens, old, adv, w, r) = policy_args(9, 700, dtype, 4)
    tokens[2] = -100
    on = (w != 0) & (tokens >= 0)
    assert on.any() and not on.all()
    for scale in (math.inf, math.nan):
        a = x.clone().requires_grad_()
        out = policy_loss(a, tokens, old, adv, w, r, kl_coef=0.1)
        for _ in range(2):  # the gradient of the forward pass, then one made from the logits
            d, = torch.autograd.grad((out.loss,), (a,), (torch.tensor(scale, device="cuda"),),
                                     retain_graph=True)
            assert torch.count_nonzero(d[~on]) == 0
            assert not d[on].isfinite().all(1).any()


# ---- routing: gradients of empty slots -----------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("experts", [5, 12, 200])
def test_route_empty_slots_take_no_gradient(dtype, normalize, experts):
    """The gradient of a gate that is 0 because its slot is empty, or its token masked, reaches
    nothing, whatever it is: the entropy of the gates has a slope of infinity there."""
    z = torch.randn(9, experts, generator=gen(1)).to(dtype)
    z[0] = -math.inf
    z[1, 2:] = -math.inf
    z[2, 1:] = -math.inf
    mask = torch.ones(9, dtype=torch.bool)
    mask[5] = mask[6] = False
    want = ref.route(z, 4, mask, normalize)
    empty = want["experts"] < 0
    assert empty.sum() == 4 + 2 + 3 + 8
    dg = torch.randn(9, 4, generator=gen(2))
    scale = 256.0 if dtype == torch.float16 else 1.0
    d, sd = ref.route_grad(want, dg * scale, torch.tensor(scale), torch.tensor(scale))
    one = torch.tensor(scale, device="cuda")
    for bad in (math.inf, -math.inf, math.nan):
        x = leaf(z)
        got = route(x, 4, token_mask=mask.cuda(), normalize=normalize)
        up = torch.where(empty, bad, dg * scale).cuda()
        dz, = torch.autograd.grad((got.gates, got.balance_loss, got.z_loss), (x,), (up, one, one))
        check(dz, d, sd, 320, dtype, bad)
    x = leaf(z)
    torch.special.entr(route(x, 4, token_mask=mask.cuda(), normalize=normalize).gates).sum().backward()
    assert x.grad.isfinite().all()


# ---- the KL term of neighbouring policies -----------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [64, 5000, 170001])
def test_policy_kl_term_of_neighbouring_policies(dtype, v):
    """exp(d) - d - 1 and its slope follow their own size, not that of exp(d), where policy and
    reference nearly agree: off by what logp is off by (256 2^-24, times the term's slope, and its
    square) and by 16 roundings of the result; and the term is never negative."""
    n = 24
    x, tokens, old, _, _, _, logp, _ = policy_case(n, v, dtype, 5, False, 1.0)
    ahead = torch.logspace(-6, 0.8, n, dtype=torch.float64) * torch.tensor([1.0, -1.0]).repeat(n // 2)
    r = (logp + ahead).float()
    ahead = r.double() - logp
    em1 = torch.expm1(ahead)
    # d^2 / 2 + d^3 / 6 + ...: the difference itself would cancel in float64 too
    series = sum(ahead ** i / float(math.factorial(i)) for i in range(2, 30))
    term = torch.where(ahead.abs() < 1, series, em1 - ahead)
    off = 256 * E
    zero, one = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    a = x.cuda()
    loss, _, rows, _ = torch.ops.muonium_amd.policy_loss(
        a, tokens.cuda(), old.cuda(), zero, one, r.cuda(), 0.2, 0.2, 1.0, 1.0, True, False)
    terms, slopes = rows[0].double().cpu(), rows[1].double().cpu()
    assert (terms >= 0).all()
    room = em1.abs() * off + (em1 + 1) * off**2 + 16 * E * term
    assert ((terms - term).abs() <= room).all(), ((terms - term).abs() / room).max()
    assert ((slopes + em1).abs() <= (em1 + 1) * off + 16 * E * em1.abs()).all()
    got = policy_loss(a, tokens.cuda(), old.cuda(), zero, one, r.cuda(), kl_coef=1.0).loss
    assert abs(got.item() - term.sum().item()) <= (room + E * term).sum().item() + E * term.sum().item()
    # exactly the reference: nothing, or next to it
    same = token_logprobs(a, tokens.cuda())
    none = policy_loss(a, tokens.cuda(), old.cuda(), zero, one, same, kl_coef=1.0).loss
    assert 0 <= none.item() <= n * (off + E * same.abs().max().item())**2


def test_policy_kl_term_of_distant_policies():
    """The same where the reference thinks a token far less, or far more, likely."""
    n = 12
    x, tokens, old, _, _, _, logp, _ = policy_case(n, 300, torch.float32, 5, False, 1.0)
    ahead = torch.linspace(1.0, 60.0, n, dtype=torch.float64) * torch.tensor([1.0, -1.0]).repeat(n // 2)
    r = (logp + ahead).float()
    ahead = r.double() - logp
    e = torch.exp(ahead)
    zero, one = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    _, _, rows, _ = torch.ops.muonium_amd.policy_loss(
        x.cuda(), tokens.cuda(), old.cuda(), zero, one, r.cuda(), 0.2, 0.2, 1.0, 1.0, True, False)
    terms, slopes = rows[0].double().cpu(), rows[1].double().cpu()
    # logp's error and the argument's rounding move the exponential, then 16 roundings
    off = (256 + 2 * ahead.abs()) * E
    assert ((terms - (e - ahead - 1)).abs() <= (e - 1).abs() * off + 16 * E * (e + ahead.abs())).all()
    assert ((slopes + e - 1).abs() <= e * off + 16 * E * (e - 1).abs()).all()


# ---- rows past the grid's second dimension ------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_more_rows_than_a_grid_has(dtype):
    """65536 rows and more, left-out ones on both sides of the line: kernels that walk over rows do
    each of them once, in both directions."""
    n, v = 70000, 40
    x, tokens, old, adv, w, r, logp, p = policy_case(n, v, dtype, 6, True, 1.0)
    out = torch.tensor([3, 65533, 65534, 65535, 65536, 65537, 69999])
    tokens[out] = -100
    w[:] = 0.5 + torch.rand(n, generator=gen(7))
    w[out[::2]] = 0.0
    w[65530], w[65540] = 0.0, 0.0
    logp, p = ref.logprobs(x, tokens)
    xl = leaf(x)
    got = token_logprobs(xl, tokens.cuda())
    check(got, logp, torch.ones(n, dtype=torch.float64), 256, torch.float32, "logp")
    g = torch.randn(n, generator=gen(8))
    d, = torch.autograd.grad((got,), (xl,), (g.cuda(),))
    check(d, *ref.logprobs_grad(p, tokens, g), 256, dtype, "dlogits")
    # fp16 reads the logits again for the gradient, bf16 makes it in the forward pass
    on = (w != 0) & (tokens >= 0)
    w = torch.where(on, w, 0.0)
    loss, slope, size, sizes = ref.policy(logp, old, adv, w, r, 0.2, 0.2, 0.1)
    args = [t.cuda() for t in (tokens, old, adv, w, r)]
    for scale in (1.0, 3.0):
        res = policy_loss(xl, *args, kl_coef=0.1)
        # 70000 terms of both signs, each rounded to fp32 before the sum in double
        check(res.loss, loss, size, 2 * 256 + 1, torch.float32, "loss")
        check(res.logprobs, torch.where(on, logp, 0.0), torch.ones(n, dtype=torch.float64), 256, torch.float32)
        d, = torch.autograd.grad((res.loss,), (xl,), (torch.tensor(scale, device="cuda"),))
        want, ds = ref.logprobs_grad(p, tokens, slope)
        _, room = ref.logprobs_grad(p, tokens, sizes)
        check(d, want * scale, (ds + 2 * room) * scale, 257, dtype, "policy dlogits")
        assert torch.count_nonzero(d[(~on).cuda()]) == 0
    plain = policy_loss(x.cuda(), *args, kl_coef=0.1)
    check(plain.loss, loss, size, 2 * 256 + 1, torch.float32, "loss without gradient")


# ---- captured graphs with a backward pass ------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_and_backward_in_a_captured_graph(dtype):
    """Every replay gives the eager results and gradients of its inputs, for any loss gradient."""
    g = gen(9)
    q = torch.randn(3, 9, 8, 64, generator=g).to(dtype).cuda().requires_grad_()
    w = torch.ones(64, device="cuda").requires_grad_()
    z = torch.randn(3000, 64, generator=g).to(dtype).cuda().requires_grad_()
    x, args = policy_args(12, 9000, dtype, 2)
    x.requires_grad_()
    ups = [torch.randn(3, 9, 8, 64, generator=g).to(dtype).cuda(), torch.randn(3000, 6, generator=g).cuda(),
           torch.tensor(0.3, device="cuda"), torch.tensor(0.01, device="cuda"),
           torch.randn(12, generator=g).cuda(), torch.tensor(1 / 3, device="cuda")]

    def run():
        a, b = qk_norm_rope(q, q, w, w)
        rt = route(z, 6)
        lp = token_logprobs(x, args[0])
        out = policy_loss(x, *args, kl_coef=0.1)
        grads = [*torch.autograd.grad((a, b), (q, w), (ups[0], ups[0])),
                 *torch.autograd.grad((rt.gates, rt.balance_loss, rt.z_loss), (z,), ups[1:4]),
                 *torch.autograd.grad((lp,), (x,), (ups[4],)),
                 *torch.autograd.grad((out.loss,), (x,), (ups[5],))]
        return [t.detach() for t in (a, b, *rt, lp, *out)] + grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i, scale in enumerate((1 / 3, 1.0, 0.0, 2.5, 1.0)):
        with torch.no_grad():
            for t in (q, z, x, *ups[:2]):
                t.copy_(torch.randn(t.shape, generator=g))
            ups[5].fill_(scale)
        graph.replay()
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(outs, run())):
            assert torch.equal(a, b), (i, j)


@pytest.mark.parametrize("dtype", TYPES)
def test_backward_alone_in_a_captured_graph(dtype):
    """A graph of the backward pass of an eager forward pass gives the gradient of each replay's loss
    gradient. (The engine runs a node on the stream of its forward pass: both are on the one that
    is captured.)"""
    x, args = policy_args(12, 3000, dtype, 2)
    x.requires_grad_()
    up = torch.tensor(3.0, device="cuda")

    def loss():
        return policy_loss(x, *args, kl_coef=0.1).loss

    def back(value):
        return torch.autograd.grad((value,), (x,), (up,), retain_graph=True)[0]

    want = back(loss()).float() / 3
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        back(loss())
        out = loss()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = back(out)
    for scale in (3.0, 3.0, 1.0, 0.5, 3.0):
        up.fill_(scale)
        graph.replay()
        torch.cuda.synchronize()
        torch.testing.assert_close(got.float(), want * scale, rtol=2.0**-6, atol=1e-6, msg=str(scale))


# ---- an outer compile ------------------------------------------------------------------------


def test_outer_compile_gives_the_same_bits():
    """Under an outer compile the same kernels run: the same bits, but for the policy loss, whose
    gradient takes two readings there, and the sums of the logits' gradient with it."""
    run = _all_calls(1)
    want = run()
    torch._dynamo.reset()
    got = torch.compile(run, backend="aot_eager")()
    torch._dynamo.reset()
    names = ["q_out", "k_out", "gates", "experts", "counts", "logprobs", "loss", "q", "k", "w", "z", "x"]
    assert len(got) == len(want) == len(names)
    for name, a, b in zip(names, got, want):
        if name in ("loss", "x"):
            tol = 2.0**-7 if a.dtype == torch.bfloat16 else 1e-5
            torch.testing.assert_close(a, b, rtol=tol, atol=1e-6, msg=lambda m: f"{name}: {m}")
        else:
            assert torch.equal(a, b), name
