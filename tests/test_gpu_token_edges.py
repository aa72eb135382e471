"""The token operators at their edges: axes of no tokens, the autograd contract, losses that nearly vanish, values that are
not finite, long axes of the forms that run on warp-level instructions, and vocabularies in several pieces.

``_check`` and its bounds are those of test_gpu_token_ops.py."""

import torch

import pytest
from test_gpu_token_ops import BF16, F32, FP32, U, _check, _gen, _inputs, _loss_ref, _ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


# ------------------------------------------------------------------------------------------ no tokens


def _leave_nan(*shape):
    """Freed blocks of NaN of this size: what the operator's next allocations are likely to get."""
    held = [torch.full(shape, float("nan"), device="cuda") for _ in range(4)]
    del held


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (33, 80), (16, 33), (48, 100), (1, 40), (65, 64), (128, 128)])
def test_no_tokens_leave_the_state(ews, dtype, dk, dv):
    """T = 0: the state is the initial one (or zero), its gradient the state's own (which passes through 1 / scale and
    scale: three roundings)."""
    g = _gen(dk * dv)
    q, k, v = (torch.zeros((2, 0, h, d), dtype=dtype, device="cuda") for h, d in ((4, dk), (2, dk), (2, dv)))
    rate = torch.tensor([0.5, 0.1, 0.02, 3.0], device="cuda")
    s0 = torch.randn((2, 4, dk, dv), device="cuda", generator=g).requires_grad_()
    ds = torch.randn((2, 4, dk, dv), device="cuda", generator=g)
    _leave_nan(2, 4, dk, dv)
    out, end = ews.decayed_attention(q, k, v, rate, initial_state=s0, return_state=True)
    assert out.shape == (2, 0, 4, dv) and torch.equal(end, s0)
    _leave_nan(2, 4, dk, dv)
    (d0,) = torch.autograd.grad(end, (s0,), ds)
    assert ((d0 - ds).abs() <= 2.0**-22 * ds.abs()).all()
    _leave_nan(2, 4, dk, dv)
    assert (ews.decayed_attention(q, k, v, rate, return_state=True)[1] == 0).all()


# ------------------------------------------------------------------------------------------ the autograd contract


def test_a_step_on_a_state_that_a_backward_needs_is_seen(ews):
    """The step overwrites its states: a backward that saved them raises, as after any operation in place."""
    q, k, v, rate, s0, _ = _inputs(FP32, 2, 5, 2, 2, 16, 16)
    leaf = q.clone().requires_grad_()
    pool = s0.clone()
    out = ews.decayed_attention(leaf, k, v, rate, initial_state=pool)
    with torch.no_grad():
        ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, pool)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with torch.inference_mode():  # tensors without a version
        ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, s0.clone())


def test_tangents_are_refused(ews):
    """No forward-mode derivative is built: a dual tensor raises instead of losing its tangent."""
    import torch.autograd.forward_ad as fw

    q, k, v, rate, s0, _ = _inputs(FP32, 2, 5, 2, 2, 16, 16)
    ids = torch.tensor([0, 1], device="cuda")
    h = torch.randn((2, 16), device="cuda")
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
        calls = [lambda: ews.decayed_attention(dual(q), k, v, rate),
                 lambda: ews.decayed_attention(q, k, v, dual(rate)),
                 lambda: ews.decayed_attention(q, k, v, rate, initial_state=dual(s0)),
                 lambda: ews.decayed_attention_step(q[:, 0], k[:, 0], dual(v[:, 0]), rate, s0),
                 lambda: ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, dual(s0)),
                 lambda: ews.token_embedding(ids, dual(h)),
                 lambda: ews.vocab_loss(dual(h), h, ids),
                 lambda: ews.vocab_loss(h, dual(h), ids)]
        was = s0.clone()
        for call in calls:
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError):
                    call()
        assert torch.equal(s0, was)
        assert ews.token_embedding(ids, h).shape == (2, 16)  # and others still run there


def test_second_derivatives_are_refused(ews):
    """A gradient taken with create_graph is usable as a number; differentiating it again raises instead of leaving the
    operator's part out, whether or not the cotangent itself depends on anything."""
    q, k, v, rate, s0, _ = _inputs(FP32, 2, 5, 2, 2, 16, 16)
    ids = torch.tensor([0, 1], device="cuda")
    h, w = (torch.randn((2, 16), device="cuda") for _ in range(2))
    leaf = lambda x: x.clone().requires_grad_()  # noqa: E731
    cases = [(lambda a, b: ews.decayed_attention(a, k, v, rate, initial_state=b), (q, s0)),
             (lambda a, b: ews.token_embedding(ids, a) * b, (w, h)),
             (lambda a, b: ews.vocab_loss(a, b, ids), (h, w))]
    for f, args in cases:
        for power in (1, 2):  # a constant cotangent, and one that depends on the result
            a, b = (leaf(x) for x in args)
            plain = torch.autograd.grad((f(a, b) ** power).sum(), (a, b))
            grads = torch.autograd.grad((f(a, b) ** power).sum(), (a, b), create_graph=True)
            for x, y in zip(plain, grads):
                assert torch.equal(x, y.detach())
            penalty = sum((x**2).sum() for x in grads) + (a**2).sum()
            with pytest.raises(RuntimeError, match="second derivative"):
                penalty.backward()


# ------------------------------------------------------------------------------------------ losses


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("offset", [0.0, 1000.0])
def test_confident_rows_keep_their_small_losses(ews, dtype, offset):
    """Logits that are exact (each row picks one column of the weight), the target's 20 to 60 above the others. The
    exponentials' sum is 1 and a remainder r, of which each of the at most 32 additions on the way rounds by 2^-24 or less,
    and never by more than what it adds; the exponentials have 2^-20 of their own."""
    D, V = 64, 700
    g = _gen(17)
    w = torch.randn((V, D), device="cuda", generator=g) + offset
    t = torch.randperm(V, device="cuda", generator=g)[:D]
    w[t, torch.arange(D, device="cuda")] += torch.linspace(20.0, 60.0, D, device="cuda")
    w = w.to(dtype)
    h = torch.eye(D, device="cuda").to(dtype)
    loss = ews.vocab_loss(h, w, t)
    z = w.t().double()
    others = torch.exp(z - z.gather(1, t[:, None])).scatter(1, t[:, None], 0.0)
    want = torch.log1p(others.sum(1))
    bound = torch.minimum(torch.full_like(want, 32 * 2.0**-24), 1.01 * want) + 2.0**-20 * want
    assert (loss >= 0).all()
    assert ((loss.double() - want).abs() <= bound).all(), float(((loss.double() - want).abs() / bound).max())


def test_losses_do_not_lose_the_logits_offset(ews):
    """Logits near 1,000 and exact: the differences that make the loss are exact too, so its error is that of the
    exponentials (2^-20) and of 40 additions (2^-24 each), not a rounding of 1,000 (2^-15)."""
    D, V = 64, 700
    g = _gen(19)
    w = 1000.0 + torch.randn((V, D), device="cuda", generator=g)
    t = torch.randint(0, V, (D,), device="cuda", generator=g)
    loss = ews.vocab_loss(torch.eye(D, device="cuda"), w, t)
    want = torch.nn.functional.cross_entropy(w.t().double(), t, reduction="none")
    assert ((loss.double() - want).abs() <= 2.0**-20 + 40 * 2.0**-24 + 2.0**-22 * want).all()


@pytest.mark.parametrize("shape", [(6,), (2, 3)])
def test_losses_may_be_weighted_in_place(ews, shape):
    g = _gen(23)
    h, w = torch.randn((*shape, 16), device="cuda", generator=g), torch.randn((30, 16), device="cuda", generator=g)
    t = torch.randint(0, 30, shape, device="cuda", generator=g)
    weight = torch.rand(shape, device="cuda", generator=g)
    hl, wl = h.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad((ews.vocab_loss(hl, wl, t) * weight).sum(), (hl, wl))
    loss = ews.vocab_loss(hl, wl, t)
    loss *= weight
    for a, b in zip(torch.autograd.grad(loss.sum(), (hl, wl)), want):
        assert torch.equal(a, b)
    with torch.no_grad():
        loss = ews.vocab_loss(h, w, t)
    factor = weight.clone().requires_grad_()
    loss *= factor  # a result without a gradient, weighted by something that has one
    loss.sum().backward()
    assert torch.equal(factor.grad, ews.vocab_loss(h, w, t))


# ------------------------------------------------------------------------------------------ values that are not finite


@pytest.mark.parametrize("dtype,dk,dv", [(BF16, 64, 64), (BF16, 128, 48), (BF16, 37, 40), (FP32, 64, 64), (FP32, 40, 72), (FP32, 100, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_key_that_is_not_finite_reaches_no_earlier_token(ews, dtype, dk, dv, value):
    """Forward: a key enters from its own token on. Backward: a token's cotangent enters dk up to its own token."""
    T, at = 300, 149  # inside a block of 32 of any chunk
    q, k, v, rate, s0, g = _inputs(dtype, 2, T, 2, 1, dk, dv, seed=41)
    do = torch.randn((2, T, 2, dv), device="cuda", generator=g).to(dtype)

    def run(k, do):
        leaf = k.clone().requires_grad_()
        out = ews.decayed_attention(q, leaf, v, rate, initial_state=s0)
        return out.detach(), torch.autograd.grad(out, (leaf,), do)[0]

    clean, dk_clean = run(k, do)
    bad = k.clone()
    bad[:, at] = value
    out = run(bad, do)[0]
    assert torch.equal(out[:, :at], clean[:, :at]) and not torch.isfinite(out[:, at]).all(-1).any()
    bad = do.clone()
    bad[:, at] = value
    grad = run(k, bad)[1]
    assert torch.equal(grad[:, at + 1 :], dk_clean[:, at + 1 :]) and not torch.isfinite(grad[:, at]).all(-1).any()


def test_rates_that_are_parameters_serve_without_gradients(ews):
    """No gradient is built for the rates, so they are refused where one would be lost, and only there."""
    q, k, v, rate, s0, _ = _inputs(FP32, 2, 5, 2, 2, 16, 16)
    p = torch.nn.Parameter(rate.clone())
    want = ews.decayed_attention(q, k, v, rate)
    step = ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, s0.clone())
    with torch.no_grad():
        assert torch.equal(ews.decayed_attention(q, k, v, p), want)
        assert torch.equal(ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], p, s0.clone()), step)
    for call in (lambda: ews.decayed_attention(q, k, v, p), lambda: ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], p, s0)):
        with pytest.raises(NotImplementedError):
            call()


# ------------------------------------------------------------------------------------------ long axes, many pieces


@pytest.mark.parametrize("dtype,B,T,H,Hk,dk,dv,lengths,state", [
    (BF16, 1, 600, 1, 1, 37, 29, None, True),  # two segments of five chunks
    (BF16, 2, 1100, 2, 1, 37, 101, [1100, 333], True),  # four, and a length that ends inside the second
    (BF16, 2, 777, 2, 2, 70, 12, [0, 640], True),  # no token, and a length at a segment's edge
    (BF16, 1, 901, 2, 2, 101, 90, None, False),
    (FP32, 1, 700, 2, 1, 100, 40, None, True),
    (FP32, 2, 1100, 1, 1, 128, 66, [321, 1100], True),
    (FP32, 1, 520, 2, 2, 72, 128, None, False),
])
def test_split_axes_of_the_warp_level_form(ews, dtype, B, T, H, Hk, dk, dv, lengths, state):
    """Odd bfloat16 widths and wide float32 heads over axes that are split: the segments' states, their join in both
    directions, and what starts and ends in them."""
    from test_gpu_token_ops import test_decayed_attention_and_gradients as whole

    whole(ews, dtype, B, T, H, Hk, dk, dv, lengths, state)


def _loss_case(ews, h, w, t, dl):
    """Loss and gradients within the bounds of test_gpu_token_ops.test_vocab_loss_and_gradients."""
    dtype = w.dtype
    hl, wl = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ews.vocab_loss(hl, wl, t)
    dh, dw = torch.autograd.grad(loss, (hl, wl), dl)
    want, wh, ww, ab, p, gg, hz = _loss_ref(h, w, t, dl)
    worst = F32 * ab.amax(1)
    assert ((loss.double() - want).abs() <= 2 * worst + 1e-6 * (want.abs() + 20)).all()
    eg = p * (2 * worst + 2e-6)[:, None] + (U if dtype == BF16 else 2.0**-21) * gg.abs()
    for got, exact, err, form in ((dh, wh, eg @ w.double().abs(), gg.abs() @ w.double().abs()), (dw, ww, eg.T @ hz.abs(), gg.abs().T @ hz.abs())):
        bound = 1.05 * err + F32 * form + (U if dtype == BF16 else 2.0**-23) * exact.abs() + 1e-30
        assert ((got.double() - exact).abs() <= bound).all(), float(((got.double() - exact).abs() / bound).max())


def test_float32_gradients_over_several_pieces(ews):
    """9,000 rows of three planes by 5,003 entries are more than one piece of the softmax gradient."""
    n, V, D = 9000, 5003, 24
    g = _gen(71)
    h = torch.randn((n, D), device="cuda", generator=g)
    w = torch.randn((V, D), device="cuda", generator=g) * 2 / D**0.5
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    t[::7] = -100
    _loss_case(ews, h, w, t, torch.rand((n,), device="cuda", generator=g) + 0.1)


@pytest.mark.parametrize("dtype,V,D,planes", [(FP32, 90001, 509, 3), (BF16, 270001, 509, 1)])
def test_packed_weights_over_several_pieces(ews, dtype, V, D, planes):
    """A weight that is packed (512 columns after padding) in two pieces: targets on both sides of the pieces' edge."""
    assert 2**27 < V * 512 * planes < 2**28
    edge = ((V + 1) // 2 + 255) // 256 * 256
    g = _gen(73)
    t = torch.tensor([0, edge - 1, edge, edge + 1, V - 1, 256, -100, V // 3], device="cuda")
    h = torch.randn((len(t), D), device="cuda", generator=g).to(dtype)
    w = (torch.randn((V, D), device="cuda", generator=g) / D**0.5).to(dtype)
    _loss_case(ews, h, w, t, torch.rand((len(t),), device="cuda", generator=g) + 0.1)


def test_backwards_in_a_cuda_graph(ews):
    """Forward and backward captured once and replayed on new contents."""
    q, k, v, rate, s0, g = _inputs(BF16, 2, 300, 2, 1, 64, 64, seed=83)
    q, k, v, s0 = (x.requires_grad_() for x in (q, k, v, s0))
    h, w = (torch.randn((n, 64), device="cuda", generator=g).to(BF16).requires_grad_() for n in (400, 500))
    t = torch.randint(0, 500, (400,), device="cuda", generator=g)
    do = torch.randn((2, 300, 2, 64), device="cuda", generator=g).to(BF16)
    dl = torch.rand((400,), device="cuda", generator=g)

    def run():
        out, end = ews.decayed_attention(q, k, v, rate, initial_state=s0, return_state=True)
        x = ews.token_embedding(t, w, scale=2.0)
        return [*torch.autograd.grad((out, end), (q, k, v, s0), (do, s0.detach())), *torch.autograd.grad(x, (w,), h.detach()),
                *torch.autograd.grad(ews.vocab_loss(h, w, t), (h, w), dl)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.no_grad():
        for x in (q, k, v, s0, h, w, do):
            x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        dl.copy_(torch.rand(dl.shape, device="cuda", generator=g))
        t.copy_(torch.randint(0, 500, (400,), device="cuda", generator=g))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, run()):
        assert torch.equal(a, b)
