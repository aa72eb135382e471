"""The token operators against plain float64 implementations: decayed attention (chunks, gradients, single-token step),
token embedding with its gradient, vocabulary loss with its gradients.

Tolerances are bounds, element by element, from the arithmetic: u = 2^-8 is bfloat16's unit roundoff. Where an operand
is rounded to bfloat16 on the way (the decayed scores, the state as an operand, the weighted softmax), the error of a
sum is at most u times the same sum over absolute values, which the float64 reference evaluates on absolute inputs;
the rounded result adds u |result|. float32 results, and the float32 parts of the others, get 2e-5 times the sum over
absolute values: products exact to 2^-21 and chains of at most some hundred truncated additions of 2^-23 each.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-8
F32 = 2e-5
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(got, want, absform, rounded, dtype, what):
    """|got - want| <= u-type bounds (see the module's docstring); rounded: some operand was rounded to bf16."""
    got, want, absform = got.double(), want.double(), absform.double()
    bound = F32 * absform + 1e-30
    if dtype == BF16:
        bound = bound + U * want.abs() + (1.05 * U * absform if rounded else 0.0)
    else:
        bound = bound + 2.0**-23 * want.abs()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound).max()):.2f} of the bound"


# ------------------------------------------------------------------------------------------ decayed attention


def _ref(q, k, v, rate, s0, lengths, scale):
    """Token by token in float64, differentiable: outputs (B, T, H, dv) and the last state."""
    B, T, H, dk = q.shape
    group = H // k.shape[2]
    k, v = (t.repeat_interleave(group, 2) for t in (k, v))
    g = torch.exp(-rate.double())[None, :, None, None]
    s = torch.zeros(B, H, dk, v.shape[3], dtype=torch.float64, device=q.device) if s0 is None else s0
    out = []
    for t in range(T):
        n = g * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        o = scale * torch.einsum("bhi,bhij->bhj", q[:, t], n)
        if lengths is not None:
            live = (t < lengths)[:, None, None, None]
            n = torch.where(live, n, s)
            o = torch.where(live[..., 0], o, torch.zeros_like(o))
        s = n
        out.append(o)
    return (torch.stack(out, 1) if out else torch.zeros(B, 0, H, v.shape[3], dtype=torch.float64, device=q.device)), s


def _inputs(dtype, B, T, H, Hk, dk, dv, seed=0, rates=None):
    g = _gen(seed)
    q, k, v = (torch.randn(s, device="cuda", generator=g).to(dtype) for s in ((B, T, H, dk), (B, T, Hk, dk), (B, T, Hk, dv)))
    rate = torch.exp2(-torch.linspace(0.5, 7.0, H, device="cuda")) if rates is None else torch.tensor(rates, device="cuda")
    return q, k, v, rate, torch.randn((B, H, dk, dv), device="cuda", generator=g), g


CASES = [
    # dtype, B, T, H, Hk, dk, dv, lengths, state
    (FP32, 1, 1, 1, 1, 1, 1, None, True),
    (BF16, 1, 1, 2, 1, 8, 8, None, True),
    (FP32, 2, 63, 2, 2, 32, 32, None, False),
    (FP32, 2, 65, 4, 2, 48, 80, [65, 3], True),
    (FP32, 3, 200, 2, 1, 128, 100, [0, 1, 200], True),
    (FP32, 1, 700, 1, 1, 33, 7, None, True),
    (BF16, 2, 127, 2, 2, 64, 64, None, False),
    (BF16, 2, 129, 4, 2, 128, 128, [129, 128], True),
    (BF16, 3, 300, 2, 1, 16, 104, [0, 1, 257], True),
    (BF16, 2, 260, 2, 2, 37, 101, [260, 5], True),
    (BF16, 1, 1100, 2, 2, 128, 64, None, True),
    (BF16, 1, 1030, 1, 1, 64, 128, None, False),
    (BF16, 170, 130, 1, 1, 24, 24, None, True),
]


@pytest.mark.parametrize("dtype,B,T,H,Hk,dk,dv,lengths,state", CASES)
def test_decayed_attention_and_gradients(ews, dtype, B, T, H, Hk, dk, dv, lengths, state):
    q, k, v, rate, s0, g = _inputs(dtype, B, T, H, Hk, dk, dv)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if ln is not None:  # what lies beyond a length must not matter
        beyond = (torch.arange(T, device="cuda")[None] >= ln[:, None])[..., None, None]
        q, k, v = (torch.where(beyond, torch.full_like(x, float("nan")), x) for x in (q, k, v))
    do = torch.randn((B, T, H, dv), device="cuda", generator=g).to(dtype)
    ds = torch.randn((B, H, dk, dv), device="cuda", generator=g)
    scale = dk**-0.5
    leaf = [x.clone().requires_grad_() for x in (q, k, v)] + ([s0.clone().requires_grad_()] if state else [])
    got = ews.decayed_attention(*leaf[:3], rate, initial_state=leaf[3] if state else None, lengths=ln, return_state=state)
    outs = got if state else (got,)
    grads = torch.autograd.grad(outs, leaf, (do, ds) if state else (do,))

    def reference(absolute):
        f = (lambda x: torch.nan_to_num(x.double()).abs()) if absolute else (lambda x: torch.nan_to_num(x.double()))
        lv = [f(x).requires_grad_() for x in (q, k, v)] + ([f(s0).requires_grad_()] if state else [])
        o = _ref(*lv[:3], rate, lv[3] if state else None, ln, scale)
        o = o if state else o[:1]
        return o, torch.autograd.grad(o, lv, (f(do), f(ds)) if state else (f(do),))

    (want, wg), (ab, ag) = reference(False), reference(True)
    _check(outs[0], want[0], ab[0], True, dtype, "out")
    if state:
        _check(outs[1], want[1], ab[1], False, FP32, "state")
    for name, a, b, c in zip(("dq", "dk", "dv"), grads, wg, ag):
        _check(a, b, c, True, dtype, name)
    if state:
        _check(grads[3], wg[3], ag[3], False, FP32, "dinitial")
    if ln is not None:
        assert (outs[0][beyond.expand_as(outs[0])] == 0).all()
        for x, y in zip(grads[:3], (q, k, v)):
            assert (x[beyond.expand_as(x)] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rate", [0.0, 3.0, 200.0, float("inf")])
def test_decay_extremes(ews, dtype, rate):
    """No decay, and decays that underflow within a chunk, an axis or a token."""
    q, k, v, r, s0, _ = _inputs(dtype, 1, 333, 2, 2, 64, 64, seed=3, rates=[rate, 0.01])
    out, end = ews.decayed_attention(q, k, v, r, initial_state=s0, return_state=True)
    want, ws = _ref(q.double(), k.double(), v.double(), r, s0.double(), None, 0.125)
    ab, abs_s = _ref(q.double().abs(), k.double().abs(), v.double().abs(), r, s0.double().abs(), None, 0.125)
    _check(out, want, ab, True, dtype, "out")
    _check(end, ws, abs_s, False, FP32, "state")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides_offsets_and_broadcast(ews, dtype):
    """(B, H, T, d) memory, sliced widths with an unaligned start, and a key shared by all samples."""
    B, T, H, dk, dv = 2, 150, 2, 32, 40
    g = _gen(5)
    q = torch.randn((B, H, T, dk), device="cuda", generator=g).to(dtype).transpose(1, 2)
    k = torch.randn((1, T, H, dk), device="cuda", generator=g).to(dtype).expand(B, -1, -1, -1)
    v = torch.randn((B, T, H, dv + 3), device="cuda", generator=g).to(dtype)[..., 3:]
    rate = torch.tensor([0.3, 0.02], device="cuda")
    a = ews.decayed_attention(q, k, v, rate)
    b = ews.decayed_attention(q.contiguous(), k.contiguous(), v.contiguous(), rate)
    want = _ref(q.double(), k.double(), v.double(), rate, None, None, dk**-0.5)[0]
    ab = _ref(q.double().abs(), k.double().abs(), v.double().abs(), rate, None, None, dk**-0.5)[0]
    _check(a, want, ab, True, dtype, "strided")
    _check(b, want, ab, True, dtype, "contiguous")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_is_bit_reproducible_and_stream_ordered(ews, dtype):
    q, k, v, rate, s0, _ = _inputs(dtype, 2, 1500, 2, 1, 64, 64, seed=9)
    a = ews.decayed_attention(q, k, v, rate, initial_state=s0, return_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ews.decayed_attention(q, k, v, rate, initial_state=s0, return_state=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gradient_against_differences(ews):
    """A float32 directional derivative of <out, w> + <state, u> by central differences of the operator itself: the
    operator is linear in v and s0, so the differences have no truncation error there, and O(h^2) in q, k together."""
    q, k, v, rate, s0, g = _inputs(FP32, 2, 150, 2, 1, 24, 40, seed=11)
    w, u = torch.randn((2, 150, 2, 40), device="cuda", generator=g), torch.randn((2, 2, 24, 40), device="cuda", generator=g)
    leaf = [x.clone().requires_grad_() for x in (q, k, v, s0)]

    def f(x):
        o, s = ews.decayed_attention(*x[:3], rate, initial_state=x[3], return_state=True)
        return (o.double() * w).sum() + (s.double() * u).sum()

    grads = torch.autograd.grad(f(leaf), leaf)
    for i in range(4):
        d = torch.randn(leaf[i].shape, device="cuda", generator=g)
        h = 0.25  # each argument enters linearly
        up, down = ([x.detach() + (h * d if j == i else 0) for j, x in enumerate(leaf)] for h in (h, -h))
        num = float(f(up) - f(down)) / (2 * h)
        ana = float((grads[i].double() * d).sum())
        size = float((grads[i].double() * d).abs().sum())
        assert abs(num - ana) <= 1e-4 * size, (i, num, ana)


@pytest.mark.parametrize("dtype,B,H,Hk,dk,dv", [(BF16, 5, 4, 2, 64, 64), (FP32, 3, 2, 1, 33, 7), (BF16, 1, 1, 1, 128, 128), (FP32, 9, 3, 3, 1, 130 - 2)])
def test_step_matches_the_recurrence(ews, dtype, B, H, Hk, dk, dv):
    g = _gen(1)
    q, k, v = (torch.randn(s, device="cuda", generator=g).to(dtype) for s in ((B, H, dk), (B, Hk, dk), (B, Hk, dv)))
    rate = torch.exp2(-torch.linspace(0.5, 7.0, H, device="cuda"))
    pool = torch.randn((B + 2, H, dk, dv), device="cuda", generator=g)
    slots = torch.arange(B, 0, -1, device="cuda", dtype=torch.int32)
    slots[B // 2] = -1
    was = pool.clone()
    out = ews.decayed_attention_step(q, k, v, rate, pool, slots=slots)
    for b in range(B):
        s = int(slots[b])
        if s < 0:
            assert (out[b] == 0).all()
            continue
        want, ws = _ref(q[None, b:b + 1].double(), k[None, b:b + 1].double(), v[None, b:b + 1].double(), rate, was[s:s + 1].double(), None, dk**-0.5)
        ab, abs_s = _ref(q[None, b:b + 1].double().abs(), k[None, b:b + 1].double().abs(), v[None, b:b + 1].double().abs(), rate, was[s:s + 1].double().abs(), None, dk**-0.5)
        _check(out[b], want[0, 0], ab[0, 0], False, dtype, "out")
        _check(pool[s], ws[0], abs_s[0], False, FP32, "state")
    idle = [i for i in range(B + 2) if i not in set(slots.tolist())]
    assert torch.equal(pool[idle], was[idle])


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_prompt_then_steps_equal_one_prompt(ews, dtype):
    q, k, v, rate, _, _ = _inputs(dtype, 2, 140, 2, 2, 64, 64, seed=21)
    whole, end = ews.decayed_attention(q, k, v, rate, return_state=True)
    _, state = ews.decayed_attention(q[:, :130], k[:, :130], v[:, :130], rate, return_state=True)
    ab = _ref(q.double().abs(), k.double().abs(), v.double().abs(), rate, None, None, 0.125)
    for t in range(130, 140):
        o = ews.decayed_attention_step(q[:, t], k[:, t], v[:, t], rate, state)
        # two results of the operator: twice the bound of one
        _check((o.double() - whole[:, t].double()) / 2 + whole[:, t].double(), whole[:, t].double(), ab[0][:, t], True, dtype, "out")
    _check((state.double() - end) / 2 + end, end, ab[1], False, FP32, "state")


def test_attention_refusals(ews):
    q, k, v, rate, s0, _ = _inputs(BF16, 2, 8, 4, 2, 16, 16)
    f = ews.decayed_attention
    with pytest.raises(TypeError):
        f(q.half(), k.half(), v.half(), rate)
    with pytest.raises(TypeError):
        f(q, k.float(), v, rate)
    with pytest.raises(ValueError):
        f(q, k[:, :7], v, rate)
    with pytest.raises(ValueError):
        f(q[:, :, :3], k, v, rate[:3])
    with pytest.raises(ValueError):
        f(q, k, v, rate[:2])
    with pytest.raises(ValueError):
        f(q, k, v, rate, initial_state=s0.bfloat16())
    with pytest.raises(ValueError):
        f(q, k, v, rate, lengths=torch.tensor([8, 8], device="cuda"))
    with pytest.raises(ValueError):
        f(q, k, v, rate, scale=0.0)
    with pytest.raises(NotImplementedError):
        f(*(torch.zeros(1, 4, 1, 136, device="cuda") for _ in range(3)), rate[:1])
    with pytest.raises(NotImplementedError):
        f(q, k, v, rate.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        f(q.cpu(), k.cpu(), v.cpu(), rate.cpu())
    step = ews.decayed_attention_step
    with pytest.raises(ValueError):
        step(q[:, 0], k[:, 0], v[:, 0], rate, s0[:1])
    with pytest.raises(ValueError):
        step(q[:, 0], k[:, 0], v[:, 0], rate, s0.transpose(2, 3))
    with pytest.raises(ValueError):
        step(q[:, 0], k[:, 0], v[:, 0], rate, s0, slots=torch.zeros(2, device="cuda", dtype=torch.int64))
    with pytest.raises(RuntimeError):
        step(q[:, 0].clone().requires_grad_(), k[:, 0], v[:, 0], rate, s0)
    assert f(q[:0], k[:0], v[:0], rate).shape == (0, 8, 4, 16)
    o, s = f(q[:, :0], k[:, :0], v[:, :0], rate, initial_state=s0, return_state=True)
    assert o.shape == (2, 0, 4, 16) and torch.equal(s, s0)


def test_slot_out_of_range_raises_on_the_next_call(ews):
    q, k, v, rate, s0, _ = _inputs(FP32, 2, 1, 2, 2, 16, 16)
    slots = torch.tensor([0, 2], device="cuda", dtype=torch.int32)
    was = s0.clone()
    out = ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, s0, slots=slots)
    torch.cuda.synchronize()
    assert (out[1] == 0).all() and torch.equal(s0[1], was[1])
    with pytest.raises(IndexError):
        ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, s0)
    ews.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], rate, s0)


# --------------------------------------------------------------------------------------------- token embedding


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (77, 100, 24), (130, 7, 33), (5000, 300, 100), (3000, 70000, 64), (20000, 50, 8), (0, 5, 4)])
def test_embedding_and_gradient(ews, dtype, wide, n, V, D):
    g = _gen(n + V)
    ids = (torch.rand(n, device="cuda", generator=g) ** 3 * V).long().clamp_(0, V - 1)
    ids = ids if wide else ids.int()
    table = torch.randn((V, D), device="cuda", generator=g).to(dtype).requires_grad_()
    do = torch.randn((n, D), device="cuda", generator=g).to(dtype)
    out = ews.token_embedding(ids, table, scale=1.7, padding_index=V - 1)
    (grad,) = torch.autograd.grad(out, (table,), do)
    s = torch.tensor(1.7, dtype=FP32).double().item()
    want = s * table.detach().double()[ids.long()]
    _check(out, want, torch.zeros_like(want), False, dtype, "out")
    gw = torch.zeros((V, D), dtype=torch.float64, device="cuda")
    ga = gw.clone()
    gw.index_add_(0, ids.long(), do.double() * s)
    ga.index_add_(0, ids.long(), do.double().abs() * s)
    gw[V - 1] = 0
    # float32 sums in order: at most n roundings of 2^-24 of the running sum, within F32 for the runs here (< 300 in a
    # chain: segments of 64 and their partials)
    _check(grad, gw, ga, False, dtype, "grad")
    assert (grad[V - 1] == 0).all()
    again = torch.autograd.grad(ews.token_embedding(ids, table, scale=1.7, padding_index=V - 1), (table,), do)[0]
    assert torch.equal(grad, again)


def test_embedding_views_and_shapes(ews):
    g = _gen(0)
    big = torch.randn((50, 40), device="cuda", generator=g)
    ids = torch.randint(0, 50, (3, 5), device="cuda", generator=g)
    assert torch.equal(ews.token_embedding(ids, big[:, 3:19]), big[:, 3:19][ids])
    assert torch.equal(ews.token_embedding(ids.t(), big), big[ids.t()])
    t = big.t().requires_grad_()  # columns as rows
    ids = ids % 40
    out = ews.token_embedding(ids, t)
    assert torch.equal(out, t[ids])
    w = torch.randn((50,), device="cuda", generator=g).expand(3, 5, 50)  # a broadcast cotangent
    (grad,) = torch.autograd.grad(out, (t,), w)
    want = torch.zeros_like(t, dtype=torch.float64).index_add_(0, ids.reshape(-1), w.reshape(-1, 50).double())
    ab = torch.zeros_like(t, dtype=torch.float64).index_add_(0, ids.reshape(-1), w.reshape(-1, 50).double().abs())
    _check(grad, want, ab, False, FP32, "grad")


def test_embedding_index_errors_and_refusals(ews):
    table = torch.randn((10, 8), device="cuda")
    ids = torch.tensor([1, 10, -1, 2], device="cuda")
    out = ews.token_embedding(ids, table)
    torch.cuda.synchronize()
    assert (out[1:3] == 0).all() and torch.equal(out[0], table[1])
    with pytest.raises(IndexError):
        ews.token_embedding(ids[:1], table)
    with pytest.raises(TypeError):
        ews.token_embedding(ids.float(), table)
    with pytest.raises(TypeError):
        ews.token_embedding(ids, table.double())
    with pytest.raises(ValueError):
        ews.token_embedding(ids, table[0])
    with pytest.raises(ValueError):
        ews.token_embedding(ids, table, padding_index=10)
    with pytest.raises(RuntimeError):
        ews.token_embedding(ids.cpu(), table.cpu())


# --------------------------------------------------------------------------------------------- vocabulary loss


def _loss_ref(h, w, t, dl):
    live = t >= 0
    h = torch.where(live[:, None], h.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    z = h @ w.double().T
    lse = torch.logsumexp(z, 1)
    loss = torch.where(live, lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    g = p.clone()
    g.scatter_add_(1, t.clamp(min=0)[:, None], torch.full((len(t), 1), -1.0, dtype=torch.float64, device="cuda"))
    d = torch.where(live, dl.double(), torch.zeros_like(lse))[:, None]
    g, p = g * d, p * d.abs()
    ab = h.abs() @ w.double().abs().T  # bounds a logit's error
    return loss, g @ w.double(), g.T @ h, ab, p, g, h


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 10, 3), (77, 501, 100), (130, 128, 64), (300, 1000, 200), (129, 2500, 8), (513, 257, 333), (64, 20000, 40)])
def test_vocab_loss_and_gradients(ews, dtype, n, V, D):
    g = _gen(n * V)
    h = torch.randn((n, D), device="cuda", generator=g).to(dtype)
    w = (torch.randn((V, D), device="cuda", generator=g) * 2 / math.sqrt(D)).to(dtype)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    if n > 8:
        t[::5] = -100
        h[::5] = float("nan")  # rows without a target must not matter
    dl = torch.rand((n,), device="cuda", generator=g) + 0.1
    hl, wl = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ews.vocab_loss(hl, wl, t)
    dh, dw = torch.autograd.grad(loss, (hl, wl), dl)
    want, wh, ww, ab, p, gg, hz = _loss_ref(h, w, t, dl)
    delta = F32 * ab  # error of a logit
    worst = delta.amax(1)
    assert loss.dtype == FP32
    assert ((loss.double() - want).abs() <= 2 * worst + 1e-6 * (want.abs() + 20)).all()
    # G's error: its rounding (bf16), and the softmax's relative error from the logits'
    eg = p * (2 * worst + 2e-6)[:, None] + (U if dtype == BF16 else 2.0**-21) * gg.abs()
    for got, exact, err, form in ((dh, wh, eg @ w.double().abs(), gg.abs() @ w.double().abs()), (dw, ww, eg.T @ hz.abs(), gg.abs().T @ hz.abs())):
        bound = 1.05 * err + F32 * form + (U if dtype == BF16 else 2.0**-23) * exact.abs() + 1e-30
        assert ((got.double() - exact).abs() <= bound).all(), float(((got.double() - exact).abs() / bound).max())
    if n > 8:
        assert (loss[::5] == 0).all() and (dh[::5] == 0).all()
    assert torch.equal(dw, torch.autograd.grad(ews.vocab_loss(hl, wl, t), (wl,), dl)[0])


def test_vocab_loss_pieces(ews):
    """Rows enough that the backward walks the vocabulary in several pieces, the last one short."""
    n, V, D = 16384, 9001, 64
    g = _gen(4)
    h = torch.randn((n, D), device="cuda", generator=g).to(BF16).requires_grad_()
    w = (torch.randn((V, D), device="cuda", generator=g) / 8).to(BF16).requires_grad_()
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    loss = ews.vocab_loss(h.view(64, 256, D), w, t.view(64, 256))
    assert loss.shape == (64, 256)
    dh, dw = torch.autograd.grad(loss.mean(), (h, w))
    dl = torch.full((n,), 1.0 / n, device="cuda")
    want, wh, ww, ab, p, gg, hz = _loss_ref(h.detach(), w.detach(), t, dl)
    assert ((loss.view(-1).double() - want).abs() <= 2 * F32 * ab.amax(1) + 3e-5).all()
    eg = p * (2 * F32 * ab.amax(1) + 2e-6)[:, None] + U * gg.abs()
    for got, exact, err, form in ((dh, wh, eg @ w.detach().double().abs(), gg.abs() @ w.detach().double().abs()), (dw, ww, eg.T @ hz.abs(), gg.abs().T @ hz.abs())):
        assert ((got.double() - exact).abs() <= 1.05 * err + F32 * form + U * exact.abs() + 1e-30).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,kept", [(700, 3), (700, 130), (300, 300), (257, 1)])
def test_vocab_loss_with_few_targets(ews, dtype, n, kept):
    """Only the rows that have a target are computed: none of the others' values matter, wherever they lie."""
    V, D = 1030, 72
    g = _gen(n + kept)
    h = torch.full((n, D), float("nan"), device="cuda").to(dtype)
    t = torch.full((n,), -100, device="cuda")
    rows = torch.randperm(n, device="cuda", generator=g)[:kept]
    h[rows] = torch.randn((kept, D), device="cuda", generator=g).to(dtype)
    t[rows] = torch.randint(0, V, (kept,), device="cuda", generator=g)
    w = (torch.randn((V, D), device="cuda", generator=g) / 4).to(dtype)
    dl = torch.rand((n,), device="cuda", generator=g) + 0.1
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


@pytest.mark.parametrize("first", [None, 0.0])
def test_a_common_loss_gradient_is_not_rounded(ews, first):
    """1 + 2^-8 lies half way between two bfloat16 numbers: rounded into every row it would put the gradients 2^-8 off.
    Left out of what is rounded, two independent roundings remain, each of 2^-7 / sqrt(12) at most. A first row whose
    gradient is another one has the ordinary rounding: 2^-8 of every entry, and that of the result."""
    n, V, D = 600, 2000, 128
    g = _gen(61)
    h = torch.randn((n, D), device="cuda", generator=g).bfloat16()
    w = (torch.randn((V, D), device="cuda", generator=g) * 0.02).bfloat16()
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    dl = torch.full((n,), (1 + 2.0**-8) / 512, device="cuda")
    if first is not None:
        dl[0] = first
    hl, wl = h.clone().requires_grad_(), w.clone().requires_grad_()
    got = torch.autograd.grad(ews.vocab_loss(hl, wl, t), (hl, wl), dl)
    want = _loss_ref(h, w, t, dl)[1:3]
    bound = 2**0.5 * 2**-7 / 12**0.5 if first is None else 2**-8 + 2**-7 / 12**0.5
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= bound * b.norm()


def test_vocab_loss_gradient_against_differences(ews):
    n, V, D = 40, 300, 24
    g = _gen(8)
    h = torch.randn((n, D), device="cuda", generator=g).requires_grad_()
    w = (torch.randn((V, D), device="cuda", generator=g) / 4).requires_grad_()
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    f = lambda a, b: ews.vocab_loss(a, b, t).double().sum()  # noqa: E731
    grads = torch.autograd.grad(f(h, w), (h, w))
    for i, x in enumerate((h, w)):
        d = torch.randn(x.shape, device="cuda", generator=g)
        d /= d.norm()
        e = 2.0**-4  # truncation e^2 |f'''| / 6 <= 1e-3 of the scale below; rounding 1e-6 * 40 * 6 / e
        args = [[y.detach() + (s * e * d if j == i else 0) for j, y in enumerate((h, w))] for s in (1, -1)]
        num = float(f(*args[0]) - f(*args[1])) / (2 * e)
        ana = float((grads[i].double() * d).sum())
        assert abs(num - ana) <= 2e-2 * float(grads[i].norm()), (num, ana)


def test_vocab_loss_strides_targets_and_refusals(ews):
    g = _gen(2)
    big = torch.randn((20, 70), device="cuda", generator=g)
    w = torch.randn((33, 64), device="cuda", generator=g)
    t = torch.randint(0, 33, (20,), device="cuda", generator=g)
    a = ews.vocab_loss(big[:, 3:67], w, t)
    b = ews.vocab_loss(big[:, 3:67].contiguous(), w.t().contiguous().t(), t.int())
    assert torch.equal(a, b)
    ig = t.clone()
    ig[:] = 7
    hl, wl = big[:, :64].clone().requires_grad_(), w.clone().requires_grad_()
    loss = ews.vocab_loss(hl, wl, ig, ignore_index=7)  # nothing has a target
    dh, dw = torch.autograd.grad(loss.sum(), (hl, wl))
    assert (loss == 0).all() and (dh == 0).all() and (dw == 0).all()
    empty = ews.vocab_loss(hl[:0], wl, ig[:0])
    assert empty.shape == (0,) and (torch.autograd.grad(empty.sum(), (wl,))[0] == 0).all()
    bad = t.clone()
    bad[3] = 33
    loss = ews.vocab_loss(big[:, :64], w, bad)
    torch.cuda.synchronize()
    assert loss[3] == 0
    with pytest.raises(IndexError):
        ews.vocab_loss(big[:, :64], w, t)
    with pytest.raises(TypeError):
        ews.vocab_loss(big[:, :64].half(), w.half(), t)
    with pytest.raises(TypeError):
        ews.vocab_loss(big[:, :64].bfloat16(), w, t)
    with pytest.raises(TypeError):
        ews.vocab_loss(big[:, :64], w, t.float())
    with pytest.raises(ValueError):
        ews.vocab_loss(big[:, :63], w, t)
    with pytest.raises(ValueError):
        ews.vocab_loss(big[:, :64], w, t[:5])
    with pytest.raises(RuntimeError):
        ews.vocab_loss(big[:, :64].cpu(), w.cpu(), t.cpu())


def test_operators_in_a_cuda_graph(ews):
    """Captured once, replayed on new contents: nothing waits on the host or keeps an input's address or values."""
    q, k, v, rate, s0, g = _inputs(BF16, 2, 300, 2, 2, 64, 64, seed=31)
    h = torch.randn((100, 64), device="cuda", generator=g).to(BF16)
    w = torch.randn((500, 64), device="cuda", generator=g).to(BF16)
    t = torch.randint(0, 500, (100,), device="cuda", generator=g)

    def run():
        x = ews.token_embedding(t, w, scale=2.0)
        return ews.decayed_attention(q, k, v, rate, initial_state=s0, return_state=True) + (x, ews.vocab_loss(h, w, t))

    with torch.no_grad():
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        for x in (q, k, v, s0, h, w):
            x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        t.copy_(torch.randint(0, 500, (100,), device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run()):
            assert torch.equal(a, b)
