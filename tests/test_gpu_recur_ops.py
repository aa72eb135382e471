"""The gated linear recurrence against its definition in 64 bits: prompts, gradients, single tokens, masks, streams, graphs.

Tolerances are bounds, element by element, from the arithmetic. In float32 one step of the recurrence adds a rounding of the
state (2^-24) and of the decay (2^-25): T 2^-23 of the sum over absolute values covers T of them. The gates and the root
cost a few units of the exponent unit's 2^-22 whatever T: 2^-19 of the same sum. Where a gradient has a factor 1 - sigmoid,
a difference of numbers of size one, the absolute form has one in its place. A result rounded to bfloat16 adds half a step,
2^-8 of itself. The absolute form is the same formula over absolute values, evaluated in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


def reference(x, decay, gate, rate, s0, lengths, do, ds, absolute=False):
    """Outputs (h, end) and gradients (dx, ddecay, dgate, drate, ds0) token by token in float64; ``absolute``: the same sums
    over absolute values."""
    f = (lambda t: t.double().abs()) if absolute else (lambda t: t.double())
    B, T, C = x.shape
    sign = 1.0 if absolute else -1.0
    rate = rate.double()
    r, i = torch.sigmoid(decay.double()), torch.sigmoid(gate.double())
    p = rate * r
    a, m = torch.exp(-p), torch.sqrt(-torch.expm1(-2 * p))
    slope = torch.where(m > 0, a * a / torch.where(m > 0, m, torch.ones_like(m)), torch.zeros_like(m))
    live = torch.ones(B, T, 1, dtype=torch.bool, device=x.device)
    if lengths is not None:
        live = (torch.arange(T, device=x.device) < lengths[:, None])[..., None]
    x = torch.where(live, f(x), 0.0)
    zero = torch.zeros(B, C, dtype=torch.float64, device=x.device)
    h = zero if s0 is None else f(s0)
    before, out = [], []
    for t in range(T):
        before.append(h)
        h = torch.where(live[:, t], a[:, t] * h + m[:, t] * i[:, t] * x[:, t], h)
        out.append(torch.where(live[:, t], h, 0.0))
    g = zero if ds is None else f(ds)
    dx, dr, di, drate = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(rate)
    for t in reversed(range(T)):
        here = torch.where(live[:, t], g + f(do[:, t]), 0.0)
        dl = here * (a[:, t] * before[t] + sign * slope[:, t] * i[:, t] * x[:, t])
        dx[:, t] = here * m[:, t] * i[:, t]
        di[:, t] = here * m[:, t] * x[:, t] * i[:, t] * (1.0 if absolute else 1 - i[:, t])
        dr[:, t] = sign * rate * r[:, t] * dl * (1.0 if absolute else 1 - r[:, t])
        drate += sign * (r[:, t] * dl).sum(0)
        g = torch.where(live[:, t], a[:, t] * here, g)
    out = torch.stack(out, 1) if T else torch.zeros(B, 0, C, dtype=torch.float64, device=x.device)
    return out, h, dx, dr, di, drate, g


def check(got, want, absform, T, what):
    bound = (T * 2.0**-23 + 2.0**-19) * absform + 1e-30
    if got.dtype == BF16:
        bound = bound + 2.0**-8 * want.abs()
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert got.shape == want.shape and not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.2f} of the bound"


def inputs(dtype, B, T, C, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, decay, gate, do = (torch.randn((B, T, C), device="cuda", generator=g).to(dtype) for _ in range(4))
    rate = torch.exp2(2.0 - 12.0 * torch.rand(C, device="cuda", generator=g))
    s0, ds = (torch.randn((B, C), device="cuda", generator=g) for _ in range(2))
    return x, decay, gate, rate, s0, do, ds


CASES = [
    # dtype, B, T, C, lengths, state
    (FP32, 1, 1, 1, None, True),
    (BF16, 1, 1, 2, None, True),
    (BF16, 3, 5, 64, [0, 1, 5], True),
    (FP32, 2, 8, 32, None, False),
    (BF16, 2, 63, 66, None, True),
    (BF16, 2, 64, 130, [64, 1], False),
    (FP32, 2, 65, 33, [65, 64], True),
    (BF16, 2, 128, 7, None, True),
    (BF16, 1, 129, 64, None, True),
    (FP32, 4, 200, 100, [0, 200, 64, 129], True),
    (BF16, 4, 300, 96, [0, 1, 257, 300], True),
    (FP32, 1, 513, 31, None, False),
    (BF16, 2, 1100, 65, [1100, 1024], True),
    (FP32, 1, 2500, 3, None, True),
    (BF16, 1, 2500, 40, None, False),
    (BF16, 70, 140, 70, None, True),
]


@pytest.mark.parametrize("dtype,B,T,C,lengths,state", CASES)
def test_outputs_and_gradients(ews, dtype, B, T, C, lengths, state):
    x, decay, gate, rate, s0, do, ds = inputs(dtype, B, T, C)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    given = (x, decay, gate)
    if ln is not None:  # what lies beyond a length must not matter
        beyond = (torch.arange(T, device="cuda") >= ln[:, None])[..., None]
        given = tuple(torch.where(beyond, torch.full_like(t, float("nan")), t) for t in given)
    leaves = [t.clone().requires_grad_() for t in (*given, rate)] + ([s0.clone().requires_grad_()] if state else [])
    got = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4] if state else None, lengths=ln, return_state=state)
    outs = got if state else (got,)
    grads = torch.autograd.grad(outs, leaves, (do, ds) if state else (do,))
    args = (x, decay, gate, rate, s0 if state else None, ln, do, ds if state else None)
    want, ab = reference(*args), reference(*args, absolute=True)
    check(outs[0].detach(), want[0], ab[0], T, "h")
    if state:
        check(outs[1].detach(), want[1], ab[1], T, "state")
    for name, a, b, c in zip(("dx", "ddecay", "dgate", "drate", "dstate"), grads, want[2:], ab[2:]):
        check(a, b, c, 2 * T, name)
    with torch.no_grad():  # without a gradient: the same numbers
        plain = ews.gated_recurrence(*(t.detach() for t in leaves[:4]), initial_state=s0 if state else None, lengths=ln, return_state=state)
    assert torch.equal(plain[0] if state else plain, outs[0].detach())


@pytest.mark.parametrize("T", [64, 65, 96, 97, 140, 333])
@pytest.mark.parametrize("C,odd", [(192, None), (192, "dout"), (192, "x"), (130, None), (129, None)])
def test_many_chains(ews, T, C, odd):
    """More chains of 64 channels than the GPU has multiprocessors, so that states are kept every 32 tokens: backward in tiles of
    32 tokens, and (where a layout does not let the forward or the backward copy tiles whole) of 64 on the same states."""
    B = 75
    x, decay, gate, rate, s0, do, ds = inputs(BF16, B, T, C, seed=T)
    ln = (torch.arange(B, device="cuda", dtype=torch.int32) * 37) % (T + 1)

    def shifted(t):
        wide = torch.full((*t.shape[:2], C + 9), float("nan"), dtype=BF16, device="cuda")
        wide[..., 1 : C + 1] = t
        return wide[..., 1 : C + 1]

    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    if odd == "x":
        leaves[0] = shifted(x).requires_grad_()
    out = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], lengths=ln, return_state=True)
    grads = torch.autograd.grad(out, leaves, (shifted(do) if odd == "dout" else do, ds))
    args = (x, decay, gate, rate, s0, ln, do, ds)
    want, ab = reference(*args), reference(*args, absolute=True)
    for k, (name, got) in enumerate(zip(("h", "state", "dx", "ddecay", "dgate", "drate", "dstate"), (out[0].detach(), out[1].detach(), *grads))):
        check(got, want[k], ab[k], T if k < 2 else 2 * T, name)


def test_the_gradient_is_the_slope(ews):
    """Against central differences of the operator's own float32 results, in 64 bits' worth of directions: the difference's
    error is its curvature (h^2) and the results' 2^-19 over h."""
    x, decay, gate, rate, s0, do, ds = inputs(FP32, 2, 70, 5)
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    f = lambda a: [t.double() for t in ews.gated_recurrence(*a[:4], initial_state=a[4], return_state=True)]  # noqa: E731
    total = lambda a: float((f(a)[0] * do).sum() + (f(a)[1] * ds).sum())  # noqa: E731
    out = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
    grads = torch.autograd.grad(out, leaves, (do, ds))
    scale = float(sum((t.detach().double().abs() * w.abs()).sum() for t, w in zip(out, (do, ds))))
    h = 2.0**-7
    for k in range(5):
        step = torch.randn(leaves[k].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k))
        if k == 3:
            step = step * rate  # stays positive
        ends = []
        for sign in (h, -h):
            a = [t.detach() for t in leaves]
            a[k] = a[k] + sign * step
            ends.append(total(a))
        slope = (ends[0] - ends[1]) / (2 * h)
        want = float((grads[k].double() * step).sum())
        size = float((grads[k].double() * step).abs().sum())
        assert abs(slope - want) <= 16 * h * h * size + 2.0**-19 * scale / h, (k, slope, want)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("value", [-float("inf"), None])
def test_a_shut_decay_gate_passes_the_state_on(ews, dtype, value):
    """-inf and the type's lowest value: no step of the clock, so the state stays and nothing is learned. Bit for bit where all
    are shut. Behind open tokens the state comes once token by token and once, for the warps that follow, as the map A h + H
    of up to 16 tokens: each way rounds A, H and the state once a token, 2^-24 each, so that the two differ by at most 2 x 3 x 16 x
    2^-24 < 2^-17 of the sum over absolute values. A result rounded to bfloat16 may then fall to the next value, 2^-7 apart."""
    x, decay, gate, rate, s0, do, ds = inputs(dtype, 2, 150, 34)
    value = torch.finfo(dtype).min if value is None else value
    decay[:, 20:140] = value
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    out, end = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
    size = reference(x, decay, gate, rate, s0, None, do, ds, absolute=True)[0][:, 19:20]
    off = (out[:, 20:140].double() - out[:, 19:20].double()).abs()
    assert (off <= 2.0**-17 * size + (2.0**-7 * out[:, 19:20].abs() if dtype == BF16 else 0.0)).all()
    assert torch.equal(out[:, 48:64], out[:, 48:49].expand(-1, 16, -1))
    grads = torch.autograd.grad((out, end), leaves, (do, ds))
    assert all(torch.isfinite(g).all() for g in grads)
    assert all((g[:, 20:140] == 0).all() for g in grads[:3])
    all_shut = torch.full_like(decay, value)
    out, end = ews.gated_recurrence(x, all_shut, gate, rate, initial_state=s0, return_state=True)
    assert torch.equal(end, s0) and torch.equal(out, s0.to(dtype)[:, None].expand_as(out))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_saturated_gates_and_rates(ews, dtype):
    """Rates of zero and of a thousand, gates at both ends: what the definition gives, gradients finite."""
    x, decay, gate, rate, s0, do, ds = inputs(dtype, 1, 140, 6)
    rate = torch.tensor([0.0, 1000.0, 1e-6, 1e-12, 88.0, 0.3499], device="cuda")
    decay[:, ::3] = 30.0
    decay[:, 1::3] = -30.0
    gate[:, ::2] = 60.0
    gate[:, 1::4] = -60.0
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    out, end = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
    grads = torch.autograd.grad((out, end), leaves, (do, ds))
    args = (x, decay, gate, rate, s0, None, do, ds)
    want, ab = reference(*args), reference(*args, absolute=True)
    check(out.detach(), want[0], ab[0], 140 + 64, "h")  # sigmoid(+-30): the argument's rounding, 60 * 2^-24 of the gate
    check(end.detach(), want[1], ab[1], 140 + 64, "state")
    for name, a, b, c in zip(("dx", "ddecay", "dgate", "drate", "dstate"), grads, want[2:], ab[2:]):
        assert torch.isfinite(a).all(), name
        check(a, b, c, 2 * 140 + 128, name)


def test_views_of_one_projection(ews):
    """x, decay and gate as parts of a wider tensor, a transposed one, strided along the last axis, and one that starts off a
    word's boundary: each within the bounds of the definition. (They need not agree bit for bit: how a tensor lies decides how
    many tokens a warp joins as one map, and maps of 8 and of 16 tokens round differently.)"""
    for dtype in (BF16, FP32):
        wide = torch.randn(2, 90, 3 * 50 + 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
        rate = torch.full((50,), 0.1, device="cuda")
        one = torch.ones(2, 90, 50, dtype=dtype, device="cuda")
        for at in (0, 1):
            parts = wide[..., at : at + 150].split(50, -1)
            args = (*parts, rate, None, None, one, None)
            want, ab = reference(*args), reference(*args, absolute=True)
            flipped = [p.transpose(0, 1).contiguous().transpose(0, 1) for p in parts]
            last = [p.mT.contiguous().mT for p in parts]  # the last axis strided
            for given in (parts, [p.contiguous() for p in parts], flipped, last):
                check(ews.gated_recurrence(*given, rate), want[0], ab[0], 90, "h")
            leaf = wide.clone().requires_grad_()
            ews.gated_recurrence(*leaf[..., at : at + 150].split(50, -1), rate).sum().backward()  # an expanded cotangent
            for k in range(3):
                check(leaf.grad[..., at + 50 * k : at + 50 * k + 50], want[2 + k], ab[2 + k], 180, k)
            assert (leaf.grad[..., 0 if at else 150] == 0).all()


def test_one_input_as_all_three(ews):
    """The same tensor in three places: its gradients add up."""
    x, _, _, rate, _, do, _ = inputs(FP32, 2, 33, 8)
    leaf = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(ews.gated_recurrence(leaf, leaf, leaf, rate), leaf, do)
    three = [x.clone().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(ews.gated_recurrence(*three, rate), three, do)
    assert torch.allclose(got, parts[0] + parts[1] + parts[2], rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_no_tokens_and_no_samples(ews, dtype):
    x, decay, gate, rate, s0, do, ds = inputs(dtype, 2, 0, 5)
    leaf, rt = s0.clone().requires_grad_(), rate.clone().requires_grad_()
    out, end = ews.gated_recurrence(x, decay, gate, rt, initial_state=leaf, return_state=True)
    assert out.shape == (2, 0, 5) and torch.equal(end, s0)
    d0, dr = torch.autograd.grad(end, (leaf, rt), ds)
    assert torch.equal(d0, ds) and (dr == 0).all()
    assert (ews.gated_recurrence(x, decay, gate, rate, return_state=True)[1] == 0).all()
    x, decay, gate, rate, s0, do, ds = inputs(dtype, 0, 7, 5)
    rt = rate.clone().requires_grad_()
    out = ews.gated_recurrence(x, decay, gate, rt)
    assert out.shape == (0, 7, 5)
    assert (torch.autograd.grad(out, rt, do)[0] == 0).all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("C", [64, 37])
def test_steps_follow_the_scan(ews, dtype, C):
    """A prompt, then tokens one by one on pooled states in another order with idle rows: the scan over all of them. The
    step runs the same float32 operations in the same order, so its states are the scan's to the maps' rounding."""
    x, decay, gate, rate, s0, _, _ = inputs(dtype, 3, 40, C)
    want, wend = ews.gated_recurrence(x, decay, gate, rate, initial_state=s0, return_state=True)
    _, mid = ews.gated_recurrence(x[:, :30], decay[:, :30], gate[:, :30], rate, initial_state=s0, return_state=True)
    pool = torch.full((6, C), 7.0, device="cuda")
    slots = torch.tensor([4, -1, 0, 5], dtype=torch.int32, device="cuda")
    rows = torch.tensor([0, 0, 1, 2], device="cuda")
    pool[slots[[0, 2, 3]].long()] = mid
    for t in range(30, 40):
        got = ews.gated_recurrence_step(x[rows, t], decay[rows, t], gate[rows, t], rate, pool, slots=slots)
        assert (got[1] == 0).all()
        for b, row in ((0, 0), (2, 1), (3, 2)):
            assert torch.allclose(got[b].float(), want[row, t].float(), rtol=2.0**-7 if dtype == BF16 else 1e-5, atol=1e-6)
    assert torch.allclose(pool[slots[[0, 2, 3]].long()], wend, rtol=1e-5, atol=1e-6)
    assert (pool[[1, 2, 3]] == 7.0).all()
    again = mid.clone()  # without slots: row b on state b
    got = ews.gated_recurrence_step(x[:, 30], decay[:, 30], gate[:, 30], rate, again)
    assert torch.allclose(got.float(), want[:, 30].float(), rtol=2.0**-7 if dtype == BF16 else 1e-5, atol=1e-6)


def test_a_slot_out_of_range_is_reported(ews):
    x, decay, gate, rate, s0, _, _ = inputs(FP32, 2, 1, 8)
    pool = s0.clone()
    slots = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    out = ews.gated_recurrence_step(x[:, 0], decay[:, 0], gate[:, 0], rate, pool, slots=slots)
    torch.cuda.synchronize()
    assert (out[1] == 0).all() and torch.equal(pool[0], s0[0])
    with pytest.raises(IndexError):
        ews.gated_recurrence_step(x[:, 0], decay[:, 0], gate[:, 0], rate, pool)
    ews.gated_recurrence_step(x[:, 0], decay[:, 0], gate[:, 0], rate, pool)


def test_a_step_counts_as_a_write(ews):
    x, decay, gate, rate, s0, do, _ = inputs(FP32, 2, 5, 8)
    leaf, pool = x.clone().requires_grad_(), s0.clone()
    out = ews.gated_recurrence(leaf, decay, gate, rate, initial_state=pool)
    with torch.no_grad():
        ews.gated_recurrence_step(x[:, 0], decay[:, 0], gate[:, 0], rate, pool)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_runs_repeat_bit_for_bit_on_any_stream(ews):
    """Many tiles that look back at one another: the sums have one order, whatever the timing."""
    x, decay, gate, rate, s0, do, ds = inputs(BF16, 6, 3000, 192)
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]

    def once():
        out = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (do, ds)))

    first = once()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for i in range(9):  # three at a time on the GPU
        with torch.cuda.stream(streams[i % 3]):
            results.append(once())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_in_a_graph(ews):
    x, decay, gate, rate, s0, do, ds = inputs(BF16, 2, 400, 64)
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    pool = s0.clone()

    def once():
        out = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
        grads = torch.autograd.grad(out, leaves, (do, ds))
        with torch.no_grad():
            step = ews.gated_recurrence_step(x[:, 0], decay[:, 0], gate[:, 0], rate, pool)
        return [t.detach() for t in out] + list(grads) + [step]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    with torch.no_grad():
        for leaf in leaves:
            leaf.mul_(0.75)
    pool.copy_(s0)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    got, end = [t.clone() for t in captured], pool.clone()
    pool.copy_(s0)
    once()
    want = once()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(end, pool)


def test_refusals_on_the_device(ews):
    x, decay, gate, rate, s0, _, _ = inputs(FP32, 2, 5, 8)
    rec, step = ews.gated_recurrence, ews.gated_recurrence_step
    for call in (lambda: rec(x, decay, gate[:, :4], rate), lambda: rec(x, decay, gate, rate[:4]), lambda: rec(x, decay, gate, rate.double()),
                 lambda: rec(x, decay, gate, rate, initial_state=s0[:1]), lambda: rec(x, decay, gate, rate, lengths=torch.zeros(2, device="cuda")),
                 lambda: rec(x[0], decay[0], gate[0], rate), lambda: rec(x, decay, gate, rate.cpu()), lambda: rec(x, decay, gate, rate[None]),
                 lambda: rec(x, decay, gate, rate, lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
                 lambda: step(x[:, 0], decay[:, 0], gate[:, 0], rate, s0[:1]), lambda: step(x[:, 0], decay[:, 0], gate[:, 0], rate, s0.mT),
                 lambda: step(x[:, 0], decay[:, 0], gate[:, 0], rate, s0, slots=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    with pytest.raises(TypeError):
        rec(x, decay.bfloat16(), gate, rate)
    with pytest.raises(TypeError):
        rec(x.half(), decay.half(), gate.half(), rate)
    with pytest.raises(RuntimeError, match="no gradient"):
        step(x[:, 0].requires_grad_(), decay[:, 0], gate[:, 0], rate, s0)
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(NotImplementedError):
        rec(fw.make_dual(x, torch.ones_like(x)), decay, gate, rate)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(rec(leaf, decay, gate, rate).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_broadcast_inputs(ews, dtype):
    """Inputs without memory of their own along the samples or the tokens; their gradients are the sums over what they stand for."""
    B, T, C = 3, 100, 32
    x, decay, gate, rate, s0, do, ds = inputs(dtype, B, T, C)
    one, two, three = x[:1].clone().requires_grad_(), decay[:, :1].clone().requires_grad_(), gate[:1, :1].clone().requires_grad_()
    given = [t.expand(B, T, C) for t in (one, two, three)]
    out = ews.gated_recurrence(*given, rate)
    whole = [t.detach().contiguous().requires_grad_() for t in given]
    want = ews.gated_recurrence(*whole, rate)
    args = (*(t.detach() for t in whole), rate, None, None, do, None)
    value, ab = reference(*args), reference(*args, absolute=True)
    check(out.detach(), value[0], ab[0], T, "h")
    check(want.detach(), value[0], ab[0], T, "h")
    grads = torch.autograd.grad(out, (one, two, three), do)
    for g, v, a, axes in zip(grads, value[2:5], ab[2:5], ((0,), (1,), (0, 1))):
        # the sum that autograd forms of the operator's gradients, each rounded (bfloat16: half a step), in the inputs' type
        n = B * T
        bound = ((2 * T * 2.0**-23 + 2.0**-19) * a).sum(axes, keepdim=True) + n * torch.finfo(dtype).eps * a.sum(axes, keepdim=True)
        assert ((g.double() - v.sum(axes, keepdim=True)).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("B,T,C", [(2, 30, 33), (3, 150, 64), (75, 140, 64), (2, 150, 34)])
@pytest.mark.parametrize("top", [1.39, None])
def test_what_a_shut_decay_gate_hides(ews, dtype, B, T, C, top):
    """A token whose decay gate is shut may hold anything: nothing of it reaches the state or a gradient, and its own gradients are
    zero. With a finite token in its place, the same numbers."""
    x, decay, gate, rate, s0, do, ds = inputs(dtype, B, T, C)
    rate = rate.clamp(max=1.39) if top else rate
    shut = torch.rand(B, T, C, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.2
    shut[:, 3] = True
    kind = torch.randint(0, 4, (B, T, C), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max], device="cuda").to(dtype)[kind]
    decay = torch.where(shut, torch.where(kind % 2 == 0, -float("inf"), torch.finfo(dtype).min).to(dtype), decay)
    results = []
    for a, b in ((x, gate), (torch.where(shut, junk, x), torch.where(shut, junk.flip(0), gate))):
        leaves = [t.clone().requires_grad_() for t in (a, decay, b, rate, s0)]
        out = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
        results.append([t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (do, ds))))
        pool = s0.clone()
        with torch.no_grad():
            results[-1] += [ews.gated_recurrence_step(a[:, 3], decay[:, 3], b[:, 3], rate, pool), pool]
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert all((g[shut] == 0).all() for g in results[1][2:5])
    assert torch.equal(results[1][8], s0)


MANY = [(FP32, 4, 300, 96), (BF16, 4, 300, 192), (BF16, 75, 140, 192), (BF16, 3, 70, 130), (FP32, 2, 200, 33), (FP32, 40, 300, 256), (BF16, 6, 3000, 192)]


@pytest.mark.parametrize("top", [1.39, None])
@pytest.mark.parametrize("dtype,B,T,C", MANY)
def test_rates_on_either_side(ews, dtype, B, T, C, top):
    """Rates of up to 1.39, all of them where decays are formed without the exponent unit, and a few beyond, where a warp forms them with
    it. In float32 more tiles than the GPU holds CTAs, so that their stages go round; in bfloat16 the same with fewer chains than
    multiprocessors (backward in tiles of 64 tokens) and with more (32)."""
    x, decay, gate, rate, s0, do, ds = inputs(dtype, B, T, C, seed=T + B)
    rate = rate.clamp(max=1.39) if top else rate
    ln = (T - (torch.arange(B, device="cuda", dtype=torch.int32) * 61) % (T // 2)).int()
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    out = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], lengths=ln, return_state=True)
    grads = torch.autograd.grad(out, leaves, (do, ds))
    args = (x, decay, gate, rate, s0, ln, do, ds)
    want, ab = reference(*args), reference(*args, absolute=True)
    for k, (name, got) in enumerate(zip(("h", "state", "dx", "ddecay", "dgate", "drate", "dstate"), (out[0].detach(), out[1].detach(), *grads))):
        check(got, want[k], ab[k], T if k < 2 else 2 * T, name)


@pytest.mark.parametrize("dtype,B,C", [(BF16, 2, 64), (BF16, 75, 192), (BF16, 2, 65), (FP32, 2, 64), (FP32, 3, 33)])
def test_gradients_of_the_end_state_alone(ews, dtype, B, C):
    """No cotangent for the outputs, on states kept every 64 and every 32 tokens."""
    x, decay, gate, rate, s0, do, ds = inputs(dtype, B, 140, C)
    leaves = [t.clone().requires_grad_() for t in (x, decay, gate, rate, s0)]
    _, end = ews.gated_recurrence(*leaves[:4], initial_state=leaves[4], return_state=True)
    grads = torch.autograd.grad(end, leaves, ds)
    args = (x, decay, gate, rate, s0, None, torch.zeros_like(do), ds)
    want, ab = reference(*args), reference(*args, absolute=True)
    for name, a, b, c in zip(("dx", "ddecay", "dgate", "drate", "dstate"), grads, want[2:], ab[2:]):
        check(a, b, c, 280, name)
