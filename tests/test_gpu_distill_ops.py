"""The loss against a teacher's top logits, against its definition in 64 bits: masks, temperatures, several pieces, graphs.

Tolerances are bounds, element by element, from the arithmetic: s = 2e-5 (products exact to 2^-21, chains of some hundred
truncated additions of 2^-23 each) of a logit's sum over absolute values bounds its error dz; a loss moves by at most twice the largest
dz of its row over the temperature, and its own sums cost 2^-19 of their absolute terms. A probability moves by the factor
2 dz / temperature; G = (q - p) w is rounded to the inputs' type once (u, half a step; float32: three planes), with one more for the
mantissa that is kept out of it, and the gradients' sums add s and their own rounding."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
S = 2e-5


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


def reference(h, w, ids, t, tau, dloss):
    """(values, bounds) of the loss, dh, dw."""
    u = torch.finfo(h.dtype).eps / 2
    h, w, ids, t = h.double(), w.double(), ids.long(), t.double() / tau
    there = (ids >= 0) & (t > -float("inf"))
    live = there.any(1)
    p = torch.softmax(t.masked_fill(~there, -float("inf")).masked_fill(~live[:, None], 0.0), 1) * live[:, None] * there
    z = h @ w.mT / tau
    dz = (S * (h.abs() @ w.abs().mT) / tau).amax(1)
    lse = torch.logsumexp(z, 1)
    at = ids.clamp(min=0)
    gap = lse[:, None] - z.gather(1, at)
    loss = (torch.special.xlogy(p, p) + p * gap).sum(1) * live
    eloss = (2 * dz + 2.0**-19 * (torch.special.xlogy(p, p).abs() + p * gap.abs() + p * (z.gather(1, at).abs() + 1)).sum(1) + 2.0**-20) * live
    q = torch.exp(z - lse[:, None])
    weight = (dloss.double() * live / tau)[:, None]
    target = torch.zeros_like(q).scatter_add_(1, at, p)
    g = (q - target) * weight
    eg = (q * (2 * dz[:, None] + 2.0**-19) + 2.0**-20 * target) * weight.abs() + 2 * u * g.abs()
    dh, dw = g @ w, g.mT @ h
    eh = (eg + S * g.abs()) @ w.abs() + u * dh.abs()
    ew = (eg + S * g.abs()).mT @ h.abs() + u * dw.abs()
    return (loss, dh, dw), (eloss, eh, ew)


def check(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound * 1.001 + 1e-30)
    assert got.shape == want.shape and not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.2f} of the bound"


def inputs(dtype, N, V, D, K, seed=0, empty=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(N, D, device="cuda", generator=g).to(dtype)
    w = (torch.randn(V, D, device="cuda", generator=g) * 1.5 * D**-0.5).to(dtype)
    ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:K] for _ in range(N)])
    t = torch.randn(N, K, device="cuda", generator=g) * 2 + 5
    if N > 2:
        ids[torch.rand(N, K, device="cuda", generator=g) < 0.1] = -1
        ids[torch.rand(N, device="cuda", generator=g) < empty] = -7
    return h, w, ids, t, torch.rand(N, device="cuda", generator=g) + 0.1


def run(ews, h, w, ids, t, tau, dloss):
    leaves = [x.clone().requires_grad_() for x in (h, w)]
    loss = ews.distill_loss(*leaves, ids, t, temperature=tau)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, dloss)]


CASES = [(1, 1, 1, 1, 1.0), (1, 7, 3, 5, 2.0), (3, 10, 8, 10, 1.0), (5, 300, 64, 1, 0.7), (130, 257, 40, 33, 1.0), (64, 1000, 128, 128, 2.0),
         (300, 5000, 72, 20, 0.5), (257, 131, 200, 100, 1.0), (2000, 700, 16, 8, 1.0), (40, 20011, 33, 64, 4.0)]


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("N,V,D,K,tau", CASES)
def test_losses_and_gradients(ews, dtype, N, V, D, K, tau):
    h, w, ids, t, dloss = inputs(dtype, N, V, D, K)
    got = run(ews, h, w, ids, t, tau, dloss)
    want, bound = reference(h, w, ids, t, tau, dloss)
    for name, a, b, c in zip(("loss", "dh", "dw"), got, want, bound):
        check(a, b, c, name)
    assert (got[0] >= 0).all()
    with torch.no_grad():
        assert torch.equal(ews.distill_loss(h, w, ids.int(), t, temperature=tau), got[0])


def test_several_pieces_of_a_vocabulary(ews):
    """Enough rows and entries that the backward forms its gradient matrix in pieces."""
    h, w, ids, t, dloss = inputs(BF16, 4096, 70001, 24, 16)
    ids[:, 0] = torch.randint(69000, 70001, (4096,), device="cuda")  # the last piece has entries too
    got = run(ews, h, w, ids, t, 1.0, dloss)
    for a in range(0, 4096, 1024):
        want, bound = reference(h[a : a + 1024], w, ids[a : a + 1024], t[a : a + 1024], 1.0, dloss[a : a + 1024])
        check(got[0][a : a + 1024], want[0], bound[0], "loss")
        check(got[1][a : a + 1024], want[1], bound[1], "dh")
        total = (want[2], bound[2]) if a == 0 else (total[0] + want[2], total[1] + bound[2])
    check(got[2], *total, "dw")


def test_the_gradient_is_the_slope(ews):
    h, w, ids, t, dloss = inputs(FP32, 20, 60, 16, 6)
    grads = run(ews, h, w, ids, t, 1.5, dloss)[1:]
    step_size = 2.0**-6
    noise = float((reference(h, w, ids, t, 1.5, dloss)[1][0] * dloss.double()).sum())
    for k, leaf in enumerate((h, w)):
        step = torch.randn(leaf.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k))
        ends = []
        for sign in (step_size, -step_size):
            a = [h, w]
            a[k] = leaf + sign * step
            ends.append(float((ews.distill_loss(*a, ids, t, temperature=1.5).double() * dloss).sum()))
        want = float((grads[k].double() * step).sum())
        size = float((grads[k].double() * step).abs().sum())
        # a loss is bent by the variance of (step's logit) under q, third derivatives below 16 of it
        assert abs((ends[0] - ends[1]) / (2 * step_size) - want) <= 64 * step_size**2 * (size + 1) + noise / step_size, k


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_masks_and_what_is_not_finite(ews, dtype):
    """Absent entries may hold anything; a logit of -inf is absent; the type's lowest value is a logit like others; NaN stays in
    its row."""
    h, w, ids, t, dloss = inputs(dtype, 8, 50, 16, 6, empty=0.0)
    ids = ids.clamp(min=0)
    ids[0] = -1
    ids[1, 2:] = -1
    t[1, 2:] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda")
    t[2] = -float("inf")
    t[3, 1:4] = -float("inf")
    t[4] = torch.finfo(FP32).min
    t[5, 1:] = torch.finfo(FP32).min
    t[6, 2] = 88.0
    got = run(ews, h, w, ids, t, 1.0, dloss)
    want, bound = reference(h, w, ids, torch.where(ids < 0, 0.0, t), 1.0, dloss)
    for name, a, b, c in zip(("loss", "dh", "dw"), got, want, bound):
        check(a, b, c, name)
    assert got[0][0] == 0 and got[0][2] == 0 and (got[1][[0, 2]] == 0).all()
    t[7, 3] = float("nan")
    bad = ews.distill_loss(h, w, ids, t)
    assert bad[7].isnan() and torch.equal(bad[:7], got[0][:7])
    h[3, 2] = float("nan")
    bad = ews.distill_loss(h, w, ids, t)
    assert bad[3].isnan() and torch.equal(bad[[0, 1, 2, 4, 5, 6]], got[0][[0, 1, 2, 4, 5, 6]])


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_orders_duplicates_and_types(ews, dtype):
    h, w, ids, t, dloss = inputs(dtype, 50, 90, 24, 12)
    want = run(ews, h, w, ids, t, 1.0, dloss)
    order = torch.randperm(12, device="cuda")
    for a, b in zip(run(ews, h, w, ids[:, order], t[:, order], 1.0, dloss), want):
        assert torch.allclose(a.float(), b.float(), rtol=2.0**-7 if dtype == BF16 else 1e-5, atol=1e-5)
    # one id twice: two entries
    ids[:, 5] = ids[:, 2]
    got = run(ews, h, w, ids, t, 1.0, dloss)
    want, bound = reference(h, w, ids, t, 1.0, dloss)
    for name, a, b, c in zip(("loss", "dh", "dw"), got, want, bound):
        check(a, b, c, name)
    assert torch.equal(ews.distill_loss(h, w, ids, t.bfloat16()), ews.distill_loss(h, w, ids, t.bfloat16().float()))
    # strided, with leading axes
    wide = torch.zeros(50, 30, dtype=ids.dtype, device="cuda")
    wide[:, 3:15] = ids
    assert torch.equal(ews.distill_loss(h.reshape(5, 10, 24), w, wide[:, 3:15].reshape(5, 10, 12), t.reshape(5, 10, 12)).reshape(-1), got[0])


def test_one_certain_entry_is_the_cross_entropy(ews):
    """K = 1: the teacher is sure, and the loss is the vocabulary loss of that id."""
    h, w, ids, t, dloss = inputs(FP32, 200, 500, 64, 1)
    got = run(ews, h, w, ids, t, 1.0, dloss)
    leaves = [x.clone().requires_grad_() for x in (h, w)]
    loss = ews.vocab_loss(*leaves, torch.where(ids[:, 0] < 0, -100, ids[:, 0]))
    want = [loss.detach(), *torch.autograd.grad(loss, leaves, dloss)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_a_student_that_agrees_has_no_loss(ews, dtype):
    """The teacher's entries are the student's whole vocabulary: the divergence and the gradient vanish."""
    h, w, _, _, dloss = inputs(dtype, 30, 100, 32, 1)
    z = h.float() @ w.float().T
    loss, dh, dw = run(ews, h, w, torch.arange(100, device="cuda").expand(30, -1), z, 2.0, dloss)
    assert (loss >= 0).all() and float(loss.max()) < 2.0**-18 * float(z.abs().max())
    assert float(dh.abs().max()) < 1e-3 and float(dw.abs().max()) < 1e-3  # q - p is a rounding of 2^-20 at most, over 100 terms


def test_an_id_beyond_the_vocabulary_is_reported(ews):
    h, w, ids, t, dloss = inputs(FP32, 6, 40, 16, 4, empty=0.0)
    ids = ids.clamp(min=0)
    ids[2, 1] = 40
    loss = ews.distill_loss(h, w, ids, t)
    torch.cuda.synchronize()
    with pytest.raises(IndexError):
        ews.distill_loss(h, w, ids, t)
    ids[2, 1] = -1
    assert torch.equal(ews.distill_loss(h, w, ids, t), loss)


def test_no_rows_and_no_live_rows(ews):
    h, w, ids, t, dloss = inputs(FP32, 6, 40, 16, 4)
    loss, dh, dw = run(ews, h[:0], w, ids[:0], t[:0], 1.0, dloss[:0])
    assert loss.shape == (0,) and dh.shape == (0, 16) and (dw == 0).all()
    loss, dh, dw = run(ews, h, w, torch.full_like(ids, -1), t, 1.0, dloss)
    assert (loss == 0).all() and (dh == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_on_streams_and_in_a_graph(ews, dtype):
    h, w, ids, t, dloss = inputs(dtype, 300, 1000, 64, 16)
    leaves = [x.clone().requires_grad_() for x in (h, w)]

    def once():
        loss = ews.distill_loss(*leaves, ids, t, temperature=2.0)
        return [loss.detach(), *torch.autograd.grad(loss, leaves, dloss)]

    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(once())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in results for a, b in zip(got, first))
    with torch.cuda.stream(streams[0]):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    with torch.no_grad():
        leaves[0].mul_(0.5)
        ids[7] = -1
    graph.replay()
    got = [x.clone() for x in captured]
    assert got[0][7] == 0
    assert all(torch.equal(a, b) for a, b in zip(got, once()))


def test_refusals_on_the_device(ews):
    h, w, ids, t, _ = inputs(FP32, 4, 30, 8, 5)
    f = ews.distill_loss
    for call in (lambda: f(h[:, :4], w, ids, t), lambda: f(h, w, ids[:3], t[:3]), lambda: f(h, w, ids, t[:, :2]), lambda: f(h, w, ids[:, :0], t[:, :0]),
                 lambda: f(h, w, ids, t, temperature=0.0), lambda: f(h, w, ids, t, temperature=float("nan")), lambda: f(h, w, ids, t, temperature=-1.0),
                 lambda: f(h, w, ids, t.cpu()), lambda: f(h, w[:0], ids, t)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    for call in (lambda: f(h, w.bfloat16(), ids, t), lambda: f(h, w, ids.float(), t), lambda: f(h, w, ids, t.double())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: f(h, w, ids.repeat(1, 26), t.repeat(1, 26)), lambda: f(h, w, ids, t.clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            call()
    leaf = h.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(leaf, w, ids, t).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_a_repeated_id_may_take_the_sum_below_zero(ews, dtype):
    """An id that occurs twice is two entries, of which a student can be surer than either: 2 (p / 2) (log(p / 2) - log q) with q near
    p is negative. Rows whose ids are distinct lie beside them; a repeated id that is absent makes no row negative."""
    h, w, ids, t, dloss = inputs(dtype, 96, 60, 24, 6, empty=0.0)
    h = h * 3
    best = (h.double() @ w.double().mT).argmax(1)
    twice = torch.arange(96, device="cuda") % 2 == 0
    ids[twice, 1], ids[twice, 4] = best[twice], best[twice]
    t[twice, 1], t[twice, 4] = 12.0, 12.0
    ids[1::4, 2:4] = -1
    got = run(ews, h, w, ids, t, 1.0, dloss)
    want, bound = reference(h, w, ids, t, 1.0, dloss)
    for name, a, b, c in zip(("loss", "dh", "dw"), got, want, bound):
        check(a, b, c, name)
    assert float(want[0].min()) < -0.3 and float(got[0].min()) < -0.3


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("tau", [0.5, 0.7, 2.0**-20, 3.0])
def test_logits_at_the_types_ends(ews, dtype, tau):
    """Only a logit of -inf is absent: the type's lowest value is a logit like others, alone in a row or beside others, at any
    temperature, and so is its largest. A constant added to a row changes nothing but the rounding of what is given."""
    h, w, ids, t, dloss = inputs(dtype, 9, 50, 16, 6, empty=0.0)
    ids = ids.clamp(min=0)
    for row in range(9):
        ids[row] = torch.randperm(50, device="cuda", generator=torch.Generator(device="cuda").manual_seed(row))[:6]
    t = t * min(tau, 1.0)
    low, high = torch.finfo(FP32).min, torch.finfo(FP32).max
    t[0] = low
    t[1, 1:] = low
    t[2] = high
    t[3, 2] = high
    t[4, :3], t[4, 3:] = low, high
    t[5] += 1000 * min(tau, 1.0)
    t[6, 2:] = -float("inf")
    t[7] = -float("inf")
    got = run(ews, h, w, ids, t, tau, dloss)
    want, bound = reference(h, w, ids, t, tau, dloss)
    for name, a, b, c in zip(("loss", "dh", "dw"), got, want, bound):
        check(a, b, c, name)
    assert (got[1][7] == 0).all() and (got[1][[0, 2]] != 0).any(1).all()
    half = torch.where(t == low, torch.finfo(BF16).min, torch.where(t == high, torch.finfo(BF16).max, t)).to(BF16)
    assert torch.equal(ews.distill_loss(h, w, ids, half, temperature=tau), ews.distill_loss(h, w, ids, half.float(), temperature=tau))


def exact_products(dtype, N, V, D, seed=0):
    """hidden and weight rows of small whole numbers: every product and every sum of them is exact."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, w = (torch.randint(-2, 3, (n, D), device="cuda", generator=g).to(dtype) for n in (N, V))
    return h, w


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("tau", [0.3, 0.013, 1e-4, 1e-18, 2.0**-90, 1e18])
def test_gradients_at_any_temperature(ews, dtype, tau):
    """Logits that are exact: what the probabilities lose is the rounding of (z - max) / temperature alone, 2^-22 of it (the difference is
    exact), and beyond 20 they are 2^-28 and less. So q is within 2^-17 of itself, G = (q - p) w within that and two roundings to the
    type, the gradients' sums within S and a rounding more."""
    h, w = exact_products(dtype, 40, 70, 12)
    _, _, ids, t, dloss = inputs(dtype, 40, 70, 12, 7, empty=0.1)
    t = t * tau
    got = run(ews, h, w, ids, t, tau, dloss)
    u = torch.finfo(dtype).eps / 2
    hd, wd, td = h.double(), w.double(), t.double() / tau
    there = ids >= 0
    live = there.any(1)
    p = torch.softmax(td.masked_fill(~there, -float("inf")).masked_fill(~live[:, None], 0.0), 1) * there
    z = hd @ wd.mT
    q = torch.softmax((z - z.amax(1, keepdim=True)) / tau, 1)
    target = torch.zeros_like(q).scatter_add_(1, ids.clamp(min=0), p)
    weight = (dloss.double() * live / tau)[:, None]
    g = (q - target) * weight
    eg = 2.0**-17 * (q + target) * weight + 2 * u * g.abs()
    for name, a, want, bound in (("dh", got[1], g @ wd, (eg + S * g.abs()) @ wd.abs()), ("dw", got[2], g.mT @ hd, (eg + S * g.abs()).mT @ hd.abs())):
        check(a, want, bound + u * want.abs(), name)


@pytest.mark.parametrize("N,V,D,dtype", [(2048, 30011, 24, FP32), (4096, 40011, 8, BF16)])
def test_several_pieces_in_planes_and_of_narrow_rows(ews, N, V, D, dtype):
    """Three planes of G in pieces, and rows narrower than a tile."""
    h, w, ids, t, dloss = inputs(dtype, N, V, D, 16)
    ids[:, 0] = torch.randint(V - 300, V, (N,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    got = run(ews, h, w, ids, t, 0.7, dloss)
    total = None
    for a in range(0, N, 1024):
        want, bound = reference(h[a : a + 1024], w, ids[a : a + 1024], t[a : a + 1024], 0.7, dloss[a : a + 1024])
        check(got[0][a : a + 1024], want[0], bound[0], "loss")
        check(got[1][a : a + 1024], want[1], bound[1], "dh")
        total = (want[2], bound[2]) if total is None else (total[0] + want[2], total[1] + bound[2])
    check(got[2], *total, "dw")


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_rows_of_wider_matrices(ews, dtype):
    """Strided rows, at offsets that TMA can and cannot start at, with their gradients."""
    h, w, ids, t, dloss = inputs(dtype, 150, 300, 40, 9)
    want, bound = reference(h, w, ids, t, 2.0, dloss)
    for at in (0, 3, 8):
        wide = [torch.full((x.shape[0], 40 + 16), float("nan"), dtype=dtype, device="cuda") for x in (h, w)]
        for big, x in zip(wide, (h, w)):
            big[:, at : at + 40] = x
        leaves = [big.requires_grad_() for big in wide]
        loss = ews.distill_loss(*(big[:, at : at + 40] for big in leaves), ids, t, temperature=2.0)
        grads = torch.autograd.grad(loss, leaves, dloss)
        check(loss.detach(), want[0], bound[0], ("loss", at))
        for k in range(2):
            check(grads[k][:, at : at + 40], want[1 + k], bound[1 + k], ("grad", k, at))
            assert (grads[k][:, :at] == 0).all() and (grads[k][:, at + 40 :] == 0).all()
