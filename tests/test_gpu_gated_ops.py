"""The gated linear layer against its definition in 64 bits: many rows, few rows, gradients, strides, graphs.

Tolerances are bounds, element by element, from the arithmetic, with u half a step of the type (bfloat16 2^-8, float32 2^-24)
and s = 2e-5 (products exact to 2^-21, chains of some hundred truncated additions of 2^-23 each) of the sum over absolute values:
a projection is off by s |X| |W|, and as it is kept for the backward by 2^-15 of itself more (24 bits, cut off). Through the product and the activation, whose slope
is at most 1.13 and whose second derivative at most 0.8, that gives the bound of H, dG and dU; dG and dU are rounded once more as
operands (float32: three planes, 2^-24). The activation itself costs 2^-20."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
S = 2e-5


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


def act_of(g, kind):
    """act, its slope, in float64."""
    if kind == "silu":
        c = torch.sigmoid(g)
        return g * c, c * (1 + g * (1 - c))
    c = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def reference(x, wg, wu, dh, kind):
    """(values, bounds) of h, dx, dwg, dwu."""
    u = torch.finfo(x.dtype).eps / 2
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    g, up = x @ wg.mT, x @ wu.mT
    eg, eu = S * (x.abs() @ wg.abs().mT), S * (x.abs() @ wu.abs().mT)
    act, slope = act_of(g, kind)
    h = act * up
    eh = 1.13 * eg * (up.abs() + eu) + act.abs() * eu + 2.0**-20 * h.abs() + u * h.abs()
    eg, eu = eg + 2.0**-15 * g.abs(), eu + 2.0**-15 * up.abs()
    dg, du = dh * up * slope, dh * act
    edg = dh.abs() * (eu * (slope.abs() + 0.8 * eg) + up.abs() * (0.8 * eg + 2.0**-20)) + u * dg.abs()
    edu = dh.abs() * (1.13 * eg + 2.0**-20 * act.abs()) + u * du.abs()
    dx, dwg, dwu = dg @ wg + du @ wu, dg.mT @ x, du.mT @ x
    ex = (edg + S * dg.abs()) @ wg.abs() + (edu + S * du.abs()) @ wu.abs() + u * dx.abs()
    ewg, ewu = (edg + S * dg.abs()).mT @ x.abs() + u * dwg.abs(), (edu + S * du.abs()).mT @ x.abs() + u * dwu.abs()
    return (h, dx, dwg, dwu), (eh, ex, ewg, ewu)


def check(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound * 1.001 + 1e-30)
    assert got.shape == want.shape and not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.2f} of the bound"


def inputs(dtype, N, D, F, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return r(N, D).to(dtype), (r(F, D) * D**-0.5).to(dtype), (r(F, D) * D**-0.5).to(dtype), r(N, F).to(dtype)


SIZES = [(1, 1, 1), (48, 136, 72), (41, 40, 130), (96, 72, 200), (81, 1000, 64), (7, 2052, 20), (12, 1301, 36), (32, 520, 40), (31, 516, 9),
         (1, 8, 16), (1, 1024, 520), (2, 33, 17), (4, 40, 31), (8, 64, 64), (9, 256, 48), (16, 128, 100), (17, 72, 33),
         (33, 96, 200), (64, 300, 24), (64, 1000, 72), (65, 64, 64), (127, 40, 129), (128, 64, 8), (129, 200, 130), (300, 512, 341),
         (1000, 136, 1000), (2050, 24, 260), (700, 1032, 2056)]


@pytest.mark.parametrize("N,D,F", SIZES)
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_outputs_and_gradients(ews, dtype, N, D, F):
    kind = "gelu" if F % 3 == 0 else "silu"
    x, wg, wu, dh = inputs(dtype, N, D, F)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    h = ews.gated_linear(*leaves, activation=kind)
    grads = torch.autograd.grad(h, leaves, dh)
    want, bound = reference(x, wg, wu, dh, kind)
    for name, a, b, c in zip(("h", "dx", "dwg", "dwu"), (h.detach(), *grads), want, bound):
        check(a, b, c, name)
    with torch.no_grad():
        assert torch.equal(ews.gated_linear(x, wg, wu, activation=kind), h.detach())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_the_gradient_is_the_slope(ews, kind):
    """Against central differences of the operator's own float32 results: their error is the curvature, h^2, and the results'
    rounding, S of the sum over absolute values, over h."""
    x, wg, wu, dh = inputs(FP32, 70, 24, 40)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(ews.gated_linear(*leaves, activation=kind), leaves, dh)
    h = 2.0**-6
    scale = float(reference(x, wg, wu, dh, kind)[1][0].mul(dh.double().abs()).sum())
    for k in range(3):
        step = torch.randn(leaves[k].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)) * (1.0 if k == 0 else 24**-0.5)
        ends = []
        for sign in (h, -h):
            a = [t.detach() for t in leaves]
            a[k] = a[k] + sign * step
            ends.append(float((ews.gated_linear(*a, activation=kind).double() * dh).sum()))
        want = float((grads[k].double() * step).sum())
        size = float((grads[k].double() * step).abs().sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - want) <= 16 * h * h * size + scale / h, k


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("N", [5, 150])
def test_strides_and_leading_axes(ews, dtype, N):
    """Rows of wider matrices, an offset that TMA cannot start at, transposed weights, one matrix as both weights."""
    x, wg, wu, dh = inputs(dtype, N, 64, 72)
    want = ews.gated_linear(x, wg, wu)
    wide = torch.zeros(N, 64 + 8 + 3, dtype=dtype, device="cuda")
    for at in (0, 3, 8):
        wide[:, at : at + 64] = x
        both = torch.zeros(72, 2 * 64 + 8, dtype=dtype, device="cuda")
        both[:, at : at + 64], both[:, at + 64 : at + 128] = wg, wu
        got = ews.gated_linear(wide[:, at : at + 64], both[:, at : at + 64], both[:, at + 64 : at + 128])
        assert torch.equal(got, want), at
    assert torch.equal(ews.gated_linear(x, wg.mT.contiguous().mT, wu), want)
    assert torch.equal(ews.gated_linear(x.reshape(N, 1, 1, 64), wg, wu), want.reshape(N, 1, 1, 72))
    assert torch.equal(ews.gated_linear(x[0], wg, wu), ews.gated_linear(x[:1], wg, wu)[0])
    # one set of weights in both places, and a cotangent of no memory: gradients add up
    leaf = wg.clone().requires_grad_()
    ews.gated_linear(x, leaf, leaf).sum().backward()
    two = [wg.clone().requires_grad_() for _ in range(2)]
    parts = torch.autograd.grad(ews.gated_linear(x, *two), two, torch.ones_like(want))
    assert torch.equal(leaf.grad, parts[0] + parts[1])


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_frozen_inputs(ews, dtype, wanted):
    x, wg, wu, dh = inputs(dtype, 300, 72, 200)
    full = [t.clone().requires_grad_() for t in (x, wg, wu)]
    all_grads = torch.autograd.grad(ews.gated_linear(*full), full, dh)
    some = [t.clone().requires_grad_(w) for t, w in zip((x, wg, wu), wanted)]
    out = ews.gated_linear(*some)
    got = torch.autograd.grad(out, [t for t in some if t.requires_grad], dh)
    want, bound = reference(x, wg, wu, dh, "silu")
    for a, b, k in zip(got, [g for g, w in zip(all_grads, wanted) if w], [k for k in range(3) if wanted[k]]):
        check(a, want[1 + k], bound[1 + k], k)
        check(b, want[1 + k], bound[1 + k], k)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("N", [3, 130])
def test_rows_stay_apart(ews, dtype, N):
    """What is not finite in one row reaches no other row's output or input gradient."""
    x, wg, wu, dh = inputs(dtype, N, 40, 56)
    clean = [t.clone().requires_grad_() for t in (x, wg, wu)]
    want = ews.gated_linear(*clean)
    (wdx,) = torch.autograd.grad(want, clean[:1], dh)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    leaf = x.clone().requires_grad_()
    got = ews.gated_linear(leaf, wg, wu)
    (dx,) = torch.autograd.grad(got, leaf, dh)
    keep = [0, *range(3, N)]
    assert torch.equal(got[keep], want[keep]) and torch.equal(dx[keep], wdx[keep])
    assert got[1].isnan().all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_large_projections(ews, dtype):
    """Gates far on either side: the activation's limits, with finite gradients."""
    x, wg, wu, dh = inputs(dtype, 70, 16, 32)
    wg = wg * 40
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    for kind in ("silu", "gelu"):
        h = ews.gated_linear(*leaves, activation=kind)
        grads = torch.autograd.grad(h, leaves, dh)
        assert all(torch.isfinite(t).all() for t in (h, *grads))
        want, bound = reference(x, wg, wu, dh, kind)
        check(h.detach(), want[0], bound[0], kind)


def test_no_rows(ews):
    x, wg, wu, dh = inputs(BF16, 0, 16, 24)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    h = ews.gated_linear(*leaves)
    assert h.shape == (0, 24)
    dx, dwg, dwu = torch.autograd.grad(h, leaves, dh)
    assert dx.shape == (0, 16) and (dwg == 0).all() and (dwu == 0).all()


@pytest.mark.parametrize("dtype,N", [(BF16, 20), (BF16, 300), (FP32, 200)])
def test_on_streams_and_in_a_graph(ews, dtype, N):
    x, wg, wu, dh = inputs(dtype, N, 128, 256)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]

    def once():
        h = ews.gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

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
        for leaf in leaves:
            leaf.mul_(0.5)
    graph.replay()
    got = [t.clone() for t in captured]
    assert all(torch.equal(a, b) for a, b in zip(got, once()))


def test_refusals_on_the_device(ews):
    x, wg, wu, _ = inputs(FP32, 4, 8, 6)
    f = ews.gated_linear
    for call in (lambda: f(x, wg, wu[:3]), lambda: f(x[:, :4], wg, wu), lambda: f(x, wg[0], wu[0]), lambda: f(x, wg, wu, activation="relu"),
                 lambda: f(x, wg[:0], wu[:0]), lambda: f(x, wg.cpu(), wu)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    with pytest.raises(TypeError):
        f(x, wg.bfloat16(), wu)
    with pytest.raises(TypeError):
        f(x.half(), wg.half(), wu.half())
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(NotImplementedError):
        f(fw.make_dual(x, torch.ones_like(x)), wg, wu)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(leaf, wg, wu).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("N", [5, 40, 150])
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_activations_to_their_ends(ews, dtype, N, kind):
    """Projections that are exact (one product each, U = 1), so that the activation shows: within 2^-15 of itself and a rounding
    (a truncated addition leaves 2^-23 of G, which an exponential of -80, or of -81 / 2, makes 2^-16.6 of the result; its argument's
    own rounding adds half of that, its last places less), both for H and, through
    dU = dH act(G) and dG = dH act'(G), for the weights' gradients, which are rounded once as operands and once as results. GELU to
    -9, where Phi is 1e-19, SiLU to -80."""
    top = 9.0 if kind == "gelu" else 80.0
    g = torch.linspace(-top, top, 145, device="cuda", dtype=torch.float64).to(dtype)
    F = len(g)
    x = torch.zeros(N, 16, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = 1, 1
    wg, wu = (torch.zeros(F, 16, device="cuda", dtype=dtype) for _ in range(2))
    wg[:, 0], wu[:, 1] = g, 1
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    dh = torch.zeros(N, F, device="cuda", dtype=dtype)
    dh[N - 1] = 1
    h = ews.gated_linear(*leaves, activation=kind)
    _, dwg, dwu = torch.autograd.grad(h, leaves, dh)
    act, slope = act_of(g.double(), kind)
    u = torch.finfo(dtype).eps / 2
    # where act' passes zero its two terms, sigmoid and g sigmoid (1 - sigmoid) or Phi and g phi, cancel
    if kind == "silu":
        terms = torch.sigmoid(g.double()) * (1 + (g.double() * torch.sigmoid(-g.double())).abs())
    else:
        terms = 0.5 * torch.special.erfc(-g.double() / math.sqrt(2)) + g.double().abs() * torch.exp(-(g.double() ** 2) / 2) / math.sqrt(2 * math.pi)
    check(h.detach(), act.expand(N, F), (2.0**-15 + u) * act.abs().expand(N, F), "h")
    # (kept in 24 bits, 2^-15 of g: exact for these numbers of bfloat16; float32 keeps all)
    check(dwu[:, 1], act, (2.0**-15 + 2 * u) * act.abs(), "dwu")
    check(dwg[:, 0], slope, 2.0**-15 * terms + 2 * u * slope.abs(), "dwg")


@pytest.mark.parametrize("N", [3, 33, 64, 200])
@pytest.mark.parametrize("kept", [False, True])
def test_float32_values_that_planes_cannot_hold(ews, N, kept):
    """Infinities and values beyond bfloat16's largest, in X and in either weight: what a row gives does not depend on how many rows
    come with it, and is the definition's."""
    x, wg, wu, _ = inputs(FP32, N, 72, 200)
    x[2, 5], x[0, 7] = float("inf"), 3.4e38
    x[1, 9] = -3.3999e38
    wg[7, 5] = 0.0  # 0 x inf: NaN
    wg[9, 4], wu[11, 6], wg[13, 3] = -float("inf"), float("inf"), float("nan")
    wg[:, 7], wu[:, 7], wu[:, 9] = wg[:, 7] * 1e-36, wu[:, 7] * 1e-36, wu[:, 9] * 1e-30  # row 0 stays small, row 1's gates are shut or huge
    g, u = x.double() @ wg.double().mT, x.double() @ wu.double().mT
    c = torch.sigmoid(g)
    want = torch.where(c == 0, torch.zeros_like(g), g * c) * u
    clean = [torch.where(torch.isfinite(t), t, 0.0) for t in (x, wg, wu)]
    bound = reference(*clean, torch.zeros(N, 200, device="cuda"), "silu")[1][0]
    weight = wg.clone().requires_grad_(kept)
    got = ews.gated_linear(x, weight, wu).detach().double()
    assert torch.equal(got.isnan(), want.isnan())
    limit = torch.finfo(FP32).max
    huge = want.abs() > limit * (1 - 2.0**-10)
    assert torch.equal(got[huge & ~want.isnan()], torch.copysign(torch.full_like(want, float("inf")), want)[huge & ~want.isnan()])
    rest = ~huge & ~want.isnan()
    assert ((got - want).abs()[rest] <= bound[rest] * 1.001 + 1e-30).all()


@pytest.mark.parametrize("dtype,N,D,F", [(BF16, 48, 2048, 5632), (BF16, 1000, 512, 1032), (BF16, 700, 64, 40000), (FP32, 500, 128, 341)])
def test_runs_repeat_bit_for_bit(ews, dtype, N, D, F):
    """Whatever the workspaces and outputs held before."""
    x, wg, wu, dh = inputs(dtype, N, D, F)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    first = None
    for fill in (0.0, float("nan"), 1e30, float("inf")):
        junk = [torch.full((16 << 20,), fill, device="cuda") for _ in range(4)]
        del junk
        h = ews.gated_linear(*leaves)
        got = [h.detach(), *torch.autograd.grad(h, leaves, dh)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
