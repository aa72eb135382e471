"""The operators of a gated recurrent token model as its users call them: the gated linear recurrence (prompts, training,
single tokens), the gated linear layer (both projections, the activation and the product, training, prompts, single
tokens), and the loss of a student against a teacher's top logits over a large vocabulary, with its gradients.

``run`` makes one pass, in plain torch operations (``own = False``) or through the package (``own = True``);
``exact`` evaluates the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # one conversation's next token: latency
        dict(name="recur-step-one", op="step", dtype="bf16", B=1, C=1024, idle=0),
        # a full serving batch over a pool of states, some rows idle
        dict(name="recur-step-batch", op="step", dtype="bf16", B=256, C=4096, idle=5),
        # one long prompt, handed over to the step as a state: one row, long axis
        dict(name="recur-prompt-long", op="scan", dtype="bf16", B=1, T=17984, C=2048, ragged=False, state=True),
        # an ordinary training batch, the rates learned
        dict(name="recur-train", op="mix", dtype="bf16", B=8, T=2048, C=2048, ragged=False, state=False),
        # float32 training at the stacked model's length: ragged, an odd width, carried state with its gradient
        dict(name="recur-train-f32", op="mix", dtype="f32", B=16, T=1440, C=333, ragged=True, state=True),
        # the channel stage of one conversation's next token: latency
        dict(name="gated-one", op="gated", dtype="bf16", N=1, D=1024, F=4096, act="silu", grad=False),
        # the channel stage of a serving batch
        dict(name="gated-batch", op="gated", dtype="bf16", N=48, D=2048, F=5632, act="silu", grad=False),
        # a prompt's channel stage, an odd number of tokens
        dict(name="gated-prompt", op="gated", dtype="bf16", N=4001, D=2048, F=8192, act="silu", grad=False),
        # an ordinary training batch
        dict(name="gated-train", op="gated", dtype="bf16", N=8192, D=1024, F=4096, act="silu", grad=True),
        # float32 training at the stacked model's width, an odd inner width, the other activation
        dict(name="gated-train-f32", op="gated", dtype="f32", N=5760, D=128, F=341, act="gelu", grad=True),
        # the stacked model's width with a small vocabulary, float32, tempered
        dict(name="distill-small-f32", op="distill", dtype="f32", N=1440, V=1000, D=128, K=10, tau=2.0, grad=True),
        # an ordinary training batch, odd vocabulary
        dict(name="distill-train", op="distill", dtype="bf16", N=8192, V=50257, D=1024, K=32, tau=1.0, grad=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "scan", "mix", "gated", "gated", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("step", "scan", "mix"):
        C = rng.choice([64, 128, 1024, 2048, 8 * _spread(rng, 1, 256), _spread(rng, 1, 2048)])
        if op == "step":
            B = _spread(rng, 1, 256)
            return dict(op=op, dtype=dtype, B=B, C=C, idle=rng.choice([0, 0, B // 8]))
        T = _spread(rng, 1, 17984)
        top = max(1, min(256, (33000000 if op == "scan" else 16000000) // (T * C)))
        if op == "mix":
            T = min(T, max(1, 16000000 // C))
        return dict(op=op, dtype=dtype, B=_spread(rng, 1, top), T=T, C=C, ragged=rng.random() < 0.4, state=rng.random() < 0.5)
    if op == "gated":
        grad = rng.random() < 0.5
        D = rng.choice([128, 1024, 2048, 8 * _spread(rng, 1, 256), _spread(rng, 1, 1024)])
        F = rng.choice([512, 4096, 8 * _spread(rng, 1, 1024), _spread(rng, 1, 4096)])
        most = (3.0e10 if dtype == "bf16" else 3.0e9) / (D * F)
        return dict(op=op, dtype=dtype, N=max(1, min(_spread(rng, 1, 8192), int(most))), D=D, F=F,
                    act=rng.choice(["silu", "silu", "gelu"]), grad=grad)
    D = rng.choice([64, 128, 512, 1024, 8 * rng.randint(2, 128), rng.randint(1, 200)])
    V = _spread(rng, 10, 131072)
    K = min(V, rng.choice([1, 8, 20, 64, rng.randint(1, 128)]))
    most = (2.0e11 if dtype == "bf16" else 6.0e10) / (V * D)
    return dict(op=op, dtype=dtype, N=max(1, min(_spread(rng, 1, 8192), int(most))), V=V, D=D, K=K,
                tau=rng.choice([1.0, 1.0, 2.0, 0.7]), grad=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ the inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        x = torch.randn(*shape, device="cuda", generator=g)
        return (x.mul_(std) if std != 1.0 else x).to(dtype)

    op = case["op"]
    s = dict(case)
    if op in ("step", "scan", "mix"):
        B, C = case["B"], case["C"]
        # half-open gates forget over 2 to 512 tokens
        s["rate"] = torch.exp2(-8.0 * torch.rand(C, device="cuda", generator=g))
    if op == "step":
        P = B + 3
        slots = torch.randperm(P, device="cuda", generator=g)[:B].to(torch.int32)
        if case["idle"]:  # rows of the batch that hold no request at the moment
            slots[torch.randperm(B, device="cuda", generator=g)[: case["idle"]]] = -1
        s.update(x=normal(B, C), decay=normal(B, C), gate=normal(B, C), slots=slots, pool=normal(P, C, dtype=torch.float32))
    elif op in ("scan", "mix"):
        T = case["T"]
        s.update(x=normal(B, T, C), decay=normal(B, T, C), gate=normal(B, T, C), s0=None, lengths=None)
        if case["state"]:
            s["s0"] = normal(B, C, dtype=torch.float32)
        if case["ragged"]:
            n = torch.randint(0, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
            n[0] = T
            s["lengths"] = n
        if op == "mix":
            s["do"] = normal(B, T, C)
            s["ds"] = normal(B, C, dtype=torch.float32) if case["state"] else None
    elif op == "gated":
        N, D, F = case["N"], case["D"], case["F"]
        s.update(x=normal(N, D), wg=normal(F, D, std=D**-0.5), wu=normal(F, D, std=D**-0.5))
        if case["grad"]:
            s["dh"] = normal(N, F)
    else:
        N, V, D, K = case["N"], case["V"], case["D"], case["K"]
        first = torch.randint(0, V, (N, 1), device="cuda", generator=g)
        gap = torch.randint(1, V // K + 1, (N, 1), device="cuda", generator=g)
        ids = (first + gap * torch.arange(K, device="cuda")) % V  # distinct within a row
        if N > 8:  # shorter lists, and positions of prompts and padding that have none
            ids[torch.rand(N, K, device="cuda", generator=g) < 0.05] = -1
            ids[torch.rand(N, device="cuda", generator=g) < 0.1] = -1
        s.update(hidden=normal(N, D), weight=normal(V, D, std=1.5 / math.sqrt(D)), ids=ids.to(torch.int32),
                 logits=normal(N, K, std=2.0, dtype=torch.float32) + 6.0)
        if case["grad"]:
            s["dloss"] = torch.full((N,), 1.0 / N, device="cuda")
    return s


# -------------------------------------------------------------------------------------------- the plain forms


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1 from zero, in log2(T) doublings."""
    T, d = a.shape[1], 1
    while d < T:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return a, b


def _gates(x, decay, gate, rate):
    """log a, a, sqrt(1 - a^2), both sigmoids, in 32 bits."""
    r, i = torch.sigmoid(decay.float()), torch.sigmoid(gate.float())
    log_a = -rate * r
    return log_a, torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a)), r, i


def _plain_recur(s, train):
    x, rate, s0, lengths = s["x"].float(), s["rate"], s["s0"], s["lengths"]
    B, T, C = x.shape
    log_a, a, m, r, i = _gates(x, s["decay"], s["gate"], rate)
    live = None
    if lengths is not None:
        live = (torch.arange(T, device=x.device) < lengths[:, None])[..., None]
        a, x, m = torch.where(live, a, 1.0), torch.where(live, x, 0.0), torch.where(live, m, 0.0)
    start = torch.zeros(B, C, device=x.device) if s0 is None else s0
    whole, h = _scan(a, m * i * x)
    h = h + whole * start[:, None]
    out = [(h if live is None else torch.where(live, h, 0.0)).to(s["x"].dtype)]
    if s["state"]:
        out.append(h[:, -1])
    if not train:
        return out
    do = s["do"].float()
    if live is not None:
        do = torch.where(live, do, 0.0)
    if s["state"]:
        do = torch.cat([do[:, :-1], do[:, -1:] + s["ds"][:, None]], 1)
    later = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _scan(later.flip(1), do.flip(1))[1].flip(1)
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    slope = torch.where(m > 0, a * a / torch.where(m > 0, m, 1.0), 0.0)
    dlog = g * (a * before - slope * i * x)
    dx, di = g * m * i, g * m * x * i * (1 - i)
    if live is not None:
        dlog = torch.where(live, dlog, 0.0)
    dr = dlog * -rate * r * (1 - r)
    out += [t.to(s["x"].dtype) for t in (dx, dr, di)] + [-(dlog * r).sum((0, 1))]
    if s["state"]:
        out.append(a[:, 0] * g[:, 0])
    return out


def _plain_step(s):
    pool, slots = s["pool"], s["slots"].long()
    _, a, m, _, i = _gates(s["x"], s["decay"], s["gate"], s["rate"])
    held = (slots >= 0)[:, None]
    at = slots.clamp(min=0)
    new = a * pool[at] + m * i * s["x"].float()
    spare = torch.cat([pool, torch.zeros_like(pool[:1])])  # idle rows write to a row of nobody
    spare[torch.where(slots < 0, pool.shape[0], slots)] = new
    pool.copy_(spare[:-1])
    return [torch.where(held, new, 0.0).to(s["x"].dtype), pool]


def _plain_gated(s):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.T, x @ wu.T
    if s["act"] == "silu":
        c = torch.sigmoid(g)
        act = g * c
    else:
        c = 0.5 * (1 + torch.erf(g * 0.5**0.5))
        act = g * c
    out = [(act * u).to(s["x"].dtype)]
    if s["grad"]:
        dh = s["dh"].float()
        slope = c * (1 + g * (1 - c)) if s["act"] == "silu" else c + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
        dg, du = dh * u * slope, dh * act
        out += [t.to(s["x"].dtype) for t in (dg @ wg + du @ wu, dg.T @ x, du.T @ x)]
    return out


def _plain_distill(s):
    h, w, ids, tau = s["hidden"].float(), s["weight"].float(), s["ids"].long(), s["tau"]
    there = ids >= 0
    live = there.any(1)
    pick = ids.clamp(min=0)
    t = torch.where(there, s["logits"] / tau, -math.inf)
    top = torch.where(live, t.amax(1), 0.0)[:, None]
    e = torch.exp(t - top)
    total = torch.where(live, e.sum(1), 1.0)[:, None]
    p = e / total
    log_p = torch.where(there, t - top - torch.log(total), 0.0)
    z = h @ w.T / tau
    most = z.amax(1, keepdim=True)
    lse = most + torch.log(torch.exp(z - most).sum(1, keepdim=True))
    out = [(p * (log_p - torch.where(there, z.gather(1, pick) - lse, 0.0))).sum(1)]
    if s["grad"]:
        g = torch.exp(z - lse)
        g.scatter_add_(1, pick, -p)
        g *= (torch.where(live, s["dloss"], 0.0) / tau)[:, None]
        out += [(g @ w).to(s["hidden"].dtype), (g.T @ h).to(s["weight"].dtype)]
    return out


# ------------------------------------------------------------------------------------------- the package's calls


def _own(s):
    import exponentially_weighted_signature_b200 as ews

    op = s["op"]
    if op == "step":
        return [ews.gated_recurrence_step(s["x"], s["decay"], s["gate"], s["rate"], s["pool"], slots=s["slots"]), s["pool"]]
    if op == "scan":
        with torch.no_grad():
            got = ews.gated_recurrence(s["x"], s["decay"], s["gate"], s["rate"], initial_state=s["s0"], lengths=s["lengths"],
                                       return_state=s["state"])
        return list(got) if s["state"] else [got]
    if op == "mix":
        x, decay, gate, rate = leaves = [s[n].detach().requires_grad_() for n in ("x", "decay", "gate", "rate")]
        if not s["state"]:
            o = ews.gated_recurrence(x, decay, gate, rate, lengths=s["lengths"])
            return [o.detach(), *torch.autograd.grad(o, leaves, s["do"])]
        leaves.append(s["s0"].detach().requires_grad_())
        o, end = ews.gated_recurrence(x, decay, gate, rate, initial_state=leaves[4], lengths=s["lengths"], return_state=True)
        return [o.detach(), end.detach(), *torch.autograd.grad((o, end), leaves, (s["do"], s["ds"]))]
    if op == "gated":
        if not s["grad"]:
            with torch.no_grad():
                return [ews.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"])]
        leaves = [s[n].detach().requires_grad_() for n in ("x", "wg", "wu")]
        o = ews.gated_linear(*leaves, activation=s["act"])
        return [o.detach(), *torch.autograd.grad(o, leaves, s["dh"])]
    if not s["grad"]:
        with torch.no_grad():
            return [ews.distill_loss(s["hidden"], s["weight"], s["ids"], s["logits"], temperature=s["tau"])]
    h, w = s["hidden"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
    loss = ews.distill_loss(h, w, s["ids"], s["logits"], temperature=s["tau"])
    return [loss.detach(), *torch.autograd.grad(loss, (h, w), s["dloss"])]


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "step":
        return _plain_step(state)
    if op in ("scan", "mix"):
        return _plain_recur(state, op == "mix")
    return _plain_gated(state) if op == "gated" else _plain_distill(state)


# ------------------------------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "step":
        return _exact_step(s)
    if op in ("scan", "mix"):
        return _exact_recur(s, op == "mix")
    return _exact_gated(s) if op == "gated" else _exact_distill(s)


def _exact_step(s):
    pool, out = s["pool"].double(), torch.zeros(s["B"], s["C"], dtype=torch.float64, device="cuda")
    for row, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            loss = -s["rate"].double() / (1 + torch.exp(-s["decay"][row].double()))
            share = 1 / (1 + torch.exp(-s["gate"][row].double()))
            pool[slot] = torch.exp(loss) * pool[slot] + (-torch.expm1(2 * loss)) ** 0.5 * share * s["x"][row].double()
            out[row] = pool[slot]
    return [out, pool]


def _exact_recur(s, train):
    """Token by token, forwards and back."""
    B, T, C = s["x"].shape
    f64, rate = torch.float64, s["rate"].double()
    h = torch.zeros(B, C, dtype=f64, device="cuda") if s["s0"] is None else s["s0"].double()
    out = torch.zeros(B, T, C, dtype=f64, device="cuda")
    n = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"]
    befores = torch.zeros_like(out) if train else None

    def token(t):
        x, r, i = (s[k][:, t].double() for k in ("x", "decay", "gate"))
        r, i = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
        return x, r, i, torch.exp(-rate * r), (-torch.expm1(-2 * rate * r)) ** 0.5, (t < n)[:, None]

    for t in range(T):
        if train:
            befores[:, t] = h
        x, r, i, a, m, live = token(t)
        h = torch.where(live, a * h + m * i * x, h)
        out[:, t] = torch.where(live, h, 0.0)
    res = [out] + ([h] if s["state"] else [])
    if not train:
        return res
    g = s["ds"].double() if s["state"] else torch.zeros(B, C, dtype=f64, device="cuda")
    dx, dr, di, drate = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out), torch.zeros(C, dtype=f64, device="cuda")
    for t in reversed(range(T)):
        x, r, i, a, m, live = token(t)
        here = torch.where(live, g + s["do"][:, t].double(), 0.0)
        # a = exp(-rate r), m = sqrt(1 - a^2): dm / d(rate r) = a^2 / m
        dp = here * (a * a / m * i * x - a * befores[:, t])
        dx[:, t] = here * m * i
        di[:, t] = here * m * x * i * (1 - i)
        dr[:, t] = dp * rate * r * (1 - r)
        drate += (dp * r).sum(0)
        g = torch.where(live, a * here, g)
    return res + [dx, dr, di, drate] + ([g] if s["state"] else [])


def _exact_gated(s):
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    grad = s["grad"]
    h = torch.empty(s["N"], s["F"], dtype=torch.float64, device="cuda")
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)
    for a in range(0, s["N"], 2048):
        rows = slice(a, a + 2048)
        g, u = x[rows] @ wg.mT, x[rows] @ wu.mT
        if s["act"] == "silu":
            e = torch.exp(-g)
            f, slope = g / (1 + e), 1 / (1 + e) + g * e / (1 + e) ** 2
        else:
            phi = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
            c = torch.special.erfc(-g / math.sqrt(2)) / 2
            f, slope = g * c, c + g * phi
        h[rows] = f * u
        if grad:
            dh = s["dh"][rows].double()
            dg, du = dh * u * slope, dh * f
            dx[rows] = dg @ wg + du @ wu
            dwg += dg.mT @ x[rows]
            dwu += du.mT @ x[rows]
    return [h, dx, dwg, dwu] if grad else [h]


def _exact_distill(s):
    h, w, tau = s["hidden"].double(), s["weight"].double(), s["tau"]
    loss = torch.zeros(s["N"], dtype=torch.float64, device="cuda")
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    rows_with = torch.nonzero((s["ids"] >= 0).any(1))[:, 0]
    for rows in rows_with.split(512):
        ids, t = s["ids"][rows].long(), s["logits"][rows].double() / tau
        p = torch.softmax(t.masked_fill(ids < 0, -math.inf), 1)
        target = torch.zeros(len(rows), s["V"] + 1, dtype=torch.float64, device="cuda")
        target.scatter_(1, torch.where(ids < 0, s["V"], ids), p)  # absent entries (of probability zero) to a column of nobody
        target = target[:, :-1]
        log_q = torch.log_softmax(h[rows] @ w.mT / tau, 1)
        loss[rows] = torch.special.xlogy(target, target).sum(1) - (target * log_q).sum(1)
        if s["grad"]:
            g = (log_q.exp_() - target) * (s["dloss"].double()[rows] / tau)[:, None]
            dh[rows] = g @ w
            dw += g.mT @ h[rows]
    return [loss, dh, dw] if s["grad"] else [loss]


# ------------------------------------------------------------------------------------------------ what a pass needs


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "step":
        rows, C = case["B"] - case["idle"], case["C"]
        return {"bytes": rows * (8 * C + 4 * e * C + 4) + 4 * C, "flops": 20 * rows * C}
    if op in ("scan", "mix"):
        n, state = case["B"] * case["T"] * case["C"], 4 * case["B"] * case["C"] if case["state"] else 0
        if op == "scan":
            return {"bytes": 4 * e * n + 2 * state + 4 * case["C"], "flops": 20 * n}
        return {"bytes": 8 * e * n + 4 * state + 8 * case["C"], "flops": 60 * n}
    if op == "gated":
        N, D, F = case["N"], case["D"], case["F"]
        once = N * D + 2 * F * D + N * F
        return {"bytes": e * once * (2 if case["grad"] else 1), "flops": (12 if case["grad"] else 4) * N * D * F}
    N, V, D, K, grad = case["N"], case["V"], case["D"], case["K"], case["grad"]
    return {"bytes": e * (N + V) * D * (2 if grad else 1) + 8 * N * K + (8 if grad else 4) * N, "flops": (6 if grad else 2) * N * V * D}
