"""The token operators as their users call them: decayed linear attention (prompts, training, single tokens), the
token embedding with its gradient, and the loss over a large vocabulary with its gradients.

``run`` makes one pass, in plain torch operations (``own = False``) or through the package (``own = True``);
``exact`` evaluates the definitions in 64 bits.
"""

import math

import torch

own = False

CHUNK = 64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # one conversation's next token: latency
        dict(name="step-one", op="step", dtype="bf16", B=1, H=8, Hk=8, dk=64, dv=64, idle=0),
        # a full serving batch over a pool of states, some rows idle
        dict(name="step-batch", op="step", dtype="bf16", B=256, H=16, Hk=16, dk=128, dv=128, idle=5),
        # a batch of short odd prompts with shared key/value heads, float32 as the EWS layers train and serve
        dict(name="prompt-short", op="scan", dtype="f32", B=48, T=37, H=8, Hk=2, dk=48, dv=80, ragged=True, state=True),
        # one long prompt, handed over to the step as a state: few rows, long axis
        dict(name="prompt-long", op="scan", dtype="bf16", B=1, T=17984, H=16, Hk=16, dk=128, dv=128, ragged=False, state=True),
        # an ordinary training batch
        dict(name="mix-train", op="mix", dtype="bf16", B=8, T=2048, H=16, Hk=16, dk=128, dv=128, ragged=False, state=False),
        # float32 training at the stacked model's length: ragged, shared heads, carried state with its gradient
        dict(name="mix-train-f32", op="mix", dtype="f32", B=16, T=1440, H=8, Hk=4, dk=64, dv=64, ragged=True, state=True),
        # the ids of one serving step
        dict(name="embed-step", op="embed", dtype="bf16", N=128, V=32000, D=1024, grad=False),
        # a training batch, natural token frequencies, odd vocabulary
        dict(name="embed-train", op="embed", dtype="bf16", N=16384, V=50257, D=768, grad=True),
        # a large training batch in float32
        dict(name="embed-train-f32", op="embed", dtype="f32", N=65536, V=131072, D=512, grad=True),
        # the stacked model's width with a small vocabulary, float32
        dict(name="loss-small-f32", op="loss", dtype="f32", N=1440, V=1000, D=128, grad=True),
        # an ordinary training batch, odd vocabulary
        dict(name="loss-train", op="loss", dtype="bf16", N=8192, V=50257, D=1024, grad=True),
        # scoring with a large vocabulary
        dict(name="loss-score", op="loss", dtype="bf16", N=4096, V=131072, D=2048, grad=False),
    ]


def _spread(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["step", "scan", "mix", "embed", "loss"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("step", "scan", "mix"):
        Hk = rng.choice([1, 2, 4, 8, 16])
        H = Hk * rng.choice([1, 1, 2, 4]) if Hk <= 4 else Hk
        dk = rng.choice([16, 32, 64, 128, 8 * rng.randint(1, 16), rng.randint(1, 128)])
        dv = rng.choice([dk, dk, 64, 128, 8 * rng.randint(1, 16), rng.randint(1, 128)])
        case = dict(op=op, dtype=dtype, H=H, Hk=Hk, dk=dk, dv=dv)
        if op == "step":
            B = _spread(rng, 1, 256)
            return dict(case, B=B, idle=rng.choice([0, 0, B // 8]))
        T = _spread(rng, 1, 17984)
        top = max(1, min(64, (32768 if op == "scan" else 16384) // T))
        return dict(case, B=_spread(rng, 1, top), T=T, ragged=rng.random() < 0.4, state=rng.random() < 0.5)
    if op == "embed":
        return dict(op=op, dtype=dtype, N=_spread(rng, 1, 65536), V=_spread(rng, 100, 131072),
                    D=rng.choice([64, 128, 512, rng.randint(1, 512), 8 * rng.randint(1, 64)]), grad=rng.random() < 0.75)
    grad = rng.random() < 0.7
    D = rng.choice([64, 128, 512, 1024, 8 * rng.randint(2, 128), rng.randint(1, 200)])
    V = _spread(rng, 10, 131072)
    most = 3.0e11 if dtype == "bf16" else 1.0e11
    return dict(op=op, dtype=dtype, N=max(1, min(_spread(rng, 1, 8192), int(most / (V * D)))), V=V, D=D, grad=grad)


# ------------------------------------------------------------------------------------------------ the inputs


def _rates(H):
    """Windows from 2 to 512 tokens over the heads."""
    return torch.exp2(-torch.linspace(1.0, 9.0, H, device="cuda")) if H > 1 else torch.full((1,), 2.0**-5, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        x = torch.randn(*shape, device="cuda", generator=g)
        return (x.mul_(std) if std != 1.0 else x).to(dtype)

    op = case["op"]
    s = dict(case)
    if op == "step":
        B, H, Hk, dk, dv = (case[n] for n in ("B", "H", "Hk", "dk", "dv"))
        P = B + 3
        slots = torch.randperm(P, device="cuda", generator=g)[:B].to(torch.int32)
        if case["idle"]:  # rows of the batch that hold no request at the moment
            slots[torch.randperm(B, device="cuda", generator=g)[: case["idle"]]] = -1
        s.update(q=normal(B, H, dk), k=normal(B, Hk, dk), v=normal(B, Hk, dv), rate=_rates(H), slots=slots,
                 pool=normal(P, H, dk, dv, dtype=torch.float32))
    elif op in ("scan", "mix"):
        B, T, H, Hk, dk, dv = (case[n] for n in ("B", "T", "H", "Hk", "dk", "dv"))
        s.update(q=normal(B, T, H, dk), k=normal(B, T, Hk, dk), v=normal(B, T, Hk, dv), rate=_rates(H), s0=None, lengths=None)
        if case["state"]:
            s["s0"] = normal(B, H, dk, dv, dtype=torch.float32)
        if case["ragged"]:
            n = torch.randint(0, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
            n[0] = T
            s["lengths"] = n
        if op == "mix":
            s["do"] = normal(B, T, H, dv)
            s["ds"] = normal(B, H, dk, dv, dtype=torch.float32) if case["state"] else None
    elif op == "embed":
        N, V, D = case["N"], case["V"], case["D"]
        u = torch.rand(N, device="cuda", generator=g, dtype=torch.float64)
        rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)  # frequencies near 1 / rank
        s.update(ids=torch.randperm(V, device="cuda", generator=g)[rank], table=normal(V, D, std=0.02), scale=math.sqrt(D))
        if case["grad"]:
            s["dout"] = normal(N, D)
    else:
        N, V, D = case["N"], case["V"], case["D"]
        t = torch.randint(0, V, (N,), device="cuda", generator=g)
        if N > 8:  # positions of prompts and padding carry no loss
            t[torch.rand(N, device="cuda", generator=g) < 0.1] = -100
        s.update(hidden=normal(N, D), weight=normal(V, D, std=1.5 / math.sqrt(D)), targets=t)
        if case["grad"]:
            s["dloss"] = torch.full((N,), 1.0 / N, device="cuda")
    return s


# -------------------------------------------------------------------------------------------- the plain forms


def _chain(q, k, v, rate, s0):
    """o_t = q_t S_t, S_t = g S_{t-1} + k_t v_t^T over (B, H, T, d), in chunks joined by a matrix of decays."""
    B, H, T, dk = q.shape
    n, dv = -(-T // CHUNK), v.shape[-1]
    if n * CHUNK > T:
        q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - T)) for x in (q, k, v))
    q, k, v = (x.reshape(B, H, n, CHUNK, -1) for x in (q, k, v))
    i = torch.arange(CHUNK, device=q.device)
    r = rate[:, None, None]
    gap = i[:, None] - i[None, :]
    inside = torch.where(gap >= 0, torch.exp(-r * gap.clamp(min=0)), torch.zeros((), device=q.device))
    o = ((q @ k.mT) * inside[:, None]) @ v
    add = (k * torch.exp(-rate[:, None] * (CHUNK - 1 - i))[:, None, :, None]).mT @ v
    c = torch.arange(n, device=q.device)
    gap = (c[:, None] - 1 - c[None, :]) * CHUNK
    join = torch.where(gap >= 0, torch.exp(-r * gap.clamp(min=0)), torch.zeros((), device=q.device))
    state = (join @ add.reshape(B, H, n, dk * dv)).reshape(B, H, n, dk, dv)
    if s0 is not None:
        state = state + torch.exp(-rate[:, None] * (c * CHUNK))[:, :, None, None] * s0[:, :, None]
    o = o + torch.exp(-rate[:, None] * (i + 1))[:, None, :, None] * (q @ state)
    return o.reshape(B, H, n * CHUNK, dv)[:, :, :T]


def _heads(x, H):
    """(B, T, Hk, d) of any type to (B, H, T, d) in 32 bits, each shared head repeated for its group."""
    x = x.float().transpose(1, 2)
    return x.repeat_interleave(H // x.shape[1], 1)


def _plain_mix(s, train):
    B, T, H, dk = s["q"].shape
    rate, s0, scale = s["rate"], s["s0"], s["dk"] ** -0.5
    q, k, v = (_heads(s[n], H) for n in ("q", "k", "v"))
    live, end = None, torch.full((B, 1, 1), float(T), device=q.device)
    t = torch.arange(T, device=q.device)
    if s["lengths"] is not None:
        end = s["lengths"].float()[:, None, None]
        live = (t < s["lengths"][:, None])[:, None, :, None]
        q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    dt = s["q"].dtype
    out = [(_chain(q, k, v, rate, s0) * scale).transpose(1, 2).to(dt)]
    r = rate[None, :, None]
    to_end = torch.exp(-r * (end - 1 - t).clamp(min=0))[..., None]  # the weight of token t in the last state
    whole = torch.exp(-r * end)[..., None]
    if s["state"]:
        out.append(whole * s0 + (k * to_end).mT @ v)
    if not train:
        return out
    do = s["do"].float().transpose(1, 2)
    if live is not None:
        do = torch.where(live, do, 0.0)
    do = do * scale
    dq = _chain(do, v, k, rate, None if s0 is None else s0.mT)
    back = [x.flip(2) for x in (q, k, v, do)]
    dk = _chain(back[2], back[3], back[0], rate, None).flip(2)
    dv = _chain(back[1], back[0], back[3], rate, None).flip(2)
    if s["state"]:
        dk = dk + to_end * (v @ s["ds"].mT)
        dv = dv + to_end * (k @ s["ds"])
    if live is not None:
        dq, dk, dv = (torch.where(live, x, 0.0) for x in (dq, dk, dv))
    Hk = s["Hk"]
    dk, dv = (x.reshape(B, Hk, H // Hk, T, -1).sum(2) for x in (dk, dv))
    out += [x.transpose(1, 2).to(dt) for x in (dq, dk, dv)]
    if s["state"]:
        out.append((q * torch.exp(-r * (t + 1))[..., None]).mT @ do + whole * s["ds"])
    return out


def _plain_step(s):
    pool, slots, H = s["pool"], s["slots"].long(), s["H"]
    B, P = slots.numel(), pool.shape[0]
    g = torch.exp(-s["rate"])
    q = s["q"].float()
    k, v = (s[n].float().repeat_interleave(H // s["Hk"], 1) for n in ("k", "v"))
    owner = torch.full((P + 1,), -1, device=pool.device)  # which row each state belongs to
    owner[torch.where(slots < 0, P, slots)] = torch.arange(B, device=pool.device)
    owner = owner[:P]
    held = (owner >= 0)[:, None]
    row = owner.clamp(min=0)
    pool.mul_(torch.where(held, g, 1.0)[:, :, None, None])
    pool.add_(torch.where(held[..., None], k[row], 0.0)[..., None] * v[row][:, :, None, :])
    o = (q[:, :, None, :] @ pool[slots.clamp(min=0)])[:, :, 0] * s["dk"] ** -0.5
    return [torch.where((slots >= 0)[:, None, None], o, 0.0).to(s["q"].dtype), pool]


def _plain_embed(s):
    out = [(s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)]
    if s["grad"]:
        d = torch.zeros(s["table"].shape, device="cuda")
        d.index_add_(0, s["ids"], s["dout"].float())
        out.append((d * s["scale"]).to(s["table"].dtype))
    return out


def _plain_loss(s):
    h, w, t = s["hidden"].float(), s["weight"].float(), s["targets"]
    live = t >= 0
    pick = t.clamp(min=0)[:, None]
    logits = h @ w.T
    top = logits.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    out = [torch.where(live, (lse - logits.gather(1, pick))[:, 0], 0.0)]
    if s["grad"]:
        g = torch.exp(logits - lse)
        g.scatter_add_(1, pick, torch.full_like(pick, -1.0, dtype=torch.float32))
        g *= torch.where(live, s["dloss"], 0.0)[:, None]
        out += [(g @ w).to(s["hidden"].dtype), (g.T @ h).to(s["weight"].dtype)]
    return out


# ------------------------------------------------------------------------------------------- the package's calls


def _own(s):
    import exponentially_weighted_signature_b200 as ews

    op = s["op"]
    if op == "step":
        return [ews.decayed_attention_step(s["q"], s["k"], s["v"], s["rate"], s["pool"], slots=s["slots"]), s["pool"]]
    if op == "scan":
        with torch.no_grad():
            got = ews.decayed_attention(s["q"], s["k"], s["v"], s["rate"], initial_state=s["s0"], lengths=s["lengths"],
                                        return_state=s["state"])
        return list(got) if s["state"] else [got]
    if op == "mix":
        q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
        if not s["state"]:
            o = ews.decayed_attention(q, k, v, s["rate"], lengths=s["lengths"])
            return [o.detach(), *torch.autograd.grad(o, (q, k, v), s["do"])]
        s0 = s["s0"].detach().requires_grad_()
        o, end = ews.decayed_attention(q, k, v, s["rate"], initial_state=s0, lengths=s["lengths"], return_state=True)
        return [o.detach(), end.detach(), *torch.autograd.grad((o, end), (q, k, v, s0), (s["do"], s["ds"]))]
    if op == "embed":
        if not s["grad"]:
            with torch.no_grad():
                return [ews.token_embedding(s["ids"], s["table"], scale=s["scale"])]
        table = s["table"].detach().requires_grad_()
        o = ews.token_embedding(s["ids"], table, scale=s["scale"])
        return [o.detach(), *torch.autograd.grad(o, (table,), s["dout"])]
    if not s["grad"]:
        with torch.no_grad():
            return [ews.vocab_loss(s["hidden"], s["weight"], s["targets"])]
    h, w = s["hidden"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
    loss = ews.vocab_loss(h, w, s["targets"])
    return [loss.detach(), *torch.autograd.grad(loss, (h, w), s["dloss"])]


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "step":
        return _plain_step(state)
    if op in ("scan", "mix"):
        return _plain_mix(state, op == "mix")
    return _plain_embed(state) if op == "embed" else _plain_loss(state)


# ------------------------------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "step":
        return _exact_step(s)
    if op in ("scan", "mix"):
        return _exact_mix(s, op == "mix")
    if op == "embed":
        table, ids = s["table"].double(), s["ids"]
        out = [s["scale"] * table[ids]]
        if case["grad"]:
            order = ids.argsort()
            total = torch.cat([torch.zeros_like(s["dout"][:1]).double(), s["dout"].double()[order].cumsum(0)])
            edge = torch.searchsorted(ids[order], torch.arange(case["V"] + 1, device="cuda"))
            out.append(s["scale"] * (total[edge[1:]] - total[edge[:-1]]))
        return out
    h, w, t = s["hidden"].double(), s["weight"].double(), s["targets"]
    loss = torch.zeros(case["N"], dtype=torch.float64, device="cuda")
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for a in range(0, case["N"], 512):
        b = min(a + 512, case["N"])
        rows = torch.nonzero(t[a:b] >= 0)[:, 0] + a
        z = h[rows] @ w.T
        p = torch.log_softmax(z, 1)
        at = t[rows][:, None]
        loss[rows] = -p.gather(1, at)[:, 0]
        if case["grad"]:
            p = p.exp_()
            p[torch.arange(len(rows), device="cuda"), at[:, 0]] -= 1
            p *= s["dloss"].double()[rows][:, None]
            dh[rows] = p @ w
            dw += p.T @ h[rows]
    return [loss, dh, dw] if case["grad"] else [loss]


def _exact_step(s):
    pool, scale = s["pool"].double(), s["dk"] ** -0.5
    out = torch.zeros(s["B"], s["H"], s["dv"], dtype=torch.float64, device="cuda")
    group = s["H"] // s["Hk"]
    g = torch.exp(-s["rate"].double())[:, None, None]
    for row, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            k, v = (s[n][row].double().repeat_interleave(group, 0) for n in ("k", "v"))
            pool[slot] = g * pool[slot] + torch.einsum("hi,hj->hij", k, v)
            out[row] = scale * torch.einsum("hi,hij->hj", s["q"][row].double(), pool[slot])
    return [out, pool]


def _exact_mix(s, train):
    """The sums over all pairs of tokens, a block of rows at a time."""
    B, T, H, dk = s["q"].shape
    Hk, dv, f64 = s["Hk"], s["dv"], torch.float64
    scale, rate, group = dk**-0.5, s["rate"].double()[:, None, None], H // Hk
    out = torch.zeros(B, T, H, dv, dtype=f64, device="cuda")
    end = s["s0"].double().clone() if s["state"] else None
    grads = [torch.zeros(x.shape, dtype=f64, device="cuda") for x in (s["q"], s["k"], s["v"])] if train else []
    d0 = s["ds"].double().clone() if train and s["state"] else None
    for b in range(B):
        n = T if s["lengths"] is None else int(s["lengths"][b])
        if not n:
            continue
        q = s["q"][b, :n].double().transpose(0, 1)
        k, v = (s[x][b, :n].double().transpose(0, 1).repeat_interleave(group, 0) for x in ("k", "v"))
        t = torch.arange(n, device="cuda", dtype=f64)
        o = torch.zeros(H, n, dv, dtype=f64, device="cuda")
        if train:
            do = scale * s["do"][b, :n].double().transpose(0, 1)
            dq, gk, gv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        block = max(1, min(n, (1 << 26) // (H * n)))
        for a in range(0, n, block):
            e = min(a + block, n)
            gap = t[a:e, None] - t[None, :e]
            w = torch.exp(-rate * gap.clamp(min=0)).masked_fill_(gap < 0, 0.0)
            p = (q[:, a:e] @ k[:, :e].mT).mul_(w)
            o[:, a:e] = p @ v[:, :e]
            if train:
                gv[:, :e] += p.mT @ do[:, a:e]
                p = (do[:, a:e] @ v[:, :e].mT).mul_(w)
                dq[:, a:e] = p @ k[:, :e]
                gk[:, :e] += p.mT @ q[:, a:e]
        if s["state"]:
            first = torch.exp(-rate * (t + 1)[:, None])
            last = torch.exp(-rate * (n - 1 - t)[:, None])
            o += first * (q @ s["s0"][b].double())
            end[b] = torch.exp(-rate * n) * s["s0"][b].double() + (k * last).mT @ v
            if train:
                ds = s["ds"][b].double()
                dq += first * (do @ s["s0"][b].double().mT)
                gk += last * (v @ ds.mT)
                gv += last * (k @ ds)
                d0[b] = torch.exp(-rate * n) * ds + (first * q).mT @ do
        out[b, :n] = scale * o.transpose(0, 1)
        if train:
            grads[0][b, :n] = dq.transpose(0, 1)
            grads[1][b, :n] = gk.reshape(Hk, group, n, dk).sum(1).transpose(0, 1)
            grads[2][b, :n] = gv.reshape(Hk, group, n, dv).sum(1).transpose(0, 1)
    return [out] + ([end] if s["state"] else []) + grads + ([d0] if d0 is not None else [])


# ------------------------------------------------------------------------------------------------ what a pass needs


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "step":
        B, H, Hk, dk, dv = (case[n] for n in ("B", "H", "Hk", "dk", "dv"))
        B -= case["idle"]
        return {"bytes": B * (8 * H * dk * dv + e * (H * (dk + dv) + Hk * (dk + dv)) + 4) + 4 * H, "flops": 4 * B * H * dk * dv}
    if op in ("scan", "mix"):
        B, T, H, Hk, dk, dv = (case[n] for n in ("B", "T", "H", "Hk", "dk", "dv"))
        q, k, v, o = H * dk, Hk * dk, Hk * dv, H * dv
        state = 4 * B * H * dk * dv if case["state"] else 0
        tokens = B * T
        if op == "scan":
            return {"bytes": e * tokens * (q + k + v + o) + 2 * state, "flops": 4 * tokens * H * dk * dv}
        return {"bytes": e * tokens * (2 * q + 2 * k + 2 * v + 2 * o) + 4 * state, "flops": 12 * tokens * H * dk * dv}
    N, V, D = case["N"], case["V"], case["D"]
    if op == "embed":
        return {"bytes": 8 * N + 2 * e * N * D + (e * (N + V) * D if case["grad"] else 0), "flops": (2 if case["grad"] else 1) * N * D}
    grad = case["grad"]
    return {"bytes": e * (N + V) * D * (2 if grad else 1) + 12 * N + (4 * N if grad else 0), "flops": (6 if grad else 2) * N * V * D}
