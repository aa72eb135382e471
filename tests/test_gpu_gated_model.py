"""The token model with gated blocks: the operators together, in training, from a teacher, over prompts and token by token."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


def _plain_hidden(model, ids, lengths):
    """The model's hidden rows in torch operations (gated blocks), in its parameters' type."""
    x = model.table[ids] * model.hidden_dim**0.5
    for block in model.blocks:
        u, decay, gate, rate = block._mixer(x)
        rate = torch.exp(block.log_rate)
        p = rate * torch.sigmoid(decay)
        a, b = torch.exp(-p), torch.sqrt(-torch.expm1(-2 * p)) * torch.sigmoid(gate) * u
        h, out = torch.zeros_like(x[:, 0, : block.width]) if block.width <= x.shape[-1] else None, []
        for t in range(x.shape[1]):
            h = a[:, t] * h + b[:, t]
            out.append(h * (t < lengths)[:, None])
        x = x + block.out(torch.stack(out, 1))
        y = block.norm2(x)
        x = x + block.ff_down(torch.nn.functional.silu(block.ff_gate(y)) * block.ff_up(y))
    return model.norm(x)


@pytest.mark.parametrize("what", ["loss", "distill"])
def test_gradients_match_plain_operations(ews, what):
    """The float32 model's gradients against the same model in float64 with torch operations in the operators' places, to the
    float32 roundings of some ten layers (2e-5 of the largest, as for the decayed attention's model)."""
    torch.manual_seed(0)
    model = ews.TokenModel(50, hidden_dim=32, mixers=("gated", "gated"), gated_kwargs=dict(width=24, ff_dim=40)).cuda()
    ids = torch.randint(0, 50, (2, 37), device="cuda")
    lengths = torch.tensor([37, 20], device="cuda", dtype=torch.int32)
    ref = copy.deepcopy(model).double()
    h = _plain_hidden(ref, ids, lengths)
    logits = h @ ref.table.T
    if what == "loss":
        targets = torch.randint(0, 50, (2, 37), device="cuda")
        targets[1, 20:] = -100
        loss = model.loss(ids, targets, lengths)
        want = torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(), ignore_index=-100)
    else:
        teacher_logits, teacher_ids = (torch.randn(2, 37, 50, device="cuda") * 3).topk(8)
        teacher_ids[1, 20:] = -1
        loss = model.distill(ids, teacher_ids, teacher_logits, lengths, temperature=2.0)
        p = torch.softmax(teacher_logits.double() / 2, -1)
        log_q = torch.log_softmax(logits / 2, -1).gather(-1, teacher_ids.clamp(min=0))
        kl = (p * (p.log() - log_q)).sum(-1) * (teacher_ids[..., 0] >= 0)
        want = 4 * kl.sum() / 57
    grads = torch.autograd.grad(loss, list(model.parameters()))
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
    for a, b in zip(grads, torch.autograd.grad(want, list(ref.parameters()))):
        assert float((a.double() - b).abs().max()) <= 2e-5 * float(b.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_student_trains_on_a_teacher(ews, dtype):
    """A wider teacher's top logits, a gated student: steps run, gradients are there for every parameter and are finite."""
    torch.manual_seed(0)
    teacher = ews.TokenModel(61, hidden_dim=64, heads=4, mixers=("decay", "gated")).cuda().to(dtype)
    student = ews.TokenModel(61, hidden_dim=32, mixers=("gated",)).cuda().to(dtype)
    ids = torch.randint(0, 61, (4, 50), device="cuda")
    with torch.no_grad():
        top = (teacher.hidden(ids) @ teacher.table.T).topk(8)
    opt = torch.optim.Adam(student.parameters(), lr=1e-3)
    for _ in range(3):
        opt.zero_grad()
        loss = student.distill(ids, top.indices, top.values, temperature=2.0) + student.loss(ids[:, :-1], ids[:, 1:])
        loss.backward()
        assert torch.isfinite(loss) and all(p.grad is not None and torch.isfinite(p.grad).all() for p in student.parameters())
        opt.step()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 6e-2)])
@pytest.mark.parametrize("mixers", [("gated", "gated"), ("gated", "decay")])
def test_prompt_and_steps_follow_the_whole_sequence(ews, dtype, tol, mixers):
    """Prompts of two lengths, then tokens one by one on pooled states in another order: the logits of the model run over
    the whole sequence. tol: float32 through two blocks; bfloat16 keeps 8 bits through some ten rounded layers."""
    torch.manual_seed(0)
    model = ews.TokenModel(97, hidden_dim=128, heads=4, mixers=mixers).cuda().to(dtype)
    ids = torch.randint(0, 97, (2, 150), device="cuda")
    with torch.no_grad():
        whole = (model.hidden(ids) @ model.table.T).float()
    lengths = torch.tensor([140, 131], device="cuda", dtype=torch.int32)
    logits, states = model.prompt(ids[:, :140], lengths)
    pools = model.states(5)
    slots = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    for pool, s in zip(pools, states):
        pool[slots.long()] = s
    for b in range(2):
        assert float((logits[b].float() - whole[b, lengths[b] - 1]).abs().max()) <= tol * float(whole[b].abs().max())
    for i in range(10):
        at = lengths.long() + i
        got = model.step(ids[torch.arange(2, device="cuda"), at], pools, slots).float()
        for b in range(2):
            assert float((got[b] - whole[b, at[b]]).abs().max()) <= tol * float(whole[b].abs().max()), (i, b)
    assert all((pool[[0, 2, 4]] == 0).all() for pool in pools)


def test_a_step_in_a_graph(ews):
    """The serving loop of a gated model as one graph, replayed on new tokens."""
    torch.manual_seed(0)
    model = ews.TokenModel(97, hidden_dim=64, mixers=("gated", "gated")).cuda().bfloat16()
    pools, eager = model.states(4), model.states(4)
    ids, slots = torch.tensor([5, 9, 11], device="cuda"), torch.tensor([2, -1, 0], device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.step(ids, [p.clone() for p in pools], slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.step(ids, pools, slots)
    for p in pools:
        p.zero_()
    for tokens in ([5, 9, 11], [1, 2, 3], [96, 0, 50]):
        ids.copy_(torch.tensor(tokens, device="cuda"))
        graph.replay()
        assert torch.equal(logits, model.step(ids, eager, slots))
    assert all(torch.equal(a, b) for a, b in zip(pools, eager))
