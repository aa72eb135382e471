"""The token model: the operators together, in training, over prompts and token by token."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ews():
    import exponentially_weighted_signature_b200 as e

    return e


@pytest.mark.parametrize("dtype,mixers", [(torch.float32, ("decay", "decay")), (torch.bfloat16, ("decay",)), (torch.float32, ("ews", "decay"))])
def test_training_steps_learn_a_repeated_sequence(ews, dtype, mixers):
    torch.manual_seed(0)
    kw = dict(m=8, n=2, series_q=4, clock_norm_constant=96.0, dropout_rate=0.0) if "ews" in mixers else None
    model = ews.TokenModel(61, hidden_dim=64, heads=4, kv_heads=2, mixers=mixers, ews_kwargs=kw).cuda().to(dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 61, (4, 24), device="cuda", generator=g).repeat(1, 4)
    targets = torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], -100)], 1)
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(30):
        opt.zero_grad()
        loss = model.loss(ids, targets)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    assert losses[-1] < 0.6 * losses[0], losses


def test_gradients_match_plain_operations(ews):
    """The float32 model's gradients against the same model in float64 with torch operations in the operators' places."""
    torch.manual_seed(0)
    model = ews.TokenModel(50, hidden_dim=32, heads=2, mixers=("decay",)).cuda()
    ids = torch.randint(0, 50, (2, 37), device="cuda")
    targets = torch.randint(0, 50, (2, 37), device="cuda")
    lengths = torch.tensor([37, 20], device="cuda", dtype=torch.int32)
    targets[1, 20:] = -100
    loss = model.loss(ids, targets, lengths)
    grads = torch.autograd.grad(loss, list(model.parameters()))

    import copy

    ref = copy.deepcopy(model).double()
    block = ref.blocks[0]
    x = ref.table[ids] * 32**0.5
    q, k, v = block._heads(x)
    t = torch.arange(37, device="cuda")
    gap = t[:, None] - t[None, :]
    w = torch.exp(-block.rate.double()[:, None, None] * gap.clamp(min=0)) * (gap >= 0)
    p = torch.einsum("bihd,bjhd->bhij", q, k) * w * (t < lengths[:, None])[:, None, None]
    o = torch.einsum("bhij,bjhd->bihd", p, v) * block.head_dim**-0.5
    o = o * (t < lengths[:, None])[..., None, None]
    h = ref.norm(block._close(x, o))
    want = torch.nn.functional.cross_entropy((h @ ref.table.T).flatten(0, 1), targets.flatten(), ignore_index=-100)
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    for a, b in zip(grads, torch.autograd.grad(want, list(ref.parameters()))):
        assert float((a.double() - b).abs().max()) <= 2e-5 * float(b.abs().max())


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 6e-2)])
def test_prompt_and_steps_follow_the_whole_sequence(ews, dtype, tol):
    """Prompts of two lengths, then tokens one by one on pooled states in another order: the logits of the model run over
    the whole sequence. tol: float32 through two blocks; bfloat16 keeps 8 bits through some ten rounded layers."""
    torch.manual_seed(0)
    model = ews.TokenModel(97, hidden_dim=128, heads=4, mixers=("decay", "decay")).cuda().to(dtype)
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


def test_serving_needs_attention_blocks(ews):
    model = ews.TokenModel(20, hidden_dim=32, heads=2, mixers=("ews",), ews_kwargs=dict(m=4)).cuda()
    with pytest.raises(NotImplementedError):
        model.states(2)
    with pytest.raises(ValueError):
        ews.TokenModel(20, mixers=("other",))
