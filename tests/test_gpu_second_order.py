"""The engines build first derivatives: a gradient taken with create_graph has the usual value, and a term that
differentiates it again raises instead of losing the engine's part."""

import pytest
import torch
from test_gpu_graph import _inputs, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,N", [("diag", 16), ("diag_clock", 8), ("logews", 8), ("dense", 32), ("block", 8)])
@pytest.mark.parametrize("power", [1, 2])
def test_engine_gradients_are_first_order(kind, N, power):
    from exponentially_weighted_signature_b200.layer import configure

    layer = _layer(kind, N).cuda()
    path, clock, lift = (x.cuda() for x in _inputs(1, 2, 40, 4, N))
    lift = torch.nn.Parameter(lift)
    path.requires_grad_()
    leaves = [path, lift, *layer.parameters()]
    configure(deterministic=True)  # the two gradients below are compared bit for bit
    try:
        f = lambda: (layer(path, clock, readout="terminal", lift=lift) ** power).sum()  # noqa: E731
        plain = torch.autograd.grad(f(), leaves)
        grads = torch.autograd.grad(f(), leaves, create_graph=True)
    finally:
        configure(deterministic=False)
    for a, b in zip(plain, grads):
        assert torch.equal(a, b.detach())
    with pytest.raises(RuntimeError, match="second derivative"):
        (sum((g**2).sum() for g in grads) + (lift**2).sum()).backward()


def test_block_gradients_are_first_order():
    from exponentially_weighted_signature_b200.block import StackedEWS

    torch.manual_seed(0)
    model = StackedEWS(1, 5, 16, 5, block_kwargs=dict(m=4, n=2, series_q=6, clock_norm_constant=24.0, dropout_rate=0.0)).cuda()
    x = torch.randn(2, 24, 5, device="cuda")
    grads = torch.autograd.grad(model(x).square().mean(), list(model.parameters()), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        sum((g**2).sum() for g in grads).backward()
