"""CPU tests of what the token operators and their model promise: derivatives, constants of the heads, seeds."""

import pytest
import torch

from exponentially_weighted_signature_b200 import engine


class _Square(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y):
        ctx.save_for_backward(x)
        return x * x + y.detach()

    @staticmethod
    @engine.first_order
    def backward(ctx, g):
        return 2 * g * ctx.saved_tensors[0], None


@pytest.mark.parametrize("power", [1, 2])
def test_a_first_order_gradient_is_a_number_and_no_more(power):
    """power 1: the cotangent is a constant; 2: it depends on the result."""
    x, y = torch.tensor([1.0, -3.0], requires_grad=True), torch.tensor([0.0, 1.0], requires_grad=True)
    plain = torch.autograd.grad((_Square.apply(x, y) ** power).sum(), x)[0]
    assert not plain.requires_grad
    grad = torch.autograd.grad((_Square.apply(x, y) ** power).sum(), x, create_graph=True)[0]
    assert torch.equal(grad.detach(), plain)
    with pytest.raises(RuntimeError, match="second derivative"):
        (grad.sum() + x.sum()).backward()
    with torch.no_grad():
        grad.mul_(2)
    assert torch.equal(grad.detach(), 2 * plain)
