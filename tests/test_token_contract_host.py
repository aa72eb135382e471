"""CPU tests of what the token operators and their model promise: derivatives, constants of the heads, seeds."""

import pytest
import torch

from exponentially_weighted_signature_b200 import _lib, engine, token_ops


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


def _block(heads=6):
    from exponentially_weighted_signature_b200 import DecayBlock

    return DecayBlock(heads * 4, heads)


def test_rates_are_the_same_in_every_type():
    want = torch.exp2(-torch.linspace(1.0, 9.0, 6))
    block = _block()
    assert torch.equal(block.rate, want)
    for cast in (lambda m: m.bfloat16(), lambda m: m.float(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.bfloat16)):
        cast(block)
        assert block.rate.dtype == torch.float32 and torch.equal(block.rate, want)
    assert block.qkv.weight.dtype == torch.bfloat16 and block._buffers["rate"] is block.rate
    assert torch.equal(torch.nn.Sequential(_block()).bfloat16()[0].rate, want)


def test_rates_that_were_set_are_kept():
    block = _block()
    block.rate.mul_(0.3)
    was = block.rate.clone()
    assert torch.equal(block.bfloat16().rate, was)


def test_rates_have_values_after_a_build_without_memory():
    want = torch.exp2(-torch.linspace(1.0, 9.0, 6))
    assert torch.equal(_block().to_empty(device="cpu").rate, want)
    with torch.device("meta"):
        block = _block()
    assert block.rate.is_meta
    assert torch.equal(block.to_empty(device="cpu").rate, want)
    assert _block().to("meta").rate.is_meta


def test_a_scale_has_to_be_a_number_that_float32_holds():
    """The backward carries a state over 1 / scale: neither may vanish or overflow."""
    for bad in (0.0, float("inf"), float("nan"), 1e300, -1e39, 1e-46, 1e-39):
        with pytest.raises(ValueError):
            token_ops._scale(bad, 64)
    for good in (-0.5, 2.0**-126, 3.4e38):
        assert token_ops._scale(good, 64) == good
    assert token_ops._scale(None, 64) == 0.125
    lib = _lib.load()
    for bad in (0.0, float("inf"), float("nan"), 1e-39):
        args = token_ops._DECAY(2, 100, 4, 2, 64, 64, 1, bad, 16, 16, 16, *([0] * 9), 16, 0, 0, 16, 0, 16, 0, 0, 0, 0, 16, 16, 16, 0, 0, 0, 0)
        assert lib.ews_decay_bwd(args, None) == 1
