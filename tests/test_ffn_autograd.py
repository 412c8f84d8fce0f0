"""Torch's autograd beside the gated block and the adapters: an input whose gradient would be lost is refused, and a Function of the
user's own around the two calls records."""
import pytest
import torch


def _cpu_calls():
    from ateniaengine_b200 import LowRankAdapters, adapter_linear, gated_ffn, gated_ffn_backward
    b = torch.bfloat16
    x = torch.zeros((4, 64), dtype=b, requires_grad=True)
    w = torch.zeros((96, 64), dtype=b), torch.zeros((96, 64), dtype=b), torch.zeros((64, 96), dtype=b)
    low = LowRankAdapters(torch.zeros((2, 8, 64), dtype=b), torch.zeros((2, 96, 8), dtype=b), torch.zeros(2))
    ids = torch.zeros(4, dtype=torch.int32)
    return (lambda: gated_ffn(x, *w), lambda: gated_ffn(x, *w, save=True), lambda: adapter_linear(x, w[0], low, ids),
            lambda: gated_ffn_backward(x, x, *w, torch.zeros((2, 24, 4, 4))))


def test_an_input_with_a_gradient_is_refused():
    """(On the CPU the calls end at the device: which refusal comes is what is asked.)"""
    *forward, backward = _cpu_calls()
    for call in forward:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="CUDA"):
        backward()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_inside_a_function_of_the_users(T):
    import ffn_helpers as ref
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward

    class Block(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, gate, up, down):
            y, saved = gated_ffn(x, gate, up, down, save=True)
            ctx.save_for_backward(x, gate, up, down, saved)
            return y

        @staticmethod
        def backward(ctx, dy):
            return gated_ffn_backward(dy, *ctx.saved_tensors)

    d, F = 272, 400
    x, w, dy = ref.rand(T, 1.0, T, d), ref.block(3, d, F), ref.rand(T + 1, 1.0, T, d)
    leaves = [t.clone().requires_grad_() for t in (x, *w)]
    y = leaves[0] + Block.apply(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    plain, saved = gated_ffn(x, *w, save=True)
    expected = gated_ffn_backward(dy, x, *w, saved)
    assert torch.equal(y.detach(), x + plain) and torch.equal(grads[0], dy + expected[0])
    assert all(torch.equal(a, b) for a, b in zip(grads[1:], expected[1:]))
    with torch.no_grad():
        assert torch.equal(gated_ffn(leaves[0], *leaves[1:]), plain)
    assert torch.equal(gated_ffn(x, *leaves[1:]), plain)  # parameters are ordinary arguments
    with pytest.raises(ValueError, match="gradient"):
        gated_ffn(leaves[0], *w)
