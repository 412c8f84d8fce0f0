"""Calls from a host thread that has made no CUDA call of its own yet, as torch's backward threads are: nothing has bound the device's
context there, which the encoding of tensor maps asks for."""
import threading

import pytest
import torch

import ffn_helpers as ref

pytestmark = pytest.mark.gpu


def in_a_new_thread(call):
    out = []

    def run():
        try:
            out.append(call())
        except Exception as e:
            out.append(e)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    return out[0]


@pytest.mark.parametrize("T", [1, 40, 300, 1100])
def test_the_dense_calls(T):
    from ateniaengine_b200 import adapter_linear, gated_ffn, gated_ffn_backward
    d, F = 528, 400
    x, dy, w, low, ids = ref.rand(T, 1.0, T, d), ref.rand(T + 1, 1.0, T, d), ref.block(2, d, F), ref.low_rank(50, 5, 16, d, F), ref.ids_of("runs", T, 5)
    y, saved = gated_ffn(x, *w, save=True)
    for call in (lambda: (gated_ffn(x, *w),), lambda: gated_ffn_backward(dy, x, *w, saved), lambda: (adapter_linear(x, w[0], low, ids),)):
        expected = call()
        torch.cuda.synchronize()
        got = in_a_new_thread(call)
        assert not isinstance(got, Exception), got
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("int8", [False, True])
def test_a_layer(int8):
    """Created in a thread of its own, and its forward in another."""
    from ateniaengine_b200 import synth
    shape = synth.MoeShape("t", 256, 128, 8, 2, True, int8=int8)
    w = synth.make_weights(shape, 1, torch.device("cuda", 0))
    x = ref.rand(1, 1.0, 40, 256)
    expected = synth.build_layer(shape, w, max_tokens=64).forward(x)
    torch.cuda.synchronize()
    layer = in_a_new_thread(lambda: synth.build_layer(shape, w, max_tokens=64))
    assert not isinstance(layer, Exception), layer
    got = in_a_new_thread(lambda: layer.forward(x))
    assert not isinstance(got, Exception), got
    assert torch.equal(got, expected)
