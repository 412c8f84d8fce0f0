"""The dense gated block and its gradients against 64 bits, element by element within the bound of their roundings (ffn_helpers)."""
import pytest
import torch

import ffn_helpers as ref

pytestmark = pytest.mark.gpu

SIZES = [(1, 16, 16), (1, 512, 1408), (2, 48, 80), (7, 272, 144), (8, 64, 64), (9, 64, 128), (16, 1040, 48), (16, 272, 2064), (64, 512, 1408), (100, 16, 2064),
         (127, 1040, 48), (128, 272, 144), (129, 272, 144), (255, 144, 272), (257, 512, 400), (700, 1040, 1424), (1021, 528, 1040),
         (2100, 768, 1552),
         # reductions cut over clusters of single CTAs and of pairs, and behind the last whole wave (tests/test_dense_choice.py)
         (300, 2064, 8208), (1021, 2048, 5632), (2600, 2064, 4112)]


@pytest.mark.parametrize("T,d,F", SIZES)
def test_forward(T, d, F):
    from ateniaengine_b200 import gated_ffn
    x, w = ref.rand(T, 1.0, T, d), ref.block(T + 10, d, F)
    out = torch.full((T + 2, d), 7.0, device="cuda", dtype=torch.bfloat16)
    y = gated_ffn(x, *w, out=out[1:T + 1], sync=True)
    expected, _ = ref.forward(x, *w)
    ref.assert_within(y, expected, "y")
    assert (out[0] == 7).all() and (out[T + 1] == 7).all()
    assert torch.equal(y, gated_ffn(x, *w))


@pytest.mark.parametrize("T,d,F", SIZES)
def test_training_step(T, d, F):
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    x, w, dy = ref.rand(T, 1.0, T, d), ref.block(T + 10, d, F), ref.rand(T + 20, 1.0, T, d)
    y, saved = gated_ffn(x, *w, save=True)
    assert torch.equal(y, gated_ffn(x, *w))
    expected, (g, eg, u, eu, *_) = ref.forward(x, *w)
    kept_g, kept_u = saved.permute(0, 2, 1, 3).reshape(2, T, F).double()
    assert ((kept_g - g).abs() <= eg).all() and ((kept_u - u).abs() <= eu).all()
    kept = saved.clone()
    grads = gated_ffn_backward(dy, x, *w, saved, sync=True)
    assert torch.equal(saved, kept)
    for got, exp, name in zip(grads, ref.backward(dy, x, *w), ("dx", "dgate", "dup", "ddown")):
        ref.assert_within(got, exp, name)
    for a, b in zip(grads, gated_ffn_backward(dy, x, *w, saved)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,d,F", [(5, 48, 80), (130, 272, 144)])
def test_gradients_against_differences(T, d, F):
    """<gradient, direction> and the central difference of sum(dy * y) in 64 bits (its own error is a third-order term, below 1e-6)."""
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    x, w, dy = ref.rand(1, 1.0, T, d), ref.block(2, d, F), ref.rand(3, 1.0, T, d)
    _, saved = gated_ffn(x, *w, save=True)
    grads = gated_ffn_backward(dy, x, *w, saved, sync=True)
    bounds = [b for _, b in ref.backward(dy, x, *w)]
    params = [t.double() for t in (x, *w)]

    def loss(ps):
        x_, g_, u_, d_ = ps
        return (dy.double() * ((torch.nn.functional.silu(x_ @ g_.T) * (x_ @ u_.T)) @ d_.T)).sum()

    for i, (got, bound) in enumerate(zip(grads, bounds)):
        step = torch.randn(params[i].shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        eps = 1e-4
        plus, minus = ([p + (sign * eps * step if j == i else 0) for j, p in enumerate(params)] for sign in (1, -1))
        slope = (loss(plus) - loss(minus)) / (2 * eps)
        allowed = (bound * step.abs()).sum() + 1e-6 * (got.double() * step).abs().sum()
        assert (slope - (got.double() * step).sum()).abs() <= allowed, i


def test_no_tokens():
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    w = ref.block(0, 64, 96)
    x = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    y, saved = gated_ffn(x, *w, save=True, sync=True)
    assert y.shape == (0, 64) and saved.shape == (2, 24, 0, 4)
    dx, *dw = gated_ffn_backward(x, x, *w, saved, sync=True)
    assert dx.shape == (0, 64) and all(g.shape == v.shape and not g.any() for g, v in zip(dw, w))


def test_large_and_small_gates():
    """The activation far out: silu(g) is g, or zero, and nothing is infinite."""
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    x, w, dy = ref.rand(1, 30.0, 33, 64), ref.block(2, 64, 96), ref.rand(3, 1.0, 33, 64)
    y, saved = gated_ffn(x, *w, save=True)
    ref.assert_within(y, ref.forward(x, *w)[0], "y")
    assert saved[0].min() < -88 or saved[0].max() > 60
    for got, exp, name in zip(gated_ffn_backward(dy, x, *w, saved, sync=True), ref.backward(dy, x, *w), ("dx", "dgate", "dup", "ddown")):
        ref.assert_within(got, exp, name)


@pytest.mark.parametrize("T", [3, 300])
def test_not_a_number_stays_in_its_row(T):
    from ateniaengine_b200 import gated_ffn
    x, w = ref.rand(1, 1.0, T, 272), ref.block(2, 272, 144)
    clean = gated_ffn(x, *w)
    x[1, 5] = float("nan")
    x[2, 0] = float("inf")
    y = gated_ffn(x, *w, sync=True)
    rows = torch.ones(T, dtype=torch.bool, device="cuda")
    rows[1] = rows[2] = False
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()


def test_strided_and_shifted_inputs():
    from ateniaengine_b200 import gated_ffn
    x, w = ref.rand(1, 1.0, 50, 2 * 64), ref.block(2, 64, 96)
    y = gated_ffn(x[::2, ::2], *w)
    assert torch.equal(y, gated_ffn(x[::2, ::2].clone(), *w))
    assert torch.equal(gated_ffn(x[7:, :64], w[0].T.contiguous().T, *w[1:]), gated_ffn(x[7:, :64].clone(), *w))
    assert torch.equal(gated_ffn(x[:, :64].contiguous()[3:], *w), gated_ffn(x[3:, :64].clone(), *w))


@pytest.mark.parametrize("T", [1, 40, 700])
def test_captured_and_replayed_beside_another_stream(T):
    """Captured training steps of two batches, replayed at once on two streams."""
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    d, F = 528, 400
    w = ref.block(2, d, F)
    steps, inputs = [], []
    for seed in (1, 2):
        x, dy = ref.rand(seed, 1.0, T, d), ref.rand(seed + 5, 1.0, T, d)
        inputs.append((x, dy))  # (a graph reads them where they are)
        y, saved = gated_ffn(x, *w, save=True)
        eager = (y, *gated_ffn_backward(dy, x, *w, saved))
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y, saved = gated_ffn(x, *w, save=True)
            out = (y, *gated_ffn_backward(dy, x, *w, saved))
        steps.append((stream, graph, eager, out))
    for _ in range(3):
        for _, _, _, out in steps:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for stream, graph, _, _ in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, eager, out in steps:
            assert all(torch.equal(a, b) for a, b in zip(eager, out))


@pytest.mark.parametrize("T", [1, 7, 16, 40])
def test_operands_on_16_byte_boundaries(T):
    """Eight elements into an allocation: the kernels that want 32 bytes leave the call to others."""
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    d, F = 272, 144

    def shifted(t):
        buf = torch.empty(t.numel() + 8, device="cuda", dtype=t.dtype)
        buf[8:] = t.flatten()
        return buf[8:].view(t.shape)

    x, w, dy = ref.rand(1, 1.0, T, d), ref.block(2, d, F), ref.rand(5, 1.0, T, d)
    sx, sw, sdy = shifted(x), [shifted(t) for t in w], shifted(dy)
    assert sx.data_ptr() % 32 == 16
    y, saved = gated_ffn(sx, *sw, save=True, out=shifted(x), sync=True)
    ref.assert_within(y, ref.forward(x, *w)[0], "y")
    for got, exp, name in zip(gated_ffn_backward(sdy, sx, *sw, saved, sync=True), ref.backward(dy, x, *w), ("dx", "dgate", "dup", "ddown")):
        ref.assert_within(got, exp, name)
    ref.assert_within(gated_ffn(x, *sw), ref.forward(x, *w)[0], "weights alone shifted")


@pytest.mark.parametrize("d,F", [(16, 16), (272, 144), (528, 2064), (2048, 5632)])
@pytest.mark.parametrize("T", [1, 3, 4, 5, 8])
def test_few_tokens_are_as_exact_as_their_last_rounding(T, d, F):
    """What the rounding of h left goes through the second product too."""
    from ateniaengine_b200 import gated_ffn
    x, w = ref.rand(T, 1.0, T, d), ref.block(2, d, F)
    ref.assert_within(gated_ffn(x, *w, sync=True), ref.forward(x, *w, h_rounding=ref.BF ** 2)[0], "y")


@pytest.mark.parametrize("T", [5, 40, 600])
def test_in_place(T):
    from ateniaengine_b200 import gated_ffn
    d, F = 272, 2064
    x, w = ref.rand(T, 1.0, T, d), ref.block(2, d, F)
    y = gated_ffn(x, *w)
    assert gated_ffn(x, *w, out=x, sync=True).data_ptr() == x.data_ptr() and torch.equal(x, y)
