"""The dense block, its gradients and the adapters on inputs whose results are known to the last bit (ffn_exact)."""
import pytest
import torch

import ffn_exact as ex

pytestmark = pytest.mark.gpu


def same(got, exact, what):
    wrong = got != exact.to(torch.bfloat16)
    assert got.shape == exact.shape and not wrong.any(), f"{what}: {int(wrong.sum())} of {wrong.numel()}, the first at {torch.nonzero(wrong)[0].tolist()}"


@pytest.mark.parametrize("T,d,F", ex.BLOCKS)
def test_block_and_gradients(T, d, F):
    from ateniaengine_b200 import gated_ffn, gated_ffn_backward
    x, w, dy = ex.make_x(T, d, T, "cuda"), ex.make_block(d, F, 1, "cuda"), ex.make_dy(T, d, 5, "cuda")
    y, g, u, h = ex.forward(x, *w)
    bx, bdy, *bw = ex.low16(x, dy, *w)
    same(gated_ffn(bx, *bw), y, "y")
    got, saved = gated_ffn(bx, *bw, save=True)
    same(got, y, "y beside the saved projections")
    kept_g, kept_u = saved.permute(0, 2, 1, 3).reshape(2, T, F).double()
    assert torch.equal(kept_g, g) and torch.equal(kept_u, u)
    for grad, exact, name in zip(gated_ffn_backward(bdy, bx, *bw, saved, sync=True), ex.backward(dy, x, *w, u, h), ("dx", "dgate", "dup", "ddown")):
        same(grad, exact, name)


@pytest.mark.parametrize("T,d,F", ex.BLOCKS)
def test_saved_projections(T, d, F):
    """Any integers in the gate: what the activation makes of them is not asked for."""
    from ateniaengine_b200 import gated_ffn
    gen = ex.generator(T, "cuda")
    x, gate, up, down = ex.signs(gen, T, d), ex.signs(gen, F, d), ex.signs(gen, F, d), torch.zeros((d, F), device="cuda").double()
    _, saved = gated_ffn(*ex.low16(x, gate, up, down), save=True, sync=True)
    kept_g, kept_u = saved.permute(0, 2, 1, 3).reshape(2, T, F).double()
    assert torch.equal(kept_g, ex.linear(x, gate)) and torch.equal(kept_u, ex.linear(x, up))


@pytest.mark.parametrize("T,d,out,n,r,kind", ex.LINEARS)
def test_linear(T, d, out, n, r, kind):
    from ateniaengine_b200 import LowRankAdapters, adapter_linear
    gen = ex.generator(T, "cuda")
    x, w, low, ids = ex.signs(gen, T, d), ex.signs(gen, out, d), ex.make_low(n, r, d, out, 7, "cuda"), ex.make_ids(kind, T, n, 3, "cuda")
    a, b, scale = low
    got = adapter_linear(*ex.low16(x, w), LowRankAdapters(*ex.low16(a, b), scale.float()), ids, sync=True)
    same(got, ex.linear(x, w, low, ids), "y")


@pytest.mark.parametrize("parts", [("gate", "up", "down"), ("gate",), ("up",), ("down",)])
@pytest.mark.parametrize("T,d,F,n,ranks,kind", ex.ADAPTED)
def test_block_with_adapters(T, d, F, n, ranks, kind, parts):
    from ateniaengine_b200 import LowRankAdapters, gated_ffn
    x, w, ids = ex.make_x(T, d, T, "cuda"), ex.make_block(d, F, 1, "cuda"), ex.make_ids(kind, T, n, 3, "cuda")
    lows = ex.make_lows(parts, n, ranks, d, F, 9, "cuda")
    sets = {p: LowRankAdapters(*ex.low16(a, b), scale.float()) for p, (a, b, scale) in lows.items()}
    got = gated_ffn(*ex.low16(x, *w), adapters=sets, adapter_ids=ids, sync=True)
    same(got, ex.forward(x, *w, lows, ids)[0], "y")
