"""The exact cases of the dense block and the adapters (ffn_exact) are exact, and show mistakes: planted in the expected results, each
changes their bits.  On the CPU; of long calls 64 tokens, half a tile, or 32 of a large block."""
import pytest
import torch

import ffn_exact as ex

ROWS = 64


def rounded(t):
    return t.to(torch.bfloat16)


def differ(a, b):
    return not torch.equal(rounded(a), rounded(b))


def blocks(k):
    """Slices of 64 of a reduction: the first, one in the middle, the last."""
    n = -(-k // 64)
    return [slice(64 * j, min(64 * j + 64, k)) for j in sorted({0, n // 2, n - 1})]


def without(a, b, part):
    """a b^T without the terms of `part`."""
    return a @ b.T - a[:, part] @ b[:, part].T


@pytest.mark.parametrize("T,d,F", ex.BLOCKS)
def test_block(T, d, F):
    rows = min(max(T, 16), ROWS if d * F < 1e7 else ROWS // 2)  # (of a shorter call the inputs of 16)
    x, gate, up, down, dy = (t.float() for t in (ex.make_x(rows, d, T, "cpu"), *ex.make_block(d, F, 1, "cpu"), ex.make_dy(rows, d, 5, "cpu")))
    y, g, u, h = ex.forward(x, gate, up, down)  # (f32 holds what ffn_exact asserts)
    dx, dgate, dup, ddown = ex.backward(dy, x, gate, up, down, u, h)
    dh = dy @ down
    dg, du = dh * u, dh * 64

    def wrong_g(part):
        other = without(x, gate, part)
        return (torch.sigmoid(other) * other * u) @ down.T

    for part in blocks(d):
        assert differ(y, wrong_g(part)) and differ(y, (g * without(x, up, part)) @ down.T), part
        other = without(dy, down.T, part)
        assert differ(dx, (other * u) @ gate + (other * 64) @ up), part
    for part in blocks(F):
        assert differ(y, without(h, down, part)), part
        assert differ(dx, without(dg, gate.T, part) + du @ up) and differ(dx, dg @ gate + without(du, up.T, part)), part
    assert differ(dx, dg @ gate) and differ(dx, du @ up)
    if F >= 128:  # partial sums kept in bf16 (those of y have more than eight bits from 8000 features on)
        cut = F // 2
        halves = [rounded(dg[:, s] @ gate[s] + du[:, s] @ up[s]).float() for s in (slice(0, cut), slice(cut, F))]
        assert differ(dx, halves[0] + halves[1])
    if F >= 8000:
        assert differ(y, rounded(h[:, :cut] @ down[:, :cut].T).float() + rounded(h[:, cut:] @ down[:, cut:].T).float())
    for part in blocks(rows):
        for exact, a, b in ((dgate, dg, x), (dup, du, x), (ddown, dy, h)):
            assert differ(exact, without(a.T, b.T, part)), part


@pytest.mark.parametrize("T,d,out,n,r,kind", ex.LINEARS)
def test_linear(T, d, out, n, r, kind):
    gen = ex.generator(T, "cpu")
    rows, n = max(min(T, ROWS), 16), min(n, ROWS)
    x, w, low, ids = ex.signs(gen, rows, d), ex.signs(gen, out, d), ex.make_low(n, r, d, out, 7, "cpu"), ex.make_ids(kind, rows, n, 3, "cpu")
    y, (a, b, scale) = ex.linear(x, w, low, ids), low
    assert differ(y, ex.linear(x, w))
    for part in blocks(d):
        assert differ(y, without(x, w, part) + ex.delta(x, low, ids, "")), part
    # a reduced row without the last columns of its reduction that any adapter in use has; without the last sixteen rank columns
    used = ids[(ids >= 0) & (ids < n)].unique().long()
    last = int(torch.nonzero(a[used].abs().sum((0, 1)))[-1])
    cut = a.clone()
    cut[:, :, last // 64 * 64:] = 0
    assert differ(y, ex.linear(x, w, (cut, b, scale), ids))
    short = b.clone()
    short[:, :, max(0, r - 16):] = 0
    assert differ(y, ex.linear(x, w, (a, short, scale), ids))


@pytest.mark.parametrize("T,d,F,n,ranks,kind", ex.ADAPTED)
def test_block_with_adapters(T, d, F, n, ranks, kind):
    rows, n = max(min(T, ROWS), 16), min(n, ROWS)
    x, w, ids = ex.make_x(rows, d, T, "cpu"), ex.make_block(d, F, 1, "cpu"), ex.make_ids(kind, rows, n, 3, "cpu")
    parts = ("gate", "up", "down")
    lows = ex.make_lows(parts, n, ranks, d, F, 9, "cpu")
    y, g, u, h = ex.forward(x, *w, lows, ids)
    gate, up, down = w

    def result(lows):
        a, b = ex.linear(x, gate, lows.get("gate"), ids, unit_w=2.0 ** -4), ex.linear(x, up, lows.get("up"), ids)
        h = rounded(torch.sigmoid(a) * a * b).double()
        y = h @ down.T
        if "down" in lows:
            a, b, scale = lows["down"]
            for i in ids.unique().tolist():
                if 0 <= i < n:
                    at = ids == i
                    y[at] += rounded(scale[i] * (h[at] @ a[i].T)).double() @ b[i].T
        return y

    assert not differ(y, result(lows))
    for p, r in zip(parts, ranks):
        assert differ(y, result({q: low for q, low in lows.items() if q != p})), p
        a, b, scale = lows[p]
        short = b.clone()
        short[:, :, r - 8:] = 0  # the last rank columns
        if p != "gate" or r > 8:  # (eight of the gate: one is all that adds)
            assert differ(y, result({**lows, p: (a, short, scale)})), p
