"""Low-rank adapters of many requests, alone and inside the gated block, against 64 bits within the bound of their roundings."""
import pytest
import torch

import ffn_helpers as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["one", "none", "distinct", "runs", "odd"])
@pytest.mark.parametrize("T,d,out,n,r", [(1, 16, 16, 1, 8), (1, 512, 1408, 4, 16), (5, 272, 144, 3, 24), (8, 512, 400, 5, 128), (13, 528, 144, 20, 40), (33, 64, 272, 40, 8),
                                         (64, 1040, 528, 70, 16), (129, 144, 400, 150, 64), (130, 272, 2064, 9, 128),
                                         (300, 528, 144, 200, 16), (1021, 1040, 1040, 12, 40), (2100, 512, 1552, 30, 64), (2100, 272, 5632, 300, 16), (1500, 144, 5008, 40, 128),
                                         # reduced rows by the tensor cores beside the kernel of a few rows; a cut last wave of CTA pairs
                                         (8, 32768, 512, 3, 128), (5000, 5632, 2048, 9, 16)])
def test_linear(T, d, out, n, r, kind):
    from ateniaengine_b200 import adapter_linear
    x, w, low, ids = ref.rand(T, 1.0, T, d), ref.rand(1, d ** -0.5, out, d), ref.low_rank(5, n, r, d, out), ref.ids_of(kind, T, n)
    buf = torch.full((T + 2, out), 7.0, device="cuda", dtype=torch.bfloat16)
    y = adapter_linear(x, w, low, ids, out=buf[1:T + 1], sync=True)
    ref.assert_within(y, ref.adapter_linear(x, w, low, ids), "y")
    assert (buf[0] == 7).all() and (buf[T + 1] == 7).all()
    assert torch.equal(y, adapter_linear(x, w, low, ids))


@pytest.mark.parametrize("parts", ["gate,up,down", "gate", "up", "down", "gate,down"])
@pytest.mark.parametrize("T,d,F,n,ranks,kind", [(1, 64, 96, 2, (8, 16, 24), "one"), (11, 272, 144, 4, (24, 8, 128), "odd"), (48, 512, 1408, 33, (16, 16, 16), "distinct"),
                                                (200, 272, 400, 7, (8, 64, 40), "odd"), (1100, 528, 1040, 16, (32, 32, 128), "runs"),
                                                (1500, 272, 3600, 40, (128, 128, 16), "distinct"), (700, 512, 5632, 50, (96, 40, 64), "odd"),
                                                (1100, 2048, 5632, 16, (24, 8, 32), "runs"),
                                                # two parts of many reduced rows beside the ring, and under the sums of a cut reduction
                                                (100, 1024, 14336, 6, (128, 128, 16), "distinct"), (128, 2048, 512, 5, (128, 128, 64), "runs"),
                                                (4, 512, 1408, 3, (128, 64, 128), "distinct")])
def test_block(T, d, F, n, ranks, kind, parts):
    from ateniaengine_b200 import gated_ffn
    x, w, ids = ref.rand(T, 1.0, T, d), ref.block(3, d, F), ref.ids_of(kind, T, n)
    sets = {p: ref.low_rank(11 * i + 30, n, ranks[i], *((F, d) if p == "down" else (d, F)))
            for i, p in enumerate(("gate", "up", "down")) if p in parts.split(",")}
    y = gated_ffn(x, *w, adapters=sets, adapter_ids=ids, sync=True)
    ref.assert_within(y, ref.forward(x, *w, sets, ids)[0], "y")
    assert torch.equal(y, gated_ffn(x, *w, adapters=sets, adapter_ids=ids))


@pytest.mark.parametrize("T,r", [(6, 16), (13, 128), (40, 16), (40, 40), (600, 64)])
def test_a_broken_adapter_stays_with_its_requests(T, r):
    """NaN and infinities in one adapter's matrices: every other row is as it is without them."""
    from ateniaengine_b200 import adapter_linear, gated_ffn
    n, d, F = 6, 272, 400
    x, w, ids = ref.rand(1, 1.0, T, d), ref.block(3, d, F), ref.ids_of("distinct", T, n, 4)
    ids[::5] = -1
    sets = {p: ref.low_rank(20 + i, n, r, *((F, d) if p == "down" else (d, F))) for i, p in enumerate(("gate", "up", "down"))}
    clean = adapter_linear(x, w[0], sets["gate"], ids), gated_ffn(x, *w, adapters=sets, adapter_ids=ids)
    for s in sets.values():
        s.a[2, 0, 3] = float("nan")
        s.b[2, 5, r - 1] = float("inf")
        s.b[4] = float("nan")
        s.scale[5] = float("inf")
    broken = adapter_linear(x, w[0], sets["gate"], ids, sync=True), gated_ffn(x, *w, adapters=sets, adapter_ids=ids, sync=True)
    sound = (ids != 2) & (ids != 4) & (ids != 5)
    for a, b in zip(clean, broken):
        assert torch.equal(a[sound], b[sound])
    assert torch.isnan(broken[0][ids == 2]).all() and torch.isnan(broken[0][ids == 4]).all()


def test_no_adapter_is_the_plain_product():
    """Ids of -1 throughout: the block's own bits, without a look at adapters full of NaN."""
    from ateniaengine_b200 import gated_ffn
    T, d, F = 77, 272, 400
    x, w = ref.rand(1, 1.0, T, d), ref.block(3, d, F)
    sets = {p: ref.low_rank(20, 3, 16, *((F, d) if p == "down" else (d, F))) for p in ("gate", "up", "down")}
    for s in sets.values():
        for t in s:
            t.fill_(float("nan"))
    ids = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(gated_ffn(x, *w, adapters=sets, adapter_ids=ids, sync=True), gated_ffn(x, *w))


def test_no_tokens():
    from ateniaengine_b200 import adapter_linear
    x, ids = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16), torch.empty(0, dtype=torch.int32, device="cuda")
    assert adapter_linear(x, ref.rand(1, 1.0, 96, 64), ref.low_rank(2, 3, 8, 64, 96), ids, sync=True).shape == (0, 96)


def test_beside_the_block_it_adapts():
    """A projection, the block and a second projection in a row on one stream, captured with new ids written in between."""
    from ateniaengine_b200 import adapter_linear, gated_ffn
    T, d, F, n, r = 45, 272, 400, 9, 16
    x, w, wo = ref.rand(1, 1.0, T, d), ref.block(3, d, F), ref.rand(9, d ** -0.5, d, d)
    sets = {p: ref.low_rank(20 + i, n, r, *((F, d) if p == "down" else (d, F))) for i, p in enumerate(("gate", "up", "down"))}
    low = ref.low_rank(50, n, r, d, d)
    ids = ref.ids_of("distinct", T, n)

    def step():
        a = adapter_linear(x, wo, low, ids)
        b = gated_ffn(a, *w, adapters=sets, adapter_ids=ids)
        return a, b, adapter_linear(b, wo, low, ids)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        ids.copy_(ref.ids_of("distinct", T, n, seed))
        x.copy_(ref.rand(seed + 60, 1.0, T, d))
        graph.replay()
        a, b, c = step()
        assert all(torch.equal(p, q) for p, q in zip(captured, (a, b, c)))
        ref.assert_within(a, ref.adapter_linear(x, wo, low, ids), "projection")
        ref.assert_within(b, ref.forward(a, *w, sets, ids)[0], "block")
        ref.assert_within(c, ref.adapter_linear(b, wo, low, ids), "second projection")


def test_threads_with_streams_of_their_own():
    """Four host threads, each its own sizes on its own stream, at the same time: the bits that each has alone."""
    import threading
    from ateniaengine_b200 import adapter_linear, gated_ffn, gated_ffn_backward
    d, F, n, r = 528, 1040, 7, 16
    w, low = ref.block(3, d, F), ref.low_rank(50, n, r, d, d)
    wo = ref.rand(9, d ** -0.5, d, d)

    def step(x, dy, ids):
        a = adapter_linear(x, wo, low, ids)
        y, saved = gated_ffn(a, *w, save=True)
        return [a, y, *gated_ffn_backward(dy, a, *w, saved)]

    jobs = []
    for i, T in enumerate((3, 48, 300, 1100)):
        args = ref.rand(T, 1.0, T, d), ref.rand(T + 1, 1.0, T, d), ref.ids_of("odd" if i % 2 else "runs", T, n, i)
        jobs.append((args, step(*args)))
    torch.cuda.synchronize()
    wrong = []

    def run(args, alone):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step(*args)
            torch.cuda.current_stream().synchronize()
            wrong.extend(not torch.equal(p, q) for p, q in zip(got, alone))

    threads = [threading.Thread(target=run, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(wrong) == 6 * len(jobs) and not any(wrong)
