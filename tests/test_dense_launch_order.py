"""The kernels of the dense block and the adapters that read before their own wait (csrc/common.cuh, chain_next): each kernel ahead of
one lets it start only behind its own wait, and the first launch of a call reads nothing early."""
import os
import re

from test_chained_launch_order import CSRC, kernels

DENSE = {"dense_rows_kernel", "dense_tile_kernel", "dense_pair_kernel", "adapter_gemv_kernel", "adapter_reduce_kernel"}


def test_the_dense_kernels_wait_before_they_let_the_next_one_start():
    seen = set()
    for _, name, body in kernels():
        if name in DENSE:
            seen.add(name)
            # every chain_next() directly behind a wait of the same branch, or behind the products
            for at in (m.start() for m in re.finditer(r"chain_next\(\)", body)):
                wait = body.rfind("chain_wait()", 0, at)
                assert wait >= 0 and "warp == 1" not in body[wait:at], name
    assert seen == DENSE


def test_the_reductions_wait_before_they_read():
    """They come first in a call: what they read may be the work of any kernel before it."""
    for _, name, body in kernels():
        if name in ("adapter_reduce_kernel", "adapter_gemv_kernel"):
            wait = body.index("chain_wait()")
            for read in (r"list_adapters\(", r"tma_load_", r"\.ids\[", r"load16\(", r"\.scale\["):
                assert all(m.start() > wait for m in re.finditer(read, body)), (name, read)


def _entry(name):
    text = re.sub(r"//.*", "", open(os.path.join(CSRC, "gated_ffn.cu"), encoding="utf-8").read())
    body = text[text.index("int " + name + "("):]
    return body[:body.index("\n}")]


def test_the_first_product_of_a_call_reads_nothing_early():
    forward, backward, linear = (_entry("atenia_" + n) for n in ("gated_ffn_forward", "gated_ffn_backward", "adapter_linear"))
    # forward: only behind the reduction of its own rows, which is launched first
    assert forward.count("g1.b_early") == 1 and forward.count("g1.a_early") == 1
    block = forward[forward.index("if (!rc && ad1) {"):]
    assert "g1.b_early = g1.a_early = true;" in block[:block.index("}\n")]
    order = [forward.index(s) for s in ("launch_adapter_reduce(first.red", "launch_dense_gemm(g1", "launch_adapter_reduce(second.red",
                                        "launch_dense_gemm(g2")]
    assert order == sorted(order) and "if (!rc && ad1) rc = launch_adapter_reduce(first.red" in forward
    assert "g2.a_early" not in forward[:forward.index("if (!rc && ad2) {")]  # (h early only behind its own reduction)
    assert "g1.b_early" not in backward and "g1.a_early" not in backward
    order = [backward.index(f"launch_dense_gemm(g{i}") for i in (1, 2, 3)]
    assert order == sorted(order) and "g2.a_early" not in backward
    assert linear.index("launch_adapter_reduce(plan.red") < linear.index("launch_dense_gemm(g,")
