"""Limits of the gated block and the adapters that the header states: what the size functions answer beyond them, on the CPU."""
import ctypes as C

import pytest

from test_ffn_refusals import _backward, _forward, _linear

P = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    from ateniaengine_b200 import _lib
    return _lib.lib()


def _low(rank):
    from ateniaengine_b200 import _lib
    return _lib.LowRank(a=P, b=P, scale=P, rank=rank)


@pytest.mark.parametrize("part", ["gate", "up", "down"])
def test_no_workspace_for_ranks_that_the_calls_refuse(lib, part):
    from ateniaengine_b200 import _lib

    def nbytes(rank):
        parts = {"gate": _low(8), "up": _low(16), "down": _low(0), part: _low(rank)}
        return lib.atenia_gated_ffn_workspace_bytes(100, 64, 96, C.byref(_lib.FfnAdapters(**parts)), 0)

    for rank in (-8, 4, 7, 12, 136, 1 << 30):
        assert nbytes(rank) == 0, rank
    assert 0 < nbytes(0) < nbytes(8) < nbytes(128)


def test_no_workspace_for_more_tokens_than_the_calls_take(lib):
    linear = lib.atenia_adapter_linear_workspace_bytes
    assert linear(1 << 24, 128) >= 1 << 32 and linear((1 << 24) + 1, 8) == 0 and linear((1 << 31) - 1, 8) == 0
    for backward in (0, 1):
        assert lib.atenia_gated_ffn_workspace_bytes((1 << 24) + 1, 64, 96, None, backward) == 0


def test_python_entries_refuse_sizes_that_the_library_does_not_take():
    """Above 2^24 tokens or a width of 2^20: at 2^32 the library's 32-bit sizes would be those of a small call."""
    import torch
    from ateniaengine_b200 import adapter_linear, ffn, gated_ffn, gated_ffn_backward

    def z(rows, cols):
        return torch.zeros((1, 1), dtype=torch.bfloat16).expand(rows, cols)

    w = z(32, 16), z(32, 16), z(16, 32)
    for T in ((1 << 24) + 1, (1 << 32) + 4):
        x = z(T, 16)
        for call in (lambda: gated_ffn(x, *w), lambda: gated_ffn_backward(x, x, *w, None), lambda: adapter_linear(x, w[0], None, None)):
            with pytest.raises(ValueError, match="at most"):
                call()
    for wide in ((1 << 20) + 16, (1 << 32) + 16):
        with pytest.raises(ValueError, match="at most"):
            ffn._block(z(4, 16), z(wide, 16), z(wide, 16), z(16, wide))
        with pytest.raises(ValueError, match="at most"):
            ffn._block(z(4, wide), z(16, wide), z(16, wide), z(wide, 16))
        with pytest.raises(ValueError, match="at most"):
            ffn._projection(z(4, 16), z(wide, 16))
        with pytest.raises(ValueError, match="at most"):
            ffn._projection(z(4, wide), z(16, wide))


@pytest.mark.parametrize("adapters", [{"gate": None}, {"gate": None, "up": None, "down": None}])
def test_a_dict_of_no_adapters_is_refused_in_python(adapters):
    import torch
    from ateniaengine_b200 import ffn
    with pytest.raises(ValueError, match="without adapters"):
        ffn._block_adapters(adapters, torch.zeros(4, dtype=torch.int32), 4, 64, 96, False, torch.device("cpu"))


def _over(call, lib, sizes, out, other):
    """The call with `out` on `other`, and with it on its last 16 bytes; everything else apart."""
    apart = {name: P + (i << 24) for i, name in enumerate(sizes)}
    return [call(lib, **{**apart, out: apart[other] + at}) for at in (0, (sizes[other] - 1) // 16 * 16)]


def test_outputs_of_the_block_over_what_it_reads_or_writes(lib):
    """T = 4, d = 64, F = 96.  (The output over x is allowed and not called here: the addresses are nobody's.)"""
    kept, w = 4 * 96 * 4, 64 * 96 * 2
    need = lib.atenia_gated_ffn_workspace_bytes(4, 64, 96, None, 0)
    sizes = dict(x=512, gate=w, up=w, down=w, y=512, sg=kept, su=kept, ws=need)
    for out, others in (("y", ("gate", "up", "down", "sg", "su", "ws")), ("sg", ("x", "gate", "up", "down", "y", "su", "ws")),
                        ("su", ("x", "gate", "up", "down", "y", "sg", "ws")), ("ws", ("x", "gate", "up", "down", "y", "sg", "su"))):
        for other in others:
            assert _over(_forward, lib, sizes, out, other) == [-2, -2], (out, other)


def test_outputs_of_the_block_over_its_adapters(lib):
    from ateniaengine_b200 import _lib
    n, r, T, d, F = 3, 16, 4, 64, 96
    places, sizes = {}, {}
    for i, part in enumerate(("gate", "up", "down")):
        n_in, n_out = (F, d) if part == "down" else (d, F)
        for j, (name, size) in enumerate((("a", n * r * n_in * 2), ("b", n * r * n_out * 2), ("scale", n * 4))):
            places[part, name], sizes[part, name] = (1 << 30) + ((3 * i + j) << 20), size
    sets = {p: _lib.LowRank(rank=r, **{k: places[p, k] for k in ("a", "b", "scale")}) for p in ("gate", "up", "down")}
    ad = _lib.FfnAdapters(ids=(1 << 30) + (10 << 20), n=n, **sets)
    places["ids"], sizes["ids"] = ad.ids, T * 4
    apart = {name: P + (i << 24) for i, name in enumerate(("x", "gate", "up", "down", "y", "ws"))}
    for other in places:
        for out in ("y", "ws"):
            for at in (0, (sizes[other] - 1) // 16 * 16):
                assert _forward(lib, adapters=C.byref(ad), **{**apart, out: places[other] + at}) == -2, (out, other, at)


def test_workspace_of_the_backward_pass_over_its_operands(lib):
    w, kept = 12288, 1536
    sizes = dict(dy=512, x=512, gate=w, up=w, down=w, sg=kept, su=kept, dx=512, dg=w, du=w, dd=w,
                 ws=lib.atenia_gated_ffn_workspace_bytes(4, 64, 96, None, 1))
    for other in sizes:
        if other != "ws":
            assert _over(_backward, lib, sizes, "ws", other) == [-2, -2], other


def test_output_of_the_projection_over_what_it_reads(lib):
    """T = 4, 64 -> 96, two adapters of rank 8."""
    from ateniaengine_b200 import _lib
    low = dict(a=2 * 8 * 64 * 2, b=2 * 8 * 96 * 2, scale=8)
    at = {name: (1 << 30) + (i << 20) for i, name in enumerate(low)}
    sizes = dict(x=512, w=12288, ids=16, y=768, ws=lib.atenia_adapter_linear_workspace_bytes(4, 8))
    for out in ("y", "ws"):
        for other in sizes:
            if other != out:
                call = lambda lib, **kw: _linear(lib, low=_lib.LowRank(rank=8, **at), **kw)
                assert _over(call, lib, sizes, out, other) == [-2, -2], (out, other)
        for name in low:
            apart = {k: P + (i << 24) for i, k in enumerate(sizes)}
            for shift in (0, (low[name] - 1) // 16 * 16):
                assert _linear(lib, low=_lib.LowRank(rank=8, **at), **{**apart, out: at[name] + shift}) == -2, (out, name)


def test_no_product_of_allowed_sizes_has_more_tiles_than_a_launch_takes(tmp_path):
    """Or it would be refused behind products that have run."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = tmp_path / "libdenselimits.so"
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", os.path.join(root, "tests", "dense_limits_probe.cpp"), "-o", str(so)])
    probe = C.CDLL(str(so))
    probe.limits_work_items.restype = probe.limits_most.restype = C.c_longlong
    most = probe.limits_most()
    assert most * 2 < 1 << 31  # (two CTAs a pair)
    widths = [16, 48, 64, 80, 128, 144, 256, 272, 1024, 1 << 14, 1 << 17, (1 << 20) - 16, 1 << 20]
    seen = 0
    for T in (1, 17, 127, 128, 129, 4096, (1 << 20) + 1, 1 << 22, (1 << 24) - 1, 1 << 24):
        for d in widths:
            for F in widths:
                blocks = [-(-v // 64) for v in (T, d, F)]
                few, gw = min(128, -(-T // 8) * 8), [F, d, blocks[0], F, d, blocks[0], d, F, blocks[0]]
                for sizes, rows, two, grad, adapters in (([T, F, blocks[1]], few, 1, 0, (0, 1, 65536)), ([T, d, blocks[2]], few, 0, 0, (0, 1, 65536)),
                                                         ([T, F, blocks[1]], few, 0, 1, (0,)), ([T, d, 2 * blocks[2]], few, 0, 0, (0,)), (gw, 128, 0, 0, (0,))):
                    for n in adapters:
                        items = probe.limits_work_items((C.c_longlong * 9)(*sizes), len(sizes) // 3, rows, two, grad, n)
                        assert items <= most, (T, d, F, two, grad, n, items)
                        seen = max(seen, items)
    assert seen > 1 << 28  # (the sizes do come near it)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_scales_and_ids_off_their_type_are_refused(lib, shift):
    """The kernels read them as 32-bit words: an address in between would be a fault on the device."""
    from ateniaengine_b200 import _lib
    low = _lib.LowRank(a=P, b=P, scale=P + shift, rank=8)
    assert _linear(lib, low=low) == -2 and _linear(lib, ids=P + shift) == -2
    good = dict(gate=_low(8), up=_low(8), down=_low(8), ids=P, n=2)
    for bad in (dict(gate=low), dict(up=low), dict(down=low), dict(ids=P + shift)):
        assert _forward(lib, adapters=C.byref(_lib.FfnAdapters(**{**good, **bad})), nbytes=0) == -2, bad
