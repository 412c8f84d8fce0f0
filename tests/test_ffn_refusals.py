"""Calls of the gated block and the adapters that are refused: by the C entries before they touch a device, and by the Python ones."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    from ateniaengine_b200 import _lib
    return _lib.lib()


P = 1 << 20  # an aligned address that nothing reads: the checks come first


def _forward(lib, **kw):
    a = dict(x=P, gate=P, up=P, down=P, T=4, d=64, F=96, adapters=None, y=P, sg=None, su=None, ws=P, nbytes=1 << 30)
    a.update(kw)
    return lib.atenia_gated_ffn_forward(a["x"], a["gate"], a["up"], a["down"], a["T"], a["d"], a["F"], a["adapters"], a["y"], a["sg"],
                                        a["su"], a["ws"], a["nbytes"], None)


def _backward(lib, **kw):
    a = dict(dy=P, x=P, gate=P, up=P, down=P, sg=P, su=P, T=4, d=64, F=96, dx=P, dg=P, du=P, dd=P, ws=P, nbytes=1 << 30)
    a.update(kw)
    return lib.atenia_gated_ffn_backward(*[a[k] for k in ("dy", "x", "gate", "up", "down", "sg", "su", "T", "d", "F", "dx", "dg", "du",
                                                          "dd", "ws", "nbytes")], None)


def _low(rank=8, **kw):
    from ateniaengine_b200 import _lib
    return _lib.LowRank(**{**dict(a=P, b=P, scale=P, rank=rank), **kw})


def _linear(lib, **kw):
    a = dict(x=P, w=P, T=4, n_in=64, n_out=96, low=_low(), ids=P, n=2, y=P + (1 << 20), ws=P, nbytes=1 << 30)
    a.update(kw)
    low = None if a["low"] is None else C.byref(a["low"])
    return lib.atenia_adapter_linear(a["x"], a["w"], a["T"], a["n_in"], a["n_out"], low, a["ids"], a["n"], a["y"], a["ws"], a["nbytes"],
                                     None)


SIZES = [dict(T=-1), dict(T=(1 << 24) + 1), dict(d=0), dict(d=24), dict(F=100), dict(F=-16), dict(d=(1 << 20) + 16)]


@pytest.mark.parametrize("call", [_forward, _backward])
def test_sizes_pointers_and_workspace_of_the_block(lib, call):
    for bad in SIZES:
        assert call(lib, **bad) == -2, bad
    for name in ("x", "gate", "up", "down", "ws"):
        assert call(lib, **{name: None}) == -1, name
        assert call(lib, **{name: P + 8}) == -2, name
    need = lib.atenia_gated_ffn_workspace_bytes(4, 64, 96, None, int(call is _backward))
    assert need > 0 and call(lib, nbytes=need - 1) == -3


def test_pointers_of_one_direction(lib):
    assert _forward(lib, y=None) == -1 and _forward(lib, sg=P) == -1 and _forward(lib, su=P) == -1
    assert _forward(lib, sg=P, su=P + 4) == -2 and _forward(lib, y=P + 2) == -2
    for name in ("dy", "sg", "su", "dx", "dg", "du", "dd"):
        assert _backward(lib, **{name: None}) == -1, name
        assert _backward(lib, **{name: P + 4}) == -2, name


def test_gradients_over_inputs_or_one_another(lib):
    apart = {n: P + (i << 16) for i, n in enumerate(("dy", "x", "gate", "up", "down", "sg", "su", "dx", "dg", "du", "dd"))}
    sizes = dict(dy=512, x=512, gate=12288, up=12288, down=12288, sg=1536, su=1536, dx=512, dg=12288, du=12288, dd=12288)
    for out in ("dx", "dg", "du", "dd"):
        for other in apart:
            if other != out:
                assert _backward(lib, **{**apart, out: apart[other]}) == -2, (out, other)
                assert _backward(lib, **{**apart, out: apart[other] + sizes[other] - 16}) == -2, (out, other)


def test_adapters_of_the_block(lib):
    from ateniaengine_b200 import _lib
    def call(**kw):
        return _forward(lib, adapters=C.byref(_lib.FfnAdapters(**{**dict(gate=_low(), up=_low(), down=_low(), ids=P, n=2), **kw})))
    assert call(ids=None) == -1 and call(n=0) == -2 and call(n=65537) == -2
    for part in ("gate", "up", "down"):
        for rank in (-8, 4, 12, 136):
            assert call(**{part: _low(rank)}) == -2
        for name in ("a", "b", "scale"):
            assert call(**{part: _low(**{name: None})}) == -1
        assert call(**{part: _low(a=P + 2)}) == -2


def test_linear(lib):
    for bad in (dict(T=-1), dict(n_in=8), dict(n_in=72), dict(n_out=40), dict(n=0), dict(n=65537), dict(low=_low(0)), dict(low=_low(7)),
                dict(low=_low(136)), dict(low=_low(b=P + 8)), dict(x=P + 2), dict(y=P + (1 << 20) + 8), dict(ws=P + 4)):
        assert _linear(lib, **bad) == -2, bad
    for bad in (dict(low=None), dict(w=None), dict(x=None), dict(ids=None), dict(y=None), dict(ws=None), dict(low=_low(a=None)),
                dict(low=_low(scale=None))):
        assert _linear(lib, **bad) == -1, bad
    assert _linear(lib, y=P) == -2 and _linear(lib, y=P + 4 * 64 * 2 - 16) == -2  # over the input
    assert _linear(lib, nbytes=63) == -3
    assert _linear(lib, T=0, x=None, y=None, ws=None, ids=None) == 0


def test_no_tokens_need_no_rows(lib):
    assert _forward(lib, T=0, x=None, y=None, ws=None) == 0


def test_workspace_bytes(lib):
    from ateniaengine_b200 import _lib
    f = lib.atenia_gated_ffn_workspace_bytes
    assert f(4, 24, 96, None, 0) == 0 and f(-1, 64, 96, None, 0) == 0 and f(0, 64, 96, None, 0) == 0
    assert f(100, 64, 96, None, 0) >= 100 * 96 * 2 and f(100, 64, 96, None, 1) >= 3 * 100 * 96 * 2
    with_ranks = f(100, 64, 96, C.byref(_lib.FfnAdapters(gate=_low(8), up=_low(16))), 0)
    assert with_ranks >= f(100, 64, 96, None, 0) + 100 * 24 * 2
    assert f(1 << 24, 64, 1 << 20, None, 0) >= (1 << 45)
    g = lib.atenia_adapter_linear_workspace_bytes
    assert g(100, 16) >= 3200 and g(100, 12) == 0 and g(-1, 16) == 0


def test_python_entries_refuse_what_is_no_cuda_bf16_matrix():
    from ateniaengine_b200 import LowRankAdapters, adapter_linear, gated_ffn, gated_ffn_backward
    b = torch.bfloat16
    x, w = torch.zeros((4, 64), dtype=b), (torch.zeros((96, 64), dtype=b), torch.zeros((96, 64), dtype=b), torch.zeros((64, 96), dtype=b))
    low = LowRankAdapters(torch.zeros((2, 8, 64), dtype=b), torch.zeros((2, 96, 8), dtype=b), torch.zeros(2))
    ids = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(TypeError):
        gated_ffn(x.float(), *w)
    with pytest.raises(TypeError):
        gated_ffn(None, *w)
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn(x, *w)
    with pytest.raises(ValueError):
        gated_ffn(x[0], *w)
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn_backward(x, x, *w, torch.zeros((2, 4, 96)))
    with pytest.raises(ValueError, match="CUDA"):
        adapter_linear(x, w[0], low, ids)


@pytest.mark.gpu
def test_python_entries_refuse_shapes_types_and_devices():
    from ateniaengine_b200 import LowRankAdapters, adapter_linear, gated_ffn, gated_ffn_backward
    def z(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device="cuda")
    x, g, u, d = z(4, 64), z(96, 64), z(96, 64), z(64, 96)
    low, low_d = LowRankAdapters(z(2, 8, 64), z(2, 96, 8), z(2, dtype=torch.float32)), LowRankAdapters(z(3, 8, 96), z(3, 64, 8), z(3, dtype=torch.float32))
    ids = z(4, dtype=torch.int32)
    for call in (lambda: gated_ffn(x, g[:, :48], u, d), lambda: gated_ffn(x, g, u[:80], d), lambda: gated_ffn(x, g, u, d.T),
                 lambda: gated_ffn(x, g, u, d.cpu()), lambda: gated_ffn(x[:, :40], g[:, :40], u[:, :40], d[:40]),
                 lambda: gated_ffn(x, g, u, d, out=z(5, 64)), lambda: gated_ffn(x, g, u, d, out=z(4, 128)[:, :64]),
                 lambda: gated_ffn(x, g, u, d, out=z(4, 64, dtype=torch.float32)), lambda: gated_ffn(x, g, u, d, adapter_ids=ids),
                 lambda: gated_ffn(x, g, u, d, adapters={"gate": low}, adapter_ids=ids, save=True),
                 lambda: gated_ffn(x, g, u, d, adapters={"router": low}, adapter_ids=ids),
                 lambda: gated_ffn(x, g, u, d, adapters={"gate": low, "down": low_d}, adapter_ids=ids),
                 lambda: gated_ffn(x, g, u, d, adapters={"down": low}, adapter_ids=ids),
                 lambda: adapter_linear(x, g, low, ids[:3]), lambda: adapter_linear(x, g, low, ids.cpu()),
                 lambda: adapter_linear(x, g, LowRankAdapters(low.a[:, :4], low.b[:, :, :4], low.scale), ids),
                 lambda: adapter_linear(x, g, low._replace(scale=low.scale[:1]), ids),
                 lambda: adapter_linear(x, g, low._replace(b=low.b[:1]), ids),
                 lambda: gated_ffn_backward(x[:3], x, g, u, d, z(2, 24, 4, 4, dtype=torch.float32)),
                 lambda: gated_ffn_backward(x, x, g, u, d, z(2, 24, 3, 4, dtype=torch.float32))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: gated_ffn(x, g.float(), u, d), lambda: gated_ffn(x, g, u, d, adapters={"gate": low}),
                 lambda: adapter_linear(x, g, low, ids.long()), lambda: adapter_linear(x, g, low._replace(scale=low.scale.double()), ids),
                 lambda: gated_ffn_backward(x, x, g, u, d, z(2, 24, 4, 4))):
        with pytest.raises(TypeError):
            call()
    from ateniaengine_b200._lib import AteniaError
    square = z(64, 64)
    square_low = LowRankAdapters(z(2, 8, 64), z(2, 64, 8), z(2, dtype=torch.float32))
    with pytest.raises(AteniaError):
        adapter_linear(x, square, square_low, ids, out=x)
