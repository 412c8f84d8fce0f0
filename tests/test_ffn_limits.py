"""Limits of the gated block and the adapters that the header states: what the size functions answer beyond them, on the CPU."""
import ctypes as C

import pytest

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
