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
