"""The choice of a dense product's kernel (csrc/dense_choice.cuh), compiled for the host: every plan is one the kernels can run, and of calls
that were measured with several kernels the one taken is near the fastest."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FORWARD, DOWN, GATE_GRAD, DX, DW = range(5)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("choice") / "libdensechoice.so"
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", os.path.join(ROOT, "tests", "dense_choice_probe.cpp"),
                           "-o", str(so)])
    return C.CDLL(str(so))


@pytest.fixture(scope="module")
def plan(lib):
    def blocks(k):
        return -(-k // 64)

    def call(kind, T, d, F, adapters=0, sms=148):
        if kind == DW:
            sizes, rows = [F, d, blocks(T), F, d, blocks(T), d, F, blocks(T)], 128
        else:
            sizes = {FORWARD: [T, F, blocks(d)], DOWN: [T, d, blocks(F)], GATE_GRAD: [T, F, blocks(d)], DX: [T, d, 2 * blocks(F)]}[kind]
            rows = min(128, -(-T // 8) * 8)
        out = (C.c_int * 4)()
        lib.choice_dense((C.c_longlong * 9)(*sizes), len(sizes) // 3, rows, kind == FORWARD, kind == GATE_GRAD, rows == 128, adapters, sms, out)
        return tuple(out) + (min(sizes[2::3]), rows)

    return call


def test_every_plan_can_be_run(plan):
    rng = random.Random(7)
    for _ in range(4000):
        T, d, F = (max(1, int(2 ** rng.uniform(0, hi))) for hi in (24, 16, 17))
        d, F = max(16, d // 16 * 16), max(16, F // 16 * 16)
        kind = rng.randrange(5)
        pairs, columns, split, tail, kb, rows = plan(kind, T, d, F, rng.choice([0, 0, 1, 40, 65536]), rng.choice([148, 148, 132, 80]))
        assert 1 <= split <= kb and 1 <= tail <= kb
        if pairs:
            assert rows == 128 and split <= 4 and tail <= 4 and (split == 1 or tail == 1)
        else:
            assert columns in (128, 256) and split in (1, 2, 3, 4, 6, 8) and tail == 1


# kind, tokens, d, F and us by (pairs, columns, split), on a B200 with weights out of L2
MEASURED = [
    (FORWARD, 8, 2048, 2816, {(0, 128, 3): 7.7, (0, 128, 6): 8.0, (0, 128, 2): 8.4, (0, 256, 4): 8.8}),
    (FORWARD, 64, 4096, 14336, {(0, 128, 1): 40.9, (0, 256, 1): 42.1, (0, 128, 2): 45.1, (0, 128, 4): 57.3}),
    (FORWARD, 333, 2048, 5632, {(0, 256, 1): 17.3, (0, 128, 1): 18.1, (1, 256, 1): 25.8, (0, 128, 2): 26.8}),
    (FORWARD, 1021, 2048, 5632, {(1, 256, 1): 36.7, (0, 256, 1): 45.5, (0, 128, 1): 46.4, (1, 256, 2): 76.9}),
    (DOWN, 8, 4096, 14336, {(0, 128, 4): 22.8, (0, 128, 6): 23.2, (0, 128, 8): 23.3, (0, 128, 2): 28.0}),
    (DOWN, 64, 512, 1408, {(0, 128, 4): 5.0, (0, 128, 6): 5.1, (0, 128, 8): 5.2, (0, 128, 1): 5.8}),
    (DOWN, 333, 4096, 14336, {(1, 256, 2): 45.4, (0, 256, 2): 49.3, (0, 256, 4): 57.4, (1, 256, 3): 62.2}),
    (DOWN, 512, 2048, 5632, {(0, 256, 4): 17.4, (0, 128, 4): 18.1, (1, 256, 3): 18.8, (0, 256, 3): 18.9, (1, 256, 4): 31.0}),
    (GATE_GRAD, 64, 2048, 2816, {(0, 128, 4): 8.3, (0, 128, 6): 8.8, (0, 128, 3): 9.6, (0, 256, 4): 9.9}),
    (GATE_GRAD, 256, 4096, 14336, {(1, 256, 1): 39.4, (0, 256, 1): 47.4, (0, 128, 1): 49.4, (0, 128, 2): 60.1}),
    (DX, 256, 2048, 5632, {(0, 256, 6): 21.0, (0, 128, 8): 21.0, (0, 128, 6): 22.0, (1, 256, 4): 23.3}),
    (DX, 1024, 2048, 2816, {(0, 256, 2): 23.2, (1, 256, 2): 23.4, (0, 128, 2): 24.9, (1, 256, 1): 31.5}),
    (DW, 64, 4096, 14336, {(1, 256, 1): 85.2, (0, 128, 1): 179.0, (0, 256, 1): 208.0}),
]


@pytest.mark.parametrize("kind,T,d,F,us", MEASURED)
def test_the_kernel_taken_is_near_the_fastest(plan, kind, T, d, F, us):
    taken = plan(kind, T, d, F)[:3]
    assert us[taken] <= 1.1 * min(us.values()), (taken, us)


def test_a_last_wave_of_few_tiles_is_cut(plan):
    """5000 x 2048 over 5632: 160 tiles on 74 pairs of SMs."""
    for adapters in (0, 9):
        assert plan(DOWN, 5000, 2048, 5632, adapters)[:2] == (1, 256) and plan(DOWN, 5000, 2048, 5632, adapters)[3] > 1


def test_pieces_of_a_few_rows(lib):
    """Every row group has its warps, every piece its steps; a small matrix is cut as far as that goes, a large one hardly."""
    out = (C.c_int * 2)()

    def rows(groups, steps, places):
        lib.choice_rows(groups, steps, 8, places, out)
        return tuple(out)

    for groups in [*range(1, 70), 128, 1000, 65536, 131072]:
        for steps in [1, 2, 3, 4, 7, 8, 16, 33, 16384]:
            for places in (80, 296, 444):
                pieces, blocks = rows(groups, steps, places)
                assert pieces in (1, 2, 4, 8) and (pieces == 1 or steps >= 2 * pieces)
                assert (blocks - 1) * (8 // pieces) < groups <= blocks * (8 // pieces)
    assert rows(2, 1, 296) == (1, 1) and rows(1, 16384, 296) == (1, 1)
    assert rows(176, 8, 296) == (4, 88) and rows(65536, 64, 444)[0] <= 2


def test_cut_and_lanes_of_the_reduced_rows(lib):
    out = (C.c_int * 2)()

    def reduce(rows, kb, n, per_pass, projections=1):
        tiles = -(-rows // 128) * projections
        lib.choice_reduce(C.c_longlong(rows), C.c_longlong(tiles), kb, n, per_pass, 148, out)
        split, lanes = out
        assert split in (1, 2, 4, 8) and (split == 1 or kb >= 2 * split) and 1 <= lanes <= max(1, -(-min(n, rows, 128) // per_pass))
        assert tiles * split * lanes < 1 << 31
        return split, lanes

    for rows in (1, 17, 128, 129, 500, 513, 5000, 1 << 24):
        for kb in (1, 2, 3, 16, 64, 16384):
            for n in (1, 3, 90, 65536):
                for per_pass in (1, 2, 16):
                    reduce(rows, kb, n, per_pass, 2)
    assert reduce(1100, 32, 16, 2) == (8, 4) and reduce(2000, 16, 60, 1) == (4, 4)
