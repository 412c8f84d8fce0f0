"""The error word that the calls without a handle share on a device (csrc/error_word.cuh): a check takes what is there, once."""
import ctypes as C
import os
import subprocess
import threading

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def take(tmp_path_factory):
    from ateniaengine_b200.csrc import build
    so = tmp_path_factory.mktemp("error_word") / "liberrorword.so"
    subprocess.check_call([build.NVCC, *build.FLAGS[:2], "-O2", "-std=c++17", "-ccbin", "g++", "-Xcompiler", "-fPIC", "-shared",
                           os.path.join(ROOT, "tests", "error_word_probe.cu"), "-o", str(so)])
    lib = C.CDLL(str(so))

    def call(word, taken, stream):
        code, site = C.c_int(), C.c_int()
        assert lib.probe_take(C.c_void_p(word.data_ptr()), C.c_void_p(taken.data_ptr()), C.c_void_p(stream.cuda_stream), C.byref(code),
                              C.byref(site)) == 0
        return code.value, site.value

    return call


def test_a_check_takes_the_error(take):
    word, taken = torch.tensor([-7, 2103], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream()
    assert take(word, taken, stream) == (-7, 2103)
    assert word[0].item() == 0 and take(word, taken, stream)[0] == 0
    word[0] = -9  # (the next one)
    assert take(word, taken, stream)[0] == -9


def test_of_many_checks_one_has_the_error(take):
    """Eight threads with streams of their own check at the same time, 40 times: each error is returned once, by one of them."""
    word, taken = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    rounds, n = 40, 8
    begin, end = threading.Barrier(n + 1), threading.Barrier(n + 1)
    seen, failed = [], []

    def run():
        stream = torch.cuda.Stream()
        for _ in range(rounds):
            begin.wait()
            try:
                seen.append(take(word, taken, stream)[0])
            except AssertionError as e:
                failed.append(e)
            end.wait()

    threads = [threading.Thread(target=run) for _ in range(n)]
    for t in threads:
        t.start()
    for i in range(rounds):
        word[0] = -1 - i
        torch.cuda.synchronize()
        begin.wait()
        end.wait()
    for t in threads:
        t.join()
    assert not failed and sorted(c for c in seen if c) == [-rounds + i for i in range(rounds)]


def test_the_library_uses_it():
    from ateniaengine_b200 import _lib
    assert _lib.lib().atenia_ffn_check(C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
