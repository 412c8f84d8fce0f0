"""What a kernel's first use prepares (csrc/first_use.cuh): a call that skips the preparation comes behind one that has succeeded, and one
that failed is tried again."""
import ctypes as C
import glob
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("first_use") / "libfirstuse.so"
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-pthread", "-shared", "-fPIC", os.path.join(ROOT, "tests", "first_use_probe.cpp"),
                           "-o", str(so)])
    return C.CDLL(str(so))


@pytest.mark.parametrize("threads", [2, 8])
def test_nobody_goes_on_before_the_preparation_has_succeeded(lib, threads):
    assert lib.first_use_too_early(threads, 50) == 0


def test_a_failure_is_returned_and_tried_again(lib):
    wrong = C.c_int()
    assert lib.first_use_runs(5, 0, C.byref(wrong)) == 1 and wrong.value == 0
    assert lib.first_use_runs(5, 2, C.byref(wrong)) == 3 and wrong.value == 0


def test_every_kernel_with_much_shared_memory_uses_it():
    """No launcher asks for the attribute behind a flag of its own."""
    uses = 0
    for path in glob.glob(os.path.join(ROOT, "ateniaengine_b200", "csrc", "*.cu*")):
        text = re.sub(r"//.*", "", open(path, encoding="utf-8").read())
        if os.path.basename(path) != "common.cuh":
            assert "MaxDynamicSharedMemorySize" not in text, path
            uses += text.count("allow_shared_memory(ready, ")
    assert uses >= 10
