"""What a kernel's or the driver's first use prepares (csrc/first_use.cuh): a call that skips the preparation comes behind one that has
succeeded, and one that failed is tried again.  And on a GPU the first calls of a process, made by several threads at once."""
import ctypes as C
import glob
import os
import re
import subprocess
import sys

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
    """No launcher asks for the attribute behind a flag of its own, and nothing else is marked as tried before it has been."""
    uses = 0
    for path in glob.glob(os.path.join(ROOT, "ateniaengine_b200", "csrc", "*.cu*")):
        text = re.sub(r"//.*", "", open(path, encoding="utf-8").read())
        if os.path.basename(path) != "common.cuh":
            assert "MaxDynamicSharedMemorySize" not in text, path
            uses += text.count("allow_shared_memory(ready, ")
        assert not re.search(r"static bool \w+\s*(\[|=|;)", text), path
    assert uses >= 10


FIRST_CALLS = """
import sys, threading
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import ffn_helpers as ref
from ateniaengine_b200 import adapter_linear, gated_ffn, gated_ffn_backward
n, r, jobs = 5, 16, []
for T, d, F in ((3, 272, 144), (40, 528, 1040), (40, 528, 1040), (300, 272, 400), (700, 528, 1040), (1100, 528, 1040), (1100, 272, 400), (2100, 768, 1552)):
    jobs.append((ref.rand(T, 1.0, T, d), ref.rand(T + 1, 1.0, T, d), ref.block(2, d, F), ref.low_rank(50, n, r, d, d), ref.rand(9, d ** -0.5, d, d),
                 ref.ids_of("runs", T, n)))
torch.cuda.synchronize()
start, results, failed = threading.Barrier(len(jobs)), [None] * len(jobs), []

def step(x, dy, w, low, wo, ids):
    a = adapter_linear(x, wo, low, ids, sync=True)
    y, saved = gated_ffn(a, *w, save=True)
    return [a, y, *gated_ffn_backward(dy, a, *w, saved, sync=True)]

def run(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            results[i] = step(*jobs[i])
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        failed.append((i, repr(e)))

threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not failed, failed
for job, got in zip(jobs, results):
    assert all(torch.equal(a, b) for a, b in zip(got, step(*job)))
print("alike")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_from_several_threads():
    """Each thread its own sizes and stream, straight into the first use of its kernels: the bits that each call has alone later."""
    code = FIRST_CALLS.format(root=ROOT, tests=os.path.join(ROOT, "tests"))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.split() == ["alike"], out.stdout + out.stderr
