"""CPU: the time limit of the product's waits, compiled for the host from the kernel's header."""
import ctypes
import os
import subprocess

import pytest

from htgs_b200 import build

SOURCE = """
#include "sequence.cuh"
// Polls at the given times until the limit is over: the number of polls it took, or -1.
extern "C" long polls(unsigned long long limit, const unsigned long long* times, long n) {
    htgs::WaitLimit wait(limit, times[0]);
    for (long i = 1; i < n; ++i) if (wait.over(times[i])) return i;
    return -1;
}
"""


@pytest.fixture(scope="module")
def polls(tmp_path_factory):
    folder = tmp_path_factory.mktemp("waits")
    (folder / "waits.cu").write_text(SOURCE)
    library = folder / "waits.so"
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-shared", "-I", build.CSRC, str(folder / "waits.cu"), "-o", str(library)], check=True)
    f = ctypes.CDLL(str(library)).polls
    f.restype = ctypes.c_long
    f.argtypes = [ctypes.c_ulonglong, ctypes.POINTER(ctypes.c_ulonglong), ctypes.c_long]
    return lambda limit, times: f(limit, (ctypes.c_ulonglong * len(times))(*times), len(times))


def test_time_in_which_the_kernel_did_not_run_is_not_counted(polls):
    begin, microsecond, second = 10 ** 18, 10 ** 3, 10 ** 9
    assert polls(2 * second, [begin, begin + 60 * second, begin + 60 * second + microsecond]) == -1
    # a minute away between any two polls of a wait that takes twenty
    assert polls(2 * second, [begin + i * 60 * second for i in range(21)]) == -1


def test_a_wait_that_polls_ends(polls):
    begin, millisecond = 10 ** 18, 10 ** 6
    assert polls(2000 * millisecond, [begin + i * millisecond for i in range(3000)]) == 2000
    assert polls(20 * millisecond, [begin + i * 1000 for i in range(30000)]) == 20000
    # however far apart the polls are, at most limit / 10 ms of them
    assert polls(2000 * millisecond, [begin + i * 3600000 * millisecond for i in range(300)]) == 200
