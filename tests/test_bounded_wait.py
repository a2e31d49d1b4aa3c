"""The bounded waits of the loss head's products run out in seconds, with a status and a context that serves on."""
import os
import subprocess

import pytest

from oxidizr_b200 import build as library

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
EXE = os.path.join(CPP, "_build", "test_bounded_wait")


def build():
    src = [os.path.join(CPP, "test_bounded_wait.cu"), os.path.join(library.CSRC, "oxz_tcgen05.cuh")]
    if os.path.exists(EXE) and os.path.getmtime(EXE) >= max(os.path.getmtime(f) for f in src):
        return
    os.makedirs(os.path.dirname(EXE), exist_ok=True)
    subprocess.run([library._nvcc(), *library.ARCH, *library._host_compiler(), "-std=c++17", "-o", EXE, src[0]], check=True)


def test_it_builds():
    build()


@pytest.mark.gpu
def test_a_wait_for_nothing_ends_in_seconds():
    build()
    out = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    first, second, dead, complete, expired, t0, t1 = out.stdout.split()
    assert (first, second) == ("0", "0") and dead == "1" and expired == "1" and complete == "1"
    assert 0.5 < float(t0) < 15.0 and 0.5 < float(t1) < 15.0, out.stdout  # the tries are counted: the clock only says of what order they are
