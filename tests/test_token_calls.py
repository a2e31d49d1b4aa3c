"""The token operators' host code over a CUDA runtime of notes (tests/cpp/fake_cuda.hpp): the order of a handle's calls, what a call
leaves that breaks off, what threads share. Runs without a GPU: no kernel is launched."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from oxidizr_b200 import build as library

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CPP = os.path.join(ROOT, "tests", "cpp")
OUT = os.path.join(CPP, "_build")
EXE = os.path.join(OUT, "test_token_calls")


def build():
    """The operators' sources and the test, with the host code under the thread sanitizer; the kernels' code is never run and is
    compiled without optimisation."""
    cu = [os.path.join(library.CSRC, f) for f in ("oxz_embed.cu", "oxz_head.cu")]
    test = [os.path.join(CPP, f) for f in ("test_token_calls.cpp", "fake_cuda.hpp")]
    used = [os.path.join(library.CSRC, f) for f in os.listdir(library.CSRC) if f.endswith((".h", ".cuh"))]
    newest = max(os.path.getmtime(f) for f in [*cu, *test, *used, os.path.join(ROOT, "include", "oxz_dpstep.h")])
    if os.path.exists(EXE) and os.path.getmtime(EXE) >= newest:
        return
    os.makedirs(OUT, exist_ok=True)
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    nvcc = library._nvcc()
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    objects = [os.path.join(OUT, os.path.basename(f) + ".calls.o") for f in cu]
    cmds = [[nvcc, "-gencode", "arch=compute_100a,code=compute_100a", "-Xcicc", "-O0", "-std=c++17", "-Xcompiler", "-fsanitize=thread,-g,-O1", *library._host_compiler(),
             "-c", "-o", o, f] for f, o in zip(cu, objects)]
    cmds.append([cxx, "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=thread", f"-I{include}", "-c", "-o", EXE + ".o", test[0]])
    with ThreadPoolExecutor() as pool:
        list(pool.map(lambda c: subprocess.run(c, check=True), cmds))
    subprocess.run([cxx, "-fsanitize=thread", "-o", EXE, EXE + ".o", *objects, "-pthread"], check=True)


def run(name):
    build()
    out = subprocess.run([EXE, name], capture_output=True, text=True, timeout=300)
    if "FATAL: ThreadSanitizer" in out.stderr:
        pytest.skip("the thread sanitizer does not start on this machine: " + out.stderr.strip().splitlines()[0])
    assert out.returncode == 0 and "all passed" in out.stdout, out.stdout[-4000:] + out.stderr[-4000:]


def test_an_error_is_reported_once():
    run("error")


def test_the_next_call_waits_for_one_that_broke_off():
    run("broke_off")


def test_the_first_failure_is_the_one_reported():
    run("first")


def test_marks_are_taken_away_after_a_call_that_broke_off():
    run("marks")


def test_threads_with_a_handle_each_share_nothing_that_is_written():
    run("threads")


def test_a_handful_of_rows_takes_no_workspace_for_tiles():
    run("handful")
