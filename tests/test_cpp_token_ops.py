"""Builds and runs the C++ mirror's token operators (tests/cpp/test_token_ops.cpp) as a compiled client of the library would."""
import os
import subprocess

import pytest

import oxidizr_b200 as ox

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "_build", "test_token_ops")


def build():
    src, hdr = os.path.join(ROOT, "tests", "cpp", "test_token_ops.cpp"), os.path.join(ROOT, "oxidizr_b200", "cpp", "oxz.hpp")
    if os.path.exists(EXE) and os.path.getmtime(EXE) >= max(os.path.getmtime(p) for p in (src, hdr, ox.ffi.LIB_PATH)):
        return
    os.makedirs(os.path.dirname(EXE), exist_ok=True)
    libdir = os.path.dirname(ox.ffi.LIB_PATH)
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", f"-I{cuda}/include", "-o", EXE, src, f"-L{libdir}", "-l:liboxz_dpstep.so",
                    f"-Wl,-rpath,{libdir}", f"-L{cuda}/lib64", "-lcudart_static", "-ldl", "-lrt", "-pthread"], check=True)


def run(*args):
    build()
    out = subprocess.run([EXE, *args], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "all passed" in out.stdout, out.stdout + out.stderr


def test_refusals_without_a_gpu():
    run()


@pytest.mark.gpu
def test_operators_on_the_gpu():
    run("--gpu")
