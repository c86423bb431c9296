"""The C++ mirrors of routing from logits and of products with 4-bit weights (include/shrike.hpp, LogitRouter and AffineProduct), built with g++ against
the library alone: their refusals on the host, and each call on the GPU on numbers whose result is known."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(tmp_path):
    exe = tmp_path / "logit_routing_harness"
    libdir = os.path.join(ROOT, "shrike_amd")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "logit_routing_harness.cpp"),
                    "-o", str(exe), "-L", libdir, "-lshrikehip", f"-Wl,-rpath,{libdir}", "-Wl,-rpath,/opt/rocm/lib"], check=True)
    return exe


def run(*command):
    out = subprocess.run([str(c) for c in command], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "all checks passed" in out.stdout


def test_the_mirror_refuses_what_the_library_refuses(tmp_path):
    run(build(tmp_path))


@pytest.mark.gpu
def test_the_mirror_s_calls_on_the_gpu(gpu, tmp_path):
    run(build(tmp_path), "gpu")
