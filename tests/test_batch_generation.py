"""The decode loop for many requests (TextGenerator::GenerateBatch in
neuraval_b200/host/neuraval_generation.hpp): the LM head with each request's adapter
and sampling with each request's options, over a toy model, compiled with g++."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _build(tmp_path):
    from neuraval_b200 import build
    libdir = os.path.dirname(build.build())
    exe = tmp_path / "batch_generation_tests"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra",
                    "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "neuraval_b200", "host"),
                    "-I", os.path.join(CUDA, "include"),
                    os.path.join(ROOT, "tests", "cpp", "batch_generation_tests.cpp"),
                    "-L", libdir, "-lnavsampler", f"-Wl,-rpath,{libdir}",
                    "-L", os.path.join(CUDA, "lib64"), "-lcudart", f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}",
                    "-o", str(exe)], check=True)
    return exe


def test_refusals_without_gpu(tmp_path):
    r = subprocess.run([str(_build(tmp_path)), "--refusals-only"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_batch_generation_on_gpu(tmp_path):
    r = subprocess.run([str(_build(tmp_path))], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
