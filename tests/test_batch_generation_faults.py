"""TextGenerator::GenerateBatch where something goes wrong for one of its requests or for the head
(tests/cpp/batch_generation_faults_tests.cpp), compiled with g++."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _build(tmp_path):
    from neuraval_b200 import build
    libdir = os.path.dirname(build.build())
    exe = tmp_path / "batch_generation_faults_tests"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra",
                    "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "neuraval_b200", "host"),
                    "-I", os.path.join(CUDA, "include"),
                    os.path.join(ROOT, "tests", "cpp", "batch_generation_faults_tests.cpp"),
                    "-L", libdir, "-lnavsampler", f"-Wl,-rpath,{libdir}",
                    "-L", os.path.join(CUDA, "lib64"), "-lcudart", "-ldl", f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}",
                    "-o", str(exe)], check=True)
    return exe


def test_without_gpu(tmp_path):
    r = subprocess.run([str(_build(tmp_path)), "--no-gpu"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_on_gpu(tmp_path):
    r = subprocess.run([str(_build(tmp_path))], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
