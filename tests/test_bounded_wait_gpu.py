"""The waits inside the head's kernels end (csrc/bounded_wait.cuh), and the head says whether one did."""
import os
import subprocess

import pytest

from neuraval_b200 import build, native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def compiled(tmp_path):
    exe = tmp_path / "bounded_wait_tests"
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "-I", os.path.join(ROOT, "neuraval_b200", "csrc"),
                    "-o", str(exe), os.path.join(ROOT, "tests", "cpp", "bounded_wait_tests.cu")], check=True)
    return exe


def test_status_without_a_head(navlib):
    assert navlib.ncb_adapter_head_status(None) == native.NCB_ERROR_NOT_INITIALIZED


def test_the_waits_compile(tmp_path):
    compiled(tmp_path)


@pytest.mark.gpu
def test_a_wait_that_nothing_answers_ends(tmp_path):
    r = subprocess.run([str(compiled(tmp_path))], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_status_of_a_head_that_works():
    import torch
    from neuraval_b200.adapter_head import CudaAdapterHead
    w = torch.ones(300, 64, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros(3, 300, device="cuda")
    with CudaAdapterHead(w, 4, 2, 8) as h:
        h.check()
        h.project_device(w[:3], torch.zeros(3, device="cuda", dtype=torch.int32), y)
        torch.cuda.synchronize()
        h.check()
    assert (y == 64).all()
    with CudaAdapterHead(w, 4) as h:  # no slots
        h.project_device(w[:3], None, y)
        torch.cuda.synchronize()
        h.check()
