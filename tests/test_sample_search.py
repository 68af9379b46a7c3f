"""CPU tests of the sampling call's searches (csrc/sample_search.cuh), compiled with g++: they find
what they should and end after a bounded number of steps."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_searches_end(tmp_path):
    exe = tmp_path / "sample_search_tests"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-ffp-contract=off",
                    "-I", os.path.join(ROOT, "neuraval_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "sample_search_tests.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
