"""The paged-cache kernels' index arithmetic (vox_amd/csrc/vh_paged_index.hpp), compiled for the host and checked there
(tests/cpp/paged_index_check.cpp): no GPU needed."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_index_arithmetic(tmp_path):
    exe = str(tmp_path / "paged_index_check")
    src = os.path.join(ROOT, "tests", "cpp", "paged_index_check.cpp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I" + os.path.join(ROOT, "vox_amd", "csrc"), src, "-o", exe],
                   check=True, capture_output=True, timeout=120)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    assert "all passed" in r.stdout
