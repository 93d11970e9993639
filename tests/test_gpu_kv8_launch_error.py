"""Test of a launch that the CUDA runtime refuses on the host (more threads than a CTA may have):
it is reported once and leaves no error behind.  Nothing runs on the device; without one the
runtime has no other error than that, so the test is marked ``gpu``."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
CSRC = Path(__file__).resolve().parent.parent / "kitty-kv_b200" / "csrc" / "kv8"

PROGRAM = r"""
#include "kv8_common.cuh"
namespace kitty8 {
int fail(int code, const char* what, const char* msg) { std::printf("%s: %s\n", what, msg); return code; }
}
__global__ void kernel(int) {}
int main() {
  cudaFree(nullptr);
  cudaGetLastError();
  const int rc = kitty8::launch_dependent("refused", kernel, dim3(1), 4096, 0, nullptr, 7);
  const cudaError_t left = cudaPeekAtLastError();
  std::printf("rc %d, left %d\n", rc, int(left));
  return rc == KITTY_ERR_CUDA && left == cudaSuccess ? 0 : 1;
}
"""


def test_a_refused_launch_leaves_no_error_behind(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("nvcc not available")
    (tmp_path / "a.cu").write_text(PROGRAM)
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", str(CSRC), "-o",
                        str(tmp_path / "a"), str(tmp_path / "a.cu")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "refused: " in r.stdout, r.stdout
