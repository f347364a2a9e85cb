"""A kernel's limit of shared memory is raised once on each device, and again after a failure: the header by itself, with stand-ins for the runtime."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
PROGRAM = r"""
#include "device_once.h"
#include <cstdio>
static int device = 0, fail = 0;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
  std::printf("%d:%d ", device, bytes);
  return fail ? cudaErrorInvalidValue : cudaSuccess;
}
int main() {
  std::atomic<uint64_t> one{0}, two{0};
  const int devices[] = {0, 0, 1, 0, 1, 70, 70};
  for (int d : devices) { device = d; if (vb_allow_smem(nullptr, 5, one) != cudaSuccess) return 1; }
  device = 3; fail = 1;
  if (vb_allow_smem(nullptr, 6, two) == cudaSuccess) return 2;
  fail = 0;
  for (int i = 0; i < 2; ++i) if (vb_allow_smem(nullptr, 6, two) != cudaSuccess) return 3;
}
"""


@pytest.mark.skipif(not shutil.which("g++") or not os.path.exists(f"{CUDA}/include/cuda_runtime_api.h"), reason="a host compiler and the runtime's header")
def test_each_device_once(tmp_path):
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-I", f"{CUDA}/include", str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    got = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, check=True).stdout
    assert got.split() == ["0:5", "1:5", "70:5", "70:5", "3:6", "3:6"]


@pytest.mark.parametrize("name", ["key_weights.cu", "scored_decode.cu"])
def test_no_kernel_asks_once_a_process(name):
    with open(os.path.join(CSRC, name)) as f:
        assert "static bool" not in f.read()
