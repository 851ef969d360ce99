"""A kernel's shared-memory limit under host threads (allow_smem of csrc/common.cuh), with a stand-in for the CUDA calls.

A small host program includes the header and runs two threads: the one with the smaller size is held inside the
attribute call until the other has had its turn.  The limit must not end below what the cache of it says.
"""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
static std::atomic<size_t> limit{0};
static std::atomic<int> inside{0};
static cudaError_t fake_device(int* d) { *d = 0; return cudaSuccess; }
template <typename K>
static cudaError_t fake_set(K, cudaFuncAttribute, int bytes) {
  if (bytes == 1000) {  // the smaller size's call takes long
    inside = 1;
    std::this_thread::sleep_for(std::chrono::milliseconds(300));
  }
  limit = bytes;
  return cudaSuccess;
}
#define cudaGetDevice fake_device
#define cudaFuncSetAttribute fake_set
#include "common.cuh"
__global__ void kern() {}
static bolt::SmemOptIn opt;
int main() {
  std::thread small([] { bolt::allow_smem(kern, 1000, opt); });
  while (!inside) std::this_thread::yield();
  std::thread large([] { bolt::allow_smem(kern, 5000, opt); });
  small.join();
  large.join();
  const bool known = bolt::allow_smem(kern, 4000, opt) == cudaSuccess;  // below the largest: no call
  std::printf("%d %zu %zu\n", known, limit.load(), opt.bytes[0].load());
  return 0;
}
"""


def test_two_threads_leave_the_larger_limit(tmp_path):
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not found")
    src, exe = tmp_path / "limit.cu", tmp_path / "limit"
    src.write_text(PROGRAM)
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-rdc=true", "-diag-suppress", "177", "-I",
           os.path.join(ROOT, "nemotron_ops_b200", "csrc"), str(src), "-o", str(exe), "-lpthread"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.stdout.split() == ["1", "5000", "5000"], out.stdout + out.stderr
