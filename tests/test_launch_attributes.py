"""What a kernel may use of shared memory, asked for by several host threads: the
helper all launches share (csrc/common.cuh) against a runtime whose answers are
recorded.  No GPU."""

from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

from kanforge_b200.build import CSRC, INCLUDE, nvcc

SOURCE = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdarg>
#include <thread>

static std::atomic<int> granted{0}, asked{0}, small_done{0};
static void wait_for(std::atomic<int>& flag) {
  for (int i = 0; i < 300 && !flag; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
static cudaError_t fake_get_device(int* dev) { *dev = 0; return cudaSuccess; }
template <typename K>
static cudaError_t fake_set(K*, cudaFuncAttribute, int bytes) {
  ++asked;
  granted = bytes;
  if (bytes == 200) wait_for(small_done);  // the other thread runs now, if it may
  return cudaSuccess;
}
#define cudaGetDevice fake_get_device
#define cudaFuncSetAttribute fake_set
#include "common.cuh"
void kf::set_error(const char*, ...) {}
void kf::register_device_error_reader(int (*)(int*)) {}

static void kernel() {}
static kf::SmemAllowed allowed;
static int allow(size_t bytes) {
  int rc = kf::allow_smem(kernel, bytes, allowed);
  return rc != KF_OK ? -1 : granted.load();
}

int main() {
  std::thread large([] { allow(200); });
  while (!asked) std::this_thread::yield();
  std::thread small([] { allow(100); small_done = 1; });
  large.join(), small.join();
  if (allow(200) < 200) return 1;  // the limit fell below what was granted before
  if (allow(50) < 200) return 2;
  const int before = asked;
  if (allow(150) < 200 || asked != before) return 3;
  return 0;
}
"""


def test_the_limit_never_falls(tmp_path: Path):
    try:
        compiler = nvcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    src, exe = tmp_path / "limit.cu", tmp_path / "limit"
    src.write_text(SOURCE)
    cmd = [compiler, "-std=c++17", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(CSRC), "-I",
           str(INCLUDE), "-o", str(exe), str(src)]
    done = subprocess.run(cmd, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert subprocess.run([str(exe)], timeout=60).returncode == 0
