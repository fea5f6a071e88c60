"""The dynamic shared-memory limit of a kernel that several threads launch with several sizes: what is
noted as set is what was set. Host code alone, with a stand-in for the CUDA calls."""

from __future__ import annotations

import os
import subprocess

from conftest import REPO

HARNESS = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

#include "common.cuh"

static std::atomic<int> attribute{0};

static void nap(int ms) { std::this_thread::sleep_for(std::chrono::milliseconds(ms)); }

extern "C" cudaError_t __wrap_cudaGetDevice(int* device) {
  *device = 0;
  return cudaSuccess;
}

// the larger size takes effect at once and returns late, the smaller one takes effect late
extern "C" cudaError_t __wrap_cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
  if (bytes < 200000) nap(50);
  attribute = bytes;
  if (bytes >= 200000) nap(200);
  return cudaSuccess;
}

int main() {
  for (int first : {200000, 100000}) {
    int done[vfl::kMaxDevices] = {};
    attribute = 0;
    std::thread a([&] { vfl::ensure_smem_attribute(nullptr, first, done); });
    nap(10);
    std::thread b([&] { vfl::ensure_smem_attribute(nullptr, 300000 - first, done); });
    a.join();
    b.join();
    std::printf("noted %d, set %d\n", done[0], attribute.load());
    if (done[0] != 200000 || attribute != 200000) return 1;
  }
  return 0;
}
"""


def test_limit_noted_is_the_limit_set(tmp_path):
    from vflorence_b200 import build

    src = tmp_path / "harness.cu"
    src.write_text(HARNESS)
    exe = str(tmp_path / "harness")
    cmd = [build._nvcc(), *build.NVCC_FLAGS, "-Xlinker", "--wrap=cudaGetDevice", "-Xlinker", "--wrap=cudaFuncSetAttribute",
           str(src), os.path.join(REPO, "vflorence_b200", "csrc", "capi.cu"), "-o", exe, "-lpthread"]
    made = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout
