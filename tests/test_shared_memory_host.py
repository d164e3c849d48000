"""What a kernel may have of shared memory, asked for by several threads at once: against a runtime that takes its time, without a GPU."""
import os
import subprocess

import pytest

from flexspmv_b200 import build

SOURCE = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>

static std::atomic<int> limit{0}, asked{0};
static cudaError_t ask_device(int* device) { *device = 0; return cudaSuccess; }
// a smaller size takes longer
static cudaError_t ask(const void*, int, int bytes) {
  std::this_thread::sleep_for(std::chrono::microseconds(60 + (200 * 1024 - bytes) / 512));
  limit = bytes;
  ++asked;
  return cudaSuccess;
}
#define cudaGetDevice ask_device
#define cudaFuncSetAttribute(kernel, what, bytes) ask((const void*)kernel, what, bytes)
#include "flex_expert_types.cuh"

template <int N> __global__ void kernel() {}

template <int N> int round_of_threads() {
  limit = 0;
  std::atomic<int> begun{0}, lowered{0};
  std::vector<std::thread> threads;
  for (int t = 0; t < 6; ++t)
    threads.emplace_back([&, t] {
      const int bytes = (50 + 25 * ((t * 5 + N) % 6)) * 1024;
      ++begun;
      while (begun < 6) {}
      if (flex::allow_smem<kernel<N>>(bytes) != 0) ++lowered;
      std::this_thread::sleep_for(std::chrono::milliseconds(1));
      if (limit < bytes) ++lowered;          // as its launch finds it
    });
  for (auto& t : threads) t.join();
  if (flex::allow_smem<kernel<N>>(175 * 1024) != 0 || limit < 175 * 1024) ++lowered;
  return lowered;
}
template <int... N> int rounds(std::integer_sequence<int, N...>) { return (round_of_threads<N>() + ...); }

int main() {
  const int lowered = rounds(std::make_integer_sequence<int, 40>());
  std::printf("%d launches without their memory, %d questions\n", lowered, (int)asked);
  return lowered != 0;
}
"""


@pytest.mark.skipif(not os.path.exists(build.NVCC), reason="needs nvcc")
def test_no_size_takes_a_larger_ones_place(tmp_path):
    source, program = tmp_path / "threads.cu", tmp_path / "threads"
    source.write_text(SOURCE)
    subprocess.run([build.NVCC, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a", "-I", build.CSRC, "-o", str(program), str(source)], check=True,
                   capture_output=True, text=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout
    assert int(done.stdout.split()[-2]) <= 40 * 7
