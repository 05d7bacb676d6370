"""The record of how many clusters a device holds (common.cuh), compiled against stand-ins for
the CUDA runtime: two threads' first questions at once, and a question that fails."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

# cudaFuncSetAttribute and cudaOccupancyMaxActiveClusters stand for the runtime's:
# a question about more shared memory than the kernel's limit of the moment is an error.
RUNTIME = r"""
#include <atomic>
#include <chrono>
#include <thread>
#include <cuda_runtime_api.h>

std::atomic<int> limit{0}, asked{0}, sets{0}, fail{0};

// (the program holds no kernels to register)
extern "C" void** __cudaRegisterFatBinary(void*) { return nullptr; }
extern "C" void __cudaRegisterFatBinaryEnd(void**) {}
extern "C" void __cudaUnregisterFatBinary(void**) {}
extern "C" char __cudaInitModule(void**) { return 0; }
extern "C" cudaError_t cudaGetLastError() { return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int v) {
  limit = v;
  ++sets;
  return cudaSuccess;
}
extern "C" cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t* c) {
  ++asked;
  if (fail > 0) {
    --fail;
    return cudaErrorUnknown;
  }
  // as long as another thread could set its own limit here, let it
  const int seen = sets;
  for (int i = 0; i < 200 && sets == seen; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  if ((int)c->dynamicSmemBytes > limit) return cudaErrorInvalidValue;
  *n = (int)(c->dynamicSmemBytes / 1000) + (int)c->gridDim.x;
  return cudaSuccess;
}
"""

PROGRAM = r"""
#include <cstdio>
#include <thread>
#include "common.cuh"

std::mutex& tsds_host_cache_lock() { static std::mutex m; return m; }
void tsds_count_launch() {}
extern std::atomic<int> asked, fail;

int main() {
  static tsds_cluster_counts large, small, other;
  void (*kernel)() = nullptr;
  auto ask = [&](size_t smem, tsds_cluster_counts& known) {
    return tsds_resident_clusters(0, kernel, 192, smem, 4, known);
  };
  int a = -1, b = -1;
  std::thread t([&] { a = ask(220000, large); });
  while (asked == 0) std::this_thread::yield();
  b = ask(70000, small);
  t.join();
  const int again_a = ask(220000, large), again_b = ask(70000, small);
  fail = 1;
  const int failed = ask(110000, other), after = ask(110000, other), calls = asked;
  ask(110000, other);
  std::printf("%d %d %d %d %d %d %d\n", a, b, again_a, again_b, failed, after, (int)asked - calls);
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no nvcc")
def test_first_questions_of_two_threads_and_a_failed_one(tmp_path):
    src, rt, exe = tmp_path / "counts.cu", tmp_path / "runtime.cpp", tmp_path / "counts"
    src.write_text(PROGRAM)
    rt.write_text(RUNTIME)
    csrc = os.path.join(ROOT, "tri_sds_b200", "csrc")
    r = subprocess.run([NVCC, "-std=c++17", "-I", csrc, "-cudart", "none", str(src), str(rt), "-o", str(exe)], capture_output=True,
                       text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    assert [int(v) for v in out.stdout.split()] == [224, 74, 224, 74, 0, 114, 0]
