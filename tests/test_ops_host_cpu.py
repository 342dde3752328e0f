"""Host helpers of the single-GPU operators (dgn_ops.h) over stand-ins for the CUDA calls that they make."""

import os
import subprocess

from dragon_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE_RUNTIME = r'''
#include "dragon_b200/csrc/dgn_ops.h"
#include <cstdio>
#include <map>
static std::map<const void*, int> limit;  // of each function; launches beyond it fail, as the runtime's do
static int launches, errors;
extern "C" {
cudaError_t cudaFuncSetAttribute(const void* fn, cudaFuncAttribute what, int value) {
  if (what != cudaFuncAttributeMaxDynamicSharedMemorySize || value > 226 << 10) return cudaErrorInvalidValue;
  limit[fn] = value;
  return cudaSuccess;
}
static cudaError_t start(const void* fn, size_t smem) {
  const int most = limit.count(fn) ? limit[fn] : 47 << 10;
  if (smem > (size_t)most) return cudaErrorInvalidValue;
  ++launches;
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* fn, dim3, dim3, void**, size_t smem, cudaStream_t) { return start(fn, smem); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* fn, void**) { return start(fn, c->dynamicSmemBytes); }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "error"; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
}
namespace dgn {
int report_error(int code, const char*) { ++errors; return code; }
void count_launch() {}
}
int main() {
  static char fn;
  // Two callers of one kernel: the one that wants less comes between the other's permission and its launch.
  if (dgn::allow_shared(&fn, 196608) != DGN_OK || dgn::allow_shared(&fn, 147456) != DGN_OK) return 1;
  if (start(&fn, 196608) != cudaSuccess) { puts("a smaller call lowered the limit"); return 2; }
  if (dgn::launch(&fn, 1, 1, 147456, 0, 0) || dgn::launch_behind(&fn, 1, 1, 196608, 0, 0) || dgn::launch(&fn, 1, 1, 64, 0, 0)) return 3;
  if (dgn::launch(&fn, 1, 1, 300 << 10, 0, 0) == DGN_OK || errors != 1) return 4;  // more than a block can have: an error
  return launches == 4 ? 0 : 5;
}
'''


def test_a_smaller_call_does_not_lower_the_limit_of_shared_memory(tmp_path):
    source, binary = tmp_path / "fake.cc", tmp_path / "fake"
    source.write_text(FAKE_RUNTIME)
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-I", ROOT, "-isystem", cuda, str(source), "-o", str(binary)], check=True)
    done = subprocess.run([str(binary)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
