// Host helpers shared by the single-GPU operators (dgn_norm.cu, dgn_experts.cu):
// error reporting, launch accounting, the device switch and alignment tests.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dgn.h"

namespace dgn {

int report_error(int code, const char* message);  // dgn_host.cu: sets dgn_last_error_string
void count_launch();                               // dgn_host.cu: dgn_launch_count

// Makes `device` current for one call and puts the caller's device back.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    err_ = cudaGetDevice(&prev_);
    if (err_ == cudaSuccess && prev_ != device) {
      err_ = cudaSetDevice(device);
      switched_ = err_ == cudaSuccess;
    }
    if (err_ != cudaSuccess) cudaGetLastError();
  }
  ~OnDevice() {
    if (switched_) cudaSetDevice(prev_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  cudaError_t error() const { return err_; }

 private:
  int prev_ = -1;
  bool switched_ = false;
  cudaError_t err_;
};

// Lets `fn` be launched with `smem` bytes of dynamic shared memory.  Without this the dynamic and the static part together
// may take 48 KiB; static parts of the kernels that have a dynamic one are below 1 KiB.  The limit belongs to the function
// and not to the launch: it is the same for every call, so that no thread lowers it between another's call and its launch.
constexpr int kMostDynamicShared = 224 << 10;  // of the 227 KiB that a block can have

inline int allow_shared(const void* fn, size_t smem) {
  if (smem <= (40 << 10)) return DGN_OK;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostDynamicShared);
  if (e == cudaSuccess) return DGN_OK;
  cudaGetLastError();
  return report_error(DGN_ERR_CUDA, cudaGetErrorString(e));
}

// One launch of `fn` on `stream`; a failure is reported and cleared.
inline int launch(const void* fn, dim3 grid, dim3 block, size_t smem, void* stream, void** args) {
  int rc = allow_shared(fn, smem);
  if (rc != DGN_OK) return rc;
  cudaError_t e = cudaLaunchKernel(fn, grid, block, args, smem, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return report_error(DGN_ERR_CUDA, cudaGetErrorString(e));
  }
  count_launch();
  return DGN_OK;
}

// The same for a kernel that reads what the launch before it on the stream has written: its
// blocks may be placed while the other's finish, and wait there (await_previous) for them all.
// Saves the gap between two short kernels.
inline int launch_behind(const void* fn, dim3 grid, dim3 block, size_t smem, void* stream, void** args) {
  int rc = allow_shared(fn, smem);
  if (rc != DGN_OK) return rc;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelExC(&config, fn, args);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return report_error(DGN_ERR_CUDA, cudaGetErrorString(e));
  }
  count_launch();
  return DGN_OK;
}

#ifdef __CUDACC__
// First statement of the kernel in front: the one behind may be placed.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;"); }
// First statement of the kernel behind: all blocks of the one in front have ended and what they wrote is there.
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

inline bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool float_dtype(int dtype) { return dtype == DGN_F16 || dtype == DGN_BF16 || dtype == DGN_F32; }

}  // namespace dgn
