// Kernel launches that report their own error code (and leave an earlier one of the thread alone), and the device
// that a call runs on.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

namespace sffft {

// Whether tensors of `size`-byte elements lie on whole elements: a kernel's access to any other address is a fault.
inline bool on_elements(size_t size, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % size != 0) return false;
  return true;
}

constexpr int kMaxShared = 227 * 1024;   // of a block on sm_100

// `smem` bytes of dynamic shared memory.  Kernels that take more than 48 KB of it have no static shared memory, which the limit
// would count too.
template <class K, class P>
cudaError_t launch(K kernel, dim3 grid, int threads, int smem, cudaStream_t st, const P& prm) {
  if (smem > 48 * 1024) {
    // A property of the kernel on the current device, which other threads' calls set too: always to the most that there
    // is, so that none takes away what another is about to launch with.  Setting it again costs under 1 us.
    const cudaError_t ce =
        cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared);
    if (ce != cudaSuccess) return ce;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, kernel, prm);
}

// Makes a call's device current and puts the caller's back at its end.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    err = cudaGetDevice(&prev_);
    // Also where it is current already: on a thread of its own that is where the device's context is bound, and a driver
    // call such as the encoding of a tensor map needs it.
    if (err == cudaSuccess) err = cudaSetDevice(device);
    back_ = err == cudaSuccess && prev_ != device;
  }
  ~DeviceScope() {
    if (back_) cudaSetDevice(prev_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t err;

 private:
  int prev_ = 0;
  bool back_ = false;
};

}  // namespace sffft
