// What a launcher asks of the CUDA runtime once for each device of the process,
// where a function-local static would ask for the first device alone.
#pragma once

#include <atomic>

namespace grx {

constexpr int kMostDevices = 64;

// One per launcher, static: zero at first.
struct PerDevice {
  std::atomic<int> known[kMostDevices];

  // What `ask` (a positive int; anything else is a failure, which is not kept)
  // answers on `device`, asked there once. Threads that come at the same time
  // may ask twice.
  template <typename Ask>
  int get(int device, Ask ask) {
    const bool in_range = device >= 0 && device < kMostDevices;
    if (in_range)
      if (const int v = known[device].load(std::memory_order_acquire)) return v;
    const int v = ask();
    if (in_range && v > 0) known[device].store(v, std::memory_order_release);
    return v;
  }
};

}  // namespace grx

#ifdef __CUDACC__
#include <cuda_runtime.h>

namespace grx {

// Lets `kernel` use `bytes` of dynamic shared memory on the current device.
template <typename Kernel>
cudaError_t allow_shared_memory(PerDevice& allowed, Kernel kernel, int bytes) {
  int device = -1;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  allowed.get(device, [&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) cudaGetLastError();  // it is in the answer, and no later call's
    return e == cudaSuccess ? 1 : -1;
  });
  return e;
}

// CTAs of `kernel` that share an SM of the current device, at least 1.
template <typename Kernel>
int resident_ctas(PerDevice& counted, Kernel kernel, int threads, int smem) {
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess) return 1;
  const int n = counted.get(device, [&] {
    int ctas = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, threads, smem) == cudaSuccess) return ctas;
    cudaGetLastError();
    return 0;
  });
  return n > 0 ? n : 1;
}

}  // namespace grx
#endif
