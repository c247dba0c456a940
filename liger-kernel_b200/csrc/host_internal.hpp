// What the host sides of the library's translation units share.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "flce_b200.h"

namespace flce {

// keeps the message for flce_b200_last_error() (per thread) and returns `code`
int fail(int code, const char* fmt, ...);

#define FLCE_CUDA(expr)                                                                             \
  do {                                                                                              \
    cudaError_t e__ = (expr);                                                                       \
    if (e__ != cudaSuccess) return fail(FLCE_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e__)); \
  } while (0)

// adds to what flce_b200_kernel_launches() reports
void count_launches(int n);

// SM count of the current device; FLCE_ERR_UNSUPPORTED unless it is an sm_100 one.  Touches no device memory and no
// stream, so the first call on a device may come while a stream is being captured.
int current_sm_count(int* sm_count);

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline int element_size(int dtype) { return dtype == FLCE_FP32 ? 4 : 2; }

// A launch that the host emulation of the tests can stand in for.  `kernel` is parenthesised: it holds commas.
#ifndef FLCE_HOST_EMULATION
#define FLCE_LAUNCH(kernel, grid, block, stream, ...) kernel<<<grid, block, 0, stream>>>(__VA_ARGS__)
#else
#define FLCE_LAUNCH(kernel, grid, block, stream, ...) \
  emu::launch(emu_dim3(grid), emu_dim3(block), [&]() { (void)(stream), (kernel)(__VA_ARGS__); })
#endif

// A launch that may start while the kernel in front of it drains; the kernel calls wait_for_previous_kernel() first.
template <auto kKernel, class... Args>
static int launch_dependent(dim3 grid, dim3 block, cudaStream_t stream, const Args&... args) {
#ifndef FLCE_HOST_EMULATION
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  FLCE_CUDA(cudaLaunchKernelEx(&config, kKernel, args...));
#else
  FLCE_LAUNCH((kKernel), grid, block, stream, args...);
#endif
  return FLCE_OK;
}

// A launch with `bytes` of dynamic shared memory; the permission for more than 48 KB is asked for once per kernel
// and device (kKernel names the instantiation).  The function is static so that what it remembers belongs to this library: the
// permission is one for the kernel in this library, not for that of another copy in the process.
constexpr int kMostDynamicShared = 220 * 1024;      // beside what such a kernel declares statically: 227 KB in all
template <auto kKernel, class... Args>
static int launch_with_shared(dim3 grid, unsigned block, size_t bytes, cudaStream_t stream, const Args&... args) {
#ifndef FLCE_HOST_EMULATION
  static std::atomic<bool> allowed[64];
  int device = 0;
  FLCE_CUDA(cudaGetDevice(&device));
  if (!allowed[device & 63].load(std::memory_order_acquire)) {
    FLCE_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostDynamicShared));
    allowed[device & 63].store(true, std::memory_order_release);
  }
  kKernel<<<grid, block, bytes, stream>>>(args...);
#else
  (void)bytes;
  FLCE_LAUNCH((kKernel), grid, block, stream, args...);
#endif
  return FLCE_OK;
}

}  // namespace flce
