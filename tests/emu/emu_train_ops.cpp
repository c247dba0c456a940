// The C entry points of the norms and of the router's balance loss, their host side and their kernels, compiled for the host and run on the host
// through simt_emulation.hpp: the library's own launch shapes, index arithmetic and argument checks, with fibers in
// the place of CUDA threads.  The "device" has three SMs, so that persistent grids walk over several rows.
//
// Test infrastructure only.
#define FLCE_HOST_EMULATION 1
#include <cuda_runtime.h>
#include "simt_emulation.hpp"

#include <cstdarg>
#include <cstdio>
#include <type_traits>

// warp votes, through the same slots as the shuffles
inline unsigned __ballot_sync(unsigned, bool v) {
  unsigned bits = 0;
  for (unsigned o = 0; o < 32; ++o) {
    const unsigned from = (emu::linear_tid() & 31u) ^ o;
    if (emu::shuffle_from(static_cast<unsigned>(v), from)) bits |= 1u << from;
  }
  return bits;
}
inline bool __any_sync(unsigned m, bool v) { return __ballot_sync(m, v) != 0; }
inline float rsqrtf(float v) { return 1.f / std::sqrt(v); }
inline int __popc(unsigned v) { return __builtin_popcount(v); }
inline int __clz(unsigned v) { return v ? __builtin_clz(v) : 32; }

template <typename T>
T __shfl_sync(unsigned, T v, int src_lane) {
  return emu::shuffle_from(v, static_cast<unsigned>(src_lane));
}
// bar.sync id, n: its own barrier per id; every id is left empty by the kernels that use it
inline void emu_named_barrier(int id, int threads) {
  static emu::Barrier named[16];
  named[id].expected = static_cast<unsigned>(threads);
  emu::barrier_wait(named[id]);
}
inline void emu_warp_sync() { emu::barrier_wait(emu::t_ctx->warp_bar[emu::linear_tid() >> 5]); }
inline void* emu_dynamic_shared() {
  alignas(128) static char bytes[227 * 1024];
  return bytes;
}

inline emu::Dim3 emu_dim3(dim3 d) { return emu::Dim3(d.x, d.y, d.z); }

#include "host_internal.hpp"

namespace flce {
static char g_message[512];
static int g_launches = 0;
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_message, sizeof(g_message), fmt, ap);
  va_end(ap);
  return code;
}
void count_launches(int n) { g_launches += n; }
int current_sm_count(int* sm_count) {
  *sm_count = 3;
  return FLCE_OK;
}
}  // namespace flce

// what the host sides call of the CUDA runtime (renamed: a process that holds the real one would get that)
static cudaError_t emu_cuda_last_error() { return cudaSuccess; }
static cudaError_t emu_cuda_memset_async(void* p, int v, size_t n, cudaStream_t) {
  std::memset(p, v, n);
  return cudaSuccess;
}
static const char* emu_cuda_error_string(cudaError_t) { return "emulated"; }
#define cudaGetLastError emu_cuda_last_error
#define cudaMemsetAsync emu_cuda_memset_async
#define cudaGetErrorString emu_cuda_error_string
extern "C" {
const char* flce_b200_last_error(void) { return flce::g_message; }
const char* flce_b200_status_string(int) { return "emulated"; }
int emu_launches(void) { return flce::g_launches; }
}

#include "norm_b200.cu"
#include "balance_b200.cu"
