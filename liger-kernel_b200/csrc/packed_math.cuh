// Arithmetic on pairs of floats in one 64-bit register (add / mul / fma .f32x2: one instruction for two elements on sm_100) and
// asynchronous 16-byte copies into shared memory, and four sums over a group of lanes at once, for kernels that are short of issue
// slots rather than of bandwidth.
//
// With FLCE_HOST_EMULATION the pairs are two floats and a copy is done when it is issued.
#pragma once

#include <cstdint>
#include <cstring>

#include "ce_kernels.cuh"
#include "simt_common.cuh"

namespace flce {

#ifdef FLCE_HOST_EMULATION
struct F2 {
  float lo, hi;
};
inline F2 f2(float lo, float hi) { return {lo, hi}; }
inline float f2_lo(F2 a) { return a.lo; }
inline float f2_hi(F2 a) { return a.hi; }
inline F2 add2(F2 a, F2 b) { return {a.lo + b.lo, a.hi + b.hi}; }
inline F2 mul2(F2 a, F2 b) { return {a.lo * b.lo, a.hi * b.hi}; }
inline F2 fma2(F2 a, F2 b, F2 c) { return {std::fma(a.lo, b.lo, c.lo), std::fma(a.hi, b.hi, c.hi)}; }
#else
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float f2_lo(F2 a) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a));
  return lo;
}
__device__ __forceinline__ float f2_hi(F2 a) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a));
  return hi;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
#endif
__device__ __forceinline__ F2 both(float v) { return f2(v, v); }

// Elements 2 i and 2 i + 1 of a run of elements held in 32-bit words (two 16-bit elements or one fp32 element per word).
template <typename T>
struct Pairs;
template <>
struct Pairs<float> {
  static constexpr int kWords = 2;             // words per pair
  __device__ static F2 get(const uint32_t* w) { return f2(__uint_as_float(w[0]), __uint_as_float(w[1])); }
  __device__ static void set(uint32_t* w, F2 v) {
    w[0] = __float_as_uint(f2_lo(v));
    w[1] = __float_as_uint(f2_hi(v));
  }
};
template <>
struct Pairs<__nv_bfloat16> {
  static constexpr int kWords = 1;
  __device__ static F2 get(const uint32_t* w) { return f2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u)); }
  __device__ static void set(uint32_t* w, F2 v) { w[0] = pack2(f2_lo(v), f2_hi(v), kOutBf16); }
};
template <>
struct Pairs<__half> {
  static constexpr int kWords = 1;
  __device__ static F2 get(const uint32_t* w) {
    __half h[2];
    memcpy(h, w, 4);
    return f2(__half2float(h[0]), __half2float(h[1]));
  }
  __device__ static void set(uint32_t* w, F2 v) { w[0] = pack2(f2_lo(v), f2_hi(v), kOutFp16); }
};

// the block's dynamic shared memory
#ifdef FLCE_HOST_EMULATION
#define FLCE_DYNAMIC_SHARED(type, name) type* name = static_cast<type*>(emu_dynamic_shared())
#else
#define FLCE_DYNAMIC_SHARED(type, name) extern __shared__ type name[]
#endif

// `bytes` (0..16) bytes from global to this CTA's shared memory (past L1), zeros up to 16; both addresses 16-byte aligned.  A
// thread sees its own copies after async_wait, its warp's after a warp_sync behind that; groups are waited for in the order
// they were committed.
__device__ __forceinline__ void async_copy16(void* dst, const void* src, int bytes) {
#ifdef FLCE_HOST_EMULATION
  std::memset(dst, 0, 16);
  if (bytes > 0) std::memcpy(dst, src, static_cast<size_t>(bytes));
#else
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src),
               "r"(bytes)
               : "memory");
#endif
}
__device__ __forceinline__ void async_commit() {
#ifndef FLCE_HOST_EMULATION
  asm volatile("cp.async.commit_group;" ::: "memory");
#endif
}
template <int kPending>
__device__ __forceinline__ void async_wait() {
#ifndef FLCE_HOST_EMULATION
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
#endif
}

// Programmatic dependent launch.  A kernel launched as a dependent may start before the kernel in front of it on the stream has
// ended (when all of that kernel's blocks have called allow_dependents or returned) and must wait before it touches anything
// that kernel, or one before it, reads or writes.
__device__ __forceinline__ void wait_for_previous_kernel() {
#ifndef FLCE_HOST_EMULATION
  asm volatile("griddepcontrol.wait;" ::: "memory");
#endif
}
__device__ __forceinline__ void allow_dependents() {
#ifndef FLCE_HOST_EMULATION
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#endif
}

__device__ __forceinline__ void warp_sync() {
#ifdef FLCE_HOST_EMULATION
  emu_warp_sync();
#else
  __syncwarp();
#endif
}

// Barrier of the `threads` threads (whole warps) that name it; ids 1..15, 0 is __syncthreads.
__device__ __forceinline__ void named_barrier(int id, int threads) {
#ifdef FLCE_HOST_EMULATION
  emu_named_barrier(id, threads);
#else
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
#endif
}

// ---- four sums at a time
//
// Lanes that differ in the group's highest bit trade two sums for the other two, those that differ in the next bit one for the
// other: 5 or 6 exchanges for four sums instead of 16 or 20.  The lane's two highest bits within its group (of its warp, if
// the group is wider) then name its sum.
__device__ __forceinline__ float low_lane_sum(float v, int lanes) {      // over `lanes` neighbouring lanes
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float lane_four_sums(const float (&v)[4], int lanes) {      // lanes: 4, 8, 16 or 32
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const int half = lanes >> 1, quarter = lanes >> 2;
  const bool up = (lane & half) != 0, right = (lane & quarter) != 0;
  const float a0 = __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], half) + (up ? v[2] : v[0]);
  const float a1 = __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], half) + (up ? v[3] : v[1]);
  return low_lane_sum(__shfl_xor_sync(0xffffffffu, right ? a0 : a1, quarter) + (right ? a1 : a0), quarter);
}

// sum number i of those of this lane's group of 1 << log2_group lanes, 32 at most
__device__ __forceinline__ float of_four(float sums, int i, int log2_group) {
  const int lanes = log2_group < 5 ? 1 << log2_group : 32;
  return __shfl_sync(0xffffffffu, sums, (static_cast<int>(threadIdx.x) & 31 & ~(lanes - 1)) | i * (lanes >> 2));
}

}  // namespace flce
