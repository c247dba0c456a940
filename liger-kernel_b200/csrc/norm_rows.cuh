// Layer norm and RMSNorm over the rows of a matrix, forward and backward (src/liger_kernel/ops/layer_norm.py and
// src/liger_kernel/ops/rms_norm.py of the reference are the operators they stand in for).
//
//   layer norm   xhat = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),   y = xhat * (offset + w) + b
//   RMSNorm      xhat = x * rstd,           rstd = 1 / sqrt(mean(x^2) + eps),            y = xhat * (offset + w)
//   backward     m = dy * (offset + w);  dx = rstd * (m - mean(m) - xhat * mean(m * xhat))   (RMSNorm: without mean(m))
//                dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Both directions are bound by HBM: forward moves a row in and out, backward two rows in and one out.  A row is read once and
// stays on the SM, so the variance is taken around the mean that is already known (no sum of squares minus square of sum)
// at no further traffic.  A *group* of 4..512 threads shares a row; a block holds as many groups as fit, so narrow rows need no
// barrier.  Everything between load and store is fp32; the only roundings to fewer bits are those of the results, and of
// xhat in the "llama" casting mode, which asks for it.
//
// A thread keeps the same columns for all its rows.  In backward the weight's and the bias's gradient are therefore sums in its
// registers; blocks leave one partial sum per column, added up in block order by a second kernel: no atomics, the same
// bits in every run.
//
// Five forms: rows of aligned 16-byte vectors, streamed (wide) or in registers (narrow); rows without that alignment, through
// windows (wide) or element by element (tiny); and rows longer than a block's threads hold (long).
#pragma once

#include <type_traits>

#include "ce_kernels.cuh"
#include "packed_math.cuh"
#include "simt_common.cuh"

namespace flce {

constexpr int kNormMaxThreads = 512;     // largest group of threads that shares a row
constexpr int kNormMaxWarps = kNormMaxThreads / 32;
constexpr int kNormColumnThreads = 256;

struct NormForwardArgs {
  const void* x;
  long long ld_x;
  const void* w;       // nullptr: a gain of one (the offset then plays no part)
  const void* b;       // nullptr: none
  void* y;             // dense rows
  float* mean;         // nullptr: not kept (also for RMSNorm)
  float* rstd;         // nullptr: not kept
  long long n_rows;
  int hidden;
  float eps, offset;
  int round_xhat;      // xhat is rounded to the rows' type before it meets the weight ("llama" casting)
  int log2_group;      // threads that share a row
  int group_warps;     // the same in warps, where they need not be a power of two
};

struct NormBackwardArgs {
  const void* dy;
  long long ld_dy;
  const void* x;
  long long ld_x;
  const void* w;
  const float* mean;
  const float* rstd;
  void* dx;            // dense rows
  float* dw_partial;   // [blocks][hidden]
  float* db_partial;   // [blocks][hidden], nullptr: not wanted
  long long n_rows;
  int hidden;
  float offset;
  int round_xhat;
  int log2_group;
  int group_warps;
};

template <typename T>
__device__ __forceinline__ float norm_round(float v) {
  T r;
  CeElem<T>::store(&r, v);
  return CeElem<T>::load(&r);
}

// 1 / sqrt(v) to the last bit or two: the hardware's estimate and one Newton step (v > 0; NaN and infinity pass through)
__device__ __forceinline__ float norm_rsqrt(float v) {
  const float r = rsqrtf(v);
  return v < INFINITY ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

// Over the `warps` whole warps of group g.  Warps meet in one of two buffers taken in turn: a thread writes a buffer
// again only behind the barrier of the call in between, which the readers of the older sums reach after reading them, so
// one barrier per call is enough.
__device__ __forceinline__ float norm_warps_four_sums(const float (&v)[4], int warps, int g, float (*scratch)[kNormMaxWarps * 4], int& phase) {
  float sum = lane_four_sums(v, 32);
  if (warps == 1) return sum;
  const int lane = static_cast<int>(threadIdx.x) & 31;
  float* buf = scratch[phase];
  phase ^= 1;
  if ((lane & 7) == 0) buf[(threadIdx.x >> 5) * 4 + (lane >> 3)] = sum;
  named_barrier(1 + g, warps * 32);
  const float* of = buf + g * warps * 4 + (lane >> 3);
  sum = 0.f;
  for (int w = lane & 7; w < warps; w += 8) sum += of[w * 4];
  return low_lane_sum(sum, 8);
}
// Rows whose warps have centred their parts on the parts' own means meet: `sum` and `square` of this warp's part of row lane >> 3
// become the mean and the sum (x - mean)^2 of the whole row.  Warp w holds part_elements(w) of the row's elements.
struct NormPartScratch {
  float sums[kNormMaxWarps * 4], squares[kNormMaxWarps * 4];
};
template <bool kCentered, class PartElements>
__device__ __forceinline__ void norm_meet(float& sum, float& square, int warps, int g, NormPartScratch (&scratch)[2], int& phase,
                                          float inv_hidden, float part_inv, PartElements part_elements) {
  if (warps == 1) {
    sum *= part_inv;
    return;
  }
  const int lane = static_cast<int>(threadIdx.x) & 31;
  NormPartScratch& buf = scratch[phase];
  phase ^= 1;                               // taken in turn, as above
  if ((lane & 7) == 0) {
    buf.squares[(threadIdx.x >> 5) * 4 + (lane >> 3)] = square;
    if (kCentered) buf.sums[(threadIdx.x >> 5) * 4 + (lane >> 3)] = sum;
  }
  named_barrier(1 + g, warps * 32);
  // eight lanes add up a row's parts
  const int of = g * warps * 4 + (lane >> 3);
  square = 0.f;
  if constexpr (kCentered) {
    sum = 0.f;
    for (int w = lane & 7; w < warps; w += 8) sum += buf.sums[of + w * 4];
    sum = low_lane_sum(sum, 8) * inv_hidden;
    for (int w = lane & 7; w < warps; w += 8) {
      const float n = part_elements(w);
      const float off = n > 0.f ? buf.sums[of + w * 4] / n - sum : 0.f;
      square += fmaf(n * off, off, buf.squares[of + w * 4]);
    }
  } else {
    for (int w = lane & 7; w < warps; w += 8) square += buf.squares[of + w * 4];
  }
  square = low_lane_sum(square, 8);
}

// sum number i of those, from a lane of the warp that holds it
__device__ __forceinline__ float norm_warp_of_four(float sums, int i) { return __shfl_sync(0xffffffffu, sums, i * 8); }

// ---- rows of whole, aligned 16-byte vectors, more than a warp's worth: streamed through shared memory
//
// One row at a time per block, in registers, loses not bandwidth but issue slots and waiting: at 32768 x 4096 bf16 such kernels
// ran at 46 % (forward) and 41 % (backward) of the copy rate, with fp32 rows, half the elements per byte, forward at 87 %.
// Here the arithmetic goes two elements to an instruction, several rows share a barrier, and the next rows are always on
// their way: every thread copies the vectors that it will read itself, with cp.async, so the ring needs no barrier and no
// wait on another thread.

constexpr int kStreamThreads = 512;

// kUnits vectors of a parameter, zeros where there is none
template <typename W, int kUnits, int kWVecs>
__device__ __forceinline__ void stream_load_parameter(const void* src, int first, int vectors, uint4 (&raw)[kUnits * kWVecs]) {
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
#pragma unroll
    for (int i = 0; i < kWVecs; ++i) {
      raw[u * kWVecs + i] = make_uint4(0u, 0u, 0u, 0u);
      if (src != nullptr && first + u * 32 < vectors)
        raw[u * kWVecs + i] = __ldg(reinterpret_cast<const uint4*>(src) + (first + u * 32) * kWVecs + i);
    }
  }
}

// Shape of the streaming kernels by the vectors per thread, 2 or 4: rows that a group takes per round (two rows of backward are
// four sums, as four rows of forward are), rounds in the ring, which takes 128 or 192 KB: one block per SM.
// With one vector per thread the groups are twice as wide and wait longer for each other: 32768 x 4096 bf16 backward 158 us
// against 127, forward 124 against 88; with four in rows that two would hold, registers run out (138 and 138 us).
// Forward with fewer rows than the device takes in one round of four goes row by row, over as many blocks as there are
// (kFew): 64 x 1024 fp32 6.9 -> 4.5 us, 1 x 8192 bf16 5.9 -> 3.9 us (kernel alone, cold caches).
template <int kUnits, bool kGrad, bool kFew = false>
struct Stream {
  static constexpr int kRows = kUnits == 4 || kFew ? 1 : (kGrad ? 2 : 4);
  static constexpr int kSlots = kFew ? 1 : (kUnits == 2 && !kGrad ? 2 : 3);
  static constexpr int kRingBytes = kSlots * kRows * (kGrad ? 2 : 1) * kUnits * kStreamThreads * 16;
};

// y and the row statistics.  Each thread of a group owns kUnits vectors of columns, their gain and bias in registers; a group takes
// kRows rows per round.  Each warp centres its part of a row on that part's own mean; across warps the parts' sums and squares
// meet behind one barrier, sum (x - mean)^2 = sum over parts of (squares + elements * (part's mean - mean)^2): nothing is
// subtracted that has to cancel.  A fixed grid walks over the rows.
template <typename T, typename W, bool kCentered, int kUnits, bool kFew>
__global__ void __launch_bounds__(kStreamThreads, 1)
norm_forward_stream_kernel(NormForwardArgs a) {
  constexpr int kRows = Stream<kUnits, false, kFew>::kRows, kSlots = Stream<kUnits, false, kFew>::kSlots;
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                    // [slot][row][unit][thread]
  __shared__ NormPartScratch scratch[2];
  const int group = 1 << a.log2_group;
  const int warps = group >> 5;
  const int groups = kStreamThreads >> a.log2_group;
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const int first = (t >> 5) * 32 * kUnits + (t & 31);        // this lane's first vector; the others follow in strides of 32
  const int vectors = a.hidden / kVec;
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  const bool rounded = !kCentered && a.round_xhat != 0;

  uint4 raw_w[kUnits * kWVecs], raw_b[kCentered ? kUnits * kWVecs : 1];
  stream_load_parameter<W, kUnits, kWVecs>(a.w, first, vectors, raw_w);
  if constexpr (kCentered) stream_load_parameter<W, kUnits, kWVecs>(a.b, first, vectors, raw_b);
  const F2 offset = both(a.w != nullptr ? a.offset : 1.f);     // without a weight the gain is one

  auto cell = [&](int slot, int r, int u) -> uint4& { return stream_ring[((slot * kRows + r) * kUnits + u) * kStreamThreads + threadIdx.x]; };
  // rows behind the last one come in as zeros and are not stored
  auto fetch = [&](long long base, int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = base + r < a.n_rows;
      const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (live ? base + r : 0) * a.ld_x) + first;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) async_copy16(&cell(slot, r, u), x + u * 32, live && first + u * 32 < vectors ? 16 : 0);
    }
    async_commit();
  };
  long long row = (static_cast<long long>(blockIdx.x) * groups + g) * kRows;
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s) fetch(row + s * step, s);
  int slot = 0, phase = 0;
  const float inv = 1.f / static_cast<float>(a.hidden);
  // elements of the row that warp w of a group holds
  auto part_elements = [&](int w) {
    const int left = vectors - w * 32 * kUnits;
    return static_cast<float>((left < 0 ? 0 : (left < 32 * kUnits ? left : 32 * kUnits)) * kVec);
  };
  const float part_inv = part_elements(t >> 5) > 0.f ? 1.f / part_elements(t >> 5) : 0.f;
  for (; row < a.n_rows; row += step) {
    // into the slot of the round before this one, which this thread, its only reader, has read for the last time
    fetch(row + (kSlots - 1) * step, slot == 0 ? kSlots - 1 : slot - 1);
    async_wait<kSlots - 1>();
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    F2 minus_mean[kRows];
    float part_sum = 0.f;                   // this warp's, of row lane >> 3
    if constexpr (kCentered) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        F2 acc = both(0.f);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const uint4 raw = cell(slot, r, u);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) acc = add2(acc, Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw) + i * Pairs<T>::kWords));
        }
        v[r] = f2_lo(acc) + f2_hi(acc);
      }
      part_sum = lane_four_sums(v, 32);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const F2 centre = both(kCentered ? -__shfl_sync(0xffffffffu, part_sum, r * 8) * part_inv : 0.f);
      F2 acc = both(0.f);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint4 raw = cell(slot, r, u);
        if (!kCentered || first + u * 32 < vectors) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            F2 e = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw) + i * Pairs<T>::kWords);
            if (kCentered) e = add2(e, centre);
            acc = fma2(e, e, acc);
          }
        }
      }
      v[r] = f2_lo(acc) + f2_hi(acc);
    }
    float square = lane_four_sums(v, 32);
    norm_meet<kCentered>(part_sum, square, warps, g, scratch, phase, inv, part_inv, part_elements);
    const float mean = part_sum;            // of row lane >> 3
    const float rstd = norm_rsqrt(fmaf(square, inv, a.eps));
#pragma unroll
    for (int r = 0; r < kRows; ++r) minus_mean[r] = both(kCentered ? -__shfl_sync(0xffffffffu, mean, r * 8) : 0.f);
    {
      const int r = lane >> 3;
      if ((t & ~24) == 0 && r < kRows && row + r < a.n_rows) {      // lanes 0, 8, 16, 24 of the group's first warp
        if (kCentered && a.mean != nullptr) a.mean[row + r] = mean;
        if (a.rstd != nullptr) a.rstd[row + r] = rstd;
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const F2 scale = both(__shfl_sync(0xffffffffu, rstd, r * 8));
      if (row + r >= a.n_rows) continue;
      uint4* y = reinterpret_cast<uint4*>(static_cast<T*>(a.y) + (row + r) * a.hidden) + first;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (first + u * 32 >= vectors) continue;
        const uint4 raw = cell(slot, r, u);
        uint4 out;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          F2 e = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw) + i * Pairs<T>::kWords);
          if (kCentered) e = add2(e, minus_mean[r]);
          e = mul2(e, scale);
          if (rounded) e = f2(norm_round<T>(f2_lo(e)), norm_round<T>(f2_hi(e)));
          const F2 gain = add2(offset, Pairs<W>::get(reinterpret_cast<const uint32_t*>(&raw_w[u * kWVecs]) + i * Pairs<W>::kWords));
          if constexpr (kCentered)
            e = fma2(e, gain, Pairs<W>::get(reinterpret_cast<const uint32_t*>(&raw_b[u * kWVecs]) + i * Pairs<W>::kWords));
          else
            e = mul2(e, gain);
          Pairs<T>::set(reinterpret_cast<uint32_t*>(&out) + i * Pairs<T>::kWords, e);
        }
        y[u * 32] = out;
      }
    }
    slot = slot + 1 == kSlots ? 0 : slot + 1;
  }
  async_wait<0>();
}

// dx, and this block's share of the parameters' gradients.  Each thread of a group owns kUnits vectors of columns; a round
// takes kRows rows per group, their sums meet in one reduction (and one barrier, if the group is wider than a warp).
template <typename T, typename W, bool kCentered, int kUnits>
__global__ void __launch_bounds__(kStreamThreads, 1)
norm_backward_stream_kernel(NormBackwardArgs a) {
  allow_dependents();      // the small kernel that adds up the partial sums
  constexpr int kRows = Stream<kUnits, true>::kRows, kSlots = Stream<kUnits, true>::kSlots;
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                // [slot][row][x, dy][unit][thread]; at the end: the blocks' folds
  __shared__ float scratch[2][kNormMaxWarps * 4];
  const int group = 1 << a.log2_group;
  const int warps = group >> 5;
  const int groups = kStreamThreads >> a.log2_group;
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int first = (t >> 5) * 32 * kUnits + (t & 31);
  const int vectors = a.hidden / kVec;
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  const bool rounded = !kCentered && a.round_xhat != 0;
  // rows are counted from the last one: what forward, or the kernel that made dy, touched last is what L2 still holds
  const long long last = a.n_rows - 1;

  uint4 raw_w[kUnits * kWVecs];
  stream_load_parameter<W, kUnits, kWVecs>(a.w, first, vectors, raw_w);
  // without a weight the gain is one: zeros plus an offset of one
  const F2 offset = both(a.w != nullptr ? a.offset : 1.f);
  auto gain = [&](int u, int i) {
    return add2(offset, Pairs<W>::get(reinterpret_cast<const uint32_t*>(&raw_w[u * kWVecs]) + i * Pairs<W>::kWords));
  };

  F2 dw[kUnits * kPairs], db[kCentered ? kUnits * kPairs : 1];
#pragma unroll
  for (int i = 0; i < kUnits * kPairs; ++i) {
    dw[i] = both(0.f);
    if (kCentered) db[i] = both(0.f);
  }

  // rows of this group in a round: consecutive ones.  A row behind the last one comes in as zeros and is not stored.
  auto cell = [&](int slot, int r, int which, int u) -> uint4& {
    return stream_ring[(((slot * kRows + r) * 2 + which) * kUnits + u) * kStreamThreads + threadIdx.x];
  };
  auto fetch = [&](long long base, int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + r;
      const bool live = row < a.n_rows;
      const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (live ? last - row : 0) * a.ld_x) + first;
      const uint4* dy = reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + (live ? last - row : 0) * a.ld_dy) + first;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        async_copy16(&cell(slot, r, 0, u), x + u * 32, live && first + u * 32 < vectors ? 16 : 0);
        async_copy16(&cell(slot, r, 1, u), dy + u * 32, live && first + u * 32 < vectors ? 16 : 0);
      }
    }
    async_commit();
  };
  float next_mean[kRows], next_rstd[kRows];
  auto fetch_statistics = [&](long long base) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = base + r < a.n_rows;
      next_mean[r] = kCentered && live ? __ldg(a.mean + last - base - r) : 0.f;
      next_rstd[r] = live ? __ldg(a.rstd + last - base - r) : 0.f;
    }
  };

  long long round = static_cast<long long>(blockIdx.x) * groups * kRows;     // the block's first row: the same in every thread
  const int mine = g * kRows;
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s) fetch(round + s * step + mine, s);
  fetch_statistics(round + mine);
  int slot = 0, phase = 0;
  for (; round < a.n_rows; round += step) {
    // the slot of the round before this one: its second reading is done, in this thread, which is the only one to read it
    fetch(round + (kSlots - 1) * step + mine, slot == 0 ? kSlots - 1 : slot - 1);
    async_wait<kSlots - 1>();
    float rstd[kRows];
    F2 minus_mean[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      minus_mean[r] = both(-next_mean[r]);
      rstd[r] = next_rstd[r];
    }
    fetch_statistics(round + step + mine);
    float v[4] = {0.f, 0.f, 0.f, 0.f};        // (sum m xhat, sum m) of each row
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      F2 s_mx = both(0.f), s_m = both(0.f);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint4 raw_x = cell(slot, r, 0, u), raw_dy = cell(slot, r, 1, u);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          // behind the row's end dy is zero, which keeps xhat out of every sum
          F2 xhat = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw_x) + i * Pairs<T>::kWords);
          if (kCentered) xhat = add2(xhat, minus_mean[r]);
          xhat = mul2(xhat, both(rstd[r]));
          const F2 d = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw_dy) + i * Pairs<T>::kWords);
          F2 xw = xhat;
          if (rounded) xw = f2(norm_round<T>(f2_lo(xhat)), norm_round<T>(f2_hi(xhat)));
          dw[u * kPairs + i] = fma2(d, xw, dw[u * kPairs + i]);
          if (kCentered) db[u * kPairs + i] = add2(db[u * kPairs + i], d);
          const F2 m = mul2(d, gain(u, i));
          s_mx = fma2(m, xhat, s_mx);
          if (kCentered) s_m = add2(s_m, m);
        }
      }
      v[2 * r] = f2_lo(s_mx) + f2_hi(s_mx);
      if (kCentered) v[2 * r + 1] = f2_lo(s_m) + f2_hi(s_m);
    }
    const float sum = norm_warps_four_sums(v, warps, g, scratch, phase);
    const float inv = 1.f / static_cast<float>(a.hidden);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float c = __shfl_sync(0xffffffffu, sum, r * 16) * inv;
      const float m_mean = kCentered ? __shfl_sync(0xffffffffu, sum, r * 16 + 8) * inv : 0.f;
      const long long row = round + mine + r;
      if (row >= a.n_rows) continue;
      uint4* dx = reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + (last - row) * a.hidden) + first;
      // rstd (m - mean(m) - xhat c), xhat = (x - mean) rstd
      const F2 minus_c = both(-c), minus_m = both(-m_mean);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (first + u * 32 >= vectors) continue;
        const uint4 raw_x = cell(slot, r, 0, u), raw_dy = cell(slot, r, 1, u);
        uint4 out;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          F2 xhat = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw_x) + i * Pairs<T>::kWords);
          if (kCentered) xhat = add2(xhat, minus_mean[r]);
          xhat = mul2(xhat, both(rstd[r]));
          F2 m = mul2(Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw_dy) + i * Pairs<T>::kWords), gain(u, i));
          if (kCentered) m = add2(m, minus_m);
          Pairs<T>::set(reinterpret_cast<uint32_t*>(&out) + i * Pairs<T>::kWords, mul2(fma2(xhat, minus_c, m), both(rstd[r])));
        }
        dx[u * 32] = out;
      }
    }
    slot = slot + 1 == kSlots ? 0 : slot + 1;
  }
  // the groups of the block, folded in halves in a fixed order; the ring is free once all copies (of zeros, behind the last
  // row) have landed
  async_wait<0>();
  float* fold = reinterpret_cast<float*>(stream_ring);
  auto leave = [&](F2* acc, float* partial) {
    for (int half = groups >> 1; half > 0; half >>= 1) {
      __syncthreads();
      if (g >= half && g < 2 * half) {
#pragma unroll
        for (int i = 0; i < kUnits * kPairs; ++i) {
          fold[((g - half) * 2 * kUnits * kPairs + 2 * i) * group + t] = f2_lo(acc[i]);
          fold[((g - half) * 2 * kUnits * kPairs + 2 * i + 1) * group + t] = f2_hi(acc[i]);
        }
      }
      __syncthreads();
      if (g < half) {
#pragma unroll
        for (int i = 0; i < kUnits * kPairs; ++i)
          acc[i] = add2(acc[i], f2(fold[(g * 2 * kUnits * kPairs + 2 * i) * group + t], fold[(g * 2 * kUnits * kPairs + 2 * i + 1) * group + t]));
      }
    }
    if (g == 0) {
      float* out = partial + static_cast<size_t>(blockIdx.x) * a.hidden;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (first + u * 32 >= vectors) continue;
        float e[kVec];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          e[2 * i] = f2_lo(acc[u * kPairs + i]);
          e[2 * i + 1] = f2_hi(acc[u * kPairs + i]);
        }
#pragma unroll
        for (int i = 0; i < kVec; i += 4) *reinterpret_cast<float4*>(out + (first + u * 32) * kVec + i) = make_float4(e[i], e[i + 1], e[i + 2], e[i + 3]);
      }
    }
  };
  if (a.dw_partial != nullptr) leave(dw, a.dw_partial);
  if constexpr (kCentered) {
    if (a.db_partial != nullptr) leave(db, a.db_partial);
  }
}

// ---- rows of at most 32 aligned 16-byte vectors: one vector per lane, several rows to a warp, kRows of them per thread in a round,
// no barrier at all.  Groups of 4 to 32 lanes.  The rounds ahead are in a ring as above: with the rows of the round loaded into
// registers, 262144 x 128 bf16 took 29 us forward and 56 us backward; now 25 and 41 us with three blocks per SM, 27 and 49 us with
// four, whose registers do not hold it all.

constexpr int kNarrowThreads = 256;
constexpr int kNarrowForwardRows = 4, kNarrowBackwardRows = 2;      // four sums either way
constexpr int kNarrowSlots = 3;
constexpr int kNarrowRingBytes = kNarrowSlots * 4 * kNarrowThreads * 16;      // 48 KB
constexpr int kNarrowBlocksPerSm = 3;

template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNarrowThreads, kNarrowBlocksPerSm)
norm_forward_narrow_kernel(NormForwardArgs a) {
  constexpr int kRows = kNarrowForwardRows;
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  const int group = 1 << a.log2_group;
  const int groups = kNarrowThreads >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const bool column = t * kVec < a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                    // [slot][row][thread]
  auto cell = [&](int slot, int r) -> uint4& { return stream_ring[(slot * kRows + r) * kNarrowThreads + threadIdx.x]; };
  // rows of a round lie `groups` apart; those behind the last one come in as zeros
  auto fetch = [&](long long base, int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + r * groups;
      const bool live = row < a.n_rows;
      async_copy16(&cell(slot, r), reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (live ? row : 0) * a.ld_x) + t, live && column ? 16 : 0);
    }
    async_commit();
  };
  F2 gain[kPairs], bias[kPairs];
  {
    uint4 w[kWVecs], b[kWVecs];
#pragma unroll
    for (int i = 0; i < kWVecs; ++i) {
      w[i] = b[i] = make_uint4(0u, 0u, 0u, 0u);
      if (column && a.w != nullptr) w[i] = __ldg(reinterpret_cast<const uint4*>(a.w) + t * kWVecs + i);
      if (column && a.b != nullptr) b[i] = __ldg(reinterpret_cast<const uint4*>(a.b) + t * kWVecs + i);
    }
    const F2 offset = both(a.w != nullptr ? a.offset : 1.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      gain[i] = add2(offset, Pairs<W>::get(reinterpret_cast<const uint32_t*>(w) + i * Pairs<W>::kWords));
      bias[i] = Pairs<W>::get(reinterpret_cast<const uint32_t*>(b) + i * Pairs<W>::kWords);
    }
  }
  const float inv = 1.f / static_cast<float>(a.hidden);
  // the same number of rounds in every thread of the block: the lanes of a warp share its shuffles
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  long long round = static_cast<long long>(blockIdx.x) * groups * kRows;
#pragma unroll
  for (int s = 0; s < kNarrowSlots - 1; ++s) fetch(round + s * step + g, s);
  int slot = 0;
  for (; round < a.n_rows; round += step) {
    const long long base = round + g;
    fetch(base + (kNarrowSlots - 1) * step, slot == 0 ? kNarrowSlots - 1 : slot - 1);
    async_wait<kNarrowSlots - 1>();
    uint4 raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) raw[r] = cell(slot, r);
    slot = slot + 1 == kNarrowSlots ? 0 : slot + 1;
    float v[4];
    float mean = 0.f;                         // of the row that this lane's sum belongs to
    if constexpr (kCentered) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        F2 acc = both(0.f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) acc = add2(acc, Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw[r]) + i * Pairs<T>::kWords));
        v[r] = f2_lo(acc) + f2_hi(acc);
      }
      mean = lane_four_sums(v, group) * inv;
    }
    F2 minus_mean[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      minus_mean[r] = both(kCentered ? -of_four(mean, r, a.log2_group) : 0.f);
      F2 acc = both(0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        F2 e = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw[r]) + i * Pairs<T>::kWords);
        if (kCentered) e = add2(e, minus_mean[r]);
        acc = fma2(e, e, acc);
      }
      v[r] = column ? f2_lo(acc) + f2_hi(acc) : 0.f;
    }
    const float rstd = norm_rsqrt(fmaf(lane_four_sums(v, group), inv, a.eps));
    {
      const int r = t / (group >> 2);
      const long long row = base + r * groups;
      if (t % (group >> 2) == 0 && row < a.n_rows) {
        if (kCentered && a.mean != nullptr) a.mean[row] = mean;
        if (a.rstd != nullptr) a.rstd[row] = rstd;
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + r * groups;
      const F2 scale = both(of_four(rstd, r, a.log2_group));
      uint4 out;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        F2 e = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw[r]) + i * Pairs<T>::kWords);
        if (kCentered) e = add2(e, minus_mean[r]);
        e = mul2(e, scale);
        if (rounded) e = f2(norm_round<T>(f2_lo(e)), norm_round<T>(f2_hi(e)));
        Pairs<T>::set(reinterpret_cast<uint32_t*>(&out) + i * Pairs<T>::kWords, kCentered ? fma2(e, gain[i], bias[i]) : mul2(e, gain[i]));
      }
      if (column && row < a.n_rows) reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.hidden)[t] = out;
    }
  }
  async_wait<0>();
}

template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNarrowThreads, kNarrowBlocksPerSm)
norm_backward_narrow_kernel(NormBackwardArgs a) {
  allow_dependents();      // the small kernel that adds up the partial sums
  constexpr int kRows = kNarrowBackwardRows;
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                    // [slot][row][x, dy][thread]; at the end: the groups' folds
  const int group = 1 << a.log2_group;
  const int groups = kNarrowThreads >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const bool column = t * kVec < a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const long long last = a.n_rows - 1;      // rows are counted from the last one, as above
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  F2 gain[kPairs], dw[kPairs], db[kPairs];
  {
    uint4 w[kWVecs];
#pragma unroll
    for (int i = 0; i < kWVecs; ++i) {
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (column && a.w != nullptr) w[i] = __ldg(reinterpret_cast<const uint4*>(a.w) + t * kWVecs + i);
    }
    const F2 offset = both(a.w != nullptr ? a.offset : 1.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      gain[i] = add2(offset, Pairs<W>::get(reinterpret_cast<const uint32_t*>(w) + i * Pairs<W>::kWords));
      dw[i] = db[i] = both(0.f);
    }
  }
  const float inv = 1.f / static_cast<float>(a.hidden);
  auto cell = [&](int slot, int r, int which) -> uint4& {
    return stream_ring[((slot * kRows + r) * 2 + which) * kNarrowThreads + threadIdx.x];
  };
  // rows of a round lie `groups` apart; those behind the last one come in as zeros
  auto fetch = [&](long long base, int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + r * groups;
      const bool live = row < a.n_rows;
      const long long from = live ? last - row : 0;
      async_copy16(&cell(slot, r, 0), reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + from * a.ld_x) + t, live && column ? 16 : 0);
      async_copy16(&cell(slot, r, 1), reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + from * a.ld_dy) + t, live && column ? 16 : 0);
    }
    async_commit();
  };
  float next_mean[kRows], next_rstd[kRows];
  auto fetch_statistics = [&](long long base) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + r * groups;
      next_mean[r] = kCentered && row < a.n_rows ? __ldg(a.mean + last - row) : 0.f;
      next_rstd[r] = row < a.n_rows ? __ldg(a.rstd + last - row) : 0.f;
    }
  };
  long long round = static_cast<long long>(blockIdx.x) * groups * kRows;
#pragma unroll
  for (int s = 0; s < kNarrowSlots - 1; ++s) fetch(round + s * step + g, s);
  fetch_statistics(round + g);
  int slot = 0;
  for (; round < a.n_rows; round += step) {
    const long long base = round + g;
    fetch(base + (kNarrowSlots - 1) * step, slot == 0 ? kNarrowSlots - 1 : slot - 1);
    async_wait<kNarrowSlots - 1>();
    uint4 raw_x[kRows], raw_dy[kRows];
    float mean[kRows], rstd[kRows], v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      raw_x[r] = cell(slot, r, 0);
      raw_dy[r] = cell(slot, r, 1);
      mean[r] = next_mean[r];
      rstd[r] = next_rstd[r];
    }
    slot = slot + 1 == kNarrowSlots ? 0 : slot + 1;
    fetch_statistics(base + step);
    auto xhat_of = [&](int r, int i) {
      F2 v = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw_x[r]) + i * Pairs<T>::kWords);
      if (kCentered) v = add2(v, both(-mean[r]));
      return mul2(v, both(rstd[r]));
    };
    auto dy_of = [&](int r, int i) { return Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw_dy[r]) + i * Pairs<T>::kWords); };
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      F2 mx = both(0.f), m = both(0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const F2 xhat = xhat_of(r, i), d = dy_of(r, i), md = mul2(d, gain[i]);
        dw[i] = fma2(d, rounded ? f2(norm_round<T>(f2_lo(xhat)), norm_round<T>(f2_hi(xhat))) : xhat, dw[i]);
        if (kCentered) db[i] = add2(db[i], d);
        mx = fma2(md, xhat, mx);
        if (kCentered) m = add2(m, md);
      }
      v[2 * r] = f2_lo(mx) + f2_hi(mx);
      v[2 * r + 1] = f2_lo(m) + f2_hi(m);
    }
    const float sums = lane_four_sums(v, group) * -inv;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + r * groups;
      const F2 minus_c = both(of_four(sums, 2 * r, a.log2_group));
      const F2 minus_m = both(kCentered ? of_four(sums, 2 * r + 1, a.log2_group) : 0.f);
      uint4 out;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        F2 m = mul2(dy_of(r, i), gain[i]);
        if (kCentered) m = add2(m, minus_m);
        Pairs<T>::set(reinterpret_cast<uint32_t*>(&out) + i * Pairs<T>::kWords, mul2(fma2(xhat_of(r, i), minus_c, m), both(rstd[r])));
      }
      if (column && row < a.n_rows) reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + (last - row) * a.hidden)[t] = out;
    }
  }
  // the groups of the block, folded in halves in a fixed order
  async_wait<0>();
  float* fold = reinterpret_cast<float*>(stream_ring);
  auto leave = [&](F2 (&acc)[kPairs], float* partial) {
    for (int half = groups >> 1; half > 0; half >>= 1) {
      __syncthreads();
      if (g >= half && g < 2 * half) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          fold[((g - half) * kVec + 2 * i) * group + t] = f2_lo(acc[i]);
          fold[((g - half) * kVec + 2 * i + 1) * group + t] = f2_hi(acc[i]);
        }
      }
      __syncthreads();
      if (g < half) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) acc[i] = add2(acc[i], f2(fold[(g * kVec + 2 * i) * group + t], fold[(g * kVec + 2 * i + 1) * group + t]));
      }
    }
    if (g == 0 && column) {
      float* out = partial + static_cast<size_t>(blockIdx.x) * a.hidden + t * kVec;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        out[2 * i] = f2_lo(acc[i]);
        out[2 * i + 1] = f2_hi(acc[i]);
      }
    }
  };
  if (a.dw_partial != nullptr) leave(dw, a.dw_partial);
  if constexpr (kCentered) {
    if (a.db_partial != nullptr) leave(db, a.db_partial);
  }
}

// ---- rows that do not start on 16-byte boundaries or do not hold whole vectors
//
// A warp fetches its part of a row as the aligned 16-byte pieces that hold it, with cp.async, into a window of its own in shared
// memory, rounds ahead like the streaming kernels, and reads its elements from there at whatever shift the row has: lane by
// lane neighbouring elements, which is free of bank conflicts.  (The first piece may begin up to 14 bytes before the row: in the
// same 16-byte granule, which belongs to the same allocation.)  Results leave as neighbouring elements, whole sectors at a
// time.  Direct element loads into registers, a round ahead, left too little under way: 10007 x 1537 fp16 35 us forward, 77 us
// backward.  A part is 32 * kEpt columns, a row `warps` parts, as many rows side by side as the block's 16 warps hold.
constexpr int kWindowThreads = 512;
constexpr int kWindowWarps = kWindowThreads / 32;
// What a round costs beside its elements (asking for the pieces, sums, barrier) is most of it, so it takes as many rows as registers
// and shared memory hold; the parameters are read from shared memory, once per round, for that.
template <typename T, int kEpt, bool kGrad>
struct Window {
  static constexpr int kPieces = 32 * kEpt * static_cast<int>(sizeof(T)) / 16 + 1;     // of one window
  static constexpr int kRows = (kEpt == 16 && sizeof(T) == 4 ? 2 : 4) / (kGrad ? 2 : 1);
  static constexpr int kRoundBytes = kRows * (kGrad ? 2 : 1) * kWindowWarps * kPieces * 16;
  static constexpr int kParameterBytes = kWindowWarps * 32 * kEpt * (kGrad ? 4 : 8);
  static constexpr int kRoom = 216 * 1024 - kParameterBytes;
  static constexpr int kSlots = 6 * kRoundBytes <= kRoom ? 6 : (4 * kRoundBytes <= kRoom ? 4 : (3 * kRoundBytes <= kRoom ? 3 : 2));
  static constexpr int kRingBytes = kSlots * kRoundBytes;          // at the end also: the groups' sums, a float per lane and element
  static constexpr int kBytes = kRingBytes + kParameterBytes;
  static_assert(kBytes <= 220 * 1024 && kRingBytes >= kWindowWarps * 32 * kEpt * 4, "shared memory");
};

// the pieces of `count` elements from `src`, asked for by the lanes of a warp; zeros in the rest of the window
template <typename T, int kPieces>
__device__ __forceinline__ void window_fetch(uint4* window, const T* src, int count, int lane) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(src);
  const int end = count > 0 ? static_cast<int>(at & 15) + count * static_cast<int>(sizeof(T)) : 0;
  const char* base = reinterpret_cast<const char*>(at & ~static_cast<uintptr_t>(15));
#pragma unroll
  for (int i = 0; i < kPieces; i += 32) {
    const int left = end - (i + lane) * 16;
    if (i + 32 <= kPieces || i + lane < kPieces)
      async_copy16(window + i + lane, left > 0 ? base + (i + lane) * 16 : base, left < 0 ? 0 : (left < 16 ? left : 16));
  }
}
// kEpt elements of this lane, in pairs, zeros behind the end
template <typename T, int kEpt>
__device__ __forceinline__ void window_read(const uint4* window, const T* src, int lane, F2 (&v)[kEpt / 2]) {
  const T* e = reinterpret_cast<const T*>(reinterpret_cast<const char*>(window) + (reinterpret_cast<uintptr_t>(src) & 15)) + lane;
#pragma unroll
  for (int i = 0; i < kEpt / 2; ++i) v[i] = f2(CeElem<T>::load(e + 64 * i), CeElem<T>::load(e + 64 * i + 32));
}
// and back; a part that is full, as all but a row's last are, needs no look at the end
template <typename T, int kEpt>
__device__ __forceinline__ void window_store(T* dst, int count, int lane, const F2 (&v)[kEpt / 2]) {
  dst += lane;
  if (count == 32 * kEpt) {
#pragma unroll
    for (int i = 0; i < kEpt / 2; ++i) {
      CeElem<T>::store(dst + 64 * i, f2_lo(v[i]));
      CeElem<T>::store(dst + 64 * i + 32, f2_hi(v[i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < kEpt / 2; ++i) {
      if (lane + 64 * i < count) CeElem<T>::store(dst + 64 * i, f2_lo(v[i]));
      if (lane + 64 * i + 32 < count) CeElem<T>::store(dst + 64 * i + 32, f2_hi(v[i]));
    }
  }
}

template <typename T, typename W, bool kCentered, int kEpt>
__global__ void __launch_bounds__(kWindowThreads, 1)
norm_forward_window_kernel(NormForwardArgs a) {
  typedef Window<T, kEpt, false> Shape;
  constexpr int kRows = Shape::kRows, kSlots = Shape::kSlots, kPairs = kEpt / 2;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                    // [slot][row][warp][piece], then (gain, bias) of every column
  __shared__ float scratch[2][kNormMaxWarps * 4];
  const int warps = a.group_warps;
  const int groups = kWindowWarps / warps;
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int g = warp / warps;
  const int column = (warp - g * warps) * 32 * kEpt;
  const int count = a.hidden - column < 32 * kEpt ? a.hidden - column : 32 * kEpt;      // of this warp's part
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const float inv = 1.f / static_cast<float>(a.hidden);
  float2* parameters = reinterpret_cast<float2*>(stream_ring + Shape::kRingBytes / 16);
  for (int c = static_cast<int>(threadIdx.x); c < warps * 32 * kEpt; c += kWindowThreads) {
    const bool in = c < a.hidden;
    parameters[c] = make_float2(in && a.w != nullptr ? a.offset + CeElem<W>::load(static_cast<const W*>(a.w) + c) : 1.f,
                                in && a.b != nullptr ? CeElem<W>::load(static_cast<const W*>(a.b) + c) : 0.f);
  }
  __syncthreads();
  if (g >= groups) return;                                    // warps that make no whole group: no block-wide barrier follows
  parameters += column + lane;
  auto window = [&](int slot, int r) { return stream_ring + ((slot * kRows + r) * kWindowWarps + warp) * Shape::kPieces; };
  auto source = [&](long long row) { return static_cast<const T*>(a.x) + row * a.ld_x + column; };
  auto fetch = [&](long long base, int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = base + r < a.n_rows;
      window_fetch<T, Shape::kPieces>(window(slot, r), source(live ? base + r : 0), live ? count : 0, lane);
    }
    async_commit();
  };
  long long row = (static_cast<long long>(blockIdx.x) * groups + g) * kRows;
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s) fetch(row + s * step, s);
  int slot = 0, phase = 0;
  for (; row < a.n_rows; row += step) {
    // into the slot of the round before this one: all lanes have read it, they have exchanged sums since
    fetch(row + (kSlots - 1) * step, slot == 0 ? kSlots - 1 : slot - 1);
    async_wait<kSlots - 1>();
    warp_sync();
    F2 x[kRows][kPairs];
    float v[4] = {0.f, 0.f, 0.f, 0.f}, mean = 0.f;            // mean of row lane >> 3
#pragma unroll
    for (int r = 0; r < kRows; ++r) window_read<T, kEpt>(window(slot, r), source(row + r < a.n_rows ? row + r : 0), lane, x[r]);
    if constexpr (kCentered) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        F2 acc = x[r][0];
#pragma unroll
        for (int i = 1; i < kPairs; ++i) acc = add2(acc, x[r][i]);
        v[r] = f2_lo(acc) + f2_hi(acc);
      }
      mean = norm_warps_four_sums(v, warps, g, scratch, phase) * inv;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if constexpr (kCentered) {
        const F2 minus_mean = both(-norm_warp_of_four(mean, r));
#pragma unroll
        for (int i = 0; i < kPairs; ++i) x[r][i] = add2(x[r][i], minus_mean);
        if (count < 32 * kEpt) {            // behind the row's end there is nothing to centre
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            x[r][i] = f2(lane + 64 * i < count ? f2_lo(x[r][i]) : 0.f, lane + 64 * i + 32 < count ? f2_hi(x[r][i]) : 0.f);
        }
      }
      F2 acc = both(0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) acc = fma2(x[r][i], x[r][i], acc);
      v[r] = f2_lo(acc) + f2_hi(acc);
    }
    const float rstd = norm_rsqrt(fmaf(norm_warps_four_sums(v, warps, g, scratch, phase), inv, a.eps));
    {
      const int r = lane >> 3;
      if (column == 0 && (lane & 7) == 0 && r < kRows && row + r < a.n_rows) {
        if (kCentered && a.mean != nullptr) a.mean[row + r] = mean;
        if (a.rstd != nullptr) a.rstd[row + r] = rstd;
      }
    }
    F2 scale[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) scale[r] = both(norm_warp_of_four(rstd, r));
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 lo = parameters[64 * i], hi = parameters[64 * i + 32];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        F2 o = mul2(x[r][i], scale[r]);
        if (rounded) o = f2(norm_round<T>(f2_lo(o)), norm_round<T>(f2_hi(o)));
        if constexpr (kCentered) x[r][i] = fma2(o, f2(lo.x, hi.x), f2(lo.y, hi.y));
        else x[r][i] = mul2(o, f2(lo.x, hi.x));
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (row + r < a.n_rows) window_store<T, kEpt>(static_cast<T*>(a.y) + (row + r) * a.hidden + column, count, lane, x[r]);
    }
    slot = slot + 1 == kSlots ? 0 : slot + 1;
  }
  async_wait<0>();
}

template <typename T, typename W, bool kCentered, int kEpt>
__global__ void __launch_bounds__(kWindowThreads, 1)
norm_backward_window_kernel(NormBackwardArgs a) {
  allow_dependents();      // the small kernel that adds up the partial sums
  typedef Window<T, kEpt, true> Shape;
  constexpr int kRows = Shape::kRows, kSlots = Shape::kSlots, kPairs = kEpt / 2;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                    // [slot][row][x, dy][warp][piece], then the gain of every column
  __shared__ float scratch[2][kNormMaxWarps * 4];
  const int warps = a.group_warps;
  const int groups = kWindowWarps / warps;
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int g = warp / warps;
  const int column = (warp - g * warps) * 32 * kEpt;
  const int count = a.hidden - column < 32 * kEpt ? a.hidden - column : 32 * kEpt;
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const long long last = a.n_rows - 1;      // rows are counted from the last one, as above
  const float inv = 1.f / static_cast<float>(a.hidden);
  float* gains = reinterpret_cast<float*>(stream_ring + Shape::kRingBytes / 16);
  for (int c = static_cast<int>(threadIdx.x); c < warps * 32 * kEpt; c += kWindowThreads)
    gains[c] = c < a.hidden && a.w != nullptr ? a.offset + CeElem<W>::load(static_cast<const W*>(a.w) + c) : 1.f;
  __syncthreads();
  gains += column + lane;
  F2 dw[kPairs], db[kCentered ? kPairs : 1];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    dw[i] = both(0.f);
    if (kCentered) db[i] = both(0.f);
  }
  auto window = [&](int slot, int r, int which) {
    return stream_ring + (((slot * kRows + r) * 2 + which) * kWindowWarps + warp) * Shape::kPieces;
  };
  auto source_x = [&](long long row) { return static_cast<const T*>(a.x) + row * a.ld_x + column; };
  auto source_dy = [&](long long row) { return static_cast<const T*>(a.dy) + row * a.ld_dy + column; };
  auto fetch = [&](long long base, int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = base + r < a.n_rows;
      window_fetch<T, Shape::kPieces>(window(slot, r, 0), source_x(live ? last - base - r : 0), live ? count : 0, lane);
      window_fetch<T, Shape::kPieces>(window(slot, r, 1), source_dy(live ? last - base - r : 0), live ? count : 0, lane);
    }
    async_commit();
  };
  float next_mean[kRows], next_rstd[kRows];
  auto fetch_statistics = [&](long long base) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = base + r < a.n_rows;
      next_mean[r] = kCentered && live ? __ldg(a.mean + last - base - r) : 0.f;
      next_rstd[r] = live ? __ldg(a.rstd + last - base - r) : 0.f;
    }
  };
  long long row = g < groups ? (static_cast<long long>(blockIdx.x) * groups + g) * kRows : a.n_rows;
  if (g < groups) {                                           // warps that make no whole group wait for the end
#pragma unroll
    for (int s = 0; s < kSlots - 1; ++s) fetch(row + s * step, s);
    fetch_statistics(row);
  }
  int slot = 0, phase = 0;
  for (; row < a.n_rows; row += step) {
    fetch(row + (kSlots - 1) * step, slot == 0 ? kSlots - 1 : slot - 1);
    async_wait<kSlots - 1>();
    warp_sync();
    F2 xhat[kRows][kPairs], m[kRows][kPairs], minus_mean[kRows], s_mx[kRows], s_m[kRows];
    float rstd[kRows], v[4] = {0.f, 0.f, 0.f, 0.f};           // (sum m xhat, sum m) of each row
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long from = row + r < a.n_rows ? last - row - r : 0;
      window_read<T, kEpt>(window(slot, r, 0), source_x(from), lane, xhat[r]);
      window_read<T, kEpt>(window(slot, r, 1), source_dy(from), lane, m[r]);
      rstd[r] = next_rstd[r];
      minus_mean[r] = both(-next_mean[r]);
      s_mx[r] = s_m[r] = both(0.f);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const F2 gain = f2(gains[64 * i], gains[64 * i + 32]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        // behind the row's end dy is zero, which keeps xhat out of every sum
        if (kCentered) xhat[r][i] = add2(xhat[r][i], minus_mean[r]);
        xhat[r][i] = mul2(xhat[r][i], both(rstd[r]));
        F2 xw = xhat[r][i];
        if (rounded) xw = f2(norm_round<T>(f2_lo(xw)), norm_round<T>(f2_hi(xw)));
        dw[i] = fma2(m[r][i], xw, dw[i]);
        if (kCentered) db[i] = add2(db[i], m[r][i]);
        m[r][i] = mul2(m[r][i], gain);
        s_mx[r] = fma2(m[r][i], xhat[r][i], s_mx[r]);
        if (kCentered) s_m[r] = add2(s_m[r], m[r][i]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      v[2 * r] = f2_lo(s_mx[r]) + f2_hi(s_mx[r]);
      v[2 * r + 1] = f2_lo(s_m[r]) + f2_hi(s_m[r]);
    }
    fetch_statistics(row + step);
    const float sums = norm_warps_four_sums(v, warps, g, scratch, phase) * -inv;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const F2 minus_c = both(norm_warp_of_four(sums, 2 * r));
      const F2 minus_m = both(kCentered ? norm_warp_of_four(sums, 2 * r + 1) : 0.f);
      if (row + r >= a.n_rows) continue;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        if (kCentered) m[r][i] = add2(m[r][i], minus_m);
        m[r][i] = mul2(fma2(xhat[r][i], minus_c, m[r][i]), both(rstd[r]));
      }
      window_store<T, kEpt>(static_cast<T*>(a.dx) + (last - row - r) * a.hidden + column, count, lane, m[r]);
    }
    slot = slot + 1 == kSlots ? 0 : slot + 1;
  }
  async_wait<0>();
  // the groups' sums, added up by the threads of the block in the groups' order
  float* fold = reinterpret_cast<float*>(stream_ring);
  auto leave = [&](F2* acc, float* partial) {
    __syncthreads();
    if (g < groups) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        fold[warp * 32 * kEpt + lane + 64 * i] = f2_lo(acc[i]);
        fold[warp * 32 * kEpt + lane + 64 * i + 32] = f2_hi(acc[i]);
      }
    }
    __syncthreads();
    float* out = partial + static_cast<size_t>(blockIdx.x) * a.hidden;
    for (int c = static_cast<int>(threadIdx.x); c < a.hidden; c += kWindowThreads) {
      float s = 0.f;
      for (int k = 0; k < groups; ++k) s += fold[k * warps * 32 * kEpt + c];
      out[c] = s;
    }
  };
  if (a.dw_partial != nullptr) leave(dw, a.dw_partial);
  if constexpr (kCentered) {
    if (a.db_partial != nullptr) leave(db, a.db_partial);
  }
}

// ---- rows of at most 32 elements without that alignment: one element per lane, groups of 4 to 32 lanes, several rows at a time
template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNarrowThreads)
norm_forward_tiny_kernel(NormForwardArgs a) {
  constexpr int kRows = kNarrowForwardRows;
  const int group = 1 << a.log2_group;
  const int groups = kNarrowThreads >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const bool column = t < a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const float inv = 1.f / static_cast<float>(a.hidden);
  const long long base = static_cast<long long>(blockIdx.x) * groups * kRows + (threadIdx.x >> a.log2_group);
  const float gain = column && a.w != nullptr ? a.offset + CeElem<W>::load(static_cast<const W*>(a.w) + t) : 1.f;
  const float bias = column && a.b != nullptr ? CeElem<W>::load(static_cast<const W*>(a.b) + t) : 0.f;
  float x[kRows], v[4], mean = 0.f;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const long long row = base + r * groups;
    x[r] = column && row < a.n_rows ? CeElem<T>::load(static_cast<const T*>(a.x) + row * a.ld_x + t) : 0.f;
  }
  if (kCentered) mean = lane_four_sums(x, group) * inv;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float m = kCentered ? of_four(mean, r, a.log2_group) : 0.f;
    x[r] = column ? x[r] - m : 0.f;
    v[r] = x[r] * x[r];
  }
  const float rstd = norm_rsqrt(fmaf(lane_four_sums(v, group), inv, a.eps));
  {
    const long long row = base + t / (group >> 2) * groups;
    if (t % (group >> 2) == 0 && row < a.n_rows) {
      if (kCentered && a.mean != nullptr) a.mean[row] = mean;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const long long row = base + r * groups;
    float o = x[r] * of_four(rstd, r, a.log2_group);
    if (rounded) o = norm_round<T>(o);
    o = kCentered ? fmaf(o, gain, bias) : o * gain;
    if (column && row < a.n_rows) CeElem<T>::store(static_cast<T*>(a.y) + row * a.hidden + t, o);
  }
}

template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNarrowThreads)
norm_backward_tiny_kernel(NormBackwardArgs a) {
  allow_dependents();      // the small kernel that adds up the partial sums
  constexpr int kRows = kNarrowBackwardRows;
  __shared__ float fold[kNarrowThreads];
  const int group = 1 << a.log2_group;
  const int groups = kNarrowThreads >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const bool column = t < a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const float inv = 1.f / static_cast<float>(a.hidden);
  const float gain = column && a.w != nullptr ? a.offset + CeElem<W>::load(static_cast<const W*>(a.w) + t) : 1.f;
  float dw = 0.f, db = 0.f;
  const long long step = static_cast<long long>(gridDim.x) * groups * kRows;
  for (long long base = static_cast<long long>(blockIdx.x) * groups * kRows; base < a.n_rows; base += step) {
    float xhat[kRows], m[kRows], rstd[kRows], v[4];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + g + r * groups;
      const bool live = row < a.n_rows;
      rstd[r] = live ? __ldg(a.rstd + row) : 0.f;
      const float mean = kCentered && live ? __ldg(a.mean + row) : 0.f;
      xhat[r] = column && live ? (CeElem<T>::load(static_cast<const T*>(a.x) + row * a.ld_x + t) - mean) * rstd[r] : 0.f;
      m[r] = column && live ? CeElem<T>::load(static_cast<const T*>(a.dy) + row * a.ld_dy + t) : 0.f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      dw = fmaf(m[r], rounded ? norm_round<T>(xhat[r]) : xhat[r], dw);
      db += m[r];
      m[r] *= gain;
      v[2 * r] = m[r] * xhat[r];
      v[2 * r + 1] = m[r];
    }
    const float sums = lane_four_sums(v, group) * inv;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + g + r * groups;
      const float c = of_four(sums, 2 * r, a.log2_group), mm = kCentered ? of_four(sums, 2 * r + 1, a.log2_group) : 0.f;
      if (column && row < a.n_rows) CeElem<T>::store(static_cast<T*>(a.dx) + row * a.hidden + t, rstd[r] * (fmaf(-xhat[r], c, m[r]) - mm));
    }
  }
  auto leave = [&](float acc, float* partial) {
    __syncthreads();
    fold[threadIdx.x] = acc;
    __syncthreads();
    if (g == 0 && column) {
      float s = 0.f;
      for (int k = 0; k < groups; ++k) s += fold[(k << a.log2_group) + t];
      partial[static_cast<size_t>(blockIdx.x) * a.hidden + t] = s;
    }
  };
  if (a.dw_partial != nullptr) leave(dw, a.dw_partial);
  if (kCentered && a.db_partial != nullptr) leave(db, a.db_partial);
}

// gradient[c] = sum over the blocks' partials; 32 columns per block, each summed by 32 threads in a fixed order.
// blockIdx.y 0: the weight's, 1: the bias's.
constexpr int kNormReduceLanes = 32;
template <typename W>
__global__ void __launch_bounds__(32 * kNormReduceLanes)
norm_parameter_gradient_kernel(const float* dw_partial, const float* db_partial, int blocks, int hidden, W* dw, W* db) {
  __shared__ float part[kNormReduceLanes][33];
  wait_for_previous_kernel();
  const float* partial = blockIdx.y == 0 ? dw_partial : db_partial;
  W* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  const int col = static_cast<int>(blockIdx.x) * 32 + static_cast<int>(threadIdx.x);
  float s = 0.f;
  if (col < hidden) {
#pragma unroll 8
    for (int b = static_cast<int>(threadIdx.y); b < blocks; b += kNormReduceLanes) s += partial[static_cast<size_t>(b) * hidden + col];
  }
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  // transposed: a warp adds up one column
  s = part[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int mine = static_cast<int>(blockIdx.x) * 32 + static_cast<int>(threadIdx.y);
  if (threadIdx.x == 0 && mine < hidden) CeElem<W>::store(out + mine, s);
}

// ---- rows longer than the registers of a block hold: one block per row, read again for every pass (from L2)

// two sums over the block, to all its threads
__device__ __forceinline__ void norm_block_sum(float& s0, float& s1, float (*scratch)[kNormMaxWarps * 4], int& phase) {
  const float v[4] = {s0, s1, 0.f, 0.f};
  const float sums = norm_warps_four_sums(v, kNormMaxWarps, 0, scratch, phase);
  s0 = norm_warp_of_four(sums, 0);
  s1 = norm_warp_of_four(sums, 1);
}

template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNormMaxThreads)
norm_forward_long_kernel(NormForwardArgs a) {
  __shared__ float scratch[2][kNormMaxWarps * 4];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const W* w = static_cast<const W*>(a.w);
  const W* b = static_cast<const W*>(a.b);
  const int tid = static_cast<int>(threadIdx.x);
  int phase = 0;
  float mean = 0.f;
  float s[2] = {0.f, 0.f};
  if constexpr (kCentered) {
    for (int c = tid; c < a.hidden; c += kNormMaxThreads) s[0] += CeElem<T>::load(x + c);
    norm_block_sum(s[0], s[1], scratch, phase);
    mean = s[0] / static_cast<float>(a.hidden);
    s[0] = 0.f;
  }
  for (int c = tid; c < a.hidden; c += kNormMaxThreads) {
    const float v = CeElem<T>::load(x + c) - mean;
    s[0] = fmaf(v, v, s[0]);
  }
  norm_block_sum(s[0], s[1], scratch, phase);
  const float rstd = norm_rsqrt(s[0] / static_cast<float>(a.hidden) + a.eps);
  if (tid == 0) {
    if (kCentered && a.mean != nullptr) a.mean[row] = mean;
    if (a.rstd != nullptr) a.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(a.y) + row * a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
  for (int c = tid; c < a.hidden; c += kNormMaxThreads) {
    float v = (CeElem<T>::load(x + c) - mean) * rstd;
    if (rounded) v = norm_round<T>(v);
    if (w != nullptr) v *= a.offset + CeElem<W>::load(w + c);
    if (b != nullptr) v += CeElem<W>::load(b + c);
    CeElem<T>::store(y + c, v);
  }
}

template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNormMaxThreads)
norm_backward_long_kernel(NormBackwardArgs a) {
  __shared__ float scratch[2][kNormMaxWarps * 4];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
  const W* w = static_cast<const W*>(a.w);
  const float mean = kCentered ? a.mean[row] : 0.f, rstd = a.rstd[row];
  int phase = 0;
  float s[2] = {0.f, 0.f};
  for (int c = static_cast<int>(threadIdx.x); c < a.hidden; c += kNormMaxThreads) {
    const float m = CeElem<T>::load(dy + c) * (w != nullptr ? a.offset + CeElem<W>::load(w + c) : 1.f);
    s[0] = fmaf(m, (CeElem<T>::load(x + c) - mean) * rstd, s[0]);
    s[1] += m;
  }
  norm_block_sum(s[0], s[1], scratch, phase);
  const float c2 = s[0] / static_cast<float>(a.hidden);
  const float c1 = kCentered ? s[1] / static_cast<float>(a.hidden) : 0.f;
  T* dx = static_cast<T*>(a.dx) + row * a.hidden;
  for (int c = static_cast<int>(threadIdx.x); c < a.hidden; c += kNormMaxThreads) {
    const float m = CeElem<T>::load(dy + c) * (w != nullptr ? a.offset + CeElem<W>::load(w + c) : 1.f);
    CeElem<T>::store(dx + c, rstd * (fmaf(-(CeElem<T>::load(x + c) - mean) * rstd, c2, m) - c1));
  }
}

// partial sums of the parameters' gradients for such rows: one thread per column, blockIdx.y = a share of the rows
template <typename T, bool kCentered>
__global__ void __launch_bounds__(kNormColumnThreads)
norm_parameter_partial_long_kernel(NormBackwardArgs a) {
  allow_dependents();      // the small kernel that adds up the partial sums
  const int c = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x);
  if (c >= a.hidden) return;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  const bool rounded = !kCentered && a.round_xhat != 0;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    const float d = CeElem<T>::load(dy + row * a.ld_dy + c);
    float xhat = (CeElem<T>::load(x + row * a.ld_x + c) - (kCentered ? a.mean[row] : 0.f)) * a.rstd[row];
    if (rounded) xhat = norm_round<T>(xhat);
    dw = fmaf(d, xhat, dw);
    db += d;
  }
  if (a.dw_partial != nullptr) a.dw_partial[static_cast<size_t>(blockIdx.y) * a.hidden + c] = dw;
  if (kCentered && a.db_partial != nullptr) a.db_partial[static_cast<size_t>(blockIdx.y) * a.hidden + c] = db;
}

}  // namespace flce
