// Layer norm and RMSNorm over the rows of a matrix, forward and backward (src/liger_kernel/ops/layer_norm.py and
// src/liger_kernel/ops/rms_norm.py of the reference are the operators they stand in for).
//
//   layer norm   xhat = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),   y = xhat * (offset + w) + b
//   RMSNorm      xhat = x * rstd,           rstd = 1 / sqrt(mean(x^2) + eps),            y = xhat * (offset + w)
//   backward     m = dy * (offset + w);  dx = rstd * (m - mean(m) - xhat * mean(m * xhat))   (RMSNorm: without mean(m))
//                dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Both directions are bound by HBM: forward moves a row in and out, backward two rows in and one out.  A row is read once and
// stays in the registers of the threads that share it, so the variance is taken around the mean that is already known (no
// sum of squares minus square of sum) at no further traffic.  A *group* of 2..512 threads shares a row; a block holds as many
// groups as fit, so narrow rows need no barrier and wide rows have one per reduction.  Everything between load and store is
// fp32; the only roundings to fewer bits are those of the results, and of xhat in the "llama" casting mode, which asks for it.
//
// In backward a thread keeps the same columns for all rows of its block, so the weight's and the bias's gradient are sums in
// its registers; blocks leave one partial sum per column, added up in block order by a second kernel: no atomics, the same
// bits in every run.  The next row is on its way while the current one is reduced.
#pragma once

#include <type_traits>

#include "ce_kernels.cuh"
#include "packed_math.cuh"
#include "simt_common.cuh"

namespace flce {

constexpr int kNormMaxThreads = 512;     // largest group, and the block of the backward kernel
constexpr int kNormForwardThreads = 256; // block of the forward kernel unless a row needs a larger group
constexpr int kNormMaxWarps = kNormMaxThreads / 32;
constexpr int kNormMaxEpt = 32;          // elements of a row per thread: rows of up to 16384 elements stay in registers

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
  int log2_group;
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
};

// One thread's share of a row: kEpt elements as kEpt / kUnit units of kUnit consecutive ones.  The units of a warp lie side by
// side in strides of 32, so that neighbouring threads touch neighbouring memory and a thread's accesses differ by constants;
// groups of fewer than 32 threads have one unit per thread.  kUnit is 1, or as many elements of the row's type as fill
// 16 bytes; then rows start on 16-byte boundaries and hold whole units.
template <int kUnit, int kEpt>
__device__ __forceinline__ int norm_first_column(int t) {
  constexpr int kUnits = kEpt / kUnit;
  return (kUnits == 1 ? t : (t >> 5) * 32 * kUnits + (t & 31)) * kUnit;
}
template <int kUnit>
__device__ __forceinline__ int norm_column(int first, int e) {
  return first + (e / kUnit) * 32 * kUnit + e % kUnit;
}

template <typename E, int kUnit, int kEpt>
struct NormChunk {
  static constexpr int kUnits = kEpt / kUnit;
  static constexpr int kPer = kUnit == 1 ? 1 : kUnit * static_cast<int>(sizeof(E)) / 16;   // words per unit
  typedef typename std::conditional<kUnit == 1, E, uint4>::type Word;
  Word q[kUnits * kPer];

  // zeros behind the row's end
  __device__ __forceinline__ void load(const E* row, int first, int hidden) {
    const Word* p = reinterpret_cast<const Word*>(row + first);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        q[u * kPer + i] = Word();
        if (first + u * 32 * kUnit < hidden) q[u * kPer + i] = p[u * 32 * kPer + i];
      }
    }
  }
  __device__ __forceinline__ float get(int e) const { return CeElem<E>::load(reinterpret_cast<const E*>(q) + e); }
  __device__ __forceinline__ void set(int e, float v) { CeElem<E>::store(reinterpret_cast<E*>(q) + e, v); }

  __device__ __forceinline__ void store(E* row, int first, int hidden) const {
    Word* p = reinterpret_cast<Word*>(row + first);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (first + u * 32 * kUnit < hidden) p[u * 32 * kPer + i] = q[u * kPer + i];
      }
    }
  }
};

// Sums of kN values over each group, returned to all its threads; every thread of the block calls it.  Groups of more than a
// warp meet in shared memory, in one of two buffers taken in turn: a thread writes a buffer again only behind the barrier
// of the call in between, which the readers of the older sums reach after reading them, so one barrier per call is enough.
template <int kN>
__device__ __forceinline__ void norm_group_sum(float (&v)[kN], int log2_group, float (*scratch)[kNormMaxWarps * kN], int& phase) {
  const int lanes = log2_group < 5 ? (1 << log2_group) : 32;
  for (int o = lanes >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if (log2_group <= 5) return;
  float* buf = scratch[phase];
  phase ^= 1;
  const int tid = static_cast<int>(threadIdx.x);
  if ((tid & 31) == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) buf[(tid >> 5) * kN + i] = v[i];
  }
  __syncthreads();
  const int warps = 1 << (log2_group - 5);
  const float* mine = buf + (tid >> log2_group) * warps * kN;
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = 0.f;
  for (int w = 0; w < warps; ++w) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] += mine[w * kN + i];
  }
}

template <typename T>
__device__ __forceinline__ float norm_round(float v) {
  T r;
  CeElem<T>::store(&r, v);
  return CeElem<T>::load(&r);
}

// y and the row statistics.  One row per group; blocks of 256 threads, or of the group if that is larger.
template <typename T, typename W, bool kCentered, int kUnit, int kEpt>
__global__ void __launch_bounds__(kNormMaxThreads)
norm_forward_kernel(NormForwardArgs a) {
  __shared__ float scratch[2][kNormMaxWarps];
  const int group = 1 << a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int first = norm_first_column<kUnit, kEpt>(t);
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> a.log2_group) + (threadIdx.x >> a.log2_group);
  const bool live = row < a.n_rows;
  const int hidden = live ? a.hidden : 0;     // a group behind the last row takes part in the barriers only
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ld_x;
  NormChunk<T, kUnit, kEpt> c;
  c.load(x, first, hidden);
  float v[kEpt];
  float s[1] = {0.f};
#pragma unroll
  for (int e = 0; e < kEpt; ++e) v[e] = c.get(e);
  int phase = 0;
  float mean = 0.f;
  if constexpr (kCentered) {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) s[0] += v[e];
    norm_group_sum<1>(s, a.log2_group, scratch, phase);
    mean = s[0] / static_cast<float>(a.hidden);
    s[0] = 0.f;
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      v[e] = norm_column<kUnit>(first, e) < hidden ? v[e] - mean : 0.f;
      s[0] = fmaf(v[e], v[e], s[0]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) s[0] = fmaf(v[e], v[e], s[0]);
  }
  norm_group_sum<1>(s, a.log2_group, scratch, phase);
  if (!live) return;
  const float rstd = 1.f / sqrtf(s[0] / static_cast<float>(a.hidden) + a.eps);
  if (t == 0) {
    if (kCentered && a.mean != nullptr) a.mean[row] = mean;
    if (a.rstd != nullptr) a.rstd[row] = rstd;
  }
  NormChunk<T, kUnit, kEpt> y;
  const bool rounded = !kCentered && a.round_xhat != 0;
#pragma unroll
  for (int e = 0; e < kEpt; ++e) {
    v[e] *= rstd;
    if (rounded) v[e] = norm_round<T>(v[e]);
  }
  if (a.w != nullptr) {
    NormChunk<W, kUnit, kEpt> w;
    w.load(static_cast<const W*>(a.w), first, hidden);
    if (a.b != nullptr) {
      NormChunk<W, kUnit, kEpt> b;
      b.load(static_cast<const W*>(a.b), first, hidden);
#pragma unroll
      for (int e = 0; e < kEpt; ++e) v[e] = fmaf(v[e], a.offset + w.get(e), b.get(e));
    } else {
#pragma unroll
      for (int e = 0; e < kEpt; ++e) v[e] *= a.offset + w.get(e);
    }
  } else if (a.b != nullptr) {
    NormChunk<W, kUnit, kEpt> b;
    b.load(static_cast<const W*>(a.b), first, hidden);
#pragma unroll
    for (int e = 0; e < kEpt; ++e) v[e] += b.get(e);
  }
#pragma unroll
  for (int e = 0; e < kEpt; ++e) y.set(e, v[e]);
  y.store(static_cast<T*>(a.y) + row * a.hidden, first, hidden);
}

// dx, and this block's share of the parameters' gradients.  A fixed grid of blocks of 512 threads walks over the rows.  The
// rows are kept as they were loaded and converted again after the reduction: the registers go to the sums and to the next row.
template <typename T, typename W, bool kCentered, int kUnit, int kEpt>
__global__ void __launch_bounds__(kNormMaxThreads)
norm_backward_kernel(NormBackwardArgs a) {
  constexpr int kSums = kCentered ? 2 : 1;
  constexpr bool kAhead = kEpt * sizeof(T) <= 32;      // room for the next row beside the current one
  __shared__ float scratch[2][kNormMaxWarps * kSums];
  __shared__ float fold[kNormMaxThreads / 2 * kEpt];
  const int group = 1 << a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int first = norm_first_column<kUnit, kEpt>(t);
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const int groups = static_cast<int>(blockDim.x) >> a.log2_group;
  const long long step = static_cast<long long>(gridDim.x) * groups;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const bool gain = a.w != nullptr;
  typedef NormChunk<T, kUnit, kEpt> Row;
  typedef NormChunk<W, kUnit, kEpt> Parameters;

  Parameters w;
  w.load(static_cast<const W*>(a.w), first, gain ? a.hidden : 0);
  float dw[kEpt], db[kCentered ? kEpt : 1];
#pragma unroll
  for (int e = 0; e < kEpt; ++e) {
    dw[e] = 0.f;
    if (kCentered) db[e] = 0.f;
  }
  struct Fetched {
    Row x, dy;
    float mean, rstd;
  };
  // a row behind the last one is loaded as zeros: it adds nothing and is not stored
  auto fetch = [&](Fetched& f, long long row) {
    const bool live = row < a.n_rows;
    const int hidden = live ? a.hidden : 0;
    const long long r = live ? row : 0;
    f.x.load(static_cast<const T*>(a.x) + r * a.ld_x, first, hidden);
    f.dy.load(static_cast<const T*>(a.dy) + r * a.ld_dy, first, hidden);
    f.mean = kCentered && live ? a.mean[r] : 0.f;
    f.rstd = live ? a.rstd[r] : 0.f;
  };
  Fetched cur;
  long long row = static_cast<long long>(blockIdx.x) * groups;
  if (kAhead) fetch(cur, row + g);
  int phase = 0;
  for (; row < a.n_rows; row += step) {       // the same number of rounds in every thread of the block
    Fetched next;
    if (kAhead) {
      if (row + step < a.n_rows) fetch(next, row + step + g);
    } else {
      fetch(cur, row + g);
    }
    float s[kSums] = {};
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      // the columns behind the row's end hold dy = 0, which keeps their xhat out of every sum
      const float xhat = (cur.x.get(e) - cur.mean) * cur.rstd;
      float d = cur.dy.get(e);
      dw[e] = fmaf(d, rounded ? norm_round<T>(xhat) : xhat, dw[e]);
      if (kCentered) db[e] += d;
      if (gain) d *= a.offset + w.get(e);
      s[0] = fmaf(d, xhat, s[0]);
      if (kCentered) s[kSums - 1] += d;
    }
    norm_group_sum<kSums>(s, a.log2_group, scratch, phase);
    const float c = s[0] / static_cast<float>(a.hidden);
    const float m = kCentered ? s[kSums - 1] / static_cast<float>(a.hidden) : 0.f;
    if (row + g < a.n_rows) {
      Row out;
#pragma unroll
      for (int e = 0; e < kEpt; ++e) {
        const float xhat = (cur.x.get(e) - cur.mean) * cur.rstd;
        float d = cur.dy.get(e);
        if (gain) d *= a.offset + w.get(e);
        out.set(e, cur.rstd * (fmaf(-xhat, c, d) - m));
      }
      out.store(static_cast<T*>(a.dx) + (row + g) * a.hidden, first, a.hidden);
    }
    if (kAhead) cur = next;
  }
  // the groups of the block, folded in halves in a fixed order
  auto leave = [&](float (&acc)[kEpt], float* partial) {
    for (int half = groups >> 1; half > 0; half >>= 1) {
      __syncthreads();
      if (g >= half && g < 2 * half) {
#pragma unroll
        for (int e = 0; e < kEpt; ++e) fold[((g - half) * kEpt + e) * group + t] = acc[e];
      }
      __syncthreads();
      if (g < half) {
#pragma unroll
        for (int e = 0; e < kEpt; ++e) acc[e] += fold[(g * kEpt + e) * group + t];
      }
    }
    if (g == 0) {
      float* mine = partial + static_cast<size_t>(blockIdx.x) * a.hidden;
#pragma unroll
      for (int e = 0; e < kEpt; ++e) {
        const int col = norm_column<kUnit>(first, e);
        if (col < a.hidden) mine[col] = acc[e];
      }
    }
  };
  if (a.dw_partial != nullptr) leave(dw, a.dw_partial);
  if constexpr (kCentered) {
    if (a.db_partial != nullptr) leave(db, a.db_partial);
  }
}

// ---- rows of whole, aligned 16-byte vectors, more than a warp's worth: streamed through shared memory
//
// What the kernels above lose is not bandwidth but issue slots and waiting: at 32768 x 4096 bf16 they ran at 46 % (forward) and
// 41 % (backward) of the copy rate with rows of one warp reaching 55 % and fp32 rows, with half the elements per byte, 87 %.
// Here the arithmetic goes two elements to an instruction, and the next rows are always on their way: every thread copies
// the vectors that it will read itself, with cp.async, so the ring needs no barrier and no wait on another thread.

constexpr int kStreamThreads = 512;

// Four sums over a group of `warps` warps.  In a warp by six exchanges: lanes that differ in bit 4 trade two sums for the other
// two, those that differ in bit 3 one for the other; bits 4 and 3 of the lane then name its sum.  Across warps through one of
// two buffers, taken in turn (see norm_group_sum).  Returns sum number lane >> 3, the same in the eight lanes that share it.
__device__ __forceinline__ float stream_four_sums(const float (&v)[4], int warps, int group_id, float (*scratch)[kNormMaxWarps * 4],
                                                  int& phase) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const bool up = (lane & 16) != 0, right = (lane & 8) != 0;
  const float a0 = __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16) + (up ? v[2] : v[0]);
  const float a1 = __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16) + (up ? v[3] : v[1]);
  float sum = __shfl_xor_sync(0xffffffffu, right ? a0 : a1, 8) + (right ? a1 : a0);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (warps == 1) return sum;
  float* buf = scratch[phase];
  phase ^= 1;
  if ((lane & 7) == 0) buf[(threadIdx.x >> 5) * 4 + (lane >> 3)] = sum;
  named_barrier(1 + group_id, warps * 32);
  const float* of = buf + group_id * warps * 4 + (lane >> 3);
  sum = 0.f;
  for (int w = lane & 7; w < warps; w += 8) sum += of[w * 4];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

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

// Shape of the streaming kernels by the vectors per thread: rows that a group takes per round, rounds in the ring, blocks per SM.
// Two rows of backward are four sums, as four rows of forward are.
template <int kUnits, bool kGrad>
struct Stream {
  static constexpr int kRows = kUnits == 4 ? 1 : (kUnits == 2 || kGrad ? 2 : 4);
  static constexpr int kSlots = 3;
  static constexpr int kBlocksPerSm = kUnits == 1 ? 2 : 1;
  static constexpr int kRingBytes = kSlots * kRows * (kGrad ? 2 : 1) * kUnits * kStreamThreads * 16;
};

// y and the row statistics.  Each thread of a group owns kUnits vectors of columns, their gain and bias in registers; a group takes
// kRows rows per round, which meet in one reduction (one barrier, if the group is wider than a warp) for the means and one for
// the variances.  A fixed grid walks over the rows.
template <typename T, typename W, bool kCentered, int kUnits>
__global__ void __launch_bounds__(kStreamThreads, (Stream<kUnits, false>::kBlocksPerSm))
norm_forward_stream_kernel(NormForwardArgs a) {
  constexpr int kRows = Stream<kUnits, false>::kRows, kSlots = Stream<kUnits, false>::kSlots;
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  FLCE_DYNAMIC_SHARED(uint4, stream_ring);                    // [slot][row][unit][thread]
  __shared__ float scratch[2][kNormMaxWarps * 4];
  const int group = 1 << a.log2_group;
  const int warps = group >> 5;
  const int groups = kStreamThreads >> a.log2_group;
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
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
      for (int u = 0; u < kUnits; ++u) async_copy16(&cell(slot, r, u), x + u * 32, live && first + u * 32 < vectors);
    }
    async_commit();
  };
  long long row = (static_cast<long long>(blockIdx.x) * groups + g) * kRows;
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s) fetch(row + s * step, s);
  int slot = 0, phase = 0;
  const float inv = 1.f / static_cast<float>(a.hidden);
  for (; row < a.n_rows; row += step) {
    // into the slot of the round before this one, which this thread, its only reader, has read for the last time
    fetch(row + (kSlots - 1) * step, slot == 0 ? kSlots - 1 : slot - 1);
    async_wait<kSlots - 1>();
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    F2 minus_mean[kRows];
    float mean = 0.f;                       // of row lane >> 3
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
      mean = stream_four_sums(v, warps, g, scratch, phase) * inv;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      minus_mean[r] = both(kCentered ? -__shfl_sync(0xffffffffu, mean, r * 8) : 0.f);
      F2 acc = both(0.f);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint4 raw = cell(slot, r, u);
        if (!kCentered || first + u * 32 < vectors) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            F2 e = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw) + i * Pairs<T>::kWords);
            if (kCentered) e = add2(e, minus_mean[r]);
            acc = fma2(e, e, acc);
          }
        }
      }
      v[r] = f2_lo(acc) + f2_hi(acc);
    }
    const float rstd = 1.f / sqrtf(fmaf(stream_four_sums(v, warps, g, scratch, phase), inv, a.eps));
    {
      const int r = static_cast<int>(threadIdx.x & 31) >> 3;
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
__global__ void __launch_bounds__(kStreamThreads, (Stream<kUnits, true>::kBlocksPerSm))
norm_backward_stream_kernel(NormBackwardArgs a) {
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
      const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (live ? row : 0) * a.ld_x) + first;
      const uint4* dy = reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + (live ? row : 0) * a.ld_dy) + first;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        async_copy16(&cell(slot, r, 0, u), x + u * 32, live && first + u * 32 < vectors);
        async_copy16(&cell(slot, r, 1, u), dy + u * 32, live && first + u * 32 < vectors);
      }
    }
    async_commit();
  };
  float next_mean[kRows], next_rstd[kRows];
  auto fetch_statistics = [&](long long base) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = base + r < a.n_rows;
      next_mean[r] = kCentered && live ? __ldg(a.mean + base + r) : 0.f;
      next_rstd[r] = live ? __ldg(a.rstd + base + r) : 0.f;
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
    const float sum = stream_four_sums(v, warps, g, scratch, phase);
    const float inv = 1.f / static_cast<float>(a.hidden);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float c = __shfl_sync(0xffffffffu, sum, r * 16) * inv;
      const float m_mean = kCentered ? __shfl_sync(0xffffffffu, sum, r * 16 + 8) * inv : 0.f;
      const long long row = round + mine + r;
      if (row >= a.n_rows) continue;
      uint4* dx = reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + row * a.hidden) + first;
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

// ---- rows of at most 32 aligned 16-byte vectors: one vector per lane, several rows to a warp, kRows of them per thread at a
// time, so that the loads and the shuffles of one row hide those of another

constexpr int kNarrowThreads = 256;

template <typename T, typename W, bool kCentered, int kRows>
__global__ void __launch_bounds__(kNarrowThreads)
norm_forward_narrow_kernel(NormForwardArgs a) {
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  const int group = 1 << a.log2_group;
  const int groups = kNarrowThreads >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const bool column = t * kVec < a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
  const long long base = static_cast<long long>(blockIdx.x) * groups * kRows + (threadIdx.x >> a.log2_group);
  uint4 raw[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const long long row = base + r * groups;
    raw[r] = make_uint4(0u, 0u, 0u, 0u);
    if (column && row < a.n_rows) raw[r] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ld_x) + t);
  }
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
  float mean[kRows], square[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    mean[r] = 0.f;
    if (kCentered) {
      F2 acc = both(0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) acc = add2(acc, Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw[r]) + i * Pairs<T>::kWords));
      mean[r] = f2_lo(acc) + f2_hi(acc);
    }
  }
  if (kCentered) {
    for (int o = group >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) mean[r] += __shfl_xor_sync(0xffffffffu, mean[r], o);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    mean[r] /= static_cast<float>(a.hidden);
    F2 acc = both(0.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const F2 v = add2(Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw[r]) + i * Pairs<T>::kWords), both(-mean[r]));
      acc = fma2(v, v, acc);
    }
    square[r] = column ? f2_lo(acc) + f2_hi(acc) : 0.f;
  }
  for (int o = group >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) square[r] += __shfl_xor_sync(0xffffffffu, square[r], o);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const long long row = base + r * groups;
    if (row >= a.n_rows) continue;
    const float rstd = 1.f / sqrtf(square[r] / static_cast<float>(a.hidden) + a.eps);
    if (t == 0) {
      if (kCentered && a.mean != nullptr) a.mean[row] = mean[r];
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    uint4 out;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      F2 v = Pairs<T>::get(reinterpret_cast<const uint32_t*>(&raw[r]) + i * Pairs<T>::kWords);
      if (kCentered) v = add2(v, both(-mean[r]));
      v = mul2(v, both(rstd));
      if (rounded) v = f2(norm_round<T>(f2_lo(v)), norm_round<T>(f2_hi(v)));
      Pairs<T>::set(reinterpret_cast<uint32_t*>(&out) + i * Pairs<T>::kWords, kCentered ? fma2(v, gain[i], bias[i]) : mul2(v, gain[i]));
    }
    if (column) reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.hidden)[t] = out;
  }
}

template <typename T, typename W, bool kCentered, int kRows>
__global__ void __launch_bounds__(kNarrowThreads)
norm_backward_narrow_kernel(NormBackwardArgs a) {
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kPairs = kVec / 2;
  constexpr int kWVecs = kVec * static_cast<int>(sizeof(W)) / 16;
  __shared__ float fold[kNarrowThreads / 2 * kVec];
  const int group = 1 << a.log2_group;
  const int groups = kNarrowThreads >> a.log2_group;
  const int t = static_cast<int>(threadIdx.x) & (group - 1);
  const int g = static_cast<int>(threadIdx.x) >> a.log2_group;
  const bool column = t * kVec < a.hidden;
  const bool rounded = !kCentered && a.round_xhat != 0;
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
  for (long long base = static_cast<long long>(blockIdx.x) * groups * kRows; base < a.n_rows; base += step) {
    uint4 raw_x[kRows], raw_dy[kRows];
    float mean[kRows], rstd[kRows], s_mx[kRows], s_m[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {       // rows behind the last one come in as zeros
      const long long row = base + g + r * groups;
      const bool live = row < a.n_rows;
      raw_x[r] = raw_dy[r] = make_uint4(0u, 0u, 0u, 0u);
      if (column && live) {
        raw_x[r] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ld_x) + t);
        raw_dy[r] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + row * a.ld_dy) + t);
      }
      mean[r] = kCentered && live ? __ldg(a.mean + row) : 0.f;
      rstd[r] = live ? __ldg(a.rstd + row) : 0.f;
    }
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
      s_mx[r] = f2_lo(mx) + f2_hi(mx);
      s_m[r] = f2_lo(m) + f2_hi(m);
    }
    for (int o = group >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        s_mx[r] += __shfl_xor_sync(0xffffffffu, s_mx[r], o);
        if (kCentered) s_m[r] += __shfl_xor_sync(0xffffffffu, s_m[r], o);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = base + g + r * groups;
      uint4 out;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        F2 m = mul2(dy_of(r, i), gain[i]);
        if (kCentered) m = add2(m, both(-s_m[r] * inv));
        Pairs<T>::set(reinterpret_cast<uint32_t*>(&out) + i * Pairs<T>::kWords,
                      mul2(fma2(xhat_of(r, i), both(-s_mx[r] * inv), m), both(rstd[r])));
      }
      if (column && row < a.n_rows) reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + row * a.hidden)[t] = out;
    }
  }
  // the groups of the block, folded in halves in a fixed order
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

// gradient[c] = sum over the blocks' partials; 32 columns per block, each summed by 32 threads in a fixed order.
// blockIdx.y 0: the weight's, 1: the bias's.
constexpr int kNormReduceLanes = 32;
template <typename W>
__global__ void __launch_bounds__(32 * kNormReduceLanes)
norm_parameter_gradient_kernel(const float* dw_partial, const float* db_partial, int blocks, int hidden, W* dw, W* db) {
  __shared__ float part[kNormReduceLanes][33];
  const float* partial = blockIdx.y == 0 ? dw_partial : db_partial;
  W* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  const int col = static_cast<int>(blockIdx.x) * 32 + static_cast<int>(threadIdx.x);
  float s = 0.f;
  if (col < hidden) {
#pragma unroll 4
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

template <int kN>
__device__ __forceinline__ void norm_block_sum(float (&v)[kN], float (*scratch)[kNormMaxWarps * kN], int& phase) {
  norm_group_sum<kN>(v, 9, scratch, phase);
}

template <typename T, typename W, bool kCentered>
__global__ void __launch_bounds__(kNormMaxThreads)
norm_forward_long_kernel(NormForwardArgs a) {
  __shared__ float scratch[2][kNormMaxWarps];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const W* w = static_cast<const W*>(a.w);
  const W* b = static_cast<const W*>(a.b);
  const int tid = static_cast<int>(threadIdx.x);
  int phase = 0;
  float mean = 0.f;
  float s[1] = {0.f};
  if constexpr (kCentered) {
    for (int c = tid; c < a.hidden; c += kNormMaxThreads) s[0] += CeElem<T>::load(x + c);
    norm_block_sum<1>(s, scratch, phase);
    mean = s[0] / static_cast<float>(a.hidden);
    s[0] = 0.f;
  }
  for (int c = tid; c < a.hidden; c += kNormMaxThreads) {
    const float v = CeElem<T>::load(x + c) - mean;
    s[0] = fmaf(v, v, s[0]);
  }
  norm_block_sum<1>(s, scratch, phase);
  const float rstd = 1.f / sqrtf(s[0] / static_cast<float>(a.hidden) + a.eps);
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
  __shared__ float scratch[2][kNormMaxWarps * 2];
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
  norm_block_sum<2>(s, scratch, phase);
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
__global__ void __launch_bounds__(kNormForwardThreads)
norm_parameter_partial_long_kernel(NormBackwardArgs a) {
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
