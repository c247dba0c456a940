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
