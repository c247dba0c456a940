// Load-balancing loss of a mixture-of-experts router over the logits of all layers, the number of tokens each expert was
// chosen by, and the gradient of the logits.
//
//   C[l][e]  tokens of layer l that have expert e among their top_k logits (equal logits: the lowest index first)
//   p        softmax of a token's logits,   S_e = sum over kept tokens of all layers of p_e,   N = kept tokens of all layers
//   loss   = E / N^2 * sum_e (sum_l C[l][e]) * S_e  +  lambda / N * sum lse^2
//   d loss / d x_j = p_j * (a_j - sum_e a_e p_e) + 2 lambda / N * lse * p_j,      a_e = E / N^2 * (sum_l C[l][e] - mean)
//
// (The mean is taken out of a: that changes nothing, as p sums to one, and in a balanced router it is nearly all of a, so the
// difference would be left with few digits.)  Tokens that the mask leaves out are not read: whatever they hold, they add
// nothing and their gradient is zero.
//
// Forward reads the logits once, backward reads them once and writes as much; nothing per token is kept in between.  A row is
// shared by a group of 1..32 lanes, each holding kEpt consecutive logits in registers, so the sums over a row are shuffles and
// several rows share a warp.  A lane keeps its columns for all rows of its block: S and C are sums in registers, left as one
// partial per block and added up in block order, in fp64 from there on: no atomics, the same bits in every run.
//
// The chosen set follows from one number per row, the top_k-th largest logit counted with multiplicity: each lane sorts its
// logits once, then the group repeatedly takes the largest of the lanes' heads.  Where more logits equal that number than places
// are left, the places go by index.
#pragma once

#include <type_traits>

#include "ce_kernels.cuh"
#include "simt_common.cuh"

namespace flce {

constexpr int kBalThreads = 256;
constexpr int kBalWarps = kBalThreads / 32;
constexpr int kBalMaxEpt = 32;               // 32 lanes x 32: up to 1024 experts
constexpr int kBalMaxLayers = 256;           // per launch: their pointers travel as kernel arguments

struct BalanceArgs {
  const void* logits[kBalMaxLayers];
  long long ld;
  long long n_tokens;
  int experts, top_k;
  const void* mask;             // nullptr: every token is kept; else n_tokens integers of mask_bytes, 0 = left out
  int mask_bytes;
  int log2_group;
  int want_lse;
};

__device__ __forceinline__ bool balance_kept(const BalanceArgs& a, long long token) {
  if (token >= a.n_tokens) return false;
  if (a.mask == nullptr) return true;
  if (a.mask_bytes == 1) return static_cast<const unsigned char*>(a.mask)[token] != 0;
  if (a.mask_bytes == 4) return static_cast<const unsigned*>(a.mask)[token] != 0;
  return static_cast<const unsigned long long*>(a.mask)[token] != 0;
}

// kEpt consecutive logits of a row from column `first`; pad behind the row's end and in rows that are not read
template <typename T, bool kVectors, int kEpt>
__device__ __forceinline__ void balance_load(const T* row, int first, int experts, bool read, float (&v)[kEpt], float pad) {
  if constexpr (kVectors) {
    constexpr int kVec = CeElem<T>::kVec;
#pragma unroll
    for (int u = 0; u < kEpt / kVec; ++u) {
      float part[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) part[i] = pad;
      if (read && first + u * kVec < experts) ce_load_vec<T>(row + first + u * kVec, part);
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[u * kVec + i] = part[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      v[e] = pad;
      if (read && first + e < experts) v[e] = CeElem<T>::load(row + first + e);
    }
  }
}

__device__ __forceinline__ float balance_group_max(float v, int log2_group) {
  for (int o = 1 << log2_group >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float balance_group_sum(float v, int log2_group) {
  for (int o = 1 << log2_group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// descending; Batcher's odd-even merge sort, its comparators are known at compile time
template <int kN>
__device__ __forceinline__ void balance_sort(float (&v)[kN]) {
#pragma unroll
  for (int p = 1; p < kN; p <<= 1) {
#pragma unroll
    for (int k = p; k >= 1; k >>= 1) {
#pragma unroll
      for (int j = k % p; j + k < kN; j += 2 * k) {
#pragma unroll
        for (int i = 0; i < k; ++i) {
          if (i + j + k < kN && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const float hi = fmaxf(v[i + j], v[i + j + k]), lo = fminf(v[i + j], v[i + j + k]);
            v[i + j] = hi;
            v[i + j + k] = lo;
          }
        }
      }
    }
  }
}

// bit e of the result: logit e of this lane is among the row's top_k.  All lanes of the warp call it.
template <int kEpt>
__device__ __forceinline__ unsigned balance_chosen(const float (&v)[kEpt], int top_k, int log2_group, int lane) {
  float head[kEpt];
#pragma unroll
  for (int e = 0; e < kEpt; ++e) head[e] = v[e];
  balance_sort<kEpt>(head);
  const unsigned group_mask = (log2_group == 5 ? 0xffffffffu : (1u << (1 << log2_group)) - 1u) << (lane >> log2_group << log2_group);
  int taken = 0, above = 0;           // logits taken so far; those larger than the last one taken
  float last = INFINITY;
  for (int round = 0; round < top_k; ++round) {
    const bool open = taken < top_k;
    if (!__any_sync(0xffffffffu, open)) break;
    const float m = balance_group_max(head[0], log2_group);
    const bool mine = head[0] == m;
    const int n = __popc(__ballot_sync(0xffffffffu, mine) & group_mask);
    if (open) {
      if (m != last) above = taken;
      last = m;
      taken += n;
    }
    if (mine) {
#pragma unroll
      for (int e = 0; e + 1 < kEpt; ++e) head[e] = head[e + 1];
      head[kEpt - 1] = -INFINITY;
    }
  }
  unsigned greater = 0, equal = 0;
#pragma unroll
  for (int e = 0; e < kEpt; ++e) {
    greater |= v[e] > last ? 1u << e : 0u;
    equal |= v[e] == last ? 1u << e : 0u;
  }
  // places left for the logits that equal the last one, by index: first those of the lanes before this one
  const int places = top_k - above;
  const int have = __popc(equal);
  int upto = have;
  for (int o = 1; o < (1 << log2_group); o <<= 1) {
    const int before = __shfl_up_sync(0xffffffffu, upto, o);
    if ((lane & ((1 << log2_group) - 1)) >= o) upto += before;
  }
  int left = places - (upto - have);
  if (left < have) {
    for (int drop = have - (left > 0 ? left : 0); drop > 0; --drop) equal &= ~(0x80000000u >> __clz(equal));
  }
  return greater | equal;
}

// partial[layer][block]: S_e [experts], the sum of lse^2, then (as int) C_e [experts] and the number of kept tokens
__host__ __device__ inline long long balance_partial_words(int experts) { return 2ll * experts + 2; }

template <typename T, bool kVectors, int kEpt>
__global__ void __launch_bounds__(kBalThreads)
balance_forward_kernel(BalanceArgs a, float* partial) {
  __shared__ float fold_s[kBalWarps][32 * kEpt];      // taken twice: for S, then for C
  __shared__ float fold_z[kBalWarps];
  __shared__ int fold_n[kBalWarps];
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int group = 1 << a.log2_group;
  const int first = (lane & (group - 1)) * kEpt;
  const int rows = kBalThreads >> a.log2_group;
  const T* logits = static_cast<const T*>(a.logits[blockIdx.y]);
  float s[kEpt], z = 0.f;
  int c[kEpt], n = 0;
#pragma unroll
  for (int e = 0; e < kEpt; ++e) {
    s[e] = 0.f;
    c[e] = 0;
  }
  float next[kEpt];
  long long token = static_cast<long long>(blockIdx.x) * rows;
  const int mine = static_cast<int>(threadIdx.x) >> a.log2_group;
  bool next_kept = balance_kept(a, token + mine);
  balance_load<T, kVectors, kEpt>(logits + (token + mine) * a.ld, first, a.experts, next_kept, next, -INFINITY);
  for (; token < a.n_tokens; token += static_cast<long long>(gridDim.x) * rows) {
    float v[kEpt];
    const bool kept = next_kept;
#pragma unroll
    for (int e = 0; e < kEpt; ++e) v[e] = next[e];
    const long long ahead = token + static_cast<long long>(gridDim.x) * rows + mine;
    next_kept = balance_kept(a, ahead);
    balance_load<T, kVectors, kEpt>(logits + ahead * a.ld, first, a.experts, next_kept, next, -INFINITY);
    if (!__any_sync(0xffffffffu, kept)) continue;
    float top = v[0];
#pragma unroll
    for (int e = 1; e < kEpt; ++e) top = fmaxf(top, v[e]);
    top = balance_group_max(top, a.log2_group);
    float p[kEpt], total = 0.f;
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      p[e] = ex2_approx((v[e] - top) * kLog2e);
      total += p[e];
    }
    total = balance_group_sum(total, a.log2_group);
    const unsigned chosen = balance_chosen<kEpt>(v, a.top_k, a.log2_group, lane);
    if (kept) {
      const float inv = 1.f / total;
#pragma unroll
      for (int e = 0; e < kEpt; ++e) {
        s[e] = fmaf(p[e], inv, s[e]);
        c[e] += (chosen >> e) & 1u;
      }
      if (first == 0) {
        ++n;
        if (a.want_lse) {
          const float lse = top + ln_approx(total);
          z = fmaf(lse, lse, z);
        }
      }
    }
  }
  // the warp's groups, then the block's warps, in a fixed order
  for (int o = 16; o >= group; o >>= 1) {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      s[e] += __shfl_xor_sync(0xffffffffu, s[e], o);
      c[e] += __shfl_xor_sync(0xffffffffu, c[e], o);
    }
    z += __shfl_xor_sync(0xffffffffu, z, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  int(*fold_c)[32 * kEpt] = reinterpret_cast<int(*)[32 * kEpt]>(fold_s);
  float* out = partial + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * balance_partial_words(a.experts);
  if (lane < group) {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) fold_s[warp][first + e] = s[e];
  }
  if (lane == 0) {
    fold_z[warp] = z;
    fold_n[warp] = n;
  }
  __syncthreads();
  for (int e = static_cast<int>(threadIdx.x); e < a.experts; e += kBalThreads) {
    float ss = 0.f;
    for (int w = 0; w < kBalWarps; ++w) ss += fold_s[w][e];
    out[e] = ss;
  }
  __syncthreads();
  if (lane < group) {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) fold_c[warp][first + e] = c[e];
  }
  __syncthreads();
  for (int e = static_cast<int>(threadIdx.x); e < a.experts; e += kBalThreads) {
    int cc = 0;
    for (int w = 0; w < kBalWarps; ++w) cc += fold_c[w][e];
    reinterpret_cast<int*>(out)[a.experts + 1 + e] = cc;
  }
  if (threadIdx.x == 0) {
    float zz = 0.f;
    int nn = 0;
    for (int w = 0; w < kBalWarps; ++w) {
      zz += fold_z[w];
      nn += fold_n[w];
    }
    out[a.experts] = zz;
    reinterpret_cast<int*>(out)[2 * a.experts + 1] = nn;
  }
}

// one block per layer: counts[layer][:], sums[layer][:] = S_e and the sum of lse^2 of that layer, kept[layer]
__global__ void __launch_bounds__(kBalThreads)
balance_layer_kernel(const float* partial, int blocks, int experts, long long* counts, double* sums, long long* kept) {
  const float* mine = partial + static_cast<long long>(blockIdx.x) * blocks * balance_partial_words(experts);
  for (int e = static_cast<int>(threadIdx.x); e < experts + 1; e += kBalThreads) {
    double s = 0.0;
    long long c = 0;
#pragma unroll 4
    for (int b = 0; b < blocks; ++b) {
      const float* row = mine + b * balance_partial_words(experts);
      s += row[e];
      c += reinterpret_cast<const int*>(row)[experts + 1 + e];
    }
    sums[static_cast<long long>(blockIdx.x) * (experts + 1) + e] = s;
    if (e < experts) counts[static_cast<long long>(blockIdx.x) * experts + e] = c;
    else kept[blockIdx.x] = c;
  }
}

// out[0] = loss, out[1] = its lse^2 term; coef[e] = a_e, coef[experts] = 2 lambda / N.  No kept token: all zero.
__global__ void __launch_bounds__(kBalThreads)
balance_total_kernel(const long long* counts, const double* sums, const long long* kept, int layers, int experts, float lambda,
                     float* out, float* coef) {
  __shared__ double scratch[kBalWarps];
  __shared__ double result;
  const int tid = static_cast<int>(threadIdx.x);
  auto block_sum = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((tid & 31) == 0) scratch[tid >> 5] = v;
    __syncthreads();
    if (tid == 0) {
      result = 0.0;
      for (int w = 0; w < kBalWarps; ++w) result += scratch[w];
    }
    __syncthreads();
    return result;
  };
  constexpr int kMine = 1024 / kBalThreads;
  double c[kMine], dot = 0.0, all = 0.0, tokens = 0.0, z = 0.0;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int e = tid + i * kBalThreads;
    c[i] = 0.0;
    if (e < experts) {
      double s = 0.0;
      for (int l = 0; l < layers; ++l) {
        c[i] += static_cast<double>(counts[static_cast<long long>(l) * experts + e]);
        s += sums[static_cast<long long>(l) * (experts + 1) + e];
      }
      dot += c[i] * s;
      all += c[i];
    }
  }
  for (int l = tid; l < layers; l += kBalThreads) {
    tokens += static_cast<double>(kept[l]);
    z += sums[static_cast<long long>(l) * (experts + 1) + experts];
  }
  dot = block_sum(dot);
  all = block_sum(all);
  tokens = block_sum(tokens);
  z = block_sum(z);
  const double inv = tokens > 0.0 ? 1.0 / tokens : 0.0;
  const double scale = experts * inv * inv;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int e = tid + i * kBalThreads;
    if (e < experts) coef[e] = static_cast<float>(scale * (c[i] - all / experts));
  }
  if (tid == 0) {
    out[0] = static_cast<float>(scale * dot + lambda * inv * z);
    out[1] = static_cast<float>(lambda * inv * z);
    coef[experts] = static_cast<float>(2.0 * lambda * inv);
  }
}

// grads[layer][token][:] (dense) = *grad_loss * d loss / d logits
template <typename T, bool kVectors, int kEpt>
__global__ void __launch_bounds__(kBalThreads)
balance_backward_kernel(BalanceArgs a, const float* coef, const float* grad_loss, T* grads) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const int group = 1 << a.log2_group;
  const int first = (lane & (group - 1)) * kEpt;
  const int rows = kBalThreads >> a.log2_group;
  const int mine = static_cast<int>(threadIdx.x) >> a.log2_group;
  const T* logits = static_cast<const T*>(a.logits[blockIdx.y]);
  T* out = grads + static_cast<long long>(blockIdx.y) * a.n_tokens * a.experts;
  const float up = *grad_loss;
  const float lse_coef = coef[a.experts] * up;
  float w[kEpt];
#pragma unroll
  for (int e = 0; e < kEpt; ++e) w[e] = first + e < a.experts ? coef[first + e] * up : 0.f;
  float next[kEpt];
  long long token = static_cast<long long>(blockIdx.x) * rows;
  bool next_kept = balance_kept(a, token + mine);
  balance_load<T, kVectors, kEpt>(logits + (token + mine) * a.ld, first, a.experts, next_kept, next, -INFINITY);
  for (; token < a.n_tokens; token += static_cast<long long>(gridDim.x) * rows) {
    float v[kEpt];
    const bool kept = next_kept;
#pragma unroll
    for (int e = 0; e < kEpt; ++e) v[e] = next[e];
    const long long ahead = token + static_cast<long long>(gridDim.x) * rows + mine;
    next_kept = balance_kept(a, ahead);
    balance_load<T, kVectors, kEpt>(logits + ahead * a.ld, first, a.experts, next_kept, next, -INFINITY);
    float top = v[0];
#pragma unroll
    for (int e = 1; e < kEpt; ++e) top = fmaxf(top, v[e]);
    top = balance_group_max(top, a.log2_group);
    float total = 0.f, dot = 0.f;
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      v[e] = ex2_approx((v[e] - top) * kLog2e);
      total += v[e];
      dot = fmaf(v[e], w[e], dot);
    }
    total = balance_group_sum(total, a.log2_group);
    dot = balance_group_sum(dot, a.log2_group);
    const float inv = 1.f / total;
    const float shift = fmaf(-dot, inv, lse_coef != 0.f ? lse_coef * (top + ln_approx(total)) : 0.f);
#pragma unroll
    for (int e = 0; e < kEpt; ++e) v[e] = kept ? v[e] * inv * (w[e] + shift) : 0.f;
    if (token + mine < a.n_tokens) {
      T* row = out + (token + mine) * a.experts;
      if constexpr (kVectors) {
        constexpr int kVec = CeElem<T>::kVec;
#pragma unroll
        for (int u = 0; u < kEpt / kVec; ++u) {
          if (first + u * kVec < a.experts) {
            float part[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) part[i] = v[u * kVec + i];
            ce_store_vec<T>(row + first + u * kVec, part);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < kEpt; ++e) {
          if (first + e < a.experts) CeElem<T>::store(row + first + e, v[e]);
        }
      }
    }
  }
}

}  // namespace flce
