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
// The largest logit is subtracted before the scaling to base 2, in every kernel: -top * log2(e) folded into one fma leaves the rounding of
// that product in all exponents of the row, |top| 2^-24, which overflows exp2 from |top| of about 1.5e9 on; a row that a mask filled with
// the type's lowest value is such a row.
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
#include "packed_math.cuh"
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
  allow_dependents();      // the small kernels that add up the partial sums
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

// ---- 32 to 256 experts in whole vectors, at most 16 of them chosen
//
// In the kernel above the choice takes most of the time: every round of it is a maximum over lanes that wait for each other
// (48 x 16384 x 128 bf16, top 8, half of the tokens padding: 351 us against about 15 us of memory traffic).  Here a warp fetches 32 rows into shared memory,
// a tile ahead, and each lane finds the 8 (or 16) largest logits of a row of its own, in registers: it sorts 8 words at a time
// with a network and merges them into a sorted list.  16-bit logits go through the network two to a word, the even and the odd columns
// as two lists, which meet at the end.  Only the top_k-th largest logit and the largest are handed on; with them the warp
// goes over the tile once more, rows shared by groups of lanes with 8 columns each, for the softmax and the sums per expert.
// Where shared memory holds two tiles for each of 16 warps, the next one is fetched while this one is worked on; else one, and
// the other warps cover the wait: more warps count for more than the second tile.
constexpr int kTileListMost = 16;

template <typename T>
struct TileWord;
template <>
struct TileWord<float> {
  typedef float Word;
  static constexpr int kPerVector = 4;
  __device__ static Word lowest() { return -INFINITY; }
  __device__ static Word larger(Word a, Word b) { return fmaxf(a, b); }
  __device__ static Word smaller(Word a, Word b) { return fminf(a, b); }
};
template <>
struct TileWord<__nv_bfloat16> {
  typedef __nv_bfloat162 Word;
  static constexpr int kPerVector = 4;
  __device__ static Word lowest() { return __nv_bfloat162(__float2bfloat16_rn(-INFINITY), __float2bfloat16_rn(-INFINITY)); }
  __device__ static Word larger(Word a, Word b) { return __hmax2(a, b); }
  __device__ static Word smaller(Word a, Word b) { return __hmin2(a, b); }
};
template <>
struct TileWord<__half> {
  typedef __half2 Word;
  static constexpr int kPerVector = 4;
  __device__ static Word lowest() { return __half2(__float2half_rn(-INFINITY), __float2half_rn(-INFINITY)); }
  __device__ static Word larger(Word a, Word b) { return __hmax2(a, b); }
  __device__ static Word smaller(Word a, Word b) { return __hmin2(a, b); }
};

template <typename T>
__device__ __forceinline__ void tile_order(typename TileWord<T>::Word& a, typename TileWord<T>::Word& b) {      // a >= b
  const auto hi = TileWord<T>::larger(a, b), lo = TileWord<T>::smaller(a, b);
  a = hi;
  b = lo;
}
// descending: Batcher's odd-even merge sort of 8, and the last merge of a bitonic one
template <typename T>
__device__ __forceinline__ void tile_sort(typename TileWord<T>::Word (&v)[8]) {
#pragma unroll
  for (int p = 1; p < 8; p <<= 1) {
#pragma unroll
    for (int k = p; k >= 1; k >>= 1) {
#pragma unroll
      for (int j = k % p; j + k < 8; j += 2 * k) {
#pragma unroll
        for (int i = 0; i < k; ++i) {
          if (i + j + k < 8 && (i + j) / (2 * p) == (i + j + k) / (2 * p)) tile_order<T>(v[i + j], v[i + j + k]);
        }
      }
    }
  }
}
template <typename T, int kN>
__device__ __forceinline__ void tile_merge(typename TileWord<T>::Word (&v)[kN]) {
#pragma unroll
  for (int k = kN / 2; k >= 1; k >>= 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if ((i & k) == 0) tile_order<T>(v[i], v[i + k]);
    }
  }
}

// bytes from one row of a tile to the next: an odd number of vectors, so that 8 lanes reading a vector of 8 rows meet all banks
__host__ __device__ inline int tile_pitch(int row_bytes) { return (row_bytes / 16 | 1) * 16; }
__host__ __device__ inline int tile_warp_bytes(int row_bytes, int buffers) { return buffers * 32 * tile_pitch(row_bytes) + 32 * 8; }
constexpr int kTileMaxWarps = 16;

template <typename T, int kList>
__global__ void __launch_bounds__(kTileMaxWarps * 32, 1)
balance_forward_tile_kernel(BalanceArgs a, int buffers, float* partial) {
  allow_dependents();      // the small kernels that add up the partial sums
  typedef TileWord<T> Tile;
  typedef typename Tile::Word Word;
  constexpr int kVec = CeElem<T>::kVec;
  constexpr int kVectors = 8 / kVec;                          // of the 8 columns of a lane
  FLCE_DYNAMIC_SHARED(uint4, tile_shared);                    // per warp: one or two tiles, and (top_k-th logit, largest) of 32 rows
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int warps = static_cast<int>(blockDim.x) >> 5;
  const int vectors = a.experts / kVec;                       // of a row
  const int pitch = tile_pitch(vectors * 16) / 16;
  uint4* tiles = tile_shared + warp * (tile_warp_bytes(vectors * 16, buffers) / 16);
  float2* chosen_of = reinterpret_cast<float2*>(tiles + buffers * 32 * pitch);
  const T* logits = static_cast<const T*>(a.logits[blockIdx.y]);

  const int group = 1 << a.log2_group, groups = 32 >> a.log2_group;
  const int quarter = group >> 2;
  const int t = lane & (group - 1), q = lane >> a.log2_group;
  const bool column = t * 8 < a.experts;
  F2 s[4], c[4];            // c counts in floats, exactly: a lane sees at most 2^24 rows
  int n = 0;
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = c[i] = both(0.f);

  // rows of a fetch side by side in the warp, for row lengths up to 32 vectors; longer rows go one at a time
  const int side = vectors < 32 ? 32 / vectors : 1;
  const int my_row = lane / vectors < side ? lane / vectors : 32, my_vector = vectors < 32 ? lane % vectors : lane;
  auto fetch = [&](long long tile, unsigned kept, uint4* to) {
    for (int r = vectors < 32 ? my_row : 0; r < 32; r += side) {
      if ((kept >> r & 1u) == 0) continue;
      const uint4* from = reinterpret_cast<const uint4*>(logits + (tile * 32 + r) * a.ld);
      for (int v = my_vector; v < vectors; v += 32) async_copy16(to + r * pitch + v, from + v, 16);
    }
    async_commit();
  };
  const long long step = static_cast<long long>(gridDim.x) * warps;
  long long tile = static_cast<long long>(blockIdx.x) * warps + warp;
  unsigned kept = __ballot_sync(0xffffffffu, balance_kept(a, tile * 32 + lane));
  bool after = balance_kept(a, (tile + step) * 32 + lane);
  fetch(tile, kept, tiles);
  int which = 0;
  for (; tile * 32 < a.n_tokens; tile += step) {
    const unsigned next_kept = __ballot_sync(0xffffffffu, after);
    after = balance_kept(a, (tile + 2 * step) * 32 + lane);
    if (buffers == 2) {
      fetch(tile + step, next_kept, tiles + (which ^ 1) * 32 * pitch);
      async_wait<1>();
    } else {
      async_wait<0>();
    }
    warp_sync();
    const uint4* here = tiles + which * 32 * pitch;
    if (kept != 0) {
      // a row per lane: its kList largest words
      {
        const uint4* row = here + lane * pitch;
        Word list[kList];
#pragma unroll
        for (int i = 0; i < kList; ++i) list[i] = Tile::lowest();
        for (int v = 0; v < vectors; v += 2) {
          Word w[8];
          const uint4 r0 = row[v];
          memcpy(w, &r0, 16);
          if (v + 1 < vectors) {
            const uint4 r1 = row[v + 1];
            memcpy(w + 4, &r1, 16);
          } else {
#pragma unroll
            for (int i = 4; i < 8; ++i) w[i] = Tile::lowest();
          }
          tile_sort<T>(w);
#pragma unroll
          for (int i = 0; i < 8; ++i) list[kList - 8 + i] = Tile::larger(list[kList - 8 + i], w[7 - i]);
          tile_merge<T, kList>(list);
        }
        float best[kList];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < kList; ++i) best[i] = list[i];
        } else {
          // the lists of the even and of the odd columns become one
          const T* e = reinterpret_cast<const T*>(list);
#pragma unroll
          for (int i = 0; i < kList; ++i) best[i] = fmaxf(CeElem<T>::load(e + 2 * i), CeElem<T>::load(e + 2 * (kList - 1 - i) + 1));
          tile_merge<float, kList>(best);
        }
        float kth = best[0];
#pragma unroll
        for (int i = 1; i < kList; ++i) kth = i < a.top_k ? best[i] : kth;
        chosen_of[lane] = make_float2(kth, best[0]);
      }
      warp_sync();
      // rows by groups of lanes, four per group at a time
      for (int r0 = q; r0 < 32; r0 += 4 * groups) {
        F2 x[4][4];
        float kth[4], total[4], taken[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = r0 + r * groups;
          uint4 raw[kVectors];
#pragma unroll
          for (int i = 0; i < kVectors; ++i) {
            raw[i] = make_uint4(~0u, ~0u, ~0u, ~0u);          // NaN behind the row's end: it compares with nothing
            if (column) raw[i] = here[row * pitch + t * kVectors + i];
          }
          const float2 of = chosen_of[row];
          const F2 counted = both((kept >> row & 1u) != 0 ? 1.f : 0.f);
          const F2 minus_top = both(-of.y);
          F2 sum = both(0.f), many = both(0.f);
          kth[r] = of.x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const F2 v = Pairs<T>::get(reinterpret_cast<const uint32_t*>(raw) + i * Pairs<T>::kWords);
            const F2 in = f2(f2_lo(v) >= of.x ? 1.f : 0.f, f2_hi(v) >= of.x ? 1.f : 0.f);
            many = add2(many, in);
            c[i] = fma2(in, counted, c[i]);
            const F2 d = mul2(add2(v, minus_top), both(kLog2e));
            x[r][i] = f2(ex2_approx(f2_lo(d)), ex2_approx(f2_hi(d)));
            sum = add2(sum, x[r][i]);
          }
          total[r] = column ? f2_lo(sum) + f2_hi(sum) : 0.f;
          taken[r] = f2_lo(many) + f2_hi(many);
        }
        const float sums = lane_four_sums(total, group);
        const float extra = lane_four_sums(taken, group) - static_cast<float>(a.top_k);
        float inv = 1.f / sums;
        const int row_of_sum = r0 + t / quarter * groups;     // the row that this lane's sums belong to
        const bool kept_of_sum = (kept >> row_of_sum & 1u) != 0;
        if (!kept_of_sum) inv = 0.f;
        if ((t & (quarter - 1)) == 0 && kept_of_sum) {
          ++n;
          if (a.want_lse) {
            const float lse = chosen_of[row_of_sum].y + ln_approx(sums);
            z = fmaf(lse, lse, z);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const F2 scale = both(of_four(inv, r, a.log2_group));
          if (kept >> (r0 + r * groups) & 1u) {               // a row that was left out may hold anything
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = fma2(x[r][i], scale, s[i]);
          }
        }
        // more logits equal the last one chosen than there are places: those of the highest columns give way
        if (__any_sync(0xffffffffu, extra > 0.f && kept_of_sum)) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            int drop = static_cast<int>(of_four(kept_of_sum ? extra : 0.f, r, a.log2_group));
            if (!__any_sync(0xffffffffu, drop > 0)) continue;
            const T* row_here = reinterpret_cast<const T*>(here + (r0 + r * groups) * pitch) + (column ? t * 8 : 0);
            unsigned equal = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) equal |= CeElem<T>::load(row_here + e) == kth[r] ? 1u << e : 0u;
            if (!column) equal = 0;
            do {
              const unsigned have = __ballot_sync(0xffffffffu, equal != 0) >> (q << a.log2_group) & (group == 32 ? 0xffffffffu : (1u << group) - 1u);
              if (drop > 0 && t == 31 - __clz(have)) {
                const int last = 31 - __clz(equal);
                equal &= ~(1u << last);
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = add2(c[i], f2(last == 2 * i ? -1.f : 0.f, last == 2 * i + 1 ? -1.f : 0.f));
              }
              --drop;
            } while (__any_sync(0xffffffffu, drop > 0));
          }
        }
      }
    }
    warp_sync();        // the tile's last readers, before a fetch overwrites it
    if (buffers == 2) which ^= 1;
    else fetch(tile + step, next_kept, tiles);
    kept = next_kept;
  }
  async_wait<0>();
  // the warp's groups, then the block's warps, in a fixed order
  __syncthreads();
  float* fold = reinterpret_cast<float*>(tile_shared);        // [warp][2 * 256 + 2]
  for (int o = group; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = add2(s[i], f2(__shfl_xor_sync(0xffffffffu, f2_lo(s[i]), o), __shfl_xor_sync(0xffffffffu, f2_hi(s[i]), o)));
      c[i] = add2(c[i], f2(__shfl_xor_sync(0xffffffffu, f2_lo(c[i]), o), __shfl_xor_sync(0xffffffffu, f2_hi(c[i]), o)));
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  float* mine = fold + warp * (2 * 256 + 2);
  if (q == 0 && column) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mine[t * 8 + e] = e % 2 ? f2_hi(s[e / 2]) : f2_lo(s[e / 2]);
      mine[256 + t * 8 + e] = __uint_as_float(static_cast<unsigned>(e % 2 ? f2_hi(c[e / 2]) : f2_lo(c[e / 2])));
    }
  }
  if (lane == 0) {
    mine[512] = z;
    mine[513] = __uint_as_float(static_cast<unsigned>(n));
  }
  __syncthreads();
  float* out = partial + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * balance_partial_words(a.experts);
  for (int e = static_cast<int>(threadIdx.x); e <= a.experts; e += static_cast<int>(blockDim.x)) {
    const int from = e < a.experts ? e : 512, from_c = e < a.experts ? 256 + e : 513;
    float ss = 0.f;
    unsigned cc = 0;
    for (int w = 0; w < warps; ++w) {
      ss += fold[w * (2 * 256 + 2) + from];
      cc += __float_as_uint(fold[w * (2 * 256 + 2) + from_c]);
    }
    out[e] = ss;
    out[a.experts + 1 + e] = __uint_as_float(cc);
  }
}

// counts[layer][:], sums[layer][:] = S_e and the sum of lse^2 of that layer, kept[layer]: one block per layer (blockIdx.y) and 32
// columns, each added up by 32 threads in a fixed order
constexpr int kBalFoldLanes = 32;
__global__ void __launch_bounds__(32 * kBalFoldLanes)
balance_layer_kernel(const float* partial, int blocks, int experts, long long* counts, double* sums, long long* kept) {
  __shared__ double part_s[kBalFoldLanes][32];
  __shared__ long long part_c[kBalFoldLanes][32];
  allow_dependents();
  wait_for_previous_kernel();
  const long long layer = blockIdx.y;
  const int e = static_cast<int>(blockIdx.x * 32 + threadIdx.x);
  double s = 0.0;
  long long c = 0;
  if (e <= experts) {
    const float* mine = partial + layer * blocks * balance_partial_words(experts) + e;
#pragma unroll 4
    for (int b = static_cast<int>(threadIdx.y); b < blocks; b += kBalFoldLanes) {
      const float* row = mine + b * balance_partial_words(experts);
      s += row[0];
      c += reinterpret_cast<const int*>(row)[experts + 1];
    }
  }
  part_s[threadIdx.y][threadIdx.x] = s;
  part_c[threadIdx.y][threadIdx.x] = c;
  __syncthreads();
  if (threadIdx.y != 0 || e > experts) return;
  for (int k = 1; k < kBalFoldLanes; ++k) {
    s += part_s[k][threadIdx.x];
    c += part_c[k][threadIdx.x];
  }
  sums[layer * (experts + 1) + e] = s;
  if (e < experts) counts[layer * experts + e] = c;
  else kept[layer] = c;
}

// out[0] = loss, out[1] = its lse^2 term; coef[e] = a_e, coef[experts] = 2 lambda / N.  No kept token: all zero.  One block: a
// thread per expert and share of the layers.  With few partials (partial != nullptr) it adds them up itself, in the place of
// balance_layer_kernel, and leaves the counts; 256 threads then do for up to 256 experts, and are launched sooner.
constexpr int kBalTotalThreads = 1024;      // at most
__global__ void __launch_bounds__(kBalTotalThreads)
balance_total_kernel(const float* partial, int blocks, long long* counts, const double* sums, const long long* kept, int layers, int experts,
                     float lambda, float* out, float* coef) {
  __shared__ double scratch[4][kBalTotalThreads / 32];
  __shared__ double part_c[kBalTotalThreads], part_s[kBalTotalThreads];
  wait_for_previous_kernel();
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
  const long long words = balance_partial_words(experts);
  int wide = 32;
  while (wide < experts) wide *= 2;
  const int e = tid & (wide - 1), shares = threads / wide;
  double c = 0.0, s = 0.0, v[4] = {0.0, 0.0, 0.0, 0.0};      // v: sum C S, sum C, N, sum lse^2
  if (e < experts) {
#pragma unroll 4
    for (int l = tid / wide; l < layers; l += shares) {
      if (partial != nullptr) {
        long long here = 0;
        for (int b = 0; b < blocks; ++b) {
          const float* row = partial + (static_cast<long long>(l) * blocks + b) * words + e;
          s += row[0];
          here += reinterpret_cast<const int*>(row)[experts + 1];
        }
        counts[static_cast<long long>(l) * experts + e] = here;
        c += static_cast<double>(here);
      } else {
        c += static_cast<double>(counts[static_cast<long long>(l) * experts + e]);
        s += sums[static_cast<long long>(l) * (experts + 1) + e];
      }
    }
  }
  if (partial != nullptr) {
    for (int r = tid; r < layers * blocks; r += threads) {
      const float* row = partial + r * words + experts;
      v[3] += row[0];
      v[2] += reinterpret_cast<const int*>(row)[experts + 1];
    }
  } else {
    for (int l = tid; l < layers; l += threads) {
      v[2] += static_cast<double>(kept[l]);
      v[3] += sums[static_cast<long long>(l) * (experts + 1) + experts];
    }
  }
  part_c[tid] = c;
  part_s[tid] = s;
  __syncthreads();
  if (tid < wide) {
    for (int k = 1; k < shares; ++k) {
      c += part_c[k * wide + tid];
      s += part_s[k * wide + tid];
    }
    v[0] = c * s;
    v[1] = c;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if ((tid & 31) == 0) scratch[i][tid >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (tid & 31) < threads >> 5 ? scratch[i][tid & 31] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  const double inv = v[2] > 0.0 ? 1.0 / v[2] : 0.0;
  const double scale = experts * inv * inv;
  if (tid < experts) coef[tid] = static_cast<float>(scale * (c - v[1] / experts));
  if (tid == 0) {
    out[0] = static_cast<float>(scale * v[0] + lambda * inv * v[3]);
    out[1] = static_cast<float>(lambda * inv * v[3]);
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

// The same for groups of 4 lanes and more with 8 logits each, four rows per group at a time: their loads are under way together,
// their sums share the exchanges.  48 x 16384 x 128 bf16: 136 us with a row at a time.
template <typename T, bool kVectors>
__global__ void __launch_bounds__(kBalThreads)
balance_backward_four_kernel(BalanceArgs a, const float* coef, const float* grad_loss, T* grads) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const int group = 1 << a.log2_group;
  const int first = (lane & (group - 1)) * 8;
  const int rows = kBalThreads >> a.log2_group;
  const int mine = static_cast<int>(threadIdx.x) >> a.log2_group;
  const T* logits = static_cast<const T*>(a.logits[blockIdx.y]);
  T* out = grads + static_cast<long long>(blockIdx.y) * a.n_tokens * a.experts;
  const float up = *grad_loss;
  const float lse_coef = coef[a.experts] * up;
  F2 w[4];
  {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = first + e < a.experts ? coef[first + e] * up : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f2(v[2 * i], v[2 * i + 1]);
  }
  for (long long base = static_cast<long long>(blockIdx.x) * rows * 4; base < a.n_tokens; base += static_cast<long long>(gridDim.x) * rows * 4) {
    F2 x[4][4];
    bool kept[4];
    float top[4], total[4], dot[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) kept[r] = balance_kept(a, base + r * rows + mine);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float v[8];
      balance_load<T, kVectors, 8>(logits + (base + r * rows + mine) * a.ld, first, a.experts, kept[r], v, -INFINITY);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[r][i] = f2(v[2 * i], v[2 * i + 1]);
      top[r] = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    }
    for (int o = group >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int r = 0; r < 4; ++r) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], o));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const F2 minus_top = both(-top[r]);
      F2 sum = both(0.f), product = both(0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 d = mul2(add2(x[r][i], minus_top), both(kLog2e));
        x[r][i] = f2(ex2_approx(f2_lo(d)), ex2_approx(f2_hi(d)));
        sum = add2(sum, x[r][i]);
        product = fma2(x[r][i], w[i], product);
      }
      total[r] = f2_lo(sum) + f2_hi(sum);
      dot[r] = f2_lo(product) + f2_hi(product);
    }
    const float sums = lane_four_sums(total, group);
    const float inv = 1.f / sums;
    const float mean = lane_four_sums(dot, group) * inv;        // sum a p
    const float ln = lse_coef != 0.f ? ln_approx(sums) : 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long long token = base + r * rows + mine;
      const float scale = of_four(inv, r, a.log2_group), m = of_four(mean, r, a.log2_group), l = of_four(ln, r, a.log2_group);
      if (token >= a.n_tokens) continue;
      const F2 shift = both(lse_coef != 0.f ? fmaf(lse_coef, top[r] + l, -m) : -m);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 g = mul2(mul2(x[r][i], both(scale)), add2(w[i], shift));
        v[2 * i] = kept[r] ? f2_lo(g) : 0.f;
        v[2 * i + 1] = kept[r] ? f2_hi(g) : 0.f;
      }
      T* row = out + token * a.experts;
      if constexpr (kVectors) {
        constexpr int kVec = CeElem<T>::kVec;
#pragma unroll
        for (int u = 0; u < 8 / kVec; ++u) {
          if (first + u * kVec < a.experts) {
            float part[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) part[i] = v[u * kVec + i];
            ce_store_vec<T>(row + first + u * kVec, part);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (first + e < a.experts) CeElem<T>::store(row + first + e, v[e]);
        }
      }
    }
  }
}

}  // namespace flce
