// Host side of the router's load-balancing loss (kernels: router_balance.cuh; documented in include/flce_b200.h).
#include "host_internal.hpp"
#include "router_balance.cuh"

#include <cstdint>

namespace flce {
namespace {


int check_balance(const flce_balance_t* p) {
  if (p == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "balance is NULL");
  if (p->n_layers <= 0 || p->n_tokens < 0 || p->n_tokens > 0x7fffffffll || p->n_experts <= 0 || p->n_layers > 0xffff)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "bad shape (n_layers=%lld n_tokens=%lld n_experts=%lld)", (long long)p->n_layers,
                (long long)p->n_tokens, (long long)p->n_experts);
  if (p->n_experts > 32 * kBalMaxEpt)
    return fail(FLCE_ERR_UNSUPPORTED, "at most %d experts, got %lld", 32 * kBalMaxEpt, (long long)p->n_experts);
  if (p->top_k <= 0 || p->top_k > p->n_experts)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "top_k must be in [1, %lld], got %lld", (long long)p->n_experts, (long long)p->top_k);
  if (p->ld < 0) return fail(FLCE_ERR_INVALID_ARGUMENT, "negative pitch %lld", (long long)p->ld);
  if (p->dtype < FLCE_BF16 || p->dtype > FLCE_FP32) return fail(FLCE_ERR_INVALID_ARGUMENT, "bad dtype %d", p->dtype);
  if (p->mask != nullptr && p->mask_bytes != 1 && p->mask_bytes != 4 && p->mask_bytes != 8)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "mask elements have 1, 4 or 8 bytes, got %d", p->mask_bytes);
  if (p->mask != nullptr && (reinterpret_cast<uintptr_t>(p->mask) % p->mask_bytes) != 0)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "the mask does not start on a multiple of its element size");
  return FLCE_OK;
}

int check_layers(const flce_balance_t* p, const void* const* logits) {
  if (logits == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "logits is NULL");
  for (int64_t l = 0; l < p->n_layers; ++l) {
    if (p->n_tokens > 0 && logits[l] == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "logits of layer %lld are NULL", (long long)l);
    if ((reinterpret_cast<uintptr_t>(logits[l]) % element_size(p->dtype)) != 0)
      return fail(FLCE_ERR_INVALID_ARGUMENT, "logits of layer %lld do not start on a multiple of their element size", (long long)l);
  }
  return FLCE_OK;
}

struct BalanceShape {
  bool vectors;             // rows of whole, aligned vectors
  bool tile;                // forward: rows by tiles of 32 per warp
  int ept, log2_group;      // logits per lane, lanes per row
  int tile_warps, tile_buffers;     // warps per block of the tile kernel and tiles per warp, as its shared memory allows
  size_t tile_bytes;
};

// Lanes that share a row: as many as it takes with 8 logits each, and more logits per lane beyond 256 experts.
BalanceShape balance_shape(const flce_balance_t* p, bool vectors) {
  BalanceShape s;
  s.vectors = vectors;
  s.ept = p->n_experts <= 256 ? 8 : (p->n_experts <= 512 ? 16 : 32);
  for (s.log2_group = 0; (s.ept << s.log2_group) < p->n_experts;) ++s.log2_group;
  s.tile = vectors && p->n_experts % 8 == 0 && p->n_experts >= 32 && p->n_experts <= 256 && p->top_k <= kTileListMost &&
           p->n_tokens <= 1 << 24;
  const int row_bytes = static_cast<int>(p->n_experts) * element_size(p->dtype);
  s.tile_buffers = kTileMaxWarps * tile_warp_bytes(row_bytes, 2) <= kMostDynamicShared ? 2 : 1;
  s.tile_warps = kMostDynamicShared / tile_warp_bytes(row_bytes, s.tile_buffers);
  if (s.tile_warps > kTileMaxWarps) s.tile_warps = kTileMaxWarps;
  const long long tiles = ceil_div(p->n_tokens, 32);       // fewer than that many: a smaller block
  if (s.tile_warps > tiles) s.tile_warps = tiles > 0 ? static_cast<int>(tiles) : 1;
  const size_t fold = static_cast<size_t>(s.tile_warps) * (2 * 256 + 2) * 4;
  s.tile_bytes = static_cast<size_t>(s.tile_warps) * tile_warp_bytes(row_bytes, s.tile_buffers);
  if (s.tile_bytes < fold) s.tile_bytes = fold;
  return s;
}

bool whole_vectors(const flce_balance_t* p, const void* const* logits, const void* out) {
  const int vec = 16 / element_size(p->dtype);
  bool yes = p->n_experts % vec == 0 && (p->n_tokens <= 1 || p->ld % vec == 0) && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  for (int64_t l = 0; l < p->n_layers; ++l) yes = yes && (reinterpret_cast<uintptr_t>(logits[l]) & 15) == 0;
  return yes;
}

// Blocks per layer of the kernels that walk over the rows: `per_sm` of them per SM over all layers, a round of rows each at least.
long long walking_blocks(const flce_balance_t* p, long long rows_per_round, int per_sm, int sm_count) {
  const long long rounds = ceil_div(p->n_tokens, rows_per_round);
  long long blocks = ceil_div(static_cast<long long>(per_sm) * sm_count, p->n_layers);
  if (blocks > rounds) blocks = rounds;
  return blocks < 1 ? 1 : blocks;
}
// Forward leaves a partial sum per block: the plain kernel has eight blocks per SM, so that the last wave costs little; the tile
// kernel as many as are resident, which its warps share evenly.
long long forward_blocks(const flce_balance_t* p, const BalanceShape& s, int sm_count) {
  if (!s.tile) return walking_blocks(p, kBalThreads >> s.log2_group, 8, sm_count);
  const long long slots = sm_count;
  const long long blocks = slots / p->n_layers;                  // one wave
  const long long rounds = ceil_div(p->n_tokens, 32 * s.tile_warps);
  return blocks > rounds ? (rounds > 0 ? rounds : 1) : (blocks > 0 ? blocks : 1);
}

BalanceArgs balance_args(const flce_balance_t* p, const void* const* logits, int64_t first_layer, int64_t layers, const BalanceShape& s) {
  BalanceArgs a{};
  for (int64_t l = 0; l < layers; ++l) a.logits[l] = logits[first_layer + l];
  a.ld = p->ld;
  a.n_tokens = p->n_tokens;
  a.experts = static_cast<int>(p->n_experts);
  a.top_k = static_cast<int>(p->top_k);
  a.mask = p->mask;
  a.mask_bytes = p->mask_bytes;
  a.log2_group = s.log2_group;
  a.want_lse = p->lse_square_scale != 0.f;
  return a;
}

template <class Fn>
void with_type(int dtype, Fn fn) {
  if (dtype == FLCE_FP32) fn(float());
  else if (dtype == FLCE_BF16) fn(__nv_bfloat16());
  else fn(__half());
}

template <typename T, bool kVectors>
void run_forward(const BalanceArgs& a, const BalanceShape& s, dim3 grid, float* partial, cudaStream_t stream) {
  switch (s.ept) {
    case 8: FLCE_LAUNCH((balance_forward_kernel<T, kVectors, 8>), grid, kBalThreads, stream, a, partial); break;
    case 16: FLCE_LAUNCH((balance_forward_kernel<T, kVectors, 16>), grid, kBalThreads, stream, a, partial); break;
    default: FLCE_LAUNCH((balance_forward_kernel<T, kVectors, 32>), grid, kBalThreads, stream, a, partial); break;
  }
}

template <typename T>
int run_forward_tile(const BalanceArgs& a, const BalanceShape& s, dim3 grid, float* partial, cudaStream_t stream) {
  const unsigned threads = static_cast<unsigned>(s.tile_warps * 32);
  if (a.top_k <= 8) return launch_with_shared<balance_forward_tile_kernel<T, 8>>(grid, threads, s.tile_bytes, stream, a, s.tile_buffers, partial);
  return launch_with_shared<balance_forward_tile_kernel<T, 16>>(grid, threads, s.tile_bytes, stream, a, s.tile_buffers, partial);
}

// With a group of 4 lanes or more the four-row kernel; smaller groups have rows short enough for a lane or two.
template <typename T, bool kVectors>
void run_backward(const BalanceArgs& a, const BalanceShape& s, dim3 grid, const float* coef, const float* up, T* out,
                  cudaStream_t stream) {
  if (s.ept == 8 && s.log2_group >= 2) {
    FLCE_LAUNCH((balance_backward_four_kernel<T, kVectors>), grid, kBalThreads, stream, a, coef, up, out);
    return;
  }
  switch (s.ept) {
    case 8: FLCE_LAUNCH((balance_backward_kernel<T, kVectors, 8>), grid, kBalThreads, stream, a, coef, up, out); break;
    case 16: FLCE_LAUNCH((balance_backward_kernel<T, kVectors, 16>), grid, kBalThreads, stream, a, coef, up, out); break;
    default: FLCE_LAUNCH((balance_backward_kernel<T, kVectors, 32>), grid, kBalThreads, stream, a, coef, up, out); break;
  }
}

// workspace: sums [layers][experts + 1] fp64, kept [layers] int64, partial [layers][blocks][2 experts + 2] 32-bit
size_t workspace_bytes(const flce_balance_t* p, long long blocks) {
  const size_t layers = static_cast<size_t>(p->n_layers), experts = static_cast<size_t>(p->n_experts);
  return layers * (experts + 1) * 8 + layers * 8 + layers * static_cast<size_t>(blocks) * (2 * experts + 2) * 4;
}

}  // namespace
}  // namespace flce

using namespace flce;

extern "C" {

size_t flce_b200_balance_workspace_bytes(const flce_balance_t* p) {
  int sms = 0;
  if (check_balance(p) != FLCE_OK || current_sm_count(&sms) != FLCE_OK) return 0;
  // whether the rows are whole, aligned vectors is not known yet: room for the larger grid
  const long long plain = forward_blocks(p, balance_shape(p, false), sms), tile = forward_blocks(p, balance_shape(p, true), sms);
  return workspace_bytes(p, plain > tile ? plain : tile);
}

int flce_b200_balance_forward(const flce_balance_t* p, const void* const* logits, float* loss, int64_t* counts, float* coef,
                              void* workspace, size_t bytes, void* stream_) {
  int rc = check_balance(p);
  if (rc != FLCE_OK) return rc;
  rc = check_layers(p, logits);
  if (rc != FLCE_OK) return rc;
  if (loss == nullptr || counts == nullptr || coef == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "NULL output");
  int sms = 0;
  rc = current_sm_count(&sms);
  if (rc != FLCE_OK) return rc;
  const BalanceShape s = balance_shape(p, whole_vectors(p, logits, nullptr));
  const long long blocks = forward_blocks(p, s, sms);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0 || bytes < workspace_bytes(p, blocks))
    return fail(FLCE_ERR_WORKSPACE, "the balance loss needs %zu bytes of 8-byte aligned workspace, got %zu", workspace_bytes(p, blocks),
                bytes);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int experts = static_cast<int>(p->n_experts);
  double* sums = static_cast<double*>(workspace);
  long long* kept = reinterpret_cast<long long*>(sums + p->n_layers * (p->n_experts + 1));
  float* partial = reinterpret_cast<float*>(kept + p->n_layers);
  int launches = 1;
  for (int64_t l = 0; l < p->n_layers; l += kBalMaxLayers) {
    const int64_t layers = p->n_layers - l < kBalMaxLayers ? p->n_layers - l : kBalMaxLayers;
    const BalanceArgs a = balance_args(p, logits, l, layers, s);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(layers));
    float* mine = partial + l * blocks * balance_partial_words(experts);
    with_type(p->dtype, [&](auto t) {
      using T = decltype(t);
      if (s.tile) rc = run_forward_tile<T>(a, s, grid, mine, stream);
      else if (s.vectors) run_forward<T, true>(a, s, grid, mine, stream);
      else run_forward<T, false>(a, s, grid, mine, stream);
    });
    if (rc != FLCE_OK) return rc;
    ++launches;
  }
  // few partials: the last kernel adds them up itself
  const bool few = p->n_layers * blocks <= 32;
  if (!few) {
    const dim3 columns(static_cast<unsigned>(ceil_div(experts + 1, 32)), static_cast<unsigned>(p->n_layers));
    rc = launch_dependent<balance_layer_kernel>(columns, dim3(32, kBalFoldLanes), stream, static_cast<const float*>(partial),
                                                static_cast<int>(blocks), experts, reinterpret_cast<long long*>(counts), sums, kept);
    if (rc != FLCE_OK) return rc;
    ++launches;
  }
  const int threads = few && experts <= 256 ? 256 : kBalTotalThreads;
  rc = launch_dependent<balance_total_kernel>(dim3(1), dim3(threads), stream, static_cast<const float*>(few ? partial : nullptr),
                                              static_cast<int>(blocks), reinterpret_cast<long long*>(counts), static_cast<const double*>(sums),
                                              static_cast<const long long*>(kept), static_cast<int>(p->n_layers), experts,
                                              p->lse_square_scale, loss, coef);
  if (rc != FLCE_OK) return rc;
  FLCE_CUDA(cudaGetLastError());
  count_launches(launches);
  return FLCE_OK;
}

int flce_b200_balance_backward(const flce_balance_t* p, const void* const* logits, const float* coef, const float* grad_loss,
                               void* grads, void* stream_) {
  int rc = check_balance(p);
  if (rc != FLCE_OK) return rc;
  rc = check_layers(p, logits);
  if (rc != FLCE_OK) return rc;
  if (p->n_tokens == 0) return FLCE_OK;
  if (coef == nullptr || grad_loss == nullptr || grads == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "NULL argument");
  if ((reinterpret_cast<uintptr_t>(grads) % element_size(p->dtype)) != 0)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "the gradients do not start on a multiple of their element size");
  int sms = 0;
  rc = current_sm_count(&sms);
  if (rc != FLCE_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const BalanceShape s = balance_shape(p, whole_vectors(p, logits, grads));
  const bool four = s.ept == 8 && s.log2_group >= 2;
  const long long blocks = walking_blocks(p, (kBalThreads >> s.log2_group) * (four ? 4 : 1), four ? 16 : 8, sms);
  int launches = 0;
  for (int64_t l = 0; l < p->n_layers; l += kBalMaxLayers) {
    const int64_t layers = p->n_layers - l < kBalMaxLayers ? p->n_layers - l : kBalMaxLayers;
    const BalanceArgs a = balance_args(p, logits, l, layers, s);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(layers));
    with_type(p->dtype, [&](auto t) {
      using T = decltype(t);
      T* out = static_cast<T*>(grads) + l * p->n_tokens * p->n_experts;
      if (s.vectors) run_backward<T, true>(a, s, grid, coef, grad_loss, out, stream);
      else run_backward<T, false>(a, s, grid, coef, grad_loss, out, stream);
    });
    ++launches;
  }
  FLCE_CUDA(cudaGetLastError());
  count_launches(launches);
  return FLCE_OK;
}

}  // extern "C"
