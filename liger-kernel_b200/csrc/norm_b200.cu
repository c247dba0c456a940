// Host side of layer norm and RMSNorm (kernels: norm_rows.cuh; documented in include/flce_b200.h): argument checks, the
// choice of a launch shape, launches.
#include "host_internal.hpp"
#include "norm_rows.cuh"

#include <cstdint>

namespace flce {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_norm(const flce_norm_t* p) {
  if (p == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "norm is NULL");
  if (p->n_rows < 0 || p->hidden <= 0 || p->hidden > 0x7fffffffll / 2 || p->n_rows > 0x7fffffffll)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "bad shape (n_rows=%lld hidden=%lld)", (long long)p->n_rows, (long long)p->hidden);
  if (p->kind != FLCE_LAYER_NORM && p->kind != FLCE_RMS_NORM) return fail(FLCE_ERR_INVALID_ARGUMENT, "bad kind %d", p->kind);
  if (p->dtype < FLCE_BF16 || p->dtype > FLCE_FP32) return fail(FLCE_ERR_INVALID_ARGUMENT, "bad dtype %d", p->dtype);
  if (p->weight_dtype != p->dtype && p->weight_dtype != FLCE_FP32)
    return fail(FLCE_ERR_UNSUPPORTED, "weight and bias have the rows' type or fp32");
  if (p->kind == FLCE_RMS_NORM && p->bias != nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "RMSNorm has no bias");
  if (p->ld_x < 0) return fail(FLCE_ERR_INVALID_ARGUMENT, "negative pitch %lld", (long long)p->ld_x);
  const int esize = element_size(p->dtype), wsize = element_size(p->weight_dtype);
  if ((reinterpret_cast<uintptr_t>(p->x) % esize) != 0 || (reinterpret_cast<uintptr_t>(p->weight) % wsize) != 0 ||
      (reinterpret_cast<uintptr_t>(p->bias) % wsize) != 0)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "a tensor does not start on a multiple of its element size");
  return FLCE_OK;
}

// How the rows are spread over threads: `share` elements (window) or 16-byte vectors (stream) per thread; the threads of a row
// as a power of two (narrow, stream, tiny) or as whole warps (stream, window).
enum NormPath { kNormStream, kNormNarrow, kNormWindow, kNormTiny, kNormLong };
struct NormPlan {
  NormPath path;
  int share, log2_group, warps;
  bool few;       // stream, forward: a row per group and round
  bool wide;      // fp32 rows
};

int log2_group_for(long long pieces, int smallest) {
  int l = smallest;
  while ((1ll << l) < pieces) ++l;
  return l;
}

// Narrow: a lane per vector, rows of up to 32 of them.  Stream: two vectors per thread if a block's 512 threads reach so, else four.
// Window: of 2, 4, 8 and 16 elements per lane the cheapest, taking a warp's part of a row to cost 8 elements beside those it
// holds: 50000 x 300 bf16 forward 45, 33, 29 and 23 us, 10007 x 1537 fp16 43, 31 and 27 us from 4 on, 100000 x 100 bf16 45, 25,
// 33 and 47 us.  Long: what is left, above 8192 elements.
NormPlan norm_plan(const flce_norm_t* p, bool vectors, int sm_count) {
  const bool wide = p->dtype == FLCE_FP32;
  const long long n = p->hidden * element_size(p->dtype) / 16;
  if (vectors && n <= 32) return {kNormNarrow, 1, log2_group_for(n, 2), 0, false, wide};
  if (vectors && n <= 4 * kStreamThreads) {
    const int share = n <= 2 * kStreamThreads ? 2 : 4;
    const int log2_group = log2_group_for(ceil_div(n, share), 5);
    const bool few = share == 2 && p->n_rows <= (static_cast<long long>(sm_count) * kStreamThreads >> log2_group);
    return {kNormStream, share, log2_group, 1 << (log2_group - 5), few, wide};
  }
  if (p->hidden <= 32) return {kNormTiny, 1, log2_group_for(p->hidden, 2), 0, false, wide};
  NormPlan best{kNormLong, 0, 9, kNormMaxWarps, false, wide};
  double least = 0.0;
  for (int share = 2; share <= 16; share *= 2) {
    const long long warps = ceil_div(p->hidden, 32 * share);
    if (warps > kWindowWarps) continue;
    const double cost = (share + 8.0) / static_cast<double>(kWindowWarps / warps);
    if (best.path == kNormLong || cost < least) {
      least = cost;
      best = {kNormWindow, share, 0, static_cast<int>(warps), false, wide};
    }
  }
  return best;
}

// fn(std::integral_constant<int, elements per lane>) for a window plan
template <class Fn>
int with_share(int share, Fn fn) {
  switch (share) {
    case 2: return fn(std::integral_constant<int, 2>());
    case 4: return fn(std::integral_constant<int, 4>());
    case 8: return fn(std::integral_constant<int, 8>());
    default: return fn(std::integral_constant<int, 16>());
  }
}

// rows that a block takes per round, and blocks that are resident on an SM
template <bool kGrad>
int rows_per_round(const NormPlan& plan) {
  switch (plan.path) {
    case kNormNarrow:
    case kNormTiny: return (kNarrowThreads >> plan.log2_group) * (kGrad ? kNarrowBackwardRows : kNarrowForwardRows);
    case kNormStream: return (kStreamThreads >> plan.log2_group) * (!kGrad && plan.few ? 1 : (plan.share == 2 ? Stream<2, kGrad>::kRows : Stream<4, kGrad>::kRows));
    case kNormWindow:
      return kWindowWarps / plan.warps * with_share(plan.share, [&](auto e) {
               constexpr int kEpt = decltype(e)::value;
               return plan.wide ? Window<float, kEpt, kGrad>::kRows : Window<__half, kEpt, kGrad>::kRows;
             });
    default: return 1;
  }
}
int blocks_per_sm(const NormPlan& plan) {
  switch (plan.path) {
    case kNormStream:
    case kNormWindow: return 1;
    case kNormNarrow: return kNarrowBlocksPerSm;
    case kNormLong: return 2;
    default: return 4;
  }
}

// Blocks that walk over the rows: as many as are resident together.  Those of the backward kernel leave `hidden` partial sums
// per parameter each.
template <bool kGrad>
long long walking_blocks(const flce_norm_t* p, const NormPlan& plan, int sm_count) {
  const long long most = ceil_div(p->n_rows, rows_per_round<kGrad>(plan));
  const long long resident = static_cast<long long>(blocks_per_sm(plan)) * sm_count;
  return most < resident ? most : resident;
}

bool whole_vectors(const flce_norm_t* p, const void* other, long long ld_other) {
  const int vec = 16 / element_size(p->dtype);
  const bool pitches = p->n_rows <= 1 || (p->ld_x % vec == 0 && ld_other % vec == 0);     // one row has no pitch
  return p->hidden % vec == 0 && pitches && aligned16(p->x) && aligned16(other) &&
         aligned16(p->weight) && aligned16(p->bias);
}

// fn(T{}, W{}) for the problem's types
template <class Fn>
void with_types(const flce_norm_t* p, Fn fn) {
  if (p->dtype == FLCE_FP32) fn(float(), float());
  else if (p->dtype == FLCE_BF16 && p->weight_dtype == FLCE_BF16) fn(__nv_bfloat16(), __nv_bfloat16());
  else if (p->dtype == FLCE_BF16) fn(__nv_bfloat16(), float());
  else if (p->weight_dtype == FLCE_FP16) fn(__half(), __half());
  else fn(__half(), float());
}

template <typename T, typename W, bool kCentered>
int run_forward(const NormForwardArgs& a, const NormPlan& plan, unsigned walking, cudaStream_t stream) {
  const dim3 grid(walking);
  switch (plan.path) {
    case kNormStream:
      if (plan.share == 2 && plan.few)
        return launch_with_shared<norm_forward_stream_kernel<T, W, kCentered, 2, true>>(grid, kStreamThreads, Stream<2, false, true>::kRingBytes, stream, a);
      if (plan.share == 2)
        return launch_with_shared<norm_forward_stream_kernel<T, W, kCentered, 2, false>>(grid, kStreamThreads, Stream<2, false>::kRingBytes, stream, a);
      return launch_with_shared<norm_forward_stream_kernel<T, W, kCentered, 4, false>>(grid, kStreamThreads, Stream<4, false>::kRingBytes, stream, a);
    case kNormNarrow:
      return launch_with_shared<norm_forward_narrow_kernel<T, W, kCentered>>(grid, kNarrowThreads, kNarrowRingBytes, stream, a);
    case kNormTiny: {
      const unsigned all = static_cast<unsigned>(ceil_div(a.n_rows, rows_per_round<false>(plan)));
      FLCE_LAUNCH((norm_forward_tiny_kernel<T, W, kCentered>), all, kNarrowThreads, stream, a);
      return FLCE_OK;
    }
    case kNormWindow:
      return with_share(plan.share, [&](auto e) {
        constexpr int kEpt = decltype(e)::value;
        return launch_with_shared<norm_forward_window_kernel<T, W, kCentered, kEpt>>(grid, kWindowThreads, Window<T, kEpt, false>::kBytes,
                                                                                    stream, a);
      });
    default:
      FLCE_LAUNCH((norm_forward_long_kernel<T, W, kCentered>), static_cast<unsigned>(a.n_rows), kNormMaxThreads, stream, a);
      return FLCE_OK;
  }
}

template <typename T, typename W, bool kCentered>
int run_backward(const NormBackwardArgs& a, const NormPlan& plan, unsigned walking, cudaStream_t stream) {
  const dim3 grid(walking);
  switch (plan.path) {
    case kNormStream:
      if (plan.share == 2)
        return launch_with_shared<norm_backward_stream_kernel<T, W, kCentered, 2>>(grid, kStreamThreads, Stream<2, true>::kRingBytes, stream, a);
      return launch_with_shared<norm_backward_stream_kernel<T, W, kCentered, 4>>(grid, kStreamThreads, Stream<4, true>::kRingBytes, stream, a);
    case kNormNarrow:
      return launch_with_shared<norm_backward_narrow_kernel<T, W, kCentered>>(grid, kNarrowThreads, kNarrowRingBytes, stream, a);
    case kNormTiny:
      FLCE_LAUNCH((norm_backward_tiny_kernel<T, W, kCentered>), grid, kNarrowThreads, stream, a);
      return FLCE_OK;
    case kNormWindow:
      return with_share(plan.share, [&](auto e) {
        constexpr int kEpt = decltype(e)::value;
        return launch_with_shared<norm_backward_window_kernel<T, W, kCentered, kEpt>>(grid, kWindowThreads, Window<T, kEpt, true>::kBytes,
                                                                                     stream, a);
      });
    default:
      FLCE_LAUNCH((norm_backward_long_kernel<T, W, kCentered>), static_cast<unsigned>(a.n_rows), kNormMaxThreads, stream, a);
      if (a.dw_partial != nullptr || a.db_partial != nullptr) {
        const dim3 columns(static_cast<unsigned>(ceil_div(a.hidden, kNormColumnThreads)), walking);
        FLCE_LAUNCH((norm_parameter_partial_long_kernel<T, kCentered>), columns, kNormColumnThreads, stream, a);
      }
      return FLCE_OK;
  }
}

}  // namespace
}  // namespace flce

using namespace flce;

extern "C" {

int flce_b200_norm_forward(const flce_norm_t* p, void* y, float* mean, float* rstd, void* stream_) {
  int rc = check_norm(p);
  if (rc != FLCE_OK) return rc;
  if (p->n_rows == 0) return FLCE_OK;
  if (p->x == nullptr || y == nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "NULL rows");
  int sms = 0;
  rc = current_sm_count(&sms);
  if (rc != FLCE_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  NormForwardArgs a;
  a.x = p->x;
  a.ld_x = p->ld_x;
  a.w = p->weight;
  a.b = p->bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.n_rows = p->n_rows;
  a.hidden = static_cast<int>(p->hidden);
  a.eps = p->eps;
  a.offset = p->offset;
  a.round_xhat = p->round_xhat;
  const NormPlan plan = norm_plan(p, whole_vectors(p, y, p->hidden), sms);
  a.log2_group = plan.log2_group;
  a.group_warps = plan.warps;
  const unsigned walking = static_cast<unsigned>(walking_blocks<false>(p, plan, sms));
  with_types(p, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    rc = p->kind == FLCE_LAYER_NORM ? run_forward<T, W, true>(a, plan, walking, stream) : run_forward<T, W, false>(a, plan, walking, stream);
  });
  if (rc != FLCE_OK) return rc;
  FLCE_CUDA(cudaGetLastError());
  count_launches(1);
  return FLCE_OK;
}

size_t flce_b200_norm_workspace_bytes(const flce_norm_t* p) {
  if (check_norm(p) != FLCE_OK) return 0;
  int sms = 0;
  if (current_sm_count(&sms) != FLCE_OK) return 0;
  // the row's spread may turn out either way (the gradient's alignment is not known yet): room for the larger grid
  const long long blocks_vec = walking_blocks<true>(p, norm_plan(p, true, sms), sms);
  const long long blocks_one = walking_blocks<true>(p, norm_plan(p, false, sms), sms);
  const long long blocks = blocks_vec > blocks_one ? blocks_vec : blocks_one;
  return static_cast<size_t>(blocks) * static_cast<size_t>(p->hidden) * sizeof(float) * (p->kind == FLCE_LAYER_NORM ? 2 : 1);
}

int flce_b200_norm_backward(const flce_norm_t* p, const void* grad_y, int64_t ld_grad, const float* mean, const float* rstd,
                            void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                            void* stream_) {
  int rc = check_norm(p);
  if (rc != FLCE_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool centered = p->kind == FLCE_LAYER_NORM;
  if (!centered && grad_bias != nullptr) return fail(FLCE_ERR_INVALID_ARGUMENT, "RMSNorm has no bias");
  const int esize = element_size(p->dtype), wsize = element_size(p->weight_dtype);
  if (p->n_rows == 0) {     // no rows: the sums over them are zero
    if (grad_weight != nullptr) FLCE_CUDA(cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(p->hidden) * wsize, stream));
    if (grad_bias != nullptr) FLCE_CUDA(cudaMemsetAsync(grad_bias, 0, static_cast<size_t>(p->hidden) * wsize, stream));
    return FLCE_OK;
  }
  if (p->x == nullptr || grad_y == nullptr || grad_x == nullptr || rstd == nullptr || (centered && mean == nullptr))
    return fail(FLCE_ERR_INVALID_ARGUMENT, "NULL argument");
  if (ld_grad < 0 || (reinterpret_cast<uintptr_t>(grad_y) % esize) != 0)
    return fail(FLCE_ERR_INVALID_ARGUMENT, "bad gradient pitch %lld or alignment", (long long)ld_grad);
  int sms = 0;
  rc = current_sm_count(&sms);
  if (rc != FLCE_OK) return rc;
  const NormPlan plan = norm_plan(p, whole_vectors(p, grad_y, ld_grad) && aligned16(grad_x), sms);
  const long long blocks = walking_blocks<true>(p, plan, sms);
  const bool parameters = grad_weight != nullptr || grad_bias != nullptr;
  const size_t plane = static_cast<size_t>(blocks) * static_cast<size_t>(p->hidden);
  const size_t planes = (grad_weight != nullptr ? 1 : 0) + (grad_bias != nullptr ? 1 : 0);
  if (parameters && (workspace == nullptr || !aligned16(workspace) ||
                     workspace_bytes < plane * planes * sizeof(float)))
    return fail(FLCE_ERR_WORKSPACE, "the norm's backward needs %zu bytes of 16-byte aligned workspace, got %zu", plane * planes * sizeof(float),
                workspace_bytes);
  NormBackwardArgs a;
  a.dy = grad_y;
  a.ld_dy = ld_grad;
  a.x = p->x;
  a.ld_x = p->ld_x;
  a.w = p->weight;
  a.mean = mean;
  a.rstd = rstd;
  a.dx = grad_x;
  a.dw_partial = grad_weight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.db_partial = grad_bias != nullptr ? static_cast<float*>(workspace) + (grad_weight != nullptr ? plane : 0) : nullptr;
  a.n_rows = p->n_rows;
  a.hidden = static_cast<int>(p->hidden);
  a.offset = p->offset;
  a.round_xhat = p->round_xhat;
  a.log2_group = plan.log2_group;
  a.group_warps = plan.warps;
  const unsigned walking = static_cast<unsigned>(blocks);
  with_types(p, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    rc = centered ? run_backward<T, W, true>(a, plan, walking, stream) : run_backward<T, W, false>(a, plan, walking, stream);
    if (rc != FLCE_OK) return;
    if (parameters) {
      const dim3 columns(static_cast<unsigned>(ceil_div(p->hidden, 32)), centered ? 2 : 1);
      rc = launch_dependent<norm_parameter_gradient_kernel<W>>(
          columns, dim3(32, kNormReduceLanes), stream, static_cast<const float*>(a.dw_partial), static_cast<const float*>(a.db_partial),
          static_cast<int>(walking), a.hidden, static_cast<W*>(grad_weight), static_cast<W*>(grad_bias));
    }
  });
  if (rc != FLCE_OK) return rc;
  FLCE_CUDA(cudaGetLastError());
  count_launches(1 + (parameters ? (plan.path == kNormLong ? 2 : 1) : 0));
  return FLCE_OK;
}

}  // extern "C"
