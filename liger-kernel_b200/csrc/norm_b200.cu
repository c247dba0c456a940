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

// How a row is spread: `unit` consecutive elements per access, `ept` elements per thread, 1 << log2_group threads.
struct NormShape {
  int unit, ept, log2_group;
  bool fits;
};

NormShape norm_shape(const flce_norm_t* p, bool whole_vectors, int preferred_threads) {
  NormShape s;
  s.unit = whole_vectors ? 16 / element_size(p->dtype) : 1;
  const long long units = ceil_div(p->hidden, s.unit);
  if (units <= 32) {        // one unit per thread, several rows to a warp
    s.ept = s.unit;
    for (s.log2_group = 0; (1ll << s.log2_group) < units;) ++s.log2_group;
    s.fits = true;
    return s;
  }
  for (s.ept = 8;; s.ept *= 2) {
    for (s.log2_group = 5; (1ll << s.log2_group) * s.ept < units * s.unit;) ++s.log2_group;
    s.fits = (1ll << s.log2_group) <= kNormMaxThreads;
    if ((1ll << s.log2_group) <= preferred_threads || s.ept == kNormMaxEpt) return s;
  }
}

// Rows of whole vectors go to the streaming kernels, or to the narrow ones if a warp's lanes hold one with a vector each.
enum NormPath { kNormGeneric, kNormStream, kNormNarrow };
constexpr int kNarrowForwardRows = 4, kNarrowBackwardRows = 2;

struct NormPlan {
  NormPath path;
  NormShape shape;      // ept holds the vectors per lane, except on the generic path
};

int log2_ceil(long long v) {
  int l = 0;
  while ((1ll << l) < v) ++l;
  return l;
}

// The streaming kernels give every thread of a 512-thread block its columns: one vector if that reaches, up to four.
NormPlan norm_plan(const flce_norm_t* p, bool vectors, int preferred_threads) {
  NormPlan plan{kNormGeneric, {}};
  const long long n = p->hidden * element_size(p->dtype) / 16;
  if (vectors && n <= 32) {
    plan.path = kNormNarrow;
    plan.shape = {1, 1, log2_ceil(n), true};
  } else if (vectors && n <= 4 * kStreamThreads) {
    int units = 1;
    while (units * kStreamThreads < n) units *= 2;
    int log2_group = 5;
    while ((units << log2_group) < n) ++log2_group;
    plan.path = kNormStream;
    plan.shape = {1, units, log2_group, true};
  } else {
    plan.shape = norm_shape(p, vectors, preferred_threads);
  }
  return plan;
}

template <bool kGrad>
int stream_rows(int units) {
  return units == 1 ? Stream<1, kGrad>::kRows : (units == 2 ? Stream<2, kGrad>::kRows : Stream<4, kGrad>::kRows);
}

bool whole_vectors(const flce_norm_t* p, const void* other, long long ld_other) {
  const int vec = 16 / element_size(p->dtype);
  const bool pitches = p->n_rows <= 1 || (p->ld_x % vec == 0 && ld_other % vec == 0);     // one row has no pitch
  return p->hidden % vec == 0 && pitches && aligned16(p->x) && aligned16(other) &&
         aligned16(p->weight) && aligned16(p->bias);
}

template <typename T, typename W, bool kCentered, int kUnit>
void run_forward(const NormForwardArgs& a, const NormShape& s, unsigned grid, int threads, cudaStream_t stream) {
  switch (s.ept) {
    case kUnit < 8 ? kUnit : -1: FLCE_LAUNCH((norm_forward_kernel<T, W, kCentered, kUnit, kUnit>), grid, threads, stream, a); break;
    case 8: FLCE_LAUNCH((norm_forward_kernel<T, W, kCentered, kUnit, 8>), grid, threads, stream, a); break;
    case 16: FLCE_LAUNCH((norm_forward_kernel<T, W, kCentered, kUnit, 16>), grid, threads, stream, a); break;
    default: FLCE_LAUNCH((norm_forward_kernel<T, W, kCentered, kUnit, 32>), grid, threads, stream, a); break;
  }
}

template <typename T, typename W, bool kCentered, int kUnit>
void run_backward(const NormBackwardArgs& a, const NormShape& s, unsigned grid, cudaStream_t stream) {
  switch (s.ept) {
    case kUnit < 8 ? kUnit : -1: FLCE_LAUNCH((norm_backward_kernel<T, W, kCentered, kUnit, kUnit>), grid, kNormMaxThreads, stream, a); break;
    case 8: FLCE_LAUNCH((norm_backward_kernel<T, W, kCentered, kUnit, 8>), grid, kNormMaxThreads, stream, a); break;
    case 16: FLCE_LAUNCH((norm_backward_kernel<T, W, kCentered, kUnit, 16>), grid, kNormMaxThreads, stream, a); break;
    default: FLCE_LAUNCH((norm_backward_kernel<T, W, kCentered, kUnit, 32>), grid, kNormMaxThreads, stream, a); break;
  }
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

// Blocks of the backward kernel: they are resident together and walk over the rows.  Each leaves hidden partial sums per
// parameter, so no more of them than it takes to fill the device.
long long backward_blocks(const flce_norm_t* p, const NormPlan& plan, int sm_count) {
  long long rows = 1, per_sm = 2;
  if (plan.path == kNormNarrow) {
    rows = (kNarrowThreads >> plan.shape.log2_group) * kNarrowBackwardRows;
    per_sm = 4;
  } else if (plan.path == kNormStream) {
    rows = (kStreamThreads >> plan.shape.log2_group) * stream_rows<true>(plan.shape.ept);
    per_sm = plan.shape.ept == 1 ? 2 : 1;
  } else if (plan.shape.fits) {
    rows = kNormMaxThreads >> plan.shape.log2_group;
  }
  const long long most = ceil_div(p->n_rows, rows);
  const long long resident = per_sm * sm_count;
  return most < resident ? most : resident;
}

template <typename T, typename W, bool kCentered>
int run_forward_stream(const NormForwardArgs& a, const NormShape& s, int sm_count, cudaStream_t stream) {
  const long long most = ceil_div(a.n_rows, (kStreamThreads >> s.log2_group) * stream_rows<false>(s.ept));
  const long long resident = (s.ept == 1 ? 2ll : 1ll) * sm_count;
  const dim3 grid(static_cast<unsigned>(most < resident ? most : resident));
  switch (s.ept) {
    case 1: return launch_with_shared<norm_forward_stream_kernel<T, W, kCentered, 1>>(grid, kStreamThreads, Stream<1, false>::kRingBytes, stream, a);
    case 2: return launch_with_shared<norm_forward_stream_kernel<T, W, kCentered, 2>>(grid, kStreamThreads, Stream<2, false>::kRingBytes, stream, a);
    default: return launch_with_shared<norm_forward_stream_kernel<T, W, kCentered, 4>>(grid, kStreamThreads, Stream<4, false>::kRingBytes, stream, a);
  }
}

template <typename T, typename W, bool kCentered>
int run_backward_stream(const NormBackwardArgs& a, const NormShape& s, unsigned blocks, cudaStream_t stream) {
  const dim3 grid(blocks);
  switch (s.ept) {
    case 1: return launch_with_shared<norm_backward_stream_kernel<T, W, kCentered, 1>>(grid, kStreamThreads, Stream<1, true>::kRingBytes, stream, a);
    case 2: return launch_with_shared<norm_backward_stream_kernel<T, W, kCentered, 2>>(grid, kStreamThreads, Stream<2, true>::kRingBytes, stream, a);
    default: return launch_with_shared<norm_backward_stream_kernel<T, W, kCentered, 4>>(grid, kStreamThreads, Stream<4, true>::kRingBytes, stream, a);
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
  const NormPlan plan = norm_plan(p, whole_vectors(p, y, p->hidden), kNormForwardThreads);
  const NormShape& s = plan.shape;
  a.log2_group = s.log2_group;
  const int threads = (1 << s.log2_group) > kNormForwardThreads ? (1 << s.log2_group) : kNormForwardThreads;
  const bool centered = p->kind == FLCE_LAYER_NORM;
  with_types(p, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int kVec = CeElem<T>::kVec;
    if (plan.path == kNormStream) {
      rc = centered ? run_forward_stream<T, W, true>(a, s, sms, stream) : run_forward_stream<T, W, false>(a, s, sms, stream);
      return;
    }
    if (plan.path == kNormNarrow) {
      const unsigned grid = static_cast<unsigned>(ceil_div(p->n_rows, (kNarrowThreads >> s.log2_group) * kNarrowForwardRows));
      if (centered) FLCE_LAUNCH((norm_forward_narrow_kernel<T, W, true, kNarrowForwardRows>), grid, kNarrowThreads, stream, a);
      else FLCE_LAUNCH((norm_forward_narrow_kernel<T, W, false, kNarrowForwardRows>), grid, kNarrowThreads, stream, a);
      return;
    }
    if (!s.fits) {
      const unsigned grid = static_cast<unsigned>(p->n_rows);
      if (centered) FLCE_LAUNCH((norm_forward_long_kernel<T, W, true>), grid, kNormMaxThreads, stream, a);
      else FLCE_LAUNCH((norm_forward_long_kernel<T, W, false>), grid, kNormMaxThreads, stream, a);
      return;
    }
    const unsigned grid = static_cast<unsigned>(ceil_div(p->n_rows, threads >> s.log2_group));
    if (s.unit == 1) {
      if (centered) run_forward<T, W, true, 1>(a, s, grid, threads, stream);
      else run_forward<T, W, false, 1>(a, s, grid, threads, stream);
    } else {
      if (centered) run_forward<T, W, true, kVec>(a, s, grid, threads, stream);
      else run_forward<T, W, false, kVec>(a, s, grid, threads, stream);
    }
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
  const long long blocks_vec = backward_blocks(p, norm_plan(p, true, kNormMaxThreads), sms);
  const long long blocks_one = backward_blocks(p, norm_plan(p, false, kNormMaxThreads), sms);
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
  const NormPlan plan = norm_plan(p, whole_vectors(p, grad_y, ld_grad) && aligned16(grad_x), kNormMaxThreads);
  const NormShape& s = plan.shape;
  const long long blocks = backward_blocks(p, plan, sms);
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
  a.log2_group = s.log2_group;
  const unsigned grid = static_cast<unsigned>(blocks);
  with_types(p, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int kVec = CeElem<T>::kVec;
    if (plan.path == kNormStream) {
      rc = centered ? run_backward_stream<T, W, true>(a, s, grid, stream) : run_backward_stream<T, W, false>(a, s, grid, stream);
      if (rc != FLCE_OK) return;
    } else if (plan.path == kNormNarrow) {
      if (centered) FLCE_LAUNCH((norm_backward_narrow_kernel<T, W, true, kNarrowBackwardRows>), grid, kNarrowThreads, stream, a);
      else FLCE_LAUNCH((norm_backward_narrow_kernel<T, W, false, kNarrowBackwardRows>), grid, kNarrowThreads, stream, a);
    } else if (!s.fits) {
      const unsigned rows = static_cast<unsigned>(p->n_rows);
      const dim3 columns(static_cast<unsigned>(ceil_div(p->hidden, kNormForwardThreads)), grid < 65535u ? grid : 65535u);
      if (centered) FLCE_LAUNCH((norm_backward_long_kernel<T, W, true>), rows, kNormMaxThreads, stream, a);
      else FLCE_LAUNCH((norm_backward_long_kernel<T, W, false>), rows, kNormMaxThreads, stream, a);
      if (parameters) {
        if (centered) FLCE_LAUNCH((norm_parameter_partial_long_kernel<T, true>), columns, kNormForwardThreads, stream, a);
        else FLCE_LAUNCH((norm_parameter_partial_long_kernel<T, false>), columns, kNormForwardThreads, stream, a);
      }
    } else if (s.unit == 1) {
      if (centered) run_backward<T, W, true, 1>(a, s, grid, stream);
      else run_backward<T, W, false, 1>(a, s, grid, stream);
    } else {
      if (centered) run_backward<T, W, true, kVec>(a, s, grid, stream);
      else run_backward<T, W, false, kVec>(a, s, grid, stream);
    }
    if (parameters) {
      const dim3 columns(static_cast<unsigned>(ceil_div(p->hidden, 32)), centered ? 2 : 1);
      FLCE_LAUNCH((norm_parameter_gradient_kernel<W>), columns, dim3(32, kNormReduceLanes), stream, 
          a.dw_partial, a.db_partial, static_cast<int>(grid), a.hidden, static_cast<W*>(grad_weight), static_cast<W*>(grad_bias));
    }
  });
  if (rc != FLCE_OK) return rc;
  FLCE_CUDA(cudaGetLastError());
  count_launches(1 + (parameters ? (s.fits ? 1 : 2) : 0));
  return FLCE_OK;
}

}  // extern "C"
