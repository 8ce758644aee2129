// RMSNorm, and residual add + RMSNorm, with an output in OCP FP8 E4M3 and fp32
// scales, for gfx950: the input of an 8-bit projection.
//
//   res   = dtype(f32(x) + f32(res))             (fused variant only)
//   y     = (f32(res) * rstd) * f32(weight),  rstd = 1 / sqrt(mean(res^2) + eps)
//   scale = max(max |y| / 448, 2^-126) over the finite y of a row, or of a group
//           of consecutive columns
//   out   = e4m3(y / scale)
// All of it is fp32 up to the one rounding to e4m3: y is not rounded to the
// input's type first. A y that is not finite becomes a NaN code.
#include <algorithm>
#include <type_traits>

#include "fp8_quant.h"
#include "hip_common.h"
#include "kl_internal.h"
#include "norm_rows.h"

namespace kl {
namespace {

__device__ __forceinline__ float wave_max(float v) { return max_xor32(max_xor16(row16_max(v))); }

// Rows of any width, element by element: the squares (writing the new
// residual), then each group's largest |y|, then its codes, all read again from
// memory.
template <typename E, bool HAS_RES>
__global__ void __launch_bounds__(kMaxThreads)
    norm8_loop_kernel(uint8_t* out, float* scales, const typename E::S* x, const typename E::S* res,
                      typename E::S* res_out, const typename E::S* weight, int hidden, int group, RowMap x_rows,
                      float eps) {
  using S = typename E::S;
  __shared__ float scratch[2][kMaxThreads / 64];
  int64_t row, x_off;
  x_rows.of_workgroup(&row, &x_off);
  const S* xr = x + x_off;
  const S* rr = HAS_RES ? res + row * hidden : nullptr;
  S* rw = HAS_RES ? res_out + row * hidden : nullptr;
  const int nw = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = __lane_id();
  float sum = 0.0f;
  for (int i = threadIdx.x; i < hidden; i += blockDim.x) {
    S v = xr[i];
    if constexpr (HAS_RES) {
      v = E::from_f32(E::to_f32(v) + E::to_f32(rr[i]));
      rw[i] = v;
    }
    sum += E::to_f32(v) * E::to_f32(v);
  }
  sum = wave_sum(sum);
  if (lane == 0) scratch[0][wave] = sum;
  __syncthreads();  // (the residual is read again by other threads of the workgroup, too)
  float total = 0.0f;
  for (int w = 0; w < nw; ++w) total += scratch[0][w];
  const float rstd = inv_rms(total, hidden, eps);
  const S* src = HAS_RES ? rw : xr;
  auto y_of = [&](int i) { return (E::to_f32(src[i]) * rstd) * E::to_f32(weight[i]); };
  // A group belongs to a wave, a whole row to all of them.
  const bool whole = group == hidden;
  const int groups = hidden / group;
  const int step = whole ? blockDim.x : 64, first = whole ? threadIdx.x : lane;
  for (int g = whole ? 0 : wave; g < groups; g += whole ? 1 : nw) {
    float most = 0.0f;
    for (int i = first; i < group; i += step) most = fmaxf(most, finite_abs(y_of(g * group + i)));
    most = wave_max(most);
    if (whole) {
      if (lane == 0) scratch[1][wave] = most;
      __syncthreads();
      for (int w = 0; w < nw; ++w) most = fmaxf(most, scratch[1][w]);
    }
    const float scale = e4m3_scale(most);
    const float inv = 1.0f / scale;
    if (first == 0) scales[row * groups + g] = scale;
    for (int i = first; i < group; i += step) out[row * hidden + g * group + i] = e4m3(y_of(g * group + i) * inv);
  }
}

template <typename E>
int launch_any(void* out, float* scales, const void* x, const void* res, void* res_out, const void* weight,
               int64_t rows, int hidden, int group, const RowMap& xm, float eps, hipStream_t stream) {
  using S = typename E::S;
  auto* o = static_cast<uint8_t*>(out);
  auto* xi = static_cast<const S*>(x);
  auto* wi = static_cast<const S*>(weight);
  const auto gx = static_cast<unsigned>(xm.swapped ? rows / xm.inner : xm.inner);
  const dim3 grid(gx, static_cast<unsigned>(rows / gx));
  if (res != nullptr) {
    norm8_loop_kernel<E, true><<<grid, 256, 0, stream>>>(o, scales, xi, static_cast<const S*>(res),
                                                         static_cast<S*>(res_out), wi, hidden, group, xm, eps);
  } else {
    norm8_loop_kernel<E, false><<<grid, 256, 0, stream>>>(o, scales, xi, nullptr, nullptr, wi, hidden, group, xm, eps);
  }
  return check_launch("rms_norm_fp8 kernel launch");
}

}  // namespace
}  // namespace kl

extern "C" int kl_rms_norm_fp8(kl_dtype dtype, void* out, float* scales, const void* x, const void* residual,
                               void* residual_out, const void* weight, int64_t groups, int64_t rows_per_group,
                               int64_t hidden, int64_t x_group_stride, int64_t x_row_stride, int64_t scale_group,
                               float eps, kl_stream_t stream) {
  using namespace kl;
  if (groups < 0 || rows_per_group < 0 || hidden < 0 || scale_group < 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "rows, hidden and scale_group must be >= 0");
  }
  if (groups == 0 || rows_per_group == 0 || hidden == 0) return ok();
  if (groups > 0x7fffffffLL || rows_per_group > 0x7fffffffLL || groups * rows_per_group > 0x7fffffffLL) {
    return fail(KL_ERR_UNSUPPORTED, "rows must be < 2^31");
  }
  if (hidden > 0x7fffffffLL) return fail(KL_ERR_UNSUPPORTED, "hidden must be < 2^31");
  const bool whole = scale_group == 0 || scale_group == hidden;
  if (!whole && scale_group != 32 && scale_group != 64 && scale_group != 128 && scale_group != 256) {
    return fail(KL_ERR_UNSUPPORTED, "scale_group must be 0 (a scale per row), hidden, 32, 64, 128 or 256");
  }
  if (!whole && hidden % scale_group != 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "hidden must be a multiple of scale_group");
  }
  if (out == nullptr || scales == nullptr || x == nullptr || weight == nullptr) {
    return fail(KL_ERR_INVALID_ARGUMENT, "out, scales, x and weight must be non-null");
  }
  if ((residual == nullptr) != (residual_out == nullptr)) {
    return fail(KL_ERR_INVALID_ARGUMENT, "residual and residual_out go together");
  }
  if ((x_row_stride < hidden && rows_per_group > 1) || (x_group_stride < hidden && groups > 1)) {
    return fail(KL_ERR_INVALID_ARGUMENT, "x_row_stride and x_group_stride must be >= hidden");
  }
  const auto s = reinterpret_cast<hipStream_t>(stream);
  const int h = static_cast<int>(hidden), g = whole ? h : static_cast<int>(scale_group);
  const int64_t rows = groups * rows_per_group;
  const RowMap xm = make_row_map(groups, rows_per_group, x_group_stride, x_row_stride);
  switch (dtype) {
    case KL_DTYPE_F32:
      return launch_any<F32>(out, scales, x, residual, residual_out, weight, rows, h, g, xm, eps, s);
    case KL_DTYPE_F16:
      return launch_any<F16>(out, scales, x, residual, residual_out, weight, rows, h, g, xm, eps, s);
    case KL_DTYPE_BF16:
      return launch_any<BF16>(out, scales, x, residual, residual_out, weight, rows, h, g, xm, eps, s);
  }
  return fail(KL_ERR_UNSUPPORTED, "dtype must be f32, f16 or bf16");
}
