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

// Largest value over the LANES (4 .. 64, run-time) lanes that hold a scale group
// or a narrow row, in every one of them.
__device__ __forceinline__ float lanes_max(float v, int lanes) {
  v = fmaxf(v, dpp<kDppQuadSwap1>(v));
  v = fmaxf(v, dpp<kDppQuadSwap2>(v));
  if (lanes >= 8) v = fmaxf(v, dpp<kDppRowHalfMirror>(v));
  if (lanes >= 16) v = fmaxf(v, dpp<kDppRowRor8>(v));
  if (lanes >= 32) v = max_xor16(v);
  if (lanes >= 64) v = max_xor32(v);
  return v;
}

__device__ __forceinline__ float wave_max(float v) { return max_xor32(max_xor16(row16_max(v))); }

struct SumMax {
  float sum, max;
};

// Sum and largest value over the workgroup, in every thread; wave results are
// joined in wave order.
__device__ __forceinline__ SumMax block_sum_max(float sum, float most, SumMax* scratch) {
  const SumMax w = {wave_sum(sum), wave_max(most)};
  const int nw = blockDim.x >> 6;
  if (__lane_id() == 0) scratch[threadIdx.x >> 6] = w;
  __syncthreads();
  SumMax total = {0.0f, 0.0f};
  for (int i = 0; i < nw; ++i) {
    total.sum += scratch[i].sum;
    total.max = fmaxf(total.max, scratch[i].max);
  }
  return total;
}

// Largest finite |v|. The maximum itself drops NaN; infinities are looked for only
// where there is one (three instructions an element less: see norm8_row).
template <int N>
__device__ __forceinline__ float most_finite(const float (&v)[N]) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) m = fmaxf(m, fabsf(v[j]));
  if (__any(m == INFINITY)) {
    m = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, finite_abs(v[j]));
  }
  return m;
}

// One thread's share of a row, NPACK packs t, t + nt, ..., as in rmsnorm.hip's
// norm_row: loaded once, kept in registers up to the codes. reduce(sum, max) joins
// both over the row's threads. group_lanes: the lanes that hold a scale group, or
// 0 for one scale a row.
//
// max |y| = rstd max |x w|, so a row's scale comes out of the reduction that its
// sum of squares needs anyway, and one barrier gives both (a product x w past
// fp32's range counts as not finite). A group lies in consecutive lanes, and its
// largest value needs no LDS.
//
// What bounds it: HBM for many rows (7 bytes an element of 16 bits with the
// residual), the launch for few. Measured (us, bf16, residual form, three sets of
// tensors in turn): 4,096 x 8,192 42.3 (5.6 TB/s; element by element from memory
// 101), a scale per 128 columns 43.2, 16,384 x 1,024 22.2, 16 x 4,096 4.5. One
// pack a thread instead of two 51.5, four 44; 16 adjacent elements a thread, whose
// codes are one 16-byte store, 48.4; non-temporal stores of the codes 41.5, but the
// projection reads them next.
template <typename E, int VEC, int NPACK, bool HAS_RES, bool ALIGNED, typename Reduce>
__device__ __forceinline__ void norm8_row(uint8_t* out, float* scales, const typename E::S* x, typename E::S* res,
                                          int64_t res_out, const typename E::S* weight, int hidden, int group_lanes,
                                          float eps, int t, int nt, bool live, Reduce&& reduce) {
  using S = typename E::S;
  using P = Pack<S, VEC>;
  const int packs = ALIGNED ? hidden / VEC : (hidden + VEC - 1) / VEC;
  int off[NPACK];
  int skip[NPACK];  // leading elements of the pack that the one before it holds
  bool valid[NPACK];
#pragma unroll
  for (int k = 0; k < NPACK; ++k) {
    const int p = t + k * nt;
    valid[k] = p < packs;
    const int at = (valid[k] ? p : packs - 1) * VEC;
    off[k] = ALIGNED ? at : min(at, hidden - VEC);
    skip[k] = at - off[k];
  }
  P a[NPACK], b[NPACK], w[NPACK];
#pragma unroll
  for (int k = 0; k < NPACK; ++k) {
    a[k] = load_at<ALIGNED, P>(x, off[k]);
    if constexpr (HAS_RES) b[k] = load_at<ALIGNED, P>(res, off[k]);
  }
#pragma unroll
  for (int k = 0; k < NPACK; ++k) w[k] = load_at<ALIGNED, P>(weight, off[k]);
  float sum_sq = 0.0f;
#pragma unroll
  for (int k = 0; k < NPACK; ++k) {
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (HAS_RES) a[k].v[j] = E::from_f32(E::to_f32(a[k].v[j]) + E::to_f32(b[k].v[j]));
      const float f = E::to_f32(a[k].v[j]);
      part += ALIGNED || j >= skip[k] ? f * f : 0.0f;
    }
    sum_sq += valid[k] ? part : 0.0f;
  }
  auto store_residual = [&] {
#pragma unroll
    for (int k = 0; k < NPACK; ++k) {
      if (valid[k] && live) store_at<ALIGNED>(residual_out(res, res_out), off[k], a[k]);
    }
  };
  if constexpr (HAS_RES && ALIGNED) store_residual();
  // x w: every scale and code comes from it.
  float p[NPACK][VEC];
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < NPACK; ++k) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) p[k][j] = E::to_f32(a[k].v[j]) * E::to_f32(w[k].v[j]);
    most = fmaxf(most, most_finite(p[k]));
  }
  const SumMax total = reduce(sum_sq, group_lanes == 0 ? most : 0.0f);
  const float rstd = inv_rms(total.sum, hidden, eps);
  // The packs of an unaligned row overlap: every thread has loaded its own by now.
  if constexpr (HAS_RES && !ALIGNED) store_residual();
  const float row_scale = e4m3_scale(rstd * total.max);
  if (group_lanes == 0 && t == 0 && live) scales[0] = row_scale;
  const float row_inv = 1.0f / row_scale;
#pragma unroll
  for (int k = 0; k < NPACK; ++k) {
    float inv = row_inv;
    if (group_lanes != 0) {
      const float scale = e4m3_scale(rstd * lanes_max(most_finite(p[k]), group_lanes));
      inv = 1.0f / scale;
      const int at = t + k * nt;
      if (valid[k] && live && (at & (group_lanes - 1)) == 0) scales[at / group_lanes] = scale;
    }
    // Two products, not one with rstd * inv, which is past fp32's range for a row
    // of next to nothing. The reciprocal is at most half a step of fp32 off, which
    // moves a code only where y / scale lies within 2^-22 of a border between two.
#pragma unroll
    for (int j = 0; j < VEC; ++j) p[k][j] = (p[k][j] * rstd) * inv;
    if (valid[k] && live) store_codes<ALIGNED>(out, off[k], p[k]);
  }
}

// A workgroup per row.
template <typename E, int NPACK, bool HAS_RES, bool ALIGNED>
__global__ void __launch_bounds__(kMaxThreads)
    norm8_kernel(uint8_t* __restrict__ out, float* __restrict__ scales, const typename E::S* __restrict__ x,
                 typename E::S* __restrict__ res, int64_t res_out, const typename E::S* __restrict__ weight, int hidden,
                 int groups, int group_lanes, RowMap x_rows, float eps) {
  __shared__ SumMax scratch[kMaxThreads / 64];
  int64_t row, x_off;
  x_rows.of_workgroup(&row, &x_off);
  norm8_row<E, 16 / E::kBytes, NPACK, HAS_RES, ALIGNED>(
      out + row * hidden, scales + row * groups, x + x_off, HAS_RES ? res + row * hidden : nullptr, res_out, weight,
      hidden, group_lanes, eps, threadIdx.x, blockDim.x, true,
      [&](float sum, float most) { return block_sum_max(sum, most, scratch); });
}

// Rows of at most a wave's packs: LANES lanes per row, 256 / LANES rows per
// workgroup, as in rmsnorm.hip's rms_norm_rows_kernel.
constexpr int kRowsThreads = 256;

template <typename E, int LANES, bool HAS_RES, bool ALIGNED>
__global__ void __launch_bounds__(kRowsThreads)
    norm8_rows_kernel(uint8_t* __restrict__ out, float* __restrict__ scales, const typename E::S* __restrict__ x,
                      typename E::S* __restrict__ res, int64_t res_out, const typename E::S* __restrict__ weight,
                      int rows, int hidden, int groups, int group_lanes, RowMap x_rows, float eps) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kRowsThreads / LANES) + threadIdx.x / LANES;
  const bool live = r < rows;
  const int64_t row = live ? r : rows - 1;
  norm8_row<E, 16 / E::kBytes, 1, HAS_RES, ALIGNED>(
      out + row * hidden, scales + row * groups, x + x_rows.x_of_row(row), HAS_RES ? res + row * hidden : nullptr,
      res_out, weight, hidden, group_lanes, eps, threadIdx.x % LANES, LANES, live, [](float sum, float most) {
        return SumMax{lanes_sum<LANES>(sum), lanes_max(most, LANES)};
      });
}

// Rows of less than a pack, and rows past the registers of a workgroup (more than 4
// packs per thread: 32,768 elements of 16 bits, 16,384 of fp32; eight packs, their
// products and the weights would spill), element by element: the squares (writing
// the new residual), then each group's largest |y|, then its codes, all read again
// from memory.
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

template <int N>
using IntC = std::integral_constant<int, N>;

constexpr int kRowsMaxPacks = 64;   // widest row of norm8_rows_kernel: a pack per lane of a wave
constexpr int kMaxPacks = 4;        // per thread of norm8_kernel
constexpr int kPacksPerThread = 2;  // aimed at beyond (rmsnorm.hip has the measurements)

template <typename E, bool HAS_RES>
int launch_typed(uint8_t* out, float* scales, const typename E::S* x, typename E::S* res, typename E::S* res_out,
                 const typename E::S* w, int64_t rows, int hidden, int group, const RowMap& xm, float eps,
                 hipStream_t stream) {
  constexpr int VEC = 16 / E::kBytes;
  const bool whole = group == hidden;
  const int groups = hidden / group, group_lanes = whole ? 0 : group / VEC;
  const int64_t rw = reinterpret_cast<intptr_t>(res_out) - reinterpret_cast<intptr_t>(res);
  const bool aligned = hidden % VEC == 0 && xm.row_stride % VEC == 0 && xm.group_stride % VEC == 0 &&
                       aligned16(out) && aligned16(x) && aligned16(w) && aligned16(res) && aligned16(res_out);
  const int packs = static_cast<int>(cdiv(hidden, VEC));
  const auto gx = static_cast<unsigned>(xm.swapped ? rows / xm.inner : xm.inner);
  const dim3 grid(gx, static_cast<unsigned>(rows / gx));
  const int threads = static_cast<int>(
      std::min<int64_t>(kMaxThreads, std::max<int64_t>(64, cdiv(cdiv(packs, kPacksPerThread), 64) * 64)));
  const int npack = static_cast<int>(cdiv(packs, threads));
  // A grid of 2^32 threads and more along x wraps without an error.
  const bool narrow = hidden >= VEC && packs <= kRowsMaxPacks;
  const int row_threads = !narrow ? kMaxThreads : packs <= 4 ? 4 : packs <= 8 ? 8 : packs <= 16 ? 16 : packs <= 32 ? 32 : 64;
  if ((narrow ? rows : static_cast<int64_t>(gx)) * row_threads > 0xffffffffLL - kRowsThreads) {
    return fail(KL_ERR_UNSUPPORTED, "too many rows for one launch");
  }
  auto rows_kernel = [&](auto lanes, auto al) {
    constexpr int L = decltype(lanes)::value;
    norm8_rows_kernel<E, L, HAS_RES, decltype(al)::value>
        <<<static_cast<unsigned>(cdiv(rows, kRowsThreads / L)), kRowsThreads, 0, stream>>>(
            out, scales, x, res, rw, w, static_cast<int>(rows), hidden, groups, group_lanes, xm, eps);
  };
  auto wide_kernel = [&](auto np, auto al) {
    norm8_kernel<E, decltype(np)::value, HAS_RES, decltype(al)::value><<<grid, threads, 0, stream>>>(
        out, scales, x, res, rw, w, hidden, groups, group_lanes, xm, eps);
  };
  auto with_alignment = [&](auto al) {
    if (packs <= 4) {
      rows_kernel(IntC<4>{}, al);
    } else if (packs <= 8) {
      rows_kernel(IntC<8>{}, al);
    } else if (packs <= 16) {
      rows_kernel(IntC<16>{}, al);
    } else if (packs <= 32) {
      rows_kernel(IntC<32>{}, al);
    } else if (packs <= kRowsMaxPacks) {
      rows_kernel(IntC<64>{}, al);
    } else if (npack <= 2) {
      wide_kernel(IntC<2>{}, al);
    } else {
      wide_kernel(IntC<kMaxPacks>{}, al);
    }
  };
  if (hidden < VEC || npack > kMaxPacks) {
    norm8_loop_kernel<E, HAS_RES><<<grid, hidden < VEC ? 64 : kMaxThreads, 0, stream>>>(
        out, scales, x, res, res_out, w, hidden, group, xm, eps);
  } else if (aligned) {
    with_alignment(std::true_type{});
  } else {
    with_alignment(std::false_type{});
  }
  return check_launch("rms_norm_fp8 kernel launch");
}

template <typename E>
int launch_any(void* out, float* scales, const void* x, const void* res, void* res_out, const void* weight,
               int64_t rows, int hidden, int group, const RowMap& xm, float eps, hipStream_t stream) {
  using S = typename E::S;
  auto* o = static_cast<uint8_t*>(out);
  auto* xi = static_cast<const S*>(x);
  auto* wi = static_cast<const S*>(weight);
  auto* r = static_cast<S*>(const_cast<void*>(res));  // read only, but for the in-place form
  return res ? launch_typed<E, true>(o, scales, xi, r, static_cast<S*>(res_out), wi, rows, hidden, group, xm, eps, stream)
             : launch_typed<E, false>(o, scales, xi, nullptr, nullptr, wi, rows, hidden, group, xm, eps, stream);
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
