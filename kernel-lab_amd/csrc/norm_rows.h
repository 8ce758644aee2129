// What the RMSNorm kernels share: where a call's rows lie, and sums over a row's
// lanes.
#pragma once

#include "hip_common.h"
#include "packs.h"

namespace kl {
namespace {

constexpr int kMaxThreads = 1024;

// Where x's rows are, in elements: row i of group g at g * group_stride + i *
// row_stride, inner rows to a group; out and the residuals hold row g * inner +
// i there. A strided view of two leading dimensions (the heads of one part of a
// fused projection) is read in place; copied first, 2,048 x 32 heads of 128
// bf16 took 15.7 us a call, the copy 9.7 of them, and 6.9 read in place (calls back
// to back; the kernel alone traces at 7.3 with the profiler's gaps).
//
// A workgroup per row takes (i, g) from the grid, the larger of the two counts
// along x: a division before the first load cost the large sizes 2 %.
struct RowMap {
  int64_t inner, row_stride, group_stride;
  int swapped;  // the grid's x counts groups
  __device__ __forceinline__ void of_workgroup(int64_t* row, int64_t* x_off) const {
    const int64_t i = swapped ? blockIdx.y : blockIdx.x;
    const int64_t g = swapped ? blockIdx.x : blockIdx.y;
    *row = g * inner + i;
    *x_off = g * group_stride + i * row_stride;
  }
  __device__ __forceinline__ int64_t x_of_row(int64_t r) const {
    if (group_stride == 0) return r * row_stride;  // one group
    const uint32_t g = static_cast<uint32_t>(r) / static_cast<uint32_t>(inner);
    return g * group_stride + (r - g * inner) * row_stride;
  }
};

// The rows of a call: one row per group, or one group, needs a single stride.
// The grid's y is at most 65,535, which the smaller of two counts whose product
// is below 2^31 meets.
inline RowMap make_row_map(int64_t groups, int64_t rows_per_group, int64_t group_stride, int64_t row_stride) {
  if (groups == 1) return RowMap{rows_per_group, row_stride, 0, 0};
  if (rows_per_group == 1) return RowMap{groups, group_stride, 0, 0};
  return RowMap{rows_per_group, row_stride, group_stride, groups > rows_per_group};
}

__device__ __forceinline__ float inv_rms(float sum_sq, int hidden, float eps) {
  // Division and square root are IEEE-rounded here (no fast-math), matching
  // torch.rsqrt on the CPU, which computes 1 / sqrt(x).
  return 1.0f / sqrtf(sum_sq / static_cast<float>(hidden) + eps);
}

// The new residual's place, `bytes` past the old one's: 0 in place. Reached
// from the same pointer, so that pointer can be __restrict__ in both forms
// (without it the large sizes lost 1 %: the weights' loads went ahead of the
// residual's).
template <typename S>
__device__ __forceinline__ S* residual_out(S* res, int64_t bytes) {
  return reinterpret_cast<S*>(reinterpret_cast<char*>(res) + bytes);
}

// Sum over the LANES (4 .. 64) lanes of a row, in every one of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<kDppQuadSwap1>(v);
  v += dpp<kDppQuadSwap2>(v);
  if constexpr (LANES >= 8) v += dpp<kDppRowHalfMirror>(v);  // the quads of each half row agree, so a mirror is a swap
  if constexpr (LANES >= 16) v += dpp<kDppRowRor8>(v);
  if constexpr (LANES >= 32) v = sum_xor16(v);
  if constexpr (LANES >= 64) v = sum_xor32(v);
  return v;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace kl
