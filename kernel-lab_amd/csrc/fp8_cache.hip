// The paged FP8 cache with a scale per page and KV head: writing new tokens into
// it (append) and choosing the pages a query attends (select).
//
// A page's codes c stand for scale * value(c). k_scale and v_scale are
// [num_pages, num_kv_heads]; k_bounds, [num_pages, num_kv_heads, 2, head_dim],
// holds the smallest and the largest code that the page's keys have in each
// dimension, in units of the page's k_scale.
#include <algorithm>
#include <type_traits>

#include "fp8_quant.h"
#include "hip_common.h"
#include "kl_internal.h"

namespace kl {
namespace {

// -------------------------------------------------------------------- append
//
// Sequence b's new tokens are rows offsets[b] .. offsets[b + 1] - 1 of k and v
// (row b alone without offsets) and take positions seq_lens[b] - n .. seq_lens[b] - 1.
// On each page they reach,
//   new   = max(max |x| / 448, 2^-126) over the finite new values of the page and head
//   scale = new, or max(scale, new) where tokens before them are on the page
//   c     = e4m3((value(c) * old scale) / scale) for those, where the scale grew
//   c     = e4m3(x / scale) for the new ones.
// Rounding is monotone, so the bounds of codes that are rounded again are their
// own bounds rounded again.
struct AppendArgs {
  const void* x[2];  // k, v
  int64_t token_stride[2], head_stride[2];
  uint8_t* cache[2];
  float* scale[2];
  uint8_t* bounds;  // null: not kept
  const int32_t* table;
  int64_t bt_stride;
  const int32_t* seq_lens;
  const int32_t* offsets;  // null: one token a sequence
  int tokens, batch, heads, dim, page, max_pages, num_pages;
};

// What a workgroup writes: new tokens [t0, t1) of a page, from row `row` on.
struct PageTile {
  int64_t phys;
  int t0, t1;
  int64_t row;
};

// Tile `i` of the launch. Without offsets it is sequence i's one token. With
// them sequence b has the tiles from offsets[b] / page + 2 b on, one for each
// page it reaches: n tokens reach at most n / page + 2 pages, so the next
// sequence's first tile lies behind its last. False where the tile has no
// tokens, and for sequences whose lengths, offsets or pages are out of range,
// which are left alone.
__device__ __forceinline__ bool page_tile(const AppendArgs& a, int i, PageTile* t) {
  int b = i, off = i, n = 1, at = 0;
  if (a.offsets != nullptr) {
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.offsets[mid] / a.page + 2 * mid <= i) {
        lo = mid;
      } else {
        hi = mid - 1;
      }
    }
    b = lo;
    off = a.offsets[b];
    const int end = a.offsets[b + 1];
    if (off < 0 || end > a.tokens || end <= off) return false;
    n = end - off;
    at = i - (off / a.page + 2 * b);
  }
  const int len = a.seq_lens[b];
  const int start = len - n;
  if (start < 0 || at < 0) return false;
  const int64_t col = start / a.page + static_cast<int64_t>(at);
  if (col * a.page >= len || col >= a.max_pages) return false;
  const int phys = a.table[b * a.bt_stride + col];
  if (phys < 0 || phys >= a.num_pages) return false;
  const int64_t base = col * a.page;
  t->phys = phys;
  t->t0 = static_cast<int>(max(static_cast<int64_t>(start) - base, static_cast<int64_t>(0)));
  t->t1 = static_cast<int>(min(static_cast<int64_t>(len) - base, static_cast<int64_t>(a.page)));
  t->row = off + (base + t->t0 - start);
  return true;
}

__device__ __forceinline__ float wave_max(float v) { return max_xor32(max_xor16(row16_max(v))); }

constexpr int kAppendThreads = 256;

// A workgroup per (tile, KV head, K or V), element by element.
template <typename E>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  using S = typename E::S;
  __shared__ float most_of[kAppendThreads / 64];
  PageTile t;
  if (!page_tile(a, static_cast<int>(blockIdx.x), &t)) return;
  const int h = blockIdx.y, which = blockIdx.z;
  const S* x = static_cast<const S*>(a.x[which]) + t.row * a.token_stride[which] + h * a.head_stride[which];
  const int64_t row_bytes = static_cast<int64_t>(a.heads) * a.dim;
  uint8_t* codes = a.cache[which] + t.phys * a.page * row_bytes + static_cast<int64_t>(h) * a.dim;
  const int n = (t.t1 - t.t0) * a.dim;
  auto x_of = [&](int i) { return E::to_f32(x[(i / a.dim) * a.token_stride[which] + i % a.dim]); };
  float most = 0.0f;
  for (int i = threadIdx.x; i < n; i += kAppendThreads) most = fmaxf(most, finite_abs(x_of(i)));
  most = wave_max(most);
  if (__lane_id() == 0) most_of[threadIdx.x >> 6] = most;
  float* scale_at = a.scale[which] + t.phys * a.heads + h;
  const float old = *scale_at;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / 64; ++w) most = fmaxf(most, most_of[w]);
  const bool held = t.t0 > 0;
  const float fresh = e4m3_scale(most);
  const float scale = held ? fmaxf(old, fresh) : fresh;
  const bool grown = held && scale > old;
  if (threadIdx.x == 0) *scale_at = scale;
  auto again = [&](uint8_t c) { return e4m3((e4m3_value(c) * old) / scale); };
  if (grown) {
    for (int i = threadIdx.x; i < t.t0 * a.dim; i += kAppendThreads) {
      uint8_t* c = codes + (i / a.dim) * row_bytes + i % a.dim;
      *c = again(*c);
    }
  }
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    codes[(t.t0 + i / a.dim) * row_bytes + i % a.dim] = e4m3(x_of(i) / scale);
  }
  if (which == 0 && a.bounds != nullptr) {
    uint8_t* edge = a.bounds + (t.phys * a.heads + h) * 2 * a.dim;
    for (int d = threadIdx.x; d < a.dim; d += kAppendThreads) {
      // NaN codes take no part.
      float lo = kE4M3Max, hi = -kE4M3Max;
      if (held) {
        lo = fminf(lo, e4m3_value(grown ? again(edge[d]) : edge[d]));
        hi = fmaxf(hi, e4m3_value(grown ? again(edge[a.dim + d]) : edge[a.dim + d]));
      }
      for (int i = 0; i < t.t1 - t.t0; ++i) {
        const float c = e4m3_value(e4m3(x_of(i * a.dim + d) / scale));
        lo = fminf(lo, c);
        hi = fmaxf(hi, c);
      }
      edge[d] = e4m3(lo);
      edge[a.dim + d] = e4m3(hi);
    }
  }
}

// -------------------------------------------------------------------- select
//
// The largest q.k that a key within the page's bounds can have, for the query
// head of the KV head's group where it is largest:
//   score = f32(k_scale * max_g sum_d max(q_gd lo_d, q_gd hi_d))
// The sum is formed in 64 bits, where it is exact for queries whose values span
// less than about 2^30 (a product has 15 bits at most), so the order of its
// terms does not decide which of two near scores is larger.
struct SelectArgs {
  const void* q;
  const uint8_t* bounds;
  const float* scale;
  const int32_t* table;
  const int32_t* seq_lens;
  int64_t bt_stride;
  float* scores;  // [batch, kv heads, max_pages]
  int32_t* out_table;
  int32_t* out_lens;
  int batch, heads, group, dim, page, max_pages, keep, first, last;
};

__device__ __forceinline__ int select_len(const SelectArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  const int64_t len = a.seq_lens[b];
  return static_cast<int>(max(static_cast<int64_t>(0), min(len, cap)));
}

// A page's score as a key that orders like it: pinned pages before all others, a
// NaN like the largest finite score.
__device__ __forceinline__ uint32_t score_key(float s) {
  s = s < 0x1.fffffep127f ? s : 0x1.fffffep127f;
  const uint32_t u = __builtin_bit_cast(uint32_t, s == 0.0f ? 0.0f : s);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A wave per page.
template <typename E>
__global__ void __launch_bounds__(256) score_kernel(const SelectArgs a) {
  const int64_t unit = blockIdx.y;
  const int b = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads);
  const int pages = (select_len(a, b) + a.page - 1) / a.page;
  const int p = blockIdx.x * 4 + wave_id();
  if (p >= pages) return;
  const int64_t phys = a.table[b * a.bt_stride + p];
  const uint8_t* edge = a.bounds + (phys * a.heads + h) * 2 * a.dim;
  const typename E::S* q = static_cast<const typename E::S*>(a.q) + unit * a.group * a.dim;
  double best = -INFINITY;
  for (int g = 0; g < a.group; ++g) {
    double sum = 0.0;
    for (int d = __lane_id(); d < a.dim; d += 64) {
      const float qv = E::to_f32(q[g * a.dim + d]);
      sum += static_cast<double>(qv) * static_cast<double>(e4m3_value(qv < 0.0f ? edge[d] : edge[a.dim + d]));
    }
    for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
    best = sum > best || sum != sum ? sum : best;
  }
  if (__lane_id() == 0) {
    a.scores[unit * a.max_pages + p] = static_cast<float>(best * static_cast<double>(a.scale[phys * a.heads + h]));
  }
}

constexpr int kPickThreads = 256;

// A workgroup per (sequence, KV head): the keep-th largest key by four passes of
// eight bits over a histogram, then the pages above it, and as many of its equals
// as are wanted, lowest first, in ascending order.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const SelectArgs a) {
  __shared__ int hist[256];
  __shared__ int wave_count[2][kPickThreads / 64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_want;
  const int64_t unit = blockIdx.x;
  const int b = static_cast<int>(unit / a.heads);
  const int len = select_len(a, b);
  const int pages = (len + a.page - 1) / a.page;
  const int kept = min(pages, a.keep);
  const float* scores = a.scores + unit * a.max_pages;
  const int32_t* table = a.table + b * a.bt_stride;
  int32_t* out = a.out_table + unit * a.keep;
  for (int i = kept + threadIdx.x; i < a.keep; i += kPickThreads) out[i] = 0;
  if (threadIdx.x == 0) a.out_lens[unit] = kept > 0 ? (kept - 1) * a.page + (len - (pages - 1) * a.page) : 0;
  if (pages <= a.keep) {
    for (int i = threadIdx.x; i < pages; i += kPickThreads) out[i] = table[i];
    return;
  }
  auto key_of = [&](int p) -> uint32_t {
    return p < a.first || p >= pages - a.last ? 0xffffffffu : score_key(scores[p]);
  };
  uint32_t prefix = 0;
  int want = kept;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < pages; p += kPickThreads) {
      const uint32_t key = key_of(p);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = want, bin = 255;
      while (bin > 0 && hist[bin] < left) left -= hist[bin--];
      s_prefix = prefix | (static_cast<uint32_t>(bin) << shift);
      s_want = left;
    }
    __syncthreads();
    prefix = s_prefix;
    want = s_want;
    __syncthreads();
  }
  // prefix is now the smallest key kept, `want` how many pages that have it.
  const int lane = __lane_id(), wave = wave_id();
  int done = 0, ties = 0;
  for (int p0 = 0; p0 < pages; p0 += kPickThreads) {
    const int p = p0 + threadIdx.x;
    const uint32_t key = p < pages ? key_of(p) : 0;
    const bool tie = p < pages && key == prefix;
    const uint64_t tie_mask = __ballot(tie);
    if (lane == 0) wave_count[0][wave] = __builtin_popcountll(tie_mask);
    __syncthreads();
    int ties_before = ties;
    for (int w = 0; w < kPickThreads / 64; ++w) {
      if (w < wave) ties_before += wave_count[0][w];
      ties += wave_count[0][w];
    }
    const uint64_t below = (1ull << lane) - 1;
    const bool take = (p < pages && key > prefix) || (tie && ties_before + __builtin_popcountll(tie_mask & below) < want);
    const uint64_t mask = __ballot(take);
    if (lane == 0) wave_count[1][wave] = __builtin_popcountll(mask);
    __syncthreads();
    int at = done + __builtin_popcountll(mask & below);
    for (int w = 0; w < kPickThreads / 64; ++w) {
      if (w < wave) at += wave_count[1][w];
      done += wave_count[1][w];
    }
    if (take && at < a.keep) out[at] = table[p];
    __syncthreads();
  }
}

bool head_dim_ok(int dim) { return dim == 64 || dim == 128 || dim == 256; }

}  // namespace
}  // namespace kl

extern "C" int kl_append_kv_fp8(kl_dtype dtype, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                void* k_bounds, const void* k, const void* v, int64_t k_token_stride,
                                int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                const int32_t* block_table, const int32_t* seq_lens, const int32_t* new_offsets,
                                int64_t tokens, int batch, int num_kv_heads, int head_dim, int page_size,
                                int num_pages, int64_t block_table_stride, int max_pages, kl_stream_t stream) {
  using namespace kl;
  if (batch < 0 || tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || num_pages < 0 || max_pages < 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "tokens, batch, heads, head_dim, page_size, num_pages and max_pages must be positive");
  }
  if (dtype != KL_DTYPE_F32 && dtype != KL_DTYPE_F16 && dtype != KL_DTYPE_BF16) {
    return fail(KL_ERR_UNSUPPORTED, "dtype must be f32, f16 or bf16");
  }
  if (!head_dim_ok(head_dim) || page_size % 16 != 0) {
    return fail(KL_ERR_UNSUPPORTED, "an FP8 cache needs head_dim 64, 128 or 256 and page_size a multiple of 16");
  }
  if (new_offsets == nullptr && tokens != batch) {
    return fail(KL_ERR_INVALID_ARGUMENT, "without new_offsets every sequence has one token");
  }
  if (batch == 0 || tokens == 0 || max_pages == 0 || num_pages == 0) return ok();
  if (!k_cache || !v_cache || !k_scale || !v_scale || !k || !v || !block_table || !seq_lens) {
    return fail(KL_ERR_INVALID_ARGUMENT, "caches, scales, k, v, block_table and seq_lens must be non-null");
  }
  if (block_table_stride < max_pages && batch > 1) {
    return fail(KL_ERR_INVALID_ARGUMENT, "block_table_stride must be >= max_pages");
  }
  const int64_t tiles = new_offsets == nullptr ? batch : tokens / page_size + 2 * static_cast<int64_t>(batch);
  if (tokens > 0x7fffffffLL || tiles > 0x7fffffffLL / kAppendThreads || num_kv_heads > 65535) {
    return fail(KL_ERR_UNSUPPORTED, "too many tokens, sequences or heads for one launch");
  }
  AppendArgs a;
  a.x[0] = k;
  a.x[1] = v;
  a.token_stride[0] = k_token_stride;
  a.token_stride[1] = v_token_stride;
  a.head_stride[0] = k_head_stride;
  a.head_stride[1] = v_head_stride;
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.bounds = static_cast<uint8_t*>(k_bounds);
  a.table = block_table;
  a.bt_stride = block_table_stride;
  a.seq_lens = seq_lens;
  a.offsets = new_offsets;
  a.tokens = static_cast<int>(tokens);
  a.batch = batch;
  a.heads = num_kv_heads;
  a.dim = head_dim;
  a.page = page_size;
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(num_kv_heads), 2);
  const auto s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case KL_DTYPE_F32:
      append_kernel<F32><<<grid, kAppendThreads, 0, s>>>(a);
      break;
    case KL_DTYPE_F16:
      append_kernel<F16><<<grid, kAppendThreads, 0, s>>>(a);
      break;
    case KL_DTYPE_BF16:
      append_kernel<BF16><<<grid, kAppendThreads, 0, s>>>(a);
      break;
  }
  return check_launch("append_kv_fp8 kernel launch");
}

extern "C" int kl_select_pages_workspace(int batch, int num_kv_heads, int max_pages, size_t* out_workspace) {
  using namespace kl;
  if (batch < 0 || num_kv_heads <= 0 || max_pages < 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "batch, num_kv_heads and max_pages must be positive");
  }
  if (out_workspace) {
    *out_workspace = static_cast<size_t>(batch) * static_cast<size_t>(num_kv_heads) * static_cast<size_t>(max_pages) * 4;
  }
  return ok();
}

extern "C" int kl_select_pages(kl_dtype dtype, int32_t* out_table, int32_t* out_lens, const void* q,
                               const void* k_bounds, const float* k_scale, const int32_t* block_table,
                               const int32_t* seq_lens, int batch, int num_q_heads, int num_kv_heads, int head_dim,
                               int page_size, int64_t block_table_stride, int max_pages, int num_selected,
                               int first_pages, int last_pages, void* workspace, size_t workspace_bytes,
                               kl_stream_t stream) {
  using namespace kl;
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || max_pages < 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "batch, heads, head_dim, page_size and max_pages must be positive");
  }
  if (num_q_heads % num_kv_heads != 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "num_q_heads must be a multiple of num_kv_heads");
  }
  if (dtype != KL_DTYPE_F16 && dtype != KL_DTYPE_BF16) {
    return fail(KL_ERR_UNSUPPORTED, "an FP8 cache needs fp16 or bf16 queries");
  }
  if (!head_dim_ok(head_dim) || page_size % 16 != 0) {
    return fail(KL_ERR_UNSUPPORTED, "an FP8 cache needs head_dim 64, 128 or 256 and page_size a multiple of 16");
  }
  if (first_pages < 0 || last_pages < 1 || num_selected < 1 || first_pages > num_selected - last_pages) {
    return fail(KL_ERR_INVALID_ARGUMENT, "first_pages >= 0 and last_pages >= 1 must fit num_selected");
  }
  const int64_t units = static_cast<int64_t>(batch) * num_kv_heads;
  if (units > 65535 || static_cast<int64_t>(max_pages) * page_size > 0x7fffffffLL ||
      static_cast<int64_t>(num_selected) * page_size > 0x7fffffffLL) {
    return fail(KL_ERR_UNSUPPORTED, "more than 65535 (sequence, KV head) pairs, or tables past 2^31 tokens");
  }
  if (batch == 0) return ok();
  if (max_pages < 1) return fail(KL_ERR_INVALID_ARGUMENT, "max_pages must be >= 1");
  if (!out_table || !out_lens || !q || !k_bounds || !k_scale || !block_table || !seq_lens) {
    return fail(KL_ERR_INVALID_ARGUMENT, "outputs, q, k_bounds, k_scale, block_table and seq_lens must be non-null");
  }
  if (block_table_stride < max_pages && batch > 1) {
    return fail(KL_ERR_INVALID_ARGUMENT, "block_table_stride must be >= max_pages");
  }
  size_t need = 0;
  kl_select_pages_workspace(batch, num_kv_heads, max_pages, &need);
  if (workspace == nullptr || workspace_bytes < need) {
    return fail(KL_ERR_WORKSPACE, "workspace smaller than kl_select_pages_workspace reported");
  }
  SelectArgs a;
  a.q = q;
  a.bounds = static_cast<const uint8_t*>(k_bounds);
  a.scale = k_scale;
  a.table = block_table;
  a.seq_lens = seq_lens;
  a.bt_stride = block_table_stride;
  a.scores = static_cast<float*>(workspace);
  a.out_table = out_table;
  a.out_lens = out_lens;
  a.batch = batch;
  a.heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.dim = head_dim;
  a.page = page_size;
  a.max_pages = max_pages;
  a.keep = num_selected;
  a.first = first_pages;
  a.last = last_pages;
  const auto s = reinterpret_cast<hipStream_t>(stream);
  if (max_pages > num_selected) {  // else every page is kept
    const dim3 grid(static_cast<unsigned>(cdiv(max_pages, 4)), static_cast<unsigned>(units));
    if (dtype == KL_DTYPE_F16) {
      score_kernel<F16><<<grid, 256, 0, s>>>(a);
    } else {
      score_kernel<BF16><<<grid, 256, 0, s>>>(a);
    }
    const int st = check_launch("select_pages score kernel launch");
    if (st != KL_OK) return st;
  }
  pick_kernel<<<static_cast<unsigned>(units), kPickThreads, 0, s>>>(a);
  return check_launch("select_pages kernel launch");
}
