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
#include "packs.h"

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
  int unit_blocks;  // workgroups a tile
};

// What a workgroup writes: new tokens [t0, t1) of a page, from row `row` on. The page
// is as the table has it, in range or not.
struct PageTile {
  int phys;
  int t0, t1;
  int64_t row;
};

// Tile `i` of the launch. Without offsets it is sequence i's one token. With
// them sequence b has the tiles from offsets[b] / page + 2 b on, one for each
// page it reaches: n tokens reach at most n / page + 2 pages, so the next
// sequence's first tile lies behind its last. False where the tile has no
// tokens, and for sequences whose lengths or offsets are out of range, which are
// left alone. Wave-uniform: the sequence is found by all lanes at once,
// 64 offsets at a time.
__device__ __forceinline__ bool page_tile(const AppendArgs& a, int i, PageTile* t) {
  int b = i, off = i, n = 1, at = 0;
  if (a.offsets != nullptr) {
    int before = 0;  // sequences whose first tile is not behind this one
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const int s = b0 + __lane_id();
      const bool reached = s < a.batch && a.offsets[s] / a.page + 2 * static_cast<int64_t>(s) <= i;
      const int count = __builtin_popcountll(__ballot(reached));
      before += count;
      if (count < 64) break;
    }
    b = before > 0 ? before - 1 : 0;
    off = as_constant(a.offsets)[b];
    const int end = as_constant(a.offsets)[b + 1];
    if (off < 0 || end > a.tokens || end <= off) return false;
    n = end - off;
    at = i - (off / a.page + 2 * b);
  }
  const int len = as_constant(a.seq_lens)[b];
  const int start = len - n;
  if (start < 0 || at < 0) return false;
  const int64_t col = start / a.page + static_cast<int64_t>(at);
  if (col * a.page >= len || col >= a.max_pages) return false;
  const int64_t base = col * a.page;
  t->phys = as_constant(a.table)[b * a.bt_stride + col];
  t->t0 = static_cast<int>(max(static_cast<int64_t>(start) - base, static_cast<int64_t>(0)));
  t->t1 = static_cast<int>(min(static_cast<int64_t>(len) - base, static_cast<int64_t>(a.page)));
  t->row = off + (base + t->t0 - start);
  return true;
}

// x / scale for many x of one scale, correctly rounded. Markstein's: a product with
// the rounded reciprocal, and one step that adds its remainder; with a correctly
// rounded reciprocal the result is the division's, in four instructions instead of
// ten. The remainder has to be exact, so scale and x are first moved from the ends of
// fp32's range by a power of two. An x that is not finite gives NaN.
struct Over {
  float pre, scale, inv;
  __device__ __forceinline__ explicit Over(float s) {
    pre = s < 0x1p-90f ? 0x1p100f : s > 0x1p90f ? 0x1p-100f : 1.0f;
    scale = s * pre;
    inv = 1.0f / scale;
  }
  __device__ __forceinline__ float operator()(float x) const {
    x *= pre;
    const float q = x * inv;
    return fmaf(fmaf(-q, scale, x), inv, q);
  }
};

// The smaller of x in this lane and the lane 32 (16) below or above it, in the lower
// half (even rows), and of y in the upper half (odd rows): v_permlane32_swap
// exchanges x's upper half with y's lower one.
__device__ __forceinline__ float min_swap32(float x, float y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
  return fminf(__builtin_bit_cast(float, static_cast<unsigned>(r[0])), __builtin_bit_cast(float, static_cast<unsigned>(r[1])));
}
__device__ __forceinline__ float min_swap16(float x, float y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
  return fminf(__builtin_bit_cast(float, static_cast<unsigned>(r[0])), __builtin_bit_cast(float, static_cast<unsigned>(r[1])));
}

// f, or NaN where it is infinite: the minimum and maximum instructions pass over it.
__device__ __forceinline__ float finite_or_nan(float f) { return fmaf(f, 0.0f, f); }

constexpr int kAppendWaves = 4;
constexpr int kAppendThreads = kAppendWaves * 64;

// A wave per (tile, KV head, K or V). A lane holds 16-byte packs of the tile's
// tokens: the LPT lanes of a token read its head_dim contiguously, TPI tokens to a
// load. Up to HOLD packs a lane stay in registers between the page's largest
// magnitude and its codes; a longer tile is read again.
//
// What bounds it: HBM for prompts (3 bytes an element of 16 bits), the launch for
// single tokens. Measured (us, 8 chunks of 2,048 .. 4,096 tokens, 8 heads of 128 bf16
// read from a fused projection, pages of 16, with bounds): 35.8 (4.5 TB/s), element by
// element 181; IEEE divisions and every lane reducing all bounds 53.5; K and V in
// workgroups of their own 42.3 (K's are longer, and the XCDs take workgroups in
// turn); tiles of one head group far apart in the launch 43.5; default-policy loads 3 to
// 10 % more; four heads one after the other in a wave, the next one loading, 51.
template <typename E, int D, int HOLD, bool ALIGNED>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  using S = typename E::S;
  constexpr int VEC = 16 / E::kBytes;
  constexpr int LPT = D / VEC;  // 8 .. 64
  constexpr int TPI = 64 / LPT;
  using P = Pack<S, VEC>;
  const uint32_t tile = blockIdx.x / static_cast<uint32_t>(a.unit_blocks);
  PageTile t;
  if (!page_tile(a, static_cast<int>(tile), &t)) return;
  const int lane = __lane_id();
  const int tok = lane / LPT, dim = VEC * (lane % LPT);
  const int n = t.t1 - t.t0;
  const int packs = (n + TPI - 1) / TPI;
  const bool once = packs <= HOLD;
  const bool held = t.t0 > 0;
  const int unit = static_cast<int>(blockIdx.x - tile * a.unit_blocks) * kAppendWaves + wave_id();
  if (unit >= 2 * a.heads) return;
  const int which = unit & 1, h = unit >> 1;
  const int64_t x_row = which ? a.token_stride[1] : a.token_stride[0];
  const S* x = static_cast<const S*>(which ? a.x[1] : a.x[0]) + t.row * x_row +
               h * (which ? a.head_stride[1] : a.head_stride[0]) + dim;
  // Pack i of the tile; a lane past the last token reads that again, which changes
  // neither the largest magnitude nor the bounds.
  auto load = [&](int i) {
    const S* p = x + min(i * TPI + tok, n - 1) * x_row;
    if constexpr (ALIGNED) {
      return __builtin_bit_cast(P, global_load16_nt(reinterpret_cast<const char*>(p)));
    } else {
      return load_at<false, P>(p, 0);
    }
  };
  P v[HOLD] = {};
  auto load_all = [&](int base) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (base + i < packs) v[i] = load(base + i);
    }
  };
  load_all(0);  // on its way while the page's entry arrives
  if (t.phys < 0 || t.phys >= a.num_pages) return;

  const int64_t row_bytes = static_cast<int64_t>(a.heads) * D;
  const int64_t head = static_cast<int64_t>(t.phys) * a.heads + h;
  uint8_t* codes = (which ? a.cache[1] : a.cache[0]) + t.phys * (a.page * row_bytes) + static_cast<int64_t>(h) * D;
  float* scale_at = (which ? a.scale[1] : a.scale[0]) + head;
  const bool bounded = which == 0 && a.bounds != nullptr;
  // The page's bounds, D smallest then D largest codes: this lane's `words` of four
  // (see the end), its sign +1 for smallest and -1 for largest.
  constexpr int SETS = LPT == 64 ? 2 : 1;
  constexpr int WORDS = LPT == 32 ? VEC / 4 : 1;  // of a set
  const bool upper = LPT < 64 && lane >= 32;
  uint32_t* edge = nullptr;
  bool edge_lane = false;
  if (bounded) {
    edge = reinterpret_cast<uint32_t*>(a.bounds + head * 2 * D + (upper ? D : 0) + dim +
                                       (VEC == 8 && LPT <= 16 ? 4 * ((lane >> 4) & 1) : 0));
    edge_lane = !(LPT == 16 && VEC == 4 && (lane & 16) != 0) && !(LPT == 8 && (lane & 8) != 0);
  }
  // What the page has.
  float old = 0.0f;
  uint32_t held_edge[SETS][WORDS] = {};
  if (held) {
    old = *scale_at;
    if (edge_lane) {
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) held_edge[s][i] = edge[s * (D / 4) + i];
      }
    }
  }

  // Largest magnitude of the finite values, or, in each dimension, their smallest
  // (end[0]) and the smallest of their negatives (end[1]).
  float end[2][VEC];
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < VEC; ++j) end[0][j] = end[1][j] = INFINITY;
  auto scan = [&](int base) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (base + i < packs) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float f = finite_or_nan(E::to_f32(v[i].v[j]));
          if (bounded) {
            end[0][j] = fminf(end[0][j], f);
            end[1][j] = fminf(end[1][j], -f);
          } else {
            most = fmaxf(most, fabsf(f));
          }
        }
      }
    }
  };
  scan(0);
  for (int base = HOLD; base < packs; base += HOLD) {
    load_all(base);
    scan(base);
  }
  if (bounded) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) most = fmaxf(most, fmaxf(finite_abs(end[0][j]), finite_abs(end[1][j])));
  }
  most = max_xor32(max_xor16(row16_max(most)));
  // The packs stay packed until here: widened once for both their scan and their
  // codes (the compiler's choice otherwise) they would take twice the registers.
#pragma unroll
  for (int i = 0; i < HOLD; ++i) {
    u32x4 r = __builtin_bit_cast(u32x4, v[i]);
    asm volatile("" : "+v"(r));
    v[i] = __builtin_bit_cast(P, r);
  }

  const float fresh = e4m3_scale(most);
  const float scale = held ? fmaxf(old, fresh) : fresh;
  const bool grown = __builtin_amdgcn_readfirstlane(held && scale > old);
  if (lane == 0) *scale_at = scale;
  const Over over(scale);
  // A held code's value, over the page's new scale.
  auto again = [&](float value) { return over(value * old); };
  if (grown) {
    constexpr int kLanes = D / 16;
    for (int s = lane / kLanes; s < t.t0; s += 64 / kLanes) {
      u32x4* c = reinterpret_cast<u32x4*>(codes + s * row_bytes + 16 * (lane % kLanes));
      const u32x4 w = *c;
      u32x4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[i] = e4m3x4(again(e4m3_value_at<0>(w[i])), again(e4m3_value_at<1>(w[i])), again(e4m3_value_at<2>(w[i])),
                      again(e4m3_value_at<3>(w[i])));
      }
      *c = r;
    }
  }
  auto write = [&](int i, const P& p) {
    const int s = i * TPI + tok;
    if (s >= n) return;
    float c[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) c[j] = over(E::to_f32(p.v[j]));
    store_codes<true>(codes + (t.t0 + s) * row_bytes, dim, c);
  };
  if (once) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (i < packs) write(i, v[i]);
    }
  } else {
    for (int i = 0; i < packs; ++i) write(i, load(i));
  }

  if (!bounded) return;
  // The lanes that hold other tokens' values of the same dimensions give theirs up
  // by halves: lanes below 32 keep the smallest and those above the largest, then,
  // of 16-bit types, even rows of 16 the first four dimensions and odd rows the last
  // four. A division by the scale and the rounding to a code are both monotone, so
  // the bounds of the codes are the codes of the bounds, and a held bound may join
  // before they are rounded. A dimension without a finite value keeps +448 and -448.
  float mine[SETS][VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    if constexpr (SETS == 2) {
      mine[0][j] = end[0][j];
      mine[1][j] = end[1][j];
    } else {
      mine[0][j] = min_swap32(end[0][j], end[1][j]);
    }
  }
  if constexpr (LPT <= 16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[0][j] = min_swap16(mine[0][j], mine[0][VEC == 8 ? j + 4 : j]);
  }
  if constexpr (LPT <= 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[0][j] = fminf(mine[0][j], dpp<kDppRowRor8>(mine[0][j]));
  }
  if (!edge_lane) return;
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    const float sign = upper || s == 1 ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      float c[4];
      const uint32_t w = held_edge[s][i];
      const float was[4] = {e4m3_value_at<0>(w), e4m3_value_at<1>(w), e4m3_value_at<2>(w), e4m3_value_at<3>(w)};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float m = mine[s][4 * i + j];
        c[j] = m < INFINITY ? over(m) : kE4M3Max;
        if (held) c[j] = fminf(c[j], sign * (grown ? again(was[j]) : was[j]));
        c[j] *= sign;
      }
      edge[s * (D / 4) + i] = e4m3x4(c[0], c[1], c[2], c[3]);
    }
  }
}

// Calls f(IntC<D>, IntC<HOLD>) for the kernel that serves the head size, pages of
// `packs` packs a lane, and single tokens or chunks.
template <int N>
using IntC = std::integral_constant<int, N>;
template <typename F>
void dispatch_append(int dim, int packs, bool chunks, F&& f) {
  auto with_dim = [&](auto d) {
    if (!chunks) {
      f(d, IntC<1>{});
    } else if (packs <= 4) {
      f(d, IntC<4>{});
    } else {
      f(d, IntC<16>{});
    }
  };
  if (dim == 64) {
    with_dim(IntC<64>{});
  } else if (dim == 128) {
    with_dim(IntC<128>{});
  } else {
    with_dim(IntC<256>{});
  }
}

template <typename E>
int launch_append(AppendArgs& a, int64_t tiles, hipStream_t stream) {
  auto aligned = [&](int i) {
    return reinterpret_cast<uintptr_t>(a.x[i]) % 16 == 0 && a.token_stride[i] * E::kBytes % 16 == 0 &&
           a.head_stride[i] * E::kBytes % 16 == 0;
  };
  const bool al = aligned(0) && aligned(1);
  const int packs = static_cast<int>(cdiv(static_cast<int64_t>(a.page) * a.dim * E::kBytes, 1024));
  int st = KL_OK;
  dispatch_append(a.dim, packs, a.offsets != nullptr, [&](auto d, auto hold) {
    constexpr int D = decltype(d)::value, HOLD = decltype(hold)::value;
    const int64_t wgs = cdiv(2 * static_cast<int64_t>(a.heads), kAppendWaves);
    if (tiles * wgs > 0xffffffffLL / kAppendThreads) {
      st = fail(KL_ERR_UNSUPPORTED, "too many tokens, sequences or heads for one launch");
      return;
    }
    a.unit_blocks = static_cast<int>(wgs);
    const auto grid = static_cast<unsigned>(tiles * wgs);
    if (al) {
      append_kernel<E, D, HOLD, true><<<grid, kAppendThreads, 0, stream>>>(a);
    } else {
      append_kernel<E, D, HOLD, false><<<grid, kAppendThreads, 0, stream>>>(a);
    }
  });
  return st != KL_OK ? st : check_launch("append_kv_fp8 kernel launch");
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
  if (reinterpret_cast<uintptr_t>(k_cache) % 16 != 0 || reinterpret_cast<uintptr_t>(v_cache) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(k_bounds) % 16 != 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "the caches and k_bounds must be 16-byte aligned");
  }
  const int64_t tiles = new_offsets == nullptr ? batch : tokens / page_size + 2 * static_cast<int64_t>(batch);
  if (tokens > 0x7fffffffLL || tiles > 0x7fffffffLL) {
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
  const auto s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case KL_DTYPE_F32:
      return launch_append<F32>(a, tiles, s);
    case KL_DTYPE_F16:
      return launch_append<F16>(a, tiles, s);
    case KL_DTYPE_BF16:
      return launch_append<BF16>(a, tiles, s);
  }
  return fail(KL_ERR_UNSUPPORTED, "dtype must be f32, f16 or bf16");
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
