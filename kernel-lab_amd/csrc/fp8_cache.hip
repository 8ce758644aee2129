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
//   score = f32(k_scale * max_g [lo hi] . [min(q_g, 0) max(q_g, 0)])
// The sum is one of 64 bits, where it is exact for queries whose values span less
// than about 2^30 (a product has 15 bits at most), so the order of its terms does
// not decide which of two near scores is larger. In 64 bits for every page, the
// scores took 25 us of 8 x 1,024 pages on 8 CUs even on the fp64 matrix cores; so:
//   1. scores of all pages on the 16-bit matrix cores, summed in fp32 and within
//      kScoreSlack of their own size;
//   2. the bin of a histogram over them that holds the smallest such score kept, T. The
//      smallest true score kept is within E, the largest error of a page, of it, so
//      pages more than 2 E above the bin are kept and those more than 2 E below it are
//      not, whatever their sums in 64 bits are;
//   3. scores in 64 bits for the pages between (some ten of a thousand), and the choice
//      among them.
// Where a score is not finite, every page is one between.
constexpr int kTile = 16;  // pages that a wave scores at once

struct SelectArgs {
  const void* q;
  const uint8_t* bounds;
  const float* scale;
  const int32_t* table;
  const int32_t* seq_lens;
  int64_t bt_stride;
  // Where a unit's scores come from several workgroups, of each unit: its pages' keys,
  // then each tile's largest k_scale.
  uint32_t* keys;
  uint32_t* arrivals;  // a counter a unit, zero and left zero; null: none
  int32_t* out_table;
  int32_t* out_lens;
  int batch, heads, group, page, max_pages, keep, first, last;
};

// Words of a unit in SelectArgs::keys.
__host__ __device__ __forceinline__ int64_t unit_words(int64_t max_pages) {
  return max_pages + (max_pages + kTile - 1) / kTile;
}

// The unit of a workgroup, by the grid's y and z, and the grid for `units`.
constexpr int kUnitsY = 32768;
__device__ __forceinline__ int64_t grid_unit() { return static_cast<int64_t>(blockIdx.z) * kUnitsY + blockIdx.y; }
inline dim3 unit_grid(int wgs, int64_t units) {
  return dim3(static_cast<unsigned>(wgs), static_cast<unsigned>(std::min<int64_t>(units, kUnitsY)),
              static_cast<unsigned>(cdiv(units, kUnitsY)));
}

__device__ __forceinline__ int select_len(const SelectArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  const int64_t len = as_constant(a.seq_lens)[b];
  return static_cast<int>(max(static_cast<int64_t>(0), min(len, cap)));
}

// A score as a key that orders like it; a NaN like the largest finite score.
__device__ __forceinline__ uint32_t score_key(float s) {
  s = s < 0x1.fffffep127f ? s : 0x1.fffffep127f;
  const uint32_t u = __builtin_bit_cast(uint32_t, s == 0.0f ? 0.0f : s);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// The score of a key made from a finite one.
__device__ __forceinline__ float key_score(uint32_t key) {
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// Keys beside those of finite scores: certainly kept (step 3), and a score that is
// not finite (step 1).
constexpr uint32_t kKeyKept = 0xfffffffeu, kKeyNotFinite = 0xffffffffu;

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = dpp_u32<CTRL>(static_cast<uint32_t>(u)), hi = dpp_u32<CTRL>(static_cast<uint32_t>(u >> 32));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// The larger of two, NaN if either is.
__device__ __forceinline__ double max_or_nan(double a, double b) { return a != a || a > b ? a : b; }

// 16-bit matrix products: 16 query heads by 16 pages, 32 bytes of the bounds a step.
// Lane l supplies A[head l % 16] and B[page l % 16] for eight k of group l / 16 and gets
// the scores of heads 4 (l / 16) .. + 3 and page l % 16, so up to four heads need no
// reduction over lanes. Which bytes a step's k are is free as long as A and B agree: a
// lane's load of 16 codes is its eight k of two steps.
template <typename E>
__device__ __forceinline__ f32x4 score_mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same_v<E, F16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
}

constexpr int kHeadsAtOnce = 16;

// Query heads g0 .. g0 + 15 of a unit as the A operands, heads past the group as zeros:
// lane l's eight values of step 2 c + half are byte 64 c + 16 (l / 16) + 8 half of
// [lo hi] on, so min(q, 0) in the first half of the steps and max(q, 0) in the others.
template <typename E, int D>
struct ScoreQueries {
  static constexpr int C = 2 * D / 64;
  u32x4 v[C][2];
  __device__ __forceinline__ ScoreQueries(const SelectArgs& a, int64_t unit, int g0) {
    const int lane = __lane_id(), g = g0 + (lane & 15);
    const auto* q = static_cast<const typename E::S*>(a.q) + (unit * a.group + min(g, a.group - 1)) * D + 16 * (lane >> 4);
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const u32x4 w = g < a.group ? load_at<false, u32x4>(q, 64 * c + 8 * half) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // 0xffff in the halves that are negative (a NaN of either sign reaches one side).
          const uint32_t sign = (w[i] >> 15) & 0x00010001u;
          const uint32_t negative = (sign << 16) - sign;
          v[c][half][i] = w[i] & negative;
          v[c + C / 2][half][i] = w[i] & ~negative;
        }
      }
    }
  }
  // max_g sum_d |q_gd|, in every lane.
  __device__ __forceinline__ float size() const {
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const auto w = __builtin_bit_cast(Pack<typename E::S, 2>, v[c][half][i] | v[c + C / 2][half][i]);
          sum += fabsf(E::to_f32(w.v[0])) + fabsf(E::to_f32(w.v[1]));
        }
      }
    }
    return row16_max(sum_xor32(sum_xor16(sum)));
  }
};

// What steps 2 and 3 need to know of a unit beside its keys, each lane's share of it.
struct Seen {
  float scale = 0.0f;                     // largest k_scale
  float size = 0.0f;                      // max_g sum_d |q_gd|
  uint32_t low = 0xffffffffu, high = 0;  // smallest and largest key
  __device__ __forceinline__ void add(uint32_t key) {
    low = min(low, key);
    high = max(high, key);
  }
};

// Step 1 for a unit's tiles first, first + step, ..., by a wave: store(page, key) by lanes
// 0 .. 15, and tile_scale(tile, largest k_scale of its pages) in every lane. The result is
// the queries' size, of waves that have a tile.
//
// What bounds it: the bounds of a unit arrive at a CU's share of HBM bandwidth, 256 KiB
// for 1,024 pages of head_dim 128 (11 us on one CU), so a unit's tiles are spread over
// several workgroups; a tile is two dependent loads, its pages' ids and their bounds, so
// the next tile's ids are loaded ahead (us: 8 x 8 units of 1,024 pages 15.7 -> 15.0; its
// bounds, too: 14.9, and others slower).
template <typename E, int D, typename Store, typename Scale>
__device__ __forceinline__ float score_unit(const SelectArgs& a, int64_t unit, int b, int h, int pages, int first,
                                            int step, Store&& store, Scale&& tile_scale) {
  constexpr int C = 2 * D / 64;  // loads of 16 bytes a lane for a tile
  const int lane = __lane_id(), k = lane >> 4;
  const int tiles = (pages + kTile - 1) / kTile;
  if (first >= tiles) return 0.0f;
  const int32_t* table = a.table + b * a.bt_stride;
  auto id_of = [&](int tile) { return table[min(kTile * tile + (lane & 15), pages - 1)]; };
  int id = id_of(first);
  float size = 0.0f;
  ScoreQueries<E, D> q(a, unit, 0);
  for (int tile = first; tile < tiles; tile += step) {
    const int page = kTile * tile + (lane & 15);
    const int64_t head = static_cast<int64_t>(id) * a.heads + h;
    id = id_of(tile + step);
    const uint8_t* edge = a.bounds + head * (2 * D) + 16 * k;
    u32x4 w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) w[c] = *reinterpret_cast<const u32x4*>(edge + 64 * c);
    const float scale = a.scale[head];
    float best = -INFINITY;
    bool finite = true;
    for (int g0 = 0; g0 < a.group; g0 += kHeadsAtOnce) {
      if (a.group > kHeadsAtOnce) q = ScoreQueries<E, D>(a, unit, g0);
      if (tile == first) size = fmaxf(size, q.size());
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        u32x4 lo, hi;
        fp8x16_to<E>(w[c], lo, hi);
        sum = score_mma<E>(q.v[c][0], lo, sum);
        sum = score_mma<E>(q.v[c][1], hi, sum);
      }
      // Lane l has heads 4 k .. + 3 of page l % 16.
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool valid = g0 + 4 * k + i < a.group;
        finite &= !valid || fabsf(sum[i]) < INFINITY;
        best = valid ? fmaxf(best, sum[i]) : best;
      }
    }
    if (a.group > 4) best = max_xor32(max_xor16(best));
    const float score = best * scale;
    finite &= k > 0 || fabsf(score) < INFINITY;
    // A score that is not finite marks its tile, and so the unit.
    const uint32_t key = __any(!finite) ? kKeyNotFinite : score_key(score);
    if (k == 0 && page < pages) store(page, key);
    tile_scale(tile, row16_max(scale));
  }
  return size;
}

// How far step 1's score may be from the true one, over the sum of its terms' sizes: a
// sum of head_dim products (the others are zeros), head_dim <= 256, takes at most 256
// roundings of 2^-23 each (or truncations), 2^-15; twice that.
constexpr float kScoreSlack = 0x1p-14f;

// max_g sum_d |q_gd| over a unit's heads g = first, first + step, ..., by a wave.
template <typename E, int D>
__device__ __forceinline__ float query_size(const SelectArgs& a, int64_t unit, int first, int step) {
  const auto* q = static_cast<const typename E::S*>(a.q) + unit * a.group * D;
  float most = 0.0f;
  for (int g = first; g < a.group; g += step) {
    float sum = 0.0f;
    for (int d = __lane_id(); d < D; d += 64) sum += fabsf(E::to_f32(q[g * D + d]));
    most = fmaxf(most, wave_sum(sum));
  }
  return most;
}

// The true score's key of a page, `head` its index in k_scale: ROWS by a row of 16 lanes
// (each row a page of its own), else by a wave (each row another query head). Each lane
// has D / 16 dimensions.
template <typename E, int D, bool ROWS>
__device__ __forceinline__ uint32_t true_key(const SelectArgs& a, int64_t unit, int64_t head) {
  constexpr int N = D / 16;
  const int lane = __lane_id(), d0 = N * (lane & 15);
  const auto* edge = reinterpret_cast<const uint32_t*>(a.bounds + head * (2 * D) + d0);
  uint32_t words[2][N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    words[0][i] = edge[i];
    words[1][i] = edge[D / 4 + i];
  }
  const double scale = a.scale[head];
  double best = -INFINITY;
  for (int g0 = 0; g0 < a.group; g0 += 4) {
    // Four heads one after the other, their loads together, or one in each row.
    constexpr int kHeads = ROWS ? 4 : 1;
    Pack<typename E::S, N> qs[kHeads];
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
      const int g = min(g0 + (ROWS ? n : lane >> 4), a.group - 1);
      __builtin_memcpy(&qs[n], static_cast<const typename E::S*>(a.q) + (unit * a.group + g) * D + d0, sizeof(qs[n]));
    }
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
      double sum = 0.0;
      static_for<N>([&](auto i) {
        constexpr int I = decltype(i)::value;
        const float v = E::to_f32(qs[n].v[I]);
        sum = fma(static_cast<double>(v < 0.0f ? v : 0.0f), static_cast<double>(e4m3_value_at<I % 4>(words[0][I / 4])), sum);
        sum = fma(static_cast<double>(v < 0.0f ? 0.0f : v), static_cast<double>(e4m3_value_at<I % 4>(words[1][I / 4])), sum);
      });
      sum += dpp64<kDppQuadSwap1>(sum);
      sum += dpp64<kDppQuadSwap2>(sum);
      sum += dpp64<kDppRowRor4>(sum);
      sum += dpp64<kDppRowRor8>(sum);
      best = max_or_nan(sum, best);  // (the last head of a group again changes nothing)
    }
  }
  if constexpr (!ROWS) {
    for (int m = 16; m <= 32; m *= 2) best = max_or_nan(best, __shfl_xor(best, m));
  }
  return score_key(static_cast<float>(best * scale));
}

// Query heads up to which a page between has a row of lanes: four pages a wave then share
// a round trip to memory.
constexpr int kRowsGroup = 8;

// Workgroups of W waves (W = 8 or 16: see wide_workgroups).
constexpr int kListed = 64;  // pages between that a wave ranks

template <int W>
struct PickLds {
  static constexpr int kBins = 64 * W;
  int count[2][3][W];  // of two rounds in turn, so that a round needs one barrier
  float scale[W], size[W];
  uint32_t not_low[W], high[W];
  alignas(16) int bins[kBins];
  int kept, between;          // pages certainly kept, pages between
  int list[kListed];          // the first of them, their ids and their keys
  int list_id[kListed];
  uint32_t list_key[kListed];
};

// Before the first barrier of pick_pages.
template <int W>
__device__ __forceinline__ void clear(PickLds<W>& lds) {
  lds.bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) lds.kept = lds.between = 0;
}

// The smallest of the `want` largest keys of pages q0, q0 + 64 W, ... < free1 of all
// threads, by a workgroup.
//
// The interval that holds it is cut in four: each round counts the keys from three
// thresholds on. It ends as soon as a threshold leaves exactly the number wanted, after
// about half of log2(pages) rounds beyond the bits that all keys share; only equal keys
// take it to the end. For selections that have many pages between (equal or nearly
// equal scores): a round's counts go through LDS, and 15 of them took 20 us.
template <int W, typename Key>
__device__ uint32_t smallest_kept(PickLds<W>& lds, int want, int q0, int free1, uint32_t low, uint32_t high, Key&& key) {
  const int wave = wave_id(), lane = __lane_id();
  // Keys from `low` on are `want` at least, from high + 1 on fewer.
  for (int round = 0; low < high; ++round) {
    const uint32_t step = (high - low) / 4;
    const uint32_t t[3] = {low + step + 1, low + 2 * step + 1, low + 3 * step + 1};
    int n[3] = {0, 0, 0};
    for (int p = q0; p < free1; p += 64 * W) {
      const uint32_t k = key(p);
#pragma unroll
      for (int i = 0; i < 3; ++i) n[i] += k >= t[i] ? 1 : 0;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int total = __builtin_amdgcn_readlane(wave_prefix_sum(n[i]), 63);
      if (lane == 0) lds.count[round & 1][i][wave] = total;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      n[i] = 0;
      for (int w = 0; w < W; ++w) n[i] += lds.count[round & 1][i][w];
    }
    const int side = n[2] >= want ? 3 : n[1] >= want ? 2 : n[0] >= want ? 1 : 0;
    if (side < 3) high = t[side] - 1;
    if (side > 0) {
      low = t[side - 1];
      if (n[side - 1] == want) break;  // the keys from low on are the ones kept
    }
  }
  __syncthreads();  // before the counts' next use
  return low;
}

__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, dpp_u32<kDppQuadSwap1>(v));
  v = max(v, dpp_u32<kDppQuadSwap2>(v));
  v = max(v, dpp_u32<kDppRowRor4>(v));
  return max(v, dpp_u32<kDppRowRor8>(v));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = row16_max(v);
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(static_cast<uint32_t>(s[0]), static_cast<uint32_t>(s[1]));
}

// Steps 2 and 3, by a workgroup: a unit's pages from its keys.
//
// What bounds it: its barriers and LDS round trips, five of them where nothing is tied,
// and one round trip to memory for the pages between. About 5 us of 1,024 pages.
template <typename E, int D, int W>
__device__ void pick_pages(const SelectArgs& a, PickLds<W>& lds, int64_t unit, int b, int h, int pages, uint32_t* keys,
                           const Seen& seen) {
  constexpr int kBins = PickLds<W>::kBins;
  const int wave = wave_id(), lane = __lane_id();
  const int kept = a.keep;  // < pages
  const int32_t* table = a.table + b * a.bt_stride;
  int32_t* out = a.out_table + unit * a.keep;
  const int free0 = a.first, free1 = pages - a.last;  // pages that are not pinned
  const int q0 = free0 + static_cast<int>(threadIdx.x);
  const int want = kept - a.first - a.last;
  auto key = [&](int p) { return keys[p]; };
  // Where the last step's pages begin, and the ids of this thread's first pages, there
  // and in step 3, on their way.
  const int range = (pages + 64 * W - 1) / (64 * W) * 64;
  const int p0 = min(wave * range, pages), p1 = min(p0 + range, pages);
  const int id_p0 = table[min(p0 + lane, pages - 1)];
  const int id_q0 = table[min(q0, pages - 1)];

  const float wave_scale = max_xor32(max_xor16(row16_max(seen.scale)));
  const uint32_t wave_not_low = wave_max(~seen.low), wave_high = wave_max(seen.high);
  if (lane == 0) {
    lds.scale[wave] = wave_scale;
    lds.size[wave] = seen.size;
    lds.not_low[wave] = wave_not_low;
    lds.high[wave] = wave_high;
  }
  __syncthreads();  // the keys are there, too
  const float scale = row16_max(lds.scale[lane % W]), most_size = row16_max(lds.size[lane % W]);
  const uint32_t low = ~row16_max(lds.not_low[lane % W]), high = row16_max(lds.high[lane % W]);
  uint32_t least = 0xffffffffu;  // the smallest key kept: none but the pinned pages
  if (want > 0) {
    // Step 2. What underflows in 16 bits adds less than the last term.
    const float reach = 2.0f * (kScoreSlack * kE4M3Max * most_size * scale) + 0x1p-100f;
    const float lowest = key_score(low), width = key_score(high) - lowest;
    const bool finite = high != kKeyNotFinite && reach < INFINITY && width < INFINITY;
    // Monotone, so a score of a higher bin is a higher one.
    const float to_bin = width > 0.0f ? fminf(kBins / width, 0x1p100f) : 0.0f;
    auto bin_of = [&](float s) { return static_cast<int>(fminf(fmaxf((s - lowest) * to_bin, -1.0f), 1.0f * kBins)); };
    int bin = 0;
    if (finite) {
      for (int p = q0; p < free1; p += 64 * W) atomicAdd(&lds.bins[min(bin_of(key_score(key(p))), kBins - 1)], 1);
      __syncthreads();
      // Lane l has the W bins below kBins - W l; every wave finds the bin by itself.
      int n[W], mine = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        n[i] = lds.bins[kBins - W * (lane + 1) + i];
        mine += n[i];
      }
      const int upto = wave_prefix_sum(mine);
      int left = want - (upto - mine), at = 0;
#pragma unroll
      for (int i = W - 1; i >= 0; --i) {
        if (left > 0) at = i;
        left -= n[i];
      }
      const uint64_t here = __ballot(upto >= want && upto - mine < want);
      const int owner = __builtin_ctzll(here);
      bin = kBins - W * (owner + 1) + __builtin_amdgcn_readlane(at, owner);
    }
    // Step 3. The pages between are listed in the order that they come in; which of them
    // are kept does not depend on it. (The last bin takes what is past its end, too.)
    int sure = 0;
    for (int base = 0; base < free1 - free0; base += 64 * W) {
      const int p = q0 + base;
      const bool valid = p < free1;
      const float s = valid ? key_score(key(p)) : 0.0f;
      const bool above = valid && finite && bin < kBins - 1 && bin_of(s - reach) > bin;
      const bool below = finite && bin_of(s + reach) < bin;
      sure += __builtin_popcountll(__ballot(above));
      if (valid) {
        keys[p] = above ? kKeyKept : below ? 0 : kKeyNotFinite;  // the last: to be scored
        if (!above && !below) {
          const int i = atomicAdd(&lds.between, 1);
          if (i < kListed) {
            lds.list[i] = p;
            lds.list_id[i] = base == 0 ? id_q0 : table[p];
          }
        }
      }
    }
    if (lane == 0 && sure > 0) atomicAdd(&lds.kept, sure);
    __syncthreads();
    const int between = lds.between;
    if (between <= kListed) {
      if (a.group <= kRowsGroup) {
        for (int i0 = 4 * wave; i0 < between; i0 += 4 * W) {
          const int i = i0 + (lane >> 4);
          const uint32_t k = true_key<E, D, true>(
              a, unit, static_cast<int64_t>(lds.list_id[min(i, between - 1)]) * a.heads + h);
          if ((lane & 15) == 0 && i < between) lds.list_key[i] = k;
        }
      } else {
        for (int i = wave; i < between; i += W) {
          const int id = __builtin_amdgcn_readfirstlane(lds.list_id[i]);
          const uint32_t k = true_key<E, D, false>(a, unit, static_cast<int64_t>(id) * a.heads + h);
          if (lane == 0) lds.list_key[i] = k;
        }
      }
      __syncthreads();
      // A row of lanes ranks a page: the ones before it are counted 16 at a time.
      for (int i0 = 4 * wave; i0 < between; i0 += 4 * W) {
        const int i = min(i0 + (lane >> 4), between - 1);
        const int p = lds.list[i];
        const uint32_t k = lds.list_key[i];
        int better = 0;
        for (int j = lane & 15; j < between; j += 16) {
          const uint32_t kj = lds.list_key[j];
          better += kj > k || (kj == k && lds.list[j] < p) ? 1 : 0;
        }
        better += static_cast<int>(dpp_u32<kDppQuadSwap1>(better));
        better += static_cast<int>(dpp_u32<kDppQuadSwap2>(better));
        better += static_cast<int>(dpp_u32<kDppRowRor4>(better));
        better += static_cast<int>(dpp_u32<kDppRowRor8>(better));
        if ((lane & 15) == 0) keys[p] = better < want - lds.kept ? kKeyKept : 0;
      }
      __syncthreads();
      least = kKeyKept;
    } else {
      for (int base = wave * 64; base < pages; base += 64 * W) {
        const int p = base + lane;
        uint64_t todo = __ballot(p >= free0 && p < free1 && keys[min(p, pages - 1)] == kKeyNotFinite);
        for (; todo != 0; todo &= todo - 1) {
          const int at = base + __builtin_ctzll(todo);
          const uint32_t k = true_key<E, D, false>(a, unit, static_cast<int64_t>(table[at]) * a.heads + h);
          if (lane == 0) keys[at] = k;
        }
      }
      __syncthreads();
      least = smallest_kept(lds, want, q0, free1, 0, kKeyKept, key);
    }
  }

  // Positions: pages above the smallest key kept, and the first ones equal to it. A wave
  // has neighbouring pages, 64 at a time, whose ranks are counts of lanes below.
  auto ranked = [&](auto&& take) {
    for (int base = p0; base < p1; base += 64) {
      const int p = base + lane;
      const bool pinned = p < free0 || p >= free1;
      const uint32_t k = p < p1 && !pinned ? key(p) : 0;
      take(p, __ballot(p < p1 && (pinned || k > least)), __ballot(p < p1 && !pinned && k == least));
    }
  };
  int above = 0, ties = 0;
  ranked([&](int, uint64_t over, uint64_t tie) {
    above += __builtin_popcountll(over);
    ties += __builtin_popcountll(tie);
  });
  if (lane == 0) {
    lds.count[1][0][wave] = above;
    lds.count[1][1][wave] = ties;
  }
  __syncthreads();
  int above_at = 0, ties_at = 0, above_all = 0;
  for (int w = 0; w < W; ++w) {
    if (w < wave) {
      above_at += lds.count[1][0][w];
      ties_at += lds.count[1][1][w];
    }
    above_all += lds.count[1][0][w];
  }
  const int room = kept - above_all;  // for keys equal to the smallest
  const uint64_t below = (1ull << lane) - 1, mine = 1ull << lane;
  ranked([&](int p, uint64_t over, uint64_t tie) {
    const int ties_here = ties_at + __builtin_popcountll(tie & below);
    const int at = above_at + __builtin_popcountll(over & below) + min(ties_here, room);
    if ((over & mine) != 0 || ((tie & mine) != 0 && ties_here < room)) {
      out[at] = p < p0 + 64 ? id_p0 : table[p];
    }
    above_at += __builtin_popcountll(over);
    ties_at += __builtin_popcountll(tie);
  });
}

// A unit's length, and its output where every page is kept, by one workgroup.
__device__ __forceinline__ void keep_all(const SelectArgs& a, int64_t unit, int b, int pages) {
  const int32_t* table = a.table + b * a.bt_stride;
  for (int i = threadIdx.x; i < a.keep; i += blockDim.x) a.out_table[unit * a.keep + i] = i < pages ? table[i] : 0;
}
__device__ __forceinline__ void write_len(const SelectArgs& a, int64_t unit, int len, int pages) {
  const int kept = min(pages, a.keep);
  if (threadIdx.x == 0) a.out_lens[unit] = kept > 0 ? (kept - 1) * a.page + (len - (pages - 1) * a.page) : 0;
}

// Pages whose keys fit LDS.
constexpr int kLdsPages = 8192;

// One launch for all steps. The workgroups along x share a unit's tiles; where more than
// one has any, they leave keys and scales in memory, device-coherent, and the last to
// arrive (paged_decode.hip's arrive_and_merge has the order of accesses) takes steps 2
// and 3. At most kLdsPages pages a unit.
template <typename E, int D, int W>
__global__ void __launch_bounds__(64 * W) select_kernel(const SelectArgs a) {
  __shared__ PickLds<W> lds;
  __shared__ uint32_t keys[kLdsPages];
  __shared__ int s_last;
  const int64_t unit = grid_unit();
  const int b = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads);
  if (b >= a.batch) return;
  const int len = select_len(a, b);
  const int pages = (len + a.page - 1) / a.page;
  const int tiles = (pages + kTile - 1) / kTile;
  const int wgs = max(1, min(static_cast<int>(gridDim.x), (tiles + W - 1) / W));
  if (pages <= a.keep) {
    if (blockIdx.x == 0) {
      write_len(a, unit, len, pages);
      keep_all(a, unit, b, pages);
    }
    return;
  }
  if (static_cast<int>(blockIdx.x) >= wgs) return;
  clear(lds);
  const int first = static_cast<int>(blockIdx.x) * W + wave_id(), step = wgs * W;
  Seen seen;
  if (wgs == 1) {
    seen.size = score_unit<E, D>(
        a, unit, b, h, pages, first, step,
        [&](int page, uint32_t key) {
          keys[page] = key;
          seen.add(key);
        },
        [&](int, float s) { seen.scale = fmaxf(seen.scale, s); });
  } else {
    uint32_t* shared = a.keys + unit * unit_words(a.max_pages);
    const auto rsrc = make_rsrc(uniform_ptr(shared));
    seen.size = score_unit<E, D>(
        a, unit, b, h, pages, first, step,
        [&](int page, uint32_t key) {
          buffer_store_f32<kCachePolicyDevice>(rsrc, static_cast<uint32_t>(page) * 4u, __builtin_bit_cast(float, key));
        },
        [&](int tile, float s) {
          if (__lane_id() == 0) {
            buffer_store_f32<kCachePolicyDevice>(rsrc, static_cast<uint32_t>(a.max_pages + tile) * 4u, s);
          }
        });
    wait_vector_memory();
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t old = __hip_atomic_fetch_add(a.arrivals + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = old + 1 == static_cast<uint32_t>(wgs);
      if (s_last) __hip_atomic_store(a.arrivals + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!__builtin_amdgcn_readfirstlane(s_last)) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");  // no load moves above the arrival
    for (int p = threadIdx.x; p < pages; p += 64 * W) {
      const uint32_t k = __builtin_bit_cast(uint32_t, buffer_load_f32<kCachePolicyDevice>(rsrc, static_cast<uint32_t>(p) * 4u));
      keys[p] = k;
      seen.add(k);
    }
    for (int t = threadIdx.x; t < tiles; t += 64 * W) {
      seen.scale = fmaxf(seen.scale, buffer_load_f32<kCachePolicyDevice>(rsrc, static_cast<uint32_t>(a.max_pages + t) * 4u));
    }
  }
  write_len(a, unit, len, pages);
  pick_pages<E, D, W>(a, lds, unit, b, h, pages, keys, seen);
}

// The same in two launches: for tables past kLdsPages, and where there are no counters.
template <typename E, int D, int W>
__global__ void __launch_bounds__(64 * W) score_kernel(const SelectArgs a) {
  const int64_t unit = grid_unit();
  const int b = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads);
  if (b >= a.batch) return;
  const int pages = (select_len(a, b) + a.page - 1) / a.page;
  if (pages <= a.keep) return;
  uint32_t* shared = a.keys + unit * unit_words(a.max_pages);
  score_unit<E, D>(a, unit, b, h, pages, static_cast<int>(blockIdx.x) * W + wave_id(),
                   W * static_cast<int>(gridDim.x), [&](int page, uint32_t key) { shared[page] = key; },
                   [&](int tile, float s) {
                     if (__lane_id() == 0) shared[a.max_pages + tile] = __builtin_bit_cast(uint32_t, s);
                   });
}

template <typename E, int D, int W>
__global__ void __launch_bounds__(64 * W) pick_kernel(const SelectArgs a) {
  __shared__ PickLds<W> lds;
  __shared__ uint32_t keys[kLdsPages];
  const int64_t unit = grid_unit();
  const int b = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads);
  if (b >= a.batch) return;
  const int len = select_len(a, b);
  const int pages = (len + a.page - 1) / a.page;
  write_len(a, unit, len, pages);
  if (pages <= a.keep) {
    keep_all(a, unit, b, pages);
    return;
  }
  clear(lds);
  uint32_t* shared = a.keys + unit * unit_words(a.max_pages);
  Seen seen;
  seen.size = query_size<E, D>(a, unit, wave_id(), W);
  for (int t = threadIdx.x; t < (pages + kTile - 1) / kTile; t += 64 * W) {
    seen.scale = fmaxf(seen.scale, __builtin_bit_cast(float, shared[a.max_pages + t]));
  }
  for (int p = threadIdx.x; p < pages; p += 64 * W) {
    const uint32_t k = shared[p];
    if (pages <= kLdsPages) keys[p] = k;
    seen.add(k);
  }
  if (pages <= kLdsPages) {
    pick_pages<E, D, W>(a, lds, unit, b, h, pages, keys, seen);
  } else {
    pick_pages<E, D, W>(a, lds, unit, b, h, pages, shared, seen);
  }
}

// Workgroups of a unit: as many as can have a tile for each of eight waves, within one
// for each CU in all (a CU holds one or two, and the others wait for a round of their
// own: 32 sequences of up to 1,024 pages 21 -> 28 us with four).
int unit_workgroups(int64_t units, int max_pages) {
  const int64_t most = cdiv(max_pages, kTile * 8);
  const int64_t wanted = cdiv(static_cast<int64_t>(current_cu_count()), std::max<int64_t>(units, 1));
  return static_cast<int>(std::max<int64_t>(1, std::min(most, wanted)));
}

// Whether a workgroup has 16 waves: where it has a unit to itself and more tiles than
// eight waves take at once, and for long tables, whose keys one workgroup ranks. Measured
// (us, 8 -> 16 waves): 32 sequences of up to 1,024 pages, 8 KV heads 21.2 -> 18.6, one
// sequence of 8,192 29.0 -> 23.8; the other way one of 1,024 12.7 -> 11.4, of 128 8.4 ->
// 7.6, and at head_dim 256, whose registers leave room for eight, 20 -> 13.3.
bool wide_workgroups(int head_dim, int wgs, int max_pages) {
  return head_dim <= 128 && ((wgs == 1 && max_pages > kTile * 8) || max_pages > 2048);
}

template <typename E, int D, int W>
int launch_select(SelectArgs& a, int64_t units, int wgs, hipStream_t stream) {
  a.arrivals = wgs > 1 && a.max_pages > a.keep && a.max_pages <= kLdsPages ? arrival_counters(units, stream) : nullptr;
  if (a.arrivals != nullptr || (wgs == 1 && a.max_pages <= kLdsPages) || a.max_pages <= a.keep) {
    select_kernel<E, D, W><<<unit_grid(a.arrivals != nullptr ? wgs : 1, units), 64 * W, 0, stream>>>(a);
    return check_launch("select_pages kernel launch");
  }
  score_kernel<E, D, W><<<unit_grid(wgs, units), 64 * W, 0, stream>>>(a);
  const int st = check_launch("select_pages score kernel launch");
  if (st != KL_OK) return st;
  pick_kernel<E, D, W><<<unit_grid(1, units), 64 * W, 0, stream>>>(a);
  return check_launch("select_pages kernel launch");
}

template <typename E>
int dispatch_select(SelectArgs& a, int dim, int64_t units, hipStream_t stream) {
  const int wgs = unit_workgroups(units, a.max_pages);
  const bool wide = wide_workgroups(dim, wgs, a.max_pages);
  if (dim == 64) {
    return wide ? launch_select<E, 64, 16>(a, units, wgs, stream) : launch_select<E, 64, 8>(a, units, wgs, stream);
  }
  if (dim == 128) {
    return wide ? launch_select<E, 128, 16>(a, units, wgs, stream) : launch_select<E, 128, 8>(a, units, wgs, stream);
  }
  return launch_select<E, 256, 8>(a, units, wgs, stream);
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
  const int64_t units = static_cast<int64_t>(batch) * num_kv_heads;
  if (out_workspace) {
    *out_workspace = unit_workgroups(units, max_pages) == 1 && max_pages <= kLdsPages
                         ? 0
                         : static_cast<size_t>(units) * static_cast<size_t>(unit_words(max_pages)) * 4;
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
  if (units > 0x7fffffffLL || static_cast<int64_t>(max_pages) * page_size > 0x7fffffffLL ||
      static_cast<int64_t>(num_selected) * page_size > 0x7fffffffLL) {
    return fail(KL_ERR_UNSUPPORTED, "more than 2^31 (sequence, KV head) pairs, or tables past 2^31 tokens");
  }
  if (batch == 0) return ok();
  if (max_pages < 1) return fail(KL_ERR_INVALID_ARGUMENT, "max_pages must be >= 1");
  if (!out_table || !out_lens || !q || !k_bounds || !k_scale || !block_table || !seq_lens) {
    return fail(KL_ERR_INVALID_ARGUMENT, "outputs, q, k_bounds, k_scale, block_table and seq_lens must be non-null");
  }
  if (block_table_stride < max_pages && batch > 1) {
    return fail(KL_ERR_INVALID_ARGUMENT, "block_table_stride must be >= max_pages");
  }
  if (reinterpret_cast<uintptr_t>(k_bounds) % 16 != 0) {
    return fail(KL_ERR_INVALID_ARGUMENT, "k_bounds must be 16-byte aligned");
  }
  size_t need = 0;
  kl_select_pages_workspace(batch, num_kv_heads, max_pages, &need);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(KL_ERR_WORKSPACE, "workspace smaller than kl_select_pages_workspace reported");
  }
  SelectArgs a;
  a.q = q;
  a.bounds = static_cast<const uint8_t*>(k_bounds);
  a.scale = k_scale;
  a.table = block_table;
  a.seq_lens = seq_lens;
  a.bt_stride = block_table_stride;
  a.keys = static_cast<uint32_t*>(workspace);
  a.out_table = out_table;
  a.out_lens = out_lens;
  a.batch = batch;
  a.heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.page = page_size;
  a.max_pages = max_pages;
  a.keep = num_selected;
  a.first = first_pages;
  a.last = last_pages;
  const auto s = reinterpret_cast<hipStream_t>(stream);
  return dtype == KL_DTYPE_F16 ? dispatch_select<F16>(a, head_dim, units, s) : dispatch_select<BF16>(a, head_dim, units, s);
}
