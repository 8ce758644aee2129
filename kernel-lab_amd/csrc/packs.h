// Packs of elements, loaded and stored at any element alignment.
#pragma once

#include "hip_common.h"

namespace kl {
namespace {

template <typename S, int N>
struct alignas(sizeof(S) * N) Pack {
  S v[N];
};

// The 16 bytes at element offset `off` of a row. Unaligned rows (any element
// alignment) use the same 16-byte memory instructions, which gfx950 takes at
// any address.
template <bool ALIGNED, typename P, typename S>
__device__ __forceinline__ P load_at(const S* row, int off) {
  P v;
  if constexpr (ALIGNED) {
    v = *reinterpret_cast<const P*>(row + off);
  } else {
    __builtin_memcpy(&v, row + off, sizeof(P));
  }
  return v;
}
template <bool ALIGNED, typename P, typename S>
__device__ __forceinline__ void store_at(S* row, int off, const P& v) {
  if constexpr (ALIGNED) {
    *reinterpret_cast<P*>(row + off) = v;
  } else {
    __builtin_memcpy(row + off, &v, sizeof(P));
  }
}

}  // namespace
}  // namespace kl
