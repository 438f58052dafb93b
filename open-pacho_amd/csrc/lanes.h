// Values and sums across the lanes of a wave without a way through LDS.
#pragma once

#include "common.h"

namespace hpd {

// Exchanges halves (BIT 5) or odd and even rows of 16 lanes (BIT 4) between a and b.
template <int BIT>
__device__ __forceinline__ void swap_lanes(uint32_t& a, uint32_t& b) {
  if constexpr (BIT == 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
  }
}
// Lane i: the value of lane i ^ 8 (8), i ^ 7 (7), i ^ 3 (3) or i ^ 1 (1).
template <int MASK>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  constexpr int kind = MASK == 8 ? 0x128 /* row_ror:8 */ : MASK == 7 ? 0x141 /* row_half_mirror */ : MASK == 3 ? 0x1B /* quad_perm 3 2 1 0 */ : 0xB1 /* 1 0 3 2 */;
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kind, 0xF, 0xF, true));
}

template <typename T>
struct Words {
  uint32_t w[sizeof(T) / 4];
};

template <int BIT, typename T>
__device__ __forceinline__ T fold_rows(T a, T b) {
  auto x = __builtin_bit_cast(Words<T>, a), y = __builtin_bit_cast(Words<T>, b);
#pragma unroll
  for (unsigned k = 0; k < sizeof(T) / 4; ++k) swap_lanes<BIT>(x.w[k], y.w[k]);
  return __builtin_bit_cast(T, x) + __builtin_bit_cast(T, y);
}
template <int MASK, typename T>
__device__ __forceinline__ T from_across(T v) {
  auto x = __builtin_bit_cast(Words<T>, v);
#pragma unroll
  for (unsigned k = 0; k < sizeof(T) / 4; ++k) x.w[k] = across<MASK>(x.w[k]);
  return __builtin_bit_cast(T, x);
}
// The sum over aligned groups of L lanes (a power of two up to 64), the same bits in all of them. The steps within
// rows of 16 lanes are additions that take their operand from another lane; exchanges join the rows.
template <int L, typename T>
__device__ __forceinline__ T lane_sum(T v) {
  if constexpr (L >= 2) v += from_across<1>(v);
  if constexpr (L >= 4) v += from_across<3>(v);
  if constexpr (L >= 8) v += from_across<7>(v);
  if constexpr (L >= 16) v += from_across<8>(v);
  if constexpr (L >= 32) v = fold_rows<4>(v, v);
  if constexpr (L >= 64) v = fold_rows<5>(v, v);
  return v;
}

}  // namespace hpd
