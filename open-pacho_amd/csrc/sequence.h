// What the operators over time share: rows that end early and start again, sums of parts.
#pragma once

#include "common.h"

namespace hpd {

// Workgroup b as number b' such that consecutive b' run on one die: workgroups start on
// the dies in turn, and neighbours read the same lines at their ends.
__device__ __forceinline__ int64_t by_die() {
  constexpr unsigned kDies = 8;
  const unsigned die = blockIdx.x % kDies, least = gridDim.x / kDies, more = gridDim.x % kDies;
  return int64_t(die) * least + (die < more ? die : more) + blockIdx.x / kDies;
}

// Stores `value`, a T or a vector of them, which is aligned as its elements are; with `past` the caches keep no
// place for it.
template <typename T, typename V>
__device__ __forceinline__ void put(T* first, V value, bool past) {
  typedef V Unaligned __attribute__((aligned(sizeof(T))));
  Unaligned* const at = reinterpret_cast<Unaligned*>(first);
  if (past) {
    asm volatile("");  // else the compiler joins the two stores into a plain one, and without the other from behind
    __builtin_nontemporal_store(value, at);
    asm volatile("");
  } else {
    *at = value;
  }
}

// Where rows begin anew and end; pointers that a call does not have are null.
struct Rows {
  const uint8_t* resets;  // (rows, time)
  const void* lengths;    // (rows,)
  int wide;               // int64, else int32
  int64_t time;

  // Steps of a row: its length, none below zero and at most `time`.
  __device__ __forceinline__ int64_t end(int64_t row) const {
    if (!lengths) return time;
    const int64_t n = wide ? static_cast<const int64_t*>(lengths)[row] : static_cast<const int32_t*>(lengths)[row];
    return n < 0 ? 0 : n < time ? n : time;
  }
  // Lane i's byte of the resets from t on, of the last step < end for lanes behind it; for a later ballot().
  __device__ __forceinline__ unsigned byte(int64_t row, int64_t t, int64_t end, int lane) const {
    return resets[row * time + (t + lane < end ? t + lane : end - 1)];
  }
  // Bit i: a reset at step t + i < end.
  template <int N>
  __device__ __forceinline__ unsigned starts(int64_t row, int64_t t, int64_t end) const {
    unsigned bits = 0;
    if (!resets) return bits;
    const uint8_t* at = resets + row * time;
    if constexpr (N % 4 == 0) {
      if (t >= 0 && t + N <= end) {
        typedef uint32_t U __attribute__((aligned(1)));
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
          // The top bit of a byte is set where it is not 0; a product gathers four of them.
          const uint32_t v = reinterpret_cast<const U*>(at + t)[j];
          bits |= ((((v & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | v) >> 7 & 0x01010101u) * 0x01020408u >> 24 << 4 * j;
        }
        return bits;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (t + i >= 0 && t + i < end) bits |= unsigned(at[t + i] != 0) << i;
    }
    return bits;
  }
};

// store(q, sum of parts[w * stride + q] over w from low to high) for the columns q that
// lanes of this workgroup of 1024 threads have, 64 from `column` on: waves on every
// sixteenth part, in a fixed order.
template <typename T, typename F>
__device__ __forceinline__ void add_parts(const T* parts, int64_t stride, int64_t low, int64_t high, int64_t column, int64_t columns, F&& store) {
  __shared__ T meet[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool valid = column + lane < columns;
  T sum[4] = {};
  if (valid) {
    int64_t w = low + wave;
    for (; w + 48 < high; w += 64) {
      T v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = parts[(w + 16 * k) * stride + column + lane];
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += v[k];
    }
    for (; w < high; w += 16) sum[0] += parts[w * stride + column + lane];
  }
  meet[wave][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (wave == 0 && valid) {
    T total = meet[0][lane];
    for (int k = 1; k < 16; ++k) total += meet[k][lane];
    store(column + lane, total);
  }
}

}  // namespace hpd

namespace hp {

constexpr int64_t kLastCache = int64_t(256) << 20;  // bytes

}  // namespace hp
