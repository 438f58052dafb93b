// Rows of logits in registers and in pieces, and sums of their losses: what the
// losses from logits share.
#pragma once

#include <type_traits>

#include "common.h"
#include "exponential.h"

namespace {

constexpr int kPieceThreads = 256, kPieceLoads = 8;
constexpr int64_t kFewPieces = 1024;
constexpr double kCountedBytes = 1 << 25;

// Elements of a piece, of which the last one of a row may have fewer.
__device__ __forceinline__ int piece_end(int64_t left, int piece) { return left < piece ? int(left) : piece; }

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  // Rows of any length follow each other: elements are aligned, vectors not.
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr int width = 4;
};
template <>
struct Vec<double> {
  typedef double type __attribute__((ext_vector_type(2), aligned(8)));
  static constexpr int width = 2;
};

__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

// log x in 64 bits. Of a float, the exponent's part exactly and the log of the
// rest, below 0.35, to a float's precision: the error is 3e-8 whatever x is.
__device__ __forceinline__ double log_wide(float x) {
  int exponent;
  float rest = frexpf(x, &exponent);
  if (rest < 0.70710678f) rest *= 2, --exponent;
  return double(exponent) * 0.6931471805599453 + double(logf(rest));
}
__device__ __forceinline__ double log_wide(double x) { return log(x); }
// What every loss of rows of logits has; pointers that a call does not have are null.
template <typename T>
struct LossCall {
  const T* logits;
  const uint8_t* mask;
  int64_t rows, vocab;
  T* grad;
  // What the sum of losses is multiplied by: a value in device memory, or the
  // one here, or where count_here is set one over the rows that the mask keeps,
  // which every workgroup counts for itself.
  const double* scale;
  double scale_value;
  bool count_here;
  double* sums;      // a workgroup's sum of losses each
  T* loss;           // their scaled sum, by the last workgroup to end, if
  unsigned* ticket;  // not null: counts the workgroups that have ended

  __device__ bool kept(int64_t row) const { return !mask || mask[row]; }
};

// A reduction over L <= 64 neighbouring lanes, all of them getting the result.
template <int L, typename T, typename Op>
__device__ __forceinline__ T team_reduce(T v, Op op) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  return v;
}

// A value that all lanes have, in scalar registers.
__device__ __forceinline__ double of_wave(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t low = __builtin_amdgcn_readfirstlane(int(bits)), high = __builtin_amdgcn_readfirstlane(int(bits >> 32));
  return __builtin_bit_cast(double, uint64_t(high) << 32 | low);
}

// What distances from a row's largest logit are multiplied by.
struct Unscaled {
  template <typename T>
  __device__ __forceinline__ T operator()(T x) const {
    return x;
  }
};

// (m, S) of a row from those of pieces in the lanes that have one, of L lanes.
template <int L = 64, typename T, typename Scale = Unscaled>
__device__ __forceinline__ void join(bool has, T piece_top, T piece_total, T& top, T& total, Scale scaled = {}) {
  const T none = -T(__builtin_huge_val());
  top = team_reduce<L>(has ? piece_top : none, [](T a, T b) { return larger(a, b); });
  T part = T(0);
  if (has) part = piece_top == none ? piece_total : piece_total * hpd::exp_down(scaled(piece_top - top));
  total = team_reduce<L>(part, [](T a, T b) { return a + b; });
}

// The same from memory, by every wave for itself; a lane's pieces join first, one after
// the other in 64 bits: a row of 2^31 floats has 4096 a lane.
template <typename T>
__device__ __forceinline__ void join_pieces(const T* tops, const T* totals, int pieces, T& top, T& total) {
  const int lane = threadIdx.x & 63;
  const T none = -T(__builtin_huge_val());
  T own = lane < pieces ? tops[lane] : none;
  double sum = lane < pieces ? totals[lane] : T(0);
  for (int k = lane + 64; k < pieces; k += 64) {
    const T next = larger(own, tops[k]);
    if (own != none) sum *= hpd::exp_down(own - next);
    sum += tops[k] == none ? double(totals[k]) : double(totals[k]) * hpd::exp_down(tops[k] - next);
    own = next;
  }
  join(lane < pieces, own, T(sum), top, total);
}

// What the waves of a workgroup leave for each other, for two rows in turn: of
// each of D pieces in depth. S: sums of a row, one or two.
template <typename T, int D, int S = 1>
struct Meet {
  T tops[2][D][16], totals[2][D][16], seconds[S == 2 ? 2 : 1][S == 2 ? D : 1][16];
};

// Logits that a second sum leaves out: none, so that there is no such sum.
struct NoNames {
  static constexpr bool some = false;
};

// A second sum (Share::statistics) below this is formed again, relative to the largest of its own logits: relative to
// the row's its terms have left the type, or are about to. Above it the terms that an exponential rounds to
// zero (2^-126, 2^-1022 and less each, of no more than 2^31 logits) are 2^-31 of it at most.
template <typename T>
constexpr T kLeastSecond = sizeof(T) == 4 ? T(0x1p-64f) : T(0x1p-900);

// A team's share of a row of `length` elements, which it takes in pieces of
// kPieceThreads x kPieceLoads vectors: kSide pieces side by side by 256 threads each,
// kDeep one after the other, a lane's vectors of a piece 256 apart. Of the elements
// after the last whole vector, the first lanes of the last piece have one each.
// Places past the row's end hold -inf. Each piece's sum is formed as stats_kernel
// forms it and they meet as there, so that a row's statistics have the same bits
// whichever kernel makes them.
template <typename T, int L, int K>
struct Share {
  static constexpr int W = Vec<T>::width;
  static constexpr int kSide = L > kPieceThreads ? L / kPieceThreads : 1, kDeep = K > kPieceLoads ? K / kPieceLoads : 1;
  static constexpr int kStep = L > kPieceThreads ? kPieceThreads : L, kLoads = K / kDeep;  // of a piece
  using V = typename Vec<T>::type;
  T z[K][W], rest;

  __device__ __forceinline__ static int index(int k, int lane) {
    const int piece = k / kLoads * kSide + lane / kStep;
    return (piece * kStep * kLoads + k % kLoads * kStep + lane % kStep) * W;
  }
  __device__ __forceinline__ static int rest_piece(int length) { return (length - 1) / (kStep * kLoads * W); }
  __device__ __forceinline__ static int rest_index(int length, int lane) {
    if (kSide > 1 && lane / kStep != rest_piece(length) % kSide) return length;
    return length / W * W + lane % kStep;
  }

  // STREAM: past the caches, for a last reading.
  template <bool STREAM>
  __device__ __forceinline__ void load(const T* row, int length, int lane) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[k][j] = -T(__builtin_huge_val());
      if (index(k, lane) + W <= length) {
        V v;
        if constexpr (STREAM) v = __builtin_nontemporal_load(reinterpret_cast<const V*>(row + index(k, lane)));
        else v = *reinterpret_cast<const V*>(row + index(k, lane));
#pragma unroll
        for (int j = 0; j < W; ++j) z[k][j] = v[j];
      }
    }
    rest = -T(__builtin_huge_val());
    if (rest_index(length, lane) < length) rest = row[rest_index(length, lane)];
  }

  // The share of a row that is not read.
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < W; ++j) z[k][j] = -T(__builtin_huge_val());
    rest = -T(__builtin_huge_val());
  }

  // Past the caches at every size (float32 with the gradient, in parentheses with a sum
  // over it right after, us, past and through the caches): 8192 x 32000 353 (512) and 392
  // (529), 65536 x 1000 103 (144) and 102 (138), 16384 x 1000 31 (46) and 34 (48), 16448 x 18
  // 15 (28) and 16 (31).
  __device__ __forceinline__ void store(T* row, int length, int lane) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (index(k, lane) + W <= length) {
        V v;
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = z[k][j];
        __builtin_nontemporal_store(v, reinterpret_cast<V*>(row + index(k, lane)));
      }
    }
    if (rest_index(length, lane) < length) row[rest_index(length, lane)] = rest;
  }

  // f(value, its index in the row, which of the lane's pieces) for every value.
  template <typename F>
  __device__ __forceinline__ void each(int length, int lane, F&& f) {
    const int last = kDeep > 1 ? rest_piece(length) / kSide : 0;
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
#pragma unroll
      for (int k = d * kLoads; k < (d + 1) * kLoads; ++k)
#pragma unroll
        for (int j = 0; j < W; ++j) f(z[k][j], index(k, lane) + j, d);
      if (d == last) f(rest, rest_index(length, lane), d);
    }
  }

  // f(value, whether `names` has it, which of the lane's pieces) for every value.
  template <typename Names, typename F>
  __device__ __forceinline__ void each_named(int length, int lane, Names names, F&& f) {
    const int last = kDeep > 1 ? rest_piece(length) / kSide : 0;
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
#pragma unroll
      for (int k = d * kLoads; k < (d + 1) * kLoads; ++k) {
        const unsigned bits = names.bits(index(k, lane));
#pragma unroll
        for (int j = 0; j < W; ++j) f(z[k][j], bits >> j & 1, d);
      }
      if (d == last) f(rest, rest_index(length, lane) < length && names.one(rest_index(length, lane)), d);
    }
  }

  // The values become exp(z - tops[d]) in the d-th piece of the lane; top and total
  // are those of the row. A barrier each after the maxima and the sums; rows take
  // the two sets of `meet` in turn.
  __device__ __forceinline__ void statistics(int length, int lane, Meet<T, kDeep>& meet, int turn, T (&tops)[kDeep], T& top, T& total) {
    T second;
    statistics(length, lane, meet, turn, tops, top, total, Unscaled(), NoNames(), second);
  }

  // The values become exp(scaled(z - tops[d])), and `second` their sum without the
  // values that `names` has, which become -exp(): names.bits(i) has a bit for each value of the vector at i.
  template <typename Scale, typename Names>
  __device__ __forceinline__ void statistics(int length, int lane, Meet<T, kDeep, Names::some ? 2 : 1>& meet, int turn, T (&tops)[kDeep], T& top, T& total,
                                             Scale scaled, Names names, T& second) {
    constexpr T kNone = -T(__builtin_huge_val());
    const auto greater = [](T a, T b) { return larger(a, b); };
    const auto plus = [](T a, T b) { return a + b; };
    const int last = kDeep > 1 ? rest_piece(length) / kSide : 0;  // the piece that has the rest
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      T m = d == last ? rest : kNone;
#pragma unroll
      for (int k = d * kLoads; k < (d + 1) * kLoads; ++k)
#pragma unroll
        for (int j = 0; j < W; ++j) m = larger(m, z[k][j]);
      tops[d] = team_reduce<L < 64 ? L : 64>(m, greater);
    }
    share_out(tops, meet.tops[turn], greater);
    T totals[kDeep], seconds[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const T reference = tops[d] == kNone ? T(0) : tops[d];
      T sum = T(0), other = T(0);
      if (d == last) {
        sum = rest = hpd::exp_down(scaled(rest - reference));
        if constexpr (Names::some) {
          const bool named = rest_index(length, lane) < length && names.one(rest_index(length, lane));
          other = named ? T(0) : rest;
          rest = named ? -rest : rest;
        }
      }
      T s[W] = {}, o[W] = {};
#pragma unroll
      for (int k = d * kLoads; k < (d + 1) * kLoads; ++k) {
        unsigned bits = 0;
        if constexpr (Names::some) bits = names.bits(index(k, lane));
#pragma unroll
        for (int j = 0; j < W; ++j) {
          z[k][j] = hpd::exp_down(scaled(z[k][j] - reference));
          s[j] += z[k][j];
          if constexpr (Names::some) {
            o[j] += bits >> j & 1 ? T(0) : z[k][j];
            z[k][j] = bits >> j & 1 ? -z[k][j] : z[k][j];
          }
        }
        if constexpr (Names::some) asm volatile("" ::: "memory");  // the bits of all vectors at once would take registers from the values
      }
#pragma unroll
      for (int j = 0; j < W; ++j) sum += s[j];
      totals[d] = team_reduce<L < 64 ? L : 64>(sum, plus);
      if constexpr (Names::some) {
#pragma unroll
        for (int j = 0; j < W; ++j) other += o[j];
        seconds[d] = team_reduce<L < 64 ? L : 64>(other, plus);
      }
    }
    if constexpr (Names::some) share_out<false>(seconds, meet.seconds[turn], plus);
    share_out(totals, meet.totals[turn], plus);
    if constexpr (Names::some) {
      if constexpr (L > 64) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) seconds[d] = of_waves(meet.seconds[turn][d], (threadIdx.x >> 6) / 4, plus);
      }
      second = seconds[0];
    }
    top = tops[0];
    total = totals[0];
    if constexpr (kSide * kDeep > 1) {
      // Lane k joins in for piece k, as in join_pieces.
      const int k = threadIdx.x & 63, d = k / kSide, side = k % kSide;
      const bool has = k <= rest_piece(length);
      T piece_top = kNone, piece_total = T(0);
      if (has) {
        piece_top = of_waves(meet.tops[turn][d], side, greater);
        piece_total = of_waves(meet.totals[turn][d], side, plus);
      }
      join(has, piece_top, piece_total, top, total, scaled);
      if constexpr (Names::some) {
        T part = T(0), again;
        if (has) part = of_waves(meet.seconds[turn][d], side, plus);
        join(has, piece_top, part, again, second, scaled);
      }
    }
  }

  // A second sum of less than kLeastSecond, from another reading of `row`: sum exp(scaled(z - top)) of the values that
  // `names` leaves out, of which `top` is the largest (-inf and 0 of none). Of several pieces those whose own sum is not as
  // small keep it. For a whole team, with what statistics() left in `meet`; its other set is free for this.
  template <typename Scale, typename Names>
  __device__ __forceinline__ static void apart(const T* row, int length, int lane, Meet<T, kDeep, 2>& meet, int turn, Scale scaled, Names names, T& top, T& sum) {
    constexpr T kNone = -T(__builtin_huge_val());
    constexpr int kPiece = kStep * kLoads * W;
    const auto greater = [](T a, T b) { return larger(a, b); };
    const auto plus = [](T a, T b) { return a + b; };
    asm volatile("" : "+v"(lane));  // what follows from it is formed here, not kept from row to row
#pragma unroll 1
    for (int d = 0; d < kDeep; ++d) {
      const int side = kSide > 1 ? lane / kStep : 0, start = (d * kSide + side) * kPiece;
      T own = kNone, part = T(0);
      if (kSide * kDeep == 1 || of_waves(meet.seconds[turn][d], side, plus) < kLeastSecond<T>) {
        for (int i = start + lane % kStep; i < length && i < start + kPiece; i += kStep) {
          const T z = row[i];
          if (names.one(i) || z == kNone) continue;
          if (z > own) part = part * hpd::exp_down(scaled(own - z)) + T(1), own = z;
          else part += hpd::exp_down(scaled(z - own));
        }
      }
      join<L < 64 ? L : 64>(true, own, part, top, sum, scaled);
      if constexpr (L > 64) {
        if ((lane & 63) == 0) meet.tops[turn ^ 1][d][lane >> 6] = top, meet.seconds[turn ^ 1][d][lane >> 6] = sum;
      }
    }
    if constexpr (L > 64) {
      __syncthreads();
      const auto joined = [&](int d, int side) {  // from the four waves of a piece
        const T *tops = meet.tops[turn ^ 1][d] + 4 * side, *sums = meet.seconds[turn ^ 1][d] + 4 * side;
        top = of_waves(tops - 4 * side, side, greater), sum = T(0);
        for (int w = 0; w < 4; ++w) sum += tops[w] == kNone ? T(0) : sums[w] * hpd::exp_down(scaled(tops[w] - top));
      };
      if constexpr (kSide * kDeep == 1) {
        joined(0, 0);
      } else {
        const int k = lane & 63, d = k / kSide, side = k % kSide;
        const bool has = k <= rest_piece(length);
        T piece_top = kNone, piece_sum = T(0);
        if (has) {
          piece_top = of_waves(meet.tops[turn][d], side, greater);
          piece_sum = of_waves(meet.seconds[turn][d], side, plus);
          if (piece_sum < kLeastSecond<T>) joined(d, side), piece_top = top, piece_sum = sum;
        }
        join(has, piece_top, piece_sum, top, sum, scaled);
      }
      __syncthreads();  // the set belongs to the next row
    }
  }

  // The share of each piece's values in the row: exp(tops[d] - top), exactly 1 of one piece.
  template <typename Scale = Unscaled>
  __device__ __forceinline__ static T part(T piece_top, T top, Scale scaled = {}) {
    return kSide * kDeep == 1 ? T(1) : hpd::exp_down(scaled(piece_top - top));
  }

 private:
  // The four waves' values of the piece at `side`.
  template <typename Op>
  __device__ __forceinline__ static T of_waves(const T* waves, int side, Op op) {
    T v = waves[4 * side];
#pragma unroll
    for (int w = 1; w < 4; ++w) v = op(v, waves[4 * side + w]);
    return v;
  }
  // From each wave's values the pieces'; without MEETS they are left for a barrier that comes.
  template <bool MEETS = true, typename Op>
  __device__ __forceinline__ static void share_out(T (&v)[kDeep], T (*waves)[16], Op op) {
    if constexpr (L > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) waves[d][wave] = v[d];
      }
      if constexpr (MEETS) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kDeep; ++d) v[d] = of_waves(waves[d], wave / 4, op);
      }
    }
  }
};

// The sum of every thread's value, for thread 0 of the workgroup.
__device__ __forceinline__ double workgroup_sum(double sum) {
  __shared__ double meet[16];
  sum = hpd::wave_sum(sum);
  __syncthreads();  // an earlier sum's values have been read
  if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = meet[0];
  for (unsigned w = 1; w < blockDim.x / 64; ++w) sum += meet[w];
  return sum;
}

// The factor of the losses.
template <typename T>
__device__ __forceinline__ double scale_of(const LossCall<T>& c) {
  if (!c.count_here) return c.scale ? *c.scale : c.scale_value;
  // Sixteen bytes at a time: the top bit of a byte is set where it is not 0.
  typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(1)));
  const int64_t vectors = c.rows / 16;
  int count = 0;
  for (int64_t i = threadIdx.x; i < vectors; i += blockDim.x) {
    const U4 v = reinterpret_cast<const U4*>(c.mask)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) count += __popc((((v[j] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | v[j]) & 0x80808080u);
  }
  const int64_t tail = vectors * 16 + threadIdx.x;
  if (threadIdx.x < 16 && tail < c.rows) count += c.mask[tail] != 0;
  const double sum = workgroup_sum(count);
  return 1.0 / (sum > 1.0 ? sum : 1.0);
}

// Leaves `sum`, which thread 0 has, as number `index` of `count`. With a ticket the
// last one to come adds all of them in their order, whichever workgroup it is. No
// fences: a sum is valid by itself, the places being all ones (which no sum is)
// between launches, and each is on its way before its ticket is taken.
template <typename T>
__device__ __forceinline__ void leave_loss(const LossCall<T>& c, double sum, double scale, unsigned index, unsigned count) {
  __shared__ bool last;
  if (!c.ticket) {
    if (threadIdx.x == 0) c.sums[index] = sum;
    return;
  }
  uint64_t* const places = reinterpret_cast<uint64_t*>(c.ticket + 64);
  if (threadIdx.x == 0) {
    uint64_t bits = __builtin_bit_cast(uint64_t, sum);
    if (bits == ~uint64_t(0)) --bits;  // a NaN as well
    __hip_atomic_store(&places[index], bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(c.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
  }
  __syncthreads();
  const bool adds = last;
  __syncthreads();
  if (!adds) return;
  double total = 0;
  for (unsigned i = threadIdx.x; i < count; i += blockDim.x) {
    uint64_t bits;
    do bits = __hip_atomic_load(&places[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    while (bits == ~uint64_t(0));
    total += __builtin_bit_cast(double, bits);
    __hip_atomic_store(&places[i], ~uint64_t(0), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  total = workgroup_sum(total);
  if (threadIdx.x == 0) {
    *c.loss = T(total * scale);
    __hip_atomic_store(c.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// 1 / max(1, rows that the mask keeps), by one workgroup.
template <typename T>
__global__ __launch_bounds__(1024) void count_kernel(LossCall<T> c, double* __restrict__ scale) {
  const double found = scale_of(c);
  if (threadIdx.x == 0) *scale = found;
}

// loss = scale x the sum of the workgroups' sums, by one workgroup.
template <typename T>
__global__ __launch_bounds__(1024) void loss_kernel(LossCall<T> c, int64_t n) {
  double sum = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) sum += c.sums[i];
  const double factor = scale_of(c);
  sum = workgroup_sum(sum);
  if (threadIdx.x == 0) *c.loss = T(sum * factor);
}

// ---- host ----------------------------------------------------------------------

// Calls f with the team (L, K) that holds rows of `vocab` logits, or returns
// false: none does.
template <typename T, typename F>
bool with_team(int64_t vocab, F&& f) {
  const int64_t vectors = hp::ceil_div(vocab, Vec<T>::width);
#define TEAM(L, K) \
  if (vectors <= L * K) return f(std::integral_constant<int, L>{}, std::integral_constant<int, K>{}), true;
  TEAM(4, 1)
  TEAM(8, 1)
  TEAM(16, 1)
  TEAM(32, 1)
  TEAM(64, 1)
  TEAM(64, 2)
  TEAM(64, 4)
  TEAM(64, 8)
  TEAM(256, 4)
  TEAM(256, 8)
  TEAM(256, 16)
  TEAM(512, 16)
  if constexpr (sizeof(T) == 4) {
    TEAM(1024, 16)
  }
#undef TEAM
  return false;
}

// Whether teams take the rows of a call with the gradient: not rows so few and so
// long that they would leave most of the chip idle.
template <typename T>
bool teams_hold(int64_t rows, int64_t vocab) {
  const int64_t vectors = hp::ceil_div(vocab, Vec<T>::width);
  return vectors <= 256 * 16 || (vectors <= (sizeof(T) == 4 ? 1024 : 512) * 16 && rows >= 128);
}

// Pieces of a row, of whole vectors: the teams' where teams would take the rows, so
// that the statistics have the same bits; else equal ones, as few as hold the row or
// as many as rows need to make kFewPieces workgroups, with a vector for every thread.
template <typename T>
struct Pieces {
  int count, length;
  Pieces(int64_t rows, int64_t vocab) {
    const int64_t vectors = hp::ceil_div(vocab, Vec<T>::width), most = kPieceThreads * kPieceLoads;
    const int64_t least = hp::ceil_div(vectors, most);
    const int64_t wanted = std::min(hp::ceil_div(kFewPieces, rows), hp::ceil_div(vectors, kPieceThreads));
    const int64_t each = teams_hold<T>(rows, vocab) ? most : hp::ceil_div(vectors, std::max(least, wanted));
    length = int(each) * Vec<T>::width;
    count = int(hp::ceil_div(vocab, length));
  }
};

unsigned loop_grid(int64_t groups) { return unsigned(std::min(groups, hp::kMaxGrid)); }

// The sum of the losses where the kernel that made them does not leave it.
template <typename T>
void final_loss(hp_ctx* ctx, const LossCall<T>& c, int64_t sums) {
  if (c.ticket && sums) return;
  loss_kernel<T><<<1, 1024, 0, ctx->stream>>>(c, sums);
  hp::check_launch("loss sum");
}

// Prepares a launch of `blocks` workgroups that leave `sums` sums of losses. Few
// sums are added by the last workgroup (up to 1024: the tickets of 4096 took 18 us more than
// a launch). The mask is counted by every workgroup for itself where that
// reads little, or little beside the logits (8192 masked rows of 32000 floats: 293 us,
// with a launch for it 297; of 6000: 71 and 67).
template <typename T>
void plan_losses(hp_ctx* ctx, hp::Scratch& scratch, LossCall<T>& c, unsigned sums, unsigned blocks) {
  if (sums <= hp::kTicketPlaces) c.ticket = ctx->ticket;
  else c.sums = scratch.take<double>(sums);
  const double counted = double(blocks) * double(c.rows), logits = double(c.rows) * double(c.vocab) * sizeof(T);
  if (!c.count_here || counted <= kCountedBytes || counted * 8 <= logits) return;
  double* scale = scratch.take<double>(1);
  count_kernel<T><<<1, 1024, 0, ctx->stream>>>(c, scale);
  hp::check_launch("token count");
  c.scale = scale;
  c.count_here = false;
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == HP_F32) f(float(0));
  else f(double(0));
}

}  // namespace
