// Divergence of rows of logits from a teacher that is known by its largest logits,
// and its gradient.
//
//   q_j = exp((z_j - m) / T) / S,  S = sum_j exp((z_j - m) / T)
//   p_e = softmax over the list's t_e / T (and the rest's logit, if there is one)
//   loss = sum_e p_e (log p_e - log q_{i(e)}) + p_r (log p_r - log (R / S))
//   T dloss/dz_j = q_j - sum_{i(e) = j} p_e            where the list names j
//                = q_j - p_r exp((z_j - m) / T) / R    elsewhere (p_r = 0 without a rest)
//
// with R the sum S without the terms that the list names. R is formed as a sum of its
// own, not as a difference: where the list holds nearly all of q the rest would lose
// its digits. Where the list holds all that the type has of q, R is formed again, relative to
// the largest logit m' that it does not name (Share::apart): log R = (m' - m) / T + log R', and
// exp((z_j - m') / T) / R' takes its place in the gradient. Such rows are read again, and
// their gradient is stored twice: 8192 x 32000 with 64 entries takes 332 us where no row is
// so and 1001 where all are.
//
// Which logits are named stands in a bit for each of a row, in LDS; a vector's
// bits are one read, and where a team holds the row the only one: named exponentials carry
// a sign from there on. (A second read for the gradient, and the bits of all vectors at
// once, took the values' registers: 451 us in place of 361.) Bound: HBM, each logit read once
// and each gradient written once, as for the losses of token_loss.hip, whose teams and
// pieces of rows it shares. 8192 x 32000 float32 with 64 entries and the rest takes
// 310-361 us with the gradient (5.8-6.8 TB/s) and 126 without, where a mask leaves rows out that are then not
// read; 4096 x 32000 float64 588 and 160.
//
// The list is the work of one wave, or of a team within one: its softmax, its bits and
// its terms of the loss, each entry's logit read again. The named places of the
// gradient are written once more, after a barrier, as p_e has no place in the registers
// that hold a row. An index that stands twice is found by the bit that it finds set;
// then every entry adds up the entries of its index.
#include "token_rows.h"

namespace {

template <typename T>
struct Call : LossCall<T> {
  const void* indices;
  int wide_indices;  // int64, else int32
  int entries;       // of a row's list
  const T *teacher, *teacher_rest;
  T* losses;
  double temperature, inverse;  // 1 / temperature

  __device__ __forceinline__ int64_t index(int64_t row, int entry) const {
    const int64_t at = row * entries + entry;
    return wide_indices ? static_cast<const int64_t*>(indices)[at] : static_cast<const int32_t*>(indices)[at];
  }
  __device__ __forceinline__ T logit(int64_t row, int entry) const { return teacher[row * entries + entry]; }
  __device__ __forceinline__ auto scaled() const {
    const T by = T(inverse);
    return [by](T x) { return x * by; };
  }
};

// Bits of the logits that a list names, those from `start` on.
struct Bits {
  static constexpr bool some = true;
  unsigned* words;

  // For the vector at i, which is a multiple of its width.
  __device__ __forceinline__ unsigned bits(int i) const { return words[i >> 5] >> (i & 31); }
  __device__ __forceinline__ bool one(int i) const { return words[i >> 5] >> (i & 31) & 1; }
};

// The team's stores to LDS and memory before are seen by its loads after.
__device__ __forceinline__ void team_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A row's list, by L <= 64 neighbouring lanes. Its logits stand as distances (t_e - t) / T from the largest of
// them, t, less the largest of these and the rest's: 0 is the largest of all. Quotients t_e / T would have lost the
// digits of their distances where they are large; not those of floats, whose quotients in 64 bits have digits to spare, so
// that t is 0 there (and takes no registers: 8 x 512 x 64000 with the gradient 352 us in place of 368).
template <typename T, int L>
struct List {
  T base;                 // t; 0 of floats and where no logit is there
  double top, log_total;  // of the distances, the rest's among them, before they end at 0; of their exponentials
  T inverse, rest;        // 1 / their sum of exponentials, and the rest's p
  T spoiled;              // 0, or NaN where an entry stands outside the vocabulary
  bool repeats;           // an index stands twice

  // A value that the team's lanes have; of a whole wave in scalar registers.
  __device__ __forceinline__ static double of_team(double v) { return L == 64 ? of_wave(v) : v; }
  __device__ __forceinline__ double distance(const Call<T>& c, T logit) const { return (double(logit) - double(base)) * c.inverse - top; }
  __device__ __forceinline__ T share(const Call<T>& c, T logit) const { return hpd::exp_down(T(distance(c, logit))) * inverse; }
  // The rest's distance from the list's largest, with what the quotient of that one's logit is rounded by put back.
  __device__ __forceinline__ double rest_distance(const Call<T>& c, T given) const {
    if constexpr (sizeof(T) == 4) return double(given);
    const double quotient = double(base) * c.inverse;
    return (double(given) - quotient) - __builtin_fma(-quotient, c.temperature, double(base)) * c.inverse;
  }

  __device__ __forceinline__ void read(const Call<T>& c, int64_t row, int lane) {
    const T none = -T(__builtin_huge_val()), given = c.teacher_rest ? c.teacher_rest[row] : none;
    T most = none;
    for (int e = lane; e < c.entries; e += L) most = larger(most, c.logit(row, e));
    most = team_reduce<L>(most, [](T a, T b) { return larger(a, b); });
    base = sizeof(T) == 4 || most == none ? T(0) : most;
    const double other = rest_distance(c, given);
    top = of_team(larger((double(most) - double(base)) * c.inverse, other));
    T sum = lane == 0 ? hpd::exp_down(T(other - top)) : T(0);
    bool outside = false;
    for (int e = lane; e < c.entries; e += L) {
      const T logit = c.logit(row, e);
      const int64_t i = c.index(row, e);
      sum += hpd::exp_down(T(distance(c, logit)));
      outside = outside || (logit != none && (i < 0 || i >= c.vocab));
    }
    sum = team_reduce<L>(sum, [](T a, T b) { return a + b; });
    outside = team_reduce<L>(int(outside), [](int a, int b) { return a | b; });
    inverse = T(1) / sum;
    log_total = of_team(log_wide(sum));
    rest = c.teacher_rest ? hpd::exp_down(T(other - top)) * inverse : T(0);
    spoiled = outside || sum != sum ? T(__builtin_nan("")) : T(0);
  }

  // f(entry, its index) for every entry of the lane that names one of [start, start + length).
  template <typename F>
  __device__ __forceinline__ static void each(const Call<T>& c, int64_t row, int lane, int64_t start, int64_t length, F&& f) {
    for (int e = lane; e < c.entries; e += L) {
      const int64_t i = c.index(row, e);
      if (i >= start && i < start + length && i < c.vocab && c.logit(row, e) != -T(__builtin_huge_val())) f(e, i);
    }
  }

  __device__ __forceinline__ void set(const Call<T>& c, Bits bits, int64_t row, int lane, int64_t start, int64_t length) {
    bool again = false;
    each(c, row, lane, start, length, [&](int, int64_t i) {
      const unsigned at = unsigned(i - start), bit = 1u << (at & 31);
      const unsigned before = atomicOr(&bits.words[at >> 5], bit);  // after a repeat too: it names the entry
      again = again || (before & bit);
    });
    repeats = team_reduce<L>(int(again), [](int a, int b) { return a | b; });
  }
  __device__ __forceinline__ static void clear(const Call<T>& c, Bits bits, int64_t row, int lane, int64_t start, int64_t length) {
    each(c, row, lane, start, length, [&](int, int64_t i) { bits.words[(i - start) >> 5] = 0; });
  }

  // The row's loss from the statistics of its logits, for every lane of the team.
  // `unlisted` is relative to `rest_top`.
  __device__ __forceinline__ double loss(const Call<T>& c, int64_t row, int lane, T row_top, T total, T rest_top, T unlisted) const {
    const double log_row = log_wide(total);
    const T given = rest != T(0) ? c.teacher_rest[row] : T(0);
    double sum = 0;
    each(c, row, lane, 0, c.vocab, [&](int e, int64_t i) {
      const double apart = distance(c, c.logit(row, e));
      const T p = hpd::exp_down(T(apart)) * inverse;
      const double log_q = (double(c.logits[row * c.vocab + i]) - double(row_top)) * c.inverse - log_row;
      if (p != T(0)) sum += double(p) * ((apart - log_total) - log_q);
    });
    if (lane == 0 && rest != T(0)) {
      const double log_q = (double(rest_top) - double(row_top)) * c.inverse + log_wide(unlisted) - log_row;
      sum += double(rest) * ((rest_distance(c, given) - top - log_total) - log_q);
    }
    sum = team_reduce<L>(sum, [](double a, double b) { return a + b; });
    return sum + double(spoiled) + (total == total ? 0.0 : double(total));
  }

  // The gradient at the named places of [start, start + length), whose other terms are
  // stored already: (q - p) weight.
  __device__ __forceinline__ void correct(const Call<T>& c, int64_t row, int lane, int64_t start, int64_t length, T row_top, T row_inverse,
                                          T weight) const {
    const auto scaled = c.scaled();
    each(c, row, lane, start, length, [&](int e, int64_t i) {
      T p = T(0);
      if (repeats) {
        for (int k = 0; k < c.entries; ++k) {
          if (c.index(row, k) == i) p += share(c, c.logit(row, k));
        }
      } else {
        p = share(c, c.logit(row, e));
      }
      const T q = hpd::exp_down(scaled(c.logits[row * c.vocab + i] - row_top)) * row_inverse;
      c.grad[row * c.vocab + i] = (q - p) * weight;
    });
  }
};

// What a gradient's value exp((z - m) / T) is multiplied by where the list does not name it.
template <typename T>
__device__ __forceinline__ T unlisted_factor(T row_inverse, T rest, T unlisted) {
  return row_inverse - (rest == T(0) || unlisted == T(0) ? T(0) : rest / unlisted);
}

// The gradient at the places of [start, start + length) that are not named, for a rest that
// is relative to its own largest logit; `by`: the rest's p over its sum.
template <int L, typename T>
__device__ __forceinline__ void correct_rest(const Call<T>& c, Bits bits, int64_t row, int lane, int64_t start, int length, T row_top, T row_inverse, T rest_top,
                                             T by, T weight) {
  const auto scaled = c.scaled();
  const T* logits = c.logits + row * c.vocab + start;
  T* out = c.grad + row * c.vocab + start;
  asm volatile("" : "+v"(lane));
  for (int i = lane; i < length; i += L) {
    const T z = logits[i];
    if (!bits.one(i)) out[i] = (hpd::exp_down(scaled(z - row_top)) * row_inverse - hpd::exp_down(scaled(z - rest_top)) * by) * weight;
  }
}

// REST: the rest of the teacher's mass is a class of its own.
template <typename T, int L, int K, bool REST>
__global__ __launch_bounds__(L > 256 ? L : 256, sizeof(T) == 8 || K < 8 ? 1 : L == 256 && K == 16 ? 3 : 4) void row_kernel(Call<T> c) {
  constexpr int kTeams = L > 256 ? 1 : 256 / L, kLanes = L < 64 ? L : 64;  // lanes that work on the list
  using S = Share<T, L, K>;
  constexpr int kWords = (L * K * S::W + 31) / 32;
  __shared__ Meet<T, S::kDeep, REST ? 2 : 1> meet;
  __shared__ unsigned words[kTeams][kWords];
  __shared__ T told[2][2];  // by the wave of the list, for two rows in turn: rest, spoiled
  const int lane = kTeams == 1 ? int(threadIdx.x) : threadIdx.x % L, team = kTeams == 1 ? 0 : threadIdx.x / L;
  const bool lists = L <= 64 || threadIdx.x < 64;
  const int length = int(c.vocab);
  const auto scaled = c.scaled();
  const Bits bits{words[team]};
  for (int i = threadIdx.x; i < kTeams * kWords; i += blockDim.x) words[0][i] = 0;
  __syncthreads();
  const double factor = scale_of(c);
  double sum = 0;
  int turn = 0;
  // Teams of several waves are alone in their workgroup, as in token_loss.hip.
  for (int64_t row = int64_t(blockIdx.x) * kTeams + team; row < c.rows; row += int64_t(gridDim.x) * kTeams) {
    T* out = c.grad ? c.grad + row * c.vocab : nullptr;
    S share;
    if (!c.kept(row)) {
      if (lane == 0) c.losses[row] = T(0);
      if (out) {
        share.each(length, lane, [](T& v, int, int) { v = T(0); });
        share.store(out, length, lane);
      }
      continue;
    }
    List<T, kLanes> list{};
    if (lists) {
      list.read(c, row, lane);
      list.set(c, bits, row, lane, 0, length);
      if constexpr (L > 64) {
        if (lane == 0) told[turn][0] = list.rest, told[turn][1] = list.spoiled;
      } else {
        team_fence();
      }
    }
    share.template load<true>(c.logits + row * c.vocab, length, lane);
    T tops[S::kDeep], top, total, unlisted = T(0);
    if constexpr (REST) share.statistics(length, lane, meet, turn, tops, top, total, scaled, bits, unlisted);
    else share.statistics(length, lane, meet, turn, tops, top, total, scaled, NoNames(), unlisted);
    const T inverse = T(1) / total, rest = L > 64 ? told[turn][0] : list.rest;
    const bool apart = REST && rest != T(0) && unlisted < kLeastSecond<T>;
    const T weight = T(factor * c.inverse) + (L > 64 ? told[turn][1] : list.spoiled);
    if (out) {
      const T inner = inverse * weight, outer = REST && !apart ? unlisted_factor(inverse, rest, unlisted) * weight : inner;
      if constexpr (REST) {
        // Named ones carry a sign: -0 too, and NaN stays NaN.
        share.each(length, lane, [&](T& v, int, int d) {
          const T value = S::part(tops[d], top, scaled) * v;
          v = __builtin_signbit(v) ? -value * inner : value * outer;
        });
      } else {
        share.each(length, lane, [&](T& v, int, int d) { v = v * (S::part(tops[d], top, scaled) * inner); });
      }
      share.store(out, length, lane);
      if constexpr (L > 64) __syncthreads();
      else team_fence();
    }
    T rest_top = top;
    if constexpr (REST) {
      if (apart) {  // here, where the row's registers are free
        S::apart(c.logits + row * c.vocab, length, lane, meet, turn, scaled, bits, rest_top, unlisted);
        if (out && unlisted != T(0)) correct_rest<L>(c, bits, row, lane, 0, length, top, inverse, rest_top, rest / unlisted, weight);
        if constexpr (L > 64) __syncthreads();  // before the list's bits are cleared
      }
    }
    if (out && lists) list.correct(c, row, lane, 0, length, top, inverse, weight);
    turn ^= 1;
    if (lists) {
      const double loss = list.loss(c, row, lane, top, total, rest_top, unlisted);
      if (lane == 0) c.losses[row] = T(loss), sum += loss;
      list.clear(c, bits, row, lane, 0, length);
      if constexpr (L <= 64) team_fence();
    }
  }
  leave_loss(c, workgroup_sum(sum), factor, blockIdx.x, gridDim.x);
}

// Statistics of pieces of rows, number row * pieces + piece.
template <typename T>
struct Statistics {
  T *tops, *totals, *seconds;
  T *rest_tops, *rests;  // the second sum relative to the largest of its own logits where it is small (Share::apart)
  int pieces, length;    // of a row, of a piece
};

template <typename T, bool REST>
__global__ __launch_bounds__(kPieceThreads) void stats_kernel(Call<T> c, Statistics<T> parts) {
  using S = Share<T, kPieceThreads, kPieceLoads>;
  __shared__ Meet<T, 1, REST ? 2 : 1> meet;
  __shared__ unsigned words[REST ? kPieceThreads * kPieceLoads * S::W / 32 : 1];
  const auto scaled = c.scaled();
  const Bits bits{words};
  if constexpr (REST) {
    for (unsigned i = threadIdx.x; i < sizeof(words) / 4; i += kPieceThreads) words[i] = 0;
    __syncthreads();
  }
  int turn = 0;
  for (int64_t part = blockIdx.x; part < c.rows * parts.pieces; part += gridDim.x) {
    const int64_t row = part / parts.pieces;
    if (!c.kept(row)) continue;
    const int64_t start = (part - row * parts.pieces) * parts.length;
    const int length = piece_end(c.vocab - start, parts.length);
    const T* logits = c.logits + row * c.vocab + start;
    T tops[1], top, total, second, rest_top, rest;
    S share;
    share.template load<true>(logits, length, threadIdx.x);
    List<T, 64> list;
    if constexpr (REST) {
      // Seen by all at the first of the statistics' barriers, and read before the second.
      if (threadIdx.x < 64) list.set(c, bits, row, threadIdx.x, start, length);
      share.statistics(length, threadIdx.x, meet, turn, tops, top, total, scaled, bits, second);
      rest_top = top, rest = second;
      if (second < kLeastSecond<T>) share.apart(logits, length, threadIdx.x, meet, turn, scaled, bits, rest_top, rest);
      if (threadIdx.x < 64) list.clear(c, bits, row, threadIdx.x, start, length);
    } else {
      share.statistics(length, threadIdx.x, meet, turn, tops, top, total, scaled, NoNames(), second);
    }
    turn ^= 1;
    if (threadIdx.x == 0) {
      parts.tops[part] = top, parts.totals[part] = total;
      if constexpr (REST) parts.seconds[part] = second, parts.rest_tops[part] = rest_top, parts.rests[part] = rest;
    }
  }
}

// What a row's pieces add up to, by every wave for itself; a lane's pieces join first,
// one after the other in 64 bits (join_pieces, with two sums).
template <typename T, bool REST, typename Scale>
__device__ __forceinline__ void join_row(const Statistics<T>& parts, int64_t row, Scale scaled, T& top, T& total, T& rest_top, T& unlisted) {
  int lane = threadIdx.x & 63;
  const int pieces = parts.pieces;
  const int64_t first = row * pieces;
  const T none = -T(__builtin_huge_val());
  const bool has = lane < pieces;
  const auto add = [&](const T* tops, const T* sums, const T* others, T& own, double& sum, double& other) __attribute__((always_inline)) {
    own = has ? tops[lane] : none;
    sum = has ? sums[lane] : T(0), other = others && has ? others[lane] : T(0);
    for (int k = lane + 64; k < pieces; k += 64) {
      const T next = larger(own, tops[k]);
      const double before = own == none ? 1.0 : double(hpd::exp_down(scaled(own - next)));
      const double here = tops[k] == none ? 1.0 : double(hpd::exp_down(scaled(tops[k] - next)));
      sum = sum * before + double(sums[k]) * here;
      if (others) other = other * before + double(others[k]) * here;
      own = next;
    }
  };
  T own;
  double sum, other;
  add(parts.tops + first, parts.totals + first, REST ? parts.seconds + first : nullptr, own, sum, other);
  join(has, own, T(sum), top, total, scaled);
  rest_top = top;
  if constexpr (REST) {
    T again;
    join(has, own, T(other), again, unlisted, scaled);
    if (unlisted < kLeastSecond<T>) {
      asm volatile("" : "+v"(lane));  // as in Share::apart
      add(parts.rest_tops + first, parts.rests + first, nullptr, own, sum, other);
      join(has, own, T(sum), rest_top, unlisted, scaled);
    }
  }
}

// The rows' losses from their pieces, a workgroup each, as wide as piece_grad_kernel, so
// that both add the losses in one order.
template <typename T, bool REST>
__global__ __launch_bounds__(kPieceThreads) void finish_kernel(Call<T> c, Statistics<T> parts) {
  const double factor = scale_of(c);
  const int64_t row = blockIdx.x;
  double loss = 0;
  if (threadIdx.x < 64) {
    if (c.kept(row)) {
      T top, total, rest_top, unlisted = T(0);
      join_row<T, REST>(parts, row, c.scaled(), top, total, rest_top, unlisted);
      List<T, 64> list;
      list.read(c, row, threadIdx.x);
      loss = list.loss(c, row, threadIdx.x, top, total, rest_top, unlisted);
    }
    if (threadIdx.x == 0) c.losses[row] = T(loss);
  }
  leave_loss(c, loss, factor, blockIdx.x, gridDim.x);
}

// The gradient of one piece of a row from the statistics of its pieces, which every
// workgroup joins for itself; that of the first piece leaves the row's loss.
template <typename T, bool REST>
__global__ __launch_bounds__(kPieceThreads, sizeof(T) == 8 && REST ? 3 : 1) void piece_grad_kernel(Call<T> c, Statistics<T> parts) {
  using S = Share<T, kPieceThreads, kPieceLoads>;
  __shared__ unsigned words[kPieceThreads * kPieceLoads * S::W / 32];
  __shared__ T told[2];
  const int lane = threadIdx.x;
  const auto scaled = c.scaled();
  const Bits bits{words};
  for (unsigned i = threadIdx.x; i < sizeof(words) / 4; i += kPieceThreads) words[i] = 0;
  __syncthreads();
  const double factor = scale_of(c);
  for (int64_t part = blockIdx.x; part < c.rows * parts.pieces; part += gridDim.x) {
    const int64_t row = part / parts.pieces;
    const bool first = part == row * parts.pieces;
    const int64_t start = (part - row * parts.pieces) * parts.length;
    const int length = piece_end(c.vocab - start, parts.length);
    T* out = c.grad + row * c.vocab + start;
    double loss = 0;
    S share;
    if (c.kept(row)) {
      share.template load<true>(c.logits + row * c.vocab + start, length, lane);
      List<T, 64> list{};
      if (lane < 64) {
        list.read(c, row, lane);
        list.set(c, bits, row, lane, start, length);
        if (lane == 0) told[0] = list.rest, told[1] = list.spoiled;
      }
      T top, total, rest_top, unlisted = T(0);
      join_row<T, REST>(parts, row, scaled, top, total, rest_top, unlisted);
      __syncthreads();
      const T inverse = T(1) / total, weight = T(factor * c.inverse) + told[1];
      const bool apart = REST && rest_top != top;
      const T inner = inverse * weight, outer = REST && !apart ? unlisted_factor(inverse, told[0], unlisted) * weight : inner;
      share.each_named(length, lane, bits, [&](T& v, bool named, int) { v = hpd::exp_down(scaled(v - top)) * (!REST || named ? inner : outer); });
      share.store(out, length, lane);
      __syncthreads();
      if (apart) {
        if (told[0] != T(0) && unlisted != T(0)) correct_rest<kPieceThreads>(c, bits, row, lane, start, length, top, inverse, rest_top, told[0] / unlisted, weight);
        __syncthreads();  // before the list's bits are cleared
      }
      if (lane < 64) {
        list.correct(c, row, lane, start, length, top, inverse, weight);
        list.clear(c, bits, row, lane, start, length);
        if (first) loss = list.loss(c, row, lane, top, total, rest_top, unlisted);
      }
    } else {
      share.each(length, lane, [](T& v, int, int) { v = T(0); });
      share.store(out, length, lane);
    }
    if (first) {
      if (lane == 0) c.losses[row] = T(loss);
      leave_loss(c, loss, factor, unsigned(row), unsigned(c.rows));
    }
  }
}

// ---- host ----------------------------------------------------------------------

// Whether a call takes teams: as the losses of token_loss.hip do.
template <typename T>
bool teams_serve(const Call<T>& c) {
  if (c.vocab <= kPieceThreads * kPieceLoads * Vec<T>::width) return true;
  return c.grad && teams_hold<T>(c.rows, c.vocab);
}

// Returns how many sums of losses there are.
template <typename T, bool REST>
int64_t rows_pass(hp_ctx* ctx, hp::Scratch& scratch, Call<T>& c) {
  unsigned blocks = 0;
  if (teams_serve(c) && with_team<T>(c.vocab, [&](auto l, auto k) {
        constexpr int L = l, K = k, threads = L > 256 ? L : 256;
        blocks = unsigned(std::min<int64_t>(hp::ceil_div(c.rows, threads / L), 16384));
        plan_losses(ctx, scratch, c, blocks, blocks);
        row_kernel<T, L, K, REST><<<blocks, threads, 0, ctx->stream>>>(c);
        hp::check_launch("distillation rows");
      })) {
    return blocks;
  }
  const Pieces<T> pieces(c.rows, c.vocab);
  const int64_t parts = c.rows * pieces.count;
  Statistics<T> found{scratch.take<T>(parts), scratch.take<T>(parts), nullptr, nullptr, nullptr, pieces.count, pieces.length};
  if constexpr (REST) found.seconds = scratch.take<T>(parts), found.rest_tops = scratch.take<T>(parts), found.rests = scratch.take<T>(parts);
  const unsigned grid = loop_grid(parts);
  hp::require(c.rows <= hp::kMaxGrid, "too many long rows for one launch");
  blocks = unsigned(c.rows);
  plan_losses(ctx, scratch, c, blocks, c.grad ? grid : blocks);
  stats_kernel<T, REST><<<grid, kPieceThreads, 0, ctx->stream>>>(c, found);
  hp::check_launch("distillation statistics");
  if (c.grad) piece_grad_kernel<T, REST><<<grid, kPieceThreads, 0, ctx->stream>>>(c, found);
  else finish_kernel<T, REST><<<blocks, kPieceThreads, 0, ctx->stream>>>(c, found);
  hp::check_launch("distillation losses");
  return blocks;
}

}  // namespace

extern "C" {

int hp_distillation_loss(hp_ctx* ctx, int dtype, int index_dtype, const void* logits, const void* indices, const void* teacher,
                         const void* teacher_rest, const void* mask, void* loss, void* losses, void* grad, int64_t rows,
                         int64_t vocab, int64_t entries, double temperature, double count) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::require(dtype == HP_F32 || dtype == HP_F64, "logits must be float32 or float64");
    hp::require(index_dtype == HP_I32 || index_dtype == HP_I64, "indices must be int32 or int64");
    hp::require(rows >= 0 && vocab > 0 && entries > 0 && entries <= 1024, "extents out of range");
    hp::require(temperature > 0 && temperature < __builtin_huge_val() && 1 / temperature < __builtin_huge_val(), "temperature out of range");
    hp::require(loss && (rows == 0 || (logits && indices && teacher && losses)), "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      hp::Scratch scratch(ctx);
      Call<T> c{};
      c.logits = static_cast<const T*>(logits);
      c.mask = static_cast<const uint8_t*>(mask);
      c.rows = rows;
      c.vocab = vocab;
      c.grad = static_cast<T*>(grad);
      c.loss = static_cast<T*>(loss);
      c.indices = indices;
      c.wide_indices = index_dtype == HP_I64;
      c.entries = int(entries);
      c.teacher = static_cast<const T*>(teacher);
      c.teacher_rest = static_cast<const T*>(teacher_rest);
      c.losses = static_cast<T*>(losses);
      c.temperature = temperature;
      c.inverse = 1 / temperature;
      if (count > 0) c.scale_value = 1 / count;
      else if (!mask) c.scale_value = 1.0 / double(std::max<int64_t>(rows, 1));
      else c.count_here = rows > 0;
      int64_t sums = 0;
      if (rows) sums = teacher_rest ? rows_pass<T, true>(ctx, scratch, c) : rows_pass<T, false>(ctx, scratch, c);
      final_loss(ctx, c, sums);
    });
  });
}

}  // extern "C"
