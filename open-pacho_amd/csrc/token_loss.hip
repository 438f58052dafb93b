// Losses of rows of logits: token log-probabilities, the clipped policy loss and
// the preference loss, and their gradients.
//
//   log p_y = z_y - m - log S,  m = max z,  S = sum_j exp(z_j - m)
//   dL/dz_j = w (1[j = y] - exp(z_j - m) / S)  where w = dL / d log p_y
//
// so that a row needs its statistics (m, S), one scalar w that follows from
// log p_y, and a pass that writes. Bound: HBM, each logit read once and each
// gradient written once where a row can stay in registers meanwhile:
//   - row_kernel, short_row_kernel: a team of L threads holds a whole row in K
//     vectors of 16 bytes each and computes m and S from registers (the terms
//     exp(z - m) replace the logits there), then the loss of its token and the
//     gradient;
//   - rows that no team holds, or so few of them that teams would leave the chip
//     idle, are cut into pieces (stats_kernel), whose (m, S) meet per row
//     (finish_kernel, policy_grad_kernel), and are read again for the gradient.
//     The preference loss needs this second reading (grad_kernel) in any case: w
//     depends on every token of both responses.
// Sums over a row are float (double of doubles) in a tree over lanes, a lane's
// vectors one after the other, and a lane's pieces of a very long row in double; the
// loss sums are double. Every order is fixed, so results repeat bit for bit.
//
// A row that the mask leaves out is not read. Pieces and teams pad with -inf,
// which adds nothing to S; the reference of a piece that is all -inf is 0, so
// that it adds 0 and no NaN. NaN and +inf logits make S NaN.
#include "token_rows.h"

namespace {

// exp and exp - 1 of a difference of log-probabilities formed in 64 bits, to a T's
// precision: a float takes the exponential of x rounded to a float and puts what that
// cuts off back to first order, exp(near + d) = exp(near) (1 + d). Without it the result
// would be off by up to |x| / 2 units of rounding. exp(-inf) and results past the type
// have nothing to put back.
__device__ __forceinline__ double exp_difference(float, double x) {
  const float near = float(x), r = expf(near);
  return r < __builtin_huge_valf() && x > -128 ? double(r) + double(r) * (x - double(near)) : double(r);
}
__device__ __forceinline__ double exp_difference(double, double x) { return exp(x); }
__device__ __forceinline__ double expm1_difference(float, double x) { return exp_difference(0.0f, x) - 1; }
__device__ __forceinline__ double expm1_difference(double, double x) { return expm1(x); }

// grown = exp(x) - 1 and excess = exp(x) - 1 - x of such a difference, both with a T's
// digits. Near 0 the difference of x and grown would lose excess's, which is some
// x^2 / 2 there: it is the series x^2/2 (1 + x/3 (1 + x/4 (...))), whose first term left
// out is below 2^-27 of it for floats up to 2 and 2^-54 for doubles up to 1. Beyond, the
// difference loses two bits at most.
template <typename T>
__device__ __forceinline__ void grow(double x, double& grown, double& excess) {
  constexpr int kTerms = sizeof(T) == 4 ? 15 : 18;
  if (fabs(x) < (sizeof(T) == 4 ? 2.0 : 1.0)) {
    double rest = 1;
#pragma unroll
    for (int k = kTerms; k > 2; --k) rest = __builtin_fma(x * (1.0 / k), rest, 1.0);
    excess = 0.5 * x * x * rest;
    grown = x + excess;
  } else {
    grown = expm1_difference(T(0), x);
    // Infinite where the policy gives a token no probability; grown - x would be NaN.
    excess = grown == __builtin_huge_val() ? grown : grown - x;
  }
}

// The values of one call; pointers that it does not have are null.
template <typename T>
struct Call : LossCall<T> {
  using LossCall<T>::logits;
  using LossCall<T>::rows;
  using LossCall<T>::vocab;
  const void* targets;
  int wide_targets;  // int64, else int32
  T* log_probs;
  double* exact;  // the log-probabilities in 64 bits (null: not wanted)
  // Policy loss (old set).
  const T *old, *advantages, *reference;
  unsigned divide, period;  // row r's advantage is number (r / divide) % period
  double low, high, kl;     // 1 - clip below, 1 + clip above, weight of the KL term
  // Statistics of every row for a later gradient pass (null: not wanted).
  T *tops, *inverses, *weights;
  // Preference loss: a weight for every `tokens` rows in place of one each.
  int64_t tokens;

  __device__ int64_t target(int64_t row) const {
    return wide_targets ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
  }
  // NaN outside the vocabulary.
  __device__ T logit(int64_t row, int64_t y) const { return y >= 0 && y < vocab ? logits[row * vocab + y] : T(__builtin_nan("")); }
  // The log-probability of a target. From here on a token's terms are differences in
  // 64 bits: float32 would lose digits of the ratio and of a pair's margin.
  __device__ double log_prob(T logit, T top, T total) const { return (double(logit) - double(top)) - log_wide(total); }
  __device__ void keep(int64_t row, double value, T top, T total) const {
    log_probs[row] = T(value);
    if (exact) exact[row] = value;
    if (tops) tops[row] = top, inverses[row] = T(1) / total;
  }
  __device__ void leave_out(int64_t row) const {
    log_probs[row] = T(0);
    if (exact) exact[row] = 0;
  }
  __device__ T advantage(int64_t row) const {
    if (divide == 1 && period == rows) return advantages[row];
    return advantages[unsigned(row) / divide % period];
  }
};

// What a row's token brings to the policy loss. Short rows read it and the target's
// logit before their own logits (2^20 x 18: 54 us, after the statistics 59), others
// where they need it: all else would wait for the target (8192 x 32000: 380 us, 355 so).
template <typename T>
struct Token {
  T old = T(0), advantage = T(0), reference = T(0);

  __device__ __forceinline__ void read(const Call<T>& c, int64_t row) {
    old = c.old[row];
    advantage = c.advantage(row);
    if (c.reference) reference = c.reference[row];
  }
};

// The policy loss of a token and its derivative by the log-probability.
template <typename T>
__device__ __forceinline__ void policy_token(const Call<T>& c, const Token<T>& token, double log_prob, double& loss, double& slope) {
  const double advantage = token.advantage;
  const double ratio = exp_difference(T(0), log_prob - double(token.old));
  const double free = ratio * advantage;
  // Not fmin/fmax: a NaN ratio stays NaN.
  const double within = ratio < c.low ? c.low : ratio > c.high ? c.high : ratio;
  const double held = within * advantage;
  const bool stopped = free > held;
  loss = -(stopped ? held : free);
  slope = stopped ? 0.0 : -free;
  if (c.reference) {
    double grown, excess;
    grow<T>(double(token.reference) - log_prob, grown, excess);
    loss += c.kl * excess;
    slope -= c.kl * grown;
  }
}

// LOSS: the policy loss and, unless c.grad is null, its gradient; else the
// statistics alone, which leave the logits in the caches for the gradient's pass.
// Floats in 8 vectors a lane and more leave room for four waves a SIMD (128 registers):
// four workgroups of 256 threads and two of 512, one of which loads while the other
// waits at its barriers; of 1024 threads it is one, which loads and then stores. 256
// threads with 16 vectors each take three workgroups.
template <typename T, int L, int K, bool LOSS>
__global__ __launch_bounds__(L > 256 ? L : 256, sizeof(T) == 8 || K < 8 ? 1 : L == 256 && K == 16 ? 3 : 4) void row_kernel(Call<T> c) {
  constexpr int kTeams = L > 256 ? 1 : 256 / L;
  using S = Share<T, L, K>;
  __shared__ Meet<T, S::kDeep> meet;
  const int lane = kTeams == 1 ? int(threadIdx.x) : threadIdx.x % L, team = kTeams == 1 ? 0 : threadIdx.x / L;
  const int length = int(c.vocab);
  const double factor = LOSS ? scale_of(c) : 1.0;
  double sum = 0;
  int turn = 0;
  // Teams of several waves are alone in their workgroup: the loop and the
  // branches on a row are uniform where they pass a barrier.
  for (int64_t row = int64_t(blockIdx.x) * kTeams + team; row < c.rows; row += int64_t(gridDim.x) * kTeams) {
    T* out = LOSS && c.grad ? c.grad + row * c.vocab : nullptr;
    S share;
    if (!c.kept(row)) {
      if (lane == 0) c.leave_out(row);
      if (out) {
        share.each(length, lane, [](T& v, int, int) { v = T(0); });
        share.store(out, length, lane);
      }
      continue;
    }
    share.template load<LOSS>(c.logits + row * c.vocab, length, lane);
    const int64_t y = c.target(row);
    T tops[S::kDeep], top, total;
    share.statistics(length, lane, meet, turn, tops, top, total);
    turn ^= 1;
    const double log_prob = c.log_prob(c.logit(row, y), top, total);
    if (lane == 0) c.keep(row, log_prob, top, total);
    if constexpr (LOSS) {
      Token<T> token;
      token.read(c, row);
      double loss, slope;
      policy_token(c, token, log_prob, loss, slope);
      if (lane == 0) sum += loss;
      if (!out) continue;
      const T w = T(slope * factor), scale = -w * (T(1) / total);
      const int at = y >= 0 && y < c.vocab ? int(y) : -1;
      share.each(length, lane, [&](T& v, int i, int d) { v = v * (scale * S::part(tops[d], top)) + (i == at ? w : T(0)); });
      share.store(out, length, lane);
    }
  }
  if constexpr (LOSS) leave_loss(c, workgroup_sum(sum), factor, blockIdx.x, gridDim.x);
}

// Rows that a team of L <= 64 lanes holds in K <= 2 vectors a lane (4 of doubles), B of
// them at a time: more loads in flight, and lane b forms the terms of the token of row b,
// so that a wave forms those of all its rows at once where every lane of a team would
// form them again for each row. 2^20 x 18 with the gradient: 54 us, one row at a time
// 85; 2^18 x 200: 104 and 155. With K = 4 the registers of a second row of
// floats cost more waves than its loads gain: 2^16 x 1000 takes 102 us so and 96 in
// row_kernel; of doubles, whose terms weigh more, 2^16 x 400 takes 125 and 139.
// LOSS: as for row_kernel.
template <typename T, int L, int K, int B, bool LOSS>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 4 : 1) void short_row_kernel(Call<T> c) {
  static_assert(B <= L && L <= 64, "a lane for each row of a team");
  constexpr int kTeams = 256 / L;
  using S = Share<T, L, K>;
  const int lane = threadIdx.x % L, team = threadIdx.x / L, first_lane = (threadIdx.x & 63) - lane;
  const int length = int(c.vocab);
  const double factor = LOSS ? of_wave(scale_of(c)) : 1.0;
  double sum = 0;
  __shared__ Meet<T, S::kDeep> meet;  // teams within a wave leave it alone
  for (int64_t base = int64_t(blockIdx.x) * (kTeams * B) + team; base < c.rows; base += int64_t(gridDim.x) * (kTeams * B)) {
    const int64_t own = base + lane * kTeams;
    const bool has = lane < B && own < c.rows, keeps = has && c.kept(own);
    Token<T> token;
    T logit = T(0);
    int at = -1;
    if (keeps) {
      const int64_t y = c.target(own);
      if (y >= 0 && y < c.vocab) at = int(y);
      logit = c.logit(own, y);
      if constexpr (LOSS) token.read(c, own);
    }
    S share[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int64_t row = base + b * kTeams;
      if (row < c.rows && c.kept(row)) share[b].template load<LOSS>(c.logits + row * c.vocab, length, lane);
      else share[b].clear();
    }
    T top = T(0), total = T(0);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      T tops[1], row_top, row_total;
      share[b].statistics(length, lane, meet, 0, tops, row_top, row_total);
      if (lane == b) top = row_top, total = row_total;
    }
    T w = T(0), scale = T(0);
    if (keeps) {
      const double log_prob = c.log_prob(logit, top, total);
      c.keep(own, log_prob, top, total);
      if constexpr (LOSS) {
        double loss, slope;
        policy_token(c, token, log_prob, loss, slope);
        sum += loss;
        w = T(slope * factor);
        scale = -w * (T(1) / total);
      }
    } else if (has) {
      c.leave_out(own);
    }
    if (!LOSS || !c.grad) continue;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      // A row that is not read has terms and weights of 0.
      const T row_w = __shfl(w, first_lane + b, 64), row_scale = __shfl(scale, first_lane + b, 64);
      const int row_at = __shfl(at, first_lane + b, 64);
      const int64_t row = base + b * kTeams;
      if (row >= c.rows) continue;
      share[b].each(length, lane, [&](T& v, int i, int) { v = v * row_scale + (i == row_at ? row_w : T(0)); });
      share[b].store(c.grad + row * c.vocab, length, lane);
    }
  }
  if constexpr (LOSS) leave_loss(c, workgroup_sum(sum), factor, blockIdx.x, gridDim.x);
}

// (m, S) of one piece of a row: parts[row * pieces + piece].
template <typename T, bool STREAM>
__global__ __launch_bounds__(kPieceThreads) void stats_kernel(Call<T> c, T* __restrict__ part_tops,
                                                              T* __restrict__ part_totals, int pieces,
                                                              int piece) {
  __shared__ Meet<T, 1> meet;
  int turn = 0;
  for (int64_t part = blockIdx.x; part < c.rows * pieces; part += gridDim.x) {
    const int64_t row = part / pieces;
    if (!c.kept(row)) continue;
    const int64_t start = (part - row * pieces) * piece;
    const int length = piece_end(c.vocab - start, piece);
    T tops[1], top, total;
    Share<T, kPieceThreads, kPieceLoads> share;
    share.template load<STREAM>(c.logits + row * c.vocab + start, length, threadIdx.x);
    share.statistics(length, threadIdx.x, meet, turn, tops, top, total);
    turn ^= 1;
    if (threadIdx.x == 0) part_tops[part] = top, part_totals[part] = total;
  }
}

// The pieces' statistics of a row meet, and with them its token's terms. LOSS: the
// policy loss, a workgroup per row, as wide as policy_grad_kernel, so that both add
// the losses in one order; else a wave per row (8192 rows: 5.1 us, a workgroup each 7.0).
template <typename T, bool LOSS>
__global__ __launch_bounds__(kPieceThreads) void finish_kernel(Call<T> c, const T* __restrict__ part_tops,
                                                               const T* __restrict__ part_totals, int pieces) {
  const double factor = LOSS ? scale_of(c) : 1.0;
  const int64_t row = LOSS ? blockIdx.x : blockIdx.x * int64_t(kPieceThreads / 64) + (threadIdx.x >> 6);
  const bool writes = (LOSS ? threadIdx.x : threadIdx.x & 63) == 0;
  if (!LOSS && row >= c.rows) return;
  double loss = 0;
  if (c.kept(row)) {
    T top, total;
    join_pieces(part_tops + row * pieces, part_totals + row * pieces, pieces, top, total);
    const double log_prob = c.log_prob(c.logit(row, c.target(row)), top, total);
    if (writes) c.keep(row, log_prob, top, total);
    if constexpr (LOSS) {
      Token<T> token;
      token.read(c, row);
      double slope;
      policy_token(c, token, log_prob, loss, slope);
    }
  } else if (writes) {
    c.leave_out(row);
  }
  if constexpr (LOSS) leave_loss(c, loss, factor, blockIdx.x, gridDim.x);
}

// The gradient of one piece of a row from the row's statistics and weight.
template <typename T, int L, int K>
__global__ __launch_bounds__(256) void grad_kernel(Call<T> c, int pieces, int piece) {
  constexpr int kTeams = 256 / L;
  const int lane = kTeams == 1 ? int(threadIdx.x) : threadIdx.x % L, team = kTeams == 1 ? 0 : threadIdx.x / L;
  for (int64_t part = int64_t(blockIdx.x) * kTeams + team; part < c.rows * pieces; part += int64_t(gridDim.x) * kTeams) {
    const int64_t row = part / pieces;
    const int64_t start = (part - row * pieces) * piece;
    const int length = piece_end(c.vocab - start, piece);
    Share<T, L, K> share;
    if (c.kept(row)) {
      share.template load<true>(c.logits + row * c.vocab + start, length, lane);
      const int64_t y = c.target(row) - start;
      const int at = y >= 0 && y < length ? int(y) : -1;
      const T w = c.weights[row / c.tokens], scale = -w * c.inverses[row], top = c.tops[row];
      share.each(length, lane, [&](T& v, int i, int) { v = hpd::exp_down(v - top) * scale + (i == at ? w : T(0)); });
    } else {
      share.each(length, lane, [](T& v, int, int) { v = T(0); });
    }
    share.store(c.grad + row * c.vocab + start, length, lane);
  }
}

// The same for the policy loss, from the statistics of the row's pieces: every
// workgroup joins them and forms the token's terms for itself, and that of the
// first piece leaves the token's log-probability and loss.
template <typename T>
__global__ __launch_bounds__(kPieceThreads) void policy_grad_kernel(Call<T> c, const T* __restrict__ part_tops,
                                                                    const T* __restrict__ part_totals, int pieces, int piece) {
  const double factor = scale_of(c);
  for (int64_t part = blockIdx.x; part < c.rows * pieces; part += gridDim.x) {
    const int64_t row = part / pieces;
    const bool first = part == row * pieces;
    const int64_t start = (part - row * pieces) * piece;
    const int length = piece_end(c.vocab - start, piece), lane = threadIdx.x;
    T* out = c.grad + row * c.vocab + start;
    double loss = 0;
    Share<T, kPieceThreads, kPieceLoads> share;
    if (c.kept(row)) {
      share.template load<true>(c.logits + row * c.vocab + start, length, lane);
      T top, total;
      join_pieces(part_tops + row * pieces, part_totals + row * pieces, pieces, top, total);
      const int64_t y = c.target(row);
      const double log_prob = c.log_prob(c.logit(row, y), top, total);
      if (first && lane == 0) c.keep(row, log_prob, top, total);
      Token<T> token;
      token.read(c, row);
      double slope;
      policy_token(c, token, log_prob, loss, slope);
      const int at = y >= start && y < start + length ? int(y - start) : -1;
      const T w = T(slope * factor), scale = -w * (T(1) / total);
      share.each(length, lane, [&](T& v, int i, int) { v = hpd::exp_down(v - top) * scale + (i == at ? w : T(0)); });
    } else {
      if (first && lane == 0) c.leave_out(row);
      share.each(length, lane, [](T& v, int, int) { v = T(0); });
    }
    share.store(out, length, lane);
    if (first) leave_loss(c, loss, factor, unsigned(row), unsigned(c.rows));
  }
}

// A workgroup per pair: the responses' log-probabilities, the pair's loss and
// its derivatives by them.
template <typename T>
__global__ __launch_bounds__(256) void pair_kernel(Call<T> c, const T* __restrict__ reference, int64_t pairs, double beta,
                                                   double smoothing, T* __restrict__ sums_out) {
  const int64_t rows[2] = {int64_t(blockIdx.x), pairs + blockIdx.x};
  const double known[2] = {double(reference[rows[0]]), double(reference[rows[1]])};
  double sums[2] = {0, 0}, ratio[2];
  for (int64_t t = threadIdx.x; t < c.tokens; t += 256) {
    for (int side = 0; side < 2; ++side) sums[side] += c.exact[rows[side] * c.tokens + t];
  }
  for (int side = 0; side < 2; ++side) {
    const double sum = workgroup_sum(sums[side]);
    if (threadIdx.x == 0) sums_out[rows[side]] = T(sum);
    ratio[side] = sum - known[side];
  }
  const double margin = beta * (ratio[0] - ratio[1]);
  // -log sigmoid(x) = max(-x, 0) + log(1 + exp(-|x|)), with a NaN margin kept.
  const double small = exp(-fabs(margin)), soft = log1p(small), large = 1.0 / (1.0 + small);
  const double yes = margin >= 0 ? large : small * large, no = margin >= 0 ? small * large : large;
  // A side of weight 0 is left out: where a response has probability 0 it is infinite.
  const double won = smoothing < 1 ? (1 - smoothing) * ((margin < 0 ? -margin : 0.0) + soft) : 0.0;
  const double lost = smoothing > 0 ? smoothing * ((margin > 0 ? margin : 0.0) + soft) : 0.0;
  const double loss = won + lost;
  if (c.weights && threadIdx.x == 0) {
    const double slope = beta * (smoothing * yes - (1 - smoothing) * no) / double(pairs);
    c.weights[blockIdx.x] = T(slope);
    c.weights[pairs + blockIdx.x] = T(-slope);
  }
  leave_loss(c, loss, c.scale_value, blockIdx.x, gridDim.x);
}

// ---- host ----------------------------------------------------------------------

// Whether a call takes teams. Without the gradient only for rows that a piece
// holds: more and smaller workgroups overlap better where nothing has to stay in
// registers (4096 x 32000 float32: pieces 101 us, teams 122; 2048 x 50257: 77 and
// 132; 8192 x 6000, one piece: 59).
template <typename T>
bool teams_serve(const Call<T>& c) {
  if (c.vocab <= kPieceThreads * kPieceLoads * Vec<T>::width) return true;
  return c.old && c.grad && teams_hold<T>(c.rows, c.vocab);
}

// The statistics, log-probabilities and, for the policy loss, the losses of
// every row and the gradient; returns how many sums of losses there are.
template <typename T>
int64_t rows_pass(hp_ctx* ctx, hp::Scratch& scratch, Call<T>& c) {
  unsigned blocks = 0;
  if (teams_serve(c) && with_team<T>(c.vocab, [&](auto l, auto k) {
        constexpr int L = l, K = k, threads = L > 256 ? L : 256;
        constexpr int several = sizeof(T) == 8 ? 4 : 2;  // short_row_kernel
        constexpr int B = L > 64 || K > several ? 1 : K == 4 ? 2 : 4 / K;
        constexpr bool both = L * K <= kPieceThreads * kPieceLoads;  // teams_serve()
        blocks = unsigned(std::min<int64_t>(hp::ceil_div(c.rows, threads / L * B), 16384));
        if (c.old) plan_losses(ctx, scratch, c, blocks, blocks);
        if constexpr (B > 1) {
          const auto kernel = c.old ? short_row_kernel<T, L, K, B, true> : short_row_kernel<T, L, K, B, false>;
          kernel<<<blocks, threads, 0, ctx->stream>>>(c);
        } else {
          const auto kernel = c.old || !both ? row_kernel<T, L, K, true> : row_kernel<T, L, K, !both>;
          kernel<<<blocks, threads, 0, ctx->stream>>>(c);
        }
        hp::check_launch("token rows");
      })) {
    return blocks;
  }
  const Pieces<T> pieces(c.rows, c.vocab);
  T* tops = scratch.take<T>(c.rows * pieces.count);
  T* totals = scratch.take<T>(c.rows * pieces.count);
  const unsigned grid = loop_grid(c.rows * pieces.count);
  const bool done = c.old && c.grad;  // the gradient follows from the pieces at once
  hp::require(c.rows <= hp::kMaxGrid, "too many long rows for one launch");
  blocks = unsigned(c.rows);
  if (c.old) plan_losses(ctx, scratch, c, blocks, done ? grid : blocks);
  const auto stats = c.grad ? stats_kernel<T, false> : stats_kernel<T, true>;
  stats<<<grid, kPieceThreads, 0, ctx->stream>>>(c, tops, totals, pieces.count, pieces.length);
  hp::check_launch("token statistics");
  if (done) policy_grad_kernel<T><<<grid, kPieceThreads, 0, ctx->stream>>>(c, tops, totals, pieces.count, pieces.length);
  else if (c.old) finish_kernel<T, true><<<blocks, kPieceThreads, 0, ctx->stream>>>(c, tops, totals, pieces.count);
  else finish_kernel<T, false><<<hp::ceil_div(blocks, 4u), kPieceThreads, 0, ctx->stream>>>(c, tops, totals, pieces.count);
  hp::check_launch("token losses");
  return blocks;
}

template <typename T>
void grad_pass(hp_ctx* ctx, const Call<T>& c) {
  const auto launch = [&](auto l, auto k, int pieces, int piece) {
    constexpr int L = l, K = k;
    const int64_t groups = hp::ceil_div(c.rows * pieces, 256 / L);
    grad_kernel<T, L, K><<<loop_grid(groups), 256, 0, ctx->stream>>>(c, pieces, piece);
    hp::check_launch("logits gradient");
  };
  const bool held = c.vocab <= kPieceThreads * kPieceLoads * Vec<T>::width && with_team<T>(c.vocab, [&](auto l, auto k) {
    if constexpr (l * k <= kPieceThreads * kPieceLoads) launch(l, k, 1, int(c.vocab));
  });
  if (held) return;
  const Pieces<T> pieces(c.rows, c.vocab);
  launch(std::integral_constant<int, kPieceThreads>{}, std::integral_constant<int, kPieceLoads>{}, pieces.count, pieces.length);
}

template <typename T>
Call<T> call_of(int index_dtype, const void* logits, const void* targets, const void* mask, int64_t rows, int64_t vocab) {
  Call<T> c{};
  c.logits = static_cast<const T*>(logits);
  c.targets = targets;
  c.wide_targets = index_dtype == HP_I64;
  c.mask = static_cast<const uint8_t*>(mask);
  c.rows = rows;
  c.vocab = vocab;
  c.tokens = 1;
  c.scale_value = 1;
  return c;
}

void check_call(int dtype, int index_dtype, int64_t rows, int64_t vocab) {
  hp::require(dtype == HP_F32 || dtype == HP_F64, "logits must be float32 or float64");
  hp::require(index_dtype == HP_I32 || index_dtype == HP_I64, "targets must be int32 or int64");
  hp::require(rows >= 0 && vocab > 0, "extents out of range");
}

}  // namespace

extern "C" {

int hp_token_log_probs(hp_ctx* ctx, int dtype, int index_dtype, const void* logits, const void* targets,
                       const void* mask, void* log_probs, int64_t rows, int64_t vocab) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_call(dtype, index_dtype, rows, vocab);
    if (rows == 0) return;
    hp::require(logits && targets && log_probs, "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      hp::Scratch scratch(ctx);
      Call<T> c = call_of<T>(index_dtype, logits, targets, mask, rows, vocab);
      c.log_probs = static_cast<T*>(log_probs);
      rows_pass(ctx, scratch, c);
    });
  });
}

int hp_policy_loss(hp_ctx* ctx, int dtype, int index_dtype, const void* logits, const void* actions, const void* old,
                   const void* advantages, int64_t divide, int64_t period, const void* reference, const void* mask,
                   void* loss, void* log_probs, void* grad, int64_t rows, int64_t vocab, double low, double high,
                   double kl_weight, double count) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_call(dtype, index_dtype, rows, vocab);
    hp::require(low >= 0 && high >= 0, "clip out of range");
    hp::require(divide > 0 && period > 0 && divide <= INT32_MAX && period <= INT32_MAX, "advantages repeat out of range");
    hp::require(rows <= INT32_MAX, "too many rows");
    hp::require(loss && (rows == 0 || (logits && actions && old && advantages && log_probs)), "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      hp::Scratch scratch(ctx);
      Call<T> c = call_of<T>(index_dtype, logits, actions, mask, rows, vocab);
      c.old = static_cast<const T*>(old);
      c.advantages = static_cast<const T*>(advantages);
      c.reference = static_cast<const T*>(reference);
      c.low = 1 - low;
      c.high = 1 + high;
      c.kl = kl_weight;
      c.log_probs = static_cast<T*>(log_probs);
      c.grad = static_cast<T*>(grad);
      c.loss = static_cast<T*>(loss);
      c.divide = unsigned(divide);
      c.period = unsigned(period);
      if (count > 0) c.scale_value = 1 / count;
      else if (!mask) c.scale_value = 1.0 / double(std::max<int64_t>(rows, 1));
      else c.count_here = rows > 0;
      int64_t sums = 0;
      if (rows) {
        sums = rows_pass(ctx, scratch, c);
      }
      final_loss(ctx, c, sums);
    });
  });
}

int hp_preference_loss(hp_ctx* ctx, int dtype, int index_dtype, const void* logits, const void* targets,
                       const void* reference, const void* mask, void* loss, void* sums, void* grad, int64_t pairs,
                       int64_t time, int64_t vocab, double beta, double smoothing) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::require(pairs >= 0 && time >= 0, "extents out of range");
    const int64_t rows = 2 * pairs * time;
    check_call(dtype, index_dtype, rows, vocab);
    hp::require(loss && (pairs == 0 || (reference && sums)) && (rows == 0 || (logits && targets)), "null pointer");
    hp::require(pairs <= hp::kMaxGrid, "too many pairs for one launch");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      hp::Scratch scratch(ctx);
      Call<T> c = call_of<T>(index_dtype, logits, targets, mask, rows, vocab);
      c.grad = static_cast<T*>(grad);
      c.tokens = time;
      c.loss = static_cast<T*>(loss);
      c.scale_value = 1.0 / double(std::max<int64_t>(pairs, 1));
      if (pairs) {
        c.log_probs = scratch.take<T>(rows);
        c.exact = scratch.take<double>(rows);
        if (grad) {
          c.tops = scratch.take<T>(rows);
          c.inverses = scratch.take<T>(rows);
        }
        if (rows) rows_pass(ctx, scratch, c);
        if (grad) c.weights = scratch.take<T>(2 * pairs);
        plan_losses(ctx, scratch, c, unsigned(pairs), unsigned(pairs));
        pair_kernel<T><<<unsigned(pairs), 256, 0, ctx->stream>>>(c, static_cast<const T*>(reference), pairs, beta,
                                                                 smoothing, static_cast<T*>(sums));
        hp::check_launch("preference pairs");
        if (grad && rows) grad_pass(ctx, c);
      }
      final_loss(ctx, c, pairs);
    });
  });
}

}  // extern "C"
