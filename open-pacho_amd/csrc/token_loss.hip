// Losses of rows of logits: token log-probabilities, the clipped policy loss and
// the preference loss, and their gradients.
//
//   log p_y = z_y - m - log S,  m = max z,  S = sum_j exp(z_j - m)
//   dL/dz_j = w (1[j = y] - exp(z_j - m) / S)  where w = dL / d log p_y
//
// so that a row needs its statistics (m, S), one scalar w that follows from
// log p_y, and a pass that writes. Bound: HBM, each logit read once and each
// gradient written once where a row can stay in registers meanwhile:
//   - rows are cut into pieces of kPieceThreads x kPieceLoads vectors (stats_kernel),
//     whose (m, S) meet per row (finish_kernel), and are read again for the
//     gradient (grad_kernel). The preference loss needs the second reading in any
//     case: w depends on every token of both responses.
// Sums over a row are float (double of doubles) in a tree; the loss sums are
// double. No atomics: every order is fixed, so results repeat bit for bit.
//
// A row that the mask leaves out is not read. Pieces and teams pad with -inf,
// which adds nothing to S; the reference of a piece that is all -inf is 0, so
// that it adds 0 and no NaN. NaN and +inf logits make S NaN.
#include "common.h"
#include "exponential.h"

namespace {

constexpr int kPieceThreads = 256, kPieceLoads = 8;

// What is left of a row from a piece on, as far as a piece can reach.
__device__ __forceinline__ int piece_end(int64_t left) { return left < (1 << 20) ? int(left) : 1 << 20; }

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

// The values of one call; pointers that it does not have are null.
template <typename T>
struct Call {
  const T* logits;
  const void* targets;
  int wide_targets;  // int64, else int32
  const uint8_t* mask;
  int64_t rows, vocab;
  T* log_probs;
  T* grad;
  double* exact;  // the log-probabilities in 64 bits (null: not wanted)
  // Policy loss (old set).
  const T *old, *advantages, *reference;
  double low, high, kl;  // 1 - clip below, 1 + clip above, weight of the KL term
  const double* scale;  // 1 / count in device memory, or
  double scale_value;   // on the host
  double* sums;         // a workgroup's sum of losses each
  // Statistics of every row for a later gradient pass (null: not wanted).
  T *tops, *inverses, *weights;
  // Preference loss: a weight for every `tokens` rows in place of one each.
  int64_t tokens;

  __device__ bool kept(int64_t row) const { return !mask || mask[row]; }
  __device__ int64_t target(int64_t row) const {
    return wide_targets ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
  }
  // The log-probability of the row's target, NaN outside the vocabulary. From
  // here on a token's terms are computed in 64 bits and rounded once: its ratio
  // and the margin of a pair are differences of such values, and exp of them.
  __device__ double log_prob(int64_t row, int64_t y, T top, T total) const {
    const T at = y >= 0 && y < vocab ? logits[row * vocab + y] : T(__builtin_nan(""));
    return (double(at) - double(top)) - log(double(total));
  }
  __device__ void keep(int64_t row, double value, T top, T total) const {
    log_probs[row] = T(value);
    if (exact) exact[row] = value;
    if (tops) tops[row] = top, inverses[row] = T(1) / total;
  }
  __device__ void leave_out(int64_t row) const {
    log_probs[row] = T(0);
    if (exact) exact[row] = 0;
  }
  __device__ T scaled(double w) const { return T(w * (scale ? *scale : scale_value)); }
};

// The policy loss of a token and its derivative by the log-probability.
// expm1 keeps the KL term's digits where the two policies nearly agree.
template <typename T>
__device__ __forceinline__ void policy_token(const Call<T>& c, int64_t row, double log_prob, double& loss, double& slope) {
  const double advantage = c.advantages[row];
  const double ratio = exp(log_prob - double(c.old[row]));
  const double free = ratio * advantage;
  // Not fmin/fmax: a NaN ratio stays NaN.
  const double within = ratio < c.low ? c.low : ratio > c.high ? c.high : ratio;
  const double held = within * advantage;
  const bool stopped = free > held;
  loss = -(stopped ? held : free);
  slope = stopped ? 0.0 : -free;
  if (c.reference) {
    const double apart = double(c.reference[row]) - log_prob;
    const double grown = expm1(apart);
    loss += c.kl * (grown - apart);
    slope -= c.kl * grown;
  }
}

// Reductions over a team of L neighbouring threads, every thread getting the
// result. Teams of several waves are a whole workgroup and meet in `meet`.
template <int L, typename T, typename Op>
__device__ __forceinline__ T team_reduce(T v, T* meet, Op op) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = v;
    __syncthreads();
    v = meet[0];
#pragma unroll
    for (int w = 1; w < L / 64; ++w) v = op(v, meet[w]);
  }
  return v;
}

// Vectors k * L + lane of a row of `length` elements, -inf past its end. All but
// the last L vectors of a row are whole, which the team's index k alone tells.
template <typename T, int L, int K>
__device__ __forceinline__ void load_row(const T* row, int length, int lane, T (&z)[K][Vec<T>::width]) {
  constexpr int W = Vec<T>::width;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (k * L + lane) * W;
    if ((k + 1) * L * W <= length || i + W <= length) {
      const auto v = *reinterpret_cast<const typename Vec<T>::type*>(row + i);
#pragma unroll
      for (int j = 0; j < W; ++j) z[k][j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) z[k][j] = i + j < length ? row[i + j] : -T(__builtin_huge_val());
    }
  }
}

template <typename T, int L, int K>
__device__ __forceinline__ void store_row(T* row, int length, int lane, const T (&z)[K][Vec<T>::width]) {
  constexpr int W = Vec<T>::width;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (k * L + lane) * W;
    if ((k + 1) * L * W <= length || i + W <= length) {
      typename Vec<T>::type v;
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = z[k][j];
      *reinterpret_cast<typename Vec<T>::type*>(row + i) = v;
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if (i + j < length) row[i + j] = z[k][j];
      }
    }
  }
}

// z becomes exp(z - top); top and total are those of the team's values.
template <typename T, int L, int K>
__device__ __forceinline__ void statistics(T (&z)[K][Vec<T>::width], T* meet, T& top, T& total) {
  constexpr int W = Vec<T>::width;
  T m = z[0][0];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < W; ++j) m = larger(m, z[k][j]);
  top = team_reduce<L>(m, meet, [](T a, T b) { return larger(a, b); });
  const T reference = top == -T(__builtin_huge_val()) ? T(0) : top;
  T s[W] = {};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < W; ++j) {
      z[k][j] = hpd::exp_down(z[k][j] - reference);
      s[j] += z[k][j];
    }
  T sum = s[0];
#pragma unroll
  for (int j = 1; j < W; ++j) sum += s[j];
  total = team_reduce<L>(sum, meet + 16, [](T a, T b) { return a + b; });
}

// Adds each thread's `sum` over the workgroup and leaves it at sums[blockIdx.x].
__device__ __forceinline__ void leave_sum(double sum, double* sums) {
  __shared__ double meet[16];
  sum = hpd::wave_sum(sum);
  if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (unsigned w = 1; w < blockDim.x / 64; ++w) sum += meet[w];
    sums[blockIdx.x] = sum;
  }
}

// (m, S) of one piece of a row: parts[row * pieces + piece].
template <typename T>
__global__ __launch_bounds__(kPieceThreads) void stats_kernel(Call<T> c, T* __restrict__ part_tops,
                                                              T* __restrict__ part_totals, int pieces) {
  constexpr int W = Vec<T>::width, K = kPieceLoads;
  __shared__ T meet[32];
  for (int64_t part = blockIdx.x; part < c.rows * pieces; part += gridDim.x) {
    const int64_t row = part / pieces;
    if (!c.kept(row)) continue;
    const int64_t start = (part - row * pieces) * (kPieceThreads * K * W);
    T z[K][W], top, total;
    load_row<T, kPieceThreads, K>(c.logits + row * c.vocab + start, piece_end(c.vocab - start), threadIdx.x, z);
    statistics<T, kPieceThreads, K>(z, meet, top, total);
    if (threadIdx.x == 0) part_tops[part] = top, part_totals[part] = total;
  }
}

// A wave per row: its pieces' statistics meet, and with them its token's loss.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(Call<T> c, const T* __restrict__ part_tops,
                                                     const T* __restrict__ part_totals, int pieces) {
  const int lane = threadIdx.x & 63;
  double sum = 0;
  for (int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); row < c.rows; row += int64_t(gridDim.x) * 4) {
    if (!c.kept(row)) {
      if (lane == 0) c.leave_out(row);
      continue;
    }
    const T* tops = part_tops + row * pieces;
    const T* totals = part_totals + row * pieces;
    const T none = -T(__builtin_huge_val());
    T top = none;
    for (int k = lane; k < pieces; k += 64) top = larger(top, tops[k]);
    top = team_reduce<64>(top, static_cast<T*>(nullptr), [](T a, T b) { return larger(a, b); });
    T total = T(0);
    for (int k = lane; k < pieces; k += 64) total += tops[k] == none ? totals[k] : totals[k] * hpd::exp_down(tops[k] - top);
    total = team_reduce<64>(total, static_cast<T*>(nullptr), [](T a, T b) { return a + b; });
    const double log_prob = c.log_prob(row, c.target(row), top, total);
    if (lane == 0) c.keep(row, log_prob, top, total);
    if (!c.old) continue;
    double loss, slope;
    policy_token(c, row, log_prob, loss, slope);
    if (lane == 0) {
      sum += loss;
      if (c.weights) c.weights[row] = c.scaled(slope);
    }
  }
  if (c.old) leave_sum(sum, c.sums);
}

// The gradient of one piece of a row from the row's statistics and weight.
template <typename T>
__global__ __launch_bounds__(kPieceThreads) void grad_kernel(Call<T> c, int pieces) {
  constexpr int W = Vec<T>::width, K = kPieceLoads;
  for (int64_t part = blockIdx.x; part < c.rows * pieces; part += gridDim.x) {
    const int64_t row = part / pieces;
    const int64_t start = (part - row * pieces) * (kPieceThreads * K * W);
    T* out = c.grad + row * c.vocab + start;
    T z[K][W];
    if (c.kept(row)) {
      load_row<T, kPieceThreads, K>(c.logits + row * c.vocab + start, piece_end(c.vocab - start), threadIdx.x, z);
      const int64_t y = c.target(row) - start;
    const int at = y >= 0 && y < piece_end(c.vocab - start) ? int(y) : -1;
      const T w = c.weights[row / c.tokens], share = -w * c.inverses[row], top = c.tops[row];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const int i = (k * kPieceThreads + int(threadIdx.x)) * W + j;
          z[k][j] = hpd::exp_down(z[k][j] - top) * share + (i == at ? w : T(0));
        }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < W; ++j) z[k][j] = T(0);
    }
    store_row<T, kPieceThreads, K>(out, piece_end(c.vocab - start), threadIdx.x, z);
  }
}

// 1 / max(1, set bytes of the mask), by one workgroup.
__global__ __launch_bounds__(1024) void count_kernel(const uint8_t* __restrict__ mask, int64_t rows, double* __restrict__ scale) {
  __shared__ double meet[16];
  unsigned count = 0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) count += mask[i] != 0;
  double sum = hpd::wave_sum(double(count));
  if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) sum += meet[w];
    *scale = 1.0 / (sum > 1.0 ? sum : 1.0);
  }
}

// loss = scale x the sum of the workgroups' sums, by one workgroup.
template <typename T>
__global__ __launch_bounds__(1024) void loss_kernel(const double* __restrict__ sums, int64_t n, const double* __restrict__ scale,
                                                    double scale_value, T* __restrict__ loss) {
  __shared__ double meet[16];
  double sum = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) sum += sums[i];
  sum = hpd::wave_sum(sum);
  if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) sum += meet[w];
    *loss = T(sum * (scale ? *scale : scale_value));
  }
}

// A workgroup per pair: the responses' log-probabilities, the pair's loss and
// its derivatives by them.
template <typename T>
__global__ __launch_bounds__(256) void pair_kernel(Call<T> c, const T* __restrict__ reference, int64_t pairs, double beta,
                                                   double smoothing, T* __restrict__ sums_out) {
  __shared__ double meet[2][4];
  double sum[2] = {0, 0};
  for (int side = 0; side < 2; ++side) {
    const int64_t first = (side * pairs + blockIdx.x) * c.tokens;
    for (int64_t t = threadIdx.x; t < c.tokens; t += 256) sum[side] += c.exact[first + t];
    sum[side] = hpd::wave_sum(sum[side]);
    if ((threadIdx.x & 63) == 0) meet[side][threadIdx.x >> 6] = sum[side];
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  double ratio[2];
  for (int side = 0; side < 2; ++side) {
    const int64_t at = side * pairs + blockIdx.x;
    const double total = meet[side][0] + meet[side][1] + meet[side][2] + meet[side][3];
    sums_out[at] = T(total);
    ratio[side] = total - double(reference[at]);
  }
  const double margin = beta * (ratio[0] - ratio[1]);
  // -log sigmoid(x) = max(-x, 0) + log(1 + exp(-|x|)), with a NaN margin kept.
  const double small = exp(-fabs(margin)), soft = log1p(small), large = 1.0 / (1.0 + small);
  const double yes = margin >= 0 ? large : small * large, no = margin >= 0 ? small * large : large;
  const double loss = (1 - smoothing) * ((margin < 0 ? -margin : 0.0) + soft) + smoothing * ((margin > 0 ? margin : 0.0) + soft);
  c.sums[blockIdx.x] = loss;
  if (c.weights) {
    const double slope = beta * (smoothing * yes - (1 - smoothing) * no) / double(pairs);
    c.weights[blockIdx.x] = T(slope);
    c.weights[pairs + blockIdx.x] = T(-slope);
  }
}

// ---- host ----------------------------------------------------------------------

// Temporaries of one call, returned to the pool when it ends.
class Scratch {
 public:
  explicit Scratch(hp_ctx* ctx) : ctx_(ctx) {}
  ~Scratch() {
    for (void* p : held_) {
      try {
        hp::scratch_free(ctx_, p);
      } catch (...) {  // a failing free would leave a destructor: the block stays allocated
      }
    }
  }
  template <typename T>
  T* take(int64_t count) {
    held_.reserve(held_.size() + 1);
    held_.push_back(hp::scratch_alloc(ctx_, size_t(count) * sizeof(T)));
    return static_cast<T*>(held_.back());
  }

 private:
  hp_ctx* ctx_;
  std::vector<void*> held_;
};

template <typename T>
constexpr int64_t piece_length() {
  return int64_t(kPieceThreads) * kPieceLoads * Vec<T>::width;
}

unsigned pieces_grid(int64_t rows, int64_t pieces) { return unsigned(std::min(rows * pieces, hp::kMaxGrid)); }

// The statistics, log-probabilities and, for the policy loss, the losses of
// every row, their sums in c.sums; returns how many sums.
template <typename T>
int64_t rows_pass(hp_ctx* ctx, Scratch& scratch, Call<T>& c) {
  const int64_t pieces = hp::ceil_div(c.vocab, piece_length<T>());
  T* tops = scratch.take<T>(c.rows * pieces);
  T* totals = scratch.take<T>(c.rows * pieces);
  const unsigned blocks = unsigned(std::min<int64_t>(hp::ceil_div(c.rows, 4), 4096));
  if (c.old) c.sums = scratch.take<double>(blocks);
  stats_kernel<T><<<pieces_grid(c.rows, pieces), kPieceThreads, 0, ctx->stream>>>(c, tops, totals, int(pieces));
  hp::check_launch("token statistics");
  finish_kernel<T><<<blocks, 256, 0, ctx->stream>>>(c, tops, totals, int(pieces));
  hp::check_launch("token losses");
  return blocks;
}

template <typename T>
void grad_pass(hp_ctx* ctx, const Call<T>& c) {
  const int64_t pieces = hp::ceil_div(c.vocab, piece_length<T>());
  grad_kernel<T><<<pieces_grid(c.rows, pieces), kPieceThreads, 0, ctx->stream>>>(c, int(pieces));
  hp::check_launch("logits gradient");
}

template <typename T>
void final_loss(hp_ctx* ctx, const Call<T>& c, int64_t sums, void* loss) {
  loss_kernel<T><<<1, 1024, 0, ctx->stream>>>(c.sums, sums, c.scale, c.scale_value, static_cast<T*>(loss));
  hp::check_launch("loss sum");
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

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == HP_F32) f(float(0));
  else f(double(0));
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
      Scratch scratch(ctx);
      Call<T> c = call_of<T>(index_dtype, logits, targets, mask, rows, vocab);
      c.log_probs = static_cast<T*>(log_probs);
      rows_pass(ctx, scratch, c);
    });
  });
}

int hp_policy_loss(hp_ctx* ctx, int dtype, int index_dtype, const void* logits, const void* actions, const void* old,
                   const void* advantages, const void* reference, const void* mask, void* loss, void* log_probs,
                   void* grad, int64_t rows, int64_t vocab, double low, double high, double kl_weight, double count) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_call(dtype, index_dtype, rows, vocab);
    hp::require(low >= 0 && high >= 0, "clip out of range");
    hp::require(loss && (rows == 0 || (logits && actions && old && advantages && log_probs)), "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      Scratch scratch(ctx);
      Call<T> c = call_of<T>(index_dtype, logits, actions, mask, rows, vocab);
      c.old = static_cast<const T*>(old);
      c.advantages = static_cast<const T*>(advantages);
      c.reference = static_cast<const T*>(reference);
      c.low = 1 - low;
      c.high = 1 + high;
      c.kl = kl_weight;
      c.log_probs = static_cast<T*>(log_probs);
      c.grad = static_cast<T*>(grad);
      if (count > 0) {
        c.scale_value = 1 / count;
      } else if (!mask) {
        c.scale_value = 1.0 / double(std::max<int64_t>(rows, 1));
      } else if (rows) {
        double* scale = scratch.take<double>(1);
        count_kernel<<<1, 1024, 0, ctx->stream>>>(c.mask, rows, scale);
        hp::check_launch("token count");
        c.scale = scale;
      }
      int64_t sums = 0;
      if (rows) {
        if (grad) {
          c.tops = scratch.take<T>(rows);
          c.inverses = scratch.take<T>(rows);
          c.weights = scratch.take<T>(rows);
        }
        sums = rows_pass(ctx, scratch, c);
        if (grad) grad_pass(ctx, c);
      }
      final_loss(ctx, c, sums, loss);
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
      Scratch scratch(ctx);
      Call<T> c = call_of<T>(index_dtype, logits, targets, mask, rows, vocab);
      c.grad = static_cast<T*>(grad);
      c.tokens = time;
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
        c.sums = scratch.take<double>(pairs);
        pair_kernel<T><<<unsigned(pairs), 256, 0, ctx->stream>>>(c, static_cast<const T*>(reference), pairs, beta,
                                                                 smoothing, static_cast<T*>(sums));
        hp::check_launch("preference pairs");
        if (grad && rows) grad_pass(ctx, c);
      }
      final_loss(ctx, c, pairs, loss);
    });
  });
}

}  // extern "C"
