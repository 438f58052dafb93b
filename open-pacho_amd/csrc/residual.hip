// The residual stream after a block and the next block's normed input, forward and backward.
//
//   rms(v) = v / sqrt(mean(v v) + eps)
//   stream = residual + scale gate (rms(x) post),  normed = rms(stream) weight
//
// With u = stream / rms', v = x / rms'', and the gradients of both results:
//   d = dstream + (dnormed weight - u mean(dnormed weight u)) / rms'     (of residual)
//   e = scale gate d,  dx = (e post - v mean(e post v)) / rms''
//   dweight = sum dnormed u,  dpost = sum e v,  dgate = scale d v post
//
// Bound: HBM. Forward reads two arrays and writes two, backward reads four and writes
// two (and the gate and its gradient where each token has one). A team of L threads
// holds a row in K vectors of 16 bytes of each array, so that each is read once: the
// squares of x give rms'', then those of the stream rms'. Rows that no team holds are
// read again from the caches (long_*_kernel). Backward 8 x 4096 x 2048 float32 with a gate
// for each token takes 411-424 us (5.1-5.2 TB/s), forward with one for each channel 194 (5.5 TB/s); rows that no team
// holds, 2048 x 12288, 324 and 143, 3 and 2 times what their bytes would.
//
// Backward a team (a worker) takes a run of neighbouring rows and sums over them in
// registers; the workers' sums meet in worker order (sums_kernel), so that results
// repeat bit for bit. Of gates that several rows share a worker leaves a sum for each
// group that it sees a part of: at most two, as groups are neighbouring rows too.
#include <type_traits>

#include "lanes.h"
#include "sequence.h"

namespace {

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr int width = 4;
};
template <>
struct Vec<double> {
  typedef double type __attribute__((ext_vector_type(2), aligned(8)));
  static constexpr int width = 2;
};

template <typename T>
struct Norm {
  const T *x, *weight, *post, *gate;
  const T *residual;                        // forward
  T *stream, *normed;
  const T *given, *grad_stream, *grad_normed;  // backward: the stream, the gradients
  T *dx, *d, *dgate;
  T *weight_sums, *post_sums, *gate_sums;  // of workers; two of the gate for each
  int64_t rows, channels, divide;  // rows that share a gate
  int64_t each;                    // rows of a worker
  T scale, eps, mean;              // mean: 1 / channels
  bool past;                       // backward: a call's arrays do not fit into the last cache
};

// A lane's part of a row: K vectors, L lanes apart. A vector that would pass the row's
// end moves back to end there, and one behind the end onto the last one: its values
// that another lane has as well are computed twice, alike, and are counted once
// (counts()). Rows of up to four elements have lanes of one element.
template <typename T, int L, int K>
struct Part {
  static constexpr int W = L == 4 ? 1 : Vec<T>::width;
  using V = typename std::conditional<W == 1, T, typename Vec<T>::type>::type;
  T v[K][W];

  // Unsigned: a row's address stays in scalar registers.
  __device__ __forceinline__ static unsigned at(int k, int lane) { return unsigned(k * L + lane) * W; }
  // Behind the end at() is past every place of the last vector.
  __device__ __forceinline__ static bool counts(int k, int j, unsigned length, int lane) { return start(k, length, lane) + j >= at(k, lane); }
  __device__ __forceinline__ static unsigned start(int k, unsigned length, int lane) {
    const unsigned i = at(k, lane), last = length - W;
    return i < last ? i : last;
  }

  __device__ __forceinline__ void load(const T* row, unsigned length, int lane) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const V found = *reinterpret_cast<const V*>(row + start(k, length, lane));
      if constexpr (W == 1) v[k][0] = found;
      else {
#pragma unroll
        for (int j = 0; j < W; ++j) v[k][j] = found[j];
      }
    }
  }
  __device__ __forceinline__ void store(T* row, unsigned length, int lane, bool past = false) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (at(k, lane) >= length) continue;
      V to;
      if constexpr (W == 1) to = v[k][0];
      else {
#pragma unroll
        for (int j = 0; j < W; ++j) to[j] = v[k][j];
      }
      hpd::put(row + start(k, length, lane), to, past);
    }
  }
  // f(k, j) for every value.
  template <typename F>
  __device__ __forceinline__ static void each(F&& f) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < W; ++j) f(k, j);
  }
  __device__ __forceinline__ void clear() {
    each([&](int k, int j) { v[k][j] = T(0); });
  }
};

// Sums of N values over a team, for all of its lanes. Teams of several waves are alone
// in their workgroup and take the sets of `meet` in turn.
template <int L, int N, typename T>
__device__ __forceinline__ void team_sums(T (&v)[N], T (*meet)[N][16]) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = hpd::lane_sum<(L < 64 ? L : 64)>(v[n]);
  if constexpr (L > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) (*meet)[n][wave] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {  // lanes read a wave's each: all of them in one lane would take its registers
      v[n] = hpd::lane_sum<L / 64>((*meet)[n][threadIdx.x % (L / 64)]);
    }
  }
}

template <typename T>
__device__ __forceinline__ T inverse_rms(const Norm<T>& c, T squares) {
  return T(1) / (sizeof(T) == 4 ? T(sqrtf(float(squares * c.mean + c.eps))) : T(sqrt(double(squares * c.mean + c.eps))));
}

template <typename T, int L, int K, bool POST, bool GATE>
__global__ __launch_bounds__(L > 256 ? L : 256) void forward_kernel(Norm<T> c) {
  constexpr int kTeams = L > 256 ? 1 : 256 / L;
  using P = Part<T, L, K>;
  __shared__ T meet[2][1][16];
  const int lane = kTeams == 1 ? int(threadIdx.x) : threadIdx.x % L, team = kTeams == 1 ? 0 : threadIdx.x / L;
  const unsigned length = unsigned(c.channels);
  for (int64_t row = int64_t(blockIdx.x) * kTeams + team; row < c.rows; row += int64_t(gridDim.x) * kTeams) {
    P x, stream, other;
    x.load(c.x + row * c.channels, length, lane);
    stream.load(c.residual + row * c.channels, length, lane);
    if constexpr (POST) {
      T sum[1] = {};
      P::each([&](int k, int j) { sum[0] += P::counts(k, j, length, lane) ? x.v[k][j] * x.v[k][j] : T(0); });
      team_sums<L>(sum, &meet[0]);
      const T inner = inverse_rms(c, sum[0]);
      other.load(c.post, length, lane);
      P::each([&](int k, int j) { x.v[k][j] = x.v[k][j] * inner * other.v[k][j]; });
    }
    if constexpr (GATE) {
      other.load(c.gate + row / c.divide * c.channels, length, lane);
      P::each([&](int k, int j) { x.v[k][j] *= c.scale * other.v[k][j]; });
    } else {
      P::each([&](int k, int j) { x.v[k][j] *= c.scale; });
    }
    T sum[1] = {};
    P::each([&](int k, int j) {
      stream.v[k][j] += x.v[k][j];
      sum[0] += P::counts(k, j, length, lane) ? stream.v[k][j] * stream.v[k][j] : T(0);
    });
    stream.store(c.stream + row * c.channels, length, lane);
    team_sums<L>(sum, &meet[1]);
    // Without a first sum the second's set is all there is: a barrier before the next row's.
    if constexpr (!POST && L > 64) __syncthreads();
    const T outer = inverse_rms(c, sum[0]);
    other.load(c.weight, length, lane);
    P::each([&](int k, int j) { stream.v[k][j] = stream.v[k][j] * outer * other.v[k][j]; });
    stream.store(c.normed + row * c.channels, length, lane);
  }
}

// Where worker w leaves its sum of the gate of group g: the group that its first row
// is in comes first.
__device__ __forceinline__ int64_t gate_slot(int64_t worker, int64_t group, int64_t divide, int64_t each) {
  return 2 * worker + (group * divide > worker * each ? 1 : 0);
}

// Backward's waves a SIMD, for the registers of K vectors of each array and sum.
template <int K, bool ALL>
constexpr int kWaves = K > 2 ? 2 : K == 2 && ALL ? 3 : 4;

// GATE: 0 none, 1 one for each row, 2 shared by rows.
template <typename T, int L, int K, bool POST, int GATE>
__global__ __launch_bounds__(L > 256 ? L : 256, (kWaves<K, (POST && GATE == 2)>)) void backward_kernel(Norm<T> c) {
  constexpr int kTeams = L > 256 ? 1 : 256 / L;
  using P = Part<T, L, K>;
  constexpr int N = POST ? 3 : 2;
  __shared__ T meet[N][16], meet_one[1][16];
  const int lane = kTeams == 1 ? int(threadIdx.x) : threadIdx.x % L, team = kTeams == 1 ? 0 : L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / L) : threadIdx.x / L;
  const unsigned length = unsigned(c.channels);
  const int64_t worker = int64_t(blockIdx.x) * kTeams + team, first = worker * c.each;
  if (first >= c.rows) return;  // whole teams; those of several waves are whole workgroups
  const int64_t end = first + c.each < c.rows ? first + c.each : c.rows;
  P weight_sum, post_sum, gate_sum;
  weight_sum.clear(), post_sum.clear(), gate_sum.clear();
  P x, u, d, dn, next_x, next_u, next_d, next_dn;
  const auto load = [&](int64_t row) __attribute__((always_inline)) {
    const int64_t start = row * c.channels;
    next_u.load(c.given + start, length, lane);
    next_dn.load(c.grad_normed + start, length, lane);
    next_x.load(c.x + start, length, lane);
    next_d.load(c.grad_stream + start, length, lane);
  };
  int64_t group = GATE == 2 ? first / c.divide : 0, next = (group + 1) * c.divide;  // a shared gate's and its end
  constexpr bool kAhead = K == 1;  // a row ahead where there are registers for it
  if (kAhead) load(first);
  for (int64_t row = first; row < end; ++row) {
    const int64_t start = row * c.channels;
    if (!kAhead) load(row);
    x = next_x, u = next_u, d = next_d, dn = next_dn;
    if (kAhead) load(row + 1 < end ? row + 1 : row);
    P other;
    other.load(c.weight, length, lane);
    T sums[N] = {};
    P::each([&](int k, int j) {
      const bool counts = P::counts(k, j, length, lane);
      sums[0] += counts ? u.v[k][j] * u.v[k][j] : T(0);
      sums[1] += counts ? u.v[k][j] * (dn.v[k][j] * other.v[k][j]) : T(0);
      if constexpr (POST) sums[N - 1] += counts ? x.v[k][j] * x.v[k][j] : T(0);
    });
    if constexpr (L > 64) __syncthreads();  // the row before has read its sums
    team_sums<L>(sums, &meet);
    const T outer = inverse_rms(c, sums[0]), along = sums[1] * outer * c.mean;
    P::each([&](int k, int j) {
      const T unit = u.v[k][j] * outer;
      weight_sum.v[k][j] += dn.v[k][j] * unit;
      d.v[k][j] += outer * (dn.v[k][j] * other.v[k][j] - unit * along);
    });
    d.store(c.d + start, length, lane, c.past);
    // From here on u holds the unit of x, or x itself, and dn the gradient of what the gate multiplies.
    T inner = T(1);
    if constexpr (POST) inner = inverse_rms(c, sums[N - 1]);
    P gate;
    if constexpr (GATE != 0) gate.load(GATE == 1 ? c.gate + start : c.gate + group * c.channels, length, lane);
    if constexpr (POST) other.load(c.post, length, lane);
    T sum[1] = {};
    P::each([&](int k, int j) {
      T e = d.v[k][j] * c.scale;
      T y = x.v[k][j];
      if constexpr (POST) y = x.v[k][j] * inner * other.v[k][j];
      if constexpr (GATE != 0) {
        const T part = e * y;
        e *= gate.v[k][j];
        if constexpr (GATE == 1) gate.v[k][j] = part;
        else gate_sum.v[k][j] += part;
      }
      if constexpr (POST) {
        const T unit = x.v[k][j] * inner;
        post_sum.v[k][j] += e * unit;
        e *= other.v[k][j];
        sum[0] += P::counts(k, j, length, lane) ? e * unit : T(0);
        x.v[k][j] = unit;
      }
      dn.v[k][j] = e;
    });
    if constexpr (GATE == 1) gate.store(c.dgate + start, length, lane, c.past);
    if constexpr (POST) {
      team_sums<L>(sum, &meet_one);
      const T shared = sum[0] * c.mean;
      P::each([&](int k, int j) { dn.v[k][j] = inner * (dn.v[k][j] - x.v[k][j] * shared); });
    }
    dn.store(c.dx + start, length, lane, c.past);
    if constexpr (GATE == 2) {
      if (row + 1 == end || row + 1 == next) {
        const bool whole = group * c.divide >= first && next <= end;
        gate_sum.store(whole ? c.dgate + group * c.channels : c.gate_sums + gate_slot(worker, group, c.divide, c.each) * c.channels, length, lane);
        gate_sum.clear();
        if (row + 1 == next) ++group, next += c.divide;
      }
    }
  }
  weight_sum.store(c.weight_sums + worker * c.channels, length, lane);
  if constexpr (POST) post_sum.store(c.post_sums + worker * c.channels, length, lane);
}

// ---- rows that no team holds: a workgroup each, which reads them again ----------------

constexpr int kLong = 1024;

template <typename T, int N, typename F>
__device__ __forceinline__ void long_sums(int64_t length, T (&sums)[N], T (*meet)[N][16], F&& f) {
#pragma unroll
  for (int n = 0; n < N; ++n) sums[n] = T(0);
  for (int64_t i = threadIdx.x; i < length; i += kLong) f(i, sums);
  __syncthreads();  // earlier sums have been read
  team_sums<kLong>(sums, meet);
}

template <typename T>
__global__ __launch_bounds__(kLong) void long_forward_kernel(Norm<T> c) {
  __shared__ T meet[1][16];
  for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const int64_t start = row * c.channels;
    const T *x = c.x + start, *residual = c.residual + start, *gate = c.gate ? c.gate + row / c.divide * c.channels : nullptr;
    T *stream = c.stream + start, *normed = c.normed + start;
    T inner = T(1), sum[1];
    if (c.post) {
      long_sums<T, 1>(c.channels, sum, &meet, [&](int64_t i, T(&s)[1]) { s[0] += x[i] * x[i]; });
      inner = inverse_rms(c, sum[0]);
    }
    // A thread reads the stream again where it wrote it.
    long_sums<T, 1>(c.channels, sum, &meet, [&](int64_t i, T(&s)[1]) {
      T y = x[i];
      if (c.post) y = y * inner * c.post[i];
      y *= gate ? c.scale * gate[i] : c.scale;
      const T value = residual[i] + y;
      stream[i] = value;
      s[0] += value * value;
    });
    const T outer = inverse_rms(c, sum[0]);
    for (int64_t i = threadIdx.x; i < c.channels; i += kLong) normed[i] = stream[i] * outer * c.weight[i];
  }
}

// A worker's sums stand in memory, each thread's own places.
template <typename T>
__global__ __launch_bounds__(kLong) void long_backward_kernel(Norm<T> c) {
  __shared__ T meet[3][16], meet_one[1][16];
  const int64_t worker = blockIdx.x, first = worker * c.each;
  const int64_t end = first + c.each < c.rows ? first + c.each : c.rows;
  T *weight_sum = c.weight_sums + worker * c.channels, *post_sum = c.post ? c.post_sums + worker * c.channels : nullptr;
  for (int64_t row = first; row < end; ++row) {
    const int64_t start = row * c.channels, group = c.gate ? row / c.divide : 0, next = (group + 1) * c.divide;
    const T *x = c.x + start, *u = c.given + start, *dn = c.grad_normed + start, *ds = c.grad_stream + start;
    const T* gate = c.gate ? c.gate + group * c.channels : nullptr;
    T *dx = c.dx + start, *d = c.d + start, *dgate = nullptr;
    if (gate && c.divide == 1) dgate = c.dgate + start;
    else if (gate) {
      const bool whole = group * c.divide >= first && next <= end;
      dgate = whole ? c.dgate + group * c.channels : c.gate_sums + gate_slot(worker, group, c.divide, c.each) * c.channels;
    }
    const bool starts = row == first, starts_group = starts || row == group * c.divide;
    T sums[3], sum[1];
    long_sums<T, 3>(c.channels, sums, &meet, [&](int64_t i, T(&s)[3]) {
      s[0] += u[i] * u[i];
      s[1] += u[i] * (dn[i] * c.weight[i]);
      s[2] += x[i] * x[i];
    });
    const T outer = inverse_rms(c, sums[0]), along = sums[1] * outer * c.mean, inner = c.post ? inverse_rms(c, sums[2]) : T(1);
    long_sums<T, 1>(c.channels, sum, &meet_one, [&](int64_t i, T(&s)[1]) {
      const T unit = u[i] * outer, value = ds[i] + outer * (dn[i] * c.weight[i] - unit * along), v = x[i] * inner;
      weight_sum[i] = (starts ? T(0) : weight_sum[i]) + dn[i] * unit;
      d[i] = value;
      T e = value * c.scale;
      if (gate) {
        const T part = e * (c.post ? v * c.post[i] : v);
        dgate[i] = (starts_group ? T(0) : dgate[i]) + part;
        e *= gate[i];
      }
      if (c.post) {
        post_sum[i] = (starts ? T(0) : post_sum[i]) + e * v;
        e *= c.post[i];
        s[0] += e * v;
      }
      dx[i] = e;
    });
    if (c.post) {
      const T shared = sum[0] * c.mean;
      for (int64_t i = threadIdx.x; i < c.channels; i += kLong) dx[i] = inner * (dx[i] - x[i] * inner * shared);
    }
  }
}

// ---- sums of workers -----------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(1024) void sums_kernel(const T* weight_sums, T* dweight, const T* post_sums, T* dpost, int64_t workers, int64_t channels) {
  const T* parts = blockIdx.y == 0 ? weight_sums : post_sums;
  T* out = blockIdx.y == 0 ? dweight : dpost;
  hpd::add_parts(parts, channels, 0, workers, int64_t(blockIdx.x) * 64, channels, [&](int64_t i, T sum) { out[i] = sum; });
}

// Groups that more than one worker has a part of: the first of them may leave it in
// its second place, all others in their first.
template <typename T>
__global__ __launch_bounds__(1024) void gate_sums_kernel(Norm<T> c, int64_t blocks) {
  const int64_t group = blockIdx.x / blocks, column = (blockIdx.x - group * blocks) * 64;
  const int64_t low = group * c.divide / c.each, high = ((group + 1) * c.divide - 1) / c.each;
  if (low == high) return;
  T* out = c.dgate + group * c.channels;
  const T* start = c.gate_sums + gate_slot(low, group, c.divide, c.each) * c.channels;
  hpd::add_parts(c.gate_sums, 2 * c.channels, low + 1, high + 1, column, c.channels, [&](int64_t i, T sum) { out[i] = start[i] + sum; });
}

template <typename T>
__global__ __launch_bounds__(256) void zeros_kernel(T* to, int64_t n) {
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) to[i] = T(0);
}

// ---- host ----------------------------------------------------------------------------

// Calls f with the team (L, K) that holds rows of `channels`, or returns false: none does.
// Two vectors of each array a lane leave backward, with its sums, room for four waves a SIMD.
template <typename T, typename F>
bool with_team(int64_t channels, F&& f) {
  const int64_t vectors = hp::ceil_div(channels, Vec<T>::width);
#define TEAM(L, K) \
  if (L == 4 ? channels <= 4 : vectors <= L * K) return f(std::integral_constant<int, L>{}, std::integral_constant<int, K>{}), true;
  TEAM(4, 1)
  TEAM(16, 1)
  TEAM(64, 1)
  TEAM(64, 2)
  TEAM(256, 1)
  TEAM(256, 2)
  TEAM(512, 2)
  TEAM(1024, 2)
#undef TEAM
  return false;
}

template <typename T>
void forward(hp_ctx* ctx, const Norm<T>& c) {
  const bool held = with_team<T>(c.channels, [&](auto l, auto k) {
    constexpr int L = l, K = k, threads = L > 256 ? L : 256;
    const int64_t blocks = std::min<int64_t>(hp::ceil_div(c.rows, threads / L), 16384);
    const auto kernel = c.post ? (c.gate ? forward_kernel<T, L, K, true, true> : forward_kernel<T, L, K, true, false>)
                               : (c.gate ? forward_kernel<T, L, K, false, true> : forward_kernel<T, L, K, false, false>);
    kernel<<<unsigned(blocks), threads, 0, ctx->stream>>>(c);
  });
  if (!held) long_forward_kernel<T><<<unsigned(std::min<int64_t>(c.rows, 4096)), kLong, 0, ctx->stream>>>(c);
  hp::check_launch("residual norm");
}

template <typename T>
void backward(hp_ctx* ctx, Norm<T> c, T* dweight, T* dpost) {
  hp::Scratch scratch(ctx);
  // Six arrays, of which the caches would hold none to its next reader: 429 us -> 422 of 8 x 4096 x 2048 float32, and of
  // rows that are no whole lines 86 -> 74 (3 x 1367 x 1537 float64), each in turn on one card.
  c.past = c.rows * c.channels * int64_t(6 * sizeof(T)) > hp::kLastCache;
  const int64_t groups = c.gate ? c.rows / c.divide : 0;
  const auto plan = [&](int64_t most) {
    // Some rows a worker, so that the sums weigh little beside the rows, unless the chip would idle.
    c.each = std::max(hp::ceil_div(c.rows, most), std::min<int64_t>(8, hp::ceil_div(c.rows, 256)));
    const int64_t workers = hp::ceil_div(c.rows, c.each);
    c.weight_sums = scratch.take<T>(workers * c.channels);
    if (c.post) c.post_sums = scratch.take<T>(workers * c.channels);
    if (c.gate && c.divide > 1) c.gate_sums = scratch.take<T>(2 * workers * c.channels);
    return workers;
  };
  int64_t workers = 0;
  const auto launch = [&](auto l, auto k, auto shared) {
    constexpr int L = l, K = k, threads = L > 256 ? L : 256, teams = threads / L;
    const auto run = [&](auto gate) {
      const auto go = [&](auto post) {
        // As many as run at once: a second round would be a short one.
        workers = plan(int64_t(256) * (4 * kWaves<K, post && gate == 2> * 64 / threads) * teams);
        backward_kernel<T, L, K, post, gate><<<unsigned(hp::ceil_div(workers, teams)), threads, 0, ctx->stream>>>(c);
      };
      if (c.post) go(std::true_type{});
      else go(std::false_type{});
    };
    if constexpr (shared) run(std::integral_constant<int, 2>{});
    else if (c.gate) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 0>{});
  };
  const bool held = with_team<T>(c.channels, [&](auto l, auto k) {
    // Teams of several waves with one vector a lane: next rows have registers. The largest cannot grow, and the third
    // sum of shared gates does not fit its threads.
    if constexpr (l == 1024) {
      if (c.gate && c.divide > 1) launch(std::integral_constant<int, 512>{}, std::integral_constant<int, 2 * k>{}, std::true_type{});
      else launch(l, k, std::false_type{});
    } else {
      constexpr int split = l >= 256 ? k : 1;
      const std::integral_constant<int, split * l> many;
      const std::integral_constant<int, k / split> of;
      if (c.gate && c.divide > 1) launch(many, of, std::true_type{});
      else launch(many, of, std::false_type{});
    }
  });
  if (!held) {
    workers = plan(1024);
    long_backward_kernel<T><<<unsigned(workers), kLong, 0, ctx->stream>>>(c);
  }
  hp::check_launch("residual norm gradient");
  const int64_t blocks = hp::ceil_div(c.channels, 64);
  sums_kernel<T><<<dim3(unsigned(blocks), c.post ? 2 : 1), 1024, 0, ctx->stream>>>(c.weight_sums, dweight, c.post_sums, dpost, workers, c.channels);
  hp::check_launch("residual norm sums");
  if (c.gate && c.divide > 1 && workers > 1) {
    hp::require(groups * blocks <= hp::kMaxThreads / 1024, "too many gates for one launch");
    gate_sums_kernel<T><<<unsigned(groups * blocks), 1024, 0, ctx->stream>>>(c, blocks);
    hp::check_launch("residual norm gates");
  }
}

void check_norm(int dtype, int64_t rows, int64_t channels, const void* gate, int64_t divide, double scale, double eps) {
  hp::require(dtype == HP_F32 || dtype == HP_F64, "norms require float32 or float64");
  hp::require(rows >= 0 && channels > 0, "extents out of range");
  hp::require(!gate || rows == 0 || (divide > 0 && rows % divide == 0), "gates do not divide the rows");
  hp::require(eps > 0 && eps < __builtin_huge_val() && scale - scale == 0, "eps or scale out of range");
}

template <typename T>
Norm<T> norm_of(const void* x, const void* weight, const void* post, const void* gate, int64_t rows, int64_t channels, int64_t divide,
                double scale, double eps) {
  Norm<T> c{};
  c.x = static_cast<const T*>(x);
  c.weight = static_cast<const T*>(weight);
  c.post = static_cast<const T*>(post);
  c.gate = static_cast<const T*>(gate);
  c.rows = rows;
  c.channels = channels;
  c.divide = gate ? divide : 1;
  c.scale = T(scale);
  c.eps = T(eps);
  c.mean = T(1.0 / double(channels));
  return c;
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == HP_F32) f(float(0));
  else f(double(0));
}

}  // namespace

extern "C" {

int hp_residual_norm(hp_ctx* ctx, int dtype, const void* x, const void* residual, const void* weight, const void* post_weight,
                     const void* gate, void* stream, void* normed, int64_t rows, int64_t channels, int64_t divide, double scale,
                     double eps) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_norm(dtype, rows, channels, gate, divide, scale, eps);
    if (rows == 0) return;
    hp::require(x && residual && weight && stream && normed, "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      Norm<T> c = norm_of<T>(x, weight, post_weight, gate, rows, channels, divide, scale, eps);
      c.residual = static_cast<const T*>(residual);
      c.stream = static_cast<T*>(stream);
      c.normed = static_cast<T*>(normed);
      forward(ctx, c);
    });
  });
}

int hp_residual_norm_grad(hp_ctx* ctx, int dtype, const void* grad_stream, const void* grad_normed, const void* x, const void* stream,
                          const void* weight, const void* post_weight, const void* gate, void* dx, void* d, void* dweight,
                          void* dpost, void* dgate, int64_t rows, int64_t channels, int64_t divide, int64_t gates, double scale,
                          double eps) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_norm(dtype, rows, channels, gate, divide, scale, eps);
    hp::require(dweight && (!post_weight || dpost) && (!gate || dgate) && gates >= 0, "null pointer");
    hp::require(!gate || rows == 0 || gates == rows / divide, "gates do not divide the rows");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      if (rows == 0) {
        const auto clear = [&](void* to, int64_t n) {
          if (to && n) zeros_kernel<T><<<unsigned(std::min<int64_t>(hp::ceil_div(n, 256), 4096)), 256, 0, ctx->stream>>>(static_cast<T*>(to), n);
        };
        clear(dweight, channels);
        if (post_weight) clear(dpost, channels);
        if (gate) clear(dgate, gates * channels);
        hp::check_launch("residual norm gradient");
        return;
      }
      hp::require(grad_stream && grad_normed && x && stream && weight && dx && d, "null pointer");
      Norm<T> c = norm_of<T>(x, weight, post_weight, gate, rows, channels, divide, scale, eps);
      c.given = static_cast<const T*>(stream);
      c.grad_stream = static_cast<const T*>(grad_stream);
      c.grad_normed = static_cast<const T*>(grad_normed);
      c.dx = static_cast<T*>(dx);
      c.d = static_cast<T*>(d);
      c.dgate = static_cast<T*>(dgate);
      backward(ctx, c, static_cast<T*>(dweight), static_cast<T*>(dpost));
    });
  });
}

}  // extern "C"
