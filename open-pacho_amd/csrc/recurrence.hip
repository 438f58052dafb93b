// Gated linear recurrence over time, forward and backward.
//
//   h_t = a_t h_{t-1} + (1 - a_t) x_t,  a_t = sigmoid(gate_t); h_{t-1} = 0 at a reset.
//
// A step is the map h -> A h + B with (A, B) = (a_t, (1 - a_t) x_t), and maps
// compose: (A2, B2) after (A1, B1) is (A2 A1, A2 B1 + B2). The gradient runs
// the other way in time on the same algebra: with the gradient g_t of h_t,
//   s_t = g_t + m_{t+1},  m_t = a_t s_t (0 at a reset)
//   dx_t = s_t (1 - a_t),  dgate_t = s_t (h_{t-1} - x_t) a_t (1 - a_t),  dinitial = m_0,
// whose step is m -> A m + B with (A, B) = (a_t, a_t g_t). A reset drops what
// comes before it by a select, not by a product: it may be infinite or NaN.
//
// Bound: HBM. Forward reads x and the gates and writes h, backward reads four
// arrays and writes two, each once. A lane owns a channel, so that a wave reads
// 64 neighbouring channels of a step at once whatever their number and
// alignment; a workgroup owns 64 channels, and its waves consecutive runs of R
// steps. Each wave loads its run into registers, composes it, leaves (A, B) in
// LDS, takes what the waves before it left, and then computes and stores its
// states: one pass over the data, one barrier for each R x waves steps. The next
// run's loads are issued before the barrier.
#include "common.h"
#include "exponential.h"

namespace {

constexpr int kMaxWaves = 8;

template <typename T>
struct Steps;
template <>
struct Steps<float> {
  static constexpr int forward = 16, backward = 8;
};
template <>
struct Steps<double> {
  static constexpr int forward = 8, backward = 4;
};

struct Extents {
  int64_t time;      // steps of a row
  int64_t total;     // rows x channels
  int64_t channels;  // of a step
  int64_t gates;     // of a step
  int64_t width;     // channels that share a gate: channels / gates
  // Backward with shared gates: lanes are laid out by heads.
  int64_t heads;  // rows x gates
  int pack;       // whole heads in a wave (width <= 64), else 1
  int pieces;     // waves that share a head (width > 64), else 1
  int piece;      // channels of a head in one wave
};

// What a lane works on: a row, a channel of it, and that channel's gate.
struct Place {
  int64_t row, channel, gate;
  bool valid;
};

__device__ __forceinline__ Place flat_place(const Extents& e, int64_t group, int lane) {
  int64_t q = group * 64 + lane;
  const bool valid = q < e.total;
  q = valid ? q : e.total - 1;  // lanes past the end load what the last one does and store nothing
  const int64_t row = q / e.channels, channel = q - row * e.channels;
  return {row, channel, channel / e.width, valid};
}

__device__ __forceinline__ Place head_place(const Extents& e, int64_t group, int lane) {
  const int64_t first = group / e.pieces * e.pack;
  const int slot = lane / e.piece, within = lane - slot * e.piece;
  const int64_t offset = (group % e.pieces) * e.piece + within;
  const bool valid = slot < e.pack && first + slot < e.heads && offset < e.width;
  const int64_t head = valid ? first + slot : e.heads - 1;
  const int64_t row = head / e.gates, gate = head - row * e.gates;
  return {row, gate * e.width + (valid ? offset : 0), gate, valid};
}

// A composed run: h -> a h + b, or h -> b where `cut` (kept in LDS as a = -1).
template <typename T>
struct Run {
  T a, b;
  bool cut;
};

template <typename T>
__device__ __forceinline__ T apply(T a, T b, T h) {
  return (a < T(0) ? T(0) : a * h) + b;
}

// R values of a column from its step t on; steps outside [0, end) hold `outside`.
template <typename T, int R>
__device__ __forceinline__ void load_steps(const T* column, int64_t stride, int64_t t, int64_t end, T outside, T (&v)[R]) {
  if (t >= 0 && t + R <= end) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = column[(t + i) * stride];
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = t + i >= 0 && t + i < end ? column[(t + i) * stride] : outside;
  }
}

// Bit i: a reset at step t + i.
template <int R>
__device__ __forceinline__ unsigned load_resets(const uint8_t* row, int64_t t, int64_t end) {
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (t + i >= 0 && t + i < end) bits |= unsigned(row[t + i] != 0) << i;
  }
  return bits;
}

template <typename T, int R, bool RESETS>
__global__ __launch_bounds__(kMaxWaves * 64) void forward_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                                 const T* __restrict__ initial,
                                                                 const uint8_t* __restrict__ resets,
                                                                 T* __restrict__ h, Extents e) {
  __shared__ T left_a[2][kMaxWaves][64], left_b[2][kMaxWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const Place at = flat_place(e, blockIdx.x, lane);
  const T* xs = x + at.row * e.time * e.channels + at.channel;
  const T* gs = gate + at.row * e.time * e.gates + at.gate;
  const uint8_t* rs = RESETS ? resets + at.row * e.time : nullptr;
  T* hs = h + at.row * e.time * e.channels + at.channel;
  T state = initial ? initial[at.row * e.channels + at.channel] : T(0);

  // Steps past the end keep the state: their gate is +inf.
  const T open = __builtin_huge_val();
  T nx[R], ng[R];
  unsigned nr = 0;
  int64_t t = int64_t(wave) * R;
  const int64_t stride = int64_t(waves) * R;
  load_steps<T, R>(xs, e.channels, t, e.time, T(0), nx);
  load_steps<T, R>(gs, e.gates, t, e.time, open, ng);
  if (RESETS) nr = load_resets<R>(rs, t, e.time);

  int turn = 0;
  for (int64_t base = 0; base < e.time; base += stride, t += stride, turn ^= 1) {
    T a[R], b[R];
    const unsigned reset = nr;
    Run<T> run{T(1), T(0), false};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      T take;
      hpd::gates(ng[i], a[i], take);
      b[i] = take * nx[i];
      const bool cut = RESETS && (reset >> i & 1);
      run.cut = run.cut || cut;
      run.b = (cut ? T(0) : a[i] * run.b) + b[i];
      run.a *= a[i];
    }
    if (base + stride < e.time) {
      load_steps<T, R>(xs, e.channels, t + stride, e.time, T(0), nx);
      load_steps<T, R>(gs, e.gates, t + stride, e.time, open, ng);
      if (RESETS) nr = load_resets<R>(rs, t + stride, e.time);
    }
    left_a[turn][wave][lane] = run.cut ? T(-1) : run.a;
    left_b[turn][wave][lane] = run.b;
    __syncthreads();
    T now = state;
    for (int w = 0; w < waves; ++w) {
      if (w == wave) now = state;
      state = apply(left_a[turn][w][lane], left_b[turn][w][lane], state);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool cut = RESETS && (reset >> i & 1);
      now = (cut ? T(0) : a[i] * now) + b[i];
      if (at.valid && t + i < e.time) hs[(t + i) * e.channels] = now;
    }
  }
}

// SHARED: gates that heads share; dgate then holds e.pieces partial sums.
template <typename T, int R, bool RESETS, bool SHARED>
__global__ __launch_bounds__(kMaxWaves * 64) void backward_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const T* __restrict__ gate, const T* __restrict__ h,
    const T* __restrict__ initial, const uint8_t* __restrict__ resets, T* __restrict__ dx, T* __restrict__ dgate,
    T* __restrict__ dinitial, Extents e) {
  __shared__ T left_a[2][kMaxWaves][64], left_b[2][kMaxWaves][64];
  __shared__ T shares[SHARED ? kMaxWaves : 1][SHARED ? R : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const Place at = SHARED ? head_place(e, blockIdx.x, lane) : flat_place(e, blockIdx.x, lane);
  const int64_t column = at.row * e.time * e.channels + at.channel;
  const int64_t gate_column = at.row * e.time * e.gates + at.gate;
  const T *xs = x + column, *hs = h + column, *ds = grad + column, *gs = gate + gate_column;
  const uint8_t* rs = RESETS ? resets + at.row * e.time : nullptr;
  const int64_t first = at.row * e.channels + at.channel;
  const T before = initial ? initial[first] : T(0);

  // Wave 0 takes the last R steps, wave 1 those before them: t is the first
  // step of a wave's run, below zero at the start of the row. Steps outside
  // the row pass the gradient on: their gate is +inf and their gradient 0.
  const T open = __builtin_huge_val();
  T nx[R], ng[R], nh[R], nd[R];
  unsigned nr = 0;
  int64_t t = e.time - int64_t(wave + 1) * R;
  const int64_t stride = int64_t(waves) * R;
  const auto load = [&](int64_t from) {
    load_steps<T, R>(xs, e.channels, from, e.time, T(0), nx);
    load_steps<T, R>(gs, e.gates, from, e.time, open, ng);
    load_steps<T, R>(ds, e.channels, from, e.time, T(0), nd);
    load_steps<T, R>(hs, e.channels, from - 1, e.time, before, nh);
    if (RESETS) nr = load_resets<R>(rs, from, e.time);
  };
  load(t);

  T carried = T(0);
  int turn = 0;
  for (int64_t base = 0; base < e.time; base += stride, t -= stride, turn ^= 1) {
    T a[R], take[R], d[R], apart[R];
    const unsigned reset = nr;
    Run<T> run{T(1), T(0), false};
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const bool cut = RESETS && (reset >> i & 1);
      hpd::gates(ng[i], a[i], take[i]);
      d[i] = nd[i];
      apart[i] = (cut ? T(0) : nh[i]) - nx[i];
      run.cut = run.cut || cut;
      run.b = cut ? T(0) : a[i] * (d[i] + run.b);
      run.a *= a[i];
    }
    if (base + stride < e.time) load(t - stride);
    left_a[turn][wave][lane] = run.cut ? T(-1) : run.a;
    left_b[turn][wave][lane] = run.b;
    __syncthreads();
    T now = carried;
    for (int w = 0; w < waves; ++w) {
      if (w == wave) now = carried;
      carried = apply(left_a[turn][w][lane], left_b[turn][w][lane], carried);
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const bool cut = RESETS && (reset >> i & 1);
      const bool inside = at.valid && t + i >= 0;
      const T slope = d[i] + now;
      now = cut ? T(0) : a[i] * slope;
      const T share = slope * apart[i] * (a[i] * take[i]);
      if (inside) dx[column + (t + i) * e.channels] = slope * take[i];
      if constexpr (SHARED) shares[wave][i][lane] = share;
      else if (inside) dgate[gate_column + (t + i) * e.gates] = share;
    }
    if constexpr (SHARED) {
      // The wave's own rows of LDS: its stores are in order before its loads.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const int64_t group = blockIdx.x;
      const int64_t head0 = group / e.pieces * e.pack;
      const int64_t left = e.width - (group % e.pieces) * e.piece;
      const int count = int(left < e.piece ? left : e.piece);
      T* out = dgate + (group % e.pieces) * (e.heads * e.time);
      for (int task = lane; task < R * e.pack; task += 64) {
        const int i = task / e.pack, slot = task - i * e.pack;
        const int64_t head = head0 + slot;
        if (head >= e.heads || t + i < 0) continue;
        T sum = T(0);
        for (int k = 0; k < count; ++k) sum += shares[wave][i][slot * e.piece + k];
        const int64_t row = head / e.gates;
        out[(row * e.time + t + i) * e.gates + (head - row * e.gates)] = sum;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (dinitial && wave == 0 && at.valid) dinitial[first] = carried;
}

// out[i] = sum over k of parts[k][i], in order.
template <typename T>
__global__ __launch_bounds__(256) void add_parts_kernel(const T* __restrict__ parts, T* __restrict__ out, int64_t n, int pieces) {
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    T sum = parts[i];
    for (int k = 1; k < pieces; ++k) sum += parts[k * n + i];
    out[i] = sum;
  }
}

Extents extents(int64_t batch, int64_t time, int64_t channels, int64_t gates) {
  hp::require(batch >= 0 && time >= 0 && channels >= 0 && gates >= 0, "negative extent");
  hp::require(channels == 0 || (gates > 0 && channels % gates == 0), "gates do not divide the channels");
  Extents e{};
  e.time = time;
  e.total = batch * channels;
  e.channels = channels;
  e.gates = gates;
  e.width = channels ? channels / gates : 1;
  e.heads = batch * gates;
  e.pieces = int(hp::ceil_div(e.width, 64));
  e.piece = int(hp::ceil_div(e.width, e.pieces));
  e.pack = 64 / e.piece;
  if (e.pieces > 1) e.pack = 1;
  return e;
}

unsigned checked_grid(int64_t groups, int threads) {
  hp::require(groups <= hp::kMaxThreads / threads, "too many channels for one launch");
  return unsigned(groups);
}

int waves_for(int64_t time, int steps) {
  int waves = 1;
  while (waves < kMaxWaves && waves * steps < time) waves *= 2;
  return waves;
}

template <typename T>
void forward(hp_ctx* ctx, const T* x, const T* gate, const T* initial, const uint8_t* resets, T* h, const Extents& e) {
  constexpr int R = Steps<T>::forward;
  const int threads = 64 * waves_for(e.time, R);
  const unsigned grid = checked_grid(hp::ceil_div(e.total, 64), threads);
  const auto kernel = resets ? forward_kernel<T, R, true> : forward_kernel<T, R, false>;
  kernel<<<grid, threads, 0, ctx->stream>>>(x, gate, initial, resets, h, e);
  hp::check_launch("recurrence forward");
}

template <typename T>
void backward(hp_ctx* ctx, const T* grad, const T* x, const T* gate, const T* h, const T* initial,
              const uint8_t* resets, T* dx, T* dgate, T* dinitial, const Extents& e) {
  constexpr int R = Steps<T>::backward;
  const bool shared = e.width > 1;
  const int64_t groups = shared ? hp::ceil_div(e.heads, e.pack) * e.pieces : hp::ceil_div(e.total, 64);
  const int threads = 64 * waves_for(e.time, R);
  const unsigned grid = checked_grid(groups, threads);
  const int64_t count = e.heads * e.time;
  T* parts = dgate;
  if (e.pieces > 1) parts = static_cast<T*>(hp::scratch_alloc(ctx, size_t(e.pieces) * size_t(count) * sizeof(T)));
  const auto kernel = shared ? (resets ? backward_kernel<T, R, true, true> : backward_kernel<T, R, false, true>)
                             : (resets ? backward_kernel<T, R, true, false> : backward_kernel<T, R, false, false>);
  kernel<<<grid, threads, 0, ctx->stream>>>(grad, x, gate, h, initial, resets, dx, parts, dinitial, e);
  const hipError_t status = hipGetLastError();
  if (e.pieces > 1) {
    if (status == hipSuccess) {
      const int64_t blocks = std::min<int64_t>(hp::ceil_div(count, 256), 4096);
      add_parts_kernel<T><<<unsigned(blocks), 256, 0, ctx->stream>>>(parts, dgate, count, e.pieces);
    }
    hp::scratch_free(ctx, parts);
  }
  hp::check_hip(status, "launch of recurrence backward");
  hp::check_launch("recurrence gate sums");
}

}  // namespace

extern "C" {

int hp_gated_recurrence(hp_ctx* ctx, int dtype, const void* x, const void* gate, const void* initial,
                        const void* resets, void* h, int64_t batch, int64_t time, int64_t channels, int64_t gates) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::require(dtype == HP_F32 || dtype == HP_F64, "recurrence requires float32 or float64");
    const Extents e = extents(batch, time, channels, gates);
    if (e.total == 0 || time == 0) return;
    hp::require(x && gate && h, "null pointer");
    const auto r = static_cast<const uint8_t*>(resets);
    if (dtype == HP_F32) {
      forward(ctx, static_cast<const float*>(x), static_cast<const float*>(gate), static_cast<const float*>(initial), r,
              static_cast<float*>(h), e);
    } else {
      forward(ctx, static_cast<const double*>(x), static_cast<const double*>(gate), static_cast<const double*>(initial),
              r, static_cast<double*>(h), e);
    }
  });
}

int hp_gated_recurrence_grad(hp_ctx* ctx, int dtype, const void* grad, const void* x, const void* gate, const void* h,
                             const void* initial, const void* resets, void* dx, void* dgate, void* dinitial,
                             int64_t batch, int64_t time, int64_t channels, int64_t gates) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::require(dtype == HP_F32 || dtype == HP_F64, "recurrence requires float32 or float64");
    const Extents e = extents(batch, time, channels, gates);
    if (e.total == 0 || time == 0) return;
    hp::require(grad && x && gate && h && dx && dgate, "null pointer");
    const auto r = static_cast<const uint8_t*>(resets);
    const auto run = [&](auto zero) {
      using T = decltype(zero);
      backward<T>(ctx, static_cast<const T*>(grad), static_cast<const T*>(x), static_cast<const T*>(gate),
                  static_cast<const T*>(h), static_cast<const T*>(initial), r, static_cast<T*>(dx),
                  static_cast<T*>(dgate), static_cast<T*>(dinitial), e);
    };
    if (dtype == HP_F32) run(float(0));
    else run(double(0));
  });
}

}  // extern "C"
