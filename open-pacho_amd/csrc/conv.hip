// A short causal convolution of each channel over time, forward and backward.
//
//   v_t = bias + sum_k w_k x_{t-K+1+k},  y_t = v_t or v_t sigmoid(v_t)
//   e_t = dy_t f'(v_t),  dx_t = sum_j w_{K-1-j} e_{t+j},  dw_k = sum_t e_t x_{t-K+1+k},  dbias = sum_t e_t
//
// Bound: HBM; forward reads an array and writes one, backward reads two and writes one.
// A thread owns a vector of 16 bytes of neighbouring channels and walks a run of steps
// with the last K inputs in registers; backward also with the K gradients of inputs that
// are not complete yet, through the K - 1 steps behind its run. So only the K - 1 steps
// around a run are read twice. What a step must not see has left the registers: a reset
// clears the inputs before it, and a count of visible steps holds its gradient back.
// Runs' sums for weights and bias meet in the runs' order. Forward 2 x 16387 x 1001 with three taps takes 40 us
// (6.5 TB/s, partly from the caches), 8 x 4096 x 2048 with four 130 (4.1 TB/s), backward 202 (4.0 TB/s); as many bytes
// of doubles 128 and 184.
#include <type_traits>

#include "exponential.h"
#include "sequence.h"

namespace {

constexpr int kMostTaps = 8;

template <typename T, int W>
struct Lane {
  typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T))));
};
template <typename T>
struct Lane<T, 1> {
  using type = T;
};

// W values of neighbouring channels.
template <typename T, int W>
struct Value {
  T v[W];

  __device__ __forceinline__ static Value of(T x) {
    Value r;
#pragma unroll
    for (int j = 0; j < W; ++j) r.v[j] = x;
    return r;
  }
  __device__ __forceinline__ static Value load(const T* at) {
    Value r;
    const auto found = *reinterpret_cast<const typename Lane<T, W>::type*>(at);
    if constexpr (W == 1) r.v[0] = found;
    else {
#pragma unroll
      for (int j = 0; j < W; ++j) r.v[j] = found[j];
    }
    return r;
  }
  __device__ __forceinline__ void store(T* at, bool past = false) const {
    typename Lane<T, W>::type to;
    if constexpr (W == 1) to = v[0];
    else {
#pragma unroll
      for (int j = 0; j < W; ++j) to[j] = v[j];
    }
    hpd::put(at, to, past);
  }
};

template <typename T>
struct Conv {
  const T *x, *weight, *bias, *initial, *grad;
  T *y, *last;            // forward
  T *dx, *dinitial, *parts;  // backward; parts: (rows x runs, taps + 1, channels)
  hpd::Rows rows;
  int64_t batch, channels;
  int64_t vectors;  // of a step
  int64_t runs;     // of a row
  int64_t steps;    // of a run
  bool silu;
  bool past;  // backward: a call's arrays do not fit into the last cache
};

// A thread's run of steps, its channels, and the inputs that its next step sees.
template <typename T, int W, int K>
struct Run {
  using V = Value<T, W>;
  int64_t row, number, first, end, channel;  // end: of the row
  V weight[K], bias, seen[K];                // seen[K - 1]: of the step itself
  int visible;                               // steps before the next one that it sees, up to K - 1
  bool valid;

  __device__ __forceinline__ explicit Run(const Conv<T>& c) {
    const int64_t item = hpd::by_die() * 256 + threadIdx.x, line = item / c.vectors;
    row = line / c.runs;
    number = line - row * c.runs;
    valid = row < c.batch;
    if (!valid) return;
    first = number * c.steps;
    end = c.rows.end(row);
    // The last vector moves back to end with the channels; what it shares it computes alike.
    channel = (item - line * c.vectors) * W;
    if (channel > c.channels - W) channel = c.channels - W;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < W; ++j) weight[k].v[j] = c.weight[(channel + j) * K + k];
    }
    bias = c.bias ? V::load(c.bias + channel) : V::of(T(0));
#pragma unroll
    for (int k = 0; k < K; ++k) seen[k] = V::of(T(0));
    visible = K - 1;
    const unsigned starts = c.rows.template starts<K - 1>(row, first - (K - 1), end);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const int64_t t = first - (K - 1) + k;
      if (starts >> k & 1) clear();
      if (t >= 0 && t < end) push(V::load(at(c, c.x, t)));
      else if (t < 0 && c.initial) push(V::load(c.initial + (row * (K - 1) + t + (K - 1)) * c.channels + channel));
      else push(V::of(T(0)));
    }
  }

  template <typename P>
  __device__ __forceinline__ P* at(const Conv<T>& c, P* array, int64_t t) const {
    return array + (row * c.rows.time + t) * c.channels + channel;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < K; ++k) seen[k] = V::of(T(0));
    visible = 0;
  }
  __device__ __forceinline__ void push(const V& x) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) seen[k] = seen[k + 1];
    seen[K - 1] = x;
    if (visible < K - 1) ++visible;
  }
  __device__ __forceinline__ V sum() const {
    V v = bias;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < W; ++j) v.v[j] = __builtin_elementwise_fma(weight[k].v[j], seen[k].v[j], v.v[j]);
    return v;
  }
};

template <typename T, int W, int K>
__global__ __launch_bounds__(256) void forward_kernel(Conv<T> c) {
  using V = Value<T, W>;
  constexpr int U = 8;
  Run<T, W, K> run(c);
  if (!run.valid) return;
  const auto leave = [&] {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) run.seen[k + 1].store(c.last + (run.row * (K - 1) + k) * c.channels + run.channel);
  };
  if (run.end == 0 && run.number == 0) leave();
  const int64_t stop = run.first + c.steps < c.rows.time ? run.first + c.steps : c.rows.time;
  for (int64_t t = run.first; t < stop; t += U) {
    V x[U];
    const unsigned starts = c.rows.template starts<U>(run.row, t, run.end);
    if (t + U <= run.end) {
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = V::load(run.at(c, c.x, t + i));
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = t + i < run.end ? V::load(run.at(c, c.x, t + i)) : V::of(T(0));
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (t + i >= stop) break;
      V y = V::of(T(0));
      if (t + i < run.end) {
        if (starts >> i & 1) run.clear();
        run.push(x[i]);
        y = run.sum();
        if (c.silu) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            T keep, rest;
            hpd::gates(y.v[j], keep, rest);
            y.v[j] *= keep;
          }
        }
        if (t + i == run.end - 1) leave();
      }
      y.store(run.at(c, c.y, t + i));
    }
  }
}

template <typename T, int W, int K>
__global__ __launch_bounds__(256) void backward_kernel(Conv<T> c) {
  using V = Value<T, W>;
  constexpr int U = K > 6 ? 2 : 4;  // steps ahead, for the registers beside the taps'
  Run<T, W, K> run(c);
  if (!run.valid) return;
  const int64_t stop = run.first + c.steps < c.rows.time ? run.first + c.steps : c.rows.time;
  V open[K];  // gradients of the last K inputs, open[j] of the step j before
  V dweight[K], dbias = V::of(T(0));
#pragma unroll
  for (int k = 0; k < K; ++k) open[k] = dweight[k] = V::of(T(0));
  // Loads of the next steps, without a branch: those behind the row's end repeat its last step's, which nothing uses.
  const uint8_t* const marks = c.rows.resets ? c.rows.resets : reinterpret_cast<const uint8_t*>(c.x);
  V next_x[U], next_d[U];
  unsigned next_marks[U];
  const auto load = [&](int64_t t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t from = t + i < run.end ? t + i : run.end - 1;
      next_x[i] = V::load(run.at(c, c.x, from));
      next_d[i] = V::load(run.at(c, c.grad, from));
      next_marks[i] = marks[run.row * c.rows.time + from];
    }
  };
  if (run.end > 0) load(run.first);
  // Through the steps behind the run that see its last ones.
  for (int64_t t = run.first; t < stop + K - 1; t += U) {
    V x[U], d[U];
    unsigned starts = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      x[i] = next_x[i], d[i] = next_d[i];
      if (c.rows.resets && next_marks[i] && t + i < run.end) starts |= 1u << i;
    }
    if (run.end > 0) load(t + U);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t now = t + i;
      if (now >= stop + K - 1) break;
      if (starts >> i & 1) run.clear();
      const int visible = run.visible;
      run.push(x[i]);
#pragma unroll
      for (int j = K - 1; j > 0; --j) open[j] = open[j - 1];
      open[0] = V::of(T(0));
      if (now < run.end) {
        if (c.silu) {
          const V v = run.sum();
#pragma unroll
          for (int j = 0; j < W; ++j) {
            T keep, rest;
            hpd::gates(v.v[j], keep, rest);
            d[i].v[j] *= keep * (T(1) + v.v[j] * rest);
          }
        }
        const auto give = [&](int j, const V& e) {
#pragma unroll
          for (int q = 0; q < W; ++q) open[j].v[q] = __builtin_elementwise_fma(run.weight[K - 1 - j].v[q], e.v[q], open[j].v[q]);
        };
#pragma unroll
        for (int j = 0; j < K; ++j) {
          if (j <= visible) give(j, d[i]);
        }
        if (now < stop) {
#pragma unroll
          for (int q = 0; q < W; ++q) {
            dbias.v[q] += d[i].v[q];
#pragma unroll
            for (int k = 0; k < K; ++k) dweight[k].v[q] = __builtin_elementwise_fma(d[i].v[q], run.seen[k].v[q], dweight[k].v[q]);
          }
        }
      }
      const int64_t done = now - (K - 1);
      if (done >= run.first) open[K - 1].store(run.at(c, c.dx, done), c.past);
      else if (done < 0 && c.dinitial) open[K - 1].store(c.dinitial + (run.row * (K - 1) + now) * c.channels + run.channel);
    }
  }
  T* parts = c.parts + (run.row * c.runs + run.number) * (K + 1) * c.channels + run.channel;
#pragma unroll
  for (int k = 0; k < K; ++k) dweight[k].store(parts + k * c.channels);
  dbias.store(parts + K * c.channels);
}

// dweight (channels, taps) and dbias from the runs' parts (parts, taps + 1, channels).
template <typename T>
__global__ __launch_bounds__(1024) void sums_kernel(const T* parts, int64_t count, int64_t channels, int taps, T* dweight, T* dbias) {
  const int64_t columns = (taps + 1) * channels;
  hpd::add_parts(parts, columns, 0, count, int64_t(blockIdx.x) * 64, columns, [&](int64_t q, T sum) {
    const int64_t k = q / channels, channel = q - k * channels;
    if (k < taps) dweight[channel * taps + k] = sum;
    else if (dbias) dbias[channel] = sum;
  });
}

template <typename T>
__global__ __launch_bounds__(256) void fill_kernel(T* to, const T* from, int64_t n) {
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) to[i] = from ? from[i] : T(0);
}

template <typename T>
void fill(hp_ctx* ctx, T* to, const T* from, int64_t n) {
  if (!to || n == 0) return;
  fill_kernel<T><<<unsigned(std::min<int64_t>(hp::ceil_div(n, 256), 4096)), 256, 0, ctx->stream>>>(to, from, n);
  hp::check_launch("convolution fill");
}

// Runs as long as there are threads enough without shorter ones.
template <typename T>
unsigned plan(Conv<T>& c, int width, int64_t longest) {
  c.vectors = hp::ceil_div(c.channels, width);
  for (c.steps = longest; c.steps > 8; c.steps /= 2) {
    if (c.batch * hp::ceil_div(c.rows.time, c.steps) * c.vectors >= 200000) break;
  }
  c.runs = hp::ceil_div(c.rows.time, c.steps);
  const int64_t blocks = hp::ceil_div(c.batch * c.runs * c.vectors, 256);
  hp::require(blocks <= hp::kMaxGrid, "too many steps for one launch");
  return unsigned(blocks);
}

template <typename F>
void with_taps(int64_t taps, F&& f) {
  switch (taps) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    case 8: return f(std::integral_constant<int, 8>{});
  }
}

// Calls f with the vectors' width: 16 bytes, or one channel where there are fewer.
template <typename T, typename F>
void with_width(int64_t channels, F&& f) {
  constexpr int W = 16 / sizeof(T);
  if (channels >= W) f(std::integral_constant<int, W>{});
  else f(std::integral_constant<int, 1>{});
}

void check_conv(int dtype, int index_dtype, int64_t batch, int64_t time, int64_t channels, int64_t taps) {
  hp::require(dtype == HP_F32 || dtype == HP_F64, "convolution requires float32 or float64");
  hp::require(index_dtype == HP_I32 || index_dtype == HP_I64, "lengths must be int32 or int64");
  hp::require(batch >= 0 && time >= 0 && channels >= 0, "negative extent");
  hp::require(taps >= 1 && taps <= kMostTaps, "taps out of range");
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == HP_F32) f(float(0));
  else f(double(0));
}

template <typename T>
Conv<T> conv_of(int index_dtype, const void* x, const void* weight, const void* bias, const void* initial, const void* resets,
                const void* lengths, int64_t batch, int64_t time, int64_t channels, int activation) {
  Conv<T> c{};
  c.x = static_cast<const T*>(x);
  c.weight = static_cast<const T*>(weight);
  c.bias = static_cast<const T*>(bias);
  c.initial = static_cast<const T*>(initial);
  c.rows = {static_cast<const uint8_t*>(resets), lengths, index_dtype == HP_I64, time};
  c.batch = batch;
  c.channels = channels;
  c.silu = activation != 0;
  return c;
}

}  // namespace

extern "C" {

int hp_causal_conv(hp_ctx* ctx, int dtype, int index_dtype, const void* x, const void* weight, const void* bias, const void* initial,
                   const void* resets, const void* lengths, void* y, void* last, int64_t batch, int64_t time, int64_t channels,
                   int64_t taps, int activation) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_conv(dtype, index_dtype, batch, time, channels, taps);
    if (batch * channels == 0) return;
    hp::require(x && weight && y && last, "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      if (time == 0) return fill(ctx, static_cast<T*>(last), static_cast<const T*>(initial), batch * (taps - 1) * channels);
      Conv<T> c = conv_of<T>(index_dtype, x, weight, bias, initial, resets, lengths, batch, time, channels, activation);
      c.y = static_cast<T*>(y);
      c.last = static_cast<T*>(last);
      with_width<T>(channels, [&](auto w) {
        const unsigned blocks = plan(c, w, 64);
        with_taps(taps, [&](auto k) { forward_kernel<T, w, k><<<blocks, 256, 0, ctx->stream>>>(c); });
      });
      hp::check_launch("convolution");
    });
  });
}

int hp_causal_conv_grad(hp_ctx* ctx, int dtype, int index_dtype, const void* grad, const void* x, const void* weight, const void* bias,
                        const void* initial, const void* resets, const void* lengths, void* dx, void* dweight, void* dbias,
                        void* dinitial, int64_t batch, int64_t time, int64_t channels, int64_t taps, int activation) {
  return hp::guarded([&] {
    hp::enter(ctx);
    check_conv(dtype, index_dtype, batch, time, channels, taps);
    if (channels == 0) return;
    hp::require(dweight, "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      if (batch * time == 0) {
        fill<T>(ctx, static_cast<T*>(dweight), nullptr, channels * taps);
        fill<T>(ctx, static_cast<T*>(dbias), nullptr, channels);
        fill<T>(ctx, static_cast<T*>(dinitial), nullptr, batch * (taps - 1) * channels);
        return;
      }
      hp::require(grad && x && weight && dx, "null pointer");
      hp::Scratch scratch(ctx);
      Conv<T> c = conv_of<T>(index_dtype, x, weight, bias, initial, resets, lengths, batch, time, channels, activation);
      c.grad = static_cast<const T*>(grad);
      c.dx = static_cast<T*>(dx);
      c.dinitial = static_cast<T*>(dinitial);
      // Three arrays, of which the caches would hold none to its next reader: 209 us -> 202 of 8 x 4096 x 2048 float32,
      // in turn on one card.
      c.past = batch * time * channels * int64_t(3 * sizeof(T)) > hp::kLastCache;
      with_width<T>(channels, [&](auto w) {
        const unsigned blocks = plan(c, w, 64);
        c.parts = scratch.take<T>(batch * c.runs * (taps + 1) * channels);
        with_taps(taps, [&](auto k) { backward_kernel<T, w, k><<<blocks, 256, 0, ctx->stream>>>(c); });
      });
      hp::check_launch("convolution gradient");
      const int64_t columns = (taps + 1) * channels, sums = hp::ceil_div(columns, 64);
      hp::require(sums <= hp::kMaxThreads / 1024, "too many channels for one launch");
      sums_kernel<T><<<unsigned(sums), 1024, 0, ctx->stream>>>(c.parts, batch * c.runs, channels, int(taps), static_cast<T*>(dweight), static_cast<T*>(dbias));
      hp::check_launch("convolution sums");
    });
  });
}

}  // extern "C"
