// The selective scan forward (scan.h). Bound: the exponentials of 16 states a channel,
// about as long as reading x, delta and the gate and writing y takes; for fewer states HBM.
#include "scan.h"

using namespace hpd;

namespace {

constexpr int kSteps = 16;  // of a tile

// SUMMARY: a part's sum of dt and the states that it ends in from zero ones, in place of y.
template <typename T, int NW, int S, bool RESETS, bool SUMMARY>
__global__ __launch_bounds__(NW * 64) void forward_kernel(Scan<T> c, const T* b_, const T* c_) {
  constexpr int kOwn = kSteps / NW;  // steps of a tile that a wave prepares and finishes
  __shared__ T shared_dt[kSteps][64], shared_u[kSteps][64];
  __shared__ T sums[SUMMARY ? 1 : NW][SUMMARY ? 1 : kSteps][64];
  const Place<T, NW, S> at(c);
  if (SUMMARY && at.part == c.parts - 1) return;
  const int lane = at.lane, own = at.wave * kOwn;
  T rate[S], h[S];
  at.read(c, c.a_log, 0, rate);
#pragma unroll
  for (int s = 0; s < S; ++s) rate[s] = rate_of(rate[s]);
  if constexpr (SUMMARY) {
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = T(0);
  } else {
    at.arrive(c, rate, h);
  }
  const T bias = c.delta_bias ? c.delta_bias[at.channel] : T(0), skip = c.skip ? c.skip[at.channel] : T(0);
  T x[kOwn], delta[kOwn], gate[kOwn], span = T(0);
  Projections<T, kSteps, S> next_b, next_c;
  bool cut = false;
  const auto load = [&](int64_t t) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int64_t step = t + own + i < at.end ? t + own + i : at.end - 1;
      x[i] = at.get(c, c.x, step);
      delta[i] = at.get(c, c.delta, step);
      if (!SUMMARY && c.gate) gate[i] = at.get(c, c.gate, step);
    }
    next_b.load(c, at, b_, t);
    if (!SUMMARY) next_c.load(c, at, c_, t);
  };
  if (at.first < at.end) load(at.first);
  for (int64_t t = at.first; t < at.end; t += kSteps) {
    const int count = at.end - t < kSteps ? int(at.end - t) : kSteps;
    T now_x[kOwn], now_gate[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool inside = own + i < count;
      T slope;
      const T dt = softplus(delta[i] + bias, slope);
      shared_dt[own + i][lane] = inside ? dt : T(0);
      shared_u[own + i][lane] = inside ? dt * x[i] : T(0);
      now_x[i] = x[i];
      if (!SUMMARY) now_gate[i] = gate[i];
    }
    Projections<T, kSteps, S> bs = next_b, cs = next_c;
    bs.keep(lane, count);
    if (!SUMMARY) cs.keep(lane, count);
    __syncthreads();
    if (t + kSteps < at.end) load(t + kSteps);
    const unsigned starts = RESETS ? __builtin_amdgcn_readfirstlane(c.rows.template starts<kSteps>(at.row, t, at.end)) : 0;
    // Tiles without a reset, nearly all of them, do without its selects.
    const auto walk = [&](auto resets) {
      for_each<kSteps>([&](auto step) {
        constexpr int i = step;
        const T dt = shared_dt[i][lane], u = shared_u[i][lane];
        T y = T(0);
        for_each<S>([&](auto state) {
          constexpr int s = state;
          if (resets) h[s] = starts >> i & 1 ? T(0) : h[s];
          h[s] = __builtin_elementwise_fma(decay(dt, rate[s]), h[s], u * bs.template get<i, s>());
          if constexpr (!SUMMARY) y = __builtin_elementwise_fma(cs.template get<i, s>(), h[s], y);
        });
        if constexpr (SUMMARY) span += dt;
        else sums[at.wave][i][lane] = y;
      });
    };
    if (RESETS && starts) walk(std::true_type{}), cut = true;
    else walk(std::false_type{});
    __syncthreads();
    if constexpr (!SUMMARY) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (t + own + i >= at.end) break;
        T y = sums[0][own + i][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) y += sums[w][own + i][lane];
        T* to = c.y + at.at(c, t + own + i);
        if (!c.starts) y += *to;
        if (c.ends) {
          if (c.skip) y = __builtin_elementwise_fma(skip, now_x[i], y);
          if (c.gate) {
            T keep, rest;
            gates(now_gate[i], keep, rest);
            y *= now_gate[i] * keep;
          }
        }
        if (at.valid) *to = y;
      }
    }
  }
  if constexpr (SUMMARY) {
    if (!at.valid) return;
    if (at.wave == 0) c.spans[(at.part * c.batch + at.row) * c.channels + at.channel] = cut ? cut_span<T>() : span;
#pragma unroll
    for (int s = 0; s < S; ++s) c.ended[at.state_at(c, at.part, s)] = h[s];
  } else {
    // Behind the row's end, by every wave for its own steps.
    const int64_t stop = at.first + c.steps < c.rows.time ? at.first + c.steps : c.rows.time;
    for (int64_t t = (at.end > at.first ? at.end : at.first) + at.wave; t < stop; t += NW) {
      if (at.valid) c.y[at.at(c, t)] = T(0);
    }
    // The part that has the row's last step, or of a row without steps the first.
    const bool last = at.length > at.first ? at.length <= at.first + c.steps : at.length == 0 && at.part == 0;
    if (last) at.write(c, c.last, at.row, h);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(T* to, const T* from, int64_t n, int64_t states, int64_t padded) {
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t step = i / padded, s = i - step * padded;
    to[i] = s < states ? from[step * states + s] : T(0);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void fill_kernel(T* to, const T* from, int64_t n) {
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) to[i] = from ? from[i] : T(0);
}

template <typename T, bool SUMMARY>
void launch(hp_ctx* ctx, const Scan<T>& c, const T* b, const T* cs, int each, int waves) {
  const unsigned blocks = unsigned(c.batch * c.groups * c.pieces * c.parts);
  const auto run = [&](auto nw) {
    const auto with = [&](auto states) {
      const auto kernel = c.rows.resets ? forward_kernel<T, nw, states, true, SUMMARY> : forward_kernel<T, nw, states, false, SUMMARY>;
      kernel<<<blocks, nw * 64, 0, ctx->stream>>>(c, b, cs);
    };
    if constexpr (nw >= 2 && nw <= 8) {
      if (each == 2) return with(std::integral_constant<int, 2>{});
    }
    with(std::integral_constant<int, 4>{});
  };
  switch (waves) {
    case 1: run(std::integral_constant<int, 1>{}); break;
    case 2: run(std::integral_constant<int, 2>{}); break;
    case 4: run(std::integral_constant<int, 4>{}); break;
    case 8: run(std::integral_constant<int, 8>{}); break;
    default: run(std::integral_constant<int, 16>{}); break;
  }
  hp::check_launch("scan");
}

}  // namespace

namespace hp {

void scan_check(int dtype, int index_dtype, int64_t batch, int64_t time, int64_t channels, int64_t groups, int64_t states) {
  require(dtype == HP_F32 || dtype == HP_F64, "scan requires float32 or float64");
  require(index_dtype == HP_I32 || index_dtype == HP_I64, "lengths must be int32 or int64");
  require(batch >= 0 && time >= 0 && channels >= 0 && groups >= 0, "negative extent");
  require(states >= 1 && states <= 256, "states out of range");
  require(channels == 0 || (groups > 0 && channels % groups == 0), "groups do not divide the channels");
}

template <typename T>
void scan_fill(hp_ctx* ctx, T* to, const T* from, int64_t n) {
  if (!to || n == 0) return;
  fill_kernel<T><<<unsigned(std::min<int64_t>(ceil_div(n, 256), 4096)), 256, 0, ctx->stream>>>(to, from, n);
  check_launch("scan fill");
}
template void scan_fill(hp_ctx*, float*, const float*, int64_t);
template void scan_fill(hp_ctx*, double*, const double*, int64_t);

template <typename T>
const T* scan_padded(hp_ctx* ctx, Scratch& scratch, const T* array, int64_t steps, int64_t states, int64_t padded) {
  if (states == padded) return array;
  T* to = scratch.take<T>(steps * padded);
  pad_kernel<T><<<unsigned(std::min<int64_t>(ceil_div(steps * padded, 256), 4096)), 256, 0, ctx->stream>>>(to, array, steps * padded, states, padded);
  check_launch("scan states");
  return to;
}
template const float* scan_padded(hp_ctx*, Scratch&, const float*, int64_t, int64_t, int64_t);
template const double* scan_padded(hp_ctx*, Scratch&, const double*, int64_t, int64_t, int64_t);

}  // namespace hp

extern "C" {

int hp_selective_scan(hp_ctx* ctx, int dtype, int index_dtype, const void* x, const void* delta, const void* a_log, const void* b,
                      const void* c, const void* skip, const void* gate, const void* initial, const void* delta_bias,
                      const void* resets, const void* lengths, void* y, void* last, int64_t batch, int64_t time, int64_t channels,
                      int64_t groups, int64_t states) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::scan_check(dtype, index_dtype, batch, time, channels, groups, states);
    if (batch * channels == 0) return;
    hp::require(last && (time == 0 || (x && delta && a_log && b && c && y)), "null pointer");
    const auto run = [&](auto zero) {
      using T = decltype(zero);
      const auto in = [](const void* p) { return static_cast<const T*>(p); };
      if (time == 0) return hp::scan_fill(ctx, static_cast<T*>(last), in(initial), batch * channels * states);
      hp::Scratch scratch(ctx);
      Scan<T> s{};
      s.x = in(x), s.delta = in(delta), s.a_log = in(a_log), s.skip = in(skip), s.gate = in(gate), s.initial = in(initial), s.delta_bias = in(delta_bias);
      s.y = static_cast<T*>(y), s.last = static_cast<T*>(last);
      s.rows = {static_cast<const uint8_t*>(resets), lengths, index_dtype == HP_I64, time};
      s.batch = batch, s.channels = channels, s.groups = groups, s.states = states;
      s.width = channels / groups, s.pieces = hp::ceil_div(s.width, 64);
      hp::scan_plan(s, kSteps);
      const int each = hp::scan_states(s), waves = hp::scan_waves(states, each, 16), width = waves * each;
      s.padded = hp::ceil_div(states, width) * width;
      const T *bs = hp::scan_padded(ctx, scratch, in(b), batch * time * groups, states, s.padded);
      const T *cs = hp::scan_padded(ctx, scratch, in(c), batch * time * groups, states, s.padded);
      if (s.parts > 1) {
        s.spans = scratch.take<T>(s.parts * batch * channels);
        s.ended = scratch.take<T>(s.parts * batch * width * channels);
      }
      for (s.first = 0; s.first < states; s.first += width) {
        s.starts = s.first == 0;
        s.ends = s.first + width >= states;
        if (s.parts > 1) launch<T, true>(ctx, s, bs, cs, each, waves);
        launch<T, false>(ctx, s, bs, cs, each, waves);
      }
    };
    if (dtype == HP_F32) run(float(0));
    else run(double(0));
  });
}

}  // extern "C"
