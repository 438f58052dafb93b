// The selective scan forward (scan.h). Bound: vector issue, 68% of the SIMDs' cycles for 16 states a
// channel; waves wait 30% of their time.
#include "scan.h"

using namespace hpd;

namespace {

// Steps of a tile, tiles that are loaded ahead (an even number), and states and waves of a
// launch, for the registers that they take.
template <typename T>
constexpr int kTile = sizeof(T) == 4 ? 16 : 8;
template <typename T, int NW>
constexpr int kTiles = sizeof(T) == 4 && NW > 2 && NW < 16 ? 4 : 2;

// SUMMARY: a part's sum of dt and the states that it ends in from zero ones, in place of y. ONE: rows of one tile, single
// tokens among them, without the loads, barriers and waits of those ahead: 8.1 us in place of 13 for 16 tokens of 2048
// channels with 16 states.
template <typename T, int NW, int S, bool RESETS, bool SUMMARY, bool ONE = false>
__global__ __launch_bounds__(NW * 64) void forward_kernel(Scan<T> c, const T* b_, const T* c_) {
  constexpr int kSteps = kTile<T>, kAhead = ONE ? 1 : kTiles<T, NW>, kOwn = kSteps / NW;  // steps of a tile that a wave prepares and finishes
  __shared__ T shared_dt[2][kSteps][64], shared_u[2][kSteps][64];
  // Two sets of sums where LDS has room: the waves then meet once a tile, not again behind its sums.
  constexpr int kSets = NW <= 8 ? 2 : 1;
  __shared__ T sums[SUMMARY ? 1 : kSets][SUMMARY ? 1 : NW][SUMMARY ? 1 : kSteps][64];
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
  T span = T(0);
  bool cut = false;
  const T* const gates_or_x = c.gate ? c.gate : c.x;
  // Loads of the tiles ahead: a tile is too short to cover the memory's latency. They are
  // issued without a branch, behind the end too, where they repeat the last step's: a wait
  // for the oldest counts the loads issued since, as many as there are on every way.
  struct Ahead {
    T x[kOwn], delta[kOwn], gate[kOwn];
    Projections<T, kSteps, S> b, c;
    unsigned resets;
  } ahead[kAhead];
  const auto load = [&](Ahead& to, int t) __attribute__((always_inline)) {
    t = t < at.end ? t : at.end - 1;
    const T *x = at.line(c, c.x, t), *delta = at.line(c, c.delta, t), *gate = at.line(c, gates_or_x, t);
    const int last = at.end - 1 - t;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const unsigned from = at.place(c, own + i < last ? own + i : last);
      to.x[i] = x[from];
      to.delta[i] = delta[from];
      if (!SUMMARY) to.gate[i] = gate[from];
    }
    to.b.load(c, at, b_, t);
    if (!SUMMARY) to.c.load(c, at, c_, t);
    if (RESETS) to.resets = c.rows.byte(at.row, t, at.end, lane);
  };
  // Leaves dt and dt x of the wave's own steps of a tile.
  const auto prepare = [&](const Ahead& from, int t, int turn) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool inside = t + own + i < at.end;
      T slope;
      const T dt = softplus(from.delta[i] + bias, slope);
      shared_dt[turn][own + i][lane] = inside ? dt : T(0);
      shared_u[turn][own + i][lane] = inside ? dt * from.x[i] : T(0);
    }
  };
  if (at.first < at.end) {
    for_each<kAhead>([&](auto k) __attribute__((always_inline)) { load(ahead[k], at.first + k * kSteps); });
    prepare(ahead[0], at.first, 0);
  }
  __syncthreads();
  // Tile t, whose loads stand in `now` and those of the next one in `next`.
  const auto tile = [&](Ahead& now, const Ahead& next, int t, int turn) __attribute__((always_inline)) {
    const int count = at.end - t < kSteps ? (at.end > t ? at.end - t : 0) : kSteps;
    T x[kOwn], gate[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) x[i] = now.x[i], gate[i] = now.gate[i];
    Projections<T, kSteps, S> bs = now.b, cs = now.c;
    bs.keep(lane, count);
    if (!SUMMARY) cs.keep(lane, count);
    const unsigned starts = RESETS ? unsigned(__ballot(now.resets != 0 && lane < count)) : 0;
    if constexpr (!ONE) {
      load(now, t + kAhead * kSteps);
      prepare(next, t + kSteps, turn ^ 1);  // of no use behind the last tile
    }
    // All of the tile's at once: the compiler would wait for those of each step in turn.
    T dts[kSteps], us[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) dts[i] = shared_dt[turn][i][lane], us[i] = shared_u[turn][i][lane];
    __builtin_amdgcn_sched_barrier(0);
    // Tiles without a reset, nearly all of them, do without its selects.
    const auto walk = [&](auto resets) __attribute__((always_inline)) {
      for_each<kSteps>([&](auto step) {
        constexpr int i = step;
        const T dt = dts[i], u = us[i];
        T y = T(0);
        for_each<S>([&](auto state) {
          constexpr int s = state;
          if (resets) h[s] = starts >> i & 1 ? T(0) : h[s];
          h[s] = __builtin_elementwise_fma(decay(dt, rate[s]), h[s], u * bs.template get<i, s>());
          // A product takes the broadcast on the way, a fused one would not.
          if constexpr (!SUMMARY) {
            const T part = cs.template get<i, s>() * h[s];
            y = s ? y + part : part;
          }
        });
        if constexpr (SUMMARY) span += dt;
        else sums[turn % kSets][at.wave][i][lane] = y;
      });
    };
    cut = cut || starts;
    if constexpr (RESETS && NW == 16) walk(std::true_type{});  // two of them would take too many registers
    else if (RESETS && starts) walk(std::true_type{});
    else if (count) walk(std::false_type{});  // (the branch also keeps the tiles' registers apart)
    __syncthreads();
    if constexpr (!SUMMARY) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (own + i >= count) break;
        T y = sums[turn % kSets][0][own + i][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) y += sums[turn % kSets][w][own + i][lane];
        T* to = at.line(c, c.y, t) + at.place(c, own + i);
        if (!c.starts) y += *to;
        if (c.ends) {
          if (c.skip) y = __builtin_elementwise_fma(skip, x[i], y);
          if (c.gate) {
            T keep, rest;
            gates(gate[i], keep, rest);
            y *= gate[i] * keep;
          }
        }
        if (at.valid) *to = y;
      }
      if (kSets == 1) __syncthreads();
    }
  };
  for (int t = at.first; t < at.end; t += kAhead * kSteps) {
    for_each<kAhead>([&](auto k) __attribute__((always_inline)) {
      tile(ahead[k], ahead[(k + 1) % kAhead], t + k * kSteps, k & 1);  // behind the end it changes nothing
    });
  }
  if constexpr (SUMMARY) {
    if (!at.valid) return;
    if (at.wave == 0) at.row_line(c, c.spans, at.part)[at.channel] = cut ? cut_span<T>() : span;
#pragma unroll
    for (int s = 0; s < S; ++s) at.state_line(c, c.ended, at.part, s)[at.channel] = h[s];
  } else {
    // Behind the row's end, by every wave for its own steps.
    const int stop = c.time - at.first < c.steps ? c.time : at.first + c.steps;
    for (int t = (at.end > at.first ? at.end : at.first) + at.wave; t < stop; t += NW) {
      if (at.valid) at.line(c, c.y, t)[at.channel] = T(0);
    }
    // The part that has the row's last step, or of a row without steps the first.
    const bool last = at.length > at.first ? at.length - at.first <= c.steps : at.length == 0 && at.part == 0;
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

template <typename T, int NW, int S>
void launch(hp_ctx* ctx, const Scan<T>& c, const T* b, const T* cs) {
  const unsigned blocks = unsigned(c.batch) * unsigned(c.groups) * unsigned(c.pieces) * unsigned(c.parts);
  if (c.parts > 1) {
    const auto kernel = c.rows.resets ? forward_kernel<T, NW, S, true, true> : forward_kernel<T, NW, S, false, true>;
    kernel<<<blocks, NW * 64, 0, ctx->stream>>>(c, b, cs);
    hp::check_launch("scan summary");
  }
  const bool one = c.time <= kTile<T> && !c.rows.resets;
  const auto kernel = c.rows.resets ? forward_kernel<T, NW, S, true, false> : one ? forward_kernel<T, NW, S, false, false, true> : forward_kernel<T, NW, S, false, false>;
  kernel<<<blocks, NW * 64, 0, ctx->stream>>>(c, b, cs);
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
      // Two states a wave, which leaves several waves a SIMD to cover each other's waits; four of many states.
      const bool many = sizeof(T) == 4 && states > 16;
      const int each = many ? 4 : 2, waves = hp::scan_waves(states, each, many ? 16 : 8), width = waves * each;
      hp::scan_sizes(s, batch, time, channels, groups, states, width);
      hp::scan_plan(s, kTile<T>);
      const T *bs = hp::scan_padded(ctx, scratch, in(b), batch * time * groups, states, s.padded);
      const T *cs = hp::scan_padded(ctx, scratch, in(c), batch * time * groups, states, s.padded);
      if (s.parts > 1) {
        s.spans = scratch.take<T>(s.parts * batch * channels);
        s.ended = scratch.take<T>(s.parts * batch * width * channels);
      }
      for (s.first = 0; s.first < states; s.first += width) {
        s.starts = s.first == 0;
        s.ends = s.first + width >= states;
        if (!many) {
          if (waves == 2) launch<T, 2, 2>(ctx, s, bs, cs);
          else if (waves == 4) launch<T, 4, 2>(ctx, s, bs, cs);
          else launch<T, 8, 2>(ctx, s, bs, cs);
        }
        if constexpr (sizeof(T) == 4) {
          if (many && waves == 8) launch<T, 8, 4>(ctx, s, bs, cs);
          else if (many) launch<T, 16, 4>(ctx, s, bs, cs);
        }
      }
    };
    if (dtype == HP_F32) run(float(0));
    else run(double(0));
  });
}

}  // extern "C"
