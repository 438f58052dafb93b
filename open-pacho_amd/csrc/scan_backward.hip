// The selective scan backward (scan.h).
//
//   g_t = dy_t silu(gate_t),  m_t = c_t g_t + e_{t+1},  e_t = exp(-dt r) m_t (0 at a reset)
//   s_t = e_t h_{t-1}
//   dc_t = sum g_t h_t,  db_t = sum dt x_t m_t over a group's channels
//   dx_t = dt sum m_t b_t + skip g_t,  ddt = x_t sum m_t b_t - sum r s_t,  da_log = -r sum_t s_t dt
//   ddelta = ddt sigmoid(delta + bias),  dgate = dy_t (sum c_t h_t + skip x_t) silu'(gate_t),  dinitial = e_0
//
// The states are not kept from forward: a first launch walks all steps and leaves the states
// before every tile, a second one walks the tiles from the last, forms a tile's states again,
// keeps them with their decays in registers, and goes back through them. A tile is as long as
// these registers allow: its states before it are as many values as a channel has states, in
// place of as many steps' values.
//
// Sums over channels (db, dc): every lane has a value for each step and state of a tile. Pairs
// of registers are folded into one whose halves, quarters, ... belong to one of the two each,
// until a register holds a sum in each lane: two or three instructions a value where a sum over
// 64 lanes by itself takes six times two. Workgroups leave these, and their sums over steps, as parts.
//
// Bound: vector issue, 29 instructions a state and step (32 with resets), 73-76% of the SIMDs' cycles. 8 x 2048 x
// 2048 float32 with 16 states and resets: 172-184 us for the first launch, 625-671 for the second, 20 for
// db and dc, where the call's bytes would take 155; 740 in all without resets.
//
// Where rows are cut into parts, the first launch also forms what a part passes back from
// nothing, sum_t D_t c_t g_t with D_t the product of the decays up to t.
#include "lanes.h"
#include "scan.h"

using namespace hpd;

namespace {

// Exponentials of doubles, small programs, one after the other: side by side they would take all registers.
template <typename T>
__device__ __forceinline__ void apart() {
  if constexpr (sizeof(T) == 8) __builtin_amdgcn_sched_barrier(0);
}

// Steps of a tile, for the registers that its states and decays take: of 16, float32 with four waves or
// more states would need accumulation registers, which leaves them a wave a SIMD.
template <typename T, int NW, int S>
constexpr int kTile = sizeof(T) == 4 && S == 2 && NW == 8 ? 16 : 8;
constexpr int kLongestTile = 16;
// Tiles that the first launch loads ahead, an even number.
template <typename T, int NW>
constexpr int kTiles = sizeof(T) == 4 && NW > 2 ? 4 : 2;

template <typename T, int NW, int S, bool RESETS, bool SPLIT>
__global__ __launch_bounds__(NW * 64) void before_kernel(Scan<T> c, const T* b_, const T* c_) {
  constexpr int L = kTile<T, NW, S>, kOwn = L / NW, kAhead = kTiles<T, NW>;
  __shared__ T shared_dt[2][L][64], shared_u[2][L][64], shared_g[2][SPLIT ? L : 1][64];
  const Place<T, NW, S> at(c);
  const int lane = at.lane, own = at.wave * kOwn;
  T rate[S], h[S], through[S], back[S], span = T(0);
  at.read(c, c.a_log, 0, rate);
#pragma unroll
  for (int s = 0; s < S; ++s) rate[s] = rate_of(rate[s]), h[s] = back[s] = T(0), through[s] = T(1);
  if (!SPLIT && c.initial) at.read(c, c.initial, at.row, h);
  const T bias = c.delta_bias ? c.delta_bias[at.channel] : T(0);
  bool cut = false;
  const T* const gates_or_x = c.gate ? c.gate : c.x;
  // Loads of the tiles ahead: a tile is too short to cover the memory's latency. They are
  // issued without a branch, behind the end too, where they repeat the last step's: a wait
  // for the oldest counts the loads issued since, as many as there are on every way.
  struct Ahead {
    T x[kOwn], delta[kOwn], grad[kOwn], gate[kOwn];
    Projections<T, L, S> b, c;
    unsigned resets;
  } ahead[kAhead];
  const auto load = [&](Ahead& to, int t) __attribute__((always_inline)) {
    t = t < at.end ? t : at.end - 1;
    const T *x = at.line(c, c.x, t), *delta = at.line(c, c.delta, t);
    const int last = at.end - 1 - t;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const unsigned from = at.place(c, own + i < last ? own + i : last);
      to.x[i] = x[from];
      to.delta[i] = delta[from];
      if constexpr (SPLIT) {
        to.grad[i] = at.line(c, c.grad, t)[from];
        to.gate[i] = at.line(c, gates_or_x, t)[from];
      }
    }
    to.b.load(c, at, b_, t);
    if (SPLIT) to.c.load(c, at, c_, t);
    if (RESETS) to.resets = c.rows.byte(at.row, t, at.end, lane);
  };
  // Leaves dt, dt x and g of the wave's own steps of a tile.
  const auto prepare = [&](const Ahead& from, int t, int turn) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool inside = t + own + i < at.end;
      T slope;
      const T dt = softplus(from.delta[i] + bias, slope);
      shared_dt[turn][own + i][lane] = inside ? dt : T(0);
      shared_u[turn][own + i][lane] = inside ? dt * from.x[i] : T(0);
      if constexpr (SPLIT) {
        T g = from.grad[i], keep, rest;
        gates(from.gate[i], keep, rest);
        g *= c.gate ? from.gate[i] * keep : T(1);
        shared_g[turn][own + i][lane] = inside ? g : T(0);
      }
    }
  };
  if (at.first < at.end) {
    for_each<kAhead>([&](auto k) __attribute__((always_inline)) { load(ahead[k], at.first + k * L); });
    prepare(ahead[0], at.first, 0);
  }
  __syncthreads();
  // Tile t, whose loads stand in `now` and those of the next one in `next`.
  const auto tile = [&](Ahead& now, const Ahead& next, int t, int turn) __attribute__((always_inline)) {
    const int count = at.end - t < L ? (at.end > t ? at.end - t : 0) : L;
    Projections<T, L, S> bs = now.b, cs = now.c;
    bs.keep(lane, count);
    if (SPLIT) cs.keep(lane, count);
    const unsigned starts = RESETS ? unsigned(__ballot(now.resets != 0 && lane < count)) : 0;
    load(now, t + kAhead * L);
    const int number = t / L;
    if (at.valid && count) {
#pragma unroll
      for (int s = 0; s < S; ++s) at.state_line(c, c.before, number, s)[at.channel] = h[s];
      if (SPLIT && at.wave == 0) at.row_line(c, c.since, number)[at.channel] = cut ? cut_span<T>() : span;
    }
    prepare(next, t + L, turn ^ 1);  // of no use behind the last tile
    // All of the tile's at once: the compiler would wait for those of each step in turn.
    T dts[L], us[L], gs[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      dts[i] = shared_dt[turn][i][lane], us[i] = shared_u[turn][i][lane];
      if constexpr (SPLIT) gs[i] = shared_g[turn][i][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    // Tiles without a reset, nearly all of them, do without its selects.
    const auto walk = [&](auto resets) __attribute__((always_inline)) {
      for_each<L>([&](auto step) {
        constexpr int i = step;
        const bool start = resets && (starts >> i & 1);
        const T dt = dts[i], u = us[i];
        T g = T(0);
        if constexpr (SPLIT) {
          cut = cut || start;
          g = RESETS && cut ? T(0) : gs[i];
          span += dt;
        }
        for_each<S>([&](auto state) {
          constexpr int s = state;
          const T keep = decay(dt, rate[s]);
          if (resets) h[s] = start ? T(0) : h[s];
          h[s] = __builtin_elementwise_fma(keep, h[s], u * bs.template get<i, s>());
          if constexpr (SPLIT) {
            through[s] *= keep;
            back[s] = __builtin_elementwise_fma(through[s], cs.template get<i, s>() * g, back[s]);
          }
        });
      });
    };
    if (RESETS && starts) walk(std::true_type{});
    else if (count) walk(std::false_type{});  // (the branch also keeps the tiles' registers apart)
    __syncthreads();
  };
  for (int t = at.first; t < at.end; t += kAhead * L) {
    for_each<kAhead>([&](auto k) __attribute__((always_inline)) {
      tile(ahead[k], ahead[(k + 1) % kAhead], t + k * L, k & 1);  // behind the end it changes nothing
    });
  }
  if constexpr (SPLIT) {
    if (!at.valid) return;
    if (at.wave == 0) at.row_line(c, c.spans, at.part)[at.channel] = cut ? cut_span<T>() : span;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      at.state_line(c, c.ended, at.part, s)[at.channel] = h[s];
      at.state_line(c, c.passed, at.part, s)[at.channel] = back[s];
    }
  }
}

template <typename T>
struct Grads {
  T *dx, *ddelta, *dgate, *dinitial;
  // (pieces, batch x time x groups, states of a launch)
  T *db, *dc;
  // (batch x parts, states of a launch, channels), (batch x parts, channels)
  T *da, *dskip, *dbias;
};

// ---- folding of registers ------------------------------------------------------------

// Lanes without `bit` get a's sums over pairs of lanes, those with it b's.
template <int MASK, typename T>
__device__ __forceinline__ T fold_pair(T a, T b, bool bit) {
  if constexpr (sizeof(T) == 4 && (MASK == 8 || MASK == 7)) {
    // Two additions that write the lanes of one kind each, in place of two selects and one;
    // what they read may be as new as the wait for it; selects or another fold read what they leave.
    T sum;
    if constexpr (MASK == 8) {
      asm("s_nop 1\n\tv_add_f32_dpp %0, %1, %1 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
          "v_add_f32_dpp %0, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xc" : "=&v"(sum) : "v"(a), "v"(b));
    } else {
      asm("s_nop 1\n\tv_add_f32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
          "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xa" : "=&v"(sum) : "v"(a), "v"(b));
    }
    return sum;
  } else {
    return (bit ? b : a) + from_across<MASK>(bit ? a : b);
  }
}

// Of values for each of S states and L steps (8 or 16) the sums over each row of 16 lanes,
// and of the rows, whose pairs the lanes' halves share, over pairs: lane i has the sum of step
// step_of_lane(i) and state state_of_lane(i). Within a row pairs of steps meet across 8, 7,
// 3 and 1 lanes, which reaches all 16: an addition that takes its operand from another
// lane costs no more than any other, where an exchange of rows takes 12 cycles or more.
template <typename T, int S, int L>
__device__ __forceinline__ T fold(const T (&pairs)[S][L / 2], int lane) {
  T of_state[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    T a[L / 4], b[L / 8];
#pragma unroll
    for (int k = 0; k < L / 4; ++k) a[k] = fold_pair<7>(pairs[s][2 * k], pairs[s][2 * k + 1], lane & 4);
#pragma unroll
    for (int k = 0; k < L / 8; ++k) b[k] = fold_pair<3>(a[2 * k], a[2 * k + 1], lane & 2);
    if constexpr (L == 16) of_state[s] = fold_pair<1>(b[0], b[1], lane & 1);
    else of_state[s] = b[0];
  }
  if constexpr (L == 8) {
    if constexpr (S == 4) {
      of_state[0] = fold_pair<1>(of_state[0], of_state[1], lane & 1);
      of_state[1] = fold_pair<1>(of_state[2], of_state[3], lane & 1);
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) of_state[s] += from_across<1>(of_state[s]);
    }
  }
  return fold_rows<5>(of_state[0], of_state[1]);
}
template <int L>
__device__ __forceinline__ int step_of_lane(int lane) {
  return (lane >> 3 & 1) | (lane >> 2 & 1) << 1 | (lane >> 1 & 1) << 2 | (L == 16 ? (lane & 1) << 3 : 0);
}
template <int S>
__device__ __forceinline__ int state_of_lane(int lane) {
  return S == 4 ? (lane & 1) | (lane >> 5 & 1) << 1 : lane >> 5 & 1;
}

// ---- backward ------------------------------------------------------------------------

template <typename T, int NW, int S, bool RESETS>
__global__ __launch_bounds__(NW * 64) void backward_kernel(Scan<T> c, Grads<T> o, const T* b_, const T* c_) {
  constexpr int L = kTile<T, NW, S>, kOwn = L / NW;
  __shared__ T shared_dt[2][L][64], shared_u[2][L][64], shared_g[2][L][64];
  __shared__ T sums_b[NW][L][64], sums_a[NW][L][64], sums_y[NW][L][64];
  const Place<T, NW, S> at(c);
  const int lane = at.lane, own = at.wave * kOwn;
  T rate[S], slow[S], e[S], da[S];
  at.read(c, c.a_log, 0, slow);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    rate[s] = rate_of(slow[s]);
    slow[s] = sizeof(T) == 4 ? -T(bounded(expf(float(slow[s])))) : rate[s];
    e[s] = da[s] = T(0);
  }
  T arrived[S] = {};
  if (c.parts > 1) {
    at.arrive(c, rate, arrived);
    if (c.grad_state) at.read(c, c.grad_state, at.row, e);
    for (int p = c.parts - 1; p > at.part; --p) {
      const T span = at.row_line(c, c.spans, p)[at.channel];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const T back = at.state_line(c, c.passed, p, s)[at.channel];
        e[s] = passed(span, rate[s], e[s], back);
      }
    }
  } else if (c.grad_state) {
    at.read(c, c.grad_state, at.row, e);
  }
#pragma unroll
  for (int s = 0; s < S; ++s) e[s] = at.valid ? e[s] : T(0);  // other lanes add nothing to db and dc
  const T bias = c.delta_bias ? c.delta_bias[at.channel] : T(0), skip = c.skip ? c.skip[at.channel] : T(0);
  T dskip = T(0), dbias = T(0);
  // Behind the row's end, by every wave for its own steps.
  const int stop = c.time - at.first < c.steps ? c.time : at.first + c.steps;
  for (int t = (at.end > at.first ? at.end : at.first) + at.wave; t < stop; t += NW) {
    if (!at.valid) continue;
    at.line(c, o.dx, t)[at.channel] = at.line(c, o.ddelta, t)[at.channel] = T(0);
    if (c.gate) at.line(c, o.dgate, t)[at.channel] = T(0);
  }
  const int tiles = at.end > at.first ? (at.end - at.first + L - 1) / L : 0;
  const T* const gates_or_x = c.gate ? c.gate : c.x;
  struct Ahead {
    T x[kOwn], delta[kOwn], gate[kOwn], grad[kOwn], before[S], since;
    Projections<T, L, S> b, c;
    unsigned resets;
  } ahead;
  const auto load = [&](int t) __attribute__((always_inline)) {
    t = t < at.first ? at.first : t;
    const int tile = t / L, last = at.end - 1 - t;
    ahead.since = c.parts > 1 ? at.row_line(c, c.since, tile)[at.channel] : cut_span<T>();
    const T *x = at.line(c, c.x, t), *delta = at.line(c, c.delta, t), *grad = at.line(c, c.grad, t), *gate = at.line(c, gates_or_x, t);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const unsigned from = at.place(c, own + i < last ? own + i : last);
      ahead.x[i] = x[from];
      ahead.delta[i] = delta[from];
      ahead.grad[i] = grad[from];
      ahead.gate[i] = gate[from];
    }
    ahead.b.load(c, at, b_, t);
    ahead.c.load(c, at, c_, t);
#pragma unroll
    for (int s = 0; s < S; ++s) ahead.before[s] = at.state_line(c, c.before, tile, s)[at.channel];
    if (RESETS) ahead.resets = c.rows.byte(at.row, t, at.end, lane);
  };
  // What a tile needs besides shared_*: of the wave's own steps x and the slopes of dt, and of y by the gate times dy.
  struct Ready {
    T x[kOwn], slope[kOwn], passes[kOwn], start[S];
    Projections<T, L, S> b, c;
    unsigned starts;
  };
  const auto prepare = [&](int t, int turn) __attribute__((always_inline)) {
    const int count = at.end - t < L ? at.end - t : L;
    Ready r;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool inside = at.valid && own + i < count;
      r.x[i] = ahead.x[i];
      const T dt = softplus(ahead.delta[i] + bias, r.slope[i]);
      T keep, rest;
      gates(ahead.gate[i], keep, rest);
      r.passes[i] = ahead.grad[i] * (keep * (T(1) + ahead.gate[i] * rest));
      const T g = c.gate ? ahead.grad[i] * (ahead.gate[i] * keep) : ahead.grad[i];
      shared_dt[turn][own + i][lane] = inside ? dt : T(0);
      shared_u[turn][own + i][lane] = inside ? dt * ahead.x[i] : T(0);
      shared_g[turn][own + i][lane] = inside ? g : T(0);
      apart<T>();
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      r.start[s] = ahead.before[s];
      if (c.parts > 1) r.start[s] = passed(ahead.since, rate[s], arrived[s], r.start[s]);
      if (!at.valid) r.start[s] = T(0);
    }
    r.b = ahead.b, r.c = ahead.c;
    r.b.keep(lane, count);
    r.c.keep(lane, count);
    r.starts = RESETS ? unsigned(__ballot(ahead.resets != 0 && lane < count)) : 0;
    return r;
  };
  Ready next{};
  if (tiles) {
    load(at.first + (tiles - 1) * L);
    next = prepare(at.first + (tiles - 1) * L, 0);
    load(at.first + (tiles - 2) * L);
  }
  __syncthreads();
  int turn = 0;
  for (int n = tiles - 1; n >= 0; --n, turn ^= 1) {
    const int t = at.first + n * L;
    const int count = at.end - t < L ? at.end - t : L;
    Ready now = next;
    auto &bs = now.b, &cs = now.c;
    const auto& start = now.start;
    const unsigned starts = now.starts;
    // The tile before it, beside this one's work: its loads are there, and, half way through the walk, so are the
    // stores of the tile behind it. (Doubles at once, while the walk does not have the registers yet.) Before the
    // first tile there is none, and nothing reads what this leaves.
    const auto prepare_next = [&]() __attribute__((always_inline)) {
      next = prepare(t - L < at.first ? at.first : t - L, turn ^ 1);
      load(t - 2 * L);
    };
    if constexpr (sizeof(T) == 8) prepare_next();
    // Read for some steps at a time, and again on the way back: all of them would take registers from the states.
    constexpr int kSome = sizeof(T) == 4 ? 8 : 2;
    T dts[L], us[L], gs[L];
    const auto walk = [&](auto resets) __attribute__((always_inline)) {
      T h[L][S], keep[L][S];
      for_each<L>([&](auto step) {
        constexpr int i = step;
        if constexpr (i % kSome == 0) {
#pragma unroll
          for (int k = i; k < i + kSome; ++k) dts[k] = shared_dt[turn][k][lane], us[k] = shared_u[turn][k][lane];
          __builtin_amdgcn_sched_barrier(0);
        }
        const T dt = dts[i], u = us[i];
        const bool cut = resets && (starts >> i & 1);
        for_each<S>([&](auto state) {
          constexpr int s = state;
          keep[i][s] = decay(dt, rate[s]);
          T before = start[s];
          if constexpr (i > 0) before = h[i - 1][s];
          h[i][s] = __builtin_elementwise_fma(keep[i][s], cut ? T(0) : before, u * bs.template get<i, s>());
        });
        apart<T>();
      });
      if constexpr (sizeof(T) == 4) prepare_next();
      bs.renew();
      T pairs_b[S][L / 2], pairs_c[S][L / 2], last_b[S], last_c[S];
      for_each<L>([&](auto step) {
        constexpr int i = L - 1 - step;
        if constexpr (step % kSome == 0) {
#pragma unroll
          for (int k = i; k > i - kSome; --k) dts[k] = shared_dt[turn][k][lane], us[k] = shared_u[turn][k][lane], gs[k] = shared_g[turn][k][lane];
          __builtin_amdgcn_sched_barrier(0);
        }
        const T dt = dts[i], u = us[i], g = gs[i];
        const bool cut = resets && (starts >> i & 1);
        T along = T(0), decays = T(0), y = T(0), to_b[S], to_c[S];
        for_each<S>([&](auto state) {
          constexpr int s = state;
          const T m = __builtin_elementwise_fma(cs.template get<i, s>(), g, e[s]);
          to_c[s] = g * h[i][s];
          to_b[s] = u * m;
          const T part = bs.template get<i, s>() * m;  // takes the broadcast on the way
          along = s ? along + part : part;
          y = __builtin_elementwise_fma(cs.template get<i, s>(), h[i][s], y);
          e[s] = cut ? T(0) : keep[i][s] * m;
          T before = start[s];
          if constexpr (i > 0) before = h[i - 1][s];
          const T share = cut ? T(0) : e[s] * before;
          decays = __builtin_elementwise_fma(share, slow[s], decays);
          da[s] = __builtin_elementwise_fma(share, dt, da[s]);
        });
        sums_b[at.wave][i][lane] = along;
        sums_a[at.wave][i][lane] = decays;
        sums_y[at.wave][i][lane] = y;  // without gates too: a branch in every step would keep the steps' work apart
#pragma unroll
        for (int s = 0; s < S; ++s) {
          if constexpr (i % 2) {
            last_b[s] = to_b[s], last_c[s] = to_c[s];
          } else {
            pairs_b[s][i / 2] = fold_pair<8>(to_b[s], last_b[s], lane & 8);
            pairs_c[s][i / 2] = fold_pair<8>(to_c[s], last_c[s], lane & 8);
          }
        }
      });
      // Rows of lanes with bit 4 get the sums of dc.
      const T all = fold_rows<4>(fold<T, S, L>(pairs_b, lane), fold<T, S, L>(pairs_c, lane));
      const int i = step_of_lane<L>(lane), s = state_of_lane<S>(lane);
      if (i < count && (S * L == 32 || !(lane & 1))) {
        const int64_t step = (int64_t(at.piece) * c.batch + at.row) * c.time + t, to = (step * c.groups + at.group) * (NW * S) + at.slot;
        ((lane & 16 ? o.dc : o.db) + to)[unsigned(i * c.groups) * (NW * S) + s] = all;
      }
    };
    if (RESETS && now.starts) walk(std::true_type{});  // few tiles have one
    else walk(std::false_type{});
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (!at.valid || t + own + i >= at.end) break;
      T along = T(0), decays = T(0), y = T(0);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        along += sums_b[w][own + i][lane];
        decays += sums_a[w][own + i][lane];
        y += sums_y[w][own + i][lane];
      }
      const unsigned to = at.place(c, own + i);
      T *to_x = at.line(c, o.dx, t) + to, *to_delta = at.line(c, o.ddelta, t) + to;
      const T dt = shared_dt[turn][own + i][lane], g = shared_g[turn][own + i][lane];
      T dx = along * dt, ddt = __builtin_elementwise_fma(along, now.x[i], decays);
      if (!c.starts) dx += *to_x, ddt += *to_delta;
      else if (c.skip) dx = __builtin_elementwise_fma(skip, g, dx);
      if (c.ends) {
        ddt *= now.slope[i];
        dbias += ddt;
        if (c.skip) dskip = __builtin_elementwise_fma(g, now.x[i], dskip);
      }
      *to_x = dx;
      *to_delta = ddt;
      if (c.gate) {
        T* to_gate = at.line(c, o.dgate, t) + to;
        if (!c.starts) y += *to_gate;
        if (c.ends) {
          if (c.skip) y = __builtin_elementwise_fma(skip, now.x[i], y);
          y *= now.passes[i];
        }
        *to_gate = y;
      }
    }
    __syncthreads();
  }
  const int64_t line = int64_t(at.row) * c.parts + at.part;
  if (at.valid) {
#pragma unroll
    for (int s = 0; s < S; ++s) (o.da + (line * (NW * S) + at.slot + s) * c.channels)[at.channel] = da[s] * slow[s];
    if (o.dinitial && at.part == 0) at.write(c, o.dinitial, at.row, e);
  }
  if (!c.ends) return;
  // The waves' sums over their own steps.
  sums_a[at.wave][0][lane] = dskip;
  sums_b[at.wave][0][lane] = dbias;
  __syncthreads();
  if (at.wave == 0 && at.valid) {
    for (int w = 1; w < NW; ++w) dskip += sums_a[w][0][lane], dbias += sums_b[w][0][lane];
    o.dskip[line * c.channels + at.channel] = dskip;
    o.dbias[line * c.channels + at.channel] = dbias;
  }
}

// db and dc (batch, time, groups, states) from the pieces' parts; zero behind the rows' ends.
template <typename T>
__global__ __launch_bounds__(256) void projections_kernel(Scan<T> c, Grads<T> o, int width, T* db, T* dc) {
  const int64_t lines = int64_t(c.batch) * c.time * c.groups, n = lines * width;
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t line = i / width, s = i - line * width + c.first;
    if (s >= c.states) continue;
    const int64_t step = line / c.groups, row = step / c.time;
    T b = T(0), d = T(0);
    if (step - row * c.time < c.rows.end(row)) {
      for (int p = 0; p < c.pieces; ++p) b += o.db[p * n + i], d += o.dc[p * n + i];
    }
    db[line * c.states + s] = b;
    dc[line * c.states + s] = d;
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void decays_kernel(Scan<T> c, const T* parts, int width, T* da) {
  const int64_t columns = int64_t(width) * c.channels;
  add_parts(parts, columns, 0, int64_t(c.batch) * c.parts, int64_t(blockIdx.x) * 64, columns, [&](int64_t q, T sum) {
    const int64_t s = q / c.channels, channel = q - s * c.channels;
    if (c.first + s < c.states) da[channel * c.states + c.first + s] = sum;
  });
}

template <typename T>
__global__ __launch_bounds__(1024) void channels_kernel(Scan<T> c, const T* skips, T* dskip, const T* biases, T* dbias) {
  T* to = blockIdx.y ? dbias : dskip;
  if (!to) return;
  add_parts(blockIdx.y ? biases : skips, c.channels, 0, int64_t(c.batch) * c.parts, int64_t(blockIdx.x) * 64, c.channels, [&](int64_t q, T sum) { to[q] = sum; });
}

}  // namespace

extern "C" {

int hp_selective_scan_grad(hp_ctx* ctx, int dtype, int index_dtype, const void* grad, const void* grad_state, const void* x,
                           const void* delta, const void* a_log, const void* b, const void* c, const void* skip, const void* gate,
                           const void* initial, const void* delta_bias, const void* resets, const void* lengths, void* dx,
                           void* ddelta, void* da_log, void* db, void* dc, void* dskip, void* dgate, void* ddelta_bias,
                           void* dinitial, int64_t batch, int64_t time, int64_t channels, int64_t groups, int64_t states) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::scan_check(dtype, index_dtype, batch, time, channels, groups, states);
    const auto run = [&](auto zero) {
      using T = decltype(zero);
      const auto in = [](const void* p) { return static_cast<const T*>(p); };
      const auto out = [](void* p) { return static_cast<T*>(p); };
      if (batch * time * channels == 0) {
        hp::scan_fill<T>(ctx, out(da_log), nullptr, channels * states);
        hp::scan_fill<T>(ctx, out(dskip), nullptr, channels);
        hp::scan_fill<T>(ctx, out(ddelta_bias), nullptr, channels);
        hp::scan_fill<T>(ctx, out(db), nullptr, batch * time * groups * states);
        hp::scan_fill<T>(ctx, out(dc), nullptr, batch * time * groups * states);
        hp::scan_fill<T>(ctx, out(dinitial), in(grad_state), batch * channels * states);
        return;
      }
      hp::require(grad && x && delta && a_log && b && c && dx && ddelta && da_log && db && dc, "null pointer");
      hp::require((!gate || dgate) && (!initial || dinitial), "null pointer");
      hp::Scratch scratch(ctx);
      Scan<T> s{};
      s.x = in(x), s.delta = in(delta), s.a_log = in(a_log), s.skip = in(skip), s.gate = in(gate), s.initial = in(initial), s.delta_bias = in(delta_bias);
      s.grad = in(grad), s.grad_state = in(grad_state);
      s.rows = {static_cast<const uint8_t*>(resets), lengths, index_dtype == HP_I64, time};
      // As forward; four states a wave would not leave as many waves their registers for more than 32. Doubles
      // take twice the registers: four waves of two states leave each what it needs, for few states too.
      const bool many = sizeof(T) == 4 && states > 16;
      const int each = many ? 4 : 2, waves = sizeof(T) == 4 ? hp::scan_waves(states, each, 8) : 4, width = waves * each;
      hp::scan_sizes(s, batch, time, channels, groups, states, width);
      hp::scan_plan(s, kLongestTile);
      const T *bs = hp::scan_padded(ctx, scratch, in(b), batch * time * groups, states, s.padded);
      const T *cs = hp::scan_padded(ctx, scratch, in(c), batch * time * groups, states, s.padded);
      const int64_t lines = batch * time * groups, rows = batch * s.parts;
      if (s.parts > 1) {
        s.spans = scratch.take<T>(rows * channels);
        s.ended = scratch.take<T>(rows * width * channels);
        s.passed = scratch.take<T>(rows * width * channels);
      }
      Grads<T> o{};
      o.dx = out(dx), o.ddelta = out(ddelta), o.dgate = out(dgate), o.dinitial = out(dinitial);
      o.db = scratch.take<T>(s.pieces * lines * width), o.dc = scratch.take<T>(s.pieces * lines * width);
      o.da = scratch.take<T>(rows * width * channels);
      o.dskip = scratch.take<T>(rows * channels), o.dbias = scratch.take<T>(rows * channels);
      const unsigned blocks = unsigned(batch * groups * s.pieces * s.parts);
      hp::require(hp::ceil_div(int64_t(width) * channels, int64_t(64)) <= hp::kMaxThreads / 1024, "too many channels for one launch");
      for (s.first = 0; s.first < states; s.first += width) {
        s.starts = s.first == 0;
        s.ends = s.first + width >= states;
        const auto launch = [&](auto nw, auto of) {
          constexpr int NW = nw, S = of;
          if (s.starts) {
            const int64_t tiles = hp::ceil_div(time, int64_t(kTile<T, NW, S>));
            s.before = scratch.take<T>(tiles * batch * width * channels);
            if (s.parts > 1) s.since = scratch.take<T>(tiles * batch * channels);
          }
          const auto first = s.parts > 1 ? (resets ? before_kernel<T, NW, S, true, true> : before_kernel<T, NW, S, false, true>)
                                         : (resets ? before_kernel<T, NW, S, true, false> : before_kernel<T, NW, S, false, false>);
          first<<<blocks, NW * 64, 0, ctx->stream>>>(s, bs, cs);
          hp::check_launch("scan states");
          const auto second = resets ? backward_kernel<T, NW, S, true> : backward_kernel<T, NW, S, false>;
          second<<<blocks, NW * 64, 0, ctx->stream>>>(s, o, bs, cs);
          hp::check_launch("scan gradient");
        };
        using Two = std::integral_constant<int, 2>;
        using Four = std::integral_constant<int, 4>;
        using Eight = std::integral_constant<int, 8>;
        if constexpr (sizeof(T) == 4) {
          if (many) launch(Eight{}, Four{});
          else if (waves == 8) launch(Eight{}, Two{});
          else if (waves == 2) launch(Two{}, Two{});
        }
        if (waves == 4) launch(Four{}, Two{});
        projections_kernel<T><<<unsigned(std::min<int64_t>(hp::ceil_div(lines * width, 256), 8192)), 256, 0, ctx->stream>>>(s, o, width, out(db), out(dc));
        hp::check_launch("scan projections");
        decays_kernel<T><<<unsigned(hp::ceil_div(width * channels, int64_t(64))), 1024, 0, ctx->stream>>>(s, o.da, width, out(da_log));
        hp::check_launch("scan rates");
      }
      channels_kernel<T><<<dim3(unsigned(hp::ceil_div(channels, 64)), 2), 1024, 0, ctx->stream>>>(s, o.dskip, out(dskip), o.dbias, out(ddelta_bias));
      hp::check_launch("scan sums");
    };
    if (dtype == HP_F32) run(float(0));
    else run(double(0));
  });
}

}  // extern "C"
