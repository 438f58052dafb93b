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
// until a register holds a sum in each lane: two instructions a value where a sum over 64 lanes
// by itself takes six times two. Workgroups leave these, and their sums over steps, as parts.
//
// Where rows are cut into parts, the first launch also forms what a part passes back from
// nothing, sum_t D_t c_t g_t with D_t the product of the decays up to t.
#include "scan.h"

using namespace hpd;

namespace {

// Steps of a tile, and waves of a launch, for the registers that a tile's states and decays take.
template <typename T, int NW, int S>
constexpr int kTile = sizeof(T) == 4 ? (S == 4 && NW == 8 ? 8 : 16) : NW == 1 ? 4 : 8;
template <typename T>
constexpr int kMostWaves = sizeof(T) == 4 ? 8 : 4;
constexpr int kLongestTile = 16;

template <typename T, int NW, int S, bool RESETS, bool SPLIT>
__global__ __launch_bounds__(NW * 64) void before_kernel(Scan<T> c, const T* b_, const T* c_) {
  constexpr int L = kTile<T, NW, S>, kOwn = L / NW;
  __shared__ T shared_dt[L][64], shared_u[L][64], shared_g[SPLIT ? L : 1][64];
  const Place<T, NW, S> at(c);
  const int lane = at.lane, own = at.wave * kOwn;
  T rate[S], h[S], through[S], back[S], span = T(0);
  at.read(c, c.a_log, 0, rate);
#pragma unroll
  for (int s = 0; s < S; ++s) rate[s] = rate_of(rate[s]), h[s] = back[s] = T(0), through[s] = T(1);
  if (!SPLIT && c.initial) at.read(c, c.initial, at.row, h);
  const T bias = c.delta_bias ? c.delta_bias[at.channel] : T(0);
  T x[kOwn], delta[kOwn], grad[kOwn], gate[kOwn];
  Projections<T, L, S> next_b, next_c;
  bool cut = false;
  const auto load = [&](int64_t t) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int64_t step = t + own + i < at.end ? t + own + i : at.end - 1;
      x[i] = at.get(c, c.x, step);
      delta[i] = at.get(c, c.delta, step);
      if constexpr (SPLIT) {
        grad[i] = at.get(c, c.grad, step);
        if (c.gate) gate[i] = at.get(c, c.gate, step);
      }
    }
    next_b.load(c, at, b_, t);
    if (SPLIT) next_c.load(c, at, c_, t);
  };
  if (at.first < at.end) load(at.first);
  for (int64_t t = at.first; t < at.end; t += L) {
    const int count = at.end - t < L ? int(at.end - t) : L;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool inside = own + i < count;
      T slope;
      const T dt = softplus(delta[i] + bias, slope);
      shared_dt[own + i][lane] = inside ? dt : T(0);
      shared_u[own + i][lane] = inside ? dt * x[i] : T(0);
      if constexpr (SPLIT) {
        T g = grad[i];
        if (c.gate) {
          T keep, rest;
          gates(gate[i], keep, rest);
          g *= gate[i] * keep;
        }
        shared_g[own + i][lane] = inside ? g : T(0);
      }
    }
    Projections<T, L, S> bs = next_b, cs = next_c;
    bs.keep(lane, count);
    if (SPLIT) cs.keep(lane, count);
    __syncthreads();
    if (t + L < at.end) load(t + L);
    const int64_t tile = t / L;
    if (at.valid) {
#pragma unroll
      for (int s = 0; s < S; ++s) c.before[at.state_at(c, tile, s)] = h[s];
      if (SPLIT && at.wave == 0) c.since[(tile * c.batch + at.row) * c.channels + at.channel] = cut ? cut_span<T>() : span;
    }
    const unsigned starts = RESETS ? __builtin_amdgcn_readfirstlane(c.rows.template starts<L>(at.row, t, at.end)) : 0;
    // Tiles without a reset, nearly all of them, do without its selects.
    const auto walk = [&](auto resets) {
      for_each<L>([&](auto step) {
        constexpr int i = step;
        const bool start = resets && (starts >> i & 1);
        const T dt = shared_dt[i][lane], u = shared_u[i][lane];
        T g = T(0);
        if constexpr (SPLIT) {
          cut = cut || start;
          g = RESETS && cut ? T(0) : shared_g[i][lane];
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
    else walk(std::false_type{});
    __syncthreads();
  }
  if constexpr (SPLIT) {
    if (!at.valid) return;
    if (at.wave == 0) c.spans[(at.part * c.batch + at.row) * c.channels + at.channel] = cut ? cut_span<T>() : span;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      c.ended[at.state_at(c, at.part, s)] = h[s];
      c.passed[at.state_at(c, at.part, s)] = back[s];
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

// Exchanges halves (BIT 5) or odd and even rows of 16 lanes (BIT 4) between a and b.
template <int BIT>
__device__ __forceinline__ void swap_lanes(uint32_t& a, uint32_t& b) {
  if constexpr (BIT == 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
  }
}
// Lane i: the value of lane i ^ 8 (8), i ^ 7 (7), i ^ 3 (3) or i ^ 1 (1).
template <int MASK>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  constexpr int kind = MASK == 8 ? 0x128 /* row_ror:8 */ : MASK == 7 ? 0x141 /* row_half_mirror */ : MASK == 3 ? 0x1B /* quad_perm 3 2 1 0 */ : 0xB1 /* 1 0 3 2 */;
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kind, 0xF, 0xF, true));
}

template <typename T>
struct Words {
  uint32_t w[sizeof(T) / 4];
};

template <int BIT, typename T>
__device__ __forceinline__ T fold_rows(T a, T b) {
  auto x = __builtin_bit_cast(Words<T>, a), y = __builtin_bit_cast(Words<T>, b);
#pragma unroll
  for (unsigned k = 0; k < sizeof(T) / 4; ++k) swap_lanes<BIT>(x.w[k], y.w[k]);
  return __builtin_bit_cast(T, x) + __builtin_bit_cast(T, y);
}
template <int MASK, typename T>
__device__ __forceinline__ T from_across(T v) {
  auto x = __builtin_bit_cast(Words<T>, v);
#pragma unroll
  for (unsigned k = 0; k < sizeof(T) / 4; ++k) x.w[k] = across<MASK>(x.w[k]);
  return __builtin_bit_cast(T, x);
}
// Lanes without `bit` get a's sums over pairs of lanes, those with it b's.
template <int MASK, typename T>
__device__ __forceinline__ T fold_pair(T a, T b, bool bit) {
  return (bit ? b : a) + from_across<MASK>(bit ? a : b);
}

// Of N values (4, 8 or 16) the sums over a row of 16 lanes: lane i has value number_of_lane(i).
// Pairs meet across 8, 7, 3 and 1 lanes, which reaches all 16.
template <typename T, int N>
__device__ __forceinline__ T fold_row(const T (&v)[N], int lane) {
  T a[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) a[k] = fold_pair<8>(v[2 * k], v[2 * k + 1], lane & 8);
  T b[N / 4];
#pragma unroll
  for (int k = 0; k < N / 4; ++k) b[k] = fold_pair<7>(a[2 * k], a[2 * k + 1], lane & 4);
  T d[N < 8 ? 1 : N / 8];
  if constexpr (N >= 8) {
#pragma unroll
    for (int k = 0; k < N / 8; ++k) d[k] = fold_pair<3>(b[2 * k], b[2 * k + 1], lane & 2);
  } else {
    d[0] = b[0] + from_across<3>(b[0]);
  }
  if constexpr (N == 16) return fold_pair<1>(d[0], d[1], lane & 1);
  else return d[0] + from_across<1>(d[0]);
}
template <int N>
__device__ __forceinline__ int number_of_lane(int lane) {
  return (lane >> 3 & 1) | (lane >> 2 & 1) << 1 | (N >= 8 ? (lane >> 1 & 1) << 2 : 0) | (N == 16 ? (lane & 1) << 3 : 0);
}

// Of S values for each of L steps the sums over all lanes: lane i has that of step
// step_of_lane(i) and state state_of_lane(i).
template <int S, typename T>
__device__ __forceinline__ T fold_states(const T (&v)[S]) {
  if constexpr (S == 4) return fold_rows<4>(fold_rows<5>(v[0], v[1]), fold_rows<5>(v[2], v[3]));
  else return fold_rows<5>(v[0], v[1]);
}
template <int S, typename T, int L>
__device__ __forceinline__ T fold_steps(const T (&v)[L], int lane) {
  if constexpr (S == 4) return fold_row<T, L>(v, lane);
  else {
    T pairs[L / 2];
#pragma unroll
    for (int k = 0; k < L / 2; ++k) pairs[k] = fold_rows<4>(v[2 * k], v[2 * k + 1]);
    return fold_row<T, L / 2>(pairs, lane);
  }
}
template <int S, int L>
__device__ __forceinline__ int step_of_lane(int lane) {
  return S == 4 ? number_of_lane<L>(lane) : (lane >> 4 & 1) | number_of_lane<L / 2>(lane) << 1;
}
template <int S>
__device__ __forceinline__ int state_of_lane(int lane) {
  return (lane >> 5 & 1) | (S == 4 ? (lane >> 4 & 1) << 1 : 0);
}
// Of the lanes that have the same sum, the one that leaves it.
template <int S, int L>
__device__ __forceinline__ bool leaves(int lane) {
  return lane % (64 / (S * L)) == 0;
}

// ---- backward ------------------------------------------------------------------------

template <typename T, int NW, int S, bool RESETS>
__global__ __launch_bounds__(NW * 64) void backward_kernel(Scan<T> c, Grads<T> o, const T* b_, const T* c_) {
  constexpr int L = kTile<T, NW, S>, kOwn = L / NW;
  __shared__ T shared_dt[L][64], shared_u[L][64], shared_g[L][64];
  __shared__ T sums_b[NW][L][64], sums_a[NW][L][64], sums_y[NW][L][64];
  const Place<T, NW, S> at(c);
  const int lane = at.lane, own = at.wave * kOwn;
  T rate[S], slow[S], e[S], da[S];
  at.read(c, c.a_log, 0, slow);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    rate[s] = rate_of(slow[s]);
    slow[s] = sizeof(T) == 4 ? -T(expf(float(slow[s]))) : rate[s];
    e[s] = da[s] = T(0);
  }
  T arrived[S] = {};
  if (c.parts > 1) {
    at.arrive(c, rate, arrived);
    if (c.grad_state) at.read(c, c.grad_state, at.row, e);
    for (int64_t p = c.parts - 1; p > at.part; --p) {
      const T span = c.spans[(p * c.batch + at.row) * c.channels + at.channel];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const T back = c.passed[at.state_at(c, p, s)];
        e[s] = span < T(0) ? back : __builtin_elementwise_fma(passed_decay(span, rate[s]), e[s], back);
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
  const int64_t stop = at.first + c.steps < c.rows.time ? at.first + c.steps : c.rows.time;
  for (int64_t t = (at.end > at.first ? at.end : at.first) + at.wave; t < stop; t += NW) {
    const int64_t to = at.at(c, t);
    if (!at.valid) continue;
    o.dx[to] = o.ddelta[to] = T(0);
    if (c.gate) o.dgate[to] = T(0);
  }
  const int64_t tiles = at.end > at.first ? (at.end - at.first + L - 1) / L : 0;
  T next_x[kOwn], delta[kOwn], gate[kOwn], grad[kOwn], before[S], since = cut_span<T>();
  Projections<T, L, S> next_b, next_c;
  const auto load = [&](int64_t t) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int64_t step = t + own + i < at.end ? t + own + i : at.end - 1;
      next_x[i] = at.get(c, c.x, step);
      delta[i] = at.get(c, c.delta, step);
      grad[i] = at.get(c, c.grad, step);
      if (c.gate) gate[i] = at.get(c, c.gate, step);
    }
    next_b.load(c, at, b_, t);
    next_c.load(c, at, c_, t);
    const int64_t tile = t / L;
#pragma unroll
    for (int s = 0; s < S; ++s) before[s] = c.before[at.state_at(c, tile, s)];
    if (c.parts > 1) since = c.since[(tile * c.batch + at.row) * c.channels + at.channel];
  };
  if (tiles) load(at.first + (tiles - 1) * L);
  for (int64_t n = tiles - 1; n >= 0; --n) {
    const int64_t t = at.first + n * L;
    const int count = at.end - t < L ? int(at.end - t) : L;
    T x[kOwn], slope[kOwn], passes[kOwn];  // of the wave's own steps; slopes of dt, and of y by the gate times dy
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool inside = at.valid && own + i < count;
      x[i] = next_x[i];
      const T dt = softplus(delta[i] + bias, slope[i]);
      T g = grad[i];
      if (c.gate) {
        T keep, rest;
        gates(gate[i], keep, rest);
        passes[i] = g * (keep * (T(1) + gate[i] * rest));
        g *= gate[i] * keep;
      }
      shared_dt[own + i][lane] = inside ? dt : T(0);
      shared_u[own + i][lane] = inside ? dt * x[i] : T(0);
      shared_g[own + i][lane] = inside ? g : T(0);
    }
    T start[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      start[s] = before[s];
      if (since >= T(0)) start[s] = __builtin_elementwise_fma(passed_decay(since, rate[s]), arrived[s], start[s]);
      if (!at.valid) start[s] = T(0);
    }
    Projections<T, L, S> bs = next_b, cs = next_c;
    bs.keep(lane, count);
    cs.keep(lane, count);
    __syncthreads();
    if (n > 0) load(t - L);
    const unsigned starts = RESETS ? __builtin_amdgcn_readfirstlane(c.rows.template starts<L>(at.row, t, at.end)) : 0;
    const auto walk = [&](auto resets) {
      T h[L][S], keep[L][S];
      for_each<L>([&](auto step) {
        constexpr int i = step;
        const T dt = shared_dt[i][lane], u = shared_u[i][lane];
        const bool cut = resets && (starts >> i & 1);
        for_each<S>([&](auto state) {
          constexpr int s = state;
          keep[i][s] = decay(dt, rate[s]);
          T before = start[s];
          if constexpr (i > 0) before = h[i - 1][s];
          h[i][s] = __builtin_elementwise_fma(keep[i][s], cut ? T(0) : before, u * bs.template get<i, s>());
        });
      });
      bs.renew();
      T rows_b[L], rows_c[L];
      for_each<L>([&](auto step) {
        constexpr int i = L - 1 - step;
        const T dt = shared_dt[i][lane], u = shared_u[i][lane], g = shared_g[i][lane];
        const bool cut = resets && (starts >> i & 1);
        T along = T(0), decays = T(0), y = T(0), to_b[S], to_c[S];
        for_each<S>([&](auto state) {
          constexpr int s = state;
          const T m = __builtin_elementwise_fma(cs.template get<i, s>(), g, e[s]);
          to_c[s] = g * h[i][s];
          to_b[s] = u * m;
          along = __builtin_elementwise_fma(bs.template get<i, s>(), m, along);
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
        if (c.gate) sums_y[at.wave][i][lane] = y;
        rows_b[i] = fold_states<S>(to_b);
        rows_c[i] = fold_states<S>(to_c);
      });
      const T all_b = fold_steps<S>(rows_b, lane), all_c = fold_steps<S>(rows_c, lane);
      const int i = step_of_lane<S, L>(lane), s = state_of_lane<S>(lane);
      if (i < count && leaves<S, L>(lane)) {
        const int64_t line = (at.row * c.rows.time + t + i) * c.groups + at.group, lines = c.batch * c.rows.time * c.groups;
        const int64_t to = (at.piece * lines + line) * (NW * S) + at.slot + s;
        o.db[to] = all_b;
        o.dc[to] = all_c;
      }
    };
    if (RESETS && starts) walk(std::true_type{});
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
        if (c.gate) y += sums_y[w][own + i][lane];
      }
      const int64_t to = at.at(c, t + own + i);
      const T dt = shared_dt[own + i][lane], g = shared_g[own + i][lane];
      T dx = along * dt, ddt = __builtin_elementwise_fma(along, x[i], decays);
      if (!c.starts) dx += o.dx[to], ddt += o.ddelta[to];
      else if (c.skip) dx = __builtin_elementwise_fma(skip, g, dx);
      if (c.ends) {
        ddt *= slope[i];
        dbias += ddt;
        if (c.skip) dskip = __builtin_elementwise_fma(g, x[i], dskip);
      }
      o.dx[to] = dx;
      o.ddelta[to] = ddt;
      if (c.gate) {
        if (!c.starts) y += o.dgate[to];
        if (c.ends) {
          if (c.skip) y = __builtin_elementwise_fma(skip, x[i], y);
          y *= passes[i];
        }
        o.dgate[to] = y;
      }
    }
  }
  const int64_t line = at.row * c.parts + at.part;
  if (at.valid) {
#pragma unroll
    for (int s = 0; s < S; ++s) o.da[(line * (NW * S) + at.slot + s) * c.channels + at.channel] = da[s] * slow[s];
    if (o.dinitial && at.part == 0) at.write(c, o.dinitial, at.row, e);
  }
  if (!c.ends) return;
  // The waves' sums over their own steps.
  __syncthreads();
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
  const int64_t lines = c.batch * c.rows.time * c.groups, n = lines * width;
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t line = i / width, s = i - line * width + c.first;
    if (s >= c.states) continue;
    const int64_t step = line / c.groups, row = step / c.rows.time;
    T b = T(0), d = T(0);
    if (step - row * c.rows.time < c.rows.end(row)) {
      for (int64_t p = 0; p < c.pieces; ++p) b += o.db[p * n + i], d += o.dc[p * n + i];
    }
    db[line * c.states + s] = b;
    dc[line * c.states + s] = d;
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void decays_kernel(Scan<T> c, const T* parts, int width, T* da) {
  const int64_t columns = width * c.channels;
  add_parts(parts, columns, 0, c.batch * c.parts, int64_t(blockIdx.x) * 64, columns, [&](int64_t q, T sum) {
    const int64_t s = q / c.channels, channel = q - s * c.channels;
    if (c.first + s < c.states) da[channel * c.states + c.first + s] = sum;
  });
}

template <typename T>
__global__ __launch_bounds__(1024) void channels_kernel(Scan<T> c, const T* skips, T* dskip, const T* biases, T* dbias) {
  T* to = blockIdx.y ? dbias : dskip;
  if (!to) return;
  add_parts(blockIdx.y ? biases : skips, c.channels, 0, c.batch * c.parts, int64_t(blockIdx.x) * 64, c.channels, [&](int64_t q, T sum) { to[q] = sum; });
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
      s.batch = batch, s.channels = channels, s.groups = groups, s.states = states;
      s.width = channels / groups, s.pieces = hp::ceil_div(s.width, 64);
            hp::scan_plan(s, kLongestTile);
      // Doubles of two states in eight waves would not fit into their registers.
      const int each = sizeof(T) == 4 ? hp::scan_states(s) : 4, waves = hp::scan_waves(states, each, kMostWaves<T>), width = waves * each;
      s.padded = hp::ceil_div(states, width) * width;
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
      hp::require(hp::ceil_div(width * channels, int64_t(64)) <= hp::kMaxThreads / 1024, "too many channels for one launch");
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
          if (each == 2 && waves == 2) launch(Two{}, Two{});
          else if (each == 2 && waves == 4) launch(Four{}, Two{});
          else if (each == 2) launch(Eight{}, Two{});
          else if (waves == 8) launch(Eight{}, Four{});
        }
        if (each == 4) {
          if (waves == 1) launch(std::integral_constant<int, 1>{}, Four{});
          else if (waves == 2) launch(Two{}, Four{});
          else if (waves == 4) launch(Four{}, Four{});
        }
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
