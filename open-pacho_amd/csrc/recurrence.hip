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
// alignment; a workgroup owns 64 channels, and its W waves consecutive runs of R
// steps. Each wave loads its run into registers, composes it, leaves (A, B) in
// LDS, takes what the waves before it left, and then computes and stores its
// states: one pass over the data, one barrier for each R x W steps. Two sets of
// registers take turns, so that the next run's loads are in flight while a run
// is computed.
//
// Few channels would leave compute units idle: then time is cut into segments
// for workgroups of their own, and a kernel before composes each segment, at the
// price of reading the gates and x (backward: the gradient) twice.
#include <type_traits>

#include "common.h"
#include "exponential.h"

namespace {

// Steps of a wave's run.
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

constexpr unsigned kDies = 8;  // of the chip, each with a cache of its own

struct Extents {
  int64_t time;      // steps of a row
  int64_t total;     // rows x channels
  int64_t channels;  // of a step
  int64_t gates;     // of a step
  int64_t width;     // channels that share a gate: channels / gates
  int64_t groups;    // of 64 lanes
  int64_t segment;   // steps of a segment
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
    const T* p = column + t * stride;
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = p[i * stride];
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = t + i >= 0 && t + i < end ? column[(t + i) * stride] : outside;
  }
}

// Bit i: a reset at step t + i.
template <int R>
__device__ __forceinline__ unsigned load_resets(const uint8_t* row, int64_t t, int64_t end) {
  unsigned bits = 0;
  if (R % 4 == 0 && t >= 0 && t + R <= end) {
    typedef uint32_t U __attribute__((ext_vector_type(R < 4 ? 1 : R / 4), aligned(1)));
    const U v = *reinterpret_cast<const U*>(row + t);
    // The top bit of a byte is set where it is not 0; a product gathers four of them.
#pragma unroll
    for (int j = 0; j < R / 4; ++j) {
      const unsigned set = (((v[j] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | v[j]) >> 7 & 0x01010101u;
      bits |= (set * 0x01020408u >> 24 & 15) << 4 * j;
    }
    return bits;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (t + i >= 0 && t + i < end) bits |= unsigned(row[t + i] != 0) << i;
  }
  return bits;
}

// What the waves of a workgroup leave for each other; two sets, so that one
// barrier is enough.
template <typename T, int W>
struct Left {
  T a[2][W][64], b[2][W][64];
};

// Takes `before` through the runs of all waves in their order: `before` becomes
// the value after the last one, the result is the one before this wave's run.
template <typename T, int W>
__device__ __forceinline__ T through(const Run<T>& run, Left<T, W>& left, int turn, int wave, int lane, T& before) {
  if constexpr (W == 1) {
    const T now = before;
    before = apply(run.cut ? T(-1) : run.a, run.b, before);
    return now;
  }
  left.a[turn][wave][lane] = run.cut ? T(-1) : run.a;
  left.b[turn][wave][lane] = run.b;
  __syncthreads();
  T now = before;
#pragma unroll
  for (int first = 0; first < W; first += 4) {  // four waves' at a time: two registers each
    T a[4], b[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) a[w] = left.a[turn][first + w][lane], b[w] = left.b[turn][first + w][lane];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (first + w == wave) now = before;
      before = apply(a[w], b[w], before);
    }
  }
  return now;
}

// The state before a segment: the value before the row through the segments
// before it, whose compositions stand in parts (A, then B) by segment.
template <typename T>
__device__ __forceinline__ T through_segments(const T* parts, int64_t total, int64_t q, int64_t segments, int64_t before, T state) {
  const T *a = parts + q, *b = parts + segments * total + q;
  int64_t s = 0;
  for (; s + 8 <= before; s += 8) {
    T av[8], bv[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) av[k] = a[(s + k) * total], bv[k] = b[(s + k) * total];
#pragma unroll
    for (int k = 0; k < 8; ++k) state = apply(av[k], bv[k], state);
  }
  for (; s < before; ++s) state = apply(a[s * total], b[s * total], state);
  return state;
}

// A workgroup's channels and steps.
struct Part {
  int64_t group, segment, begin, end;
};

__device__ __forceinline__ Part part_of(const Extents& e) {
  // Consecutive workgroups start on different dies; consecutive groups of a
  // segment, which share lines where rows are not whole lines, go to one.
  const unsigned die = blockIdx.x % kDies, least = gridDim.x / kDies, more = gridDim.x % kDies;
  const int64_t place = die * least + (die < more ? die : more) + blockIdx.x / kDies;
  const int64_t segment = place / e.groups, begin = segment * e.segment;
  return {place - segment * e.groups, segment, begin, begin + e.segment < e.time ? begin + e.segment : e.time};
}

// ---- forward ---------------------------------------------------------------------

template <typename T, int R>
struct ForwardLoads {
  T x[R], gate[R];
  unsigned resets = 0;

  // Steps past the end keep the state: their gate is +inf.
  template <bool RESETS>
  __device__ __forceinline__ void load(const T* xs, const T* gs, const uint8_t* rs, const Extents& e, int64_t t, int64_t end) {
    load_steps<T, R>(xs, e.channels, t, end, T(0), x);
    load_steps<T, R>(gs, e.gates, t, end, T(__builtin_huge_val()), gate);
    if (RESETS) resets = load_resets<R>(rs, t, end);
  }

  // x and gate become (1 - a) x and a; `run` goes on through the steps.
  template <bool RESETS>
  __device__ __forceinline__ void compose(Run<T>& run) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      T keep, take;
      hpd::gates(gate[i], keep, take);
      gate[i] = keep;
      x[i] *= take;
      const bool cut = RESETS && (resets >> i & 1);
      run.b = (cut ? T(0) : keep * run.b) + x[i];
      run.a *= keep;
    }
    run.cut = run.cut || (RESETS && resets);
  }
};

template <typename T, int R, int W, bool RESETS>
__global__ __launch_bounds__(W * 64) void forward_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                         const T* __restrict__ initial, const uint8_t* __restrict__ resets,
                                                         T* __restrict__ h, const T* __restrict__ parts, Extents e) {
  __shared__ Left<T, W> left;
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Part part = part_of(e);
  const Place at = flat_place(e, part.group, lane);
  const T* xs = x + at.row * e.time * e.channels + at.channel;
  const T* gs = gate + at.row * e.time * e.gates + at.gate;
  const uint8_t* rs = RESETS ? resets + at.row * e.time : nullptr;
  T* hs = h + at.row * e.time * e.channels + at.channel;
  const int64_t q = at.row * e.channels + at.channel;
  T state = initial ? initial[q] : T(0);
  if (parts) state = through_segments(parts, e.total, q, gridDim.x / e.groups, part.segment, state);

  constexpr int64_t stride = int64_t(W) * R;
  int64_t t = part.begin + int64_t(wave) * R;
  ForwardLoads<T, R> one, two;
  const auto steps = [&](ForwardLoads<T, R>& now, ForwardLoads<T, R>& next, int turn) {
    if (t + stride < part.end) next.template load<RESETS>(xs, gs, rs, e, t + stride, part.end);
    Run<T> run{T(1), T(0), false};
    now.template compose<RESETS>(run);
    T value = through<T, W>(run, left, turn, wave, lane, state);
    const bool whole = t + R <= part.end;
    T* out = hs + t * e.channels;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool cut = RESETS && (now.resets >> i & 1);
      now.x[i] = value = (cut ? T(0) : now.gate[i] * value) + now.x[i];
    }
    if (at.valid) {
      if (whole) {
#pragma unroll
        for (int i = 0; i < R; ++i) out[i * e.channels] = now.x[i];
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (t + i < part.end) out[i * e.channels] = now.x[i];
        }
      }
    }
    t += stride;
  };
  one.template load<RESETS>(xs, gs, rs, e, t, part.end);
  for (int64_t base = part.begin; base < part.end; base += 2 * stride) {
    steps(one, two, 0);
    if (base + stride < part.end) steps(two, one, 1);
  }
}

// ---- backward --------------------------------------------------------------------

template <typename T, int R>
struct BackwardLoads {
  T x[R], gate[R], h[R], grad[R];
  unsigned resets = 0;

  // Steps outside the segment pass the gradient on: their gate is +inf and their
  // gradient 0. h is that of the step before. STATES: with x and h.
  template <bool RESETS, bool STATES = true>
  __device__ __forceinline__ void load(const T* xs, const T* gs, const T* hs, const T* ds, const uint8_t* rs, T before,
                                       const Extents& e, int64_t t, int64_t begin) {
    load_steps<T, R>(gs, e.gates, t, e.time, T(__builtin_huge_val()), gate);
    load_steps<T, R>(ds, e.channels, t, e.time, T(0), grad);
    if constexpr (STATES) {
      load_steps<T, R>(xs, e.channels, t, e.time, T(0), x);
      load_steps<T, R>(hs, e.channels, t - 1, e.time, before, h);
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) x[i] = h[i] = T(0);
    }
    if (RESETS) resets = load_resets<R>(rs, t, e.time);
    if (t < begin) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (t + i < begin) gate[i] = T(__builtin_huge_val()), grad[i] = T(0), resets &= ~(1u << i);
      }
    }
  }

  // gate becomes a, h - x (0 - x at a reset) stands in h and 1 - a in x; `run`
  // goes on through the steps, from the last.
  template <bool RESETS>
  __device__ __forceinline__ void compose(Run<T>& run) {
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      T keep, take;
      hpd::gates(gate[i], keep, take);
      gate[i] = keep;
      const bool cut = RESETS && (resets >> i & 1);
      h[i] = (cut ? T(0) : h[i]) - x[i];
      x[i] = take;
      run.b = cut ? T(0) : keep * (grad[i] + run.b);
      run.a *= keep;
    }
    run.cut = run.cut || (RESETS && resets);
  }
};

// Lanes that share one of a wave's R x pack sums of gate gradients: a power of two.
template <int R>
struct SumLanes {
  __device__ __forceinline__ static int of(int pack) {
    int lanes = 1;
    while (lanes * 2 * R * pack <= 64) lanes *= 2;
    return lanes;
  }
};

// SHARED: gates that heads share; dgate then holds e.pieces partial sums.
template <typename T, int R, int W, bool RESETS, bool SHARED>
__global__ __launch_bounds__(W * 64) void backward_kernel(const T* __restrict__ grad, const T* __restrict__ x,
                                                          const T* __restrict__ gate, const T* __restrict__ h,
                                                          const T* __restrict__ initial, const uint8_t* __restrict__ resets,
                                                          T* __restrict__ dx, T* __restrict__ dgate, T* __restrict__ dinitial,
                                                          const T* __restrict__ parts, Extents e) {
  __shared__ Left<T, W> left;
  __shared__ T shares[SHARED ? W : 1][SHARED ? R : 1][65];  // rows of a task's lanes in banks of their own
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Part part = part_of(e);
  const Place at = SHARED ? head_place(e, part.group, lane) : flat_place(e, part.group, lane);
  const int64_t column = at.row * e.time * e.channels + at.channel;
  const int64_t gate_column = at.row * e.time * e.gates + at.gate;
  const T *xs = x + column, *hs = h + column, *ds = grad + column, *gs = gate + gate_column;
  const uint8_t* rs = RESETS ? resets + at.row * e.time : nullptr;
  const int64_t q = at.row * e.channels + at.channel;
  const T before = initial ? initial[q] : T(0);
  const int64_t segments = gridDim.x / e.groups;
  T carried = T(0);
  // Segments are kept from the last one on, in the order of this pass.
  if (parts) carried = through_segments(parts, e.total, q, segments, segments - 1 - part.segment, carried);

  // Wave 0 takes the last R steps, wave 1 those before them: t is the first
  // step of a wave's run, before the segment at its start.
  constexpr int64_t stride = int64_t(W) * R;
  int64_t t = part.end - int64_t(wave + 1) * R;
  BackwardLoads<T, R> one, two;
  const auto steps = [&](BackwardLoads<T, R>& now, BackwardLoads<T, R>& next, int turn, bool more) {
    if (more) next.template load<RESETS>(xs, gs, hs, ds, rs, before, e, t - stride, part.begin);
    Run<T> run{T(1), T(0), false};
    now.template compose<RESETS>(run);
    T value = through<T, W>(run, left, turn, wave, lane, carried);
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const bool cut = RESETS && (now.resets >> i & 1);
      const T slope = now.grad[i] + value;
      value = cut ? T(0) : now.gate[i] * slope;
      now.h[i] = slope * now.h[i] * (now.gate[i] * now.x[i]);
      now.x[i] = slope * now.x[i];
    }
    T* out = dx + column + t * e.channels;
    T* out_gate = dgate + gate_column + t * e.gates;
    if (at.valid) {
      if (t >= part.begin) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          out[i * e.channels] = now.x[i];
          if (!SHARED) out_gate[i * e.gates] = now.h[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (t + i >= part.begin) {
            out[i * e.channels] = now.x[i];
            if (!SHARED) out_gate[i * e.gates] = now.h[i];
          }
        }
      }
    }
    if constexpr (SHARED) {
      // The wave's own rows of LDS: its stores are in order before its loads.
#pragma unroll
      for (int i = 0; i < R; ++i) shares[wave][i][lane] = now.h[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const int64_t piece = part.group % e.pieces, head0 = part.group / e.pieces * e.pack;
      const int64_t rest = e.width - piece * e.piece;
      const int count = int(rest < e.piece ? rest : e.piece);
      T* sums = dgate + piece * (e.heads * e.time);
      // One sum for each step and head of the wave, by neighbouring lanes.
      const int lanes = SumLanes<R>::of(e.pack), sub = lane % lanes;
      for (int first = 0; first < R * e.pack; first += 64 / lanes) {
        const int task = first + lane / lanes, i = task / e.pack, slot = task - i * e.pack;
        T sum = T(0);
        if (i < R) {
          for (int k = sub; k < count; k += lanes) sum += shares[wave][i][slot * e.piece + k];
        }
        for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const int64_t head = head0 + slot;
        if (sub != 0 || i >= R || head >= e.heads || t + i < part.begin) continue;
        const int64_t row = head / e.gates;
        sums[(row * e.time + t + i) * e.gates + (head - row * e.gates)] = sum;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    t -= stride;
  };
  one.template load<RESETS>(xs, gs, hs, ds, rs, before, e, t, part.begin);
  for (int64_t base = part.begin; base < part.end; base += 2 * stride) {
    const bool second = base + stride < part.end;
    steps(one, two, 0, second);
    if (second) steps(two, one, 1, base + 2 * stride < part.end);
  }
  if (dinitial && part.segment == 0 && wave == 0 && at.valid) dinitial[q] = carried;
}

// ---- segments --------------------------------------------------------------------

// The composition of every segment but the last one in the pass's order, per
// channel. A wave composes one W-th of a segment.
template <typename T, int R, int W, bool RESETS, bool BACKWARD>
__global__ __launch_bounds__(W * 64) void segments_kernel(const T* __restrict__ values, const T* __restrict__ gate,
                                                          const uint8_t* __restrict__ resets, T* __restrict__ parts,
                                                          Extents e) {
  __shared__ T left_a[W][64], left_b[W][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Part part = part_of(e);
  const int64_t place = part.segment, composed = gridDim.x / e.groups;  // one less than segments
  if (BACKWARD) {
    part.begin = (composed - place) * e.segment;
    part.end = part.begin + e.segment < e.time ? part.begin + e.segment : e.time;
  }
  const Place at = flat_place(e, part.group, lane);
  const T* vs = values + at.row * e.time * e.channels + at.channel;
  const T* gs = gate + at.row * e.time * e.gates + at.gate;
  const uint8_t* rs = RESETS ? resets + at.row * e.time : nullptr;
  const int64_t share = (e.segment + W * R - 1) / (W * R) * R;
  Run<T> run{T(1), T(0), false};
  if (!BACKWARD) {
    const int64_t begin = part.begin + wave * share, end = begin + share < part.end ? begin + share : part.end;
    ForwardLoads<T, R> one, two;
    one.template load<RESETS>(vs, gs, rs, e, begin, end);
    for (int64_t t = begin; t < end; t += 2 * R) {
      two.template load<RESETS>(vs, gs, rs, e, t + R, end);
      one.template compose<RESETS>(run);
      one.template load<RESETS>(vs, gs, rs, e, t + 2 * R, end);
      two.template compose<RESETS>(run);
    }
  } else {
    const int64_t end = part.end - wave * share, begin = end - share > part.begin ? end - share : part.begin;
    BackwardLoads<T, R> one, two;
    const auto load = [&](BackwardLoads<T, R>& to, int64_t t) {
      to.template load<RESETS, false>(nullptr, gs, nullptr, vs, rs, T(0), e, t, begin);
    };
    load(one, end - R);
    for (int64_t t = end - R; t + R > begin; t -= 2 * R) {
      load(two, t - R);
      one.template compose<RESETS>(run);
      load(one, t - 2 * R);
      two.template compose<RESETS>(run);
    }
  }
  left_a[wave][lane] = run.cut ? T(-1) : run.a;
  left_b[wave][lane] = run.b;
  __syncthreads();
  if (wave != 0 || !at.valid) return;
  Run<T> all{T(1), T(0), false};
  for (int w = 0; w < W; ++w) {
    const T a = left_a[w][lane];
    all.b = apply(a, left_b[w][lane], all.b);
    all.cut = all.cut || a < T(0);
    all.a *= a;
  }
  const int64_t q = at.row * e.channels + at.channel, segments = composed + 1;
  parts[place * e.total + q] = all.cut ? T(-1) : all.a;
  parts[(segments + place) * e.total + q] = all.b;
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

constexpr int kWaves = 16, kSegmentWaves = 8;

// Cuts time where groups are too few to fill the chip; returns the number of
// segments.
int64_t plan_segments(const hp_ctx* ctx, Extents& e, int steps) {
  const int64_t least = int64_t(kWaves) * steps;  // of a segment
  int64_t segments = 1;
  if (e.groups * 2 <= ctx->compute_units) segments = std::min(ctx->compute_units / e.groups, e.time / least);
  e.segment = segments > 1 ? hp::ceil_div(hp::ceil_div(e.time, segments), least) * least : e.time;
  return hp::ceil_div(e.time, e.segment);
}

// Calls f with the waves of a workgroup and the steps of a run.
template <int R, typename F>
void with_shape(int64_t time, F&& f) {
  using Int = std::integral_constant<int, R>;
  if (time == 1) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  else if (time <= R) f(std::integral_constant<int, 1>{}, Int{});
  else if (time <= 4 * R) f(std::integral_constant<int, 4>{}, Int{});
  else f(std::integral_constant<int, kWaves>{}, Int{});
}

// The compositions of the segments, in scratch memory; null for one segment.
template <typename T, int R, bool BACKWARD>
T* compose_segments(hp_ctx* ctx, const T* values, const T* gate, const uint8_t* resets, Extents e, int64_t segments) {
  if (segments == 1) return nullptr;
  e.groups = hp::ceil_div(e.total, 64);
  T* parts = static_cast<T*>(hp::scratch_alloc(ctx, size_t(2 * segments) * size_t(e.total) * sizeof(T)));
  constexpr int W = kSegmentWaves;
  const unsigned grid = checked_grid(e.groups * (segments - 1), 64 * W);
  const auto kernel = resets ? segments_kernel<T, R, W, true, BACKWARD> : segments_kernel<T, R, W, false, BACKWARD>;
  kernel<<<grid, 64 * W, 0, ctx->stream>>>(values, gate, resets, parts, e);
  return parts;
}

// Returns a call's scratch memory, then reports a failed launch.
void finish(hp_ctx* ctx, const char* name, void* one, void* two) {
  const hipError_t status = hipGetLastError();
  if (one) hp::scratch_free(ctx, one);
  if (two) hp::scratch_free(ctx, two);
  hp::check_hip(status, name);
}

template <typename T>
void forward(hp_ctx* ctx, const T* x, const T* gate, const T* initial, const uint8_t* resets, T* h, Extents e) {
  constexpr int R = Steps<T>::forward;
  e.groups = hp::ceil_div(e.total, 64);
  const int64_t segments = plan_segments(ctx, e, R);
  T* parts = nullptr;
  with_shape<R>(e.time, [&](auto waves, auto steps) {
    constexpr int W = waves, S = steps;
    const unsigned grid = checked_grid(e.groups * segments, 64 * W);
    parts = compose_segments<T, R, false>(ctx, x, gate, resets, e, segments);
    const auto kernel = resets ? forward_kernel<T, S, W, true> : forward_kernel<T, S, W, false>;
    kernel<<<grid, 64 * W, 0, ctx->stream>>>(x, gate, initial, resets, h, parts, e);
  });
  finish(ctx, "launch of the recurrence", parts, nullptr);
}

template <typename T>
void backward(hp_ctx* ctx, const T* grad, const T* x, const T* gate, const T* h, const T* initial,
              const uint8_t* resets, T* dx, T* dgate, T* dinitial, Extents e) {
  constexpr int R = Steps<T>::backward;
  const bool shared = e.width > 1;
  e.groups = shared ? hp::ceil_div(e.heads, e.pack) * e.pieces : hp::ceil_div(e.total, 64);
  const int64_t segments = plan_segments(ctx, e, R);
  const int64_t count = e.heads * e.time;
  T *parts = nullptr, *sums = dgate;
  with_shape<R>(e.time, [&](auto waves, auto steps) {
    constexpr int W = waves, S = steps;
    const unsigned grid = checked_grid(e.groups * segments, 64 * W);
    if (e.pieces > 1) sums = static_cast<T*>(hp::scratch_alloc(ctx, size_t(e.pieces) * size_t(count) * sizeof(T)));
    parts = compose_segments<T, R, true>(ctx, grad, gate, resets, e, segments);
    const auto kernel = shared ? (resets ? backward_kernel<T, S, W, true, true> : backward_kernel<T, S, W, false, true>)
                               : (resets ? backward_kernel<T, S, W, true, false> : backward_kernel<T, S, W, false, false>);
    kernel<<<grid, 64 * W, 0, ctx->stream>>>(grad, x, gate, h, initial, resets, dx, sums, dinitial, parts, e);
  });
  if (e.pieces > 1) {
    const int64_t blocks = std::min<int64_t>(hp::ceil_div(count, 256), 4096);
    add_parts_kernel<T><<<unsigned(blocks), 256, 0, ctx->stream>>>(sums, dgate, count, e.pieces);
  }
  finish(ctx, "launch of the recurrence's gradient", parts, e.pieces > 1 ? sums : nullptr);
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
