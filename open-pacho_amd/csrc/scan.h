// The selective scan: what its forward and backward kernels share.
//
//   dt = softplus(delta + bias),  r_n = exp(a_log_n)
//   h_t,n = exp(-dt r_n) h_{t-1},n + dt x_t b_t,n,  y_t = (sum_n c_t,n h_t,n + skip x_t) silu(gate_t)
//
// A lane owns a channel, a wave S (2, or 4 of many) of its states, a workgroup all states of up to 64
// channels that share b and c. So b and c are the same in a whole wave: a register holds
// those of four steps in the lanes of each row of 16, and an instruction that multiplies by
// one of them takes it from its lane on the way (a row broadcast). Bound: vector issue. An
// exponential, two products and two fused multiply-adds make a state's step, 10.4 instructions with its
// share of the rest: 8 x 2048 x 2048 float32 with 16 states takes 230 us, of which 159 are issue, and whose bytes
// would take 89. (Scalar loads of b and c in each step, whose waits no other work covers, took 1458.) Two states a wave leave enough
// waves; from 17 states on (33 forward in 16 waves) four save the steps' common work. Only the sums over states meet in LDS, once for a tile of
// steps: each wave has some of the tile's steps as its own, whose dt and dt x it leaves for
// all waves before they walk the tile, and whose sums it adds up afterwards. Steps of a
// tile behind the row's end have dt, x, b and c of zero and change nothing.
//
// Where a call has few channels the steps of a row are cut into parts with workgroups of
// their own. A part from zero states ends in states E; from states h it ends in E + D h,
// D = exp(-r sum dt): each part needs the sum of its dt and its E from a launch before,
// which reads everything once more.
#pragma once

#include <type_traits>

#include "exponential.h"
#include "sequence.h"

namespace hpd {

// The arrays of a call; pointers that it does not have are null.
template <typename T>
struct Scan {
  const T *x, *delta, *a_log, *skip, *gate, *initial, *delta_bias;
  T *y, *last;
  Rows rows;
  // 32 bits: products of them are formed in 64.
  int batch, time, channels, groups;
  int width;    // channels of a group
  int pieces;   // of a group's channels, 64 each
  int states;   // of a channel
  int padded;   // of a step and group in b and c: states, up to whole launches
  int first;    // state of this launch, which takes S for each wave
  int starts, ends;  // the first and the last launch over the states
  int parts;    // of a row's steps
  int steps;    // of a part, a multiple of the tile
  // (parts, batch, channels): sums of dt; (parts, batch, states of a launch, channels): states that parts end in.
  T *spans, *ended;
  // Backward, (tiles, batch, states of a launch, channels): states before each tile, from the
  // part's zero states where there are several; (tiles, batch, channels): sums of dt from the
  // part's start; (parts, batch, states of a launch, channels): what a part passes back.
  T *before, *since, *passed;
  const T *grad, *grad_state;
};

template <typename T, int S>
struct Several {
  typedef T type __attribute__((ext_vector_type(S), aligned(sizeof(T))));
};

// exp(dt rate) of rates that are -r, for floats -r log2 e: the rounding of the product is off
// by 2^-24 of an exponent whose power is at most 0.37 of its inverse, so by half a unit of 1.
__device__ __forceinline__ float decay(float dt, float rate) { return __builtin_amdgcn_exp2f(dt * rate); }
__device__ __forceinline__ double decay(double dt, double rate) { return exp(dt * rate); }
// Rates end at the type's largest number: in steps that have a dt of 0 to change nothing an infinite one
// would make NaN, as it would of a decay of 0 in the gradients. A NaN stays one.
__device__ __forceinline__ float bounded(float rate) { return rate > 0x1.fffffep+127f ? 0x1.fffffep+127f : rate; }
__device__ __forceinline__ double bounded(double rate) { return rate > 0x1.fffffffffffffp+1023 ? 0x1.fffffffffffffp+1023 : rate; }
__device__ __forceinline__ float rate_of(float a_log) { return -bounded(expf(a_log) * 0x1.715476p+0f); }
__device__ __forceinline__ double rate_of(double a_log) { return -bounded(exp(a_log)); }
// What a state is behind steps whose dt add up to `span` (cut_span(): a reset is among them) and which end in
// `end` from nothing. An infinite one passes them also where the product of their decays is 0 in the type, though
// none of them is.
template <typename T>
__device__ __forceinline__ T passed(T span, T rate, T state, T end) {
  T kept = decay(span, rate);
  kept = kept == T(0) && __builtin_elementwise_abs(state) == T(__builtin_huge_val()) ? T(1) : kept;
  T behind = __builtin_elementwise_fma(kept, state, end);
  // Formed by all lanes, without a branch: where registers are short the compiler has put a copy of another value
  // behind such a branch, before the lanes that skipped it are back (tests/test_build_exec.py looks for that).
  asm("" : "+v"(behind));
  return span < T(0) ? end : behind;
}

// What a workgroup and its lanes work on.
template <typename T, int NW, int S>
struct Place {
  int lane, wave;
  int row, group, piece, part;
  int first, end, length;  // steps [first, end) of a row of `length`
  int slot, state;         // the wave's first state, within the launch and the channel
  unsigned channel;
  bool valid;

  __device__ __forceinline__ explicit Place(const Scan<T>& c) {
    lane = threadIdx.x & 63;
    wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int block = int(by_die());
    part = block % c.parts, block /= c.parts;
    piece = block % c.pieces, block /= c.pieces;
    group = block % c.groups;
    row = block / c.groups;
    const int within = piece * 64 + lane;
    valid = within < c.width;
    channel = unsigned(group * c.width + (valid ? within : c.width - 1));  // lanes behind it load what the last one does
    length = int(c.rows.end(row));
    first = part * c.steps;
    end = length - first < c.steps ? length : first + c.steps;
    slot = wave * S;
    state = c.first + slot;
  }
  // Of x's shape: a scalar address of step t and this lane's places in steps after it.
  template <typename P>
  __device__ __forceinline__ P* line(const Scan<T>& c, P* array, int t) const {
    return array + (int64_t(row) * c.time + t) * c.channels;
  }
  __device__ __forceinline__ unsigned place(const Scan<T>& c, int i) const { return unsigned(i * c.channels) + channel; }
  // Of (..., batch, states of a launch, channels): a scalar address of the wave's state s.
  template <typename P>
  __device__ __forceinline__ P* state_line(const Scan<T>& c, P* array, int lead, int s) const {
    return array + ((int64_t(lead) * c.batch + row) * (NW * S) + slot + s) * c.channels;
  }
  // Of (..., batch, channels).
  template <typename P>
  __device__ __forceinline__ P* row_line(const Scan<T>& c, P* array, int lead) const {
    return array + (int64_t(lead) * c.batch + row) * c.channels;
  }
  // Values of the wave's states in an array (batch, channels, states), zero for those that pad.
  __device__ __forceinline__ void read(const Scan<T>& c, const T* array, int lead, T (&to)[S]) const {
    const T* from = array + (int64_t(lead) * c.channels + channel) * c.states + state;
    if (state + S <= c.states) {
      const auto v = *reinterpret_cast<const typename Several<T, S>::type*>(from);
#pragma unroll
      for (int s = 0; s < S; ++s) to[s] = v[s];
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) to[s] = state + s < c.states ? from[s] : T(0);
    }
  }
  __device__ __forceinline__ void write(const Scan<T>& c, T* array, int lead, const T (&from)[S]) const {
    if (!valid) return;
    T* to = array + (int64_t(lead) * c.channels + channel) * c.states + state;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (state + s < c.states) to[s] = from[s];
    }
  }
  // The states before the part, from its predecessors' sums and ends.
  __device__ __forceinline__ void arrive(const Scan<T>& c, const T (&rate)[S], T (&h)[S]) const {
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = T(0);
    if (c.initial) read(c, c.initial, row, h);
    for (int p = 0; p < part; ++p) {
      const T span = row_line(c, c.spans, p)[channel];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const T end = state_line(c, c.ended, p, s)[channel];
        h[s] = passed(span, rate[s], h[s], end);
      }
    }
  }
};

// f(std::integral_constant<int, i>) for i from 0 to N - 1.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void for_each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each<N, I + 1>(f);
  }
}

// The value that lane I of each row of 16 lanes has.
template <int I>
__device__ __forceinline__ float of_row(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + I, 0xF, 0xF, true));
}
template <int I>
__device__ __forceinline__ double of_row(double v) {
  struct Words {
    int low, high;
  } w = __builtin_bit_cast(Words, v);
  w.low = __builtin_amdgcn_update_dpp(0, w.low, 0x150 + I, 0xF, 0xF, true);
  w.high = __builtin_amdgcn_update_dpp(0, w.high, 0x150 + I, 0xF, 0xF, true);
  return __builtin_bit_cast(double, w);
}

// b or c of the wave's states in the L steps of a tile: 16 / S steps a register.
template <typename T, int L, int S>
struct Projections {
  static constexpr int kSteps = 16 / S;
  T v[L / kSteps];

  // Of the tile at t < end; those of steps behind the end are what the last one's are, until keep() clears them.
  template <int NW>
  __device__ __forceinline__ void load(const Scan<T>& c, const Place<T, NW, S>& at, const T* array, int t) {
    const T* from = array + ((int64_t(at.row) * c.time + t) * c.groups + at.group) * c.padded + at.state;
    const unsigned stride = unsigned(c.groups * c.padded), last = unsigned(at.end - 1 - t);
#pragma unroll
    for (int q = 0; q < L / kSteps; ++q) {
      const unsigned i = q * kSteps + (at.lane & 15) / S;
      v[q] = from[(i < last ? i : last) * stride + at.lane % S];
    }
  }
  __device__ __forceinline__ void keep(int lane, int count) {
#pragma unroll
    for (int q = 0; q < L / kSteps; ++q) v[q] = q * kSteps + (lane & 15) / S < count ? v[q] : T(0);
  }
  // What was taken from lanes before is taken again after this, in place of staying in registers.
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int q = 0; q < L / kSteps; ++q) asm("" : "+v"(v[q]));
  }
  // Of step I and state J.
  template <int I, int J>
  __device__ __forceinline__ T get() const {
    return of_row<I % kSteps * S + J>(v[I / kSteps]);
  }
};

// The sum of dt of a part in which a reset cuts off what came before: below zero.
template <typename T>
__device__ __forceinline__ T cut_span() {
  return T(-1);
}

}  // namespace hpd

namespace hp {

// Waves of a launch with `each` states a wave: 2, 4, ... up to `most`.
inline int scan_waves(int64_t states, int each, int most) {
  int waves = 2;
  while (waves < most && int64_t(waves) * each < states) waves *= 2;
  return waves;
}

void scan_check(int dtype, int index_dtype, int64_t batch, int64_t time, int64_t channels, int64_t groups, int64_t states);
// b or c (steps, states) with zeros up to `padded` states, or as they are where there are so many.
template <typename T>
const T* scan_padded(hp_ctx* ctx, Scratch& scratch, const T* array, int64_t steps, int64_t states, int64_t padded);
template <typename T>
void scan_fill(hp_ctx* ctx, T* to, const T* from, int64_t n);

// Parts of rows: one, or as many as make enough workgroups. 128 workgroups in four parts each take 165 us
// forward and 455 backward where whole rows take 230 and 732 (4 x 2048 x 2048 float32, 16 states); 256 in
// two parts lose more in the launch before than they gain (380 against 250, and 1371 against 1188). Whole rows of 160,
// 192 and 224 workgroups take 228 and 734-739, in two parts 308-311 and 840-851, in three 277-279 and
// 861-869 of the last two; three of 160, which fill the chip twice as 128 in four do, would take 217 and 589.
template <typename T>
void scan_plan(hpd::Scan<T>& c, int tile) {
  const int64_t blocks = int64_t(c.batch) * c.groups * c.pieces, tiles = ceil_div(c.time, tile);
  int64_t parts = 1;
  if (blocks <= 128) parts = std::min<int64_t>(std::min<int64_t>(ceil_div(512, blocks), 64), std::max<int64_t>(1, tiles / 4));
  c.steps = int(ceil_div(tiles, parts)) * tile;
  c.parts = int(ceil_div(c.time, c.steps));
  require(blocks * c.parts <= kMaxThreads / 1024, "too many channels for one launch");
}

// Sizes that fit what the kernels form in 32 bits.
template <typename T>
void scan_sizes(hpd::Scan<T>& c, int64_t batch, int64_t time, int64_t channels, int64_t groups, int64_t states, int width) {
  const int64_t padded = ceil_div(states, width) * width;
  require(batch <= INT32_MAX && time <= INT32_MAX - 128 && channels <= INT32_MAX / 32 && groups * padded <= INT32_MAX / 32, "extents out of range");
  c.batch = int(batch), c.time = int(time), c.channels = int(channels), c.groups = int(groups), c.states = int(states);
  c.width = c.channels / c.groups, c.pieces = int(ceil_div(c.width, 64)), c.padded = int(padded);
}

}  // namespace hp
