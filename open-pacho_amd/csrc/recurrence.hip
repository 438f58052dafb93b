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
// states: one pass over the data.
//
// Longer rows are cut into tiles of W x R steps with a workgroup each (the chained
// kernels), still in one pass. A tile publishes its composition as soon as it has
// it. Tiles count in blocks of `span`: the state before a tile is the one before its
// block, which the last tile of the block before publishes, through the compositions
// of the block's earlier tiles, always in the same order, so that results repeat bit
// for bit. Workgroups take tiles in time order from queues, so a tile only ever
// waits for tiles whose workgroups have started, and those for earlier ones: every
// wait ends. A published word is valid by itself, without fences: memory is all
// ones before, which no published value is. One workgroup that walks all tiles of
// its channels with the next tile's loads in flight took 163 us forward and 327
// backward for 8 x 4096 x 2048 float32 where chained tiles took 150 and 294: its
// waves wait for each other every tile. For 1 x 65536 x 1024, segments of time in two
// passes took 278 and 448 us, chained tiles 174 and 331. Past the caches, as they are
// now, tiles take 141 and 275 us, 5.7 and 5.9 TB/s, and 160 and 306 (forward just
// this size goes through them, 147, for its reader's sake).
//
// A head that has whole waves computes the sigmoid of a step once in the wave; its
// gate's gradient is summed over the lanes through LDS. Shared gates are furthest from
// the bytes' time: 65536 x 1024 in 8 heads takes 243 us backward where they take 177,
// 4.4 TB/s, and 65536 x 1000 308 of 173. The sums over lanes make a quarter more vector
// instructions than gates of their own have (85.7 million against 68.6, 57% of the
// SIMDs' cycles against 42%) and twice the scalar ones, and with 16 groups a wave waits
// 58% of its time (53%); which of these bounds it has not been separated. Rows that are
// no whole lines add the rest: in waves of 63 and 62 channels dies read 1.29 times the
// arrays, with 1024 channels 1.04, as each die has a head, whose lines the next one
// shares at both ends in every step. Accesses past the caches make that worse (360 us),
// and tiles of other dies' time would wait for workgroups that need not have started.
//
// Runs of 16 and 8 steps (forward, backward; half as many float64) fill 78 and 96
// registers, so that three and two workgroups share a compute unit. Half as many
// steps take 2 to 25% longer, twice as many backward 4 to 8%, four waves 3 to 15%.
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
constexpr double kLastCache = 1 << 28;  // bytes of the cache that they share

struct Extents {
  int64_t time;      // steps of a row
  int64_t total;     // rows x channels
  int64_t channels;  // of a step
  int64_t gates;     // of a step
  int64_t width;     // channels that share a gate: channels / gates
  int64_t groups;    // of 64 lanes
  int64_t tiles;     // of a group (chained kernels)
  int span;          // tiles of a block
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
  const int64_t head = valid ? first + slot : first;
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

// An infinite state passes steps whose gates' product is too small for the type, and is
// NaN past a gate of 0. Runs and tiles tell the two apart: a product that has become 0 of
// gates above 0 is kept as -0. apply() makes NaN of both; where a NaN turns up the values
// are formed again by apply_all(). (8 x 4096 x 2048 float32: forward, past the caches,
// 139.1 us without any of this and 139.4, backward 273 and 275-278; 1 x 65536 x 1024 in 8 heads 120.6 and 121.9,
// 243.6 and 244.4. Products and states told apart in every step of the way: 143 and 292,
// 129 and 263.)
template <typename T>
__device__ __forceinline__ T apply_all(T a, T b, T h) {
  const bool passes = a == T(0) && __builtin_signbit(a) && __builtin_elementwise_abs(h) == T(__builtin_huge_val());
  return passes ? h + b : apply(a, b, h);
}

// R values of a column from its step t on; steps outside [0, end) hold `outside`.
// STREAM: past the caches.
template <bool STREAM, typename T, int R>
__device__ __forceinline__ void load_steps(const T* column, int64_t stride, int64_t t, int64_t end, T outside, T (&v)[R]) {
  if (t >= 0 && t + R <= end) {
    const T* p = column + t * stride;
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = STREAM ? __builtin_nontemporal_load(p + i * stride) : p[i * stride];
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
  const T start = before;
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
  if (__any(now != now || before != before)) {
    before = start;
    for (int w = 0; w < W; ++w) {
      if (w == wave) now = before;
      before = apply_all(left.a[turn][w][lane], left.b[turn][w][lane], before);
    }
  }
  return now;
}

// Workgroup b as number b' such that consecutive b' run on one die: workgroups
// start on the dies in turn, and neighbouring groups share lines where rows are
// not whole lines.
__device__ __forceinline__ int64_t by_die() {
  const unsigned die = blockIdx.x % kDies, least = gridDim.x / kDies, more = gridDim.x % kDies;
  return int64_t(die) * least + (die < more ? die : more) + blockIdx.x / kDies;
}

// ---- chained tiles -----------------------------------------------------------------

template <typename T>
struct Word;
template <>
struct Word<float> {
  using type = uint32_t;
};
template <>
struct Word<double> {
  using type = uint64_t;
};

constexpr int kTicketWords = 32;  // of 4 bytes, apart for each die's queue

// Memory of a chained launch, all ones at its start: a queue for each die, the
// compositions of the tiles (A of 64 lanes, then B), and the states after blocks.
template <typename T>
struct Chain {
  unsigned* tickets;
  typename Word<T>::type *runs, *states;

  __device__ __forceinline__ static void publish(typename Word<T>::type* at, T value) {
    typename Word<T>::type bits;
    __builtin_memcpy(&bits, &value, sizeof(T));
    if (bits == ~typename Word<T>::type(0)) bits = ~typename Word<T>::type(0) - 1;  // a NaN as well
    __hip_atomic_store(at, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ __forceinline__ static typename Word<T>::type peek(const typename Word<T>::type* at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // The value at `at`, first seen as `bits`, once it is there.
  __device__ __forceinline__ static T await(const typename Word<T>::type* at, typename Word<T>::type bits) {
    while (bits == ~typename Word<T>::type(0)) {
      __builtin_amdgcn_s_sleep(1);
      bits = peek(at);
    }
    T value;
    __builtin_memcpy(&value, &bits, sizeof(T));
    return value;
  }
};

// Groups of a die's queue: [first(die), first(die + 1)).
__device__ __forceinline__ int64_t first_group(const Extents& e, int die) { return die * e.groups / kDies; }

struct Tile {
  int64_t group, number;
};

// The next tile of this die's queue, or of another's when it is empty. There are as
// many workgroups as tiles, so each finds one (a number below 0 would be none).
__device__ __forceinline__ Tile take_tile(unsigned* tickets, const Extents& e) {
  __shared__ int64_t found[2];
  if (threadIdx.x == 0) {
    found[1] = -1;
    for (unsigned turn = 0; turn < kDies; ++turn) {
      const int die = (blockIdx.x + turn) % kDies;
      const int64_t first = first_group(e, die), groups = first_group(e, die + 1) - first;
      if (groups == 0) continue;
      // All ones counts as -1.
      const unsigned ticket = 1 + __hip_atomic_fetch_add(tickets + die * kTicketWords, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (ticket >= uint64_t(groups) * uint64_t(e.tiles)) continue;
      const int64_t number = ticket / groups;
      found[0] = first + (ticket - number * groups);
      found[1] = number;
      break;
    }
  }
  __syncthreads();
  return {found[0], found[1]};
}

// a composed with what came before it: `before` where a < 0 is dropped.
template <typename T>
__device__ __forceinline__ void then(T& all_a, T& all_b, T a, T b) {
  all_b = apply(a, b, all_b);
  all_a = a < T(0) || all_a < T(0) ? T(-1) : all_a * a;
}

// The same as apply_all has it.
template <typename T>
__device__ __forceinline__ void then_all(T& all_a, T& all_b, T a, T b) {
  const auto shut = [](T v) { return v == T(0) && !__builtin_signbit(v); };
  const bool is_shut = shut(all_a) || shut(a);
  all_b = apply_all(a, b, all_b);
  all_a = a < T(0) || all_a < T(0) ? T(-1) : all_a * a;
  if (all_a == T(0)) all_a = is_shut ? T(0) : -T(0);
}

template <typename T, int W>
struct ChainLeft {
  T a[W][64], b[W][64], earlier_a[W][64], earlier_b[W][64], state[64];
};

// The value before this wave's run; `after` becomes the value after the tile.
// `first` is the value before the row.
template <typename T, int W>
__device__ __forceinline__ T through_chain(const Run<T>& run, ChainLeft<T, W>& left, const Chain<T>& chain, const Extents& e,
                                           const Tile& tile, int wave, int lane, T first, T& after) {
  using C = Chain<T>;
  using Bits = typename Word<T>::type;
  const int64_t block = tile.number / e.span;
  const int inner = int(tile.number - block * e.span);
  const bool last = inner == e.span - 1;
  left.a[wave][lane] = run.cut ? T(-1) : run.a;
  left.b[wave][lane] = run.b;
  __syncthreads();
  T all_a = T(1), all_b = T(0), own_a = T(1), own_b = T(0);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == wave) own_a = all_a, own_b = all_b;
    then(all_a, all_b, left.a[w][lane], left.b[w][lane]);
  }
  Bits* const runs = chain.runs + (tile.number * e.groups + tile.group) * 128 + lane;
  if (wave == 0 && !last) {
    T a = all_a, b = all_b;
    if (__any(a == T(0) || b != b)) {
      a = T(1), b = T(0);
      for (int w = 0; w < W; ++w) then_all(a, b, left.a[w][lane], left.b[w][lane]);
    }
    C::publish(runs, a), C::publish(runs + 64, b);
  }
  // Each wave takes a run of the block's earlier tiles.
  const int each = (inner + W - 1) / W, low = wave * each, high = low + each < inner ? low + each : inner;
  T win_a = T(1), win_b = T(0);
  for (int p = low; p < high; p += 4) {
    Bits a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const Bits* at = runs - (inner - (p + k < high ? p + k : high - 1)) * e.groups * 128;
      a[k] = C::peek(at), b[k] = C::peek(at + 64);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (p + k >= high) break;
      const Bits* at = runs - (inner - (p + k)) * e.groups * 128;
      const T va = C::await(at, a[k]);
      then(win_a, win_b, va, C::await(at + 64, b[k]));
    }
  }
  left.earlier_a[wave][lane] = win_a;
  left.earlier_b[wave][lane] = win_b;
  Bits* const states = chain.states + (block * e.groups + tile.group) * 64 + lane;
  if (wave == W - 1) {
    const Bits* at = states - e.groups * 64;
    left.state[lane] = block == 0 ? first : C::await(at, C::peek(at));
  }
  __syncthreads();
  T state = left.state[lane];
#pragma unroll
  for (int w = 0; w < W; ++w) state = apply(left.earlier_a[w][lane], left.earlier_b[w][lane], state);
  after = apply(all_a, all_b, state);
  T value = apply(own_a, own_b, state);
  if (__any(value != value || after != after)) {
    state = left.state[lane];
    for (int p = 0; p < inner; ++p) {
      const Bits* at = runs - (inner - p) * e.groups * 128;
      const T a = C::await(at, C::peek(at));
      state = apply_all(a, C::await(at + 64, C::peek(at + 64)), state);
    }
    after = state;
    for (int w = 0; w < W; ++w) {
      if (w == wave) value = after;
      after = apply_all(left.a[w][lane], left.b[w][lane], after);
    }
  }
  if (wave == 0 && last) C::publish(states, after);
  return value;
}

// ---- forward ---------------------------------------------------------------------

// Where a lane's gates come from: kOwn: each channel has its own; kShared: heads
// share them; kWave: one head has the whole wave.
enum Gating { kOwn, kShared, kWave };

// The gates of a run: raw ones, +inf (a step that keeps the state) outside [0, end),
// which open() turns into sigmoids.
template <typename T, int R, Gating G>
struct Gates {
  T v[R];

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* gs, const Extents& e, int64_t t, int64_t end, int) {
    load_steps<STREAM && G == kOwn>(gs, e.gates, t, end, T(__builtin_huge_val()), v);
  }
  __device__ __forceinline__ void open() {}
  // a_i, once; then keep(i) has it and the result is 1 - a_i.
  __device__ __forceinline__ T take(int i) {
    T keep, take;
    hpd::gates(v[i], keep, take);
    v[i] = keep;
    return take;
  }
  __device__ __forceinline__ T keep(int i) const { return v[i]; }
};

// Lane i has step i's: one load and one sigmoid a lane in place of R.
template <typename T, int R>
struct Gates<T, R, kWave> {
  T own, taken;

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* gs, const Extents& e, int64_t t, int64_t end, int lane) {
    own = T(__builtin_huge_val());
    if (lane < R && t + lane >= 0 && t + lane < end) own = gs[(t + lane) * e.gates];
  }
  __device__ __forceinline__ void open() {
    const T raw = own;
    hpd::gates(raw, own, taken);
  }
  __device__ __forceinline__ T take(int i) const { return of_lane(taken, i); }
  __device__ __forceinline__ T keep(int i) const { return of_lane(own, i); }

 private:
  __device__ __forceinline__ static float of_lane(float v, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
  }
  __device__ __forceinline__ static double of_lane(double v, int i) {
    const int64_t bits = __builtin_bit_cast(int64_t, v);
    const uint32_t low = uint32_t(__builtin_amdgcn_readlane(int(bits), i)), high = uint32_t(__builtin_amdgcn_readlane(int(bits >> 32), i));
    return __builtin_bit_cast(double, uint64_t(high) << 32 | low);
  }
};

template <typename T, int R, Gating G>
struct ForwardLoads {
  T x[R];
  Gates<T, R, G> gates;
  unsigned resets = 0;

  template <bool RESETS>
  __device__ __forceinline__ void load(const T* xs, const T* gs, const uint8_t* rs, const Extents& e, int64_t t, int lane) {
    load_steps<true>(xs, e.channels, t, e.time, T(0), x);
    gates.template load<true>(gs, e, t, e.time, lane);
    if (RESETS) resets = load_resets<R>(rs, t, e.time);
  }

  // x becomes (1 - a) x; `run` goes on through the steps.
  template <bool RESETS>
  __device__ __forceinline__ void compose(Run<T>& run) {
    gates.open();
    T least = T(1);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      x[i] *= gates.take(i);
      const bool cut = RESETS && (resets >> i & 1);
      run.b = (cut ? T(0) : gates.keep(i) * run.b) + x[i];
      run.a *= gates.keep(i);
      least = __builtin_elementwise_min(least, gates.keep(i));
    }
    run.cut = run.cut || (RESETS && resets);
    if (run.a == T(0) && least > T(0)) run.a = -T(0);
  }
};

// The arrays of a call.
template <typename T>
struct Forward {
  const T *x, *gate, *initial;
  const uint8_t* resets;
  T* h;
};

// A lane's columns of them. STREAM: states are stored past the caches.
template <typename T, Gating G, bool STREAM>
struct ForwardColumns {
  const T *x, *gate;
  const uint8_t* resets;
  T *h, first;
  bool valid;

  __device__ __forceinline__ ForwardColumns(const Forward<T>& f, const Extents& e, int64_t group, int lane) {
    const Place at = G == kWave ? head_place(e, group, lane) : flat_place(e, group, lane);
    const int64_t column = at.row * e.time * e.channels + at.channel;
    x = f.x + column;
    h = f.h + column;
    gate = f.gate + at.row * e.time * e.gates + at.gate;
    resets = f.resets + at.row * e.time;
    first = f.initial ? f.initial[at.row * e.channels + at.channel] : T(0);
    valid = at.valid;
  }

  // The states of composed steps from t on.
  template <int R, bool RESETS>
  __device__ __forceinline__ void finish(ForwardLoads<T, R, G>& now, const Extents& e, int64_t t, T value) const {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool cut = RESETS && (now.resets >> i & 1);
      now.x[i] = value = (cut ? T(0) : now.gates.keep(i) * value) + now.x[i];
    }
    if (!valid) return;
    T* out = h + t * e.channels;
    if (t + R <= e.time) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if constexpr (STREAM) __builtin_nontemporal_store(now.x[i], out + i * e.channels);
        else out[i * e.channels] = now.x[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (t + i < e.time) out[i * e.channels] = now.x[i];
      }
    }
  }
};

// Rows of at most W x R steps, or of two times as many where DOUBLE.
template <typename T, int R, int W, bool DOUBLE, bool RESETS, Gating G, bool STREAM>
__global__ __launch_bounds__(W * 64) void forward_kernel(Forward<T> f, Extents e) {
  __shared__ Left<T, W> left;
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ForwardColumns<T, G, STREAM> c(f, e, by_die(), lane);
  T state = c.first;
  constexpr int stride = W * R;
  ForwardLoads<T, R, G> loads[DOUBLE ? 2 : 1];
#pragma unroll
  for (int n = 0; n < (DOUBLE ? 2 : 1); ++n) {
    loads[n].template load<RESETS>(c.x, c.gate, c.resets, e, n * stride + wave * R, lane);
  }
#pragma unroll
  for (int n = 0; n < (DOUBLE ? 2 : 1); ++n) {
    Run<T> run{T(1), T(0), false};
    loads[n].template compose<RESETS>(run);
    const T value = through<T, W>(run, left, n, wave, lane, state);
    c.template finish<R, RESETS>(loads[n], e, n * stride + wave * R, value);
  }
}

template <typename T, int R, int W, bool RESETS, Gating G, bool STREAM>
__global__ __launch_bounds__(W * 64) void forward_chained_kernel(Forward<T> f, Extents e, Chain<T> chain) {
  __shared__ ChainLeft<T, W> left;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = take_tile(chain.tickets, e);
  if (tile.number < 0) return;
  const ForwardColumns<T, G, STREAM> c(f, e, tile.group, lane);
  const int64_t t = (tile.number * W + wave) * R;
  ForwardLoads<T, R, G> now;
  now.template load<RESETS>(c.x, c.gate, c.resets, e, t, lane);
  Run<T> run{T(1), T(0), false};
  now.template compose<RESETS>(run);
  T after;
  const T value = through_chain<T, W>(run, left, chain, e, tile, wave, lane, c.first, after);
  c.template finish<R, RESETS>(now, e, t, value);
}

// ---- backward --------------------------------------------------------------------

template <typename T, int R, Gating G>
struct BackwardLoads {
  T x[R], h[R], grad[R];
  Gates<T, R, G> gates;
  unsigned resets = 0;

  // Steps before the row pass the gradient on: their gate is +inf and their
  // gradient 0. h is that of the step before.
  template <bool RESETS, bool STREAM>
  __device__ __forceinline__ void load(const T* xs, const T* gs, const T* hs, const T* ds, const uint8_t* rs, T before,
                                       const Extents& e, int64_t t, int lane) {
    gates.template load<STREAM>(gs, e, t, e.time, lane);
    load_steps<STREAM>(ds, e.channels, t, e.time, T(0), grad);
    load_steps<STREAM>(xs, e.channels, t, e.time, T(0), x);
    load_steps<STREAM>(hs, e.channels, t - 1, e.time, before, h);
    if (RESETS) resets = load_resets<R>(rs, t, e.time);
  }

  // h - x (0 - x at a reset) stands in h and 1 - a in x; `run` goes on through the
  // steps, from the last.
  template <bool RESETS>
  __device__ __forceinline__ void compose(Run<T>& run) {
    gates.open();
    T least = T(1);
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const bool cut = RESETS && (resets >> i & 1);
      h[i] = (cut ? T(0) : h[i]) - x[i];
      x[i] = gates.take(i);
      run.b = cut ? T(0) : gates.keep(i) * (grad[i] + run.b);
      run.a *= gates.keep(i);
      least = __builtin_elementwise_min(least, gates.keep(i));
    }
    run.cut = run.cut || (RESETS && resets);
    if (run.a == T(0) && least > T(0)) run.a = -T(0);
  }
};

// The arrays of a call. dgate holds e.pieces partial sums where heads share gates.
template <typename T>
struct Backward {
  const T *grad, *x, *gate, *h, *initial;
  const uint8_t* resets;
  T *dx, *dgate, *dinitial;
};

template <typename T, Gating G, bool STREAM>
struct BackwardColumns {
  static constexpr bool SHARED = G != kOwn;
  const T *x, *gate, *h, *grad;
  const uint8_t* resets;
  T *dx, *dgate, *dinitial, before;
  bool valid;

  __device__ __forceinline__ BackwardColumns(const Backward<T>& f, const Extents& e, int64_t group, int lane) {
    const Place at = SHARED ? head_place(e, group, lane) : flat_place(e, group, lane);
    const int64_t column = at.row * e.time * e.channels + at.channel;
    const int64_t gate_column = at.row * e.time * e.gates + at.gate, q = at.row * e.channels + at.channel;
    x = f.x + column;
    h = f.h + column;
    grad = f.grad + column;
    dx = f.dx + column;
    gate = f.gate + gate_column;
    dgate = SHARED ? f.dgate : f.dgate + gate_column;
    resets = f.resets + at.row * e.time;
    before = f.initial ? f.initial[q] : T(0);
    dinitial = f.dinitial ? f.dinitial + q : nullptr;
    valid = at.valid;
  }

  template <bool RESETS, int R>
  __device__ __forceinline__ void load(BackwardLoads<T, R, G>& to, const Extents& e, int64_t t, int lane) const {
    to.template load<RESETS, STREAM>(x, gate, h, grad, resets, before, e, t, lane);
  }

  __device__ __forceinline__ static void store(T* to, T v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, to);
    else *to = v;
  }

  // The gradients of composed steps from t on; `shares`: LDS of this wave.
  template <int R, bool RESETS>
  __device__ __forceinline__ void finish(BackwardLoads<T, R, G>& now, const Extents& e, int64_t group, int64_t t, int lane,
                                         T (*shares)[65], T value) const {
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const bool cut = RESETS && (now.resets >> i & 1);
      const T slope = now.grad[i] + value;
      value = cut ? T(0) : now.gates.keep(i) * slope;
      now.h[i] = slope * now.h[i] * (now.gates.keep(i) * now.x[i]);
      now.x[i] = slope * now.x[i];
    }
    T* out = dx + t * e.channels;
    T* out_gate = dgate + t * e.gates;
    if (valid) {
      if (t >= 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          store(out + i * e.channels, now.x[i]);
          if (!SHARED) store(out_gate + i * e.gates, now.h[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (t + i >= 0) {
            out[i * e.channels] = now.x[i];
            if (!SHARED) out_gate[i * e.gates] = now.h[i];
          }
        }
      }
    }
    if constexpr (SHARED) add_shares<R>(now, e, group, t, lane, shares);
  }

  // One sum for each step and head of the wave, by neighbouring lanes.
  template <int R>
  __device__ __forceinline__ void add_shares(const BackwardLoads<T, R, G>& now, const Extents& e, int64_t group, int64_t t,
                                             int lane, T (*shares)[65]) const {
    // The wave's own rows of LDS: its stores are in order before its loads.
#pragma unroll
    for (int i = 0; i < R; ++i) shares[i][lane] = now.h[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int64_t piece = group % e.pieces, head0 = group / e.pieces * e.pack;
    const int64_t rest = e.width - piece * e.piece;
    const int count = int(rest < e.piece ? rest : e.piece);
    T* sums = dgate + piece * (e.heads * e.time);
    int lanes = 1;  // that share a sum: a power of two
    while (lanes * 2 * R * e.pack <= 64) lanes *= 2;
    const int sub = lane % lanes;
    for (int first = 0; first < R * e.pack; first += 64 / lanes) {
      const int task = first + lane / lanes, i = task / e.pack, slot = task - i * e.pack;
      T sum = T(0);
      if (i < R) {
        for (int k = sub; k < count; k += lanes) sum += shares[i][slot * e.piece + k];
      }
      for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
      const int64_t head = head0 + slot;
      if (sub != 0 || i >= R || head >= e.heads || t + i < 0) continue;
      const int64_t row = head / e.gates;
      sums[(row * e.time + t + i) * e.gates + (head - row * e.gates)] = sum;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
};

// Rows as in forward_kernel. Wave 0 takes the last R steps, wave 1 those before them:
// a wave's first step is below zero at the start of the row.
template <typename T, int R, int W, bool DOUBLE, bool RESETS, Gating G, bool STREAM>
__global__ __launch_bounds__(W * 64) void backward_kernel(Backward<T> f, Extents e) {
  __shared__ Left<T, W> left;
  constexpr bool SHARED = G != kOwn;
  __shared__ T shares[SHARED ? W : 1][SHARED ? R : 1][65];  // rows of a sum's lanes in banks of their own
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t group = by_die();
  const BackwardColumns<T, G, STREAM> c(f, e, group, lane);
  T carried = T(0);
  const int64_t t = e.time - int64_t(wave + 1) * R;
  BackwardLoads<T, R, G> loads[DOUBLE ? 2 : 1];
#pragma unroll
  for (int n = 0; n < (DOUBLE ? 2 : 1); ++n) c.template load<RESETS>(loads[n], e, t - n * W * R, lane);
#pragma unroll
  for (int n = 0; n < (DOUBLE ? 2 : 1); ++n) {
    Run<T> run{T(1), T(0), false};
    loads[n].template compose<RESETS>(run);
    const T value = through<T, W>(run, left, n, wave, lane, carried);
    c.template finish<R, RESETS>(loads[n], e, group, t - n * W * R, lane, shares[SHARED ? wave : 0], value);
  }
  if (c.dinitial && wave == 0 && c.valid) *c.dinitial = carried;
}

template <typename T, int R, int W, bool RESETS, Gating G, bool STREAM>
__global__ __launch_bounds__(W * 64) void backward_chained_kernel(Backward<T> f, Extents e, Chain<T> chain) {
  __shared__ ChainLeft<T, W> left;
  constexpr bool SHARED = G != kOwn;
  __shared__ T shares[SHARED ? W : 1][SHARED ? R : 1][65];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = take_tile(chain.tickets, e);
  if (tile.number < 0) return;
  const BackwardColumns<T, G, STREAM> c(f, e, tile.group, lane);
  const int64_t t = e.time - (tile.number * W + wave + 1) * R;
  BackwardLoads<T, R, G> now;
  c.template load<RESETS>(now, e, t, lane);
  Run<T> run{T(1), T(0), false};
  now.template compose<RESETS>(run);
  T after;
  const T value = through_chain<T, W>(run, left, chain, e, tile, wave, lane, T(0), after);
  c.template finish<R, RESETS>(now, e, tile.group, t, lane, shares[SHARED ? wave : 0], value);
  if (c.dinitial && tile.number == e.tiles - 1 && wave == 0 && c.valid) *c.dinitial = after;
}

__global__ __launch_bounds__(256) void ones_kernel(uint4* __restrict__ to, int64_t n) {
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    to[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
  }
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

constexpr int kWaves = 8;

// Calls f with the steps of a run, the waves of a workgroup, and whether it takes
// two runs of each.
template <int R, typename F>
void with_shape(int64_t time, F&& f) {
  const auto shape = [&](auto steps, auto waves, auto twice) { f(steps, waves, twice); };
  using Int = std::integral_constant<int, R>;
  using One = std::integral_constant<int, 1>;
  using Four = std::integral_constant<int, 4>;
  using All = std::integral_constant<int, kWaves>;
  if (time == 1) shape(One{}, One{}, std::false_type{});
  else if (time <= 4) shape(Four{}, One{}, std::false_type{});
  else if (time <= R) shape(Int{}, One{}, std::false_type{});
  else if (time <= 4 * R) shape(Int{}, Four{}, std::false_type{});
  else if (time <= kWaves * R) shape(Int{}, All{}, std::false_type{});
  else shape(Int{}, All{}, std::true_type{});
}

// Whether tiles are chained: from three on. (With one workgroup that walks two
// tiles 128 x 256 x 2048 float32 forward takes 152 us and 154 chained, with eight
// 32 x 1024 x 2048 164 and 154.)
bool plan_chain(Extents& e, int steps) {
  e.tiles = hp::ceil_div(e.time, int64_t(kWaves) * steps);
  if (e.tiles < 3) return false;
  // Few groups are long in waiting from block to block: 65536 x 1000 in 8 heads, 16
  // groups, takes 308 us backward in blocks of 64 and 321 of 16; with 256 groups,
  // 8 x 4096 x 2048, the readings of a block's tiles weigh more, 281 and 274. Between
  // them nothing was measured. The order in which a row's tiles meet, and with it the
  // rounding, so depends on the rows beside it.
  e.span = e.groups >= 32 ? 16 : 64;
  return true;
}

// Memory of a chained launch, all ones.
template <typename T>
Chain<T> make_chain(hp_ctx* ctx, hp::Scratch& scratch, const Extents& e) {
  const int64_t tickets = int64_t(kDies) * kTicketWords * 4, runs = e.tiles * e.groups * 128 * int64_t(sizeof(T));
  const int64_t states = hp::ceil_div(e.tiles, e.span) * e.groups * 64 * int64_t(sizeof(T));
  char* memory = scratch.take<char>(tickets + runs + states);
  const int64_t n = (tickets + runs + states) / 16;
  ones_kernel<<<unsigned(std::min<int64_t>(hp::ceil_div(n, 256), 2048)), 256, 0, ctx->stream>>>(reinterpret_cast<uint4*>(memory), n);
  hp::check_launch("recurrence memory");
  using Bits = typename Word<T>::type;
  return {reinterpret_cast<unsigned*>(memory), reinterpret_cast<Bits*>(memory + tickets), reinterpret_cast<Bits*>(memory + tickets + runs)};
}

template <typename T, Gating G, bool STREAM>
void forward(hp_ctx* ctx, const Forward<T>& f, Extents e) {
  constexpr int R = Steps<T>::forward;
  hp::Scratch scratch(ctx);
  e.groups = G == kWave ? e.heads * e.pieces : hp::ceil_div(e.total, 64);
  if (plan_chain(e, R)) {
    const unsigned grid = checked_grid(e.groups * e.tiles, 64 * kWaves);
    const Chain<T> chain = make_chain<T>(ctx, scratch, e);
    const auto kernel = f.resets ? forward_chained_kernel<T, R, kWaves, true, G, STREAM>
                                 : forward_chained_kernel<T, R, kWaves, false, G, STREAM>;
    kernel<<<grid, 64 * kWaves, 0, ctx->stream>>>(f, e, chain);
  } else {
    with_shape<R>(e.time, [&](auto steps, auto waves, auto twice) {
      constexpr int S = steps, W = waves;
      const unsigned grid = checked_grid(e.groups, 64 * W);
      const auto kernel = f.resets ? forward_kernel<T, S, W, twice, true, G, STREAM> : forward_kernel<T, S, W, twice, false, G, STREAM>;
      kernel<<<grid, 64 * W, 0, ctx->stream>>>(f, e);
    });
  }
  hp::check_launch("recurrence");
}

template <typename T, Gating G, bool STREAM>
void backward(hp_ctx* ctx, Backward<T> f, Extents e) {
  constexpr int R = Steps<T>::backward;
  hp::Scratch scratch(ctx);
  e.groups = G == kOwn ? hp::ceil_div(e.total, 64) : hp::ceil_div(e.heads, e.pack) * e.pieces;
  T* const dgate = f.dgate;
  const int64_t count = e.heads * e.time;
  if (e.pieces > 1) f.dgate = scratch.take<T>(e.pieces * count);
  if (plan_chain(e, R)) {
    const unsigned grid = checked_grid(e.groups * e.tiles, 64 * kWaves);
    const Chain<T> chain = make_chain<T>(ctx, scratch, e);
    const auto kernel = f.resets ? backward_chained_kernel<T, R, kWaves, true, G, STREAM>
                                 : backward_chained_kernel<T, R, kWaves, false, G, STREAM>;
    kernel<<<grid, 64 * kWaves, 0, ctx->stream>>>(f, e, chain);
  } else {
    with_shape<R>(e.time, [&](auto steps, auto waves, auto twice) {
      constexpr int S = steps, W = waves;
      const unsigned grid = checked_grid(e.groups, 64 * W);
      const auto kernel = f.resets ? backward_kernel<T, S, W, twice, true, G, STREAM> : backward_kernel<T, S, W, twice, false, G, STREAM>;
      kernel<<<grid, 64 * W, 0, ctx->stream>>>(f, e);
    });
  }
  hp::check_launch("recurrence gradient");
  if (e.pieces > 1) {
    const int64_t blocks = std::min<int64_t>(hp::ceil_div(count, 256), 4096);
    add_parts_kernel<T><<<unsigned(blocks), 256, 0, ctx->stream>>>(f.dgate, dgate, count, e.pieces);
    hp::check_launch("recurrence gate sums");
  }
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
    const auto run = [&](auto zero) {
      using T = decltype(zero);
      const Forward<T> f{static_cast<const T*>(x), static_cast<const T*>(gate), static_cast<const T*>(initial), r, static_cast<T*>(h)};
      // Heads of whole waves are laid out by waves, for one sigmoid a step (65536 x 1024
      // float32 in 8 heads: 125 us, 131 with a sigmoid a lane; 65536 x 1000 in 8 heads,
      // waves of 63: 157 and 148).
      // States are stored past the caches where steps are whole lines and all of them are
      // more than the last cache holds (16 x 4096 x 2048 float32: 264 us, 284 through it;
      // with a product of 18 columns right after, 460 and 487). Fewer are left there for
      // their reader: of 8 x 4096 x 2048, just what it holds, 141 us and 147, but with a sum
      // or a product of 512 columns right after 186 and 170, 615 and 605.
      const bool stream = channels * int64_t(sizeof(T)) % 128 == 0 && double(e.total) * double(time) * sizeof(T) > kLastCache;
      const auto launch = e.width == 1                      ? (stream ? forward<T, kOwn, true> : forward<T, kOwn, false>)
                          : e.pack == 1 && e.piece == 64    ? (stream ? forward<T, kWave, true> : forward<T, kWave, false>)
                                                            : (stream ? forward<T, kShared, true> : forward<T, kShared, false>);
      launch(ctx, f, e);
    };
    if (dtype == HP_F32) run(float(0));
    else run(double(0));
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
      const Backward<T> f{static_cast<const T*>(grad), static_cast<const T*>(x), static_cast<const T*>(gate),
                          static_cast<const T*>(h), static_cast<const T*>(initial), r, static_cast<T*>(dx),
                          static_cast<T*>(dgate), static_cast<T*>(dinitial)};
      // Past the caches where steps are whole lines and the call's arrays together are more
      // than the last one holds (float32, us: 8 x 4096 x 2048 275 against 292 through the
      // caches, 4 x 4096 x 2048 145 and 153, with sums over the gradients right after 367 and
      // 377, 196 and 196; but 8 x 512 x 2048, 192 MiB in all, 44 and 38, 66 and 57). Without
      // whole lines neighbouring groups meet in the lines that they share (2 x 8192 x 3001
      // 298 against 255).
      const double bytes = (4.0 * double(e.total) + 2.0 * double(e.heads)) * double(time) * sizeof(T);
      const bool stream = channels * int64_t(sizeof(T)) % 128 == 0 && bytes > kLastCache;
      const auto launch = e.width == 1  ? (stream ? backward<T, kOwn, true> : backward<T, kOwn, false>)
                          : e.pack == 1 ? (stream ? backward<T, kWave, true> : backward<T, kWave, false>)
                                        : (stream ? backward<T, kShared, true> : backward<T, kShared, false>);
      launch(ctx, f, e);
    };
    if (dtype == HP_F32) run(float(0));
    else run(double(0));
  });
}

}  // extern "C"
