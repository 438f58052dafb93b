// AdamW over a list of tensors, with moments in the parameters' type or in 8 bits.
//
//   m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g g
//   p' = p - (decay p + step m' / (root sqrt(v') + eps)),  step = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
//
// Bound: HBM. Four arrays are read and three written (float32: 28 bytes a
// parameter: 201 million in 948 us, 5.9 TB/s), with 8-bit moments two arrays and two
// bytes read, one array and two bytes written and 16 bytes of scales for every 256
// parameters (98 million: 1.6 GB in 264-306 us). There the vector unit comes
// next: divisions and roots as the compiler expands them took 131 instructions a
// parameter and bound the kernel at 340 us, the ones below take about 80.
//
// A launch takes up to kTensors tensors: the table of their addresses is a
// kernel argument, so that no table has to be copied to the device first. A
// workgroup works on kChunk elements of one tensor and finds it by bisection
// in the table. State and new parameters lie in chunks in the order of the
// workgroups: a chunk's number is its place there.
//
// 8 bits: blocks of 256 elements of a tensor, one wave each, share a scale, the
// largest |m| and the largest u = sqrt(v) of the block. A code is the share in
// it, rounded to the nearest (ties to even), with 4 bits below the leading one:
// 3 exponent bits and a sign for m, 4 exponent bits for u; the lowest 16 codes
// are evenly spaced down to 0. A share of 1 has an exact code, so that the
// largest element of a block keeps all its digits. u is kept rather than v, since
// a root has half the range; one above 0 never becomes 0, which would divide by
// eps alone. A block with an infinite or NaN moment becomes NaN. The update takes
// the moments before they are rounded. Products and sums of the moments are
// rounded one by one, so that codes do not depend on how a compiler fuses them.
#include "common.h"

namespace {

constexpr int kBlock = 256;              // elements that share a scale: a wave's
constexpr int kChunk = 4 * kBlock;       // elements of a workgroup
constexpr int kTensors = 96;             // of one launch

template <typename T>
struct Tensor {
  const T* param;
  const T* grad;
  int64_t size;
  int64_t chunk;  // its first
  double decay;
};

template <typename T>
struct Table {
  Tensor<T> tensor[kTensors];
  int count;
  int64_t first_chunk;  // of this launch
};

struct Scalars {
  double beta1, beta2, rest1, rest2, step, root, eps;
};

// The moments' storage: arrays of whole chunks.
template <typename T>
struct Moments {
  T *first, *second;            // 0: in the parameters' type
  uint8_t *codes1, *codes2;     // 8 bits
  float *top1, *top2;           // a scale for each block
};

template <typename T, int W>
struct Pack {
  T v[W];
};

// W values from `p`; one access if `whole`, else those below `count`. Past the
// caches, as the stores: everything is read and written once (201 million float32
// parameters 998 -> 948 us, 98 million with 8-bit states 483 -> 419).
template <typename T, int W>
__device__ __forceinline__ Pack<T, W> load_pack(const T* p, bool whole, int64_t count) {
  typedef T V __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  Pack<T, W> r;
  if (whole) {
    const V v = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
#pragma unroll
    for (int j = 0; j < W; ++j) r.v[j] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) r.v[j] = j < count ? p[j] : T(0);
  }
  return r;
}

template <typename T, int W>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, W>& r) {
  typedef T V __attribute__((ext_vector_type(W), aligned(sizeof(T) * W)));
  V v;
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = r.v[j];
  __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
}

// 1 / x of a normal x > 0 or infinity to a unit in the last place: the hardware's
// estimate, which is 0 from 2^126 on, and a Newton step.
__device__ __forceinline__ float reciprocal(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return r == 0.0f ? 0.0f : __builtin_fmaf(r, __builtin_fmaf(-x, r, 1.0f), r);
}
__device__ __forceinline__ double reciprocal(double x) { return 1.0 / x; }

// `root_v`: sqrt(v).
template <typename T>
__device__ __forceinline__ T update(T p, T m, T root_v, T decay, T step, T root, T eps) {
  return p - (decay * p + step * m * reciprocal(root_v * root + eps));
}

// The correctly rounded root. Between 2^-96 and 2^96 (and of 0) by the coupled
// iteration of Markstein (Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990) without the scaling that the ends of the type need:
// eleven instructions in place of about eighteen.
__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(v);
  float g = v * y, h = 0.5f * y;
  const float r = __builtin_fmaf(-h, g, 0.5f);
  g = __builtin_fmaf(g, r, g);
  h = __builtin_fmaf(h, r, h);
  g = __builtin_fmaf(__builtin_fmaf(-g, g, v), h, g);
  return v == 0.0f ? v : g;
}

// Roots of a lane's elements; all lanes of a wave take one way.
__device__ __forceinline__ Pack<float, 4> roots(const Pack<float, 4>& v) {
  bool plain = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) plain = plain && (v.v[j] == 0.0f || (v.v[j] > 0x1p-96f && v.v[j] < 0x1p96f));
  Pack<float, 4> r;
  if (__all(plain)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = root_of(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = __builtin_sqrtf(v.v[j]);
  }
  return r;
}
__device__ __forceinline__ Pack<double, 4> roots(const Pack<double, 4>& v) {
  Pack<double, 4> r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.v[j] = __builtin_sqrt(v.v[j]);
  return r;
}

// ---- 8-bit shares ----------------------------------------------------------------

// LOW: the lowest 16 codes are multiples of 2^-LOW; from the octave 2^(4 - LOW) on
// each octave has 16 codes. A share plus 1.5 x 2^(octave + 19) is rounded to its
// octave's step, 2^(octave - 4), and has the number of steps in its last bits.
template <int LOW>
__device__ __forceinline__ unsigned encode(float share) {
  constexpr unsigned kLowest = (127 + 4 - LOW) << 23, kMagic = (19u << 23) + 0x400000u;
  const unsigned octave = max(__float_as_uint(share) & 0x7F800000u, kLowest);
  const unsigned steps = __float_as_uint(share + __uint_as_float(octave + kMagic));
  return steps - octave + (octave >> 19) - (kMagic + (kLowest >> 19));
}

// A code's bits, put to the top of a float below its sign, are its share times
// 2^(LOW - 130), with the float's own denormal numbers for the lowest 16.
template <int LOW>
__device__ __forceinline__ float decode(unsigned top_bits) {
  constexpr unsigned kScale = (127 + 130 - LOW) << 23;
  return __uint_as_float(top_bits) * __uint_as_float(kScale);
}

constexpr int kFirst = 10, kSecond = 18;

__device__ __forceinline__ float decode_first(unsigned code, float top) {
  return decode<kFirst>((code & 128) << 24 | (code & 127) << 19) * top;
}

__device__ __forceinline__ float decode_second(unsigned code, float top) {
  const float u = decode<kSecond>(code << 19) * top;
  return u * u;
}

// The largest of values >= 0 over a wave; NaN if one is NaN or infinite.
__device__ __forceinline__ float block_top(const Pack<float, 4>& v) {
  // Bits of floats >= 0 order as integers, infinity and then NaN above all others.
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(v.v[j]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, unsigned(__shfl_xor(int(top), o, 64)));
  return top >= 0x7F800000u ? __builtin_nanf("") : __uint_as_float(top);
}

// Shares in `top`, each correctly rounded: two corrections of the product with the
// reciprocal (Markstein, as above), or where that could leave the type, divisions.
__device__ __forceinline__ Pack<float, 4> shares(const Pack<float, 4>& v, float top) {
  Pack<float, 4> r;
  if (top > 0x1p-60f && top < 0x1p60f) {
    const float inverse = reciprocal(top);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float q = v.v[j] * inverse;
      q = __builtin_fmaf(__builtin_fmaf(-q, top, v.v[j]), inverse, q);
      r.v[j] = __builtin_fmaf(__builtin_fmaf(-q, top, v.v[j]), inverse, q);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = v.v[j] / top;
  }
  return r;
}

// Codes of four moments a lane of a block of 256 (`root`: of the second), and the
// block's scales.
__device__ __forceinline__ void encode_block(const Pack<float, 4>& m, const Pack<float, 4>& root, int64_t block,
                                             const Moments<float>& to, int lane) {
  Pack<float, 4> size;
#pragma unroll
  for (int j = 0; j < 4; ++j) size.v[j] = __builtin_fabsf(m.v[j]);
  const float top1 = block_top(size), top2 = block_top(root);
  uint32_t codes1 = 0, codes2 = 0;
  // Comparisons that a NaN scale fails leave code 0, which stands for 0 times NaN.
  if (top1 > 0) {
    const Pack<float, 4> share = shares(size, top1);
#pragma unroll
    for (int j = 0; j < 4; ++j) codes1 |= encode<kFirst>(share.v[j]) << 8 * j;
  }
  if (top2 > 0) {
    const Pack<float, 4> share = shares(root, top2);
#pragma unroll
    for (int j = 0; j < 4; ++j) codes2 |= max(encode<kSecond>(share.v[j]), root.v[j] > 0 ? 1u : 0u) << 8 * j;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) codes1 |= (__float_as_uint(m.v[j]) >> 31) << (8 * j + 7);
  reinterpret_cast<uint32_t*>(to.codes1)[block * 64 + lane] = codes1;
  reinterpret_cast<uint32_t*>(to.codes2)[block * 64 + lane] = codes2;
  if (lane == 0) to.top1[block] = top1, to.top2[block] = top2;
}

// ---- kernels -----------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ int find(const Table<T>& table, int64_t chunk) {
  int low = 0, high = table.count;
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (table.tensor[middle].chunk <= chunk) low = middle;
    else high = middle;
  }
  return low;
}

template <typename T>
__global__ __launch_bounds__(256) void step_kernel(Table<T> table, Moments<T> from, Moments<T> to, T* __restrict__ params,
                                                   Scalars s) {
  constexpr int W = 4;
  const int64_t chunk = table.first_chunk + blockIdx.x;
  const Tensor<T>& t = table.tensor[find(table, chunk)];
  const int lane = threadIdx.x & 63;
  const int64_t block = chunk * (kChunk / kBlock) + (threadIdx.x >> 6);
  const int64_t place = block * kBlock + lane * W;                  // in the state
  const int64_t at = place - t.chunk * kChunk, left = t.size - at;  // in the tensor
  const bool whole = left >= W;
  const Pack<T, W> p = load_pack<T, W>(t.param + at, whole, left), g = load_pack<T, W>(t.grad + at, whole, left);
  Pack<T, W> m, v, out;
  uint32_t codes1 = 0, codes2 = 0;
  float top1 = 0, top2 = 0;
  if constexpr (sizeof(T) == 4) {
    if (from.codes1) {
      codes1 = reinterpret_cast<const uint32_t*>(from.codes1)[block * 64 + lane];
      codes2 = reinterpret_cast<const uint32_t*>(from.codes2)[block * 64 + lane];
      top1 = from.top1[block], top2 = from.top2[block];
    }
  }
  if (sizeof(T) == 8 || !from.codes1) {
    m = load_pack<T, W>(from.first + place, true, W);
    v = load_pack<T, W>(from.second + place, true, W);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      m.v[j] = decode_first(codes1 >> 8 * j & 255, top1);
      v.v[j] = decode_second(codes2 >> 8 * j & 255, top2);
    }
  }
  const T beta1 = T(s.beta1), beta2 = T(s.beta2), rest1 = T(s.rest1), rest2 = T(s.rest2);
  const T step = T(s.step), root = T(s.root), eps = T(s.eps), decay = T(t.decay);
#pragma unroll
  for (int j = 0; j < W; ++j) {
    m.v[j] = m.v[j] * beta1 + g.v[j] * rest1;
    v.v[j] = v.v[j] * beta2 + (g.v[j] * g.v[j]) * rest2;
  }
  const Pack<T, W> root_v = roots(v);
#pragma unroll
  for (int j = 0; j < W; ++j) out.v[j] = update(p.v[j], m.v[j], root_v.v[j], decay, step, root, eps);
  store_pack<T, W>(params + place, out);
  if constexpr (sizeof(T) == 4) {
    if (to.codes1) {
      encode_block(m, root_v, block, to, lane);
      return;
    }
  }
  store_pack<T, W>(to.first + place, m);
  store_pack<T, W>(to.second + place, v);
}

// Moments given as tensors (param: the first, grad: the second) into the state.
template <typename T>
__global__ __launch_bounds__(256) void load_kernel(Table<T> table, Moments<T> to) {
  constexpr int W = 4;
  const int64_t chunk = table.first_chunk + blockIdx.x;
  const Tensor<T>& t = table.tensor[find(table, chunk)];
  const int lane = threadIdx.x & 63;
  const int64_t block = chunk * (kChunk / kBlock) + (threadIdx.x >> 6), place = block * kBlock + lane * W;
  const int64_t at = place - t.chunk * kChunk, left = t.size - at;
  const Pack<T, W> m = load_pack<T, W>(t.param + at, left >= W, left), v = load_pack<T, W>(t.grad + at, left >= W, left);
  if constexpr (sizeof(T) == 4) {
    if (to.codes1) {
      encode_block(m, roots(v), block, to, lane);
      return;
    }
  }
  store_pack<T, W>(to.first + place, m);
  store_pack<T, W>(to.second + place, v);
}

// The values of the codes of one moment, in the state's order.
__global__ __launch_bounds__(256) void values_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ tops,
                                                     float* __restrict__ values, int64_t blocks, bool first) {
  const int lane = threadIdx.x & 63;
  for (int64_t block = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); block < blocks; block += int64_t(gridDim.x) * 4) {
    const uint32_t four = reinterpret_cast<const uint32_t*>(codes)[block * 64 + lane];
    const float top = tops[block];
    Pack<float, 4> r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned code = four >> 8 * j & 255;
      r.v[j] = first ? decode_first(code, top) : decode_second(code, top);
    }
    store_pack<float, 4>(values + block * kBlock + lane * 4, r);
  }
}

// ---- host ----------------------------------------------------------------------

int64_t chunks_of(int64_t size) { return hp::ceil_div(size, kChunk); }

// The state's arrays in one allocation: two moments, or two arrays of codes
// and two of scales.
template <typename T>
Moments<T> moments_at(void* state, int bits, int64_t chunks) {
  Moments<T> m{};
  const int64_t elements = chunks * kChunk, blocks = elements / kBlock;
  if (bits == 8) {
    m.codes1 = static_cast<uint8_t*>(state);
    m.codes2 = m.codes1 + elements;
    m.top1 = reinterpret_cast<float*>(m.codes2 + elements);
    m.top2 = m.top1 + blocks;
  } else {
    m.first = static_cast<T*>(state);
    m.second = m.first + elements;
  }
  return m;
}

int64_t check_tensors(int dtype, int bits, int64_t count, const int64_t* sizes) {
  hp::require(dtype == HP_F32 || dtype == HP_F64, "AdamW requires float32 or float64");
  hp::require(bits == 0 || (bits == 8 && dtype == HP_F32), "states are of the parameters' type, or of 8 bits for float32");
  hp::require(count >= 0 && (count == 0 || sizes), "bad list of tensors");
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    hp::require(sizes[i] >= 0, "negative size");
    chunks += chunks_of(sizes[i]);
  }
  return chunks;
}

// Launches over the list, tensors of no elements left out, a table at a time
// and at most kMaxGrid workgroups.
template <typename T, typename Launch>
void over_tensors(int64_t count, const void* const* one, const void* const* two, const int64_t* sizes, const double* decays,
                  Launch&& launch) {
  Table<T> table{};
  int64_t chunk = 0;
  const auto flush = [&] {
    const int64_t end = chunk;
    for (int64_t at = table.first_chunk; at < end; at += hp::kMaxGrid) {
      table.first_chunk = at;
      launch(table, unsigned(std::min(end - at, hp::kMaxGrid)));
    }
    table.count = 0;
    table.first_chunk = end;
  };
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    hp::require(one[i] && two[i], "null tensor");
    table.tensor[table.count++] = {static_cast<const T*>(one[i]), static_cast<const T*>(two[i]), sizes[i], chunk,
                                   decays ? decays[i] : 0.0};
    chunk += chunks_of(sizes[i]);
    if (table.count == kTensors) flush();
  }
  if (table.count) flush();
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == HP_F32) f(float(0));
  else f(double(0));
}

}  // namespace

extern "C" {

int hp_adamw_layout(int dtype, int bits, int64_t count, const int64_t* sizes, int64_t* offsets, int64_t* elements,
                    int64_t* state_bytes) {
  return hp::guarded([&] {
    hp::require(elements && state_bytes && (count == 0 || offsets), "null output");
    const int64_t chunks = check_tensors(dtype, bits, count, sizes);
    int64_t chunk = 0;
    for (int64_t i = 0; i < count; ++i) {
      offsets[i] = chunk * kChunk;
      chunk += chunks_of(sizes[i]);
    }
    *elements = chunks * kChunk;
    const int64_t size = int64_t(hp::dtype_size(dtype));
    *state_bytes = bits == 8 ? 2 * *elements + 2 * (*elements / kBlock) * 4 : 2 * *elements * size;
  });
}

int hp_adamw_load(hp_ctx* ctx, int dtype, int bits, int64_t count, const void* const* first, const void* const* second,
                  const int64_t* sizes, void* state) {
  return hp::guarded([&] {
    hp::enter(ctx);
    const int64_t chunks = check_tensors(dtype, bits, count, sizes);
    if (chunks == 0) return;
    hp::require(state && first && second, "null pointer");
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      const Moments<T> to = moments_at<T>(state, bits, chunks);
      over_tensors<T>(count, first, second, sizes, nullptr, [&](const Table<T>& table, unsigned grid) {
        load_kernel<T><<<grid, 256, 0, ctx->stream>>>(table, to);
        hp::check_launch("AdamW load");
      });
    });
  });
}

int hp_adamw_values(hp_ctx* ctx, int64_t elements, const void* state, int which, void* values) {
  return hp::guarded([&] {
    hp::enter(ctx);
    hp::require(elements >= 0 && elements % kChunk == 0, "elements are no whole chunks");
    hp::require(which == 0 || which == 1, "no such moment");
    if (elements == 0) return;
    hp::require(state && values, "null pointer");
    const Moments<float> m = moments_at<float>(const_cast<void*>(state), 8, elements / kChunk);
    const int64_t blocks = elements / kBlock;
    values_kernel<<<unsigned(std::min(hp::ceil_div(blocks, 4), hp::kMaxGrid)), 256, 0, ctx->stream>>>(
        which ? m.codes2 : m.codes1, which ? m.top2 : m.top1, static_cast<float*>(values), blocks, which == 0);
    hp::check_launch("AdamW values");
  });
}

int hp_adamw_step(hp_ctx* ctx, int dtype, int bits, int64_t count, const void* const* params, const void* const* grads,
                  const int64_t* sizes, const double* decays, const void* state, void* new_state, void* new_params,
                  double beta1, double beta2, double step, double root, double eps) {
  return hp::guarded([&] {
    hp::enter(ctx);
    const int64_t chunks = check_tensors(dtype, bits, count, sizes);
    if (chunks == 0) return;
    hp::require(params && grads && decays && state && new_state && new_params, "null pointer");
    hp::require(state != new_state, "the new state takes a place of its own");
    const Scalars s{beta1, beta2, 1 - beta1, 1 - beta2, step, root, eps};
    by_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      const Moments<T> from = moments_at<T>(const_cast<void*>(state), bits, chunks);
      const Moments<T> to = moments_at<T>(new_state, bits, chunks);
      over_tensors<T>(count, params, grads, sizes, decays, [&](const Table<T>& table, unsigned grid) {
        step_kernel<T><<<grid, 256, 0, ctx->stream>>>(table, from, to, static_cast<T*>(new_params), s);
        hp::check_launch("AdamW step");
      });
    });
  });
}

}  // extern "C"
