// AdamW (Adam with decoupled weight decay) over many tensors in one launch, moments in 32 bits or in 8, and what comes before it in a
// step: the norm of all gradients together, by which they are clipped, and the corrections of step counts kept on the device.
//
//   m = b1 m + (1 - b1) c g,  v = b2 v + (1 - b2) (c g)^2,  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// with c = min(1, max_norm / (|g| + 1e-6)) where a norm is given. Every tensor has its own rates and step count. Parameters and gradients
// are float32, float16 or bfloat16 (rounded to nearest once, when they are stored); the moments are float32 or the 8-bit blocks below.
//
// Moments in 8 bits. Adam's moments move by parts in ten (m) and in a thousand (v) of a step, far less than the spacing of 8-bit
// values: rounding to the nearest one would leave them where they are for good. They are rounded down after a number in [0, 1) spacings
// has been added, 16 bits of a hash of (element, step count, seed), so that the mean of what is kept is the value (of v itself: rounding
// its root in that way would raise the mean of v by the variance of the root). A block is 256 consecutive elements, four for each lane of
// a wavefront, under one power of two for each moment, the smallest for which the highest code is not below the largest value (a
// value above it could only be rounded down).
//   m  sign, 4 bits of exponent, 3 of fraction: 18 binades
//   v  5 bits of exponent, 3 of fraction: 34 binades, 17 of the root; a value above 0 is kept above 0, since an element whose
//      second moment vanished before its first would be divided by eps alone
// Both are the top of a float with a small exponent: decoding shifts the code to its place in a float32 and scales by a power of two; encoding
// scales a float64, adds the noise below the last kept bit of its upper word and shifts, subnormal values of the format included, with no
// case of its own.
// A state is one allocation: codes of m [256 b], codes of v [256 b], exponents (m, v) [b][2] for b blocks. Exponents are those of
// float32 (biased by 127); 0 is a block of zeros, 255 one that held an infinity or a NaN, all of whose values read as NaN.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <cmath>

#include "../../include/fsgs.h"
#include "common.hpp"

namespace fsgs {
namespace {

constexpr int kBlock = 256;        // elements of an 8-bit block
constexpr int kMaxTensors = 48;    // a launch's table is passed by value: 80 bytes a tensor of the 4 KB that arguments may have
constexpr int kNormBlocks = 1024;  // of the sum of squares: a sum each
constexpr int kNormChunk = 8192;   // elements that a block sums before it looks for its next ones

struct Rates {  // of one tensor's step, formed on the host or by adamw_rates_kernel
  float step_size, inv_root_c2;
  uint32_t key;  // of the step's noise
  uint32_t pad;
};

struct AdamwTable {
  void* param[kMaxTensors];
  const void* grad[kMaxTensors];
  void* m[kMaxTensors];  // 8-bit moments: the state
  float* v[kMaxTensors];
  int64_t count[kMaxTensors];
  Rates rates[kMaxTensors];
  float keep[kMaxTensors];  // 1 - lr wd
  float eps[kMaxTensors];
  unsigned first_block[kMaxTensors + 1];
  int n;
};
static_assert(sizeof(AdamwTable) <= 4032, "kernel arguments");

// The tensor that block `b` of a launch works on.
__device__ __forceinline__ int tensor_of(const unsigned* first, int n, unsigned b) {
  int low = 0, high = n;  // first[low] <= b < first[high]
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (b >= first[mid]) low = mid;
    else high = mid;
  }
  return low;
}

// ---- four elements at a time --------------------------------------------------------------------------------------------------
template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T x[4];
};
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half(x); }
template <>
__device__ __forceinline__ __hip_bfloat16 from_float<__hip_bfloat16>(float x) { return __float2bfloat16(x); }

// One access of sizeof(Q) bytes; `kStream`: past the caches, which what is touched once a step would empty.
template <bool kStream, typename Q>
__device__ __forceinline__ Q get(const void* p) {
  typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(Q) / 4)));
  const Raw raw = kStream ? __builtin_nontemporal_load((const Raw*) p) : *(const Raw*) p;
  return __builtin_bit_cast(Q, raw);
}
template <bool kStream, typename Q>
__device__ __forceinline__ void put(void* p, const Q& q) {
  typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(Q) / 4)));
  if (kStream) __builtin_nontemporal_store(__builtin_bit_cast(Raw, q), (Raw*) p);
  else *(Raw*) p = __builtin_bit_cast(Raw, q);
}

// Four elements as they lie in memory. `kWhole`: all are there, and their address allows one access; otherwise `left` of them are. Loads of
// a whole block stand one behind the other, with no branch and no conversion between them: a wavefront waits for memory once.
template <bool kWhole, bool kStream, typename T>
__device__ __forceinline__ Four<T> load4(const T* p, int64_t left) {
  if (kWhole) return get<kStream, Four<T>>(p);
  Four<T> q;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) q.x[k] = p[k];
    else q.x[k] = from_float<T>(0.0f);
  return q;
}
template <bool kWhole, bool kStream, typename T>
__device__ __forceinline__ void store4(T* p, int64_t left, const float in[4]) {
  Four<T> q;
#pragma unroll
  for (int k = 0; k < 4; ++k) q.x[k] = from_float<T>(in[k]);
  if (kWhole) {
    put<kStream>(p, q);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = q.x[k];
  }
}

struct Step {
  float b1, b2, c1, c2;  // c = 1 - b
};
// What the norm of the gradients leaves for the step.
struct Norm {
  float norm, factor;
  double exact;  // factor, before it was rounded
};

// One element, whose moments are the step's already. The root and the reciprocal are the hardware's, one unit in the last place each. The root's
// instruction takes subnormal numbers for 0, so v counts as 2^-126 at least: the smallest root is 1e-19, a hundred-thousandth of an eps
// of 1e-15 (scenes' own), and nothing is divided by 0 where eps is. A NaN stays one.
__device__ __forceinline__ float updated(const Rates& r, float keep, float eps, float p, float m, float v) {
  const float root = __builtin_amdgcn_sqrtf(v < 0x1p-126f ? 0x1p-126f : v);
  return fmaf(p, keep, -(r.step_size * m * __builtin_amdgcn_rcpf(fmaf(root, r.inv_root_c2, eps))));
}

// ---- 32-bit moments -------------------------------------------------------------------------------------------------------------
// A block steps 1024 elements of one tensor, found by a binary search in the table that the launch carries: one launch whatever the tensors'
// number and sizes, no job list in memory. 28 bytes an element in float32 (22 in 16 bits) for some fifteen operations: memory. 174M elements
// of six tensors 805 - 821 us (6.0 TB/s), 8M in bfloat16 29 us, 0.5M in 25 tensors 5.1 us, which is the launch and two dependent loads.
// What a block needs of its tensor, in scalar registers.
template <typename T>
struct Part {
  T* param;
  const T* grad;
  void* m;
  float* v;
  int64_t count, first;  // first: of the block's elements
  Rates rate;
  float keep, eps, factor;
  double exact_factor;
  bool aligned;  // param and grad, for four elements at once

  __device__ __forceinline__ Part(const AdamwTable& t, const Norm* norm, const Rates* rates) {
    const int q = tensor_of(t.first_block, t.n, blockIdx.x);
    param = (T*) t.param[q], grad = (const T*) t.grad[q], m = t.m[q], v = t.v[q], count = t.count[q];
    first = (int64_t) (blockIdx.x - t.first_block[q]) * 1024;
    rate = t.rates[q], keep = t.keep[q], eps = t.eps[q], factor = 1.0f, exact_factor = 1.0;
    if (rates) {
      const Rates on_device = rates[q];
      rate = on_device;
    }
    if (norm) factor = norm->factor, exact_factor = norm->exact;
    aligned = (((uintptr_t) param | (uintptr_t) grad) & (4 * sizeof(T) - 1)) == 0;
  }
};

template <typename T, bool kStream, bool kWhole>
__device__ __forceinline__ void adamw_block(const Part<T>& t, const Step& s) {
  const int64_t e = t.first + threadIdx.x * 4, left = t.count - e;
  if (!kWhole && left <= 0) return;
  float *first = (float*) t.m + e, *second = t.v + e;
  const Four<T> param = load4<kWhole, kStream>(t.param + e, left), grad = load4<kWhole, kStream>(t.grad + e, left);
  Four<float> m = load4<kWhole, kStream>(first, left), v = load4<kWhole, kStream>(second, left);
  float p[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float g = t.factor * to_float(grad.x[k]);
    m.x[k] = fmaf(s.c1, g, s.b1 * m.x[k]), v.x[k] = fmaf(s.c2 * g, g, s.b2 * v.x[k]);
    p[k] = updated(t.rate, t.keep, t.eps, to_float(param.x[k]), m.x[k], v.x[k]);
  }
  store4<kWhole, kStream>(t.param + e, left, p);
  store4<kWhole, kStream>(first, left, m.x), store4<kWhole, kStream>(second, left, v.x);
}

template <typename T, bool kStream>
__global__ void __launch_bounds__(256) adamw_kernel(AdamwTable t, Step s, const Norm* __restrict__ norm,
                                                    const Rates* __restrict__ rates) {
  const Part<T> part(t, norm, rates);
  if (part.aligned && (((uintptr_t) part.m | (uintptr_t) part.v) & 15) == 0 && part.first + 1024 <= part.count)
    adamw_block<T, kStream, true>(part, s);
  else
    adamw_block<T, kStream, false>(part, s);
}

// ---- 8-bit moments ----------------------------------------------------------------------------------------------------------------
// 16 bytes an element in float32 (10 in 16 bits), the exponents 4 in 256: memory in float32, 171M elements 432 - 447 us (6.1 - 6.3 TB/s). In 16 bits
// decoding, the step, the hash and encoding take longer than the accesses: 8M in bfloat16 24 us (3.3 TB/s), 21 with ten operations an element
// less (314 vector instructions for 256 elements; the vector units issue in 0.95 of the busy cycles, with 64M elements in all of them, in float32
// in 0.86). Two blocks for each wavefront were slower.
__host__ __device__ __forceinline__ uint32_t mixed(uint32_t x) {
  x = (x ^ (x >> 16)) * 0xBB67AE85u;
  x = (x ^ (x >> 15)) * 0x3C6EF373u;
  return x ^ (x >> 16);
}
constexpr uint32_t kStride = 0x9E3779B1u;  // between the hashes' arguments of neighbouring elements, and of seeds
__host__ __device__ __forceinline__ uint32_t noise_key(uint32_t step, uint32_t seed) { return mixed(step + seed * kStride); }

// Largest of a value over the wavefront's lanes, in scalar registers: four rotations within rows of 16 lanes, then the rows.
template <int kCtrl>
__device__ __forceinline__ uint32_t max_step(uint32_t x) {
  return max(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max_step<0x128>(x), x = max_step<0x124>(x), x = max_step<0x122>(x), x = max_step<0x121>(x);  // row_ror:8, 4, 2, 1
  const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  return max(max(a, b), max(c, d));
}

constexpr int kBias = 1023 - 127;  // of a float64's exponent over a float32's
__device__ __forceinline__ uint32_t upper(double x) { return (uint32_t) (__builtin_bit_cast(uint64_t, x) >> 32); }

// From a code's place in a float32 (exponent 1 is its lowest binade) to that of its block, whose highest one is 2^kBits - 1.
template <int kBits>  // of exponent
__device__ __forceinline__ float decoded(uint32_t bits, int exponent) {
  return ldexpf(__builtin_bit_cast(float, bits), exponent + 1 - (1 << kBits));
}
// The same the other way round, of a float64, whose upper word has all the bits that count: 3 kept ones and the 16 below them that the noise
// is added to. Betas are decimal numbers: gradients of few bits put moments on a border that the betas' binary neighbours miss by parts
// in 10^16. A border counts as reached from 256 units in the last place below it on (2^-44 of the binade, 6e-14); farther from it a
// code is that of the float64 moment.
constexpr uint64_t kHair = 256;
template <int kBits>
__device__ __forceinline__ uint32_t encoded(double x, int exponent, uint32_t noise16, uint32_t least) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, ldexp(x, (1 << kBits) - 1 - kBias - exponent));
  const uint32_t y = (uint32_t) ((bits + kHair) >> 32);
  return min(max((y + (noise16 << 1)) >> 17, least), (8u << kBits) - 1);
}
// Element k of the four whose codes are in a word each.
template <int k>
__device__ __forceinline__ void decode(uint32_t codes_m, uint32_t codes_v, int exponent_m, int exponent_v, float& m, float& v) {
  // a code's magnitude to bits 20 to 26 (m) or 27 (v), m's sign to bit 31
  const uint32_t a = k == 0 ? codes_m << 20 : k == 1 ? codes_m << 12 : k == 2 ? codes_m << 4 : codes_m >> 4;
  const uint32_t b = k == 0 ? codes_v << 20 : k == 1 ? codes_v << 12 : k == 2 ? codes_v << 4 : codes_v >> 4;
  m = decoded<4>((a & 0x07f00000u) | ((codes_m << (24 - 8 * k)) & 0x80000000u), exponent_m);
  v = decoded<5>(b & 0x0ff00000u, exponent_v);
}
__device__ __forceinline__ void decode4(uint32_t codes_m, uint32_t codes_v, int exponent_m, int exponent_v, float m[4], float v[4]) {
  decode<0>(codes_m, codes_v, exponent_m, exponent_v, m[0], v[0]), decode<1>(codes_m, codes_v, exponent_m, exponent_v, m[1], v[1]);
  decode<2>(codes_m, codes_v, exponent_m, exponent_v, m[2], v[2]), decode<3>(codes_m, codes_v, exponent_m, exponent_v, m[3], v[3]);
  if (exponent_m == 255)
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = __builtin_nanf("");
  if (exponent_v == 255)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __builtin_nanf("");
}
// A block's exponent byte from the upper word of its largest magnitude (a NaN is larger than any; the last bit stands for all bits
// of the lower word): that of the next binade where the value is above 1.875 of its own. What float32 cannot hold is an infinity or 0. Below the
// normal numbers the lowest normal exponent stands for all; 254 is the last of finite values.
__device__ __forceinline__ int block_exponent(uint32_t top) {
  if (top >= (uint32_t) (kBias + 255) << 20) return 255;
  if (top < (uint32_t) (kBias + 1 - 23) << 20) return 0;
  return min(max((int) ((top + 0x1ffffu) >> 20) - kBias, 1), 254);
}
__device__ __forceinline__ uint32_t magnitude(double x) {
  return (upper(x) & 0x7fffffffu) | min((uint32_t) __builtin_bit_cast(uint64_t, x), 1u);
}

// Codes of four elements of a block, and the block's exponents; the noise of m in the low half of a word, of v in the high one. The moments come
// in 64 bits: rounded to 32 before, one value in a million falls on the other side of a border, and equal inputs give other codes than the
// definition does. Ten more operations an element, at the rate of 32-bit ones: 64M elements in float32 181 us against 174, in bfloat16 154
// against 143.
__device__ __forceinline__ void encode4(const double m[4], const double v[4], const uint32_t noise[4], uint32_t& codes_m,
                                        uint32_t& codes_v, int& exponent_m, int& exponent_v) {
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) top_m = max(top_m, magnitude(m[k])), top_v = max(top_v, magnitude(v[k]));
  exponent_m = block_exponent(wave_max(top_m)), exponent_v = block_exponent(wave_max(top_v));
  codes_m = codes_v = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t a = encoded<4>(fabs(m[k]), exponent_m, noise[k] & 0xffffu, 0);
    const uint32_t b = encoded<5>(v[k], exponent_v, noise[k] >> 16, (float) v[k] > 0.0f ? 1 : 0);
    codes_m |= (a | ((upper(m[k]) >> 24) & 128u)) << (8 * k);
    codes_v |= b << (8 * k);
  }
}

struct Shares {  // of the new gradient, 1 - b, in the moments
  double c1, c2;
};
struct StateView {  // of a tensor's 8-bit moments
  uint8_t *m, *v, *exponents;
};
__host__ __device__ __forceinline__ StateView view_state(void* state, int64_t count) {
  const int64_t b = (count + kBlock - 1) / kBlock;
  uint8_t* at = (uint8_t*) state;
  return {at, at + b * kBlock, at + 2 * b * kBlock};
}

// A wavefront steps a block: a lane has four elements of it.
template <typename T, bool kStream, bool kWhole>
__device__ __forceinline__ void adamw8_block(const Part<T>& t, const Shares& s, int64_t block) {
  const int lane = threadIdx.x & 63;
  const int64_t e = block * kBlock + lane * 4, left = t.count - e;
  const StateView state = view_state(t.m, t.count);
  const Four<T> param = load4<kWhole, kStream>(t.param + e, left), grad = load4<kWhole, kStream>(t.grad + e, left);
  uint32_t codes_m = get<kStream, uint32_t>(state.m + e), codes_v = get<kStream, uint32_t>(state.v + e);
  const int exponents = __builtin_amdgcn_readfirstlane(*(const uint16_t*) (state.exponents + 2 * block));
  float old_m[4], old_v[4], p[4];
  double m[4], v[4];
  uint32_t noise[4];
  decode4(codes_m, codes_v, exponents & 255, exponents >> 8, old_m, old_v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double g = t.exact_factor * (double) to_float(grad.x[k]);
    // as b m + (1 - b) g, but what the gradient does not move stays where it is to the last bit, on its code's border
    m[k] = fma(s.c1, g - (double) old_m[k], (double) old_m[k]), v[k] = fma(s.c2, fma(g, g, -(double) old_v[k]), (double) old_v[k]);
    p[k] = updated(t.rate, t.keep, t.eps, to_float(param.x[k]), (float) m[k], (float) v[k]);
    if (!kWhole && k >= left) m[k] = v[k] = 0.0;
    noise[k] = mixed((uint32_t) (e + k) * kStride + t.rate.key);
  }
  int exponent_m, exponent_v;
  encode4(m, v, noise, codes_m, codes_v, exponent_m, exponent_v);
  store4<kWhole, kStream>(t.param + e, left, p);
  put<kStream>(state.m + e, codes_m), put<kStream>(state.v + e, codes_v);
  if (lane == 0) *(uint16_t*) (state.exponents + 2 * block) = (uint16_t) (exponent_m | exponent_v << 8);
}

template <typename T, bool kStream>
__global__ void __launch_bounds__(256) adamw8_kernel(AdamwTable t, Shares s, const Norm* __restrict__ norm,
                                                     const Rates* __restrict__ rates) {
  const Part<T> part(t, norm, rates);
  const int64_t block = part.first / kBlock + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (block * kBlock >= part.count) return;  // the whole wavefront
  if (part.aligned && (block + 1) * kBlock <= part.count) adamw8_block<T, kStream, true>(part, s, block);
  else adamw8_block<T, kStream, false>(part, s, block);
}

struct MomentsTable {
  void* state[kMaxTensors];
  void* m[kMaxTensors];
  void* v[kMaxTensors];
  int64_t count[kMaxTensors];
  unsigned first_block[kMaxTensors + 1];
  int n;
};

// The values that 8-bit moments stand for; a lane writes 16 bytes of each. 171M elements in bfloat16 162 us (6.3 TB/s), 8M 10.5 us.
template <typename T, bool kStream>
__global__ void __launch_bounds__(256) adamw8_unpack_kernel(MomentsTable t) {
  constexpr int kWords = 4 / sizeof(T);  // of four codes
  const int q = tensor_of(t.first_block, t.n, blockIdx.x);
  const int64_t e = ((int64_t) (blockIdx.x - t.first_block[q]) * 256 + threadIdx.x) * 4 * kWords, left = t.count[q] - e;
  if (left <= 0) return;
  const StateView state = view_state(t.state[q], t.count[q]);
  T *first = (T*) t.m[q] + e, *second = (T*) t.v[q] + e;
  const int exponent_m = state.exponents[2 * (e / kBlock)], exponent_v = state.exponents[2 * (e / kBlock) + 1];
  const bool whole = left >= 4 * kWords && (((uintptr_t) first | (uintptr_t) second) & 15) == 0;
  struct alignas(16) Values { T x[4 * kWords]; } pm, pv;
  struct alignas(4 * kWords) Codes { uint32_t x[kWords]; };
  const Codes codes_m = get<kStream, Codes>(state.m + e), codes_v = get<kStream, Codes>(state.v + e);
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    float m[4], v[4];
    decode4(codes_m.x[w], codes_v.x[w], exponent_m, exponent_v, m, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) pm.x[4 * w + k] = from_float<T>(m[k]), pv.x[4 * w + k] = from_float<T>(v[k]);
  }
  if (whole) {
    put<kStream>(first, pm), put<kStream>(second, pv);
  } else {
#pragma unroll
    for (int k = 0; k < 4 * kWords; ++k)
      if (k < left) first[k] = pm.x[k], second[k] = pv.x[k];
  }
}

// 8-bit moments of given values (m, v), rounded to the nearest: they are taken over once, not step after step. Element by element: 8M 25 us, 64M 196 us
// (3.4 TB/s, 1.4 of a copy's time).
__global__ void __launch_bounds__(256) adamw8_pack_kernel(MomentsTable t) {
  const int q = tensor_of(t.first_block, t.n, blockIdx.x);
  const int64_t block = (int64_t) (blockIdx.x - t.first_block[q]) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (block * kBlock >= t.count[q]) return;
  const int64_t e = block * kBlock + lane * 4, left = t.count[q] - e;
  const StateView state = view_state(t.state[q], t.count[q]);
  const Four<float> m = load4<false, false>((const float*) t.m[q] + e, left), v = load4<false, false>((const float*) t.v[q] + e, left);
  const uint32_t noise[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
  const double exact_m[4] = {m.x[0], m.x[1], m.x[2], m.x[3]}, exact_v[4] = {v.x[0], v.x[1], v.x[2], v.x[3]};
  uint32_t codes_m, codes_v;
  int exponent_m, exponent_v;
  encode4(exact_m, exact_v, noise, codes_m, codes_v, exponent_m, exponent_v);
  *(uint32_t*) (state.m + e) = codes_m, *(uint32_t*) (state.v + e) = codes_v;
  if (lane == 0) *(uint16_t*) (state.exponents + 2 * block) = (uint16_t) (exponent_m | exponent_v << 8);
}

// ---- the norm of all gradients --------------------------------------------------------------------------------------------------
struct NormTable {
  const void* grad[kMaxTensors];
  int64_t count[kMaxTensors];
  unsigned first_chunk[kMaxTensors + 1];
  int n;
};

// Sum over the block's 256 threads, in a fixed order; valid in thread 0.
__device__ __forceinline__ double block_sum(double x, double* s_wave) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_down(x, d);
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = x;
  __syncthreads();
  return ((s_wave[0] + s_wave[1]) + s_wave[2]) + s_wave[3];
}

// Sums of squares, in float64 from the first element on: its multiply-adds go at the rate of float32's, and the pass waits for memory. A
// chunk's eight loads are on their way together. 174M float32 104 us (6.7 TB/s), 8M bfloat16 9 us.
template <typename T, bool kStream>
__global__ void __launch_bounds__(256) square_sums_kernel(NormTable t, double* __restrict__ sums) {
  __shared__ double s_wave[4];
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  const auto add = [&](const Four<T>& g) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double x = (double) to_float(g.x[k]);
      sum[k] = fma(x, x, sum[k]);
    }
  };
  for (unsigned chunk = blockIdx.x; chunk < t.first_chunk[t.n]; chunk += gridDim.x) {
    const int q = tensor_of(t.first_chunk, t.n, chunk);
    const int64_t at = (int64_t) (chunk - t.first_chunk[q]) * kNormChunk + threadIdx.x * 4, count = t.count[q];
    const T* grad = (const T*) t.grad[q];
    const bool aligned = ((uintptr_t) grad & (4 * sizeof(T) - 1)) == 0;
    if (aligned && (int64_t) (chunk - t.first_chunk[q] + 1) * kNormChunk <= count) {
      Four<T> g[kNormChunk / 1024];
#pragma unroll
      for (int j = 0; j < kNormChunk / 1024; ++j) g[j] = load4<true, kStream>(grad + at + j * 1024, 4);
#pragma unroll
      for (int j = 0; j < kNormChunk / 1024; ++j) add(g[j]);
    } else {
      for (int64_t e = at; e < count && e < at + kNormChunk; e += 1024) add(load4<false, kStream>(grad + e, count - e));
    }
  }
  const double total = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]), s_wave);
  if (threadIdx.x == 0) sums[blockIdx.x] = total;
}

__global__ void __launch_bounds__(256) norm_factor_kernel(int n, const double* __restrict__ sums, double max_norm, Norm* __restrict__ out) {
  __shared__ double s_wave[4];
  double total = 0.0;
  for (int k = threadIdx.x; k < n; k += 256) total += sums[k];
  total = block_sum(total, s_wave);
  if (threadIdx.x != 0) return;
  const double norm = sqrt(total), factor = max_norm / (norm + 1e-6);
  // a NaN passes, as a comparison with it would not let it
  const double exact = factor > 1.0 ? 1.0 : factor;
  *out = Norm{(float) norm, (float) exact, exact};
}

// ---- step counts on the device ------------------------------------------------------------------------------------------------
struct StepTable {
  float* step[kMaxTensors];
  double lr[kMaxTensors];
  int n;
};
__global__ void __launch_bounds__(64) adamw_rates_kernel(StepTable t, double b1, double b2, uint32_t seed, Rates* __restrict__ rates) {
  const int q = threadIdx.x;
  if (q >= t.n) return;
  const float step = *t.step[q] + 1.0f;
  *t.step[q] = step;
  Rates r{};
  r.step_size   = (float) (t.lr[q] / (1.0 - pow(b1, (double) step)));
  r.inv_root_c2 = (float) (1.0 / sqrt(1.0 - pow(b2, (double) step)));
  r.key         = noise_key((uint32_t) step, seed);
  rates[q] = r;
}

enum Type { kFloat32 = FSGS_DTYPE_F32, kFloat16 = FSGS_DTYPE_F16, kBfloat16 = FSGS_DTYPE_BF16 };
size_t type_size(int type) { return type == kFloat32 ? 4 : 2; }
bool is_type(int type) { return type == kFloat32 || type == kFloat16 || type == kBfloat16; }

// A launch that moves this many MiB goes past the caches: less may still be, or stay, in the 256 MB memory-side cache. us of a step of n
// elements, three sets of tensors in turn, ordinary and streaming accesses: float32 4M (117 MB) 18.3 and 21.7, 8M 46.1 and 41.0, 16M
// 92.1 and 82.2, 64M 351 and 334; bfloat16 4M 15.0 and 16.9, 8M (185 MB) 32.9 and 32.3, 16M 68.7 and 60.7, 64M 270 and 250; 8-bit
// moments, float32 8M (134 MB) 23.6 and 26.0, 16M 52.3 and 48.6, 64M 193 and 176. One set again and again, with nothing in between, gains by
// the cache up to 20M elements (16M 65.9 and 79.7), which no training loop does.
constexpr int kStepMiB = 160;
// What is read back is mostly writes, which the cache takes in longer: float32 16M (168 MB) 26.1 and 31.4, 28M 45.7 and 50.4, 32M (336 MB)
// 60.0 and 59.1, 64M 114.7 and 114.0; bfloat16 40M (252 MB) 42.3 and 43.9, 48M 51.2 and 52.6, 64M (403 MB) 73.5 and 68.5. The sum of squares,
// reads alone, goes by the step's limit.
constexpr int kReadBackMiB = 320;
bool streams(int n, const int64_t* count, size_t bytes_an_element, int mib = kStepMiB) {
  int64_t sum = 0;
  for (int q = 0; q < n; ++q) sum += count[q];
  return sum >= ((int64_t) mib << 20) / (int64_t) bytes_an_element;
}
// kernel<type, streaming>
#define FSGS_BY_TYPE(kernel, dtype, stream)                                                          \
  ((dtype) == kFloat32   ? ((stream) ? kernel<float, true> : kernel<float, false>)                   \
   : (dtype) == kFloat16 ? ((stream) ? kernel<__half, true> : kernel<__half, false>)                 \
                         : ((stream) ? kernel<__hip_bfloat16, true> : kernel<__hip_bfloat16, false>))

// first[q]: blocks before tensor q at `per_block` elements a block. A launch has 2^32 threads at most, in blocks of 256.
template <typename Table>
int lay_out(const char* what, Table& t, unsigned* first, int n, const int64_t* count, int64_t per_block) {
  int64_t blocks = 0;
  for (int q = 0; q < n; ++q) {
    FSGS_REQUIRE(count[q] >= 0, "%s: bad tensor %d", what, q);
    t.count[q] = count[q], first[q] = (unsigned) blocks;
    blocks += (count[q] + per_block - 1) / per_block;
    FSGS_REQUIRE(blocks < (int64_t) 1 << 24, "%s: more than %lld elements in a launch", what, (long long) (per_block << 24));
  }
  first[n] = (unsigned) blocks;
  t.n = n;
  return kOk;
}

}  // namespace
}  // namespace fsgs

using namespace fsgs;

FSGS_API int fsgs_adamw_max_tensors(void) { return kMaxTensors; }
FSGS_API size_t fsgs_adamw8_state_bytes(int64_t count) {
  return count <= 0 ? 0 : (size_t) ((count + kBlock - 1) / kBlock) * (2 * kBlock + 2);
}
FSGS_API int fsgs_grad_square_sums_max(void) { return kNormBlocks; }
FSGS_API size_t fsgs_adamw_rates_bytes(int n_tensors) { return (size_t) (n_tensors > 0 ? n_tensors : 0) * sizeof(Rates); }

FSGS_API int fsgs_grad_square_sums(int n_tensors, int dtype, const int64_t* count, const void* const* grad, int n_sums, double* sums,
                                   void* stream) {
  const char* what = "grad_norm";
  FSGS_REQUIRE(n_tensors > 0 && n_tensors <= kMaxTensors && is_type(dtype) && n_sums > 0 && n_sums <= kNormBlocks,
               "%s: bad arguments (at most %d tensors)", what, kMaxTensors);
  FSGS_REQUIRE(count && grad && sums, "%s: null pointer", what);
  NormTable t{};
  if (const int rc = lay_out(what, t, t.first_chunk, n_tensors, count, kNormChunk)) return rc;
  for (int q = 0; q < n_tensors; ++q) {
    FSGS_REQUIRE(count[q] == 0 || (grad[q] && (uintptr_t) grad[q] % type_size(dtype) == 0), "%s: bad tensor %d", what, q);
    t.grad[q] = grad[q];
  }
  auto kernel = FSGS_BY_TYPE(square_sums_kernel, dtype, streams(n_tensors, count, type_size(dtype)));
  hipLaunchKernelGGL(kernel, dim3(n_sums), dim3(256), 0, (hipStream_t) stream, t, sums);
  return check_launch(what);
}

FSGS_API size_t fsgs_grad_norm_bytes(void) { return sizeof(Norm); }
FSGS_API int fsgs_grad_norm_factor(int n_sums, const double* sums, double max_norm, float* norm_and_factor, void* stream) {
  FSGS_REQUIRE(n_sums >= 0 && (n_sums == 0 || sums) && norm_and_factor, "grad_norm: null pointer");
  FSGS_REQUIRE((uintptr_t) norm_and_factor % 8 == 0, "grad_norm: misaligned address");
  hipLaunchKernelGGL(norm_factor_kernel, dim3(1), dim3(256), 0, (hipStream_t) stream, n_sums, sums, max_norm, (Norm*) norm_and_factor);
  return check_launch("grad_norm");
}

FSGS_API int fsgs_adamw_rates(int n_tensors, float* const* step, const double* lr, double b1, double b2, uint32_t seed, void* rates,
                              void* stream) {
  const char* what = "adamw";
  FSGS_REQUIRE(n_tensors >= 0 && n_tensors <= kMaxTensors, "%s: at most %d tensors", what, kMaxTensors);
  if (n_tensors == 0) return kOk;
  FSGS_REQUIRE(step && lr && rates && ((uintptr_t) rates & 15) == 0, "%s: null pointer", what);
  StepTable t{};
  t.n = n_tensors;
  for (int q = 0; q < n_tensors; ++q) {
    FSGS_REQUIRE(step[q], "%s: bad tensor %d", what, q);
    t.step[q] = step[q], t.lr[q] = lr[q];
  }
  hipLaunchKernelGGL(adamw_rates_kernel, dim3(1), dim3(64), 0, (hipStream_t) stream, t, b1, b2, seed, (Rates*) rates);
  return check_launch(what);
}

namespace {
int adamw_update(const char* what, int bits, int n, int dtype, const int64_t* count, const double* step, const double* lr, double b1,
                 double b2, const double* eps, const double* decay, uint32_t seed, const void* rates, const float* factor,
                 void* const* param, const void* const* grad, void* const* m, float* const* v, void* stream) {
  FSGS_REQUIRE(n >= 0 && n <= kMaxTensors && is_type(dtype), "%s: bad arguments (at most %d tensors)", what, kMaxTensors);
  if (n == 0) return kOk;
  FSGS_REQUIRE(count && lr && eps && decay && param && grad && m && (v || bits == 8) && (step || rates), "%s: null pointer", what);
  AdamwTable t{};
  if (const int rc = lay_out(what, t, t.first_block, n, count, 1024)) return rc;
  if (t.first_block[n] == 0) return kOk;
  double known = 0.0, c1 = 1.0;
  float inv_root_c2 = 1.0f;
  for (int q = 0; q < n; ++q) {
    const uintptr_t wide = (uintptr_t) m[q] | (v ? (uintptr_t) v[q] : 0), narrow = (uintptr_t) param[q] | (uintptr_t) grad[q];
    FSGS_REQUIRE(count[q] == 0 || (param[q] && grad[q] && m[q] && (!v || v[q]) && wide % (bits == 8 ? 16 : 4) == 0 && narrow % type_size(dtype) == 0),
                 "%s: bad tensor %d", what, q);
    t.param[q] = param[q], t.grad[q] = grad[q], t.m[q] = m[q], t.v[q] = v ? v[q] : nullptr;
    t.keep[q] = (float) (1.0 - lr[q] * decay[q]), t.eps[q] = (float) eps[q];
    if (rates) continue;
    FSGS_REQUIRE(step[q] >= 1.0, "%s: tensor %d has taken no step", what, q);
    if (step[q] != known) {  // the tensors of a call mostly share their count, and powers take their time
      known = step[q];
      c1 = 1.0 - std::pow(b1, known), inv_root_c2 = (float) (1.0 / std::sqrt(1.0 - std::pow(b2, known)));
    }
    t.rates[q].step_size   = (float) (lr[q] / c1);
    t.rates[q].inv_root_c2 = inv_root_c2;
    t.rates[q].key         = noise_key((uint32_t) (int64_t) known, seed);
  }
  FSGS_REQUIRE((uintptr_t) factor % 8 == 0, "%s: misaligned address", what);
  const Norm* norm = (const Norm*) factor;
  const bool past = streams(n, count, 3 * type_size(dtype) + (bits == 8 ? 4 : 16));
  const dim3 grid(t.first_block[n]);
  if (bits == 8) {
    const Shares s{1.0 - b1, 1.0 - b2};
    hipLaunchKernelGGL(FSGS_BY_TYPE(adamw8_kernel, dtype, past), grid, dim3(256), 0, (hipStream_t) stream, t, s, norm, (const Rates*) rates);
  } else {
    const Step s{(float) b1, (float) b2, (float) (1.0 - b1), (float) (1.0 - b2)};
    hipLaunchKernelGGL(FSGS_BY_TYPE(adamw_kernel, dtype, past), grid, dim3(256), 0, (hipStream_t) stream, t, s, norm, (const Rates*) rates);
  }
  return check_launch(what);
}

int moments(const char* what, int n, const int64_t* count, const void* const* state, const void* const* m, const void* const* v,
            size_t size, int64_t per_block, MomentsTable& t) {
  FSGS_REQUIRE(n >= 0 && n <= kMaxTensors, "%s: at most %d tensors", what, kMaxTensors);
  if (n == 0) return kOk;
  FSGS_REQUIRE(count && state && m && v, "%s: null pointer", what);
  if (const int rc = lay_out(what, t, t.first_block, n, count, per_block)) return rc;
  for (int q = 0; q < n; ++q) {
    FSGS_REQUIRE(count[q] == 0 || (state[q] && m[q] && v[q] && (uintptr_t) state[q] % 16 == 0 &&
                                   ((uintptr_t) m[q] | (uintptr_t) v[q]) % size == 0), "%s: bad tensor %d", what, q);
    t.state[q] = (void*) state[q], t.m[q] = (void*) m[q], t.v[q] = (void*) v[q];
  }
  return kOk;
}
}  // namespace

FSGS_API int fsgs_adamw_update_multi(int n_tensors, int dtype, const int64_t* count, const double* step, const double* lr, double b1,
    double b2, const double* eps, const double* decay, const void* rates, const float* norm_and_factor, void* const* param,
    const void* const* grad, float* const* m, float* const* v, void* stream) {
  FSGS_REQUIRE(n_tensors == 0 || v, "adamw: null pointer");
  return adamw_update("adamw", 32, n_tensors, dtype, count, step, lr, b1, b2, eps, decay, 0, rates, norm_and_factor, param, grad,
                      (void* const*) m, v, stream);
}

FSGS_API int fsgs_adamw8_update_multi(int n_tensors, int dtype, const int64_t* count, const double* step, const double* lr, double b1,
    double b2, const double* eps, const double* decay, uint32_t seed, const void* rates, const float* norm_and_factor,
    void* const* param, const void* const* grad, void* const* state, void* stream) {
  return adamw_update("adamw8", 8, n_tensors, dtype, count, step, lr, b1, b2, eps, decay, seed, rates, norm_and_factor, param, grad,
                      state, nullptr, stream);
}

FSGS_API int fsgs_adamw8_unpack_multi(int n_tensors, int dtype, const int64_t* count, const void* const* state, void* const* m,
                                      void* const* v, void* stream) {
  const char* what = "adamw8_moments";
  FSGS_REQUIRE(is_type(dtype), "%s: element type not supported", what);
  MomentsTable t{};
  if (const int rc = moments(what, n_tensors, count, state, m, v, type_size(dtype), 4096 / type_size(dtype), t)) return rc;
  if (t.first_block[t.n] == 0) return kOk;
  auto kernel = FSGS_BY_TYPE(adamw8_unpack_kernel, dtype, streams(n_tensors, count, 2 + 2 * type_size(dtype), kReadBackMiB));
  hipLaunchKernelGGL(kernel, dim3(t.first_block[t.n]), dim3(256), 0, (hipStream_t) stream, t);
  return check_launch(what);
}

FSGS_API int fsgs_adamw8_pack_multi(int n_tensors, const int64_t* count, const float* const* m, const float* const* v,
                                    void* const* state, void* stream) {
  const char* what = "adamw8_pack";
  MomentsTable t{};
  if (const int rc = moments(what, n_tensors, count, state, (const void* const*) m, (const void* const*) v, 4, 1024, t)) return rc;
  if (t.first_block[t.n] == 0) return kOk;
  hipLaunchKernelGGL(adamw8_pack_kernel, dim3(t.first_block[t.n]), dim3(256), 0, (hipStream_t) stream, t);
  return check_launch(what);
}
