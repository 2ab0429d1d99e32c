// Balance of an association: how evenly points spread over the M superpoints they may belong to, with gradients.
//
//   P_m = (1 / T) sum_n p_nm      mean weight of a superpoint over the T points that count
//   c_m                           how often a superpoint is chosen; f_m = c_m / sum c
//   loss = M sum_m f_m P_m        1 where both are even, M where one superpoint takes all; f carries no gradient
//
// Over logits [N, M]: p_n = softmax(logits_n), chosen are a point's K largest logits, the lowest index first among equals. A row of -inf
// alone, or one that the row mask leaves out, does not count; no entry of -inf is ever chosen. Over neighbour weights [N, K] with indices
// [N, K]: p_n is what the weights give, chosen is the neighbour of largest weight, the first among equals.
//
//   d loss / d logit_nj = p_nj (a_j - sum_m p_nm a_m),   d loss / d weight_nk = a_index[n,k],   a = (g_loss M f + g_P) / T
//
// The pass over the rows keeps a block's sums to itself (in registers, one column's in one lane; neighbour weights as integers in LDS, where
// the order of additions does not matter) and writes them once; a second launch adds the blocks' sums in a fixed order and forms
// the loss: equal calls give equal results.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "../../include/fsgs.h"
#include "common.hpp"

namespace fsgs {
namespace {

constexpr int kMostChoices   = 64;
constexpr int kRowBlocks     = 768;   // of the pass over logits
// Threads of its blocks, and wavefronts that share a SIMD's registers: with 64 values in each lane one has them to itself.
constexpr int row_threads(int vals) { return vals >= 32 ? 256 : 512; }
constexpr int row_waves(int vals) { return vals == 64 ? 1 : vals >= 16 ? 3 : 4; }
constexpr int kMostInLanes   = 4096;  // superpoints whose row is held by the lanes of one wavefront
constexpr int kNeighbourBlocks = 256;
constexpr int kNeighbourThreads = 1024;
constexpr int kMostInLds     = 5400;  // superpoints whose sums (8 bytes) and counts (4) of a block fit in 64 KB beside a few words
constexpr int kMostRanges    = 16;    // of so many superpoints, for each of which the weights are read again
constexpr int kSlopeThreads  = 512;   // of their backward
constexpr int kSlopeBlocks   = 1024;
constexpr int kMostSlopes    = 8192;  // that it keeps in LDS
constexpr float kLog2e       = 1.44269504f;
constexpr float kLowest      = -3.402823466e38f;

// What a block of a pass leaves: sums and counts of every superpoint, the rows that counted, whether something was no weight or no index.
struct BlockRows {
  int counted, invalid;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, float& y) { y = x; }
__device__ __forceinline__ void from_float(float x, __half& y) { y = __float2half(x); }
__device__ __forceinline__ void from_float(float x, __hip_bfloat16& y) { y = __float2bfloat16(x); }
template <typename T, int n>
struct alignas(n * sizeof(T)) Pack {
  T x[n];
};

__device__ __forceinline__ float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ uint32_t as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }

// ---- reductions over the kLanes lanes of a row; every one of them gets the result ----------------------------------------------
template <int kCtrl>
__device__ __forceinline__ int moved(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kCtrl, 0xf, 0xf, true);
}
// `none`: what f leaves its other argument as it is with
template <int kLanes, typename F>
__device__ __forceinline__ int over_lanes(int x, int none, F f) {
  x = f(x, moved<0xB1>(x)), x = f(x, moved<0x4E>(x));  // quad_perm: neighbours, then pairs of them
  if (kLanes >= 8) x = f(x, moved<0x141>(x));          // row_half_mirror
  if (kLanes >= 16) x = f(x, moved<0x140>(x));         // row_mirror
  if (kLanes == 64) {
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x142, 0xa, 0xf, false));  // row_bcast15: of 16 lanes to the next 16
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x143, 0xc, 0xf, false));  // row_bcast31: of 32 to the next
    x = __builtin_amdgcn_readlane(x, 63);
  }
  return x;
}
template <int kLanes>
__device__ __forceinline__ int row_max(int x) {
  return over_lanes<kLanes>(x, (int) 0x80000000, [](int a, int b) { return max(a, b); });
}
template <int kLanes>
__device__ __forceinline__ int row_min(int x) {
  return over_lanes<kLanes>(x, 0x7fffffff, [](int a, int b) { return min(a, b); });
}
template <int kLanes>
__device__ __forceinline__ int row_count(int x) {
  return over_lanes<kLanes>(x, 0, [](int a, int b) { return a + b; });
}
template <int kLanes>
__device__ __forceinline__ float row_sum(float x) {
  return as_float(over_lanes<kLanes>((int) as_uint(x), 0, [](int a, int b) { return (int) as_uint(as_float(a) + as_float(b)); }));
}
// Floats as integers of the same order (-0 directly below 0): their maximum takes one instruction with a lane's exchange, where that
// of floats quiets its operands first. It is its own inverse.
__device__ __forceinline__ int ordered(int bits) { return bits ^ ((bits >> 31) & 0x7fffffff); }
__device__ __forceinline__ int ordered(float x) { return ordered((int) as_uint(x)); }
__device__ __forceinline__ float unordered(int x) { return as_float((uint32_t) ordered(x)); }

// ---- rows of logits in the lanes of a wavefront ------------------------------------------------------------------------------------
// kLanes lanes have a row, kVals of its columns each, in pieces of 16 bytes: piece i of lane l begins at column (i kLanes + l) 16 / size.
template <typename T, int kLanes>
__device__ __forceinline__ int column(int lane, int j) {
  constexpr int kPiece = 16 / sizeof(T);
  return (j / kPiece * kLanes + lane) * kPiece + j % kPiece;
}
// How logits are read: element by element; in pieces, which are aligned and end where the row ends; in pieces past the caches.
enum Access { kSingle, kWhole, kStream };

// Element j of words as they lie in memory.
template <typename T>
__device__ __forceinline__ float element(const uint32_t* word, int j);
template <>
__device__ __forceinline__ float element<float>(const uint32_t* word, int j) { return as_float(word[j]); }
template <>
__device__ __forceinline__ float element<__hip_bfloat16>(const uint32_t* word, int j) {
  return as_float(j & 1 ? word[j / 2] & 0xffff0000u : word[j / 2] << 16);
}
template <>
__device__ __forceinline__ float element<__half>(const uint32_t* word, int j) {
  return (float) __builtin_bit_cast(_Float16, (uint16_t) (word[j / 2] >> (j & 1) * 16));
}

// A lane's part of a row as it lies in memory. A row that is not `on` is read where the first one is, a column that there is not where the
// row begins: no branch stands between the loads, so that they stay in flight while the row before is worked on. It is kept in words: the
// compiler would take elements of 16 bits apart as they arrive and put them into place again.
template <typename T, int kLanes, int kVals>
struct Row {
  static constexpr int kPiece = 16 / sizeof(T);
  uint32_t word[kVals * sizeof(T) / 4];

  template <Access kAccess>
  __device__ __forceinline__ void load(const T* __restrict__ row, int M, int lane) {
#pragma unroll
    for (int i = 0; i < kVals / kPiece; ++i) {
      const int c = column<T, kLanes>(lane, i * kPiece);
      typedef uint32_t Raw __attribute__((ext_vector_type(4)));
      Raw q;
      if (kAccess == kSingle) {
        typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type x[kPiece];
#pragma unroll
        for (int k = 0; k < kPiece; ++k) __builtin_memcpy(&x[k], row + (c + k < M ? c + k : 0), sizeof(T));
        q = __builtin_bit_cast(Raw, x);
      } else if (kAccess == kWhole) {
        q = *(const Raw*) (row + (c < M ? c : 0));
      } else {
        q = __builtin_nontemporal_load((const Raw*) (row + (c < M ? c : 0)));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) word[4 * i + k] = q[k];
    }
  }
  // -inf for what there is not; `full`: every lane has kVals columns
  template <Access kAccess>
  __device__ __forceinline__ void values(float x[kVals], int M, bool full, bool on, int lane) const {
#pragma unroll
    for (int j = 0; j < kVals; ++j) x[j] = element<T>(word, j);
    if (wave_ballot(!on)) {
#pragma unroll
      for (int j = 0; j < kVals; ++j) x[j] = on ? x[j] : -INFINITY;
    }
    if (full) return;
    const int l = keep_local(lane);
#pragma unroll
    for (int i = 0; i < kVals; i += kPiece) {
      if ((i / kPiece + 1) * kLanes * kPiece <= M) continue;  // of all lanes
#pragma unroll
      for (int k = 0; k < kPiece; ++k) x[i + k] = column<T, kLanes>(l, i + (kAccess == kSingle ? k : 0)) < M ? x[i + k] : -INFINITY;
    }
  }
};

// Counts the row's K largest values above -inf, the lowest column first among equals. `lane_top`: the largest of the lane, `top` of the row,
// ordered. The K-th largest of the lanes' own largest is reached by at least K values, and mostly by no other: 4 of 512 values lie
// in 4 of 64 lanes in 9 rows of 10. What reaches it is counted at once, in the columns' registers (a row that has the wavefront to itself is
// counted by the comparisons' lane masks). Where there are more, those equal to the threshold are taken back and the threshold rises to the
// next value, until K are left or fewer; then the first of the last ones taken back are counted after all, in LDS. Where the K-th value is
// nearer to the top than to the threshold, a walk down from the top comes first.
template <typename T, int kLanes, int kVals>
__device__ __forceinline__ void choose(const float x[kVals], int lane_top, int top, int K, int lane, int count[kVals], int* s_count) {
  const int lowest = ordered(-INFINITY);
  int t_ordered = top;
  for (int r = 1; r < K; ++r) t_ordered = row_max<kLanes>(lane_top < t_ordered ? lane_top : lowest);
  float t = unordered(max(t_ordered, ordered(kLowest)));
  int n = 0;
#pragma unroll
  for (int j = 0; j < kVals; ++j) {
    const bool hit = x[j] >= t;
    n += kLanes == 64 ? (int) __popcll(wave_ballot(hit)) : hit ? 1 : 0;
    // counted here and now, by an addition that takes the comparison as its carry
    count[j] = keep_local(count[j] + (hit ? 1 : 0));
  }
  if (kLanes != 64) n = row_count<kLanes>(n);
  if (!wave_ballot(n > K)) return;
  if (wave_ballot(n > 2 * K)) {
    const bool walk = n > 2 * K;
    const float counted = as_float((uint32_t) keep_local((int) as_uint(t)));  // or the comparisons' results are kept, in 64 scalar registers
    float s = unordered(top);
    for (int r = 1; r < K; ++r) {
      float below = -INFINITY;
#pragma unroll
      for (int j = 0; j < kVals; ++j) below = fmaxf(below, x[j] < s ? x[j] : -INFINITY);
      s = unordered(row_max<kLanes>(ordered(below)));
    }
    s = fmaxf(s, kLowest);
    int m = 0;
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
      const bool hit = x[j] >= s;
      m += kLanes == 64 ? (int) __popcll(wave_ballot(hit)) : hit ? 1 : 0;
      count[j] -= walk && x[j] >= counted && !hit ? 1 : 0;
    }
    if (kLanes != 64) m = row_count<kLanes>(m);
    if (walk) t = s, n = m;
  }
  int left = 0;  // to be chosen of the values equal to t
  while (wave_ballot(n > K)) {
    const float gone = n > K ? t : __builtin_nanf("");
    int equal = 0;
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
      const bool hit = x[j] == gone;
      equal += kLanes == 64 ? (int) __popcll(wave_ballot(hit)) : hit ? 1 : 0;
      count[j] = keep_local(count[j] - (hit ? 1 : 0));
    }
    if (kLanes != 64) equal = row_count<kLanes>(equal);
    const bool higher = n - equal > K;
    if (n > K && !higher) left = K - (n - equal);
    n = higher ? n - equal : 0;
    if (!wave_ballot(higher)) break;
    float above = INFINITY;
#pragma unroll
    for (int j = 0; j < kVals; ++j) above = fminf(above, x[j] > t ? x[j] : INFINITY);
    above = unordered(row_min<kLanes>(ordered(above)));
    if (higher) t = above;
  }
  if (kLanes == 64) {
    // columns rise with the piece, the lane, the value of the piece: over the comparisons' lane masks
    constexpr int kPiece = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kVals; i += kPiece) {
      if (left <= 0) break;
      unsigned long long equal[kPiece], any = 0;
#pragma unroll
      for (int k = 0; k < kPiece; ++k) equal[k] = wave_ballot(x[i + k] == t), any |= equal[k];
      for (; any && left > 0; any &= any - 1) {
        const int l = __builtin_ctzll(any);
#pragma unroll
        for (int k = 0; k < kPiece; ++k)
          if (((equal[k] >> l) & 1) && left > 0) {
            if (lane == 0) atomicAdd(&s_count[column<T, kLanes>(l, i + k)], 1);
            --left;
          }
      }
    }
    return;
  }
  for (int at = -1; wave_ballot(left > 0); --left) {
    const int l = keep_local(lane);  // or every column's index stays in a register of its own
    int where = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
      const int c = column<T, kLanes>(l, j);
      where = min(where, x[j] == t && c > at ? c : 0x7fffffff);
    }
    at = row_min<kLanes>(where);
    if (left > 0 && lane == 0) atomicAdd(&s_count[at], 1);
  }
}

// exp(x - shift) of the row's values. The shift's product with log2 e is rounded once for the whole row, a factor that the row's sum has too:
// one multiply-add a value. That factor is 2 to half an ulp of the product: within 2^(1/16) up to a shift of 2^20, beyond float32 from 2^32 on
// (2^440 in a row of -1e10). From 2^20 on the difference is taken first.
template <int kVals>
__device__ __forceinline__ void exponentials(float x[kVals], float shift) {
  const bool far = fabsf(shift) >= 0x1p20f;
  if (wave_ballot(far)) {
#pragma unroll
    for (int j = 0; j < kVals; ++j) x[j] = far ? x[j] - shift : x[j];
  }
  const float s = far ? 0.0f : shift * kLog2e;
#pragma unroll
  for (int j = 0; j < kVals; ++j) x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], kLog2e, -s));
}

// One pass: maximum, exponentials, their sum and the choice from registers, the next row's loads in flight meanwhile; a column's sum and count
// stay in the registers of the lane that reads it, for all rows of a wavefront. Vector instructions for each row: 127 of 512 float32 with 4
// chosen (300 000 x 512 105 - 122 us, 5.0 - 5.8 TB/s: memory), 142 of 512 bfloat16 (300 000 x 512 105 us, 2.9 TB/s, 0.9 of the cycles issue),
// 498 of 2000 bfloat16 with 8 chosen (400 000 x 2000 539 us, 3.0 TB/s, 0.7 of the cycles, three wavefronts a SIMD; one chosen 4.4 TB/s), 22
// of 64 bfloat16 (200 000 x 64 19 us, of 1M 52 us, 2.4 TB/s, 0.95 of the cycles). Rows that do not begin and end with pieces of 16 bytes take three
// times the loads: 300 000 x 501 161 - 174 us in float32, 158 - 167 in bfloat16.
template <typename T, int kLanes, int kVals, Access kAccess>
__global__ void __launch_bounds__(row_threads(kVals), row_waves(kVals)) balance_rows_kernel(int64_t N, int M, int64_t ld, int K,
    const T* __restrict__ logits, const uint8_t* __restrict__ rows, float2* __restrict__ stats, float* __restrict__ sums,
    int* __restrict__ counts, BlockRows* __restrict__ blocks, unsigned* __restrict__ ticket) {
  constexpr int kRows = 64 / kLanes, kThreads = row_threads(kVals), kWaves = kThreads / 64;
  __shared__ float s_sum[kLanes * kVals];
  __shared__ int s_count[kLanes * kVals];
  __shared__ int s_rows[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (kLanes - 1);
  const int group = kLanes == 64 ? 0 : (threadIdx.x & 63) / kLanes;
  const bool full = M == kLanes * kVals;
  float sum[kVals];
  int count[kVals], counted = 0;
#pragma unroll
  for (int j = 0; j < kVals; ++j) sum[j] = 0.0f, count[j] = 0;
  for (int c = threadIdx.x; c < kLanes * kVals; c += kThreads) s_count[c] = 0;
  __syncthreads();
  const int64_t step = (int64_t) gridDim.x * kWaves * kRows;
  int64_t base = ((int64_t) blockIdx.x * kWaves + wave) * kRows;

  // whether a row counts is known a row before its values are asked for, those a row before they are worked on
  auto mask_of = [&](int64_t row) { return rows ? (int) rows[row < N ? row : 0] : 1; };
  auto on_of = [&](int64_t row, int mask) { return row < N && mask != 0; };
  auto address = [&](int64_t row, bool on) { return logits + (on ? row : 0) * ld; };
  auto work = [&](const Row<T, kLanes, kVals>& row, int64_t at, bool on) {
    float x[kVals];
    row.template values<kAccess>(x, M, full, on, lane);
    float lane_top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVals; ++j) lane_top = fmaxf(lane_top, x[j]);
    // -0 becomes +0, to which it compares equal: as integers they would be two values, and the K-th of the lanes' largest, which sets the first
    // threshold, could lie above the K-th value of the row
    const int lane_top_ordered = ordered(lane_top + 0.0f), top_ordered = row_max<kLanes>(lane_top_ordered);
    choose<T, kLanes, kVals>(x, lane_top_ordered, top_ordered, K, lane, count, s_count);
    // a row without a number (top is -inf): the sum is 0, or NaN where one of its values is, which counts
    const float top = unordered(top_ordered), shift = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    exponentials<kVals>(x, shift);
#pragma unroll
    for (int j = 0; j < kVals; ++j) total += x[j];
    total = row_sum<kLanes>(total);
    const bool counts_in = !(total == 0.0f);
    const float scale = counts_in ? __builtin_amdgcn_rcpf(total) : 0.0f;
#pragma unroll
    for (int j = 0; j < kVals; ++j) sum[j] = fmaf(x[j], scale, sum[j]);
    if (lane == 0 && at < N) {
      if (stats) stats[at] = make_float2(shift, scale);
      counted += counts_in ? 1 : 0;
    }
  };
  Row<T, kLanes, kVals> a, b;
  bool on_a = on_of(base + group, mask_of(base + group)), on_b;
  int mask = mask_of(base + step + group);
  a.template load<kAccess>(address(base + group, on_a), M, lane);
  for (; base < N; base += 2 * step) {
    const int64_t at = base + group;
    on_b = on_of(at + step, mask);
    mask = mask_of(at + 2 * step);
    b.template load<kAccess>(address(at + step, on_b), M, lane);
    work(a, at, on_a);
    on_a = on_of(at + 2 * step, mask);
    mask = mask_of(at + 3 * step);
    a.template load<kAccess>(address(at + 2 * step, on_a), M, lane);
    if (base + step < N) work(b, at + step, on_b);
  }
  // the rows' groups of a wavefront, then the wavefronts one after the other
#pragma unroll
  for (int j = 0; j < kVals; ++j)
#pragma unroll
    for (int d = kLanes; d < 64; d <<= 1) sum[j] += __shfl_xor(sum[j], d), count[j] += __shfl_xor(count[j], d);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) counted += __shfl_xor(counted, d);
  if ((threadIdx.x & 63) == 0) s_rows[wave] = counted;
  __syncthreads();  // ties are counted
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave && group == 0)
#pragma unroll
      for (int j = 0; j < kVals; ++j) {
        const int c = column<T, kLanes>(lane, j);
        s_sum[c] = w ? s_sum[c] + sum[j] : sum[j], s_count[c] += count[j];
      }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < M; c += kThreads)
    sums[(size_t) blockIdx.x * M + c] = s_sum[c], counts[(size_t) blockIdx.x * M + c] = s_count[c];
  if (threadIdx.x == 0) {
    int all = 0;
    for (int w = 0; w < kWaves; ++w) all += s_rows[w];
    blocks[blockIdx.x] = BlockRows{all, 0};
    if (blockIdx.x == 0) *ticket = 0;
  }
}

// The access also of the gradient's rows. The weights are formed again from the row's shift and scale, 8 bytes a row: reading N M and writing
// N M is what bounds it. 300 000 x 512 float32 210 - 221 us (5.6 - 5.9 TB/s), 200 000 x 64 bfloat16 with a third of the rows left out 15 us. Element by
// element (rows that are not whole pieces) 300 000 x 501 takes 391 us, in bfloat16 334 (119 of 512).
template <typename T, int kLanes, int kVals, Access kAccess>
__global__ void __launch_bounds__(256) balance_rows_backward_kernel(int64_t N, int M, int64_t ld, const T* __restrict__ logits,
    const float2* __restrict__ stats, const int* __restrict__ counts, const int64_t* __restrict__ totals,
    const float* __restrict__ g_loss, const float* __restrict__ g_importance, T* __restrict__ grad) {
  constexpr int kRows = 64 / kLanes, kPiece = 16 / sizeof(T);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (kLanes - 1);
  const int group = kLanes == 64 ? 0 : (threadIdx.x & 63) / kLanes;
  const bool full = M == kLanes * kVals;
  const float rows = (float) max(totals[1], (int64_t) 1);
  const float of_counts = g_loss ? *g_loss * (float) M / (float) max(totals[0], (int64_t) 1) / rows : 0.0f;
  float slope[kVals];
#pragma unroll
  for (int j = 0; j < kVals; ++j) {
    const int c = column<T, kLanes>(lane, j);
    slope[j] = c < M ? of_counts * (float) counts[c] + (g_importance ? g_importance[c] / rows : 0.0f) : 0.0f;
  }
  // weights of 0 do not make 0 of slopes that are no numbers
  bool finite = true;
#pragma unroll
  for (int j = 0; j < kVals; ++j) finite = finite && fabsf(slope[j]) < INFINITY;
  const bool any_odd = wave_ballot(!finite) != 0;
  const int64_t step = (int64_t) gridDim.x * 4 * kRows;
  int64_t base = ((int64_t) blockIdx.x * 4 + wave) * kRows;

  // y is 0 in rows that did not count: they are not read
  auto stat_of = [&](int64_t row) { return stats[row < N ? row : 0]; };
  auto on_of = [&](int64_t row, float2 stat) { return row < N && !(stat.y == 0.0f); };
  auto address = [&](int64_t row, bool on) { return logits + (on ? row : 0) * ld; };
  auto work = [&](const Row<T, kLanes, kVals>& row, int64_t at, float2 stat) {
    const bool on = on_of(at, stat);
    float x[kVals], mean = 0.0f;
    row.template values<kAccess>(x, M, full, on, lane);
    exponentials<kVals>(x, stat.x);
#pragma unroll
    for (int j = 0; j < kVals; ++j) x[j] *= stat.y, mean = fmaf(x[j], slope[j], mean);
    mean = row_sum<kLanes>(mean);
    if (at >= N) return;
#pragma unroll
    for (int j = 0; j < kVals; ++j) x[j] *= slope[j] - mean;
    if (any_odd)
#pragma unroll
      for (int j = 0; j < kVals; ++j) x[j] = on ? x[j] : 0.0f;
    T* out = grad + at * M;
#pragma unroll
    for (int j = 0; j < kVals; j += kPiece) {
      const int c = column<T, kLanes>(lane, j);
      Pack<T, kPiece> q;
#pragma unroll
      for (int k = 0; k < kPiece; ++k) from_float(x[j + k], q.x[k]);
      if (kAccess == kStream) {
        typedef uint32_t Raw __attribute__((ext_vector_type(4)));
        if (c < M) __builtin_nontemporal_store(__builtin_bit_cast(Raw, q), (Raw*) (out + c));
      } else if (kAccess == kWhole) {
        if (c < M) *(Pack<T, kPiece>*) (out + c) = q;
      } else {
#pragma unroll
        for (int k = 0; k < kPiece; ++k)
          if (c + k < M) out[c + k] = q.x[k];
      }
    }
  };
  Row<T, kLanes, kVals> a, b;
  float2 stat_a = stat_of(base + group), stat_b = stat_of(base + step + group), after;
  a.template load<kAccess>(address(base + group, on_of(base + group, stat_a)), M, lane);
  for (; base < N; base += 2 * step) {
    const int64_t at = base + group;
    after = stat_of(at + 2 * step);
    b.template load<kAccess>(address(at + step, on_of(at + step, stat_b)), M, lane);
    work(a, at, stat_a);
    stat_a = after, after = stat_of(at + 3 * step);
    a.template load<kAccess>(address(at + 2 * step, on_of(at + 2 * step, stat_a)), M, lane);
    if (base + step < N) work(b, at + step, stat_b);
    stat_b = after;
  }
}

// ---- rows of more superpoints than a wavefront's lanes hold: a block a row ----------------------------------------------------------
// kPer: values of the row in each thread's registers, its columns' sums and counts beside them; 0: of more than 16 384 superpoints, read
// again for every step, the sums in memory. Most of the time goes to the 2 + 2 K reductions over the block, two barriers each (vector units 0.61 of
// the busy cycles, the rest waits): 20 000 x 5000 in float32, 4 chosen, 411 - 431 us forward and 551 - 571 with the backward (0.9 and 2.1
// TB/s), 1179 and 1484 read again by 256 threads; 2000 x 50 000 1154 and 1457.
constexpr int kWideThreads = 1024, kMostPer = 16;
template <typename F>
__device__ __forceinline__ int over_block(int x, int none, F f, int* s) {  // all threads get the result; as over_lanes
  x = over_lanes<64>(x, none, f);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  static_assert(kWideThreads / 64 == 16, "a row of lanes has a value of every wavefront");
  return __builtin_amdgcn_readfirstlane(over_lanes<16>(s[threadIdx.x & 15], none, f));
}
__device__ __forceinline__ float block_max(float x, int* s) {
  return unordered(over_block(ordered(x), (int) 0x80000000, [](int a, int b) { return max(a, b); }, s));
}
__device__ __forceinline__ float block_sum(float x, int* s) {
  return as_float(over_block((int) as_uint(x), 0, [](int a, int b) { return (int) as_uint(as_float(a) + as_float(b)); }, s));
}

// f(column, value, place) of the row's values that are this thread's; -inf for columns that there are not.
template <int kPer, typename T, typename F>
__device__ __forceinline__ void each_of_row(const T* __restrict__ row, const float* x, int M, F f) {
  if constexpr (kPer > 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) f((int) threadIdx.x + i * kWideThreads, x[i], i);
  } else {
    for (int c = threadIdx.x; c < M; c += kWideThreads) f(c, to_float(row[c]), 0);
  }
}
template <int kPer, typename T>
__device__ __forceinline__ void load_row(const T* __restrict__ row, float* x, int M) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = threadIdx.x + i * kWideThreads;
    const float value = to_float(row[c < M ? c : 0]);
    x[i] = c < M ? value : -INFINITY;
  }
}

template <typename T, int kPer>
__global__ void __launch_bounds__(kWideThreads) balance_wide_kernel(int64_t N, int M, int64_t ld, int K, const T* __restrict__ logits,
    const uint8_t* __restrict__ rows, float2* __restrict__ stats, float* __restrict__ sums, int* __restrict__ counts,
    BlockRows* __restrict__ blocks, unsigned* __restrict__ ticket) {
  constexpr int kHeld = kPer > 0 ? kPer : 1;
  __shared__ int s_part[kWideThreads / 64];
  // a column's sums belong to one thread
  float *sum = sums + (size_t) blockIdx.x * M, held_sum[kHeld], x[kHeld] = {};
  int *count = counts + (size_t) blockIdx.x * M, held_count[kHeld], counted = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held_sum[i] = 0.0f, held_count[i] = 0;
  if (kPer == 0)
    for (int c = threadIdx.x; c < M; c += kWideThreads) sum[c] = 0.0f, count[c] = 0;
  for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
    const T* row = logits + n * ld;
    const bool on = !rows || rows[n];
    float top = -INFINITY, total = 0.0f;
    if (on) {
      load_row<kPer>(row, x, M);
      each_of_row<kPer>(row, x, M, [&](int, float y, int) { top = fmaxf(top, y); });
      top = block_max(top, s_part);
    }
    const float shift = top == -INFINITY ? 0.0f : top;
    const auto power = [&](float y) { return __builtin_amdgcn_exp2f((y - shift) * kLog2e); };
    if (on) {
      each_of_row<kPer>(row, x, M, [&](int, float y, int) { total += power(y); });
      total = block_sum(total, s_part);
    }
    const bool counts_in = !(total == 0.0f);
    const float scale = counts_in ? 1.0f / total : 0.0f;
    if (threadIdx.x == 0 && stats) stats[n] = make_float2(shift, scale);
    if (!counts_in) continue;
    ++counted;
    each_of_row<kPer>(row, x, M, [&](int c, float y, int i) {
      if constexpr (kPer > 0) held_sum[i] = fmaf(power(y), scale, held_sum[i]);
      else sum[c] = fmaf(power(y), scale, sum[c]);
    });
    float value = INFINITY;
    int at = 0;
    for (int r = 0; r < K; ++r) {
      float best = -INFINITY;
      int where = 0x7fffffff;
      each_of_row<kPer>(row, x, M, [&](int c, float y, int) {
        const bool after = r == 0 || y < value || (y == value && c > at);
        if (after && y > best) best = y, where = c;
      });
      const float most = block_max(best, s_part);
      if (!(most > -INFINITY)) break;
      at = over_block(best == most ? where : 0x7fffffff, 0x7fffffff, [](int a, int b) { return min(a, b); }, s_part);
      value = most;
      if constexpr (kPer > 0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) held_count[i] += at == (int) threadIdx.x + i * kWideThreads ? 1 : 0;
      } else if (at % kWideThreads == (int) threadIdx.x) {
        ++count[at];
      }
    }
  }
  if constexpr (kPer > 0)
    each_of_row<kPer>(logits, x, M, [&](int c, float, int i) {
      if (c < M) sum[c] = held_sum[i], count[c] = held_count[i];
    });
  if (threadIdx.x == 0) {
    blocks[blockIdx.x] = BlockRows{counted, 0};
    if (blockIdx.x == 0) *ticket = 0;
  }
}

template <typename T, int kPer>
__global__ void __launch_bounds__(kWideThreads) balance_wide_backward_kernel(int64_t N, int M, int64_t ld, const T* __restrict__ logits,
    const float2* __restrict__ stats, const int* __restrict__ counts, const int64_t* __restrict__ totals,
    const float* __restrict__ g_loss, const float* __restrict__ g_importance, T* __restrict__ grad) {
  constexpr int kHeld = kPer > 0 ? kPer : 1;
  __shared__ int s_part[kWideThreads / 64];
  const float of_rows = (float) max(totals[1], (int64_t) 1);
  const float of_counts = g_loss ? *g_loss * (float) M / (float) max(totals[0], (int64_t) 1) / of_rows : 0.0f;
  auto slope_of = [&](int c) { return of_counts * (float) counts[c] + (g_importance ? g_importance[c] / of_rows : 0.0f); };
  float slope[kHeld], x[kHeld] = {};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = threadIdx.x + i * kWideThreads;
    slope[i] = c < M ? slope_of(c) : 0.0f;
  }
  auto slope_at = [&](int c, int i) { return kPer > 0 ? slope[i] : slope_of(c); };
  for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
    const float2 stat = stats[n];
    const T* row = logits + n * ld;
    T* out = grad + n * M;
    if (stat.y == 0.0f) {  // did not count, and is not read
      for (int c = threadIdx.x; c < M; c += kWideThreads) from_float(0.0f, out[c]);
      continue;
    }
    auto weight = [&](float y) { return __builtin_amdgcn_exp2f((y - stat.x) * kLog2e) * stat.y; };
    load_row<kPer>(row, x, M);
    float mean = 0.0f;
    each_of_row<kPer>(row, x, M, [&](int c, float y, int i) { mean = fmaf(weight(y), slope_at(c, i), mean); });
    mean = block_sum(mean, s_part);
    each_of_row<kPer>(row, x, M, [&](int c, float y, int i) {
      if (c < M) from_float(weight(y) * (slope_at(c, i) - mean), out[c]);
    });
  }
}

// ---- neighbour weights ----------------------------------------------------------------------------------------------------------------
// Weights lie in [0, 1] (roundings above 1 are let pass, up to kMostWeight): in units of 2^-31 a block's sums are integers of 64 bits. A weight that
// is none, or an index that is none, is reported and left out.
constexpr float kWeightUnits = 2147483648.0f;
constexpr float kMostWeight = 1.0001f;  // its units fit in 32 bits

// A thread takes a row, four neighbours at a time: all loads of four are on their way before the first is looked at. kQuads: K is a
// multiple of four and the addresses allow 16 bytes. A block keeps the superpoints of one range in LDS (blockIdx.y); beyond kMostRanges of
// them the sums are global ones (kLds false). 3M points with 8 neighbours, us: 72 with 2048 superpoints, 109 if all are one and the same;
// with 8000, in two ranges, 96 and 205, by global atomics 1030 and 288 000; with 86 000 in 16 ranges 514 and 1580. Of the 69 us of a pass over
// 288 MB (4.2 TB/s) what is above the copy rate is LDS atomics, one a neighbour and one a point; 512 blocks instead of 256 were slower.
template <bool kLds, bool kQuads>
__global__ void __launch_bounds__(kNeighbourThreads) balance_neighbours_kernel(int64_t N, int M, int K,
    const float* __restrict__ weights, const int64_t* __restrict__ indices, const uint8_t* __restrict__ rows,
    unsigned long long* __restrict__ sums, int* __restrict__ counts, BlockRows* __restrict__ blocks, unsigned* __restrict__ ticket) {
  extern __shared__ unsigned long long s_sums[];  // [M], then the counts [M]
  __shared__ int s_rows[2];
  const int first = kLds ? blockIdx.y * kMostInLds : 0, in_range = kLds ? min(M - first, kMostInLds) : M;
  unsigned long long* sum = kLds ? s_sums : sums;
  int* count = kLds ? (int*) (s_sums + in_range) : counts;
  if (kLds)
    for (int c = threadIdx.x; c < in_range; c += kNeighbourThreads) sum[c] = 0, count[c] = 0;
  if (threadIdx.x < 2) s_rows[threadIdx.x] = 0;
  __syncthreads();
  int counted = 0, invalid = 0;
  for (int64_t n = (int64_t) blockIdx.x * kNeighbourThreads + threadIdx.x; n < N; n += (int64_t) gridDim.x * kNeighbourThreads) {
    if (rows && !rows[n]) continue;
    ++counted;
    float best = -1.0f;
    int where = 0;
    const float* row_w     = weights + n * K;
    const int64_t* row_i = indices + n * K;
    for (int k = 0; k < K; k += 4) {
      float w[4];
      int64_t m[4];
      if (kQuads) {
        const float4 q = *(const float4*) (row_w + k);
        const longlong2 i = *(const longlong2*) (row_i + k), j = *(const longlong2*) (row_i + k + 2);
        w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
        m[0] = i.x, m[1] = i.y, m[2] = j.x, m[3] = j.y;
      } else {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int at = min(k + d, K - 1);
          w[d] = row_w[at], m[d] = row_i[at];
        }
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if (!kQuads && k + d >= K) continue;
        const bool valid = w[d] >= 0.0f && w[d] <= kMostWeight && (uint64_t) m[d] < (uint64_t) M;
        if (!valid) {
          invalid = 1;
          continue;
        }
        const unsigned at = (unsigned) ((int) m[d] - first);
        if (at < (unsigned) in_range) atomicAdd(&sum[at], (unsigned long long) __float2uint_rn(w[d] * kWeightUnits));
        if (w[d] > best) best = w[d], where = (int) m[d];
      }
    }
    if (best >= 0.0f && (unsigned) (where - first) < (unsigned) in_range) atomicAdd(&count[where - first], 1);
  }
  if (counted) atomicAdd(&s_rows[0], counted);
  if (invalid) atomicOr(&s_rows[1], 1);
  __syncthreads();
  if (kLds)
    for (int c = threadIdx.x; c < in_range; c += kNeighbourThreads)
      sums[(size_t) blockIdx.x * M + first + c] = sum[c], counts[(size_t) blockIdx.x * M + first + c] = count[c];
  if (threadIdx.x == 0 && blockIdx.y == 0) {
    blocks[blockIdx.x] = BlockRows{s_rows[0], s_rows[1]};
    if (blockIdx.x == 0) *ticket = 0;
  }
}

// A thread takes four pairs. kLds: the slopes of all superpoints lie in LDS, which answers 64 lanes' addresses at once where the cache
// takes them line by line. 24M pairs, 288 MB, 47 us (6.1 TB/s).
template <bool kLds>
__global__ void __launch_bounds__(kSlopeThreads) balance_neighbours_backward_kernel(int64_t N, int M, int K,
    const int64_t* __restrict__ indices, const uint8_t* __restrict__ rows, const int* __restrict__ counts,
    const int64_t* __restrict__ totals, const float* __restrict__ g_loss, const float* __restrict__ g_importance,
    float* __restrict__ grad) {
  extern __shared__ float s_slope[];
  const float of_rows = (float) max(totals[1], (int64_t) 1);
  const float of_counts = g_loss ? *g_loss * (float) M / (float) max(totals[0], (int64_t) 1) / of_rows : 0.0f;
  auto slope = [&](int m) { return of_counts * (float) counts[m] + (g_importance ? g_importance[m] / of_rows : 0.0f); };
  if (kLds) {
    for (int m = threadIdx.x; m < M; m += kSlopeThreads) s_slope[m] = slope(m);
    __syncthreads();
  }
  const bool aligned = (((uintptr_t) indices | (uintptr_t) grad) & 15) == 0;
  const double per_row = 1.0 / (double) K;
  const int64_t pairs = N * K;
  for (int64_t e = ((int64_t) blockIdx.x * kSlopeThreads + threadIdx.x) * 4; e < pairs; e += (int64_t) gridDim.x * kSlopeThreads * 4) {
    const bool whole = aligned && e + 4 <= pairs;
    int64_t m[4];
    if (whole) {
      const longlong2 i = *(const longlong2*) (indices + e), j = *(const longlong2*) (indices + e + 2);
      m[0] = i.x, m[1] = i.y, m[2] = j.x, m[3] = j.y;
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d) m[d] = indices[min(e + d, pairs - 1)];
    }
    bool on[4] = {true, true, true, true};
    if (rows) {
      // the row of the first pair: the product is off by one at most, pairs being fewer than 2^53
      int64_t row = (int64_t) ((double) e * per_row);
      int k = (int) (e - row * K);
      if (k < 0) --row, k += K;
      if (k >= K) ++row, k -= K;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        on[d] = rows[min(row, N - 1)] != 0;
        if (++k == K) k = 0, ++row;
      }
    }
    float g[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const bool valid = (uint64_t) m[d] < (uint64_t) M;
      const int at = valid && on[d] ? (int) m[d] : 0;
      const float a = kLds ? s_slope[at] : slope(at);
      g[d] = !on[d] ? 0.0f : valid ? a : __builtin_nanf("");
    }
    if (whole) {
      *(float4*) (grad + e) = make_float4(g[0], g[1], g[2], g[3]);
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (e + d < pairs) grad[e + d] = g[d];
    }
  }
}

__global__ void __launch_bounds__(256) clear_kernel(int M, unsigned long long* sums, int* counts) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < M) sums[c] = 0, counts[c] = 0;
}

// ---- the blocks' sums together -----------------------------------------------------------------------------------------------------------
// A block takes 16 superpoints, 64 threads of it a superpoint's blocks in turn; the last block to end forms the loss of all of them. 5 to 10
// us: the launch, loads of two arrays by 64 threads in turn, a fence and a ticket.
constexpr int kTotalColumns = 16;
__device__ __forceinline__ double value_of(float s) { return (double) s; }
__device__ __forceinline__ double value_of(unsigned long long s) { return (double) s * (1.0 / kWeightUnits); }
__device__ __forceinline__ double added(double a, float s) { return a + (double) s; }
__device__ __forceinline__ unsigned long long added(unsigned long long a, unsigned long long s) { return a + s; }
template <typename S> struct TotalOf { using type = double; };
template <> struct TotalOf<unsigned long long> { using type = unsigned long long; };
__device__ __forceinline__ double value_of(double s) { return s; }

template <typename S>
__global__ void __launch_bounds__(1024) balance_totals_kernel(int G, int G_rows, int M, const S* __restrict__ sums,
    const int* __restrict__ block_counts, const BlockRows* __restrict__ blocks, double* __restrict__ parts, unsigned* __restrict__ ticket,
    float* __restrict__ loss, int* __restrict__ counts, float* __restrict__ importance, int64_t* __restrict__ totals) {
  using Total = typename TotalOf<S>::type;
  constexpr int kSlices = 1024 / kTotalColumns, kWaves = 16;
  static_assert(kTotalColumns == 16 && kSlices == 4 * kWaves, "a wavefront has four slices of 16 columns");
  __shared__ Total s_sum[kWaves][kTotalColumns];
  __shared__ int s_count[kWaves][kTotalColumns], s_rows[kWaves], s_invalid[kWaves], s_last;
  const int c = threadIdx.x % kTotalColumns, slice = threadIdx.x / kTotalColumns, m = blockIdx.x * kTotalColumns + c;
  const int wave = threadIdx.x >> 6;
  int rows = 0, invalid = 0, count = 0;
  for (int g = threadIdx.x; g < G_rows; g += 1024) rows += blocks[g].counted, invalid |= blocks[g].invalid;
  Total sum = 0;
  if (m < M)
#pragma unroll 8
    for (int g = slice; g < G; g += kSlices) sum = added(sum, sums[(size_t) g * M + m]), count += block_counts[(size_t) g * M + m];
  // in a fixed order: the slices of a wavefront, then the wavefronts
#pragma unroll
  for (int d = 16; d < 64; d <<= 1) sum += __shfl_xor(sum, d), count += __shfl_xor(count, d);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) rows += __shfl_xor(rows, d), invalid |= __shfl_xor(invalid, d);
  if ((threadIdx.x & 63) < kTotalColumns) s_sum[wave][c] = sum, s_count[wave][c] = count;
  if ((threadIdx.x & 63) == 0) s_rows[wave] = rows, s_invalid[wave] = invalid;
  __syncthreads();
  int T = 0, any_invalid = 0;
  for (int w = 0; w < kWaves; ++w) T += s_rows[w], any_invalid |= s_invalid[w];
  const int of = max(T, 1);
  if (wave == 0) {  // the block's share of the loss
    double chosen = 0.0, both = 0.0;
    if (slice == 0 && m < M) {
      sum = 0, count = 0;
      for (int w = 0; w < kWaves; ++w) sum += s_sum[w][c], count += s_count[w][c];
      const double s = any_invalid ? __builtin_nan("") : value_of(sum);
      counts[m] = count, importance[m] = (float) (s / of);
      chosen = (double) count, both = chosen * s;
    }
#pragma unroll
    for (int d = kTotalColumns / 2; d; d >>= 1) chosen += __shfl_xor(chosen, d), both += __shfl_xor(both, d);
    if (threadIdx.x == 0) {
      parts[2 * blockIdx.x] = chosen, parts[2 * blockIdx.x + 1] = both;
      __threadfence();
      s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!s_last || wave != 0) return;
  __threadfence();
  double chosen = 0.0, both = 0.0;
  for (int b = threadIdx.x; b < (int) gridDim.x; b += 64)
    chosen += __builtin_nontemporal_load(parts + 2 * b), both += __builtin_nontemporal_load(parts + 2 * b + 1);
#pragma unroll
  for (int d = 32; d; d >>= 1) chosen += __shfl_xor(chosen, d), both += __shfl_xor(both, d);
  if (threadIdx.x == 0) {
    *loss = (float) ((double) M * both / ((chosen > 0.0 ? chosen : 1.0) * (double) of));
    totals[0] = (int64_t) chosen, totals[1] = T;
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------------
struct Workspace {
  size_t counts, blocks, parts, ticket, bytes;  // sums come first
  Workspace(int G, int64_t M, size_t sum_bytes, int G_rows) {
    counts = align_up((size_t) G * M * sum_bytes, 256);
    blocks = counts + align_up((size_t) G * M * 4, 256);
    parts  = blocks + align_up((size_t) G_rows * sizeof(BlockRows), 256);
    ticket = parts + align_up((size_t) div_up(M, kTotalColumns) * 16, 256);
    bytes  = ticket + 256;
  }
};

// Lanes that have a row: the fewest of 4, 8 and 16 that hold it in a piece of 16 bytes each, 16 with two pieces, or 64 and as many as it takes.
int lanes_of(int M, int piece) { return M <= 4 * piece ? 4 : M <= 8 * piece ? 8 : M <= 32 * piece ? 16 : 64; }
int pass_blocks(int64_t N, int M, int dtype) {
  if (N == 0) return 0;
  // two rows for a wavefront's lanes, which ask for both at once. With one the blocks' sums are more: 20 000 x 64 in bf16 12.8 us against
  // 11.1 with both launches, 10 000 x 512 16.1 against 15.4 (500 x 512 9.7 against 10.2); with four 12.4, 15.2 and 11.8.
  const int rows = M > kMostInLanes ? 1 : 2 * row_threads(M > 1024 ? 32 : 16) / lanes_of(M, dtype == FSGS_DTYPE_F32 ? 4 : 8);
  const int64_t blocks = (N + rows - 1) / rows;
  // sums and counts of M superpoints for each block: 256 MB of them at most, or what 32 blocks take
  const int64_t most = std::min<int64_t>(kRowBlocks, std::max<int64_t>(32, ((int64_t) 1 << 25) / M));
  return (int) std::min(blocks, most);
}
bool in_lds(int64_t M) { return M <= (int64_t) kMostRanges * kMostInLds; }
int neighbour_blocks(int64_t N, int64_t M) {
  const int64_t blocks = (N + kNeighbourThreads - 1) / kNeighbourThreads;
  const int64_t ranges = in_lds(M) ? (M + kMostInLds - 1) / kMostInLds : 1;
  return (int) std::min(blocks, kNeighbourBlocks / ranges);
}

// Logits that exceed the 256 MB memory-side cache are read past it, and their gradients written past it, where a row is made of whole lines of
// 128 bytes or is long: of lines that two wavefronts share, streaming moves the halves apart. us of forward and backward, ordinary and
// streaming: float32 320 000 x 512 419 and 367, 1M x 128 341 and 314, 500 000 x 256 360 and 347, 80 000 x 1000 212 and 202, bfloat16 2M x 128
// 451 and 439; but float32 1M x 100 280 and 320, 600 000 x 200 360 and 376, 500 000 x 300 417 and 444, bfloat16 400 000 x 1000 564 and 576.
// Rows of 32 values a lane and more are bound by their registers and read either way as fast (100 000 x 2000 173 us both).
bool past_caches(int64_t N, int M, size_t size) {
  const int64_t row = (int64_t) (M * size);
  return N >= ((int64_t) 160 << 20) / row && (row % 128 == 0 || row > 2048);
}

// kernel<T, lanes, values>(...) for the narrowest rows that hold M columns
#define FSGS_ROW_KERNELS(T, LAUNCH)                         \
  do {                                                      \
    constexpr int kPiece = 16 / sizeof(T);                  \
    if (M <= 4 * kPiece) LAUNCH(T, 4, kPiece);              \
    else if (M <= 8 * kPiece) LAUNCH(T, 8, kPiece);         \
    else if (M <= 16 * kPiece) LAUNCH(T, 16, kPiece);       \
    else if (M <= 32 * kPiece) LAUNCH(T, 16, 2 * kPiece);   \
    else if (M <= 64 * kPiece) LAUNCH(T, 64, kPiece);       \
    else if (M <= 512) LAUNCH(T, 64, 8);                    \
    else if (M <= 1024) LAUNCH(T, 64, 16);                  \
    else if (M <= 2048) LAUNCH(T, 64, 32);                  \
    else LAUNCH(T, 64, 64);                                 \
  } while (0)

template <typename T>
void launch_rows(int G, int64_t N, int M, int64_t ld, int K, const void* logits, const uint8_t* rows, float2* stats, float* sums,
                 int* counts, BlockRows* blocks, unsigned* ticket, hipStream_t s) {
  const T* x = (const T*) logits;
  if (M > kMostInLanes) {
    hipLaunchKernelGGL((M <= 8 * kWideThreads          ? balance_wide_kernel<T, 8>
                        : M <= kMostPer * kWideThreads ? balance_wide_kernel<T, kMostPer>
                                                       : balance_wide_kernel<T, 0>),
                       dim3(G), dim3(kWideThreads), 0, s, N, M, ld, K, x, rows, stats, sums, counts, blocks, ticket);
    return;
  }
  const bool whole = M % (16 / sizeof(T)) == 0 && ld * sizeof(T) % 16 == 0 && (uintptr_t) logits % 16 == 0;
#define LAUNCH(T, L, V)                                                                                                               \
  hipLaunchKernelGGL((!whole ? balance_rows_kernel<T, L, V, kSingle>                                                                  \
                      : past_caches(N, M, sizeof(T)) ? balance_rows_kernel<T, L, V, V < 32 ? kStream : kWhole>                        \
                                                     : balance_rows_kernel<T, L, V, kWhole>),                                         \
                     dim3(G), dim3(row_threads(V)), 0, s, N, M, ld, K, x, rows, stats, sums, counts, blocks, ticket)
  FSGS_ROW_KERNELS(T, LAUNCH);
#undef LAUNCH
}

template <typename T>
void launch_rows_backward(int G, int64_t N, int M, int64_t ld, const void* logits, const float2* stats, const int* counts,
                          const int64_t* totals, const float* g_loss, const float* g_importance, void* grad, hipStream_t s) {
  const T* x = (const T*) logits;
  T* out = (T*) grad;
  if (M > kMostInLanes) {
    hipLaunchKernelGGL((M <= 8 * kWideThreads          ? balance_wide_backward_kernel<T, 8>
                        : M <= kMostPer * kWideThreads ? balance_wide_backward_kernel<T, kMostPer>
                                                       : balance_wide_backward_kernel<T, 0>),
                       dim3(G), dim3(kWideThreads), 0, s, N, M, ld, x, stats, counts, totals, g_loss,
                       g_importance, out);
    return;
  }
  const bool whole = M % (16 / sizeof(T)) == 0 && ld * sizeof(T) % 16 == 0 && ((uintptr_t) logits | (uintptr_t) grad) % 16 == 0;
#define LAUNCH(T, L, V)                                                                                                             \
  hipLaunchKernelGGL((!whole ? balance_rows_backward_kernel<T, L, V, kSingle>                                                       \
                      : past_caches(N, M, sizeof(T)) ? balance_rows_backward_kernel<T, L, V, V < 32 ? kStream : kWhole>             \
                                                     : balance_rows_backward_kernel<T, L, V, kWhole>),                              \
                     dim3(G), dim3(256), 0, s, N, M, ld, x, stats, counts, totals, g_loss, g_importance, out)
  FSGS_ROW_KERNELS(T, LAUNCH);
#undef LAUNCH
}
#undef FSGS_ROW_KERNELS

// The totals' launch has 1024 threads for 16 superpoints, and a launch fewer than 2^32 threads.
constexpr int kMostSuperpoints = (1 << 26) - 16;
// Sums of weights have 64 bits, 31 of them below the point.
constexpr int64_t kMostPairs = ((int64_t) 1 << 33) - 1;

bool is_type(int type) { return type == FSGS_DTYPE_F32 || type == FSGS_DTYPE_F16 || type == FSGS_DTYPE_BF16; }

}  // namespace
}  // namespace fsgs

using namespace fsgs;

FSGS_API int fsgs_balance_max_choices(void) { return kMostChoices; }
FSGS_API int fsgs_balance_max_superpoints(void) { return kMostSuperpoints; }

FSGS_API size_t fsgs_balance_loss_workspace_bytes(int64_t N, int M, int dtype) {
  if (N < 0 || M <= 0) return 0;
  const int G = pass_blocks(N, M, dtype);
  return Workspace(G, M, 4, G).bytes;
}

FSGS_API int fsgs_balance_loss_forward(int64_t N, int M, int64_t ld, int K, int dtype, const void* logits, const uint8_t* rows,
    float* loss, int32_t* counts, float* importance, int64_t* totals, float* stats, void* workspace, size_t workspace_bytes,
    void* stream) {
  const char* what = "balance_loss";
  FSGS_REQUIRE(N >= 0 && N < (int64_t) 0x7fffffff && M > 0 && is_type(dtype) && (N <= 1 || ld >= M), "%s: bad arguments", what);
  FSGS_REQUIRE(M <= kMostSuperpoints, "%s: more than %d superpoints", what, kMostSuperpoints);
  FSGS_REQUIRE(K >= 1 && K <= M && K <= kMostChoices, "%s: K must be in [1, min(M, %d)]", what, kMostChoices);
  FSGS_REQUIRE((N == 0 || logits) && loss && counts && importance && totals && workspace, "%s: null pointer", what);
  FSGS_REQUIRE((uintptr_t) logits % (dtype == FSGS_DTYPE_F32 ? 4 : 2) == 0 && (uintptr_t) stats % 8 == 0 && (uintptr_t) workspace % 8 == 0,
               "%s: misaligned address", what);
  const int G = pass_blocks(N, M, dtype);
  const Workspace ws(G, M, 4, G);
  if (workspace_bytes < ws.bytes) return fsgs::fail(kWorkspaceSmall, "%s: the workspace is too small", what);
  char* at = (char*) workspace;
  float* sums = (float*) at;
  int* block_counts = (int*) (at + ws.counts);
  BlockRows* blocks = (BlockRows*) (at + ws.blocks);
  unsigned* ticket = (unsigned*) (at + ws.ticket);
  hipStream_t s = (hipStream_t) stream;
  if (G == 0) {
    hipLaunchKernelGGL(clear_kernel, dim3(1), dim3(256), 0, s, 1, (unsigned long long*) ticket, (int*) ticket + 2);
  } else {
    auto launch = dtype == FSGS_DTYPE_F32 ? launch_rows<float> : dtype == FSGS_DTYPE_F16 ? launch_rows<__half> : launch_rows<__hip_bfloat16>;
    launch(G, N, M, ld, K, logits, rows, (float2*) stats, sums, block_counts, blocks, ticket, s);
  }
  if (const int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(balance_totals_kernel<float>, dim3(div_up(M, kTotalColumns)), dim3(1024), 0, s, G, G, M, sums, block_counts, blocks,
                     (double*) (at + ws.parts), ticket, loss, counts, importance, totals);
  return check_launch(what);
}

FSGS_API int fsgs_balance_loss_backward(int64_t N, int M, int64_t ld, int dtype, const void* logits, const float* stats,
    const int32_t* counts, const int64_t* totals, const float* g_loss, const float* g_importance, void* grad, void* stream) {
  const char* what = "balance_loss_backward";
  FSGS_REQUIRE(N >= 0 && N < (int64_t) 0x7fffffff && M > 0 && is_type(dtype) && (N <= 1 || ld >= M), "%s: bad arguments", what);
  if (N == 0) return kOk;
  FSGS_REQUIRE(logits && stats && counts && totals && grad && (g_loss || g_importance), "%s: null pointer", what);
  const size_t size = dtype == FSGS_DTYPE_F32 ? 4 : 2;
  FSGS_REQUIRE(((uintptr_t) logits | (uintptr_t) grad) % size == 0 && (uintptr_t) stats % 8 == 0, "%s: misaligned address", what);
  // four rows in turn at least for a wavefront, which has its columns' slopes to form first
  const int rows = M > kMostInLanes ? 1 : 16 * (64 / lanes_of(M, (int) (16 / size)));
  const int64_t blocks = (N + rows - 1) / rows;
  const int G = (int) (blocks < 4096 ? blocks : 4096);
  auto launch = dtype == FSGS_DTYPE_F32 ? launch_rows_backward<float> : dtype == FSGS_DTYPE_F16 ? launch_rows_backward<__half> : launch_rows_backward<__hip_bfloat16>;
  launch(G, N, M, ld, logits, (const float2*) stats, counts, totals, g_loss, g_importance, grad, (hipStream_t) stream);
  return check_launch(what);
}

FSGS_API size_t fsgs_neighbour_balance_workspace_bytes(int64_t N, int M) {
  if (N < 0 || M <= 0) return 0;
  const int G = neighbour_blocks(N, M);
  return Workspace(in_lds(M) ? G : 1, M, 8, G).bytes;
}

FSGS_API int fsgs_neighbour_balance_forward(int64_t N, int M, int K, const float* weights, const int64_t* indices, const uint8_t* rows,
    float* loss, int32_t* counts, float* importance, int64_t* totals, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "neighbour_balance";
  FSGS_REQUIRE(N >= 0 && N < (int64_t) 0x7fffffff && M > 0 && K >= 1, "%s: bad arguments", what);
  FSGS_REQUIRE(M <= kMostSuperpoints, "%s: more than %d superpoints", what, kMostSuperpoints);
  FSGS_REQUIRE(N * K <= kMostPairs, "%s: more than %lld pairs of points and neighbours", what, (long long) kMostPairs);
  FSGS_REQUIRE((N == 0 || (weights && indices)) && loss && counts && importance && totals && workspace, "%s: null pointer", what);
  FSGS_REQUIRE((uintptr_t) weights % 4 == 0 && (uintptr_t) indices % 8 == 0 && (uintptr_t) workspace % 8 == 0, "%s: misaligned address", what);
  const int G = neighbour_blocks(N, M), G_sums = in_lds(M) ? G : 1;
  const Workspace ws(G_sums, M, 8, G);
  if (workspace_bytes < ws.bytes) return fsgs::fail(kWorkspaceSmall, "%s: the workspace is too small", what);
  char* at = (char*) workspace;
  unsigned long long* sums = (unsigned long long*) at;
  int* block_counts = (int*) (at + ws.counts);
  BlockRows* blocks = (BlockRows*) (at + ws.blocks);
  unsigned* ticket = (unsigned*) (at + ws.ticket);
  hipStream_t s = (hipStream_t) stream;
  if (!in_lds(M)) hipLaunchKernelGGL(clear_kernel, dim3(div_up(M, 256)), dim3(256), 0, s, M, sums, block_counts);
  if (G == 0)
    hipLaunchKernelGGL(clear_kernel, dim3(1), dim3(256), 0, s, 1, (unsigned long long*) ticket, (int*) ticket + 2);
  else {
    const bool quads = K % 4 == 0 && ((uintptr_t) weights | (uintptr_t) indices) % 16 == 0;
    auto kernel = in_lds(M) ? (quads ? balance_neighbours_kernel<true, true> : balance_neighbours_kernel<true, false>)
                            : (quads ? balance_neighbours_kernel<false, true> : balance_neighbours_kernel<false, false>);
    const dim3 grid(G, in_lds(M) ? div_up(M, kMostInLds) : 1);
    hipLaunchKernelGGL(kernel, grid, dim3(kNeighbourThreads), in_lds(M) ? (size_t) std::min(M, kMostInLds) * 12 : 0, s, N, M, K, weights,
                       indices, rows, sums, block_counts, blocks, ticket);
  }
  if (const int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(balance_totals_kernel<unsigned long long>, dim3(div_up(M, kTotalColumns)), dim3(1024), 0, s, G_sums, G, M, sums, block_counts,
                     blocks, (double*) (at + ws.parts), ticket, loss, counts, importance, totals);
  return check_launch(what);
}

FSGS_API int fsgs_neighbour_balance_backward(int64_t N, int M, int K, const int64_t* indices, const uint8_t* rows,
    const int32_t* counts, const int64_t* totals, const float* g_loss, const float* g_importance, float* grad, void* stream) {
  const char* what = "neighbour_balance_backward";
  FSGS_REQUIRE(N >= 0 && N < (int64_t) 0x7fffffff && M > 0 && K >= 1, "%s: bad arguments", what);
  if (N == 0) return kOk;
  FSGS_REQUIRE(indices && counts && totals && grad && (g_loss || g_importance), "%s: null pointer", what);
  FSGS_REQUIRE((uintptr_t) indices % 8 == 0 && (uintptr_t) grad % 4 == 0, "%s: misaligned address", what);
  const int64_t blocks = (N * K + 4 * kSlopeThreads - 1) / (4 * kSlopeThreads);
  const bool lds = M <= kMostSlopes;
  hipLaunchKernelGGL((lds ? balance_neighbours_backward_kernel<true> : balance_neighbours_backward_kernel<false>),
                     dim3((unsigned) (blocks < kSlopeBlocks ? blocks : kSlopeBlocks)), dim3(kSlopeThreads), lds ? (size_t) M * 4 : 0,
                     (hipStream_t) stream, N, M, K, indices, rows, counts, totals, g_loss, g_importance, grad);
  return check_launch(what);
}
