// Verification of drafted tokens against the model's probabilities, and the token that follows them (kb200_cache_verify).  Rules: include/kb200.h.
//
// What bounds it: the bytes of the logits, which one pass reads (maxima and sums of all drafted tokens' rows, over the whole GPU); what a sequence does with them is
// decided by a cluster of CTAs in a second launch, which reads one more row, or two with the draft's probabilities, to draw the token that follows.
//
// The drawn token is the one in whose share of the sum a random number falls, and with a hundred thousand tokens the shares' borders lie closer than float32
// resolves: with sums that are off by 1e-7 one draw in a hundred gives a neighbour.  So the row that is drawn from is summed in float64, exponentials included; a token's
// own chance, which only a border that is as near as float32's errors could turn, is compared with float32's sums, and with float64's where it is that near.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "cache.h"
#include "tc_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kWalkThreads = 512, kWalkWarps = kWalkThreads / 32, kMostCluster = 16;
constexpr int kMostTokens = 512;       // of a row
constexpr double kLog2e = 1.4426950408889634074;
// What float32's sums may be off by, relatively.  A thread sums weights 2^(scale (x - m)) for a reference m that its maximum is kSlack above at most, and follows it by a factor in
// float64, however often.  A weight is off by 2^-22, and by ln 2 of what its exponent is: three roundings (difference, scale, product) of 2^-24 of the way from x to m and on to
// the largest of the CTA's m.  On the average over the weights that way is 2 kSlack longer at most than the distance to the row's maximum, and that is the entropy at most, log2 of the
// vocabulary: 1.24e-7 x (30 + 8) = 4.8e-6.  The factor from m to the largest: 2^-22.  Sums of eight, three joins and what is stored: 11 x 2^-24.  Together 6e-6.
constexpr double kUnsure = 8e-6;
constexpr float kSlack = 4.0f;         // log2 of a weight

struct VerifyParams {
  CacheView c;
  const void *logits, *draft;
  int64_t logits_stride[2], draft_stride[2];
  const int32_t *tokens, *parents;
  int64_t parents_stride;
  const float *uniform, *temperature;
  const int32_t *counts, *slots;
  int rows, width, vocab, chunks;
  int draft_dtype;
  float2* partial;         // [rows, width, chunks]: what a sum is relative to, and the sum (temperature 0: the maximum and, as bits, its index)
  int32_t *accepted_n, *accepted, *following;
};

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's elements in 16-byte vectors of the memory's own borders, whatever its alignment: vector i has elements i kVec - off .. of the row, some of which
// the first and the last one lack.
template <typename T>
struct RowOf {
  static constexpr int kVec = 16 / (int)sizeof(T);
  const T* row;
  int off, n;
  __device__ __forceinline__ RowOf(const T* at, int elements) : row(at), off((int)((reinterpret_cast<uintptr_t>(at) & 15) / sizeof(T))), n(elements) {}
  __device__ __forceinline__ int vectors() const { return (off + n + kVec - 1) / kVec; }
  __device__ __forceinline__ int first(int i) const { return i * kVec - off; }
  __device__ __forceinline__ bool whole(int i) const { return first(i) >= 0 && first(i) + kVec <= n; }
  // -inf where there is none.
  __device__ __forceinline__ uint4 load(int i) const {
    const int at = first(i);
    if (at >= 0 && at + kVec <= n) return *reinterpret_cast<const uint4*>(row + at);
    return load_part(at);
  }
  __device__ __noinline__ uint4 load_part(int at) const {
    uint4 v;
    T* const e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) e[j] = at + j >= 0 && at + j < n ? row[at + j] : T(-CUDART_INF_F);
    return v;
  }
  static __device__ __forceinline__ uint4 nothing() {
    uint4 v;
    T* const e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) e[j] = T(-CUDART_INF_F);
    return v;
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[kVec]) {
    const T* const e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = as_float(e[j]);
  }
};

// A row's sequence, or -1 where that is not the row's; drafted tokens, none where the row is left out.  By all threads of a CTA.
__device__ __forceinline__ int row_slot(const VerifyParams& p, int b, int* count, float* temperature, bool tell) {
  const int slot = p.slots != nullptr ? p.slots[b] : b;
  int n = p.counts != nullptr ? p.counts[b] : p.width;
  const float t = p.temperature != nullptr ? p.temperature[b] : 1.0f;
  bool bad = (unsigned)slot >= (unsigned)p.c.sequences, again = false;
  const bool cold = !(t >= 0.0f && t < CUDART_INF_F);
  if (p.slots != nullptr) {              // a sequence that an earlier row names is that row's
    for (int i = threadIdx.x; i < b; i += blockDim.x) again = again || p.slots[i] == slot;
    again = __syncthreads_or(again);
  }
  bad = bad || again;
  if ((bad || cold || n < 0 || n > p.width) && tell && threadIdx.x == 0) cache_fault(p.c, KB200_CACHE_BAD_INDEX);
  *count = cold ? 0 : min(max(n, 0), p.width);
  *temperature = t;
  return bad ? -1 : slot;
}

// Maxima and sums of exponentials of a drafted token's row, by chunks.
template <typename T>
__global__ void __launch_bounds__(kStatThreads, 4) verify_stats_kernel(const __grid_constant__ VerifyParams p) {
  using Row = RowOf<T>;
  constexpr int VEC = Row::kVec, AT_ONCE = 4;
  __shared__ float maxima[kStatThreads / 32];
  __shared__ double sums[kStatThreads / 32];
  __shared__ int indexes[kStatThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // What sequences get that no row names.
  if (p.slots != nullptr || p.rows < p.c.sequences) {
    const int64_t all = (int64_t)p.c.sequences * p.width;
    for (int64_t i = (int64_t)blockIdx.x * kStatThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kStatThreads) {
      p.accepted[i] = -1;
      if (i < p.c.sequences) p.accepted_n[i] = 0, p.following[i] = -1;
    }
    for (int64_t i = all + (int64_t)blockIdx.x * kStatThreads + threadIdx.x; i < p.c.sequences; i += (int64_t)gridDim.x * kStatThreads) p.accepted_n[i] = 0, p.following[i] = -1;
  }
  const int64_t units = (int64_t)p.rows * p.width * p.chunks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int chunk = (int)(u % p.chunks), node = (int)(u / p.chunks % p.width), b = (int)(u / p.chunks / p.width);
    if (node >= (p.counts != nullptr ? p.counts[b] : p.width)) continue;
    const float t = p.temperature != nullptr ? p.temperature[b] : 1.0f, scale = fminf((float)(kLog2e / t), 1e38f);
    const Row row(static_cast<const T*>(p.logits) + b * p.logits_stride[0] + node * p.logits_stride[1], p.vocab);
    const int vectors = row.vectors(), lo = (int)((int64_t)vectors * chunk / p.chunks), hi = (int)((int64_t)vectors * (chunk + 1) / p.chunks);
    float m = -CUDART_INF_F;             // what the sum's weights are relative to (temperature 0: the maximum)
    double s = 0.0;
    int index = INT_MAX;
    auto add = [&](const uint4 (&v)[AT_ONCE], int i0) {
      float x[AT_ONCE][VEC];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) Row::unpack(v[j], x[j]);
      if (t == 0.0f) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int at = row.first(i0 + j * kStatThreads) + e;
            if (x[j][e] > m || (x[j][e] == m && at < index)) m = x[j][e], index = at;      // (a row's first vector comes last)
            if (x[j][e] != x[j][e]) s = CUDART_NAN;
          }
        return;
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
        for (int e = 0; e < VEC; e += 2) top = tc::fmax3(top, x[j][e], x[j][e + 1]);
      if (!((top - m) * scale > kSlack)) top = m;
      const float2 behind = top == -CUDART_INF_F ? make_float2(0.0f, 0.0f) : make_float2(-top, -top), scale2 = make_float2(scale, scale);      // (nothing but -inf so far: weights of 0; NaN: NaN)
      float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const float2 y = tc::fmul2(tc::fadd2(make_float2(x[j][e], x[j][e + 1]), behind), scale2);
          sum[e >> 1 & 1] = tc::fadd2(sum[e >> 1 & 1], make_float2(exp2_fast(y.x), exp2_fast(y.y)));
        }
      if (top > m && m > -CUDART_INF_F) s *= exp2(((double)m - (double)top) * (double)scale);
      m = top;
      s += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    };
    // Whole vectors, the next of which are under way while these are summed; the row's first and last may not be whole.
    const int from = max(lo, 1), to = min(hi, vectors - 1);
    const uint4* const whole = reinterpret_cast<const uint4*>(row.row + row.first(1));
    uint4 ahead[AT_ONCE];
    auto ask = [&](int i0) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) ahead[j] = i0 + j * kStatThreads < to ? __ldcg(whole + i0 + j * kStatThreads - 1) : Row::nothing();
    };
    ask(from + threadIdx.x);
    for (int i0 = from + threadIdx.x; i0 < to; i0 += kStatThreads * AT_ONCE) {
      uint4 now[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) now[j] = ahead[j];
      ask(i0 + kStatThreads * AT_ONCE);
      add(now, i0);
    }
    if ((lo == 0 || hi == vectors) && threadIdx.x < 32) {
      const int i = threadIdx.x == 0 && lo == 0 ? 0 : threadIdx.x == 1 && hi == vectors && vectors > 1 ? vectors - 1 : -1;
      uint4 edge[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) edge[j] = Row::nothing();
      if (i >= 0) edge[0] = row.load(i);
      add(edge, max(i, 0));
    }
    // of the CTA
    float all = m;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, d));
    if (lane == 0) maxima[warp] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatThreads / 32; ++w) all = fmaxf(all, maxima[w]);
    s *= t == 0.0f || m == all ? 1.0 : m == -CUDART_INF_F ? (s != s ? CUDART_NAN : 0.0) : (double)exp2_fast((m - all) * scale);
    index = m == all ? index : INT_MAX;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    index = __reduce_min_sync(0xffffffffu, index);
    if (lane == 0) sums[warp] = s, indexes[warp] = index;
    __syncthreads();
    if (threadIdx.x == 0) {
      s = 0.0;
      for (int w = 0; w < kStatThreads / 32; ++w) s += sums[w], index = min(index, indexes[w]);
      p.partial[u] = make_float2(s != s ? CUDART_NAN_F : all, t == 0.0f ? __int_as_float(index) : (float)s);
    }
    __syncthreads();
  }
}

// 2^y for y <= 0 to about 3e-15: a table of 32nds and a polynomial, 2^f = sum (f ln 2)^k / k!, |f| <= 1/64 (the sixth power is 2e-15).  (More 32nds would save a
// multiplication and cost as much: 32 doubles lie two to a bank of shared memory.)
constexpr double kLn2 = 0.69314718055994530942;
__device__ __forceinline__ double exp2_wide(double y, const double* table) {
  if (!(y > -1000.0)) return y != y ? y : 0.0;
  constexpr double kRound = 211106232532992.0;       // 3 x 2^46: the sum's last bits are 32nds
  const double t = y + kRound, f = y - (t - kRound);
  const int n = __double2loint(t);
  double r = __fma_rn(f, kLn2 * kLn2 * kLn2 * kLn2 * kLn2 / 120.0, kLn2 * kLn2 * kLn2 * kLn2 / 24.0);
  r = __fma_rn(f, r, kLn2 * kLn2 * kLn2 / 6.0);
  r = __fma_rn(f, r, kLn2 * kLn2 / 2.0);
  r = __fma_rn(f, r, kLn2);
  const double power = table[n & 31];
  r = __fma_rn(power, f * r, power);
  return __hiloint2double(__double2hiint(r) + ((n >> 5) << 20), __double2loint(r));
}

__device__ __forceinline__ float draft_at(const VerifyParams& p, int64_t at) {
  if (p.draft_dtype == KB200_DTYPE_FP32) return static_cast<const float*>(p.draft)[at];
  if (p.draft_dtype == KB200_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.draft)[at]);
  return __half2float(static_cast<const __half*>(p.draft)[at]);
}

// What is known of the drafted tokens of a row.
struct Drafted {
  double *sum, *weight;                  // a token's row: the sum; its own weight in the row of the one that it follows, 2^((logit - maximum) / T log2 e)
  double* chance;                        // ... by that row's sum
  double* divisors;                      // see Left
  float *top, *uniform, *chance_q;       // a token's row: its maximum; the random number; the draft's probability of it
  int *parent, *token, *best;            // best: the largest logit's index (temperature 0)
  int* out;                              // see Left
};
constexpr int kDraftedBytes = 4 * 8 + 3 * 4 + 4 * 4;

// What is left of a token's row: weights 2^(scale (logit - top)), the first of them without what was refused, or, with a draft, in units of their sum, from which the draft's
// probabilities were taken `depth` times (divisors: the reciprocals of what was left before each time, of the first also the sum's).
struct Left {
  double scale, top;
  const double *table = nullptr, *divisors = nullptr;
  const int* out = nullptr;
  int64_t draft = 0;                     // the row's first element in p.draft
  int refused = 0, depth = 0;
};
// What nearly every row needs: sums over the vocabulary are bounded by the instructions of an exponential, 20 here (10 of float64).  (logit - top) scale is one multiply-add, off by 2^-53 of
// top scale, for rows where that is 2^12 at most, 5e-13 of a weight; and there is one power of f less than in exp2_wide, 1.2e-12.
constexpr double kNearTop = 4096.0;
struct Power {
  double e;
  bool any;                              // y >= -1000; if not e is nothing
};
__device__ __forceinline__ Power power_of(double y, uint32_t table) {
  constexpr double kRound = 211106232532992.0;
  const double t = y + kRound, f = y - (t - kRound);
  const int n = __double2loint(t);
  double r = __fma_rn(f, kLn2 * kLn2 * kLn2 * kLn2 / 24.0, kLn2 * kLn2 * kLn2 / 6.0), power;
  r = __fma_rn(f, r, kLn2 * kLn2 / 2.0);
  r = __fma_rn(f, r, kLn2);
  asm("ld.shared.f64 %0, [%1];" : "=d"(power) : "r"(table + ((n & 31) << 3)));
  r = __fma_rn(power, f * r, power);
  return Power{__hiloint2double(__double2hiint(r) + ((n & ~31) << 15), __double2loint(r)), (unsigned)__double2hiint(y) <= 0xC08F4000u};
}

__device__ __forceinline__ bool near_top(const Left& left) { return fabs(left.top * left.scale) <= kNearTop; }
// A token's weight, by the same steps wherever it is needed: what a draft leaves of one is a difference that is divided by what is left, refusal by refusal, and where a quarter is left each
// time a weight that is off by 10^-12 of itself is another number after twenty.
__device__ __forceinline__ double weight_of(const Left& left, double logit) {
  if (!near_top(left)) return exp2_wide((logit - left.top) * left.scale, left.table);
  const double shift = -left.top * left.scale;
  const Power y = power_of(__fma_rn(logit, left.scale, shift), tc::smem_u32(left.table));
  return y.any ? y.e : 0.0;
}
__device__ __forceinline__ double value_of(const VerifyParams& p, const Left& left, int v, float logit) {
  double r = weight_of(left, (double)logit);
  for (int j = 0; j < left.refused; ++j)
    if (left.out[j] == v) r = 0.0;
  if (left.depth > 0) {
    const double q = draft_at(p, left.draft + v);
    for (int k = 0; k < left.depth; ++k) r = fmax(__fma_rn(r, left.divisors[k], -q), 0.0);
  }
  return r;
}
// Sums of vectors lo .. hi of a row, by a warp.
struct Sums {
  double left;                           // what is left
  double all, of_left, near;             // (sum_first) the weights; those of what is left; the draft's probabilities that a weight is near
};
// Of whatever is left.
template <typename T>
__device__ __noinline__ Sums sum_any(const VerifyParams& p, const RowOf<T>& row, const Left& left, int lo, int hi) {
  double x = 0.0;
  for (int i = lo + (threadIdx.x & 31); i < hi; i += 32)
    for (int j = 0; j < RowOf<T>::kVec; ++j) {
      const int v = row.first(i) + j;
      if (v >= 0 && v < row.n) x += value_of(p, left, v, as_float(row.row[v]));
    }
  return Sums{x, 0.0, 0.0, 0.0};
}

// A vector's elements, as they lie.
template <typename T, int VEC>
struct Vector {
  uint32_t w[VEC * sizeof(T) / 4];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (std::is_same<T, float>::value) return __uint_as_float(w[i]);
    else if constexpr (std::is_same<T, __half>::value) return i & 1 ? __high2float(*reinterpret_cast<const __half2*>(&w[i / 2])) : __low2float(*reinterpret_cast<const __half2*>(&w[i / 2]));
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};
template <typename T>
using Logits = Vector<T, RowOf<T>::kVec>;
template <typename T>
__device__ __forceinline__ Logits<T> logits_of(const RowOf<T>& row, int i, int hi) {
  const uint4 v = i < hi ? row.load(i) : RowOf<T>::nothing();
  return Logits<T>{{v.x, v.y, v.z, v.w}};
}
// As many of a draft's probabilities as a vector of logits has: in 16 bytes or twice that where they lie so, or one by one.
template <typename T, typename Q>
struct DraftOf {
  static constexpr int kVec = RowOf<T>::kVec, kWords = kVec * (int)sizeof(Q) / 4, kEach = kWords < 4 ? kWords : 4;
  using Chances = Vector<Q, kVec>;
  struct alignas(kEach * 4) Words {
    uint32_t w[kEach];
  };
  const Q* q;
  bool aligned;
  __device__ __forceinline__ DraftOf(const VerifyParams& p, const Left& left, const RowOf<T>& row)
      : q(static_cast<const Q*>(p.draft) + left.draft), aligned(reinterpret_cast<uintptr_t>(q + row.first(0)) % sizeof(Words) == 0) {}
  __device__ __forceinline__ Chances load(const RowOf<T>& row, int i, int hi) const {
    Chances x = {};
    if (i >= hi) return x;
    if (!aligned || !row.whole(i)) return load_part(q, row.first(i), row.n);
#pragma unroll
    for (int k = 0; k < kWords; k += kEach) {
      const Words v = *reinterpret_cast<const Words*>(q + row.first(i) + k * 4 / (int)sizeof(Q));
#pragma unroll
      for (int j = 0; j < kEach; ++j) x.w[k + j] = v.w[j];
    }
    return x;
  }
  static __device__ __noinline__ Chances load_part(const Q* q, int first, int n) {
    Chances x = {};
    Q* const e = reinterpret_cast<Q*>(x.w);
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (first + j >= 0 && first + j < n) e[j] = q[first + j];
    return x;
  }
};
constexpr int kAhead = 1;                // vectors of a lane that are under way (more are moved from register to register: 64 rows of 8 drafts, 128000 tokens, 52.9, 53.6 and 56.6 us with 1, 2 and 4)

// Of weights, without those refused.
template <typename T>
__device__ __noinline__ Sums sum_weights(const VerifyParams& p, const RowOf<T>& row, const Left& left, int lo, int hi) {
  const double scale = left.scale, shift = -left.top * left.scale;
  const uint32_t table = tc::smem_u32(left.table);
  const int refused = left.refused;
  double x = 0.0;
  int i = lo + (threadIdx.x & 31);
  Logits<T> ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) ahead[j] = logits_of(row, i + 32 * j, hi);
  for (; i < hi; i += 32) {
    const Logits<T> now = ahead[0];                    // (-inf, a weight of 0, where there is none)
#pragma unroll
    for (int j = 1; j < kAhead; ++j) ahead[j - 1] = ahead[j];
    ahead[kAhead - 1] = logits_of(row, i + 32 * kAhead, hi);
    float logit[RowOf<T>::kVec];
#pragma unroll
    for (int j = 0; j < RowOf<T>::kVec; ++j) logit[j] = now[j];
    for (int k = 0; k < refused; ++k) {
      const int at = left.out[k] - row.first(i);
#pragma unroll
      for (int j = 0; j < RowOf<T>::kVec; ++j) logit[j] = at == j ? -CUDART_INF_F : logit[j];
    }
#pragma unroll
    for (int j = 0; j < RowOf<T>::kVec; ++j) {
      const Power y = power_of(__fma_rn((double)logit[j], scale, shift), table);
      if (y.any) x += y.e;
    }
  }
  return Sums{x, 0.0, 0.0, 0.0};
}
// Of weights, and of what the draft's probabilities leave of them when the sum is only known to float32 (its reciprocal: divisors[0]).  Where that turns out to be off by d, kUnsure at
// most, what is left is sum (e / sum' - q) = left + of_left (1 / sum' - 1 / sum), but for elements where |e / sum - q| is less than d q, which may have been counted or left out wrongly: d q
// at most for each.  Those of 2^-16 q and less are summed (near); 64 in 128000 of such logits' differences are.  Where d near is more than kMostOff of what is left, that is summed again
// with the sum that is then known.  (That always: twice the time.)
constexpr double kMostOff = 1e-10;
template <typename T, typename Q>
__device__ __noinline__ Sums sum_first(const VerifyParams& p, const RowOf<T>& row, const Left& left, int lo, int hi) {
  const DraftOf<T, Q> draft(p, left, row);
  const double scale = left.scale, shift = -left.top * left.scale, unit = left.divisors[0];
  const uint32_t table = tc::smem_u32(left.table);
  Sums x{0.0, 0.0, 0.0, 0.0};
  float near = 0.0f;
  int i = lo + (threadIdx.x & 31);
  Logits<T> ahead[kAhead];
  typename DraftOf<T, Q>::Chances q_ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) ahead[j] = logits_of(row, i + 32 * j, hi), q_ahead[j] = draft.load(row, i + 32 * j, hi);
  for (; i < hi; i += 32) {
    const Logits<T> now = ahead[0];
    const typename DraftOf<T, Q>::Chances q = q_ahead[0];
#pragma unroll
    for (int j = 1; j < kAhead; ++j) ahead[j - 1] = ahead[j], q_ahead[j - 1] = q_ahead[j];
    ahead[kAhead - 1] = logits_of(row, i + 32 * kAhead, hi), q_ahead[kAhead - 1] = draft.load(row, i + 32 * kAhead, hi);
#pragma unroll
    for (int j = 0; j < RowOf<T>::kVec; ++j) {
      const Power y = power_of(__fma_rn((double)now[j], scale, shift), table);
      const double e = y.any ? y.e : 0.0, chance = (double)q[j], r = __fma_rn(e, unit, -chance);
      if ((__double2hiint(r) & 0x7fffffff) < (int)((unsigned)__double2hiint(chance) - (16u << 20))) near += q[j];      // (16 of the exponent)
      x.all += e;
      if (r > 0.0) x.left += r, x.of_left += e;
    }
  }
  x.near = (double)near;
  return x;
}
// Of what they leave, taken off any number of times.
template <typename T, typename Q>
__device__ __noinline__ Sums sum_beyond(const VerifyParams& p, const RowOf<T>& row, const Left& left, int lo, int hi) {
  const DraftOf<T, Q> draft(p, left, row);
  const double scale = left.scale, shift = -left.top * left.scale;
  const uint32_t table = tc::smem_u32(left.table);
  double x = 0.0;
  int i = lo + (threadIdx.x & 31);
  Logits<T> ahead = logits_of(row, i, hi);
  typename DraftOf<T, Q>::Chances q_ahead = draft.load(row, i, hi);
  for (; i < hi; i += 32) {
    const Logits<T> now = ahead;
    const typename DraftOf<T, Q>::Chances q = q_ahead;
    ahead = logits_of(row, i + 32, hi), q_ahead = draft.load(row, i + 32, hi);
    double r[RowOf<T>::kVec];
#pragma unroll
    for (int j = 0; j < RowOf<T>::kVec; ++j) {
      const Power y = power_of(__fma_rn((double)now[j], scale, shift), table);
      r[j] = y.any ? y.e : 0.0;
    }
    for (int k = 0; k < left.depth; ++k) {
      const double unit = left.divisors[k];
#pragma unroll
      for (int j = 0; j < RowOf<T>::kVec; ++j) r[j] = fmax(__fma_rn(r[j], unit, -(double)q[j]), 0.0);
    }
#pragma unroll
    for (int j = 0; j < RowOf<T>::kVec; ++j) x += r[j];
  }
  return Sums{x, 0.0, 0.0, 0.0};
}
template <typename T, typename Q>
__device__ __forceinline__ Sums sum_drafted(const VerifyParams& p, const RowOf<T>& row, const Left& left, int lo, int hi, bool first) {
  return first ? sum_first<T, Q>(p, row, left, lo, hi) : sum_beyond<T, Q>(p, row, left, lo, hi);
}
template <typename T>
__device__ __forceinline__ Sums sum_of(const VerifyParams& p, const RowOf<T>& row, const Left& left, int lo, int hi, bool first) {
  Sums x;
  if (!near_top(left)) x = sum_any<T>(p, row, left, lo, hi);
  else if (left.depth == 0) x = sum_weights<T>(p, row, left, lo, hi);
  else if (p.draft_dtype == KB200_DTYPE_FP32) x = sum_drafted<T, float>(p, row, left, lo, hi, first);
  else if (p.draft_dtype == KB200_DTYPE_BF16) x = sum_drafted<T, __nv_bfloat16>(p, row, left, lo, hi, first);
  else x = sum_drafted<T, __half>(p, row, left, lo, hi, first);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    x.left += __shfl_xor_sync(0xffffffffu, x.left, o);
    if (first) {
      x.all += __shfl_xor_sync(0xffffffffu, x.all, o);
      x.of_left += __shfl_xor_sync(0xffffffffu, x.of_left, o);
      x.near += __shfl_xor_sync(0xffffffffu, x.near, o);
    }
  }
  return x;
}
template <typename T>
__global__ void __launch_bounds__(kWalkThreads, 1) verify_walk_kernel(const __grid_constant__ VerifyParams p) {
  using Row = RowOf<T>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ double table[32], shares[4][kWalkWarps], totals[2][4][kMostCluster];      // (as in Sums)
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks(), b = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  tc::cluster_arrive_relaxed();
  if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
  pdl_wait();
  pdl_launch_dependents();
  tc::cluster_wait();                    // (all of the cluster's CTAs have started: what they write into each other's shared memory finds it)
  int count;
  float temperature;
  const int slot = row_slot(p, b, &count, &temperature, rank == 0);
  if (slot < 0) return;                  // (all of the cluster)
  const bool writes = rank == 0 && threadIdx.x == 0, greedy = temperature == 0.0f;
  int32_t* const accepted = p.accepted + (int64_t)slot * p.width;
  if (rank == 0)
    for (int i = threadIdx.x; i < p.width; i += kWalkThreads) accepted[i] = i == 0 && count > 0 ? 0 : -1;
  if (count == 0) {
    if (writes) p.accepted_n[slot] = 0, p.following[slot] = -1;
    return;
  }
  const double scale = fmin(kLog2e / (double)temperature, 1e38);
  const T* const logits = static_cast<const T*>(p.logits) + b * p.logits_stride[0];
  Drafted d;
  {
    double* at = reinterpret_cast<double*>(smem);
    d.sum = at, d.weight = at + p.width, d.chance = at + 2 * p.width, d.divisors = at + 3 * p.width;
    float* of = reinterpret_cast<float*>(at + 4 * p.width);
    d.top = of, d.uniform = of + p.width, d.chance_q = of + 2 * p.width;
    int* to = reinterpret_cast<int*>(of + 3 * p.width);
    d.parent = to, d.token = to + p.width, d.best = to + 2 * p.width, d.out = to + 3 * p.width;
  }
  __syncthreads();                       // (the table)
  // What is given of the drafted tokens, by the last warps, and every row's chunks together, a warp to a row: at the same time, as far as there are warps.
  for (int i = kWalkThreads - 1 - threadIdx.x; i < count; i += kWalkThreads) {
    int parent = p.parents != nullptr ? p.parents[b * p.parents_stride + i] : i - 1;
    const int token = p.tokens[(int64_t)b * p.width + i];
    const float uniform = p.uniform[(int64_t)b * p.width + i];
    if (i > 0 && (parent < -1 || parent >= i || (unsigned)token >= (unsigned)p.vocab)) {
      if (rank == 0) cache_fault(p.c, KB200_CACHE_BAD_INDEX);
      parent = -1;
    }
    if (i > 0 && parent >= 0 && !greedy) {
      d.weight[i] = (double)as_float(logits[parent * p.logits_stride[1] + token]);
      d.chance_q[i] = p.draft != nullptr ? draft_at(p, b * p.draft_stride[0] + parent * p.draft_stride[1] + token) : 1.0f;
    }
    d.parent[i] = i > 0 ? parent : -1;
    d.token[i] = token;
    d.uniform[i] = fmaxf(uniform, 0.0f);
  }
  for (int i = warp; i < count; i += kWalkWarps) {
    const float2* const parts = p.partial + ((int64_t)b * p.width + i) * p.chunks;
    const float2 none_there = make_float2(-CUDART_INF_F, 0.0f), first = lane < p.chunks ? parts[lane] : none_there, second = lane + 32 < p.chunks ? parts[lane + 32] : none_there;
    float top = fmaxf(first.x, second.x);
    bool nan = first.x != first.x || second.x != second.x;
#pragma unroll
    for (int x = 16; x > 0; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    nan = __any_sync(0xffffffffu, nan) != 0;
    double sum = 0.0;
    int best = INT_MAX;
#pragma unroll 1
    for (int j = 0; j < 2; ++j) {
      const float2 part = j == 0 ? first : second;
      if (greedy && part.x == top) best = min(best, __float_as_int(part.y));
      if (!greedy && part.x > -CUDART_INF_F) sum += (double)part.y * exp2_wide(((double)part.x - (double)top) * scale, table);
    }
#pragma unroll
    for (int x = 16; x > 0; x /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    best = __reduce_min_sync(0xffffffffu, best);
    // no distribution: a NaN, an infinity or nothing but -inf
    const bool none = nan || !(top > -CUDART_INF_F) || (!greedy && !(top < CUDART_INF_F && sum > 0.0));
    if (lane == 0) d.top[i] = top, d.sum[i] = none ? -1.0 : sum, d.best[i] = best;
  }
  __syncthreads();
  if (!greedy)
    for (int i = threadIdx.x; i < count; i += kWalkThreads)
      if (d.parent[i] >= 0) {
        const int of = d.parent[i];
        d.weight[i] = weight_of(Left{scale, (double)d.top[of], table}, d.weight[i]);
        d.chance[i] = d.weight[i] / d.sum[of];
      }
  __syncthreads();

  // The first warp of every CTA of the cluster takes the same steps with the same numbers (by all threads they took 400 cycles for a token), and only the sums over the
  // vocabulary are shared out: it says which one it needs, and goes on behind it.
  enum { kNothing, kExactly, kFirst, kTaken, kRefused, kLast, kDone };
  struct Plan {
    int wants, at, steps, refused, depth;
    bool known;
    double total;
  };
  __shared__ Plan plan;
  int at = 0, steps = 1, c = 1, wants = kNothing, refused = 0, depth = 0, turn = 0;
  double sum = d.sum[0], left = 1.0, total = 0.0;
  bool exact = false;          // `sum` is float64's
  bool shared = false;         // shares and totals are of what is left now
  bool known = sum >= 0.0;
  auto removed = [&](int token) {
    bool is = false;
    for (int j = 0; j < refused; ++j) is = is || d.out[j] == token;
    return is;
  };
  while (true) {
    if (warp == 0) {
      while (wants == kNothing) {
        while (c < count && (!known || d.parent[c] != at)) ++c;
        if (c == count) {
          wants = !known || greedy || shared ? kDone : kLast;
          break;
        }
        bool take;
        if (greedy) {
          take = d.token[c] == d.best[at];
        } else {
          const double u = (double)d.uniform[c] * (double)d.chance_q[c];
          const bool again = p.draft == nullptr && removed(d.token[c]);
          double chance = again ? 0.0 : depth > 0 ? d.weight[c] : exact ? d.weight[c] / sum : d.chance[c];
          for (int k = 0; k < depth; ++k) chance = fmax(__fma_rn(chance, d.divisors[k], -(double)d.chance_q[c]), 0.0);
          take = u * left < chance;
          if (!exact && fabs(u * left - chance) <= kUnsure * (u + chance)) {
            wants = kExactly;            // (what is left without a draft is 1 less the refused ones' chances, which are as near as the sum)
          } else if (!take && p.draft != nullptr) {
            wants = exact ? kTaken : near_top(Left{scale, (double)d.top[at]}) ? kFirst : kExactly;
          } else if (!take && !again) {
            const double rest = left - chance;
            if (rest >= 1e-3) {
              if (lane == 0) d.out[refused] = d.token[c];
              __syncwarp();
              left = rest, shared = false, ++refused;
            } else {                     // little is left: float64 says how much
              wants = exact ? kRefused : kExactly;
            }
          }
        }
        if (wants != kNothing) break;
        if (take) {
          at = c;
          if (writes) accepted[steps] = c;
          ++steps;
          sum = d.sum[at], left = 1.0, exact = shared = false, refused = depth = 0;
          known = sum >= 0.0;
        }
        ++c;
      }
      if (lane == 0) {
        Plan next{wants, at, steps, refused, depth, known, total};
        if (wants == kExactly) next.refused = next.depth = 0;
        if (wants == kTaken || wants == kFirst) d.divisors[next.depth++] = 1.0 / (depth == 0 ? sum : left);
        if (wants == kRefused) d.out[next.refused++] = d.token[c];
        plan = next;
      }
    }
    __syncthreads();
    if (plan.wants == kDone) break;
    // ---- a sum over the vocabulary ----
    const Row row(logits + plan.at * p.logits_stride[1], p.vocab);
    const Left of{scale, (double)d.top[plan.at], table, d.divisors, d.out, b * p.draft_stride[0] + plan.at * p.draft_stride[1], plan.refused, plan.depth};
    const int64_t vectors = row.vectors(), of_all = ranks * kWalkWarps, mine = rank * kWalkWarps + warp;
    const int lo = (int)(vectors * mine / of_all), hi = (int)(vectors * (mine + 1) / of_all);
    const bool first = plan.wants == kFirst;
    const Sums mine_of = sum_of<T>(p, row, of, lo, hi, first);
    if (lane == 0) shares[0][warp] = mine_of.left, shares[1][warp] = mine_of.all, shares[2][warp] = mine_of.of_left, shares[3][warp] = mine_of.near;
    __syncthreads();
    if (warp < (first ? 4 : 1)) {
      double x = lane < kWalkWarps ? shares[warp][lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o /= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (lane < ranks) cluster.map_shared_rank(&totals[turn][warp][0], lane)[rank] = x;
    }
    cluster.sync();
    double off = 0.0;
    if (first) {                         // with the sum as it is now known
      double all = 0.0;
      for (int r = 0; r < ranks; ++r) all += totals[turn][1][r];
      const double change = 1.0 / all - d.divisors[0];
      if (lane == 0) shares[0][warp] = fmax(__fma_rn(mine_of.of_left, change, mine_of.left), 0.0);
      __syncthreads();
      if (warp == 0) {
        if (lane < ranks) totals[turn][0][lane] = fmax(__fma_rn(totals[turn][2][lane], change, totals[turn][0][lane]), 0.0);
        if (lane == 0) d.divisors[0] = 1.0 / all;
        off = fabs(change) * sum;
        sum = all, exact = true;
      }
    }
    if (warp == 0) {
      __syncwarp();
      double all = 0.0, near = 0.0;
      for (int r = 0; r < ranks; ++r) all += totals[turn][0][r], near += first ? totals[turn][3][r] : 0.0;
      if (near * off > kMostOff * all) {
        shared = false, wants = kNothing;
      } else if (wants == kExactly) {
        if (p.draft == nullptr) left = 1.0 - (1.0 - left) * (sum / all);
        sum = total = all, exact = true;
        shared = refused == 0;
        wants = kNothing;
      } else if (wants == kLast) {
        total = all, wants = kDone;
      } else {                           // (where nothing is left it stays as it was)
        const double rest = wants == kRefused ? all / sum : all;
        shared = rest > 0.0;
        if (shared) left = rest, total = all, refused = plan.refused, depth = plan.depth;
        ++c;
        wants = kNothing;
      }
    }
    turn ^= 1;
  }
  at = plan.at;
  if (writes) p.accepted_n[slot] = plan.steps;
  if (!plan.known || greedy) {
    if (writes) p.following[slot] = plan.known ? d.best[at] : -1;
    if (writes && !plan.known) cache_fault(p.c, KB200_CACHE_BAD_VALUE);
    return;
  }
  const Left now{scale, (double)d.top[at], table, d.divisors, d.out, b * p.draft_stride[0] + at * p.draft_stride[1], plan.refused, plan.depth};
  // ---- the token that follows: the CTA, the warp's part, a part of that, and in it the token, in whose share the target falls ----
  const Row row(logits + at * p.logits_stride[1], p.vocab);
  double target = (double)d.uniform[0] * plan.total;
  // Of up to 32 shares, one in each lane, the first that reaches beyond the target, which becomes what it is beyond those before; where roundings leave none, the last
  // that has any.
  bool reached = false;                  // whether the one found is of the first kind
  double below = 0.0, all = 0.0;         // the shares in front of it; all of them
  auto find = [&](double x) {
    double upto = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const unsigned any = __ballot_sync(0xffffffffu, x > 0.0), beyond = __ballot_sync(0xffffffffu, x > 0.0 && target < upto);
    const int found = beyond != 0 ? __ffs(beyond) - 1 : 31 - __clz(any);      // (-1: there are none)
    all = __shfl_sync(0xffffffffu, upto, 31);
    below = __shfl_sync(0xffffffffu, upto - x, max(found, 0));
    reached = beyond != 0;
    return found;
  };
  const int owner = find(lane < ranks ? totals[turn ^ 1][0][lane] : 0.0);
  if (owner < 0 && writes) p.following[slot] = -1;
  if (rank != owner) return;
  target -= below;
  const int w1 = find(lane < kWalkWarps ? shares[0][lane] : 0.0);
  target -= below;
  const int64_t vectors = row.vectors(), of_all = ranks * kWalkWarps, mine = rank * kWalkWarps + w1;
  const int lo = (int)(vectors * mine / of_all), hi = (int)(vectors * (mine + 1) / of_all);
  auto part = [&](int i) { return lo + (int)((int64_t)(hi - lo) * i / kWalkWarps); };
  const double share = sum_of<T>(p, row, now, part(warp), part(warp + 1), false).left;
  __syncthreads();
  if (lane == 0) shares[0][warp] = share;
  __syncthreads();
  if (warp != 0) return;
  const int w2 = find(lane < kWalkWarps ? shares[0][lane] : 0.0);
  target -= below;
  const int begin = max(row.first(part(w2)), 0), end = min(row.first(part(w2 + 1)), p.vocab);
  int last = -1;
  for (int v0 = begin; v0 < end; v0 += 32) {
    const int v = v0 + lane;
    const int found = find(v < end ? value_of(p, now, v, as_float(row.row[v])) : 0.0);
    if (found >= 0) last = v0 + found;
    if (reached) break;
    target -= all;
  }
  if (lane == 0) p.following[slot] = last;
}

// ---- host --------------------------------------------------------------------------------------

// Chunks of a row: as many CTAs as an SM holds of them, four, and a row's part is 8 KB at least.  (With four times as many, of which half had a row behind its sequence's last, 8 rows of
// 12 tokens took 14.5 us.)
int chunks_of(const Cache& c, int rows, int tokens, int vocab) {
  const int64_t nodes = (int64_t)rows * tokens, wanted = (4 * (int64_t)c.sm_count + nodes - 1) / nodes;
  return (int)std::min<int64_t>(std::min<int64_t>(wanted, 64), std::max(1, vocab / 2048));      // (64: two to a lane)
}
int cluster_of(const Cache& c, int rows) {
  int n = c.verify_cluster;
  while (n > 1 && (int64_t)rows * n > c.sm_count) n /= 2;
  return n;
}

template <typename T>
cudaError_t launch_verify(const Cache& c, const VerifyParams& p, cudaStream_t s) {
  const int64_t units = (int64_t)p.rows * p.width * p.chunks;
  cudaError_t e = launch_kernel(true, verify_stats_kernel<T>, dim3((unsigned)std::min<int64_t>(units, 1 << 20)), dim3(kStatThreads), 0, s, p);
  if (e != cudaSuccess) return e;
  const int ranks = cluster_of(c, p.rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * ranks);
  cfg.blockDim = dim3(kWalkThreads);
  cfg.dynamicSmemBytes = (size_t)p.width * kDraftedBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_walk_kernel<T>, p);
}

// The largest cluster, of up to kMostCluster CTAs, that the device takes.
template <typename T>
cudaError_t most_of_cluster(int* most) {
  cudaError_t e = cudaFuncSetAttribute(verify_walk_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (; e == cudaSuccess && *most > 8; *most /= 2) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(*most);
    cfg.blockDim = dim3(kWalkThreads);
    cfg.dynamicSmemBytes = (size_t)kMostTokens * kDraftedBytes;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = *most;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int fit = 0;
    if (cudaOccupancyMaxActiveClusters(&fit, verify_walk_kernel<T>, &cfg) == cudaSuccess && fit > 0) break;
    cudaGetLastError();
  }
  return e;
}
bool verify_ok(const Cache& c, int rows, int tokens, int vocab) {
  return rows >= 0 && rows <= (1 << 20) && tokens >= 0 && tokens <= kMostTokens && vocab >= 1 && vocab < (1 << 30);
}

}  // namespace

int cache_verify_prepare(Cache& c) {
  c.verify_cluster = kMostCluster;
  KB200_CUDA(most_of_cluster<float>(&c.verify_cluster));
  KB200_CUDA(most_of_cluster<__nv_bfloat16>(&c.verify_cluster));
  KB200_CUDA(most_of_cluster<__half>(&c.verify_cluster));
  return KB200_OK;
}

}  // namespace kb200

using namespace kb200;

KB200_EXPORT uint64_t kb200_cache_verify_workspace(const kb200_cache* handle, int rows, int tokens, int vocab) {
  if (handle == nullptr) return 0;
  const Cache& c = *cache_of(handle);
  if (!verify_ok(c, rows, tokens, vocab) || rows == 0 || tokens == 0) return 0;
  return (uint64_t)rows * tokens * chunks_of(c, rows, tokens, vocab) * sizeof(float2);
}

KB200_EXPORT int kb200_cache_verify(kb200_cache* handle, const kb200_scores* logits, const kb200_scores* draft, int rows, int tokens, int vocab, const int32_t* drafted,
                                    const int32_t* parents, int64_t parents_stride, const float* uniform, const float* temperature, const int32_t* counts,
                                    const int32_t* slots, int32_t* n_accepted, int32_t* accepted, int32_t* following, void* workspace, uint64_t workspace_bytes,
                                    void* stream) {
  KB200_CACHE_ENTER("kb200_cache_verify");
  if (!verify_ok(c, rows, tokens, vocab) || (slots == nullptr && rows > c.view.sequences))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_verify: %d rows of %d tokens, %d in the vocabulary (%d sequences, up to %d tokens)", rows, tokens, vocab, c.view.sequences,
                kMostTokens);
  if (n_accepted == nullptr || following == nullptr || (accepted == nullptr && tokens > 0)) return fail(KB200_ERR_ARGUMENT, "kb200_cache_verify: a result is null");
  const bool any = rows > 0 && tokens > 0;
  if (any) {
    if (logits == nullptr || logits->data == nullptr || drafted == nullptr || uniform == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_verify: logits, tokens or uniform is null");
    for (const kb200_scores* x : {logits, draft})
      if (x != nullptr && (x->data == nullptr || x->dtype < KB200_DTYPE_FP32 || x->dtype > KB200_DTYPE_FP16 ||
                           reinterpret_cast<uintptr_t>(x->data) % (x->dtype == KB200_DTYPE_FP32 ? 4 : 2) != 0))
        return fail(KB200_ERR_ARGUMENT, "kb200_cache_verify: logits and draft must be float32, bfloat16 or float16");
  }
  const uint64_t need = kb200_cache_verify_workspace(handle, rows, tokens, vocab);
  if (need > 0 && (workspace == nullptr || !tc::aligned16(workspace) || workspace_bytes < need))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_verify: a workspace of %llu bytes on 16 bytes is needed", (unsigned long long)need);
  if (!any) {
    KB200_CUDA(cudaMemsetAsync(n_accepted, 0, (size_t)c.view.sequences * 4, s));
    KB200_CUDA(cudaMemsetAsync(following, 0xff, (size_t)c.view.sequences * 4, s));
    if (tokens > 0) KB200_CUDA(cudaMemsetAsync(accepted, 0xff, (size_t)c.view.sequences * tokens * 4, s));
    return KB200_OK;
  }
  VerifyParams p{};
  p.c = c.view;
  p.logits = logits->data;
  p.draft = draft != nullptr ? draft->data : nullptr;
  p.draft_dtype = draft != nullptr ? draft->dtype : 0;
  for (int i = 0; i < 2; ++i) p.logits_stride[i] = logits->stride[i], p.draft_stride[i] = draft != nullptr ? draft->stride[i] : 0;
  p.tokens = drafted;
  p.parents = parents;
  p.parents_stride = parents_stride;
  p.uniform = uniform;
  p.temperature = temperature;
  p.counts = counts;
  p.slots = slots;
  p.rows = rows;
  p.width = tokens;
  p.vocab = vocab;
  p.chunks = chunks_of(c, rows, tokens, vocab);
  p.partial = static_cast<float2*>(workspace);
  p.accepted_n = n_accepted;
  p.accepted = accepted;
  p.following = following;
  KB200_CUDA(logits->dtype == KB200_DTYPE_FP32 ? launch_verify<float>(c, p, s)
             : logits->dtype == KB200_DTYPE_BF16 ? launch_verify<__nv_bfloat16>(c, p, s) : launch_verify<__half>(c, p, s));
  return KB200_OK;
}
