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

constexpr int kStatThreads = 256, kWalkThreads = 512, kWalkWarps = kWalkThreads / 32, kMostCluster = 8;
constexpr int kMostTokens = 512;       // of a row
constexpr double kLog2e = 1.4426950408889634074;
// What float32's sums may be off by, relatively: sums of 32 at a time (2^-19 at most) of exponentials that are off by 2^-22 each.
constexpr double kUnsure = 4e-6;

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
  float2* partial;         // [rows, width, chunks]: maximum and sum (temperature 0: maximum and, as bits, its index)
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
  __device__ __forceinline__ void load(int i, float (&x)[kVec]) const {
    const int at = first(i);
    if (at >= 0 && at + kVec <= n) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + at);
      const T* const e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[j] = as_float(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[j] = at + j >= 0 && at + j < n ? as_float(row[at + j]) : -CUDART_INF_F;
    }
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
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int VEC = RowOf<T>::kVec, AT_ONCE = 32 / VEC;
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
    const RowOf<T> row(static_cast<const T*>(p.logits) + b * p.logits_stride[0] + node * p.logits_stride[1], p.vocab);
    const int vectors = row.vectors(), lo = (int)((int64_t)vectors * chunk / p.chunks), hi = (int)((int64_t)vectors * (chunk + 1) / p.chunks);
    float m = -CUDART_INF_F;
    double s = 0.0;
    int index = INT_MAX;
    for (int i0 = lo + threadIdx.x; i0 < hi; i0 += kStatThreads * AT_ONCE) {
      float x[AT_ONCE][VEC];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int i = i0 + j * kStatThreads;
        if (i < hi) {
          row.load(i, x[j]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[j][e] = -CUDART_INF_F;
        }
      }
      if (t == 0.0f) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if (x[j][e] > m) m = x[j][e], index = row.first(i0 + j * kStatThreads) + e;
            if (x[j][e] != x[j][e]) s = CUDART_NAN;
          }
        continue;
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) top = fmaxf(top, x[j][e]);
      if (top == -CUDART_INF_F) {        // (NaN alone are such a maximum too)
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (x[j][e] != x[j][e]) s = CUDART_NAN;
        continue;
      }
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += exp2_fast((x[j][e] - top) * scale);
      if (top > m) s *= exp2_fast((m - top) * scale), m = top;
      s += sum;
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

// 2^y for y <= 0 to about 2e-16: a table of 32nds and a polynomial, 2^f = sum (f ln 2)^k / k!, |f| <= 1/64.
__device__ __forceinline__ double exp2_wide(double y, const double* table) {
  if (!(y > -1000.0)) return y != y ? y : 0.0;
  constexpr double kRound = 6755399441055744.0;      // 3 x 2^51: the sum's last bits are a whole number
  const double t = __fma_rn(y, 32.0, kRound);
  const int n = __double2loint(t);
  const double f = __fma_rn(t - kRound, -1.0 / 32.0, y), z = f * 0.69314718055994530942;
  double r = __fma_rn(z, 1.0 / 720.0, 1.0 / 120.0);
  r = __fma_rn(z, r, 1.0 / 24.0);
  r = __fma_rn(z, r, 1.0 / 6.0);
  r = __fma_rn(z, r, 0.5);
  r = __fma_rn(z, r, 1.0);
  r = __fma_rn(z, r, 1.0) * table[n & 31];
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
  double* divisors;                      // see below
  float *top, *uniform, *chance_q;       // a token's row: its maximum; the random number; the draft's probability of it
  int *parent, *token, *best;            // best: the largest logit's index (temperature 0)
  int* out;                              // followers that were refused (no draft)
};
constexpr int kDraftedBytes = 3 * 8 + 3 * 4 + 4 * 4;

template <typename T>
__global__ void __launch_bounds__(kWalkThreads, 1) verify_walk_kernel(const __grid_constant__ VerifyParams p) {
  using Row = RowOf<T>;
  constexpr int VEC = Row::kVec;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ double table[32], shares[kWalkWarps], totals[2][kMostCluster];
  pdl_wait();
  pdl_launch_dependents();
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks(), b = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
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
    d.sum = at, d.weight = at + p.width, d.divisors = at + 2 * p.width;
    float* of = reinterpret_cast<float*>(at + 3 * p.width);
    d.top = of, d.uniform = of + p.width, d.chance_q = of + 2 * p.width;
    int* to = reinterpret_cast<int*>(of + 3 * p.width);
    d.parent = to, d.token = to + p.width, d.best = to + 2 * p.width, d.out = to + 3 * p.width;
  }
  __syncthreads();                       // (the table)
  // Every row's chunks together, a warp to a row.
  for (int i = warp; i < count; i += kWalkWarps) {
    const float2* const parts = p.partial + ((int64_t)b * p.width + i) * p.chunks;
    float top = -CUDART_INF_F;
    bool nan = false;
    for (int j = lane; j < p.chunks; j += 32) top = fmaxf(top, parts[j].x), nan = nan || parts[j].x != parts[j].x;
#pragma unroll
    for (int x = 16; x > 0; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    nan = __any_sync(0xffffffffu, nan) != 0;
    double sum = 0.0;
    int best = INT_MAX;
    for (int j = lane; j < p.chunks; j += 32) {
      if (greedy && parts[j].x == top) best = min(best, __float_as_int(parts[j].y));
      if (!greedy && parts[j].x > -CUDART_INF_F) sum += (double)parts[j].y * exp2_wide(((double)parts[j].x - (double)top) * scale, table);
    }
#pragma unroll
    for (int x = 16; x > 0; x /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    best = __reduce_min_sync(0xffffffffu, best);
    // no distribution: a NaN, an infinity or nothing but -inf
    const bool none = nan || !(top > -CUDART_INF_F) || (!greedy && !(top < CUDART_INF_F && sum > 0.0));
    if (lane == 0) d.top[i] = top, d.sum[i] = none ? -1.0 : sum, d.best[i] = best;
  }
  for (int i = threadIdx.x; i < count; i += kWalkThreads) {
    int parent = p.parents != nullptr ? p.parents[b * p.parents_stride + i] : i - 1;
    const int token = p.tokens[(int64_t)b * p.width + i];
    if (i > 0 && (parent < -1 || parent >= i || (unsigned)token >= (unsigned)p.vocab)) {
      if (rank == 0) cache_fault(p.c, KB200_CACHE_BAD_INDEX);
      parent = -1;
    }
    d.parent[i] = i > 0 ? parent : -1;
    d.token[i] = token;
    d.uniform[i] = fmaxf(p.uniform[(int64_t)b * p.width + i], 0.0f);
  }
  __syncthreads();
  if (!greedy)
    for (int i = 1 + threadIdx.x; i < count; i += kWalkThreads) {
      if (d.parent[i] < 0) continue;
      const int of = d.parent[i], token = d.token[i];
      d.weight[i] = exp2_wide(((double)as_float(logits[of * p.logits_stride[1] + token]) - (double)d.top[of]) * scale, table);
      d.chance_q[i] = p.draft != nullptr ? draft_at(p, b * p.draft_stride[0] + of * p.draft_stride[1] + token) : 1.0f;
    }
  __syncthreads();

  // From here on every thread of the cluster takes the same steps with the same numbers, and only the sums over the vocabulary are shared out.
  int at = 0, steps = 1, turn = 0;
  int depth = 0;               // how many times the draft's probabilities have been taken off the row of `at`, by which divisors
  int refused = 0;             // (no draft) how many of the followers' tokens have been taken out of it
  double sum = d.sum[0], left = 1.0;
  bool exact = false;          // `sum` is float64's
  bool shared = false;         // shares and totals are of what is left now
  double total = 0.0;
  auto removed = [&](int token, int n) {
    bool is = false;
    for (int j = 0; j < n; ++j) is = is || d.out[j] == token;
    return is;
  };
  // What is left of element v of the row of `at`, in units of the row's sum with a draft, of its largest weight without.
  auto value = [&](int v, float logit, int out) {
    const double e = exp2_wide(((double)logit - (double)d.top[at]) * scale, table);
    if (out > 0) return removed(v, out) ? 0.0 : e;
    if (depth == 0) return e;
    const double q = draft_at(p, b * p.draft_stride[0] + at * p.draft_stride[1] + v);
    double r = e / sum;
    for (int k = 0; k < depth; ++k) r = fmax(r / d.divisors[k] - q, 0.0);
    return r;
  };
  auto sum_of = [&](const Row& row, int lo, int hi, int out) {      // of vectors lo .. hi, by a warp
    double x = 0.0;
    for (int i = lo + lane; i < hi; i += 32) {
      float logit[VEC];
      row.load(i, logit);
      const int first = row.first(i);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (first + j >= 0 && first + j < p.vocab) x += value(first + j, logit[j], out);
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  };
  auto row_at = [&]() { return Row(logits + at * p.logits_stride[1], p.vocab); };
  auto part_of = [](int lo, int hi, int i, int n, int* from, int* to) {
    *from = lo + (int)((int64_t)(hi - lo) * i / n);
    *to = lo + (int)((int64_t)(hi - lo) * (i + 1) / n);
  };
  // The sum of what is left, over the cluster; the first `out` of the refused tokens are out of it.
  auto sum_left = [&](int out) {
    const Row row = row_at();
    int lo, hi, from, to;
    part_of(0, row.vectors(), rank, ranks, &lo, &hi);
    part_of(lo, hi, warp, kWalkWarps, &from, &to);
    const double mine = sum_of(row, from, to, out);
    __syncthreads();                     // (the last shares have been read)
    if (lane == 0) shares[warp] = mine;
    __syncthreads();
    if (threadIdx.x < ranks) {
      double x = 0.0;
      for (int w = 0; w < kWalkWarps; ++w) x += shares[w];
      cluster.map_shared_rank(&totals[turn][0], threadIdx.x)[rank] = x;
    }
    cluster.sync();
    double x = 0.0;
    for (int r = 0; r < ranks; ++r) x += totals[turn][r];
    turn ^= 1;
    return x;
  };
  auto sum_exactly = [&]() {               // (nothing has been taken off by a draft yet)
    if (exact) return;
    total = sum = sum_left(0);
    exact = true;
    shared = refused == 0;
  };

  bool known = sum > 0.0 || greedy;
  if (d.sum[0] < 0.0) known = false;
  for (int c = 1; c < count && known; ++c) {
    if (d.parent[c] != at) continue;
    bool take;
    if (greedy) {
      take = d.token[c] == d.best[at];
    } else {
      const double u = (double)d.uniform[c] * (double)d.chance_q[c];
      for (int pass = 0; pass < 2; ++pass) {
        double chance = d.weight[c] / sum;
        if (p.draft != nullptr) {
          for (int k = 0; k < depth; ++k) chance = fmax(chance / d.divisors[k] - (double)d.chance_q[c], 0.0);
        } else if (removed(d.token[c], refused)) {
          chance = 0.0;
        }
        take = u * left < chance;
        if (exact || pass > 0 || fabs(u * left - chance) > kUnsure * (u + chance)) break;
        // (what is left without a draft is 1 less the refused ones' chances, which are as near as the sum)
        const double before = sum;
        sum_exactly();
        if (p.draft == nullptr && refused != 0) left = 1.0 - (1.0 - left) * (before / sum);
      }
    }
    if (take) {
      at = c;
      if (writes) accepted[steps] = c;
      ++steps;
      depth = 0, refused = 0, left = 1.0, exact = false, shared = false;
      sum = d.sum[at];
      if (d.sum[at] < 0.0) known = false;
    } else if (!greedy) {
      if (p.draft != nullptr) {
        sum_exactly();
        if (threadIdx.x == 0) d.divisors[depth] = left;
        __syncthreads();
        ++depth;
        const double rest = sum_left(0);
        shared = rest > 0.0;
        if (shared) left = rest, total = rest;
        else --depth;                    // (where nothing is left it stays as it was)
      } else if (!removed(d.token[c], refused)) {
        if (threadIdx.x == 0) d.out[refused] = d.token[c];
        __syncthreads();
        double rest = left - d.weight[c] / sum;
        if (rest < 1e-3) {               // little is left: float64 says how much
          sum_exactly();
          rest = sum_left(refused + 1) / sum;
        }
        shared = false;
        if (rest > 0.0) left = rest, ++refused;
      }
    }
  }
  if (writes) p.accepted_n[slot] = steps;
  if (!known) {
    if (writes) p.following[slot] = -1, cache_fault(p.c, KB200_CACHE_BAD_VALUE);
    return;
  }
  if (greedy) {
    if (writes) p.following[slot] = d.best[at];
    return;
  }
  // ---- the token that follows ----
  if (!shared) total = sum_left(refused);
  double target = (double)d.uniform[0] * total;
  const int last_turn = turn ^ 1;
  int owner = -1;
  for (int r = 0; r < ranks; ++r) {      // the first whose share reaches beyond the target; where roundings leave none, the last that has any
    const double x = totals[last_turn][r];
    if (x > 0.0) owner = r;
    if (target < x) break;
    if (r + 1 < ranks) {
      bool more = false;
      for (int r2 = r + 1; r2 < ranks; ++r2) more = more || totals[last_turn][r2] > 0.0;
      if (!more) break;
    }
    target -= x;
  }
  if (owner < 0 && writes) p.following[slot] = -1;
  if (rank != owner) return;
  const Row row = row_at();
  // Of parts' sums (of all warps), the one that the target falls into.
  auto find = [&]() {
    int found = 0;
    for (int w = 0, had = -1; w < kWalkWarps; ++w) {
      const double x = shares[w];
      if (x > 0.0) {
        had = w;
        if (target < x) {
          found = w;
          break;
        }
      }
      found = max(had, 0);
      bool more = false;
      for (int w2 = w + 1; w2 < kWalkWarps; ++w2) more = more || shares[w2] > 0.0;
      if (!more) break;
      target -= x;
    }
    return found;
  };
  int lo, hi, from, to;
  part_of(0, row.vectors(), rank, ranks, &lo, &hi);
  const int w1 = find();
  part_of(lo, hi, w1, kWalkWarps, &from, &to);
  lo = from, hi = to;
  part_of(lo, hi, warp, kWalkWarps, &from, &to);
  const double mine = sum_of(row, from, to, refused);
  __syncthreads();
  if (lane == 0) shares[warp] = mine;
  __syncthreads();
  const int w2 = find();
  part_of(lo, hi, w2, kWalkWarps, &from, &to);
  if (warp != 0) return;
  int last = -1;
  for (int i0 = from; i0 < to; i0 += 32) {
    const int i = i0 + lane, first = row.first(i);
    double x[VEC], of_lane = 0.0;
    float logit[VEC];
    if (i < to) row.load(i, logit);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[j] = i < to && first + j >= 0 && first + j < p.vocab ? value(first + j, logit[j], refused) : 0.0;
      of_lane += x[j];
    }
    double before = of_lane;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    const double all = __shfl_sync(0xffffffffu, before, 31);
    before -= of_lane;
    int mine_at = INT_MAX, mine_last = -1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      before += x[j];
      if (x[j] > 0.0) {
        mine_last = first + j;
        if (mine_at == INT_MAX && before > target) mine_at = first + j;
      }
    }
    const int found = __reduce_min_sync(0xffffffffu, mine_at);
    last = max(last, __reduce_max_sync(0xffffffffu, mine_last));
    if (found != INT_MAX) {
      last = found;
      break;
    }
    target -= all;
  }
  if (lane == 0) p.following[slot] = last;
}

// ---- host --------------------------------------------------------------------------------------

// Chunks of a row: so many CTAs that each of them has a row's part of 16 KB or so, and the GPU is full a few times over.
int chunks_of(const Cache& c, int rows, int tokens, int vocab) {
  const int64_t nodes = (int64_t)rows * tokens, wanted = (16 * (int64_t)c.sm_count + nodes - 1) / nodes;
  return (int)std::min<int64_t>(std::min<int64_t>(wanted, 64), std::max(1, vocab / 2048));
}
int cluster_of(const Cache& c, int rows) {
  int n = kMostCluster;
  while (n > 2 && rows * n > 2 * c.sm_count) n /= 2;
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

bool verify_ok(const Cache& c, int rows, int tokens, int vocab) {
  return rows >= 0 && rows <= (1 << 20) && tokens >= 0 && tokens <= kMostTokens && vocab >= 1 && vocab < (1 << 30);
}

}  // namespace
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
