// What a warp of the attention over a paged cache does with a tile of keys: on the tensor cores for 16-bit caches (MmaMath), by float32
// multiply-adds for float32 ones (FmaMath).  Both keep maxima, sums and output rows of up to 16 query rows in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

#include "cache_attention.h"
#include "tc_common.cuh"

namespace kb200 {
namespace cache_math {

using namespace tc;

// A stage of the ring: blocks of 128-byte columns, as the map's 128-byte swizzle wants them: K's, then V's.
template <typename T, int DP>
struct Tile {
  static constexpr int kBlocks = DP * (int)sizeof(T) / 128;
  static constexpr int kKeys = kBlocks <= 2 ? 64 : 128 / kBlocks;        // 16 KB of K and of V at most
  static constexpr int kBlockBytes = kKeys * 128;
  static constexpr int kHalf = kBlocks * kBlockBytes;                    // K
  static constexpr int kBytes = 2 * kHalf;
  // The address of an element in K or V of a stage.
  static __device__ __forceinline__ T* at(uint8_t* half, int key, int d) {
    const int byte = d * (int)sizeof(T);
    return reinterpret_cast<T*>(half + (byte / 128) * kBlockBytes + key * 128 + ((((byte % 128) >> 4) ^ (key & 7)) << 4) + byte % 16);
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ void store2(T* to, float a, float b) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(to) = make_float2(a, b);
  else *reinterpret_cast<uint32_t*>(to) = pack<T>(a, b);
}
// Sets the top bit of every element of a 32-bit word that is infinite or NaN, and may set others below it: the exponent's ones and one more.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (sizeof(T) == 4) return (w & 0x7f800000u) + 0x00800000u;
  else if constexpr (std::is_same<T, __half>::value) return (w & 0x7c007c00u) + 0x04000400u;
  else return (w & 0x7f807f80u) + 0x00800080u;
}
// Two 16-bit elements with zeros in place of infinities and NaN.
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  if ((w & kExponent) == kExponent) w &= 0xffff0000u;
  if ((w >> 16 & kExponent) == kExponent) w &= 0xffffu;
  return w;
}
template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// 16-bit caches: a maximum of this size is a power of two's exponent that its rounding has moved by up to a half, which all weights of a row share and the division by
// their sum takes back.  Larger ones (float16 reaches 2^36) could be off by hundreds, and weights overflow; there an exponent is cut at its value at the maximum.
constexpr float kFarScore = 4194304.0f;
// The exponent of the largest weight.  float16 has 14 powers of two below 1 and 15 above: with a largest weight of 1, weights below 2^-14 would lose bits and those
// below 2^-25 vanish, and where a first token draws nearly all of the weight and its V is small the result is such weights' (3000 tokens whose scores are 17 behind its:
// off by 28 times what a rounding to float16 gives).  From 2^12 on it is 2^-26 and 2^-37 of the largest; sums and rows have the same factor, and their division takes it out.
template <typename T>
constexpr float kTopExponent = std::is_same<T, __half>::value ? 12.0f : 0.0f;
template <typename T>
__device__ __forceinline__ float exponent_of_top(float top, float scale) {
  const float e = __fmul_rd(top, scale);
  if constexpr (kTopExponent<T> != 0.0f) return __fadd_rd(e, -kTopExponent<T>);
  else return e;
}
template <typename T>
__device__ __forceinline__ float behind_top(float score, float scale, float shift) {
  const float e = fmaf(score, scale, shift);
  return e > kTopExponent<T> ? kTopExponent<T> : e;        // (NaN stays)
}

// Where a warp is: its tile and rows.
struct Place {
  uint8_t *k, *v;              // the stage
  int key0, sure;              // the tile's first key; keys that every row sees
  int row0, rows_here;         // the warp's first row of the item's row tile; rows of that
  int hidden;                  // (a window) keys from here on are not hidden from any row
  int warp, lane, row_group, key_group;
};

// A window hides some of a tile's keys from some rows.
__device__ __forceinline__ bool window_hides(const CacheAttnParams& p, int key0, int keys, int hidden) { return key0 < hidden && key0 + keys > p.sinks; }
// ... the bits of those that are hidden from a row of place `place`; drafted tokens are the mask's matter where there is one.
__device__ __forceinline__ unsigned long long hidden_keys(const CacheAttnParams& p, int length, int place, int key0) {
  const int begin = length + place - p.window + 1, end = p.mask != nullptr ? min(begin, length) : begin;
  if (end <= key0) return 0ull;            // (first: with a window of 2^31 - 1, end - key0 may be below -2^31)
  const int from = max(0, p.sinks - key0), to = end - key0;
  if (to <= from || from >= 64) return 0ull;
  return (to >= 64 ? ~0ull : (1ull << to) - 1) & ~((1ull << from) - 1);
}
__device__ __forceinline__ void write_lse(const CacheAttnParams& p, int b, const CacheRow& r, float value) {
  if (p.lse != nullptr) p.lse[b * p.lse_stride[0] + r.token * p.lse_stride[1] + r.head * p.lse_stride[2]] = value;
}

// What a warp's rows see of the drafted tokens.  Lane i has row i % 16 of the warp's, and of its drafted tokens the 32 from `first` on.  Small code on purpose, here
// and below: a launch meets it cold, once or twice, and its instructions come from L2 (unrolled over rows and keys this was 13000 cycles).
template <int ROWS>
__device__ __forceinline__ uint32_t mask_word(const CacheAttnParams& p, const CacheCursor& now, const Place& at, int first) {
  const int row = at.row0 + (at.lane & 15);
  if (row >= at.rows_here) return 0u;
  const CacheRow r = row_of<ROWS>(p, now, row);
  const uint8_t* const mask = p.mask + now.b * p.mask_stride[0] + r.token * p.mask_stride[1];
  const int lo = max(0, -first), hi = min(32, now.it.count - first);
  uint32_t word = 0u;
#pragma unroll 8
  for (int j = lo; j < hi; ++j) word |= mask[(first + j) * p.mask_stride[2]] != 0 ? 1u << j : 0u;
  return word;
}
// Of up to this many drafted tokens the words are fetched when an item begins, under the way of its first keys.
constexpr int kMaskAhead = 64;

// The keys of a tile with drafted tokens that the warp's rows see: row i of the warp's in sees[i].
template <int ROWS, int WARP_ROWS, int KEYS, bool WINDOW>
__device__ __forceinline__ void look_at_mask(const CacheAttnParams& p, const CacheCursor& now, const Place& at, uint32_t ahead, uint2* sees) {
  const int row = at.lane & 15, off = now.it.length - at.key0;         // where the first drafted token is in the tile
  unsigned long long shows = 0ull;
  if (p.mask == nullptr) {
    const int n = off + row_of<ROWS>(p, now, at.row0 + row).token + 1;
    shows = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
  } else {
    uint32_t low = ahead, high;
    if (p.tokens > kMaskAhead) low = mask_word<ROWS>(p, now, at, (at.lane >> 4) * 32 - off);
    high = __shfl_sync(0xffffffffu, low, row + 16);
    low = __shfl_sync(0xffffffffu, low, row);
    shows = (unsigned long long)high << 32 | low;
    if (p.tokens <= kMaskAhead) shows = off >= 64 || off <= -64 ? 0ull : off >= 0 ? shows << off : shows >> -off;
    if (off > 0) shows |= off >= 64 ? ~0ull : (1ull << off) - 1;
  }
  const int last = now.it.end - at.key0;
  if (last < 64) shows &= last <= 0 ? 0ull : (1ull << last) - 1;
  if constexpr (WINDOW) {
    if (at.row0 + row < at.rows_here) shows &= ~hidden_keys(p, now.it.length, place_of(p, now.b, row_of<ROWS>(p, now, at.row0 + row).token), at.key0);
  }
  if (at.lane < WARP_ROWS) sees[row] = make_uint2((uint32_t)shows, (uint32_t)(shows >> 32));
  __syncwarp();
}

// V behind the sequence's end is what an earlier tenant left, as far as its last page goes (pages that it has not come as zeros), and V of a drafted token that some
// rows do not see may hold infinities or NaN; 0 times those is NaN.  The former become zeros (every warp that reads the tile writes them, and looks at none of
// them).  True: the latter are there.
template <typename T, int DP, bool WINDOW>
__device__ __forceinline__ bool look_at_values(const CacheAttnParams& p, const CacheCursor& now, const Place& at) {
  using G = Tile<T, DP>;
  constexpr int kChunks = G::kBlocks * 8;
  const int in_page = (1 << p.c.page_log2) - 1, last = now.it.end - at.key0;
  const int from = WINDOW && window_hides(p, at.key0, G::kKeys, at.hidden) ? 0 : max(0, at.sure - at.key0), to = min(G::kKeys, ((now.it.end + in_page) & ~in_page) - at.key0);
  uint32_t odd = 0u;
#pragma unroll 2
  for (int i = from * kChunks + at.lane; i < to * kChunks; i += 32) {
    const int key = i / kChunks, chunk = i % kChunks;
    uint4* const x = reinterpret_cast<uint4*>(G::at(at.v, key, chunk * (16 / (int)sizeof(T))));
    if (key >= last) *x = make_uint4(0, 0, 0, 0);
    else odd |= not_finite<T>(x->x) | not_finite<T>(x->y) | not_finite<T>(x->z) | not_finite<T>(x->w);
  }
  const bool any = __any_sync(0xffffffffu, (odd & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u)) != 0u) != 0;
  __syncwarp();
  return any;
}

// 16-bit caches: mma.sync m16n8k16, the scores' accumulators being the weights' operands.  A thread holds rows g and g + 8.
template <typename T, int DP>
struct MmaMath {
  using Type = T;
  static constexpr bool kByRows = false;
  static constexpr int kDim = DP, kRows = 16, kOut = DP / 2;             // rows of a warp; output registers of a thread
  using G = Tile<T, DP>;
  static constexpr int NT = G::kKeys / 8, DT = DP / 8;                   // 8-wide column tiles of the scores, of the output rows
  uint32_t q[DP / 16][4];
  float o[DT][4], m[2], l[2];
  // Maxima are powers of two's exponents: the scale and the maximum go into one multiply-add per score, and a rounding of the maximum cancels.  It is rounded
  // down, so that the largest weight is not below 2^kTopExponent; see kFarScore for where it would be far above.
  static __device__ __forceinline__ float exponent(float behind, float) { return behind; }
  // The logarithm of a row's sum.
  static __device__ __forceinline__ float log_sum(float top, float sum, float) { return sum == 0.0f ? -CUDART_INF_F : fmaf(top, 0.69314718f, logf(sum)); }

  template <int ROWS>
  __device__ __forceinline__ void begin(const CacheAttnParams& p, const CacheCursor& now, const Place& at) {
    const int g = at.lane >> 2, t4 = at.lane & 3;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.0f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = at.row0 + g + 8 * half;
      const bool there = row < at.rows_here;
      const CacheRow r = row_of<ROWS>(p, now, there ? row : 0);
      const int64_t from = now.b * p.q_stride[0] + r.token * p.q_stride[1] + r.head * p.q_stride[2];
      auto pair = [&](int i) {                       // two elements
        if (!p.q_fp32) return reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + from)[i];
        const float2 x = reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + from)[i];
        return pack<T>(x.x, x.y);
      };
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const bool in = there && k * 16 < p.c.head_dim;
        q[k][half] = in ? pair(k * 8 + t4) : 0u;
        q[k][2 + half] = in ? pair(k * 8 + 4 + t4) : 0u;
      }
    }
  }

  // The weights times V; CLEAN: with zeros in place of infinities and NaN in V.
  template <bool CLEAN>
  __device__ __forceinline__ void times_values(const float (&s)[NT][4], uint32_t v_tile, int lane) {
    const uint32_t v_row = v_tile + (((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
#pragma unroll
    for (int k = 0; k < NT / 2; ++k) {
      const uint32_t a[4] = {pack<T>(s[2 * k][0], s[2 * k][1]), pack<T>(s[2 * k][2], s[2 * k][3]), pack<T>(s[2 * k + 1][0], s[2 * k + 1][1]),
                             pack<T>(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
      for (int d = 0; d < DT; d += 2) {
        uint32_t b[4];
        ldmatrix4_t(b, v_row + k * 16 * 128 + (d / 8) * G::kBlockBytes + (((d % 8 + (lane >> 4)) ^ (lane & 7)) << 4));
        if constexpr (CLEAN) {
#pragma unroll
          for (int i = 0; i < 4; ++i) b[i] = finite_pair<T>(b[i]);
        }
        mma16<T>(o[d], a, b[0], b[1]);
        mma16<T>(o[d + 1], a, b[2], b[3]);
      }
    }
  }

  template <int ROWS, bool WINDOW>
  __device__ __forceinline__ void tile(const CacheAttnParams& p, const CacheCursor& now, const Place& at, uint32_t ahead, uint2* sees) {
    const int lane = at.lane, g = lane >> 2, t4 = lane & 3;
    const uint32_t k_tile = smem_u32(at.k), v_tile = smem_u32(at.v);
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
    const uint32_t k_row = k_tile + ((lane >> 4) * 8 + (lane & 7)) * 128;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint32_t in_row = (k / 4) * G::kBlockBytes + ((((k % 4) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t b[4];
        ldmatrix4(b, k_row + n * 8 * 128 + in_row);
        mma16<T>(s[n], q[k], b[0], b[1]);
        mma16<T>(s[n + 1], q[k], b[2], b[3]);
      }
    }

    const bool drafted = at.key0 + G::kKeys > at.sure || (WINDOW && window_hides(p, at.key0, G::kKeys, at.hidden));
    bool infinite = false;
    if (drafted) {
      look_at_mask<ROWS, 16, G::kKeys, WINDOW>(p, now, at, ahead, sees);
      infinite = look_at_values<T, DP, WINDOW>(p, now, at);
      unsigned long long shows[2];                   // the tile's keys that rows g and g + 8 see
#pragma unroll
      for (int h = 0; h < 2; ++h) shows[h] = sees[g + 8 * h].x | (unsigned long long)sees[g + 8 * h].y << 32;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(shows[j >> 1] >> (n * 8 + t4 * 2 + (j & 1)) & 1)) s[n][j] = -CUDART_INF_F;
    }

    // softmax: two rows of a thread, their keys over the four lanes of a group
    float top[2] = {-CUDART_INF_F, -CUDART_INF_F}, shift[2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) top[j >> 1] = fmaxf(top[j >> 1], s[n][j]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = exponent_of_top<T>(fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2)), p.scale_log2);
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], m[h]);
        alpha[h] = top[h] == -CUDART_INF_F ? 1.0f : ex2(m[h] - top[h]);
        m[h] = top[h];
        l[h] *= alpha[h];
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][j] *= alpha[j >> 1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) shift[h] = m[h] == -CUDART_INF_F ? 0.0f : -m[h];          // nothing seen so far: every weight is 2^-inf
    float scale = p.scale_log2;
    if (fabsf(shift[0]) > kFarScore || fabsf(shift[1]) > kFarScore) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = behind_top<T>(s[n][j], scale, shift[j >> 1]);
      scale = 1.0f, shift[0] = shift[1] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] = ex2(fmaf(s[n][j], scale, shift[j >> 1]));
        l[j >> 1] += s[n][j];
      }

    if (infinite) {  // infinities and NaN: one by one, to the rows that give them any weight; they are zero in the product
#pragma unroll
      for (int n = 0; n < NT; ++n)
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float w[2] = {__shfl_sync(0xffffffffu, s[n][e], (lane & ~3) | t), __shfl_sync(0xffffffffu, s[n][2 + e], (lane & ~3) | t)};
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float x = to_float(*G::at(at.v, n * 8 + t * 2 + e, d * 8 + t4 * 2 + (j & 1)));
                if (!(fabsf(x) < CUDART_INF_F) && w[j >> 1] != 0.0f) o[d][j] += w[j >> 1] * x;
              }
          }
    }

    if (infinite) times_values<true>(s, v_tile, lane);
    else times_values<false>(s, v_tile, lane);
    if (drafted) fence_async_smem();                 // (the zeros, in front of the next copy to this stage)
  }

  __device__ __forceinline__ void sum_up() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (l[h] != l[h]) m[h] = 0.0f;                 // (NaN, which a maximum passes over, reaches the result)
    }
  }
  __device__ __forceinline__ void put_states(int lane, float2* states) const {
    if ((lane & 3) == 0) states[lane >> 2] = make_float2(m[0], l[0]), states[(lane >> 2) + 8] = make_float2(m[1], l[1]);
  }
  __device__ __forceinline__ void rescale(int lane, const float* factors) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float f = factors[(lane >> 2) + 8 * h];
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][2 * h] *= f, o[d][2 * h + 1] *= f;
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_out(F&& f) {
#pragma unroll
    for (int i = 0; i < kOut; ++i) f(i, o[i / 4][i % 4]);
  }
  // Where a row's column is among the 32 x kOut values of a warp.
  static __device__ __forceinline__ int place(int row, int d) { return (d / 8 * 4 + (row >> 3) * 2 + (d & 1)) * 32 + (row & 7) * 4 + d % 8 / 2; }
  // The rows, divided by their sums; states: of all the item's warps together.
  template <int ROWS, bool WINDOW>
  __device__ __forceinline__ void write(const CacheAttnParams& p, const CacheCursor& now, const Place& at, const float2* states, float*) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int in_warp = (at.lane >> 2) + 8 * h, row = at.row0 + in_warp;
      if (row >= at.rows_here) continue;
      const float sum = states[in_warp].y, inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const CacheRow r = row_of<ROWS>(p, now, row);
      T* const to = static_cast<T*>(p.out) + now.b * p.out_stride[0] + r.token * p.out_stride[1] + r.head * p.out_stride[2] + (at.lane & 3) * 2;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        if (d * 8 < p.c.head_dim) store2<T>(to + d * 8, o[d][2 * h] * inv, o[d][2 * h + 1] * inv);
      if constexpr (WINDOW) {
        if ((at.lane & 3) == 0) write_lse(p, now.b, r, log_sum(states[in_warp].x, sum, p.scale_log2));
      }
    }
  }
};

// float32 caches: multiply-adds, two to an instruction.  (Three TF32 products of split operands by mma.sync took 9200 cycles for 64 keys of 64 whatever the
// number of rows was, and were off by twice as much.  A tile's multiply-adds take the SM 64 cycles a row; with five warps at it a warp needs 5000 to 7000 for 16 rows.)
// For the scores a lane has keys (two lanes share one where a tile has 16), for the output it has DP / 32 columns of all rows; weights go from one to the
// other through shared memory.
template <int DP, int R>
struct FmaMath {
  using Type = float;
  static constexpr bool kByRows = false;
  static constexpr int kDim = DP, kRows = R, kOut = R * DP / 32;
  using G = Tile<float, DP>;
  static constexpr int KEYS = G::kKeys >= 32 ? G::kKeys / 32 : 1;        // of a lane
  static constexpr int SHARE = G::kKeys >= 32 ? 1 : 32 / G::kKeys;       // lanes to a key, each with part of the columns
  static constexpr int kVec = R < 4 ? R : 4, kWeightRow = R < 4 ? R : R + 4;       // (the weights of a key: rows apart by banks that lanes do not share)
  static constexpr int C = DP / 32;                                      // output columns of a lane: C lane .. C lane + C - 1
  float2 o[C][R / 2];                                // rows 2i and 2i + 1
  float m[R], l[R];                                  // (l: of the lane's keys)
  // Scores and maxima are kept as they were summed, and the scale is applied to differences: a rounding then goes with the distance from the maximum, not with
  // the score's size.  (Scores of 8000 that were scaled and rounded first gave errors of 1e-4.)
  static __device__ __forceinline__ float exponent(float behind, float scale) { return behind * scale; }
  static __device__ __forceinline__ float log_sum(float top, float sum, float scale) { return sum == 0.0f ? -CUDART_INF_F : fmaf(top * scale, 0.69314718f, logf(sum)); }

  // The query rows go to shared memory, [R][DP] of the warp's own.
  template <int ROWS>
  __device__ __forceinline__ void begin(const CacheAttnParams& p, const CacheCursor& now, const Place& at, float* q) {
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -CUDART_INF_F, l[r] = 0.0f;
#pragma unroll 2
    for (int i = at.lane; i < R * (DP / 4); i += 32) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      const bool there = at.row0 + r < at.rows_here && d < p.c.head_dim;
      const CacheRow row = row_of<ROWS>(p, now, there ? at.row0 + r : 0);
      const float* const from = static_cast<const float*>(p.q) + now.b * p.q_stride[0] + row.token * p.q_stride[1] + row.head * p.q_stride[2];
      *reinterpret_cast<float4*>(q + i * 4) = there ? *reinterpret_cast<const float4*>(from + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < R / 2; ++i) o[c][i] = make_float2(0.0f, 0.0f);
  }

  template <bool CLEAN>
  __device__ __forceinline__ void times_values(const Place& at, const float* weights) {
    constexpr int kUnroll = CLEAN ? 1 : 4;
#pragma unroll kUnroll
    for (int k = 0; k < G::kKeys; ++k) {
      float x[C];
      constexpr int kAtOnce = C < 4 ? C : 4;
#pragma unroll
      for (int c = 0; c < C; c += kAtOnce) {
        const float* const from = G::at(at.v, k, C * at.lane + c);
        if constexpr (kAtOnce == 4) {
          const float4 v = *reinterpret_cast<const float4*>(from);
          x[c] = v.x, x[c + 1] = v.y, x[c + 2] = v.z, x[c + 3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(from);
          x[c] = v.x, x[c + 1] = v.y;
        }
      }
      float w[R];
#pragma unroll
      for (int r = 0; r < R; r += kVec) {
        const float* const from = weights + k * kWeightRow + r;
        if constexpr (kVec == 4) {
          const float4 v = *reinterpret_cast<const float4*>(from);
          w[r] = v.x, w[r + 1] = v.y, w[r + 2] = v.z, w[r + 3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(from);
          w[r] = v.x, w[r + 1] = v.y;
        }
      }
      if constexpr (CLEAN) {                         // infinities and NaN: to the rows that give them any weight; they are zero in the product
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (fabsf(x[c]) < CUDART_INF_F) continue;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (w[r] != 0.0f) (r & 1 ? o[c][r / 2].y : o[c][r / 2].x) += w[r] * x[c];
          x[c] = 0.0f;
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < R / 2; ++i) o[c][i] = ffma2(make_float2(w[2 * i], w[2 * i + 1]), make_float2(x[c], x[c]), o[c][i]);
    }
  }

  template <int ROWS, bool WINDOW>
  __device__ __forceinline__ void tile(const CacheAttnParams& p, const CacheCursor& now, const Place& at, uint32_t ahead, uint2* sees, const float* q, float* weights) {
    const int lane = at.lane;
    // Few rows: sums in two parts, so that half as many roundings follow each other (one token over 128 keys: 2.0e-7 to 3.3e-7 off, 2.9e-7 to 4.0e-7 in one part, in the
    // same time; with more rows there are no registers for it).
    constexpr int kSums = R <= 4 ? 2 : 1;
    float2 sum[KEYS][R][kSums];
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < kSums; ++j) sum[i][r][j] = make_float2(0.0f, 0.0f);
    const int key = lane % (32 / SHARE);
    const uint8_t* const k_row = at.k + key * 128;
    const int dims = p.c.head_dim / SHARE, first = lane / (32 / SHARE) * dims;       // (of 8 or more, a multiple of four)
#pragma unroll 4
    for (int d = 0; d < dims; d += 4) {
      const int at_d = first + d, in_row = (at_d / 32) * G::kBlockBytes + (((at_d % 32 / 4) ^ (key & 7)) << 4);
      float4 x[KEYS];
#pragma unroll
      for (int i = 0; i < KEYS; ++i) x[i] = *reinterpret_cast<const float4*>(k_row + i * 32 * 128 + in_row);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 y = *reinterpret_cast<const float4*>(q + r * DP + at_d);
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
          sum[i][r][0] = ffma2(make_float2(x[i].x, x[i].y), make_float2(y.x, y.y), sum[i][r][0]);
          sum[i][r][kSums - 1] = ffma2(make_float2(x[i].z, x[i].w), make_float2(y.z, y.w), sum[i][r][kSums - 1]);
        }
      }
    }
    float s[KEYS][R], top[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < KEYS; ++i) s[i][r] = kSums == 1 ? sum[i][r][0].x + sum[i][r][0].y : (sum[i][r][0].x + sum[i][r][0].y) + (sum[i][r][kSums - 1].x + sum[i][r][kSums - 1].y);
    if constexpr (SHARE > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int d = 32 / SHARE; d < 32; d *= 2) s[0][r] += __shfl_xor_sync(0xffffffffu, s[0][r], d);
    }
    const bool drafted = at.key0 + G::kKeys > at.sure || (WINDOW && window_hides(p, at.key0, G::kKeys, at.hidden));
    bool infinite = false;
    if (drafted) {
      look_at_mask<ROWS, R, G::kKeys, WINDOW>(p, now, at, ahead, sees);
      infinite = look_at_values<float, DP, WINDOW>(p, now, at);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint2 shows = sees[r];
#pragma unroll
        for (int i = 0; i < KEYS; ++i)
          if (!((i == 0 ? shows.x : shows.y) >> (key & 31) & 1)) s[i][r] = -CUDART_INF_F;
      }
    }
    bool grown = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      top[r] = s[0][r];
#pragma unroll
      for (int i = 1; i < KEYS; ++i) top[r] = fmaxf(top[r], s[i][r]);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
#pragma unroll
      for (int r = 0; r < R; ++r) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], d));
#pragma unroll
    for (int r = 0; r < R; ++r) grown = grown || top[r] > m[r];          // (the same in all lanes)
    if (grown) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        top[r] = fmaxf(top[r], m[r]);
        const float alpha = top[r] == -CUDART_INF_F ? 1.0f : ex2(exponent(m[r] - top[r], p.scale_log2));
        m[r] = top[r];
        l[r] *= alpha;
#pragma unroll
        for (int c = 0; c < C; ++c) (r & 1 ? o[c][r / 2].y : o[c][r / 2].x) *= alpha;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float shift = m[r] == -CUDART_INF_F ? 0.0f : m[r];           // nothing seen so far: every weight is 2^-inf
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        s[i][r] = ex2(exponent(s[i][r] - shift, p.scale_log2));
        if (SHARE == 1 || lane < 32 / SHARE) l[r] += s[i][r];
      }
    }
    if (SHARE == 1 || lane < 32 / SHARE) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i)
#pragma unroll
        for (int r = 0; r < R; r += kVec) {
          float* const to = weights + (key + 32 * i) * kWeightRow + r;
          if constexpr (kVec == 4) *reinterpret_cast<float4*>(to) = make_float4(s[i][r], s[i][r + 1], s[i][r + 2], s[i][r + 3]);
          else *reinterpret_cast<float2*>(to) = make_float2(s[i][r], s[i][r + 1]);
        }
    }
    __syncwarp();
    if (infinite) times_values<true>(at, weights);
    else times_values<false>(at, weights);
    if (drafted) fence_async_smem();
    __syncwarp();                                    // (the weights have been read)
  }

  __device__ __forceinline__ void sum_up() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int d = 16; d > 0; d /= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
      if (l[r] != l[r]) m[r] = 0.0f;
    }
  }
  __device__ __forceinline__ void put_states(int lane, float2* states) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (lane == r) states[r] = make_float2(m[r], l[r]);
  }
  __device__ __forceinline__ void rescale(int, const float* factors) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float f = factors[r];
#pragma unroll
      for (int c = 0; c < C; ++c) (r & 1 ? o[c][r / 2].y : o[c][r / 2].x) *= f;
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_out(F&& f) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < R / 2; ++i) f((c * (R / 2) + i) * 2, o[c][i].x), f((c * (R / 2) + i) * 2 + 1, o[c][i].y);
  }
  static __device__ __forceinline__ int place(int row, int d) { return ((d % C * (R / 2) + row / 2) * 2 + (row & 1)) * 32 + d / C; }
  // (by way of the query rows' place, so that a small loop does: a launch meets this code cold)
  template <int ROWS, bool WINDOW>
  __device__ __forceinline__ void write(const CacheAttnParams& p, const CacheCursor& now, const Place& at, const float2* states, float* query) {
    const int lane = at.lane;
    __syncwarp();
    each_out([&](int i, float x) { query[i * 32 + lane] = x; });
    __syncwarp();
#pragma unroll 2
    for (int i = lane; i < R * (DP / 2); i += 32) {
      const int in_warp = i / (DP / 2), row = at.row0 + in_warp, d = i % (DP / 2) * 2;
      if (row >= at.rows_here || d >= p.c.head_dim) continue;
      const float sum = states[in_warp].y, inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const CacheRow r = row_of<ROWS>(p, now, row);
      store2<float>(static_cast<float*>(p.out) + now.b * p.out_stride[0] + r.token * p.out_stride[1] + r.head * p.out_stride[2] + d,
                    query[place(in_warp, d)] * inv, query[place(in_warp, d + 1)] * inv);
      if constexpr (WINDOW) {
        if (d == 0) write_lse(p, now.b, r, log_sum(states[in_warp].x, sum, p.scale_log2));
      }
    }
    __syncwarp();
  }
};

}  // namespace cache_math
}  // namespace kb200
