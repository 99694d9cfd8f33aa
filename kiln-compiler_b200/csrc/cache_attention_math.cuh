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
// Does one of the elements in a 32-bit word hold an infinity or NaN?
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  if constexpr (sizeof(T) == 4) return (w & 0x7f800000u) == 0x7f800000u;
  else if constexpr (std::is_same<T, __half>::value) return (w & 0x7c000000u) == 0x7c000000u || (w & 0x7c00u) == 0x7c00u;
  else return (w & 0x7f800000u) == 0x7f800000u || (w & 0x7f80u) == 0x7f80u;
}
template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// Where a warp is: its tile and rows.
struct Place {
  uint8_t *k, *v;              // the stage
  int key0, sure;              // the tile's first key; keys that every row sees
  int row0, rows_here;         // the warp's first row of the item's row tile; rows of that
  int warp, lane, row_group, key_group;
};

// The keys of a tile with drafted tokens that the warp's rows see, a word per 32, by all lanes: row i of the warp's in sees[i].  All
// loads are in flight together (where there is nothing to look up they read the mask's first byte).
template <int ROWS, int WARP_ROWS, int KEYS>
__device__ __forceinline__ void look_at_mask(const CacheAttnParams& p, const CacheCursor& now, const Place& at, uint32_t (*sees)[2]) {
  constexpr int W = (KEYS + 31) / 32;
  uint8_t bytes[WARP_ROWS][W];
  const int first = now.row_tile * ROWS + at.row0;
  int token = first / p.group, in_group = first - token * p.group;
  const uint8_t* const mask = p.mask + now.b * p.mask_stride[0];
#pragma unroll
  for (int i = 0; i < WARP_ROWS; ++i) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int j = at.key0 + w * 32 + at.lane - now.it.length;
      const bool looked_up = j >= 0 && j < now.it.count && at.row0 + i < at.rows_here;
      bytes[i][w] = *(looked_up ? mask + token * p.mask_stride[1] + j * p.mask_stride[2] : p.mask);
    }
    if (++in_group == p.group) in_group = 0, ++token;
  }
#pragma unroll
  for (int i = 0; i < WARP_ROWS; ++i)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int key = at.key0 + w * 32 + at.lane;
      const bool visible = key < now.it.length || (bytes[i][w] != 0 && at.row0 + i < at.rows_here);
      const uint32_t word = __ballot_sync(0xffffffffu, visible && key < now.it.end && w * 32 + at.lane < KEYS);
      if (at.lane == 0) sees[i][w] = word;
    }
  __syncwarp();
}
// ... of a row where no mask is given: drafted tokens up to its own.
template <int ROWS>
__device__ __forceinline__ unsigned long long shown_by_order(const CacheAttnParams& p, const CacheCursor& now, const Place& at, int row) {
  const int n = min(now.it.end, now.it.length + row_of<ROWS>(p, now, row).token + 1) - at.key0;
  return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
}

// V behind the sequence's end is what an earlier tenant left, and V of a drafted token that some rows do not see may hold infinities or NaN; 0 times
// those is NaN.  True: such elements are among the tile's keys.  (The former are made zeros where the warp has the tile for itself.)
template <typename T, int DP, bool ALONE>
__device__ __forceinline__ bool look_at_values(const CacheCursor& now, const Place& at) {
  using G = Tile<T, DP>;
  const int last = now.it.end - at.key0;
  bool odd = false;
#pragma unroll 8
  for (int i = at.lane; i < G::kKeys * G::kBlocks * 8; i += 32) {
    const int key = i / (G::kBlocks * 8), chunk = i % (G::kBlocks * 8);
    uint4* const x = reinterpret_cast<uint4*>(G::at(at.v, key, chunk * (16 / (int)sizeof(T))));
    if (ALONE && key >= last) *x = make_uint4(0, 0, 0, 0);
    else if (key < last) odd = odd || not_finite<T>(x->x) || not_finite<T>(x->y) || not_finite<T>(x->z) || not_finite<T>(x->w);
  }
  odd = __any_sync(0xffffffffu, odd) != 0;
  __syncwarp();
  return odd;
}
// The warps that read a tile meet, make what must not enter the product zero, and meet again.  (Warps of other rows: each waits for all to
// have seen the tile as it was.)
template <int RG>
__device__ __forceinline__ void meet_rows(int key_group) {
  if constexpr (RG > 1) asm volatile("bar.sync %0, %1;" ::"r"(2 + key_group), "n"(32 * RG) : "memory");
  else __syncwarp();
}
template <typename T, int DP, int RG>
__device__ __forceinline__ void clear_values(const CacheCursor& now, const Place& at) {
  using G = Tile<T, DP>;
  meet_rows<RG>(at.key_group);
  const int last = now.it.end - at.key0;
  for (int i = at.row_group * 32 + at.lane; i < G::kKeys * DP; i += 32 * RG) {
    T* const x = G::at(at.v, i / DP, i % DP);
    if (i / DP >= last || !(fabsf(to_float(*x)) < CUDART_INF_F)) *x = T(0.0f);
  }
  meet_rows<RG>(at.key_group);
}

// 16-bit caches: mma.sync m16n8k16, the scores' accumulators being the weights' operands.  A thread holds rows g and g + 8.
template <typename T, int DP, int RG>
struct MmaMath {
  using Type = T;
  static constexpr int kDim = DP, kRows = 16, kOut = DP / 2;             // rows of a warp; output registers of a thread
  using G = Tile<T, DP>;
  static constexpr int NT = G::kKeys / 8, DT = DP / 8;                   // 8-wide column tiles of the scores, of the output rows
  uint32_t q[DP / 16][4];
  float o[DT][4], m[2], l[2];

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

  template <int ROWS>
  __device__ __forceinline__ void tile(const CacheAttnParams& p, const CacheCursor& now, const Place& at, uint32_t (*sees)[2]) {
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

    const bool drafted = at.key0 + G::kKeys > at.sure;
    bool infinite = false;
    unsigned long long shows[2] = {~0ull, ~0ull};    // the tile's keys that rows g and g + 8 see
    if (drafted) {
      if (p.mask != nullptr) look_at_mask<ROWS, 16, G::kKeys>(p, now, at, sees);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        shows[h] = p.mask == nullptr ? shown_by_order<ROWS>(p, now, at, at.row0 + g + 8 * h)
                                     : sees[g + 8 * h][0] | (G::kKeys > 32 ? (unsigned long long)sees[g + 8 * h][1] << 32 : 0ull);
      infinite = look_at_values<T, DP, RG == 1>(now, at);
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
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2)) * p.scale_log2;
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
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] = ex2(fmaf(s[n][j], p.scale_log2, shift[j >> 1]));
        l[j >> 1] += s[n][j];
      }

    if (infinite)                                    // such elements are added to the rows that see them one by one, and are zero in the product
      for (int key = 0; key < G::kKeys; ++key)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = to_float(*G::at(at.v, key, d * 8 + t4 * 2 + (j & 1)));
            if (!(fabsf(x) < CUDART_INF_F) && (shows[j >> 1] >> key & 1)) o[d][j] += x;
          }
    if (drafted && (RG > 1 || infinite)) clear_values<T, DP, RG>(now, at);

    const uint32_t v_row = v_tile + (((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
#pragma unroll
    for (int k = 0; k < NT / 2; ++k) {
      const uint32_t a[4] = {pack<T>(s[2 * k][0], s[2 * k][1]), pack<T>(s[2 * k][2], s[2 * k][3]), pack<T>(s[2 * k + 1][0], s[2 * k + 1][1]),
                             pack<T>(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
      for (int d = 0; d < DT; d += 2) {
        uint32_t b[4];
        ldmatrix4_t(b, v_row + k * 16 * 128 + (d / 8) * G::kBlockBytes + (((d % 8 + (lane >> 4)) ^ (lane & 7)) << 4));
        mma16<T>(o[d], a, b[0], b[1]);
        mma16<T>(o[d + 1], a, b[2], b[3]);
      }
    }
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
  // Maxima and sums of the warp's rows out and in, f(row, maximum, sum) once per row ...
  template <typename F>
  __device__ __forceinline__ void states(int lane, F&& f) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if ((lane & 3) == 0) f((lane >> 2) + 8 * h, m[h], l[h]);
  }
  // ... to a new maximum, top(row), and with another warp's sums added, more(row).
  template <typename F>
  __device__ __forceinline__ void rescale(int lane, F&& top) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float t = top((lane >> 2) + 8 * h), mine = m[h] == -CUDART_INF_F ? 0.0f : ex2(m[h] - t);
      l[h] *= mine;
      m[h] = t;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][2 * h] *= mine, o[d][2 * h + 1] *= mine;
    }
  }
  template <typename F>
  __device__ __forceinline__ void add_sums(int lane, F&& more) {
#pragma unroll
    for (int h = 0; h < 2; ++h) l[h] += more((lane >> 2) + 8 * h);
  }
  template <typename F>
  __device__ __forceinline__ void each_out(F&& f) {
#pragma unroll
    for (int i = 0; i < kOut; ++i) f(i, o[i / 4][i % 4]);
  }
  // f(row, its sum, its maximum, a function that hands the row's columns over: f2(column, two values))
  template <typename F>
  __device__ __forceinline__ void each_row(int lane, F&& f) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      f((lane >> 2) + 8 * h, l[h], m[h], (lane & 3) == 0, [&](auto&& f2) {
#pragma unroll
        for (int d = 0; d < DT; ++d) f2(d * 8 + (lane & 3) * 2, o[d][2 * h], o[d][2 * h + 1]);
      });
  }
};

// float32 caches: multiply-adds, two to an instruction.  (Three TF32 products of split operands by mma.sync took 9200 cycles for 64 keys of 64, whatever
// the number of rows, and lost a bit: these take ~1000 for 4 rows and ~3300 for 16.)  For the scores a lane has keys (two lanes share one where a
// tile has 16), for the output it has DP / 32 columns of all rows; weights go from one to the other through shared memory.
template <int DP, int R, int RG>
struct FmaMath {
  using Type = float;
  static constexpr int kDim = DP, kRows = R, kOut = R * DP / 32;
  using G = Tile<float, DP>;
  static constexpr int KEYS = G::kKeys >= 32 ? G::kKeys / 32 : 1;        // of a lane
  static constexpr int SHARE = G::kKeys >= 32 ? 1 : 32 / G::kKeys;       // lanes to a key, each with part of the columns
  static constexpr int C = DP / 32;                                      // output columns of a lane: C lane .. C lane + C - 1
  float2 o[C][R / 2];                                // rows 2i and 2i + 1
  float m[R], l[R];                                  // (l: of the lane's keys)

  // The query rows go to shared memory, [R][DP] of the warp's own.
  template <int ROWS>
  __device__ __forceinline__ void begin(const CacheAttnParams& p, const CacheCursor& now, const Place& at, float* q) {
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -CUDART_INF_F, l[r] = 0.0f;
#pragma unroll 8
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

  template <int ROWS>
  __device__ __forceinline__ void tile(const CacheAttnParams& p, const CacheCursor& now, const Place& at, uint32_t (*sees)[2], const float* q, float* weights) {
    const int lane = at.lane;
    float2 sum[KEYS][R];
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) sum[i][r] = make_float2(0.0f, 0.0f);
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
          sum[i][r] = ffma2(make_float2(x[i].x, x[i].y), make_float2(y.x, y.y), sum[i][r]);
          sum[i][r] = ffma2(make_float2(x[i].z, x[i].w), make_float2(y.z, y.w), sum[i][r]);
        }
      }
    }
    const bool drafted = at.key0 + G::kKeys > at.sure;
    bool infinite = false;
    if (drafted) {
      if (p.mask != nullptr) look_at_mask<ROWS, R, G::kKeys>(p, now, at, sees);
      infinite = look_at_values<float, DP, RG == 1>(now, at);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[KEYS], top = -CUDART_INF_F;
      unsigned long long shows = ~0ull;
      if (drafted) shows = p.mask == nullptr ? shown_by_order<ROWS>(p, now, at, at.row0 + r) : sees[r][0] | (G::kKeys > 32 ? (unsigned long long)sees[r][1] << 32 : 0ull);
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        s[i] = sum[i][r].x + sum[i][r].y;
#pragma unroll
        for (int d = 32 / SHARE; d < 32; d *= 2) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
        s[i] = shows >> (key + 32 * i) & 1 ? s[i] * p.scale_log2 : -CUDART_INF_F;
        top = fmaxf(top, s[i]);
      }
#pragma unroll
      for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      if (top > m[r]) {                              // (the same in all lanes)
        const float alpha = ex2(m[r] - top);
        m[r] = top;
        l[r] *= alpha;
#pragma unroll
        for (int c = 0; c < C; ++c) (r & 1 ? o[c][r / 2].y : o[c][r / 2].x) *= alpha;
      }
      const float shift = m[r] == -CUDART_INF_F ? 0.0f : m[r];
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        s[i] = ex2(s[i] - shift);
        if (lane < 32 / SHARE) l[r] += s[i];
        if (SHARE == 1 || lane < 32 / SHARE) weights[(key + 32 * i) * R + r] = s[i];
      }
    }
    __syncwarp();
    if (infinite) {
      for (int k = 0; k < G::kKeys; ++k)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float x = *G::at(at.v, k, C * lane + c);
          if (fabsf(x) < CUDART_INF_F) continue;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const unsigned long long shows = p.mask == nullptr ? shown_by_order<ROWS>(p, now, at, at.row0 + r)
                                                               : sees[r][0] | (G::kKeys > 32 ? (unsigned long long)sees[r][1] << 32 : 0ull);
            if (shows >> k & 1) (r & 1 ? o[c][r / 2].y : o[c][r / 2].x) += x;
          }
        }
    }
    if (drafted && (RG > 1 || infinite)) clear_values<float, DP, RG>(now, at);
#pragma unroll 4
    for (int k = 0; k < G::kKeys; ++k) {
      float x[C];
      constexpr int kVec = C < 4 ? C : 4;
#pragma unroll
      for (int c = 0; c < C; c += kVec) {
        const float* const from = G::at(at.v, k, C * lane + c);
        if constexpr (kVec == 4) *reinterpret_cast<float4*>(x + c) = *reinterpret_cast<const float4*>(from);
        else *reinterpret_cast<float2*>(x + c) = *reinterpret_cast<const float2*>(from);
      }
      float w[R];
      if constexpr (R >= 4) {
#pragma unroll
        for (int r = 0; r < R; r += 4) *reinterpret_cast<float4*>(w + r) = *reinterpret_cast<const float4*>(weights + k * R + r);
      } else {
        *reinterpret_cast<float2*>(w) = *reinterpret_cast<const float2*>(weights + k * R);
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < R / 2; ++i) o[c][i] = ffma2(make_float2(w[2 * i], w[2 * i + 1]), make_float2(x[c], x[c]), o[c][i]);
    }
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
  template <typename F>
  __device__ __forceinline__ void states(int lane, F&& f) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (lane == r) f(r, m[r], l[r]);
  }
  template <typename F>
  __device__ __forceinline__ void rescale(int, F&& top) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float t = top(r), mine = m[r] == -CUDART_INF_F ? 0.0f : ex2(m[r] - t);
      l[r] *= mine;
      m[r] = t;
#pragma unroll
      for (int c = 0; c < C; ++c) (r & 1 ? o[c][r / 2].y : o[c][r / 2].x) *= mine;
    }
  }
  template <typename F>
  __device__ __forceinline__ void add_sums(int, F&& more) {
#pragma unroll
    for (int r = 0; r < R; ++r) l[r] += more(r);
  }
  template <typename F>
  __device__ __forceinline__ void each_out(F&& f) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < R / 2; ++i) f((c * (R / 2) + i) * 2, o[c][i].x), f((c * (R / 2) + i) * 2 + 1, o[c][i].y);
  }
  template <typename F>
  __device__ __forceinline__ void each_row(int lane, F&& f) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
      f(r, l[r], m[r], lane == 0, [&](auto&& f2) {
#pragma unroll
        for (int c = 0; c < C; c += 2)
          f2(C * lane + c, r & 1 ? o[c][r / 2].y : o[c][r / 2].x, r & 1 ? o[c + 1][r / 2].y : o[c + 1][r / 2].x);
      });
  }
};

}  // namespace cache_math
}  // namespace kb200
