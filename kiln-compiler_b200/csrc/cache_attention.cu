// Attention of drafted tokens over a paged K/V cache (kb200_cache_attend): softmax(scale q K^T, masked) V for the few query rows of
// each sequence, one pass over its keys with a running maximum and sum.
//
// What bounds it: the cache's bytes.  A key head's K and V are read once for all query rows that share them (drafted tokens x heads per key head).
// Products run on the tensor cores by warp (mma.sync): the rows of a decoding step do not fill more, and at up to ~64 rows per key
// they take less time than the bytes.
//
// A CTA of four warps walks its run of key tiles (cache_attention.h).  K and V tiles come by asynchronous 16-byte copies, kStages tiles in
// flight across the borders of sequences and heads, rows found through the page table a tile ahead.  With
// 16 query rows the warps take 16 keys of a tile each and join their sums at the end of an item; with 32 or 64 rows two or four of them take rows.
// Scores, maxima, sums and output rows are float32 in registers.  16-bit caches: the weights of a tile are rounded to the cache's type for the product with V
// (half a step, 2^-9 for bfloat16, of every summand; the sum of the weights is kept of the unrounded ones).  float32 caches: both operands of both
// products as a TF32 head and tail, three products; what is dropped is 2^-22 of a summand.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "cache_attention.h"
#include "tc_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

constexpr int kThreads = 128;

// Sizes by type and padded head width.  A tile's rows are padded so that the fragments' loads do not collide in
// shared memory: 16-bit rows by 16 bytes (ldmatrix), float32 K rows by 32 (64-bit loads), V rows by 16 bytes (rows 2t, 2t + 1 by four lanes).
template <typename T, int DP>
struct Shape {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kTile = kWide && DP > 64 ? 32 : 64;               // keys
  static constexpr int kPadK = kWide ? 8 : 8, kPadV = kWide ? 4 : 8;
  static constexpr int kRowK = DP + kPadK, kRowV = DP + kPadV;           // elements
  static constexpr int kStageBytes = kTile * (kRowK + kRowV) * (int)sizeof(T);
  static constexpr int kStages = kStageBytes > 40000 ? 2 : 3;
  static constexpr int kChunks = DP * (int)sizeof(T) / 16;               // 16-byte chunks of a padded row
  static constexpr int kRowsPerPass = kThreads / kChunks;
  static constexpr int kPasses = kTile / kRowsPerPass;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {      // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as a TF32 head, rounded to nearest, and the rest, rounded as well.
__device__ __forceinline__ void split(float x, uint32_t* head, uint32_t* tail) {
  uint32_t h, t;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(h) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(t) : "f"(x - __uint_as_float(h)));
  *head = h;
  *tail = t;
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
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// Where a run is: an item (batch row, key head, row tile) and a key tile of it.
struct Cursor {
  int b, head, row_tile, tile;
  CacheItems it;
};
template <int ROWS, int TILE>
__device__ __forceinline__ void to_row(const CacheAttnParams& p, Cursor& u, int b) {       // the first batch row from b on that has units
  u.b = b;
  u.head = u.row_tile = u.tile = 0;
  while (u.b < p.rows) {
    u.it = cache_items<ROWS, TILE>(p, u.b);
    if (u.it.units > 0) return;
    ++u.b;
  }
}
template <int ROWS, int TILE>
__device__ __forceinline__ bool advance(const CacheAttnParams& p, Cursor& u) {      // true: another item
  if (++u.tile < u.it.key_tiles) return false;
  u.tile = 0;
  if (++u.row_tile == u.it.row_tiles) {
    u.row_tile = 0;
    if (++u.head == p.c.kv_heads) to_row<ROWS, TILE>(p, u, u.b + 1);
  }
  return true;
}

// All units, and the run of the CTA `part`.  shared: 2 * 4 values.
template <int ROWS, int TILE>
__device__ int64_t find_run(const CacheAttnParams& p, int part, int64_t* shared, int64_t* lo, int64_t* hi, int* parts, Cursor* at) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t all = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.rows; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const int64_t units = b < p.rows ? cache_items<ROWS, TILE>(p, b).units : 0;
      int64_t sum = units;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int64_t below = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += below;
      }
      __syncthreads();
      if (lane == 31) shared[warp] = sum;
      __syncthreads();
      int64_t before = 0, total = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        before += w < warp ? shared[w] : 0;
        total += shared[w];
      }
      const int64_t from = base + before + sum - units;
      if (pass == 1 && *lo >= from && *lo < from + units) shared[4] = b, shared[5] = *lo - from;
      base += total;
    }
    if (pass == 0) {
      all = base;
      const int64_t n = min((int64_t)p.parts, (all + p.min_units - 1) / p.min_units);
      *parts = (int)n;
      if (part >= n) return all;
      *lo = all * part / n;
      *hi = all * (part + 1) / n;
    }
  }
  __syncthreads();
  at->b = (int)shared[4];
  int64_t rest = shared[5];
  at->it = cache_items<ROWS, TILE>(p, at->b);
  const int64_t per_head = (int64_t)at->it.row_tiles * at->it.key_tiles;
  at->head = (int)(rest / per_head);
  rest -= at->head * per_head;
  at->row_tile = (int)(rest / at->it.key_tiles);
  at->tile = (int)(rest - (int64_t)at->row_tile * at->it.key_tiles);
  return all;
}

// A part: ROWS output rows (not divided by their sums), then their maxima and sums.
template <int DP, int ROWS>
constexpr int64_t part_floats() { return (int64_t)ROWS * (DP + 2); }

template <typename T, int DP, int RW>
__global__ void __launch_bounds__(kThreads) cache_attention_kernel(const __grid_constant__ CacheAttnParams p) {
  using Z = Shape<T, DP>;
  constexpr int KW = 4 / RW, ROWS = 16 * RW, TILE = Z::kTile;
  constexpr int KEYS = TILE / KW;                  // of a warp in a tile
  constexpr int NT = KEYS / 8, DT = DP / 8;        // 8-wide column tiles of its scores, of its output rows
  constexpr bool kWide = Z::kWide;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t run[6];
  __shared__ uint32_t sees[ROWS][TILE / 32];       // a tile with drafted tokens: which row sees which key
  __shared__ float states[4][16][2];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row_warp = warp % RW, key_warp = warp / RW;
  const int g = lane >> 2, t4 = lane & 3;          // fragment coordinates
  const uint32_t stage0 = tc::smem_u32(smem);
  float* const q_rows = reinterpret_cast<float*>(smem + Z::kStages * Z::kStageBytes);      // float32: the item's query rows, as wide as K's

  pdl_wait();
  pdl_launch_dependents();

  // rows behind a sequence's drafted tokens
  if (p.counts != nullptr) {
    const int width = p.heads * p.c.head_dim;
    for (int64_t r = blockIdx.x; r < (int64_t)p.rows * p.tokens; r += gridDim.x) {
      const int b = (int)(r / p.tokens), i = (int)(r % p.tokens);
      const int slot = p.slots != nullptr ? p.slots[b] : b;
      if (i < p.counts[b] && (unsigned)slot < (unsigned)p.c.sequences) continue;
      for (int x = threadIdx.x; x < width; x += kThreads)
        static_cast<T*>(p.out)[b * p.out_stride[0] + i * p.out_stride[1] + (x / p.c.head_dim) * p.out_stride[2] + x % p.c.head_dim] = T(0.0f);
    }
  } else if (p.slots != nullptr) {
    const int width = p.heads * p.c.head_dim;
    for (int64_t r = blockIdx.x; r < (int64_t)p.rows * p.tokens; r += gridDim.x) {
      const int b = (int)(r / p.tokens), i = (int)(r % p.tokens);
      if ((unsigned)p.slots[b] < (unsigned)p.c.sequences) continue;
      for (int x = threadIdx.x; x < width; x += kThreads)
        static_cast<T*>(p.out)[b * p.out_stride[0] + i * p.out_stride[1] + (x / p.c.head_dim) * p.out_stride[2] + x % p.c.head_dim] = T(0.0f);
    }
  }

  int64_t lo = 0, hi = 0;
  int parts;
  Cursor now;
  find_run<ROWS, TILE>(p, blockIdx.x, run, &lo, &hi, &parts, &now);
  if ((int)blockIdx.x >= parts || lo >= hi) return;
  __syncthreads();
  Cursor ahead = now;                              // the tile whose copies are issued next
  int64_t to_issue = hi - lo;

  // ---- copies ----
  const int chunk = threadIdx.x % Z::kChunks, first_row = threadIdx.x / Z::kChunks;
  const int in_page = (1 << p.c.page_log2) - 1;
  int pages[Z::kPasses];
  auto look_up = [&]() {                           // the pages of the rows that this thread copies of the tile `ahead`
#pragma unroll
    for (int i = 0; i < Z::kPasses; ++i) {
      const int at = ahead.tile * TILE + first_row + i * Z::kRowsPerPass;
      pages[i] = at < ahead.it.end
                     ? p.c.table[(int64_t)ahead.it.slot * p.c.max_pages + (at >> p.c.page_log2)] : -1;
    }
  };
  auto issue = [&](int stage) {
    if (to_issue > 0) {
      const uint32_t k_to = stage0 + stage * Z::kStageBytes, v_to = k_to + TILE * Z::kRowK * (int)sizeof(T);
      const int64_t v_from = ((int64_t)p.c.pages * p.c.kv_heads << p.c.page_log2) * p.c.row_chunks;
      if (chunk < p.c.row_chunks) {
#pragma unroll
        for (int i = 0; i < Z::kPasses; ++i) {
          const int row = first_row + i * Z::kRowsPerPass, at = ahead.tile * TILE + row;
          const bool there = cache_page_ok(p.c, pages[i]);
          if (!there && at < ahead.it.end) cache_fault(p.c, KB200_CACHE_BAD_INDEX);
          const uint4* const from = static_cast<const uint4*>(p.c.pool) +
                                    (there ? (cache_row(p.c, p.layer, 0, pages[i], ahead.head) + (at & in_page)) * p.c.row_chunks + chunk : 0);
          copy16(k_to + (row * Z::kRowK) * (int)sizeof(T) + chunk * 16, from, there);
          copy16(v_to + (row * Z::kRowV) * (int)sizeof(T) + chunk * 16, from + (there ? v_from : 0), there);
        }
      }
      --to_issue;
      if (to_issue > 0) {
        advance<ROWS, TILE>(p, ahead);
        look_up();
      }
    }
    copy_commit();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < Z::kStages - 1; ++i) issue(i);

  // ---- per item ----
  uint32_t q_frag[kWide ? 1 : DP / 16][4];
  float o[DT][4], m[2], l[2];
  int rows_here = 0;                               // of the item's row tile
  auto q_at = [&](int row) -> const void* {        // a row of the tile: token, then head of the group
    const int r = now.row_tile * ROWS + row;
    const int64_t at = now.b * p.q_stride[0] + (r / p.group) * p.q_stride[1] + (now.head * p.group + r % p.group) * p.q_stride[2];
    return static_cast<const uint8_t*>(p.q) + at * (kWide || p.q_fp32 ? 4 : 2);
  };
  auto begin = [&]() {
    rows_here = min(ROWS, now.it.count * p.group - now.row_tile * ROWS);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.0f;
    if constexpr (kWide) {
      __syncthreads();                             // (the last item's rows have been read)
      for (int i = threadIdx.x; i < ROWS * Z::kChunks; i += kThreads) {
        const int row = i / Z::kChunks, c = i % Z::kChunks;
        const float4 x = row < rows_here && c < p.c.row_chunks ? static_cast<const float4*>(q_at(row))[c] : make_float4(0, 0, 0, 0);
        *reinterpret_cast<float4*>(q_rows + row * Z::kRowK + c * 4) = x;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = row_warp * 16 + g + half * 8;
        const bool there = row < rows_here;
        const void* const from = there ? q_at(row) : nullptr;
        auto pair = [&](int i) {                   // two elements
          if (!p.q_fp32) return static_cast<const uint32_t*>(from)[i];
          const float2 x = static_cast<const float2*>(from)[i];
          return pack<T>(x.x, x.y);
        };
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const bool in = there && k * 16 < p.c.head_dim;
          q_frag[k][half] = in ? pair(k * 8 + t4) : 0u;
          q_frag[k][2 + half] = in ? pair(k * 8 + 4 + t4) : 0u;
        }
      }
    }
  };

  // ---- a tile ----
  auto compute = [&](int stage) {
    T* const k_tile = reinterpret_cast<T*>(smem + stage * Z::kStageBytes);
    T* const v_tile = k_tile + TILE * Z::kRowK;
    const int key0 = now.tile * TILE, end = now.it.end;
    const bool drafted = key0 + TILE > now.it.length;
    bool infinite = false;
    if (drafted) {
      // Which row sees which key: a ballot per row and 32 keys.
      for (int i = warp; i < ROWS * (TILE / 32); i += kThreads / 32) {
        const int row = i / (TILE / 32), key = key0 + (i % (TILE / 32)) * 32 + lane;
        const int token = (now.row_tile * ROWS + row) / p.group, j = key - now.it.length;
        bool s = key < now.it.length;
        if (!s && key < end && row < rows_here)
          s = p.mask == nullptr ? j <= token : p.mask[now.b * p.mask_stride[0] + token * p.mask_stride[1] + j * p.mask_stride[2]] != 0;
        const uint32_t word = __ballot_sync(0xffffffffu, s && key < end);
        if (lane == 0) sees[row][i % (TILE / 32)] = word;
      }
      // V of a drafted token that some rows do not see may hold infinities or NaN, and 0 times those is NaN: such elements are added to the rows that see them one by
      // one, below, and are zero in the product.
      bool odd = false;
      for (int i = threadIdx.x; i < TILE * Z::kChunks; i += kThreads) {
        if (i % Z::kChunks >= p.c.row_chunks) continue;
        const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(v_tile) + (i / Z::kChunks) * Z::kRowV * (int)sizeof(T) + (i % Z::kChunks) * 16);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kWide) odd = odd || (w[j] & 0x7f800000u) == 0x7f800000u;
          else if constexpr (std::is_same<T, __half>::value) odd = odd || (w[j] & 0x7c000000u) == 0x7c000000u || (w[j] & 0x7c00u) == 0x7c00u;
          else odd = odd || (w[j] & 0x7f800000u) == 0x7f800000u || (w[j] & 0x7f80u) == 0x7f80u;
        }
      }
      infinite = __syncthreads_or(odd) != 0;
    }

    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
    if constexpr (!kWide) {
      const uint32_t at = tc::smem_u32(k_tile) + ((key_warp * KEYS + (lane >> 4) * 8 + (lane & 7)) * Z::kRowK + ((lane >> 3) & 1) * 8) * 2;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          if (k * 16 >= p.c.head_dim) continue;    // (columns behind the head's hold anything)
          uint32_t b[4];
          ldmatrix4(b, at + (n * 8 * Z::kRowK + k * 16) * 2);
          mma16<T>(s[n], q_frag[k], b[0], b[1]);
          mma16<T>(s[n + 1], q_frag[k], b[2], b[3]);
        }
    } else {
      // dims 2t and 2t + 1 of eight stand in fragment columns t and t + 4, in both operands: 64-bit loads
      const float* const q0 = q_rows + (row_warp * 16 + g) * Z::kRowK + 2 * t4;
      const float* const k0 = reinterpret_cast<const float*>(k_tile) + (key_warp * KEYS + g) * Z::kRowK + 2 * t4;
#pragma unroll 4
      for (int k = 0; k < p.c.head_dim / 8; ++k) {
        const float2 qa = *reinterpret_cast<const float2*>(q0 + k * 8), qb = *reinterpret_cast<const float2*>(q0 + 8 * Z::kRowK + k * 8);
        uint32_t ah[4], al[4];
        split(qa.x, ah + 0, al + 0);
        split(qb.x, ah + 1, al + 1);
        split(qa.y, ah + 2, al + 2);
        split(qb.y, ah + 3, al + 3);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float2 kb = *reinterpret_cast<const float2*>(k0 + n * 8 * Z::kRowK + k * 8);
          uint32_t bh[2], bl[2];
          split(kb.x, bh + 0, bl + 0);
          split(kb.y, bh + 1, bl + 1);
          mma_tf32(s[n], al, bh[0], bh[1]);
          mma_tf32(s[n], ah, bl[0], bl[1]);
          mma_tf32(s[n], ah, bh[0], bh[1]);
        }
      }
    }

    // ---- softmax: two rows of a thread, their keys over the four lanes of a group ----
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] *= p.scale_log2;
        if (drafted) {
          const int key = key_warp * KEYS + n * 8 + t4 * 2 + (j & 1);
          if (!(sees[row_warp * 16 + g + (j >> 1) * 8][key / 32] >> (key % 32) & 1)) s[n][j] = -CUDART_INF_F;
        }
        top[j >> 1] = fmaxf(top[j >> 1], s[n][j]);
      }
    float shift[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      shift[h] = top[h] == -CUDART_INF_F ? 0.0f : top[h];          // nothing seen so far: every weight is 2^-inf
      const float alpha = ex2(m[h] - shift[h]);
      m[h] = top[h];
      l[h] *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][2 * h] *= alpha, o[d][2 * h + 1] *= alpha;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] = ex2(s[n][j] - shift[j >> 1]);
        l[j >> 1] += s[n][j];
      }

    if (infinite) {
      for (int key = key_warp * KEYS; key < (key_warp + 1) * KEYS; ++key)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = to_float(v_tile[key * Z::kRowV + d * 8 + t4 * 2 + (j & 1)]);
            if (!(fabsf(x) < CUDART_INF_F) && (sees[row_warp * 16 + g + (j >> 1) * 8][key / 32] >> (key % 32) & 1)) o[d][j] += x;
          }
      __syncthreads();
      for (int i = threadIdx.x; i < TILE * DP; i += kThreads) {
        T& x = v_tile[(i / DP) * Z::kRowV + i % DP];
        if (!(fabsf(to_float(x)) < CUDART_INF_F)) x = T(0.0f);
      }
      __syncthreads();
    }

    // ---- P V ----
    if constexpr (!kWide) {
      const uint32_t at = tc::smem_u32(v_tile) + ((key_warp * KEYS + ((lane >> 3) & 1) * 8 + (lane & 7)) * Z::kRowV + (lane >> 4) * 8) * 2;
#pragma unroll
      for (int k = 0; k < KEYS / 16; ++k) {
        const uint32_t a[4] = {pack<T>(s[2 * k][0], s[2 * k][1]), pack<T>(s[2 * k][2], s[2 * k][3]), pack<T>(s[2 * k + 1][0], s[2 * k + 1][1]),
                               pack<T>(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
        for (int d = 0; d < DT; d += 2) {
          uint32_t b[4];
          ldmatrix4_t(b, at + (k * 16 * Z::kRowV + d * 8) * 2);
          mma16<T>(o[d], a, b[0], b[1]);
          mma16<T>(o[d + 1], a, b[2], b[3]);
        }
      }
    } else {
      // keys 2t and 2t + 1 of eight stand in fragment columns t and t + 4: the scores are where the product wants them
      const float* const v0 = reinterpret_cast<const float*>(v_tile) + (key_warp * KEYS + 2 * t4) * Z::kRowV + g;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        uint32_t ah[4], al[4];
        split(s[k][0], ah + 0, al + 0);
        split(s[k][2], ah + 1, al + 1);
        split(s[k][1], ah + 2, al + 2);
        split(s[k][3], ah + 3, al + 3);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          uint32_t bh[2], bl[2];
          split(v0[k * 8 * Z::kRowV + d * 8], bh + 0, bl + 0);
          split(v0[(k * 8 + 1) * Z::kRowV + d * 8], bh + 1, bl + 1);
          mma_tf32(o[d], al, bh[0], bh[1]);
          mma_tf32(o[d], ah, bl[0], bl[1]);
          mma_tf32(o[d], ah, bh[0], bh[1]);
        }
      }
    }
  };

  // ---- the end of an item, or of the run inside one: the warps' sums, then the rows or a part ----
  auto finish = [&](int stage, bool whole, int64_t slot) {
    float* const sums = reinterpret_cast<float*>(smem + stage * Z::kStageBytes);     // (the tile has been read; nothing is copied to it before the next one)
    constexpr int kRow = DP + 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (l[h] != l[h]) m[h] = 0.0f;               // (NaN, which a maximum passes over, reaches the result)
      if (t4 == 0) states[warp][g + 8 * h][0] = m[h], states[warp][g + 8 * h][1] = l[h];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < KW; ++w) top = fmaxf(top, states[w * RW + row_warp][g + 8 * h][0]);
      const float mine = m[h] == -CUDART_INF_F ? 0.0f : ex2(m[h] - top);
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<float2*>(sums + (warp * 16 + g + 8 * h) * kRow + d * 8 + t4 * 2) = make_float2(o[d][2 * h] * mine, o[d][2 * h + 1] * mine);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * (DP / 4); i += kThreads) {
      const int row = i / (DP / 4), d = i % (DP / 4) * 4;
      if (row >= rows_here || d >= p.c.head_dim) continue;
      float top = -CUDART_INF_F, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < KW; ++w) top = fmaxf(top, states[w * RW + row / 16][row % 16][0]);
      float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float* const st = states[w * RW + row / 16][row % 16];
        sum += st[0] == -CUDART_INF_F ? 0.0f : st[1] * ex2(st[0] - top);
        const float4 y = *reinterpret_cast<const float4*>(sums + ((w * RW + row / 16) * 16 + row % 16) * kRow + d);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int r = now.row_tile * ROWS + row;
        T* const to = static_cast<T*>(p.out) + now.b * p.out_stride[0] + (r / p.group) * p.out_stride[1] + (now.head * p.group + r % p.group) * p.out_stride[2] + d;
        if constexpr (kWide) *reinterpret_cast<float4*>(to) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        else *reinterpret_cast<uint2*>(to) = make_uint2(pack<T>(x.x * inv, x.y * inv), pack<T>(x.z * inv, x.w * inv));
      } else {
        float* const part = p.partial + slot * p.partial_floats;
        *reinterpret_cast<float4*>(part + (int64_t)row * DP + d) = x;
        if (d == 0) part[ROWS * DP + row] = top, part[ROWS * DP + ROWS + row] = sum;
      }
    }
  };

  int stage = 0;
  bool fresh = true;
  int64_t first_tile = 0;
  for (int64_t u = lo; u < hi; ++u) {
    copy_wait<Z::kStages - 2>();
    __syncthreads();                               // everybody's copies of this tile; the tile before has been read
    issue((stage + Z::kStages - 1) % Z::kStages);
    if (fresh) {
      begin();
      first_tile = now.tile;
      fresh = false;
    }
    compute(stage);
    const bool ends = now.tile + 1 == now.it.key_tiles;
    if (ends || u + 1 == hi) {
      __syncthreads();                             // the tile has been read by all warps
      // a part that begins with the run is the run's first, else its second
      finish(stage, ends && first_tile == 0, 2 * (int64_t)blockIdx.x + (u - (now.tile - first_tile) == lo ? 0 : 1));
      fresh = true;
    }
    if (u + 1 < hi) advance<ROWS, TILE>(p, now);
    stage = (stage + 1) % Z::kStages;
  }
  copy_wait<0>();
}

// Joins the parts of an item.  CTA x sees to the item that ends in the run of CTA x of the first launch and began before it.
template <typename T, int DP, int RW, int TILE>
__global__ void __launch_bounds__(kThreads) cache_attention_join_kernel(const __grid_constant__ CacheAttnParams p) {
  constexpr int ROWS = 16 * RW;
  __shared__ int64_t run[6];
  pdl_wait();
  pdl_launch_dependents();
  int64_t lo = 0, hi = 0;
  int parts;
  Cursor at;
  const int64_t all = find_run<ROWS, TILE>(p, blockIdx.x, run, &lo, &hi, &parts, &at);
  if ((int)blockIdx.x >= parts || lo >= hi || at.tile == 0 || at.it.key_tiles - at.tile > hi - lo) return;
  const int64_t begins = lo - at.tile;             // the item's first unit
  int first = (int)(((begins + 1) * parts - 1) / all);       // the run that it is in
  const int rows_here = min(ROWS, at.it.count * p.group - at.row_tile * ROWS);
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < rows_here * (DP / 4); i += gridDim.y * kThreads) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= p.c.head_dim) continue;
    float top = -CUDART_INF_F, sum = 0.0f;
    float4 x = make_float4(0, 0, 0, 0);
    for (int r = first; r <= (int)blockIdx.x; ++r) {
      // (a run that the item begins in, but not with, has left it as its second part)
      const int64_t slot = 2 * (int64_t)r + (r == first && all * r / parts != begins ? 1 : 0);
      const float* const part = p.partial + slot * p.partial_floats;
      const float m = part[ROWS * DP + row], l = part[ROWS * DP + ROWS + row];
      if (m == -CUDART_INF_F) continue;
      const float4 y = *reinterpret_cast<const float4*>(part + (int64_t)row * DP + d);
      const float next = fmaxf(top, m), a = ex2(top - next), b = ex2(m - next);
      sum = sum * a + l * b;
      x.x = x.x * a + y.x * b, x.y = x.y * a + y.y * b, x.z = x.z * a + y.z * b, x.w = x.w * a + y.w * b;
      top = next;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int r = at.row_tile * ROWS + row;
    T* const to = static_cast<T*>(p.out) + at.b * p.out_stride[0] + (r / p.group) * p.out_stride[1] + (at.head * p.group + r % p.group) * p.out_stride[2] + d;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    else *reinterpret_cast<uint2*>(to) = make_uint2(pack<T>(x.x * inv, x.y * inv), pack<T>(x.z * inv, x.w * inv));
  }
}

// ---- host --------------------------------------------------------------------------------------

struct Variant {
  void (*kernel)(CacheAttnParams);
  void (*join)(CacheAttnParams);
  int smem, rows, tile;            // rows and keys of a tile
  int64_t part_floats;
};

template <typename T, int DP, int RW>
Variant variant() {
  using Z = Shape<T, DP>;
  return Variant{cache_attention_kernel<T, DP, RW>, cache_attention_join_kernel<T, DP, RW, Z::kTile>,
                 Z::kStages * Z::kStageBytes + (Z::kWide ? 16 * RW * Z::kRowK * 4 : 0), 16 * RW, Z::kTile, part_floats<DP, 16 * RW>()};
}

// Tiles of 16, 32 and 64 query rows (64 where the registers, for float32 also the shared memory, allow it).
template <typename T>
Variant variant_of(int head_dim, int index) {
  if (head_dim <= 64) return index == 0 ? variant<T, 64, 1>() : index == 1 ? variant<T, 64, 2>() : variant<T, 64, 4>();
  if constexpr (sizeof(T) == 2)
    if (head_dim <= 128) return index == 0 ? variant<T, 128, 1>() : index == 1 ? variant<T, 128, 2>() : variant<T, 128, 4>();
  if (head_dim <= 128) return index == 0 ? variant<T, 128, 1>() : variant<T, 128, 2>();
  return index == 0 ? variant<T, 256, 1>() : variant<T, 256, 2>();
}
Variant variant_at(const Cache& c, int index) {
  return c.dtype == KB200_DTYPE_FP32 ? variant_of<float>(c.view.head_dim, index)
         : c.dtype == KB200_DTYPE_BF16 ? variant_of<__nv_bfloat16>(c.view.head_dim, index) : variant_of<__half>(c.view.head_dim, index);
}

// As many rows to a tile as there are: every row tile reads the keys again.
int variant_index(const Cache& c, int tokens, int heads) {
  const int64_t rows = (int64_t)tokens * (heads / c.view.kv_heads);
  return rows <= 16 ? 0 : rows <= 32 ? 1 : 2;
}

// CTAs that share the work: all that fit, but no more than there can be units.
int parts_of(const Cache& c, const Variant& v, int resident, int rows, int tokens, int heads) {
  const int64_t row_tiles = ((int64_t)tokens * (heads / c.view.kv_heads) + v.rows - 1) / v.rows;
  const int64_t tiles = (((int64_t)c.view.max_pages << c.view.page_log2) + v.tile - 1) / v.tile;
  const double units = (double)rows * c.view.kv_heads * row_tiles * tiles;
  return (int)std::min<double>(units, (double)c.sm_count * resident);
}

Cache* cache_of(const kb200_cache* c) { return reinterpret_cast<Cache*>(const_cast<kb200_cache*>(c)); }

bool call_ok(const Cache& c, int rows, int tokens, int heads) {
  return rows >= 0 && tokens >= 0 && heads >= 1 && heads % c.view.kv_heads == 0 && (int64_t)tokens * (heads / c.view.kv_heads) < (1 << 24) &&
         (int64_t)rows * std::max(tokens, 1) < ((int64_t)1 << 31);
}

}  // namespace

int cache_attention_prepare(Cache& c) {
  for (int i = 0; i < 3; ++i) {
    const Variant v = variant_at(c, i);
    KB200_CUDA(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem));
    KB200_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&c.attention_resident[i], v.kernel, kThreads, v.smem));
    if (c.attention_resident[i] < 1) return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: the attention kernel does not fit this GPU");
  }
  return KB200_OK;
}

}  // namespace kb200

using namespace kb200;

KB200_EXPORT uint64_t kb200_cache_attend_workspace(const kb200_cache* handle, int rows, int tokens, int heads) {
  if (handle == nullptr) return 0;
  const Cache& c = *cache_of(handle);
  if (!call_ok(c, rows, tokens, heads) || rows == 0 || tokens == 0) return 0;
  const int index = variant_index(c, tokens, heads);
  const Variant v = variant_at(c, index);
  return (uint64_t)parts_of(c, v, c.attention_resident[index], rows, tokens, heads) * 2 * v.part_floats * sizeof(float);
}

KB200_EXPORT int kb200_cache_attend(kb200_cache* handle, int layer, const kb200_rows* q, const kb200_rows* out, int rows, int tokens,
                                    const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale,
                                    void* workspace, uint64_t workspace_bytes, void* stream) {
  if (handle == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: cache is null");
  const Cache& c = *cache_of(handle);
  if (layer < 0 || layer >= c.view.layers) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: layer %d of %d", layer, c.view.layers);
  if (q == nullptr || out == nullptr || q->heads != out->heads || !call_ok(c, rows, tokens, q->heads) || (slots == nullptr && rows > c.view.sequences))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: rows and tokens do not suit the cache, or heads are no multiple of its %d", c.view.kv_heads);
  if (rows == 0 || tokens == 0) return KB200_OK;
  for (const kb200_rows* r : {q, out}) {
    const bool wide = r->dtype == KB200_DTYPE_FP32;
    if (r->data == nullptr || !tc::aligned16(r->data) || (r->dtype != c.dtype && (r == out || !wide)))
      return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: q and out must be of the cache's type (q of that or float32) and on 16 bytes");
    for (const int64_t s : r->stride)
      if (s % (wide ? 4 : 8) != 0) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: strides of q and out must be multiples of 16 bytes");
  }
  if (mask != nullptr && mask_stride == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: a mask without strides");
  if (!(scale > 0.0f) || !(scale < 1e30f)) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: scale must be positive and finite");
  const int index = variant_index(c, tokens, q->heads);
  const Variant v = variant_at(c, index);
  const int parts = parts_of(c, v, c.attention_resident[index], rows, tokens, q->heads);
  const uint64_t need = (uint64_t)parts * 2 * v.part_floats * sizeof(float);
  if (workspace == nullptr || !tc::aligned16(workspace) || workspace_bytes < need)
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: a workspace of %llu bytes on 16 bytes is needed", (unsigned long long)need);
  const DeviceGuard guard(c.device);
  if (guard.error != cudaSuccess) return cuda_fail(guard.error, "kb200_cache_attend");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  CacheAttnParams p{};
  p.c = c.view;
  p.q = q->data;
  p.out = out->data;
  for (int i = 0; i < 3; ++i) p.q_stride[i] = q->stride[i], p.out_stride[i] = out->stride[i], p.mask_stride[i] = mask != nullptr ? mask_stride[i] : 0;
  p.mask = mask;
  p.counts = counts;
  p.slots = slots;
  p.partial = static_cast<float*>(workspace);
  p.partial_floats = v.part_floats;
  p.layer = layer;
  p.rows = rows;
  p.tokens = tokens;
  p.heads = q->heads;
  p.group = q->heads / c.view.kv_heads;
  p.parts = parts;
  p.min_units = 2;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.q_fp32 = q->dtype != c.dtype;
  KB200_CUDA(launch_kernel(true, v.kernel, dim3(parts), dim3(kThreads), v.smem, s, p));
  KB200_CUDA(launch_kernel(true, v.join, dim3(parts, (v.rows * 32 + kThreads - 1) / kThreads / 2), dim3(kThreads), 0, s, p));
  return KB200_OK;
}
