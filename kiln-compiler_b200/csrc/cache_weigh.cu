// What weight the tokens of a sequence draw (kb200_cache_weigh): for every key the sum, over query rows and heads, of exp(scale q k - lse).
//
// What bounds it: the bytes of K, which is read once; nothing comes back but a number per key.  K needs no layout but its own: a key's 16-byte chunks go to the four lanes that hold it in
// mma.sync's second operand, and since the order in which a dot product's elements are summed is free, the query rows are read in the same order.  (Which chunks a lane has: t4, t4 + 4, ...)
// Few rows (weigh_few_kernel): a warp walks a run of keys for query rows that stay.  Many rows, and float32 (weigh_kernel): a warp takes 8 to 32 keys of a head straight into
// registers and walks the rows.
//
// Every key belongs to one CTA, whose warps share out the heads and are added up in their order: no atomics, the same bits every time.
#include <algorithm>
#include <cmath>

#include "cache_attention_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

using namespace cache_math;

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct WeighParams {
  CacheAttnParams a;       // with one head to a sequence, so that a unit is a tile of keys in all heads (find_run)
  int kv_heads, group;
  const float* lse;
  int64_t lse_stride[3];
  float* out;
  int64_t out_stride;
  const float* weights;    // what is added to; null: zeros.  Or out, and then `rest` is not to be written
  int64_t weights_stride;
  bool rest;               // entries that no key of the call has are written too (batch row b is sequence b)
  int split;               // warps that share the heads of a tile; the others have other tiles
};

// Keys of a warp at a time: 16 registers of K to 4 lanes and 8 keys of 128 columns in 16 bits, 64 in all.
template <typename T, int DP>
struct WeighTile {
  static constexpr int kChunks = DP * (int)sizeof(T) / 64;      // 16-byte chunks of a key in a lane
  static constexpr int kGroups = kChunks <= 2 ? 4 : kChunks <= 4 ? 2 : 1;        // of 8 keys
  static constexpr int kKeys = 8 * kGroups;
};

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

// A lane's chunks of a query row, rounded to the cache's type where they are float32; zeros where there is no row.
template <typename T, int DP>
__device__ __forceinline__ void load_row(const WeighParams& p, int b, int token, int head, bool there, int t4, uint4 (&x)[WeighTile<T, DP>::kChunks]) {
  constexpr int kElements = 16 / (int)sizeof(T);
  const int64_t from = b * p.a.q_stride[0] + token * p.a.q_stride[1] + head * p.a.q_stride[2];
#pragma unroll
  for (int i = 0; i < WeighTile<T, DP>::kChunks; ++i) {
    const int chunk = 4 * i + t4;
    x[i] = zero4();
    if (!there || chunk >= p.a.c.row_chunks) continue;
    if (sizeof(T) == 2 && p.a.q_fp32) {
      const float4* const q = reinterpret_cast<const float4*>(static_cast<const float*>(p.a.q) + from) + chunk * 2;
      const float4 u = q[0], v = q[1];
      x[i] = make_uint4(pack<T>(u.x, u.y), pack<T>(u.z, u.w), pack<T>(v.x, v.y), pack<T>(v.z, v.w));
    } else {
      x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.q) + from + chunk * kElements);
    }
  }
}

__device__ __forceinline__ bool sees_key(const WeighParams& p, int b, int token, int drafted) {
  if (p.a.mask == nullptr) return drafted <= token;
  return p.a.mask[b * p.a.mask_stride[0] + token * p.a.mask_stride[1] + drafted * p.a.mask_stride[2]] != 0;
}

__device__ __forceinline__ float added_to(const WeighParams& p, int s, int key) { return p.weights == nullptr ? 0.0f : p.weights[s * p.weights_stride + key]; }
// The entries that no key of the call has, 1024 to a CTA at a time.  (A sequence to a CTA: 10 us for 32 of 8192.)
__device__ __forceinline__ void write_rest(const WeighParams& p) {
  if (!p.rest) return;
  const int width = p.a.c.max_pages << p.a.c.page_log2, pieces = (width + 4 * kThreads - 1) / (4 * kThreads);
  for (int64_t u = blockIdx.x; u < (int64_t)p.a.c.sequences * pieces; u += gridDim.x) {
    const int s = (int)(u / pieces), from = (int)(u % pieces) * 4 * kThreads + threadIdx.x;
    int end = 0;
    if (s < p.a.rows) {
      const CacheItems it = cache_items<1 << 24, 8, kOrCommitted>(p.a, s);
      end = it.count > 0 ? it.end : 0;
    }
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = from + j * kThreads >= end && from + j * kThreads < width ? added_to(p, s, from + j * kThreads) : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (from + j * kThreads >= end && from + j * kThreads < width) p.out[s * p.out_stride + from + j * kThreads] = x[j];
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 2) weigh_kernel(const __grid_constant__ WeighParams p) {
  using W = WeighTile<T, DP>;
  constexpr int KEYS = W::kKeys, GROUPS = W::kGroups, CHUNKS = W::kChunks, ROWS = 1 << 24;
  __shared__ CacheRunShared found;
  __shared__ float sums[2][kWarps][KEYS];
  __shared__ bool gone[2][kWarps][GROUPS];         // of a tile's groups of eight keys, which no page's border cuts: their page is missing
  pdl_wait();
  pdl_launch_dependents();
  write_rest(p);
  const int lane = threadIdx.x & 31, warp = warp_index(), g = lane >> 2, t4 = lane & 3;
  CacheRun run;
  if (!find_run<ROWS, KEYS, kThreads, kOrCommitted>(p.a, blockIdx.x, found, &run)) return;
  const CacheView& c = p.a.c;
  const int beside = kWarps / p.split, mine = warp / p.split, part = warp % p.split, in_page = (1 << c.page_log2) - 1;
  const float scale = p.a.scale_log2;
  int turn = 0;
  for (int tiles; (tiles = run.tiles(p.a)) > 0; run.pass<ROWS, KEYS, kOrCommitted>(p.a, tiles)) {
    const CacheItems& it = run.at.it;
    const int b = run.at.b, rows = it.count * p.group;
    if (p.a.slots != nullptr) {                    // a sequence that an earlier row names is that row's
      bool again = false;
      for (int i = threadIdx.x; i < b; i += kThreads) again = again || p.a.slots[i] == it.slot;
      if (__syncthreads_or(again)) {
        if (threadIdx.x == 0) cache_fault(c, KB200_CACHE_BAD_INDEX);
        continue;
      }
    }
    for (int i0 = 0; i0 < tiles; i0 += beside) {
      const bool there = i0 + mine < tiles;
      const int key0 = (run.at.tile + i0 + mine) * KEYS;
      float sum[GROUPS][2];                        // 16 bits: of keys 2 t4 and 2 t4 + 1 of a group; float32: the first, of key g of group t4
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) sum[i][0] = sum[i][1] = 0.0f;
      if (there) {
        const T* keys[GROUPS];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
          const int key = key0 + 8 * i + g;
          int page = -1;
          if (key < it.end) {
            page = c.table[(int64_t)it.slot * c.max_pages + (key >> c.page_log2)];
            if (!cache_page_ok(c, page)) cache_fault(c, KB200_CACHE_BAD_INDEX), page = -1;
          }
          if (lane == 0) gone[turn][warp][i] = page < 0;
          keys[i] = page < 0 ? nullptr : static_cast<const T*>(c.pool) + (((((int64_t)p.a.layer * 2 * c.pages + page) * p.kv_heads) << c.page_log2) + (key & in_page)) * c.head_dim;
        }
        const bool drafted = key0 + KEYS > it.length;
        for (int head = part; head < p.kv_heads; head += p.split) {
          uint4 k[GROUPS][CHUNKS];
#pragma unroll
          for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
              k[i][j] = zero4();
              if (keys[i] != nullptr && 4 * j + t4 < c.row_chunks)
                k[i][j] = __ldg(reinterpret_cast<const uint4*>(keys[i] + (((int64_t)head << c.page_log2) * c.head_dim)) + 4 * j + t4);
            }
          if constexpr (sizeof(T) == 2) {
            for (int row0 = 0; row0 < rows; row0 += 16) {
              uint4 q[2][CHUNKS];
              float shift[2];
              int token[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int row = row0 + g + 8 * h;
                token[h] = row / p.group;
                const int of = head * p.group + row - token[h] * p.group;
                load_row<T, DP>(p, b, token[h], of, row < rows, t4, q[h]);
                // (no row, or one that sees nothing: 2^-inf of whatever is finite, and nothing else is summed)
                shift[h] = row < rows ? p.lse[b * p.lse_stride[0] + token[h] * p.lse_stride[1] + of * p.lse_stride[2]] : -CUDART_INF_F;
                shift[h] = shift[h] == -CUDART_INF_F ? CUDART_INF_F : shift[h] * 1.4426950408889634f;
                if (row >= rows) token[h] = -1;
              }
#pragma unroll
              for (int i = 0; i < GROUPS; ++i) {
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j) {
                  const uint32_t low[4] = {q[0][j].x, q[1][j].x, q[0][j].y, q[1][j].y}, high[4] = {q[0][j].z, q[1][j].z, q[0][j].w, q[1][j].w};
                  mma16<T>(s, low, k[i][j].x, k[i][j].y);
                  mma16<T>(s, high, k[i][j].z, k[i][j].w);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int h = e >> 1, key = key0 + 8 * i + 2 * t4 + (e & 1);
                  bool visible = shift[h] != CUDART_INF_F;
                  if (drafted && visible) visible = key < it.end && (key < it.length || sees_key(p, b, token[h], key - it.length));
                  if (visible) sum[i][e & 1] += ex2(fmaf(s[e], scale, -shift[h]));
                }
              }
            }
          } else {
            for (int row = 0; row < rows; ++row) {
              const int token = row / p.group, of = head * p.group + row - token * p.group;
              uint4 q[CHUNKS];
              load_row<T, DP>(p, b, token, of, true, t4, q);
              const float lse = p.lse[b * p.lse_stride[0] + token * p.lse_stride[1] + of * p.lse_stride[2]];
              if (lse == -CUDART_INF_F) continue;
              float s[GROUPS];
#pragma unroll
              for (int i = 0; i < GROUPS; ++i) {
                float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j) {
                  x = ffma2(make_float2(__uint_as_float(k[i][j].x), __uint_as_float(k[i][j].y)), make_float2(__uint_as_float(q[j].x), __uint_as_float(q[j].y)), x);
                  x = ffma2(make_float2(__uint_as_float(k[i][j].z), __uint_as_float(k[i][j].w)), make_float2(__uint_as_float(q[j].z), __uint_as_float(q[j].w)), x);
                }
                s[i] = x.x + x.y;
                s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
                s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
              }
              float score = s[0];
#pragma unroll
              for (int i = 1; i < GROUPS; ++i) score = t4 == i ? s[i] : score;
              const int key = key0 + 8 * t4 + g;
              bool visible = t4 < GROUPS;
              if (drafted && visible) visible = key < it.end && (key < it.length || sees_key(p, b, token, key - it.length));
              if (visible) sum[0][0] += ex2(fmaf(score, scale, -lse * 1.4426950408889634f));
            }
          }
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int d = 4; d < 32; d *= 2) sum[i][e] += __shfl_xor_sync(0xffffffffu, sum[i][e], d);
              if (g == 0) sums[turn][warp][8 * i + 2 * t4 + e] = sum[i][e];
            }
        } else if (t4 < GROUPS) {
          sums[turn][warp][8 * t4 + g] = sum[0][0];
        }
      }
      __syncthreads();                             // (of two sets in turn: the last step's has been read)
      if (there && part == 0 && lane < KEYS && key0 + lane < it.end) {
        float x = 0.0f;
        for (int w = 0; w < p.split; ++w) x += sums[turn][warp + w][lane];
        p.out[it.slot * p.out_stride + key0 + lane] = added_to(p, it.slot, key0 + lane) + (gone[turn][warp][lane >> 3] ? 0.0f : x);
      }
      turn ^= 1;
    }
  }
}

// Up to 16 query rows to a key head, 16 bits: what single tokens and the last few of a prompt are.  A warp's query rows of a head stay in registers over a run of tiles, the next of
// which are under way to a ring of the warp's own, eight keys to a copy; its keys' sums over heads are kept in shared memory, and the warps' are added up behind a run.  (With the rows looked up at every tile, 650 instructions for 4 KB
// of K: 83 us for 32 sequences of up to 8192 tokens, 16 rows to each of eight key heads.)
constexpr int kRunKeys = 512, kStages = 3;
// What beginning and ending a sequence costs, in keys: runs of 600 keys that went from one sequence to the next took 53.6 us, the others 44.1.  A call: 62.2 us without, 59.1
// with 64 keys, 56.8 with 128, 56.0 with 256.
constexpr int kItemKeys = 256;

template <typename T, int DP>
struct WeighRing {
  static constexpr int kTileBytes = WeighTile<T, DP>::kGroups * WeighTile<T, DP>::kChunks * 512, kRunTiles = kRunKeys / WeighTile<T, DP>::kKeys;
  static constexpr int kSmem = kWarps * (kStages * kTileBytes + kRunKeys * (int)sizeof(float));
};
__device__ __forceinline__ void copy_bulk(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 2) weigh_few_kernel(const __grid_constant__ WeighParams p) {
  using W = WeighTile<T, DP>;
  constexpr int KEYS = W::kKeys, GROUPS = W::kGroups, CHUNKS = W::kChunks, ROWS = 1 << 24;
  using Ring = WeighRing<T, DP>;
  constexpr int kRunTiles = Ring::kRunTiles;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ CacheRunShared found;
  __shared__ __align__(8) uint64_t bars[kWarps * kStages];
  __shared__ unsigned gone[kWarps][2];             // of a warp's run: groups of eight keys whose page is missing
  __shared__ int gave_up;
  float* const sums = reinterpret_cast<float*>(smem + kWarps * kStages * Ring::kTileBytes);      // [kWarps][kRunKeys]
  const int lane = threadIdx.x & 31, warp = warp_index(), g = lane >> 2, t4 = lane & 3;
  if (lane < kStages) mbar_init(smem_u32(&bars[warp * kStages + lane]), 1);
  if (threadIdx.x == 0) gave_up = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();
  write_rest(p);
  __syncthreads();
  const uint32_t ring = smem_u32(smem) + warp * kStages * Ring::kTileBytes, full = smem_u32(&bars[warp * kStages]);
  uint32_t asked = 0, taken = 0;                   // tiles, over all runs
  CacheRun run;
  if (!find_run<ROWS, KEYS, kThreads, kOrCommitted>(p.a, blockIdx.x, found, &run)) return;
  const CacheView& c = p.a.c;
  const int beside = kWarps / p.split, mine = warp / p.split, part = warp % p.split, in_page = (1 << c.page_log2) - 1;
  const float scale = p.a.scale_log2;
  const int64_t head_stride = (int64_t)c.head_dim << c.page_log2;
  // Of a lane's sums, one per key, those of all lanes that have the same keys: each lane is left with one key's.
  const int my_key = GROUPS == 4 ? (lane >> 3 & 1) * 16 + (lane >> 4 & 1) * 8 + 2 * t4 + (lane >> 2 & 1) : GROUPS == 2 ? (lane >> 3 & 1) * 8 + 2 * t4 + (lane >> 2 & 1) : 2 * t4 + (lane >> 2 & 1);
  for (int tiles; (tiles = run.tiles(p.a)) > 0; run.pass<ROWS, KEYS, kOrCommitted>(p.a, tiles)) {
    const CacheItems& it = run.at.it;
    const int b = run.at.b, rows = it.count * p.group;
    if (p.a.slots != nullptr) {                    // a sequence that an earlier row names is that row's
      bool again = false;
      for (int i = threadIdx.x; i < b; i += kThreads) again = again || p.a.slots[i] == it.slot;
      if (__syncthreads_or(again)) {
        if (threadIdx.x == 0) cache_fault(c, KB200_CACHE_BAD_INDEX);
        continue;
      }
    }
    int token[2], in_group[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = min(g + 8 * h, rows - 1);
      token[h] = row / p.group;
      in_group[h] = row - token[h] * p.group;
    }
    const int32_t* const table = c.table + (int64_t)it.slot * c.max_pages;
    for (int i0 = 0; i0 < tiles; i0 += kRunTiles * beside) {
      const int n = min(tiles - i0, kRunTiles * beside), per = (n + beside - 1) / beside;
      const int first = i0 + mine * per, last = min(i0 + n, first + per);
      // Where the run's groups of eight keys are, which no page's border cuts: two to a lane.  (Behind the keys there are the last ones again, which no row sees, and where a page is
      // missing the pool's first page, whose sums are left out.)
      constexpr int PLACES = GROUPS * kRunTiles / 32;
      static_assert(PLACES == 2, "a bit of `gone` to a group");
      int64_t places[PLACES];
#pragma unroll
      for (int i = 0; i < PLACES; ++i) {
        const int key = (run.at.tile + first) * KEYS + 8 * (lane + 32 * i), there = max(min(key, (it.end - 1) & ~7), 0);
        int page = first < last ? table[there >> c.page_log2] : 0;
        const bool missing = !cache_page_ok(c, page);
        if (missing) {
          if (key < it.end && key < (run.at.tile + last) * KEYS) cache_fault(c, KB200_CACHE_BAD_INDEX);
          page = 0;
        }
        places[i] = (((((int64_t)p.a.layer * 2 * c.pages + page) * p.kv_heads) << c.page_log2) + (there & in_page)) * c.head_dim;
        const unsigned lacks = __ballot_sync(0xffffffffu, missing);
        if (lane == 0) gone[warp][i] = lacks;
      }
      // (what the first of the keys' sums are added to is asked for in front of them)
      const int key_first = (run.at.tile + i0) * KEYS + threadIdx.x;
      float before[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) before[j] = threadIdx.x + j * kThreads < n * KEYS && key_first + j * kThreads < it.end ? added_to(p, it.slot, key_first + j * kThreads) : 0.0f;
      for (int head = part; head < p.kv_heads; head += p.split) {
        uint4 q[2][CHUNKS];
        float shift[2];
        bool adds[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int of = head * p.group + in_group[h];
          const float lse = g + 8 * h < rows ? p.lse[b * p.lse_stride[0] + token[h] * p.lse_stride[1] + of * p.lse_stride[2]] : -CUDART_INF_F;
          adds[h] = lse != -CUDART_INF_F;          // (a row, and one that sees something)
          load_row<T, DP>(p, b, token[h], of, adds[h], t4, q[h]);
          shift[h] = lse * -1.4426950408889634f;
        }
        const T* const base = static_cast<const T*>(c.pool) + head * head_stride;
        const uint32_t row_bytes = c.row_chunks * 16;
        auto ask = [&](int tile) {                 // by a lane for each eight keys
          int64_t at = 0;
#pragma unroll
          for (int i = 0; i < PLACES; ++i) {
            const int64_t of = __shfl_sync(0xffffffffu, places[i], ((tile - first) * GROUPS + lane) & 31);
            if ((((tile - first) * GROUPS) >> 5) == i) at = of;
          }
          const uint32_t stage = asked % kStages, bar = full + 8 * stage;
          if (lane == 0) mbar_expect_tx(bar, GROUPS * 8 * row_bytes);
          __syncwarp();
          if (lane < GROUPS) copy_bulk(ring + stage * Ring::kTileBytes + lane * 8 * row_bytes, base + at, 8 * row_bytes, bar);
          ++asked;
        };
        for (int j = 0; j < kStages - 1 && first + j < last; ++j) ask(first + j);
        for (int tile = first; tile < last; ++tile) {
          if (tile + kStages - 1 < last) ask(tile + kStages - 1);
          const uint32_t stage = taken % kStages;
          const bool ok = warp_waits(full + 8 * stage, (taken / kStages) & 1, &gave_up);
          ++taken;
          float s[GROUPS][4];
#pragma unroll
          for (int i = 0; i < GROUPS; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
          if (ok) {
            const uint32_t at = ring + stage * Ring::kTileBytes + g * row_bytes + t4 * 16;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
              const uint32_t low[4] = {q[0][j].x, q[1][j].x, q[0][j].y, q[1][j].y}, high[4] = {q[0][j].z, q[1][j].z, q[0][j].w, q[1][j].w};
#pragma unroll
              for (int i = 0; i < GROUPS; ++i) {
                uint4 k = zero4();
                if (4 * j + t4 < c.row_chunks)
                  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(k.x), "=r"(k.y), "=r"(k.z), "=r"(k.w) : "r"(at + i * 8 * row_bytes + j * 64) : "memory");
                mma16<T>(s[i], low, k.x, k.y);
                mma16<T>(s[i], high, k.z, k.w);
              }
            }
          }
          __syncwarp();                            // (the tile has been read; its stage is the next one's)
          // What a row does not add is left out behind the exponential: a key with an infinity makes NaN even of a row of zeros, and a row's lse may be NaN.
          const int key0 = (run.at.tile + tile) * KEYS;
          float sum[2 * GROUPS];
          auto add = [&](auto&& sees) {
#pragma unroll
            for (int i = 0; i < GROUPS; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = key0 + 8 * i + 2 * t4 + e;
                const float x = ex2(fmaf(s[i][e], scale, shift[0])), y = ex2(fmaf(s[i][2 + e], scale, shift[1]));
                sum[2 * i + e] = (adds[0] && sees(0, key) ? x : 0.0f) + (adds[1] && sees(1, key) ? y : 0.0f);
              }
          };
          if (key0 + KEYS <= it.length)
            add([](int, int) { return true; });
          else                                     // drafted tokens, or what is behind them
            add([&](int h, int key) { return key < it.end && (key < it.length || sees_key(p, b, token[h], key - it.length)); });
          // over the lanes with other rows: as many sums as there are halve at every step
#pragma unroll
          for (int d = 4, m = GROUPS; d < 32; d *= 2, m /= 2) {
            const bool upper = (lane & d) != 0;
            if (m >= 1) {
              // (the first step is between the two keys of a lane, the others between groups)
#pragma unroll
              for (int i = 0; i < (m < 1 ? 1 : m); ++i) {
                const int low = d == 4 ? 2 * i : i, high = d == 4 ? 2 * i + 1 : i + m;
                const float give = upper ? sum[low] : sum[high], keep = upper ? sum[high] : sum[low];
                sum[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
              }
            } else {
              sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], d);
            }
          }
          if (GROUPS == 4 || (lane & (GROUPS == 2 ? 16 : 24)) == 0) {
            float* const to = &sums[warp * kRunKeys + (tile - first) * KEYS + my_key];
            *to = (head == part ? 0.0f : *to) + sum[0];
          }
        }
      }
      __syncthreads();
      // the heads' warps, in their order
      for (int k = threadIdx.x; k < n * KEYS; k += kThreads) {
        const int tile = k / KEYS, of = tile / per, key = (run.at.tile + i0) * KEYS + k;
        if (key >= it.end) continue;
        const int in_run = k - of * per * KEYS;
        float x = 0.0f;
        for (int w = 0; w < min(p.split, p.kv_heads); ++w) x += sums[(of * p.split + w) * kRunKeys + in_run];
        if (gone[of * p.split][in_run >> 8] >> (in_run >> 3 & 31) & 1u) x = 0.0f;
        p.out[it.slot * p.out_stride + key] = (k < kThreads ? before[0] : k < 2 * kThreads ? before[1] : added_to(p, it.slot, key)) + x;
      }
      __syncthreads();
    }
  }
  if (gave_up) {                                   // (a wait ran out: what is under way lands before shared memory is given back)
    if (threadIdx.x == 0) cache_fault(c, kCacheWaitFault);
    let_copies_land();
  }
}

// What is added to, where that is another tensor: weights, or zeros.
__global__ void __launch_bounds__(kThreads) weigh_begin_kernel(float* out, int64_t out_stride, const float* weights, int64_t weights_stride, int rows, int width) {
  pdl_wait();
  pdl_launch_dependents();
  for (int s = blockIdx.y; s < rows; s += gridDim.y) {
    const float* const from = weights + s * weights_stride;
    float* const to = out + s * out_stride;
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < width; i += gridDim.x * kThreads) to[i] = weights == nullptr ? 0.0f : from[i];
  }
}

struct Variant {
  void (*kernel)(WeighParams);
  int keys, smem;
};
template <typename T>
Variant few_variant_of(int head_dim) {
  return head_dim <= 64 ? Variant{weigh_few_kernel<T, 64>, WeighTile<T, 64>::kKeys, WeighRing<T, 64>::kSmem} : head_dim <= 128 ? Variant{weigh_few_kernel<T, 128>, WeighTile<T, 128>::kKeys, WeighRing<T, 128>::kSmem}
                                                                                                      : Variant{weigh_few_kernel<T, 256>, WeighTile<T, 256>::kKeys, WeighRing<T, 256>::kSmem};
}
template <typename T>
Variant variant_of(int head_dim) {
  return head_dim <= 64 ? Variant{weigh_kernel<T, 64>, WeighTile<T, 64>::kKeys, 0} : head_dim <= 128 ? Variant{weigh_kernel<T, 128>, WeighTile<T, 128>::kKeys, 0}
                                                                                                  : Variant{weigh_kernel<T, 256>, WeighTile<T, 256>::kKeys, 0};
}
// 16 rows are what a product of weigh_few_kernel has and all that its warps keep.  (32 sequences of up to 8192, heads of 128, four to a key head, BF16: 4 tokens take 48.8 us by it and 80.7 by weigh_kernel; of
// 8192 each 96 and 167, and there 5 tokens, 20 rows, take 236 by weigh_kernel.)
Variant variant_for(const Cache& c, int rows) {
  if (rows <= 16 && c.dtype != KB200_DTYPE_FP32) return c.dtype == KB200_DTYPE_BF16 ? few_variant_of<__nv_bfloat16>(c.view.head_dim) : few_variant_of<__half>(c.view.head_dim);
  return c.dtype == KB200_DTYPE_FP32 ? variant_of<float>(c.view.head_dim)
         : c.dtype == KB200_DTYPE_BF16 ? variant_of<__nv_bfloat16>(c.view.head_dim) : variant_of<__half>(c.view.head_dim);
}

}  // namespace

int cache_weigh_prepare(const Cache& c) {
  if (c.dtype == KB200_DTYPE_FP32) return KB200_OK;
  const Variant v = variant_for(c, 1);
  KB200_CUDA(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem));
  return KB200_OK;
}

}  // namespace kb200

using namespace kb200;

KB200_EXPORT int kb200_cache_weigh(kb200_cache* handle, int layer, const kb200_rows* q, const float* lse, const int64_t* lse_stride, int rows, int tokens,
                                   const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale, int committed, const float* weights,
                                   int64_t weights_stride, float* out, int64_t out_stride, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_weigh");
  if (layer < 0 || layer >= c.view.layers) return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: layer %d of %d", layer, c.view.layers);
  if (q == nullptr || !cache_attention_call_ok(c, rows, tokens, q->heads) || (slots == nullptr && rows > c.view.sequences))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: rows and tokens do not suit the cache, or heads are no multiple of its %d", c.view.kv_heads);
  const int64_t width = (int64_t)c.view.max_pages << c.view.page_log2;
  if (out == nullptr || (c.view.sequences > 1 && (out_stride < width || (weights != nullptr && weights_stride < width))))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: rows of weights and out are %lld long", (long long)width);
  const bool any = rows > 0 && tokens > 0;
  if (any) {
    const bool wide = q->dtype == KB200_DTYPE_FP32;
    if (q->data == nullptr || !tc::aligned16(q->data) || (q->dtype != c.dtype && !wide))
      return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: q must be of the cache's type or float32 and on 16 bytes");
    for (const int64_t x : q->stride)
      if (x % (wide ? 4 : 8) != 0) return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: strides of q must be multiples of 16 bytes");
    if (lse == nullptr || lse_stride == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: lse is null");
    if (mask != nullptr && mask_stride == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: a mask without strides");
    if (!(scale >= 1e-30f) || !(scale <= 1e30f)) return fail(KB200_ERR_ARGUMENT, "kb200_cache_weigh: scale must be from 1e-30 to 1e30");
  }
  const bool rest = any && slots == nullptr && out != weights;
  if (out != weights && !rest) {
    const dim3 grid((unsigned)std::min<int64_t>((width + kThreads - 1) / kThreads, 64), (unsigned)std::min(c.view.sequences, 65535));
    KB200_CUDA(launch_kernel(true, weigh_begin_kernel, grid, dim3(kThreads), 0, s, out, out_stride, weights, weights_stride, c.view.sequences, (int)width));
  }
  if (!any) return KB200_OK;
  const Variant v = variant_for(c, tokens * (q->heads / c.view.kv_heads));
  WeighParams p{};
  p.a.c = c.view;
  p.a.c.kv_heads = 1;
  p.a.q = q->data;
  for (int i = 0; i < 3; ++i) p.a.q_stride[i] = q->stride[i], p.lse_stride[i] = lse_stride[i], p.a.mask_stride[i] = mask != nullptr ? mask_stride[i] : 0;
  p.a.mask = mask;
  p.a.counts = counts;
  p.a.slots = slots;
  p.a.layer = layer;
  p.a.committed = committed != 0;
  p.a.rows = rows;
  p.a.tokens = tokens;
  p.a.heads = q->heads;
  p.a.group = 1;
  p.a.scale_log2 = scale * 1.4426950408889634f;
  p.a.q_fp32 = q->dtype != c.dtype;
  p.kv_heads = c.view.kv_heads;
  p.group = q->heads / c.view.kv_heads;
  p.lse = lse;
  p.out = out;
  p.out_stride = out_stride;
  p.weights = rest ? weights : out;
  p.weights_stride = rest ? weights_stride : out_stride;
  p.rest = rest;
  p.split = 1;
  while (p.split < kWarps && p.split < c.view.kv_heads) p.split *= 2;
  // Two CTAs to an SM, but no more than have a tile for each group of warps.
  p.a.min_units = kWarps / p.split;
  if (v.smem > 0) p.a.item_units = kItemKeys / v.keys;
  const double units = (double)rows * (std::ceil((double)width / v.keys) + p.a.item_units);
  p.a.parts = (int)std::min<double>(std::ceil(units / p.a.min_units), 2.0 * c.sm_count);
  KB200_CUDA(launch_kernel(true, v.kernel, dim3(p.a.parts), dim3(kThreads), v.smem, s, p));
  return KB200_OK;
}
