// What the kernels of the attention over a paged cache share: the producer of tiles, bounded waits, the rows that hold nothing, and the join of
// parts.
#pragma once

#include "cache_attention_math.cuh"

namespace kb200 {
namespace {

using namespace cache_math;

// A wait of 2^31 cycles at most, about a second (a poll may suspend the thread, so a number of polls says little).  Where the barrier is ready it is one poll and
// nothing else: the warp that issues the tensor core's instructions waits twice a tile.
__device__ __forceinline__ bool polled(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool wait_a_second(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const long long t0 = clock64();
  while (true) {
    for (int i = 0; i < 16; ++i)
      if (polled(bar, parity)) return true;
    if (*abort_flag || clock64() - t0 > (1ll << 31)) return false;
  }
}
// By a converged warp: ends for all lanes or none (a lane may have a barrier of its own).  Where it runs out the CTA's other waits do too.
__device__ __forceinline__ bool warp_waits(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, polled(bar, parity))) return true;
  const bool got = wait_a_second(bar, parity, abort_flag);
  if (!got) *abort_flag = 1;
  return __all_sync(0xffffffffu, got) != 0;
}

// Asks L2 for an item's query rows and masks in front of its keys.  All rings together are 28 MB of reads that are under way, 4 us of the memory's time, and what is asked
// for behind them comes that much later: an item began 16000 cycles after the last had ended (trees of 32 tokens over long sequences).
template <typename T, int ROWS>
__device__ __forceinline__ void ask_for_rows(const CacheAttnParams& p, const CacheCursor& now, int lane) {
  const int rows = min(ROWS, now.it.count * p.group - now.row_tile * ROWS);
  const int element = p.q_fp32 ? 4 : (int)sizeof(T), lines = (p.c.head_dim * element + 127) / 128;
  for (int i = lane; i < rows * lines; i += 32) {
    const CacheRow r = row_of<ROWS>(p, now, i / lines);
    const char* const at = static_cast<const char*>(p.q) + (now.b * p.q_stride[0] + r.token * p.q_stride[1] + r.head * p.q_stride[2]) * element + i % lines * 128;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
  }
  if (p.mask == nullptr) return;
  const int first = now.row_tile * ROWS / p.group, tokens = (now.row_tile * ROWS + rows - 1) / p.group - first + 1;
  for (int i = lane; i < 2 * tokens; i += 32)                            // (both ends of a row: of up to 64 tokens all of it)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p.mask + now.b * p.mask_stride[0] + (first + i / 2) * p.mask_stride[1] + (i & 1) * (now.it.count - 1) * p.mask_stride[2]));
}

// The producer warp: brings the run's tiles, page by page, as the ring's stages become free.
template <typename T, int DP, int ROWS, int STAGES, typename Wait>
__device__ __forceinline__ void bring_tiles(const CUtensorMap& map, const CacheAttnParams& p, CacheRun& run, uint32_t stage0, uint32_t full, uint32_t empty, Wait&& wait) {
  using G = Tile<T, DP>;
  constexpr int TILE = G::kKeys;
  const int lane = threadIdx.x & 31;
  CacheCursor& now = run.at;
  const int box = min(TILE, 1 << p.c.page_log2), boxes = TILE / box;       // rows of a box; of a tile
  const int none = p.c.layers * 2 * p.c.pages;                             // beyond the map: zeros
  uint32_t u = 0;
  // 32 entries of a sequence's table row as far as a batch row's keys go, one per lane (rows that name the same sequence may end apart)
  int page_base = -1, page_slot = -1, page_end = -1, my_page = -1;
  int left = run.tiles(p), tiles = left;
  if (left > 0) ask_for_rows<T, ROWS>(p, now, lane);
  while (left > 0) {
    const int first = now.tile * TILE >> p.c.page_log2;
    const int wanted = first & ~31;
    if (page_slot != now.it.slot || page_end != now.it.end || wanted != page_base) {
      page_slot = now.it.slot;
      page_end = now.it.end;
      page_base = wanted;
      const int k = wanted + lane;
      my_page = k << p.c.page_log2 < now.it.end ? p.c.table[(int64_t)now.it.slot * p.c.max_pages + k] : -1;
      if (my_page >= p.c.pages || (my_page < 0 && k << p.c.page_log2 < now.it.end)) {
        cache_fault(p.c, KB200_CACHE_BAD_INDEX);
        my_page = -1;
      }
    }
    const int stage = u % STAGES;
    if (!wait(empty + 8 * stage, ((u / STAGES) & 1) ^ 1)) break;
    const uint32_t to = stage0 + stage * G::kBytes, bar = full + 8 * stage;
    if (lane == 0) mbar_expect_tx(bar, G::kBytes);
    __syncwarp();
    // K and V of every box, block by block: as many loads as there are, spread over the lanes
    const int in_page = now.tile * TILE & ((1 << p.c.page_log2) - 1);
    for (int i0 = 0; i0 < boxes * G::kBlocks * 2; i0 += 32) {
      const int i = i0 + lane, which = i & 1, block = (i >> 1) % G::kBlocks, j = (i >> 1) / G::kBlocks;
      const int page = __shfl_sync(0xffffffffu, my_page, (first + j) & 31);
      if (i < boxes * G::kBlocks * 2)
        tma_load_3d(to + which * G::kHalf + block * G::kBlockBytes + j * box * 128, &map, bar, block * (128 / (int)sizeof(T)),
                    (now.head << p.c.page_log2) + in_page, page < 0 ? none : (p.layer * 2 + which) * p.c.pages + page);
    }
    ++u;
    ++now.tile;
    if (--left == 0) {
      run.pass<ROWS, TILE>(p, tiles);
      left = tiles = run.tiles(p);
      if (left > 0) ask_for_rows<T, ROWS>(p, now, lane);
    }
  }
}

// Rows behind a sequence's drafted tokens, and those of no sequence: zeros.  By every warp, when it has nothing else to do: 32 rows are looked at at a time, which lie
// apart, so that neighbours go to other SMs (32 neighbours to a warp: 249 us where 231 are, a few warps cleared whole sequences).
template <typename T>
__device__ __forceinline__ void clear_rows_behind(const CacheAttnParams& p, int warp, int warps) {
  if (p.counts == nullptr && p.slots == nullptr) return;
  const int lane = threadIdx.x & 31, chunks = p.heads * p.c.row_chunks;
  const int64_t rows = (int64_t)p.rows * p.tokens;
  const int64_t step = (int64_t)gridDim.x * warps;
  for (int64_t r0 = (int64_t)warp * gridDim.x + blockIdx.x; r0 < rows; r0 += 32 * step) {
    const int64_t r = r0 + lane * step;
    const int b = (int)(r / p.tokens);
    const bool empty = r < rows && ((p.counts != nullptr && (int)(r - (int64_t)b * p.tokens) >= p.counts[b]) ||
                                    (p.slots != nullptr && (unsigned)p.slots[b] >= (unsigned)p.c.sequences));
    for (unsigned left = __ballot_sync(0xffffffffu, empty); left != 0; left &= left - 1) {
      const int64_t at = r0 + (__ffs(left) - 1) * step;
      T* const row = static_cast<T*>(p.out) + at / p.tokens * p.out_stride[0] + at % p.tokens * p.out_stride[1];
      for (int x = lane; x < chunks; x += 32)
        *reinterpret_cast<uint4*>(row + x / p.c.row_chunks * p.out_stride[2] + x % p.c.row_chunks * (16 / (int)sizeof(T))) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// A part, by groups of rows: a warp's output registers, not divided by their sums, then its rows' maxima and sums.
template <typename Math>
constexpr int kPartOfWarp = Math::kOut * 32 + 2 * Math::kRows;

// Joins the parts of the item that CTA x of the first launch has left (CacheJoin).
constexpr int kJoinThreads = 128, kJoinAtOnce = 4;      // parts whose loads are in flight together

template <typename Math, int RG>
__global__ void __launch_bounds__(kJoinThreads) cache_attention_join_kernel(const __grid_constant__ CacheAttnParams p) {
  using T = typename Math::Type;
  constexpr int DP = Math::kDim, ROWS = Math::kRows * RG;
  pdl_wait();
  pdl_launch_dependents();
  const CacheJoin at = p.joins[blockIdx.x];
  const int rows_here = at.rows;
  for (int i = blockIdx.y * kJoinThreads + threadIdx.x; i < rows_here * (DP / 4); i += gridDim.y * kJoinThreads) {
    // (neighbours in a part to neighbouring lanes)
    const int row = Math::kByRows ? i % rows_here : i / (DP / 4), d = (Math::kByRows ? i / rows_here : i % (DP / 4)) * 4;
    if (d >= p.c.head_dim) continue;
    const int in_warp = row % Math::kRows;
    const int at0 = Math::place(in_warp, d), at1 = Math::place(in_warp, d + 1), at2 = Math::place(in_warp, d + 2), at3 = Math::place(in_warp, d + 3);
    float top = -CUDART_INF_F, sum = 0.0f;
    float4 x = make_float4(0, 0, 0, 0);
    for (int r0 = at.first; r0 <= (int)blockIdx.x; r0 += kJoinAtOnce) {
      float m[kJoinAtOnce], l[kJoinAtOnce], next = top;
      float4 y[kJoinAtOnce];
#pragma unroll
      for (int j = 0; j < kJoinAtOnce; ++j) {
        const int r = min(r0 + j, (int)blockIdx.x);
        const float* const part = p.partial + (2 * (int64_t)r + (r == at.first ? at.later : 0)) * p.partial_floats + row / Math::kRows * kPartOfWarp<Math>;
        const float2 state = reinterpret_cast<const float2*>(part + Math::kOut * 32)[in_warp];
        m[j] = state.x;
        l[j] = state.y;
        y[j] = make_float4(part[at0], part[at1], part[at2], part[at3]);
      }
#pragma unroll
      for (int j = 0; j < kJoinAtOnce; ++j) {
        if (r0 + j > (int)blockIdx.x) m[j] = -CUDART_INF_F;
        next = fmaxf(next, m[j]);
      }
      if (next == -CUDART_INF_F) continue;           // nothing seen so far
      const float a = ex2(Math::exponent(top - next, p.scale_log2));
      sum *= a, x.x *= a, x.y *= a, x.z *= a, x.w *= a;
#pragma unroll
      for (int j = 0; j < kJoinAtOnce; ++j) {
        if (m[j] == -CUDART_INF_F) continue;
        const float b = ex2(Math::exponent(m[j] - next, p.scale_log2));
        sum += l[j] * b, x.x += y[j].x * b, x.y += y[j].y * b, x.z += y[j].z * b, x.w += y[j].w * b;
      }
      top = next;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const CacheRow r = row_of<ROWS>(p, at.row_tile, at.head, row);
    T* const to = static_cast<T*>(p.out) + at.b * p.out_stride[0] + r.token * p.out_stride[1] + r.head * p.out_stride[2] + d;
    store2<T>(to, x.x * inv, x.y * inv);
    store2<T>(to + 2, x.z * inv, x.w * inv);
  }
}

}  // namespace

// A kernel of the attention for a size of row tiles.
struct CacheAttnVariant {
  void (*kernel)(CUtensorMap, CacheAttnParams);
  void (*join)(CacheAttnParams);
  int threads, smem, rows, tile;   // rows and keys of a tile
  int groups;                      // tiles at work at once
  int item_units;                  // see cache_attention.h
  int64_t part_floats;
};
CacheAttnVariant cache_attention_tc_variant(int dtype, int head_dim, int tokens);      // (cache_attention_tc.cu) tiles of 128 query rows; 16-bit types, heads up to 128

}  // namespace kb200
