// Attention of drafted tokens over a paged K/V cache (kb200_cache_attend): softmax(scale q K^T, masked) V for the few query rows of
// each sequence, one pass over its keys with a running maximum and sum.
//
// What bounds it: the cache's bytes.  A key head's K and V are read once for all query rows that share them (drafted tokens x heads per key head).
// Products run on the tensor cores by warp (mma.sync): the rows of a decoding step do not fill more.
//
// A CTA has one producer warp and up to six consumer warps (from the eighth on a scheduler holds three warps and a thread 168 registers) and walks its run of key tiles (cache_attention.h).  The producer brings
// tiles of K and V through a tensor map of the pool, page by page, as far ahead as the ring of stages goes, across the borders of sequences and
// heads.  A consumer warp takes a WHOLE tile for 16 query rows and keeps maxima, sums and output rows in registers; the
// warps' sums are joined at the end of an item only.  Every stage of the ring belongs to one warp (or the group of warps with the other rows of the row
// tile), which therefore sees each of its fillings: a barrier's parity tells no more than the last one.  (With the tile's keys divided among the warps, and copies issued by them, a warp
// paid the rescaling, the shuffles and the addresses for 16 keys instead of 64: 985 instructions per warp and tile at 5.8 cycles each, two warps to
// a scheduler, 187 us for 32 sequences of up to 8192 tokens, 52 % of the bandwidth.)
//
// Scores, maxima, sums and output rows are float32.  16-bit caches: the weights of a tile are rounded to the cache's type for the product with V
// (half a step, 2^-9 for bfloat16, of every summand; the sum of the weights is kept of the unrounded ones).  float32 caches: both operands of both
// products as a TF32 head and tail, three products, what is dropped is 2^-22 of a summand; the tensor core cuts
// off what does not fit a sum, so products with tails are summed apart from those of heads, and a tile's rows start from zero and are added by FMA.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "cache_attention.h"
#include "tc_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

using namespace tc;

// Sizes by type and padded head width.  A tile is blocks of 128-byte columns, as the map's 128-byte swizzle wants them: K's, then V's.
template <typename T, int DP, int RG>
struct Shape {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kGroups = RG == 4 ? 1 : DP > 128 ? 6 / RG - 1 : 6 / RG;     // of warps, each for tiles of its own
  static constexpr int kWarps = kGroups * RG;                            // consumers
  static constexpr bool kKeepsQ = !kWide || DP <= 64;                    // query rows in registers
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kBlocks = DP * (int)sizeof(T) / 128;
  static constexpr int kTile = kBlocks <= 2 ? 64 : 128 / kBlocks;        // keys: 16 KB of K and of V at most
  static constexpr int kBlockBytes = kTile * 128;
  static constexpr int kStageBytes = 2 * kBlocks * kBlockBytes;
  static constexpr int kStages = kGroups * ((DP > 128 ? 160 : 192) * 1024 / kStageBytes / kGroups);      // (a multiple: see above)
  static constexpr int kSlots = 2;                                       // warps whose rows are in shared memory at a time when sums are joined
  static constexpr int kSlotRow = DP + 4;                                // floats
  static constexpr int kSmem = kStages * kStageBytes + kSlots * 16 * kSlotRow * 4;
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

// A wait of 2^31 cycles at most, about a second (a poll may suspend the thread, so a number of polls says little).
__device__ __forceinline__ bool wait_a_second(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const long long t0 = clock64();
  while (true) {
    for (int i = 0; i < 16; ++i) {
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(bar), "r"(parity)
          : "memory");
      if (ok != 0) return true;
    }
    if (*abort_flag || clock64() - t0 > (1ll << 31)) return false;
  }
}

// A part: ROWS output rows (not divided by their sums), then their maxima and sums.
template <int DP, int ROWS>
constexpr int64_t part_floats() { return (int64_t)ROWS * (DP + 2); }

template <typename T, int DP, int RG>
__global__ void __launch_bounds__(Shape<T, DP, RG>::kThreads, 1)
cache_attention_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CacheAttnParams p) {
  using Z = Shape<T, DP, RG>;
  constexpr int KG = Z::kGroups, ROWS = 16 * RG, TILE = Z::kTile;      // groups of warps by keys, by rows
  constexpr int NT = TILE / 8, DT = DP / 8;        // 8-wide column tiles of a warp's scores, of its output rows
  constexpr bool kWide = Z::kWide;
  static_assert(Z::kStages > 0 && Z::kStages % KG == 0 && (KG == 1 || Z::kSlots % RG == 0), "a stage belongs to one group, a slot to a warp of each row group");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[2 * Z::kStages];
  __shared__ CacheRunShared found;
  __shared__ uint32_t sees[Z::kWarps][16][2];      // a tile with drafted tokens under a mask: which row sees which key
  __shared__ float states[Z::kWarps][16][2];
  __shared__ int abort_flag;

  const int lane = threadIdx.x & 31, warp = warp_index();
  const uint32_t stage0 = smem_u32(smem), full = smem_u32(bars), empty = full + 8 * Z::kStages;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    prefetch_tensormap(&map);
    for (int i = 0; i < Z::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, RG);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  CacheRun run;
  const bool any = find_run<ROWS, TILE, Z::kThreads>(p, blockIdx.x, found, &run);       // (a barrier for all that is above, too)
  CacheCursor& now = run.at;
  volatile int* const abort_ptr = &abort_flag;
  // A wait that ends for all lanes of a warp or none.  Where it runs out the warps do no more work, but meet each other as if they did.
  auto wait = [&](uint32_t bar, uint32_t parity) {
    const bool got = wait_a_second(bar, parity, abort_ptr);
    if (!got) *abort_ptr = 1;
    return __all_sync(0xffffffffu, got ? 1 : 0) != 0;
  };

  if (warp == Z::kWarps) {
    // ---------------- producer ----------------
    if (any) {
      const int box = min(TILE, 1 << p.c.page_log2), boxes = TILE / box;       // rows of a box; of a tile
      const int none = p.c.layers * 2 * p.c.pages;                             // beyond the map: zeros
      int64_t left = run.hi - run.lo;
      uint32_t u = 0;
      int page_base = -1, page_slot = -1, my_page = -1;                        // 32 entries of a sequence's table row, one per lane
      while (left > 0) {
        const int first = now.tile * TILE >> p.c.page_log2;
        const int wanted = first & ~31;
        if (page_slot != now.it.slot || wanted != page_base) {
          page_slot = now.it.slot;
          page_base = wanted;
          const int k = wanted + lane;
          my_page = k << p.c.page_log2 < now.it.end ? p.c.table[(int64_t)now.it.slot * p.c.max_pages + k] : -1;
          if (my_page >= p.c.pages || (my_page < 0 && k << p.c.page_log2 < now.it.end)) {
            cache_fault(p.c, KB200_CACHE_BAD_INDEX);
            my_page = -1;
          }
        }
        const int stage = u % Z::kStages;
        if (!wait(empty + 8 * stage, ((u / Z::kStages) & 1) ^ 1)) break;
        const uint32_t to = stage0 + stage * Z::kStageBytes, bar = full + 8 * stage;
        if (lane == 0) mbar_expect_tx(bar, Z::kStageBytes);
        __syncwarp();
        // K and V of every box, block by block: as many loads as there are, spread over the lanes
        const int in_page = now.tile * TILE & ((1 << p.c.page_log2) - 1);
        for (int i0 = 0; i0 < boxes * Z::kBlocks * 2; i0 += 32) {
          const int i = i0 + lane, which = i & 1, block = (i >> 1) % Z::kBlocks, j = (i >> 1) / Z::kBlocks;
          const int page = __shfl_sync(0xffffffffu, my_page, (first + j) & 31);
          if (i < boxes * Z::kBlocks * 2)
            tma_load_3d(to + which * Z::kBlocks * Z::kBlockBytes + block * Z::kBlockBytes + j * box * 128, &map, bar, block * (128 / (int)sizeof(T)),
                        (now.head << p.c.page_log2) + in_page, page < 0 ? none : (p.layer * 2 + which) * p.c.pages + page);
        }
        ++u;
        --left;
        if (++now.tile == now.it.key_tiles) next_item<ROWS, TILE>(p, now);
      }
    }
  } else {
    // ---------------- consumers ----------------
    const int row_group = warp % RG, key_group = warp / RG;
    const int g = lane >> 2, t4 = lane & 3;          // fragment coordinates
    float* const slots = reinterpret_cast<float*>(smem + Z::kStages * Z::kStageBytes);
    auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::kWarps) : "memory"); };

    // rows behind a sequence's drafted tokens
    if (p.counts != nullptr || p.slots != nullptr) {
      const int width = p.heads * p.c.head_dim;
      for (int64_t r = blockIdx.x + (int64_t)warp * gridDim.x; r < (int64_t)p.rows * p.tokens; r += (int64_t)gridDim.x * Z::kWarps) {
        const int b = (int)(r / p.tokens), i = (int)(r % p.tokens);
        if ((p.counts == nullptr || i < p.counts[b]) && (p.slots == nullptr || (unsigned)p.slots[b] < (unsigned)p.c.sequences)) continue;
        for (int x = lane; x < width; x += 32)
          static_cast<T*>(p.out)[b * p.out_stride[0] + i * p.out_stride[1] + (x / p.c.head_dim) * p.out_stride[2] + x % p.c.head_dim] = T(0.0f);
      }
    }

    const int row = row_group * 16 + g;              // this thread's rows of the row tile: row and row + 8
    uint32_t q16[kWide ? 1 : DP / 16][4];
    float q32[kWide && Z::kKeepsQ ? DP / 8 : 1][4];
    const float* q_from[2] = {nullptr, nullptr};     // ... or where they are
    float o[DT][4], m[2], l[2];
    int rows_here = 0;                               // of the item's row tile
    auto begin = [&]() {
      rows_here = min(ROWS, now.it.count * p.group - now.row_tile * ROWS);
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
      m[0] = m[1] = -CUDART_INF_F;
      l[0] = l[1] = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bool there = row + 8 * half < rows_here;
        const CacheRow r = row_of<ROWS>(p, now, there ? row + 8 * half : 0);
        const int64_t at = now.b * p.q_stride[0] + r.token * p.q_stride[1] + r.head * p.q_stride[2];
        if constexpr (kWide) {
          // dims 2t and 2t + 1 of eight stand in fragment columns t and t + 4, in both operands: 64-bit loads
          if constexpr (Z::kKeepsQ) {
#pragma unroll
            for (int k = 0; k < DP / 8; ++k) {
              const float2 x = there && k * 8 < p.c.head_dim ? reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + at)[k * 4 + t4] : make_float2(0, 0);
              q32[k][half] = x.x;
              q32[k][2 + half] = x.y;
            }
          } else {
            q_from[half] = there ? static_cast<const float*>(p.q) + at : nullptr;
          }
        } else {
          auto pair = [&](int i) {                   // two elements
            if (!p.q_fp32) return reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + at)[i];
            const float2 x = reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + at)[i];
            return pack<T>(x.x, x.y);
          };
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const bool in = there && k * 16 < p.c.head_dim;
            q16[k][half] = in ? pair(k * 8 + t4) : 0u;
            q16[k][2 + half] = in ? pair(k * 8 + 4 + t4) : 0u;
          }
        }
      }
    };

    // ---- a tile ----
    auto compute = [&](int tile, uint32_t k_tile, uint32_t v_tile) {
      float s[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
      if constexpr (!kWide) {
        const uint32_t at = k_tile + ((lane >> 4) * 8 + (lane & 7)) * 128;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t in_row = (k / 4) * Z::kBlockBytes + ((((k % 4) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t b[4];
            ldmatrix4(b, at + n * 8 * 128 + in_row);
            mma16<T>(s[n], q16[k], b[0], b[1]);
            mma16<T>(s[n + 1], q16[k], b[2], b[3]);
          }
        }
      } else {
        float low[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) low[i][j] = 0.0f;
        const uint8_t* const at = smem + (k_tile - stage0) + g * 128 + (t4 & 1) * 8;
#pragma unroll
        for (int k = 0; k < DP / 8; ++k) {
          const int in_row = (k / 4) * Z::kBlockBytes + ((((k % 4) * 2 + (t4 >> 1)) ^ g) << 4);
          uint32_t ah[4], al[4];
          if constexpr (Z::kKeepsQ) {
#pragma unroll
            for (int j = 0; j < 4; ++j) split(q32[k][j], ah + j, al + j);
          } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float2 x = q_from[half] != nullptr && k * 8 < p.c.head_dim ? reinterpret_cast<const float2*>(q_from[half])[k * 4 + t4] : make_float2(0, 0);
              split(x.x, ah + half, al + half);
              split(x.y, ah + 2 + half, al + 2 + half);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 x = *reinterpret_cast<const float2*>(at + n * 8 * 128 + in_row);
            uint32_t bh[2], bl[2];
            split(x.x, bh + 0, bl + 0);
            split(x.y, bh + 1, bl + 1);
            mma_tf32(low[n], al, bh[0], bh[1]);
            mma_tf32(low[n], ah, bl[0], bl[1]);
            mma_tf32(s[n], ah, bh[0], bh[1]);
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] += low[i][j];
      }

      const int key0 = tile * TILE;
      const bool drafted = key0 + TILE > min(now.it.length, now.it.end);
      bool infinite = false;
      unsigned long long shows[2] = {~0ull, ~0ull};  // the tile's keys that rows g and g + 8 see
      if (drafted) {
        if (p.mask == nullptr) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = min(now.it.end, now.it.length + row_of<ROWS>(p, now, row + 8 * h).token + 1) - key0;
            shows[h] = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
          }
        } else {
          // a ballot per row and 32 keys, all loads in flight together (where there is nothing to look up they read the mask's first byte)
          uint8_t bytes[16][(TILE + 31) / 32];
          const uint8_t* const mask = p.mask + now.b * p.mask_stride[0];
          const int first = now.row_tile * ROWS + row_group * 16;
          int token = first / p.group, in_group = first - token * p.group;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
#pragma unroll
            for (int w = 0; w < (TILE + 31) / 32; ++w) {
              const int j = key0 + w * 32 + lane - now.it.length;
              const bool looked_up = j >= 0 && j < now.it.count && row_group * 16 + i < rows_here;
              bytes[i][w] = *(looked_up ? mask + token * p.mask_stride[1] + j * p.mask_stride[2] : p.mask);
            }
            if (++in_group == p.group) in_group = 0, ++token;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int w = 0; w < (TILE + 31) / 32; ++w) {
              const int key = key0 + w * 32 + lane;
              const bool visible = key < now.it.length || (bytes[i][w] != 0 && row_group * 16 + i < rows_here);
              const uint32_t word = __ballot_sync(0xffffffffu, visible && key < now.it.end && w * 32 + lane < TILE);
              if (lane == 0) sees[warp][i][w] = word;
            }
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) shows[h] = sees[warp][g + 8 * h][0] | (TILE > 32 ? (unsigned long long)sees[warp][g + 8 * h][1] << 32 : 0ull);
          __syncwarp();
        }
        // V behind the sequence's end is what an earlier tenant left, and V of a drafted token that some rows do not see may hold infinities or NaN; 0 times
        // those is NaN.  The former become zeros here, the latter below.
        const int last = now.it.end - key0;
        bool odd = false;
#pragma unroll 8
        for (int i = lane; i < TILE * Z::kBlocks * 8; i += 32) {
          const int key = i / (Z::kBlocks * 8), chunk = i % (Z::kBlocks * 8);
          uint4* const x = reinterpret_cast<uint4*>(smem + (v_tile - stage0) + (chunk / 8) * Z::kBlockBytes + key * 128 + (((chunk % 8) ^ (key & 7)) << 4));
          if (RG == 1 && key >= last) *x = make_uint4(0, 0, 0, 0);
          else if (key < last) odd = odd || not_finite<T>(x->x) || not_finite<T>(x->y) || not_finite<T>(x->z) || not_finite<T>(x->w);
        }
        infinite = __any_sync(0xffffffffu, odd) != 0;
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = n * 8 + t4 * 2 + (j & 1);
            if (!(shows[j >> 1] >> key & 1)) s[n][j] = -CUDART_INF_F;
          }
      }

      // ---- softmax: two rows of a thread, their keys over the four lanes of a group ----
      float top[2] = {-CUDART_INF_F, -CUDART_INF_F}, shift[2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) top[j >> 1] = fmaxf(top[j >> 1], s[n][j]);
      float alpha[2] = {1.0f, 1.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2)) * p.scale_log2;
      }
      const bool grown = __any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1]);
      if (grown) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(top[h], m[h]);
          alpha[h] = top[h] == -CUDART_INF_F ? 1.0f : ex2(m[h] - top[h]);
          m[h] = top[h];
          l[h] *= alpha[h];
        }
        if constexpr (!kWide)
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

      auto v_at = [&](int key, int d) -> T* {
        const int byte = d * (int)sizeof(T);
        return reinterpret_cast<T*>(smem + (v_tile - stage0) + (byte / 128) * Z::kBlockBytes + key * 128 + ((((byte % 128) >> 4) ^ (key & 7)) << 4) + byte % 16);
      };
      // Elements that are not finite are added to the rows that see them one by one, and are zero in the product.
      if (infinite) {
        if constexpr (kWide)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[d][j] *= alpha[j >> 1];
        alpha[0] = alpha[1] = 1.0f;
        for (int key = 0; key < TILE; ++key)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = to_float(*v_at(key, d * 8 + t4 * 2 + (j & 1)));
              if (!(fabsf(x) < CUDART_INF_F) && (shows[j >> 1] >> key & 1)) o[d][j] += x;
            }
      }
      if (drafted && (RG > 1 || infinite)) {
        // (warps of other rows read the same tile: each waits for all to have seen it as it was)
        if (RG > 1) asm volatile("bar.sync %0, %1;" ::"r"(2 + key_group), "n"(32 * RG) : "memory");
        else __syncwarp();
        const int last = now.it.end - key0;
        for (int i = row_group * 32 + lane; i < TILE * DP; i += 32 * RG) {
          T* const x = v_at(i / DP, i % DP);
          if (i / DP >= last || !(fabsf(to_float(*x)) < CUDART_INF_F)) *x = T(0.0f);
        }
        if (RG > 1) asm volatile("bar.sync %0, %1;" ::"r"(2 + key_group), "n"(32 * RG) : "memory");
        else __syncwarp();
      }

      // ---- P V ----
      if constexpr (!kWide) {
        const uint32_t at = v_tile + (((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
#pragma unroll
        for (int k = 0; k < NT / 2; ++k) {
          const uint32_t a[4] = {pack<T>(s[2 * k][0], s[2 * k][1]), pack<T>(s[2 * k][2], s[2 * k][3]), pack<T>(s[2 * k + 1][0], s[2 * k + 1][1]),
                                 pack<T>(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
          for (int d = 0; d < DT; d += 2) {
            uint32_t b[4];
            ldmatrix4_t(b, at + k * 16 * 128 + (d / 8) * Z::kBlockBytes + (((d % 8 + (lane >> 4)) ^ (lane & 7)) << 4));
            mma16<T>(o[d], a, b[0], b[1]);
            mma16<T>(o[d + 1], a, b[2], b[3]);
          }
        }
      } else {
        // keys 2t and 2t + 1 of eight stand in fragment columns t and t + 4: the scores are where the product wants them
        uint32_t ah[NT][4], al[NT][4];
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          split(s[k][0], ah[k] + 0, al[k] + 0);
          split(s[k][2], ah[k] + 1, al[k] + 1);
          split(s[k][1], ah[k] + 2, al[k] + 2);
          split(s[k][3], ah[k] + 3, al[k] + 3);
        }
        const uint8_t* const at = smem + (v_tile - stage0) + 2 * t4 * 128 + (g & 3) * 4;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          float high[4] = {0.0f, 0.0f, 0.0f, 0.0f}, low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const int block = (d / 4) * Z::kBlockBytes, chunk = (d % 4) * 2 + (g >> 2);
#pragma unroll
          for (int k = 0; k < NT; ++k) {
            uint32_t bh[2], bl[2];
            split(*reinterpret_cast<const float*>(at + block + k * 8 * 128 + ((chunk ^ (2 * t4)) << 4)), bh + 0, bl + 0);
            split(*reinterpret_cast<const float*>(at + block + (k * 8 + 1) * 128 + ((chunk ^ (2 * t4 + 1)) << 4)), bh + 1, bl + 1);
            mma_tf32(low, al[k], bh[0], bh[1]);
            mma_tf32(low, ah[k], bl[0], bl[1]);
            mma_tf32(high, ah[k], bh[0], bh[1]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) o[d][j] = fmaf(o[d][j], alpha[j >> 1], high[j] + low[j]);
        }
      }
      if (drafted) fence_async_smem();               // (the zeros, in front of the next copy to this stage)
    };

    // ---- the end of an item, or of the run inside one: the warps' sums, then the rows or a part ----
    // `order`: this warp's place among those that had a tile of it, in the order of the keys.
    auto finish = [&](int order, int tiles, bool whole, int64_t part) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (l[h] != l[h]) m[h] = 0.0f;               // (NaN, which a maximum passes over, reaches the result)
      }
      int n = min(KG, tiles);                        // groups of keys that had a tile
      if (n > 1) {
        // to the largest maximum
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (t4 == 0) states[order * RG + row_group][g + 8 * h][0] = m[h];
        meet();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = -CUDART_INF_F;
          for (int w = 0; w < n; ++w) top = fmaxf(top, states[w * RG + row_group][g + 8 * h][0]);
          const float mine = m[h] == -CUDART_INF_F ? 0.0f : ex2(m[h] - top);
          l[h] *= mine;
          m[h] = top;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][2 * h] *= mine, o[d][2 * h + 1] *= mine;
          if (t4 == 0) states[order * RG + row_group][g + 8 * h][1] = l[h];
        }
        while (n > 1) {                              // the upper half's rows go to the lower half, as many at a time as there are slots
          const int half = (n + 1) / 2;
          for (int from = half; from < n; from += Z::kSlots / RG) {
            const int to = min(n, from + Z::kSlots / RG);
            float* const slot = slots + ((order >= half ? order - from : order + half - from) * RG + row_group) * 16 * Z::kSlotRow + t4 * 2;
            if (order >= from && order < to)
#pragma unroll
              for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(slot + (g + 8 * h) * Z::kSlotRow + d * 8) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
            meet();
            if (order + half >= from && order + half < to)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                  const float2 x = *reinterpret_cast<const float2*>(slot + (g + 8 * h) * Z::kSlotRow + d * 8);
                  o[d][2 * h] += x.x;
                  o[d][2 * h + 1] += x.y;
                }
                l[h] += states[(order + half) * RG + row_group][g + 8 * h][1];
                __syncwarp();
                if (t4 == 0) states[order * RG + row_group][g + 8 * h][1] = l[h];
              }
            meet();
          }
          n = half;
        }
      }
      if (order != 0) return;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row + 8 * h >= rows_here) continue;
        if (whole) {
          const float inv = l[h] == 0.0f ? 0.0f : 1.0f / l[h];
          const CacheRow r = row_of<ROWS>(p, now, row + 8 * h);
          T* const to = static_cast<T*>(p.out) + now.b * p.out_stride[0] + r.token * p.out_stride[1] + r.head * p.out_stride[2] + t4 * 2;
#pragma unroll
          for (int d = 0; d < DT; ++d)
            if (d * 8 < p.c.head_dim) store2<T>(to + d * 8, o[d][2 * h] * inv, o[d][2 * h + 1] * inv);
        } else {
          float* const to = p.partial + part * p.partial_floats;
#pragma unroll
          for (int d = 0; d < DT; ++d)
            if (d * 8 < p.c.head_dim) *reinterpret_cast<float2*>(to + (int64_t)(row + 8 * h) * DP + d * 8 + t4 * 2) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
          if (t4 == 0) to[ROWS * DP + row + 8 * h] = m[h], to[ROWS * DP + ROWS + row + 8 * h] = l[h];
        }
      }
    };

    int64_t left = any ? run.hi - run.lo : 0;
    uint32_t u0 = 0;
    while (left > 0) {
      const int tiles = (int)min(left, (int64_t)now.it.key_tiles - now.tile);      // of this item, in this run
      begin();
      const int order = (int)((key_group + KG - u0 % KG) % KG);
      for (int i = order; i < tiles; i += KG) {
        const uint32_t u = u0 + i, stage = u % Z::kStages;
        if (wait(full + 8 * stage, (u / Z::kStages) & 1)) {
          const uint32_t k_tile = stage0 + stage * Z::kStageBytes;
          compute(now.tile + i, k_tile, k_tile + Z::kBlocks * Z::kBlockBytes);
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * stage);
        } else if (RG > 1 && (now.tile + i + 1) * TILE > min(now.it.length, now.it.end)) {
          for (int j = 0; j < 2; ++j) asm volatile("bar.sync %0, %1;" ::"r"(2 + key_group), "n"(32 * RG) : "memory");
        }
      }
      // a part that begins with the run is the run's first, else its second
      finish(order, tiles, now.tile == 0 && tiles == now.it.key_tiles, 2 * (int64_t)blockIdx.x + (u0 == 0 ? 0 : 1));
      u0 += tiles;
      left -= tiles;
      if (left > 0) next_item<ROWS, TILE>(p, now);
    }
  }
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) {
    cache_fault(p.c, kCacheWaitFault);
    let_copies_land();
  }
  __syncthreads();
}

// Joins the parts of an item.  CTA x sees to the item that ends in the run of CTA x of the first launch and began before it.
constexpr int kJoinThreads = 128;

template <typename T, int DP, int ROWS, int TILE>
__global__ void __launch_bounds__(kJoinThreads) cache_attention_join_kernel(const __grid_constant__ CacheAttnParams p) {
  __shared__ CacheRunShared found;
  pdl_wait();
  pdl_launch_dependents();
  CacheRun run;
  if (!find_run<ROWS, TILE, kJoinThreads>(p, blockIdx.x, found, &run)) return;
  const CacheCursor& at = run.at;
  if (at.tile == 0 || at.it.key_tiles - at.tile > run.hi - run.lo) return;
  const int64_t begins = run.lo - at.tile;         // the item's first unit
  const int first = (int)(((begins + 1) * run.parts - 1) / run.all);       // the run that it is in
  const int rows_here = min(ROWS, at.it.count * p.group - at.row_tile * ROWS);
  for (int i = blockIdx.y * kJoinThreads + threadIdx.x; i < rows_here * (DP / 4); i += gridDim.y * kJoinThreads) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= p.c.head_dim) continue;
    float top = -CUDART_INF_F, sum = 0.0f;
    float4 x = make_float4(0, 0, 0, 0);
    for (int r = first; r <= (int)blockIdx.x; ++r) {
      // (a run that the item begins in, but not with, has left it as its second part)
      const int64_t slot = 2 * (int64_t)r + (r == first && run.all * r / run.parts != begins ? 1 : 0);
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
    const CacheRow r = row_of<ROWS>(p, at, row);
    T* const to = static_cast<T*>(p.out) + at.b * p.out_stride[0] + r.token * p.out_stride[1] + r.head * p.out_stride[2] + d;
    store2<T>(to, x.x * inv, x.y * inv);
    store2<T>(to + 2, x.z * inv, x.w * inv);
  }
}

// ---- host --------------------------------------------------------------------------------------

struct Variant {
  void (*kernel)(CUtensorMap, CacheAttnParams);
  void (*join)(CacheAttnParams);
  int threads, smem, rows, tile;   // rows and keys of a tile
  int64_t part_floats;
};

template <typename T, int DP, int RG>
Variant variant() {
  using Z = Shape<T, DP, RG>;
  return Variant{cache_attention_kernel<T, DP, RG>, cache_attention_join_kernel<T, DP, 16 * RG, Z::kTile>, Z::kThreads, Z::kSmem, 16 * RG, Z::kTile,
                 part_floats<DP, 16 * RG>()};
}

// Tiles of 16, 32 and 64 query rows.
template <typename T, int DP>
Variant variant_of(int index) { return index == 0 ? variant<T, DP, 1>() : index == 1 ? variant<T, DP, 2>() : variant<T, DP, 4>(); }
template <typename T>
Variant variant_of(int head_dim, int index) {
  return head_dim <= 64 ? variant_of<T, 64>(index) : head_dim <= 128 ? variant_of<T, 128>(index) : variant_of<T, 256>(index);
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
int parts_of(const Cache& c, const Variant& v, int rows, int tokens, int heads) {
  const int64_t row_tiles = ((int64_t)tokens * (heads / c.view.kv_heads) + v.rows - 1) / v.rows;
  const int64_t tiles = (((int64_t)c.view.max_pages << c.view.page_log2) + v.tile - 1) / v.tile;
  const double units = (double)rows * c.view.kv_heads * row_tiles * tiles;
  return (int)std::min<double>(units, (double)c.sm_count);
}

Cache* cache_of(const kb200_cache* c) { return reinterpret_cast<Cache*>(const_cast<kb200_cache*>(c)); }

bool call_ok(const Cache& c, int rows, int tokens, int heads) {
  return rows >= 0 && tokens >= 0 && heads >= 1 && heads % c.view.kv_heads == 0 && (int64_t)tokens * (heads / c.view.kv_heads) < (1 << 24) &&
         (int64_t)rows * std::max(tokens, 1) < ((int64_t)1 << 31);
}

}  // namespace

int cache_attention_prepare(Cache& c) {
  const EncodeFn encode = encode_fn();
  if (encode == nullptr) return fail(KB200_ERR_CUDA, "kb200_cache_create: the driver has no cuTensorMapEncodeTiled");
  const CacheView& v = c.view;
  const int page = 1 << v.page_log2, columns = 128 / c.element, tile = variant_at(c, 0).tile;
  const cuuint64_t dims[3] = {(cuuint64_t)v.head_dim, (cuuint64_t)v.kv_heads * page, (cuuint64_t)v.layers * 2 * v.pages};
  const cuuint64_t strides[2] = {(cuuint64_t)v.head_dim * c.element, dims[1] * v.head_dim * c.element};
  const cuuint32_t box[3] = {(cuuint32_t)columns, (cuuint32_t)std::min(page, tile), 1}, steps[3] = {1, 1, 1};
  const CUtensorMapDataType type = c.dtype == KB200_DTYPE_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : c.dtype == KB200_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (dims[1] >= (1ull << 31) || dims[2] >= (1ull << 31))
    return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: 2^31 or more rows of a page, or pages of all layers");
  const CUresult r = encode(&c.map, type, 3, v.pool, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: the pool cannot be described to the copy engine (error %d)", (int)r);
  for (int i = 0; i < 3; ++i) {
    const Variant of = variant_at(c, i);
    KB200_CUDA(cudaFuncSetAttribute(of.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, of.smem));
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
  return (uint64_t)parts_of(c, v, rows, tokens, heads) * 2 * v.part_floats * sizeof(float);
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
  const int parts = parts_of(c, v, rows, tokens, q->heads);
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
  KB200_CUDA(launch_kernel(true, v.kernel, dim3(parts), dim3(v.threads), v.smem, s, c.map, p));
  KB200_CUDA(launch_kernel(true, v.join, dim3(parts, v.rows / 8), dim3(kJoinThreads), 0, s, p));
  return KB200_OK;
}
