// Attention of drafted tokens over a paged K/V cache with many query rows to a key head (wide trees, pieces of a prompt, many heads per key head):
// 128-row tiles on tcgen05, 16-bit caches with heads up to 128.  Work, ring and parts as in cache_attention.cu.
//
// What bounds it: the cache's bytes up to about 128 rows (a tile of 64 keys of 128 is 32 KB, 1365 cycles of an SM's share of the memory; its products are 512
// cycles of the tensor core, its exponentials 512 of the special-function unit), beyond that the exponentials.
//
// 320 threads: warp 0 brings tiles, warp 1 issues the products, and two groups of four warps take turns at the tiles, a query row to a thread of each
// (tensor-memory lane = row of the tile): from a tile's scores to its weights a warp needs ~1500 cycles, of which the exponentials are 512, so that one group
// alone holds the memory up (304 us for 32 sequences of up to 16384 tokens and 32 drafted ones).  Each group has maxima, sums and output rows of its own,
// joined at the end of an item.  448 columns of tensor memory: two sets of output rows, scores and weights (two to a column) of two tiles.  An instruction costs
// the issuing warp ~60 cycles, a commit ~100, a tile ~1000: so a group's next scores are asked for as soon as it has read the last ones, under its exponentials.
// (With the weights over the scores they had to wait for them: 3400 cycles for two tiles.)  Output rows stay in tensor memory over an item and are rescaled
// only when a row's maximum has grown.  Q is put into shared memory by the threads that own its rows, from any strides, rounded on the way where it is float32.
#include <algorithm>

#include "cache_attention_common.cuh"

namespace kb200 {
namespace {

constexpr int kRows = 128, kThreads = 64 + 2 * kRows;
constexpr uint32_t kColumns = 512, kColS = 256, kColP = 384;      // a group's output rows, the other's, two tiles' scores of 64 columns, their weights

template <typename T, int DP>
struct TcShape {
  using G = Tile<T, DP>;
  static constexpr int kQBlock = kRows * 128, kQBytes = DP / 64 * kQBlock;
  static constexpr int kStages = (224 * 1024 - kQBytes) / G::kBytes;
  static constexpr int kSmem = kQBytes + kStages * G::kBytes;
};

// Where a part's values are, for the join: a thread's row, column by column.
template <typename T, int DP>
struct TcMath {
  using Type = T;
  static constexpr bool kByRows = true;
  static constexpr int kDim = DP, kRows = kb200::kRows, kOut = DP * kb200::kRows / 32;
  static __device__ __forceinline__ int place(int row, int d) { return d * kb200::kRows + row; }
  static __device__ __forceinline__ float exponent(float behind, float) { return behind; }       // (maxima are exponents, as MmaMath's)
};

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Two 8-column loads in flight at once.
__device__ __forceinline__ void tmem_ld8x2(uint32_t addr_a, uint32_t addr_b, float (&va)[8], float (&vb)[8]) {
  uint32_t a[8], b[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%16];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%17];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]),
        "=r"(b[5]), "=r"(b[6]), "=r"(b[7])
      : "r"(addr_a), "r"(addr_b)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) va[i] = __uint_as_float(a[i]), vb[i] = __uint_as_float(b[i]);
}

// More drafted tokens than are looked up ahead: what the rows see of those in one tile, two words per token, a warp a word in four.  (64 sequences, trees of 300 tokens behind
// 100, four heads to a key head: 222 us; 285 when each row's thread read its own bytes.)
template <int ROWS>
__device__ __forceinline__ void look_at_tile(const CacheAttnParams& p, int b, int row_tile, int length, int count, int key0, uint32_t* to) {
  const int quarter = ((threadIdx.x >> 5) - 2) & 3, lane = threadIdx.x & 31;
  const int first_token = row_tile * ROWS / p.group, words = 2 * ((min((row_tile + 1) * ROWS, count * p.group) - 1) / p.group - first_token + 1);
  const int j = key0 + (quarter & 1) * 32 + lane - length;
  const bool is_drafted = j >= 0 && j < count;
  const uint8_t* const column = p.mask + b * p.mask_stride[0] + (is_drafted ? j : 0) * p.mask_stride[2];
  const int64_t step = p.mask_stride[1];
#pragma unroll 8
  for (int w = quarter; w < words; w += 4) {
    const uint32_t word = __ballot_sync(0xffffffffu, column[(first_token + w / 2) * step] != 0 && is_drafted);
    if (lane == 0) to[w] = word;
  }
}

// V of a drafted token holds infinities or NaN: they are zero in the product, and this adds them to the output row of a thread that gives the token weight w.
template <typename T, int DP>
__device__ __noinline__ void add_infinite(const CacheAttnParams& p, const CacheItems& it, int head, int at, float w, uint32_t out_addr) {
  const int page = p.c.table[(int64_t)it.slot * p.c.max_pages + (at >> p.c.page_log2)];
  if (!cache_page_ok(p.c, page)) return;
  const T* const v = static_cast<const T*>(p.c.pool) + (cache_row(p.c, p.layer, 1, page, head) + (at & ((1 << p.c.page_log2) - 1))) * p.c.head_dim;
  for (int c = 0; c < DP; c += 32) {
    float o[32];
    tmem_ld32(out_addr + c, o);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float x = c + j < p.c.head_dim ? to_float(v[c + j]) : 0.0f;
      if (!(fabsf(x) < CUDART_INF_F) && w != 0.0f) o[j] += w * x;
    }
    tmem_st32(out_addr + c, o);
    tmem_st_wait();
  }
}

// MANY: more than kMaskAhead drafted tokens.  (Two kernels: with both ways in one, its registers cost a call of few tokens up to 9%: 109 us where 100 are.)
template <typename T, int DP, bool MANY>
__global__ void __launch_bounds__(kThreads, 1)
cache_attention_tc_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CacheAttnParams p) {
  using Z = TcShape<T, DP>;
  using G = Tile<T, DP>;
  constexpr int TILE = G::kKeys;
  static_assert(TILE == 64, "64 columns of scores");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[2 * Z::kStages + 9];
  __shared__ CacheRunShared found;
  __shared__ unsigned long long odd_keys[2];         // keys of a group's tile whose V is not finite
  __shared__ float2 states[2][kRows];                // the groups' maxima and sums at the end of an item
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;

  const int lane = threadIdx.x & 31, warp = warp_index();
  const uint32_t q_smem = smem_u32(smem), stage0 = q_smem + Z::kQBytes;
  const uint32_t full = smem_u32(bars), empty = full + 8 * Z::kStages, q_full = empty + 8 * Z::kStages, s_full = q_full + 8, p_full = s_full + 16, o_full = p_full + 16, s_free = o_full + 16;
  if (threadIdx.x == 0) {
    gave_up = 0;
    prefetch_tensormap(&map);
    for (int i = 0; i < 2 * Z::kStages; ++i) mbar_init(full + 8 * i, 1);
    mbar_init(q_full, 2 * kRows / 32);
    for (int i = 0; i < 2; ++i) mbar_init(s_full + 8 * i, 1), mbar_init(p_full + 8 * i, kRows / 32), mbar_init(o_full + 8 * i, 1), mbar_init(s_free + 8 * i, kRows / 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  CacheRun run;
  const bool any = find_run<kRows, TILE, kThreads>(p, blockIdx.x, found, &run);
  CacheCursor& now = run.at;
  volatile int* const abort_ptr = &gave_up;
  // A wait that ends for all lanes of a warp or none.  Where it runs out the softmax warps do no more work, but meet each other as if they did.
  auto wait = [&](uint32_t bar, uint32_t parity) { return warp_waits(bar, parity, abort_ptr); };

  if (warp == 0) {
    if (lane == 0) leave_join<kRows>(p, any, run);
    if (any) bring_tiles<T, DP, kRows, Z::kStages>(map, p, run, stage0, full, empty, wait);
  } else if (warp == 1) {
    // ---------------- products ----------------
    // Tiles are numbered over all items; scores, weights and the output's barrier take turns of two.
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
    const uint32_t idesc_qk = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
    const uint32_t idesc_pv = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
    uint32_t items = 0;
    auto issue_qk = [&](uint32_t t, bool first, bool behind) {       // `behind`: the scores of the tile before the last one, in the same place, are of this item
      const uint32_t stage = t % Z::kStages;
      if (first && !wait(q_full, items++ & 1)) return false;
      // (both at once, half of the lanes each)
      const bool scores = behind && (lane & 1) != 0;
      if (!wait(scores ? s_free + 8 * (t & 1) : full + 8 * stage, scores ? ((t - 2) >> 1) & 1 : (t / Z::kStages) & 1)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t k = stage0 + stage * G::kBytes, on = elect_one() ? 1u : 0u;
#pragma unroll
      for (int kd = 0; kd < DP / 16; ++kd)
        umma_if(on, tmem + kColS + (t & 1) * TILE, make_desc(q_smem + kd / 4 * Z::kQBlock + kd % 4 * 32, 16, 1024),
                make_desc(k + kd / 4 * G::kBlockBytes + kd % 4 * 32, 16, 1024), idesc_qk, kd != 0 ? 1u : 0u, true);
      if (on) umma_commit(s_full + 8 * (t & 1));
      __syncwarp();
      return true;
    };
    auto issue_pv = [&](uint32_t t, bool first) {
      const uint32_t stage = t % Z::kStages;
      if (!wait(p_full + 8 * (t & 1), (t >> 1) & 1)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t v = stage0 + stage * G::kBytes + G::kHalf, on = elect_one() ? 1u : 0u;
      // 16 keys = 8 columns of weights and 16 128-byte rows of V per instruction
#pragma unroll
      for (int kk = 0; kk < TILE / 16; ++kk)
        umma_ts_if(on, tmem + (t & 1) * DP, tmem + kColP + (t & 1) * (TILE / 2) + kk * 8, make_desc(v + kk * 2048, G::kBlockBytes, 1024), idesc_pv, !first || kk != 0 ? 1u : 0u, true);
      if (on) {
        umma_commit(o_full + 8 * (t & 1));
        umma_commit(empty + 8 * stage);
      }
      __syncwarp();
      return true;
    };
    uint32_t t = 0;
    bool ok = any;
    for (int tiles; ok && (tiles = run.tiles(p)) > 0; run.pass<kRows, TILE>(p, tiles)) {
      ok = issue_qk(t, true, false) && (tiles == 1 || issue_qk(t + 1, false, false));
      for (int i = 0; i < tiles && ok; ++i, ++t) {
        if (i + 2 < tiles) ok = issue_qk(t + 2, false, true);
        ok = ok && issue_pv(t, i < 2);
      }
    }
  } else {
    // ---------------- softmax: a thread per query row and group ----------------
    const int group = (warp - 2) >> 2, quad = warp & 3, row = quad * 32 + lane, worker = (threadIdx.x - 64) & (kRows - 1);
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16), out_addr = lane_addr + group * DP, scores = lane_addr + kColS + group * TILE, weights = lane_addr + kColP + group * (TILE / 2);
    auto arrive = [&](uint32_t bar) {                // after this warp's last tensor-memory access that the barrier speaks of
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto meet_group = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kRows) : "memory"); };
    auto meet_both = [&]() { asm volatile("bar.sync 3, %0;" ::"n"(2 * kRows) : "memory"); };
    uint32_t t0 = 0;                                 // the item's first tile
    for (int tiles; any && (tiles = run.tiles(p)) > 0; run.pass<kRows, TILE>(p, tiles)) {
      const int rows_here = min(kRows, now.it.count * p.group - now.row_tile * kRows), sure = min(now.it.length, now.it.end);
      const bool there = row < rows_here, warp_there = quad * 32 < rows_here;
      const CacheRow r = row_of<kRows>(p, now, there ? row : 0);
      // What the rows see of up to 64 drafted tokens: a lane has a drafted token and a warp a word in eight of two per token.  All of these loads and those of Q are
      // under way before any is waited for, and they are under the way of the first keys.
      const uint8_t* const mask = p.mask + now.b * p.mask_stride[0];
      const bool masked = !MANY && p.mask != nullptr && (now.tile + tiles) * TILE > sure;
      const int first_token = now.row_tile * kRows / p.group, words = 2 * ((now.row_tile * kRows + rows_here - 1) / p.group - first_token + 1);
      uint32_t seen = 0u;
      if (masked) {
        const int j = (warp & 1) * 32 + lane;                // (the words of a warp are all even or all odd)
        const uint8_t* const column = mask + (j < now.it.count ? j : 0) * p.mask_stride[2];
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int w = warp - 2 + 8 * n;
          if (w < words && column[(first_token + w / 2) * p.mask_stride[1]] != 0 && j < now.it.count) seen |= 1u << n;
        }
      }
      // half a row of Q (the products that read the last item's have been executed: its output was read); zeros for rows that are not there
      if (warp_there) {
        const int64_t from = now.b * p.q_stride[0] + r.token * p.q_stride[1] + r.head * p.q_stride[2];
        uint4 x[DP / 16];
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          const int at = group * (DP / 16) + c;
          x[c] = make_uint4(0u, 0u, 0u, 0u);
          if (there && at * 8 < p.c.head_dim) {
            if (p.q_fp32) {
              const float4* const q = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + from) + at * 2;
              const float4 a = q[0], b = q[1];
              x[c] = make_uint4(pack<T>(a.x, a.y), pack<T>(a.z, a.w), pack<T>(b.x, b.y), pack<T>(b.z, b.w));
            } else {
              x[c] = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + from)[at];
            }
          }
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          const int at = group * (DP / 16) + c;
          *reinterpret_cast<uint4*>(smem + at / 8 * Z::kQBlock + row * 128 + (((at % 8) ^ (row & 7)) << 4)) = x[c];
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      unsigned long long tree = 0ull;
      if (masked) {
        uint32_t* const to = reinterpret_cast<uint32_t*>(states);        // (free between items)
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const uint32_t word = __ballot_sync(0xffffffffu, (seen >> n & 1u) != 0u);
          if (lane == 0 && warp - 2 + 8 * n < words) to[warp - 2 + 8 * n] = word;
        }
        meet_both();
        if (there) tree = to[2 * (r.token - first_token)] | (unsigned long long)to[2 * (r.token - first_token) + 1] << 32;
        meet_both();
      }
      float m = -CUDART_INF_F, l = 0.0f;
      uint32_t done = 0;                             // the group's last tile, plus one
      for (int i = (int)((group + t0) & 1); i < tiles; i += 2) {
        const uint32_t t = t0 + i, stage = t % Z::kStages;
        const int key0 = (now.tile + i) * TILE;
        const bool ok = wait(s_full + 8 * group, (t >> 1) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const bool drafted = key0 + TILE > sure, work = ok && warp_there;
        unsigned long long odd = 0ull;
        if (drafted) {
          // V behind the sequence's end becomes zeros, and so do infinities and NaN (see look_at_values), by all rows' threads of the group together.
          uint8_t* const values = smem + Z::kQBytes + stage * G::kBytes + G::kHalf;
          constexpr int kChunks = G::kBlocks * 8;
          const int in_page = (1 << p.c.page_log2) - 1, last = now.it.end - key0;
          const int from = max(0, sure - key0) * kChunks, to = min(TILE, ((now.it.end + in_page) & ~in_page) - key0) * kChunks;
          if (worker == 0) odd_keys[group] = 0ull;
          meet_group();
          if (wait(full + 8 * stage, (t / Z::kStages) & 1))
            for (int c = from + worker; c < to; c += kRows) {
              uint4* const x = reinterpret_cast<uint4*>(G::at(values, c / kChunks, c % kChunks * 8));
              if (c / kChunks >= last) *x = make_uint4(0u, 0u, 0u, 0u);
              else if ((not_finite<T>(x->x) | not_finite<T>(x->y) | not_finite<T>(x->z) | not_finite<T>(x->w)) & 0x80008000u) {
                atomicOr(&odd_keys[group], 1ull << (c / kChunks));
                *x = make_uint4(finite_pair<T>(x->x), finite_pair<T>(x->y), finite_pair<T>(x->z), finite_pair<T>(x->w));
              }
            }
          fence_async_smem();
          // more drafted tokens than are looked up ahead: those of this tile, the same way
          uint32_t* const to_see = reinterpret_cast<uint32_t*>(states[group]);
          const bool look = MANY && p.mask != nullptr;
          if (look) look_at_tile<kRows>(p, now.b, now.row_tile, now.it.length, now.it.count, key0, to_see);
          meet_group();
          odd = odd_keys[group];
          if (look && there) tree = to_see[2 * (r.token - first_token)] | (unsigned long long)to_see[2 * (r.token - first_token) + 1] << 32;
          meet_group();
        }
        float v[64];
        if (work) {
          {
            float a[32], b[32];
            tmem_ld32x2(scores, scores + 32, a, b);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = a[j], v[32 + j] = b[j];
          }
          arrive(s_free + 8 * group);
          // the product of the group's last tile has read its weights, and the output rows so far are there
          if (done != 0) wait(o_full + 8 * group, ((t - 2) >> 1) & 1);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (drafted) {
            const int off = now.it.length - key0, last = now.it.end - key0;      // where the first drafted token is in the tile; where the keys end
            unsigned long long shows;
            if (p.mask == nullptr) {
              const int n = off + r.token + 1;
              shows = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
            } else {
              shows = MANY ? tree : off >= 64 || off <= -64 ? 0ull : off >= 0 ? tree << off : tree >> -off;
              if (off > 0) shows |= off >= 64 ? ~0ull : (1ull << off) - 1;
            }
            if (last < 64) shows &= last <= 0 ? 0ull : (1ull << last) - 1;
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (!((j < 32 ? (uint32_t)shows : (uint32_t)(shows >> 32)) >> (j & 31) & 1u)) v[j] = -CUDART_INF_F;
          }
          float top[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) top[q] = fmaxf(v[2 * q], v[2 * q + 1]);
#pragma unroll
          for (int j = 8; j < 64; j += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) top[q] = fmax3(top[q], v[j + 2 * q], v[j + 2 * q + 1]);
          const float mx = exponent_of_top<T>(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), p.scale_log2);
          if (done == 0) {
            m = mx;
          } else if (__any_sync(0xffffffffu, mx > m)) {
            const float grown = fmaxf(m, mx), alpha = grown == -CUDART_INF_F ? 1.0f : ex2(m - grown);
            m = grown;
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              float o[32];
              tmem_ld32(out_addr + c, o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] *= alpha;
              tmem_st32(out_addr + c, o);
            }
          }
          float shift = m == -CUDART_INF_F ? 0.0f : -m, scale = p.scale_log2;          // nothing seen so far: every weight is 2^-inf
          if (fabsf(shift) > kFarScore) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = behind_top<T>(v[j], scale, shift);
            scale = 1.0f, shift = 0.0f;
          }
          const float2 scale2 = make_float2(scale, scale), shift2 = make_float2(shift, shift);
          float2 sum2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            uint32_t packed[16];
#pragma unroll
            for (int j = h; j < h + 32; j += 2) {
              const float2 e = ffma2(make_float2(v[j], v[j + 1]), scale2, shift2);
              v[j] = ex2(e.x);
              v[j + 1] = ex2(e.y);
              sum2[j >> 1 & 1] = fadd2(sum2[j >> 1 & 1], make_float2(v[j], v[j + 1]));
              packed[(j - h) / 2] = pack<T>(v[j], v[j + 1]);
            }
            tmem_st16(weights + h / 2, packed);
          }
          l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
          tmem_st_wait();
        } else {
          arrive(s_free + 8 * group);
          if (done != 0) wait(o_full + 8 * group, ((t - 2) >> 1) & 1);       // (no warp arrives for a tile's weights before all have for the last one's)
        }
        arrive(p_full + 8 * group);
        done = t + 1;
        if (odd != 0ull && work) {
          wait(o_full + 8 * group, (t >> 1) & 1);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (odd >> j & 1) add_infinite<T, DP>(p, now.it, now.head, key0 + j, v[j], out_addr);
        }
      }
      // ---- the end of the item, or of the run inside it: both groups' rows, half of the columns each ----
      bool ok = true;
      if (done != 0) ok = wait(o_full + 8 * group, ((done - 1) >> 1) & 1);
      if (l != l) m = 0.0f;                          // (NaN, which a maximum passes over, reaches the result)
      states[group][row] = make_float2(m, l);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      meet_both();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (ok && warp_there) {
        const bool whole = now.tile == 0 && tiles == now.it.key_tiles;
        const float2 a = states[0][row], b = states[1][row];
        const float top = fmaxf(a.x, b.x);
        float fa = a.x == -CUDART_INF_F ? 0.0f : ex2(a.x - top), fb = b.x == -CUDART_INF_F ? 0.0f : ex2(b.x - top);
        const float sum = a.y * fa + b.y * fb;
        if (whole) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          fa *= inv, fb *= inv;
        }
        const bool first = t0 % 2 == 0 || tiles > 1, second = t0 % 2 == 1 || tiles > 1;       // which groups had a tile
        // a part that begins with the run is the run's first, else its second
        float* const part = p.partial + (2 * (int64_t)blockIdx.x + (t0 == 0 ? 0 : 1)) * p.partial_floats;
        T* const to = static_cast<T*>(p.out) + now.b * p.out_stride[0] + r.token * p.out_stride[1] + r.head * p.out_stride[2];
        // (small code: a launch meets it cold)
#pragma unroll 1
        for (int c = group * (DP / 2); c < (group + 1) * (DP / 2); c += 8) {
          float o[8], o2[8];
          tmem_ld8x2(lane_addr + c, lane_addr + DP + c, o, o2);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = (first ? o[j] * fa : 0.0f) + (second ? o2[j] * fb : 0.0f);
          if (there && whole && c < p.c.head_dim) {
            *reinterpret_cast<uint4*>(to + c) = make_uint4(pack<T>(o[0], o[1]), pack<T>(o[2], o[3]), pack<T>(o[4], o[5]), pack<T>(o[6], o[7]));
          } else if (there && !whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j) part[TcMath<T, DP>::place(row, c + j)] = o[j];
          }
          __syncwarp();
        }
        if (!whole && there && group == 0) reinterpret_cast<float2*>(part + TcMath<T, DP>::kOut * 32)[row] = make_float2(top, sum);
      }
      // the next item's products write the output rows behind both groups' next weights
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      meet_both();
      t0 += tiles;
    }
  }

  clear_rows_behind<T>(p, warp, kThreads / 32);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (gave_up && threadIdx.x == 0) {
    cache_fault(p.c, kCacheWaitFault);
    let_copies_land();
  }
  __syncthreads();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
}

// What beginning and ending an item costs, in tiles: 32 sequences of 2000 to 16384 tokens, trees of 32: 269.8 us without, 263.9 with four, 258.9 with eight; five row
// tiles of 20 tiles and more: 101.7, 86.8, 82.0.
constexpr int kItemUnits = 8;

template <typename T, int DP, bool MANY>
CacheAttnVariant tc_variant() {
  using Z = TcShape<T, DP>;
  return CacheAttnVariant{cache_attention_tc_kernel<T, DP, MANY>, cache_attention_join_kernel<TcMath<T, DP>, 1>, kThreads, Z::kSmem, kRows, Z::G::kKeys, 4, kItemUnits,
                          kPartOfWarp<TcMath<T, DP>>};
}
template <typename T, bool MANY>
CacheAttnVariant tc_variant(int head_dim) {
  return head_dim <= 64 ? tc_variant<T, 64, MANY>() : tc_variant<T, 128, MANY>();
}

}  // namespace

CacheAttnVariant cache_attention_tc_variant(int dtype, int head_dim, int tokens) {
  const bool many = tokens > kMaskAhead;
  if (dtype == KB200_DTYPE_BF16) return many ? tc_variant<__nv_bfloat16, true>(head_dim) : tc_variant<__nv_bfloat16, false>(head_dim);
  return many ? tc_variant<__half, true>(head_dim) : tc_variant<__half, false>(head_dim);
}

}  // namespace kb200
