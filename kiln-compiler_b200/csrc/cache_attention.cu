// Attention of drafted tokens over a paged K/V cache (kb200_cache_attend): softmax(scale q K^T, masked) V for the few query rows of
// each sequence, one pass over its keys with a running maximum and sum.
//
// What bounds it: the cache's bytes.  A key head's K and V are read once for all query rows that share them (drafted tokens x heads per key head).
// Products run by warp (cache_attention_math.cuh): the rows of a decoding step do not fill larger units.
//
// A CTA has one producer warp and up to six consumer warps (from the eighth on a scheduler holds three warps and a thread 168 registers) and walks
// its run of key tiles (cache_attention.h).  The producer brings tiles of K and V through a tensor map of the pool, page by page, as far ahead as the ring of stages goes, across the borders of sequences and
// heads.  A consumer warp takes a WHOLE tile for up to 16 query rows and keeps maxima, sums and output rows in registers; the
// warps' sums are joined at the end of an item only.  Every stage of the ring belongs to one warp (or the group of warps with the other rows
// of the row tile), which therefore sees each of its fillings: a barrier's parity tells no more than the last one.  (With the tile's keys divided among the
// warps, and copies issued by them, a warp paid the rescaling, the shuffles and the addresses for 16 keys instead of 64: 985 instructions per warp and tile at 5.8 cycles each, two warps to
// a scheduler, 187 us for 32 sequences of up to 8192 tokens in BF16, 52 % of the bandwidth; now 110, 0.88 of the
// measured copy bandwidth.)
//
// Scores, maxima, sums and output rows are float32.  16-bit caches: the weights of a tile are rounded to the cache's type for the product with V
// (half a step, 2^-9 for bfloat16, of every summand; the largest is 2^12 in float16, so that smaller ones keep their bits too; the sum of the weights is kept of the
// unrounded ones).  float32 caches are not rounded anywhere.
//
// WINDOW: the kernels with a window (kb200_cache_attend_window), which cache_attention_window.cu compiles from the same text.
#include <limits.h>

#include <algorithm>
#include <cmath>

#include "cache_attention_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

using namespace cache_math;

// Warps, ring and shared memory by what the warps do; RG: groups of warps with other rows of the same row tile.
template <typename Math, int RG>
struct Shape {
  using T = typename Math::Type;
  using G = Tile<T, Math::kDim>;
  static constexpr bool kWide = sizeof(T) == 4;
  // groups of warps, each for tiles of its own: as many as there are stages, with what a warp keeps in shared memory beside them
  static constexpr int kMost = kWide ? (Math::kDim <= 64 ? 5 : Math::kDim <= 128 ? 4 : 3) : Math::kDim > 128 ? 5 : 6;
  static constexpr int kGroups = RG == 4 ? 1 : kMost / RG;
  static constexpr int kWarps = kGroups * RG;                            // consumers
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kSlots = RG == 1 && !kWide && Math::kDim <= 128 ? 3 : 2;      // warps whose rows are in shared memory at a time when sums are joined
  static constexpr int kSlotFloats = Math::kOut * 32;
  static constexpr int kQuery = kWide ? Math::kRows * Math::kDim : 0, kWeights = kWide ? G::kKeys * (Math::kRows + 4) : 0;      // floats of a warp
  static constexpr int kBeside = (kSlots * kSlotFloats + kWarps * (kQuery + kWeights)) * 4;
  static constexpr int kStages = kGroups * ((222 * 1024 - kBeside) / G::kBytes / kGroups);      // (a multiple: see above)
  static constexpr int kSmem = kStages * G::kBytes + kBeside;
  static constexpr int kRows = Math::kRows * RG;                         // of a row tile
};

template <typename Math, int RG, bool WINDOW>
__global__ void __launch_bounds__(Shape<Math, RG>::kThreads, 1)
cache_attention_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CacheAttnParams p) {
  using Z = Shape<Math, RG>;
  using T = typename Math::Type;
  using G = typename Z::G;
  constexpr int KG = Z::kGroups, ROWS = Z::kRows, TILE = G::kKeys;
  static_assert(Z::kStages > 0 && Z::kStages % KG == 0 && (KG == 1 || Z::kSlots % RG == 0), "a stage belongs to one group, a slot to a warp of each row group");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[2 * Z::kStages];
  __shared__ CacheRunShared found;
  __shared__ uint2 sees[Z::kWarps][16];            // a tile with drafted tokens: which row sees which key
  __shared__ float2 states[Z::kWarps][Math::kRows];       // maxima and sums, by place in an item that several groups had a tile of
  __shared__ float2 own_states[Z::kWarps][Math::kRows];   // ... of all of them, or of a warp that had it alone: others may be at other items
  __shared__ float factors[Z::kWarps][Math::kRows];
  __shared__ int gave_up;

  const int lane = threadIdx.x & 31, warp = warp_index();
  const uint32_t stage0 = smem_u32(smem), full = smem_u32(bars), empty = full + 8 * Z::kStages;
  if (threadIdx.x == 0) {
    gave_up = 0;
    prefetch_tensormap(&map);
    for (int i = 0; i < Z::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, RG);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  CacheRun run;
  const bool any = find_run<ROWS, TILE, Z::kThreads, WINDOW>(p, blockIdx.x, found, &run);       // (a barrier for all that is above, too)
  CacheCursor& now = run.at;
  volatile int* const abort_ptr = &gave_up;
  // A wait that ends for all lanes of a warp or none.  Where it runs out the warps do no more work, but meet each other as if they did.
  auto wait = [&](uint32_t bar, uint32_t parity) { return warp_waits(bar, parity, abort_ptr); };

  if (warp == Z::kWarps) {
    if (lane == 0) leave_join<ROWS>(p, any, run);
    if (any) bring_tiles<T, Math::kDim, ROWS, Z::kStages, WINDOW>(map, p, run, stage0, full, empty, wait);
  } else {
    // ---------------- consumers ----------------
    const int row_group = warp % RG, key_group = warp / RG;
    float* const slots = reinterpret_cast<float*>(smem + Z::kStages * G::kBytes);
    float* const query = slots + Z::kSlots * Z::kSlotFloats + warp * (Z::kQuery + Z::kWeights);
    auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::kWarps) : "memory"); };

    Math math;
    Place at{nullptr, nullptr, 0, 0, row_group * Math::kRows, 0, 0, warp, lane, row_group, key_group};

    // The end of an item, or of the run inside one: the warps' sums, then the rows or a part.  `order`: this warp's place among those that had a tile of
    // it, in the order of the keys.
    auto finish = [&](int order, int tiles, bool whole, int64_t part) {
      math.sum_up();
      int n = min(KG, tiles);                        // groups of keys that had a tile
      math.put_states(lane, n > 1 ? states[order * RG + row_group] : own_states[warp]);
      if (n > 1) {
        meet();
        // to the largest maximum
        float factor = 0.0f;
        float2 all = make_float2(-CUDART_INF_F, 0.0f);
        const int row = lane % Math::kRows;
        const float top = states[order * RG + row_group][row].x;
        for (int w = 0; w < n; ++w) all.x = fmaxf(all.x, states[w * RG + row_group][row].x);
        for (int w = 0; w < n; ++w) {
          const float2 state = states[w * RG + row_group][row];
          if (state.x != -CUDART_INF_F) all.y += state.y * ex2(Math::exponent(state.x - all.x, p.scale_log2));
        }
        if (top != -CUDART_INF_F) factor = ex2(Math::exponent(top - all.x, p.scale_log2));
        if (lane < Math::kRows) factors[warp][lane] = factor;
        meet();                                      // (which also says that the states have been read)
        math.rescale(lane, factors[warp]);
        if (lane < Math::kRows) own_states[warp][lane] = all;
        while (n > 1) {                              // the upper half's rows go to the lower half, as many at a time as there are slots
          const int half = (n + 1) / 2;
          for (int from = half; from < n; from += Z::kSlots / RG) {
            const int to = min(n, from + Z::kSlots / RG);
            float* const slot = slots + ((order >= half ? order - from : order + half - from) * RG + row_group) * Z::kSlotFloats + lane;
            if (order >= from && order < to) math.each_out([&](int i, float x) { slot[i * 32] = x; });
            meet();
            if (order + half >= from && order + half < to) math.each_out([&](int i, float& x) { x += slot[i * 32]; });
            meet();
          }
          n = half;
        }
      }
      __syncwarp();
      if (order != 0) return;
      if (whole) {
        math.template write<ROWS, WINDOW>(p, now, at, own_states[warp], query);
      } else {
        float* const to = p.partial + part * p.partial_floats + row_group * kPartOfWarp<Math>;
        math.each_out([&](int i, float x) { to[i * 32 + lane] = x; });
        if (lane < Math::kRows) reinterpret_cast<float2*>(to + Math::kOut * 32)[lane] = own_states[warp][lane];
      }
    };

    uint32_t u0 = 0;
    for (int tiles; any && (tiles = run.tiles(p)) > 0; run.pass<ROWS, TILE, WINDOW>(p, tiles)) {
      at.rows_here = min(ROWS, now.it.count * p.group - now.row_tile * ROWS);
      at.sure = min(now.it.length, now.it.end);
      CacheGap gap{0, 0};
      if constexpr (WINDOW) {
        gap = gap_of<ROWS, TILE>(p, now);
        at.sure = min(sure_keys<ROWS>(p, now), now.it.end);
        at.hidden = now.it.length + last_place<ROWS>(p, now.row_tile, at.rows_here) - p.window + 1;
      }
      auto key_of = [&](int tile) { return (WINDOW ? gap.tile(tile) : tile) * TILE; };
      if constexpr (Z::kWide) math.template begin<ROWS>(p, now, at, query);
      else math.template begin<ROWS>(p, now, at);
      const int order = (int)((key_group + KG - u0 % KG) % KG);
      uint32_t ahead = 0u;
      if (p.mask != nullptr && p.tokens <= kMaskAhead && order < tiles && key_of(now.tile + tiles - 1) + TILE > at.sure)
        ahead = mask_word<ROWS>(p, now, at, (lane >> 4) * 32);
      for (int i = order; i < tiles; i += KG) {
        const uint32_t u = u0 + i, stage = u % Z::kStages;
        at.key0 = key_of(now.tile + i);
        if (wait(full + 8 * stage, (u / Z::kStages) & 1)) {
          at.k = smem + stage * G::kBytes;
          at.v = at.k + G::kHalf;
          if constexpr (Z::kWide) math.template tile<ROWS, WINDOW>(p, now, at, ahead, sees[warp], query, query + Z::kQuery);
          else math.template tile<ROWS, WINDOW>(p, now, at, ahead, sees[warp]);
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * stage);
        }
      }
      // a part that begins with the run is the run's first, else its second
      finish(order, tiles, now.tile == 0 && tiles == now.it.key_tiles, 2 * (int64_t)blockIdx.x + (u0 == 0 ? 0 : 1));
      u0 += tiles;
    }
  }
  clear_rows_behind<T, WINDOW>(p, warp, Z::kWarps + 1);
  __syncthreads();
  if (gave_up && threadIdx.x == 0) {
    cache_fault(p.c, kCacheWaitFault);
    let_copies_land();
  }
  __syncthreads();
}

using Variant = CacheAttnVariant;

// What beginning and ending an item costs, in tiles.  32 sequences of 1000 to 8192 tokens, BF16: 128.5 us without, 119.9 with two tiles, 115.2 with four, 111.2 with
// six, 110.1 with eight (but 17.0 instead of 16.0 us for 36 items of 28 tiles); trees of 9 in FP32: 40.1, 37.9, 36.5, 37.0, 37.9.
template <typename Math>
constexpr int kItemUnits = sizeof(typename Math::Type) == 4 ? 4 : 6;

template <typename Math, int RG, bool WINDOW>
Variant variant() {
  using Z = Shape<Math, RG>;
  return Variant{cache_attention_kernel<Math, RG, WINDOW>, cache_attention_join_kernel<Math, RG, WINDOW>, Z::kThreads, Z::kSmem,
                 Z::kRows, Z::G::kKeys, Z::kGroups, kItemUnits<Math>, (int64_t)RG * kPartOfWarp<Math>};
}

// By the rows of an item, up to 64 to a row tile.
template <typename T, int DP, bool WINDOW>
Variant variant_of(int rows) {
  if constexpr (sizeof(T) == 4)
    return rows <= 2 ? variant<FmaMath<DP, 2>, 1, WINDOW>() : rows <= 4 ? variant<FmaMath<DP, 4>, 1, WINDOW>() : rows <= 8 ? variant<FmaMath<DP, 8>, 1, WINDOW>()
           : rows <= 12 ? variant<FmaMath<DP, 12>, 1, WINDOW>() : rows <= 16 ? variant<FmaMath<DP, 16>, 1, WINDOW>() : rows <= 32 ? variant<FmaMath<DP, 16>, 2, WINDOW>() : variant<FmaMath<DP, 16>, 4, WINDOW>();
  else if constexpr (DP <= 128)
    return rows <= 16 ? variant<MmaMath<T, DP>, 1, WINDOW>() : variant<MmaMath<T, DP>, 2, WINDOW>();       // (more: tcgen05)
  else
    return rows <= 16 ? variant<MmaMath<T, DP>, 1, WINDOW>() : rows <= 32 ? variant<MmaMath<T, DP>, 2, WINDOW>() : variant<MmaMath<T, DP>, 4, WINDOW>();
}
template <typename T, bool WINDOW>
Variant variant_of(int head_dim, int rows) {
  return head_dim <= 64 ? variant_of<T, 64, WINDOW>(rows) : head_dim <= 128 ? variant_of<T, 128, WINDOW>(rows) : variant_of<T, 256, WINDOW>(rows);
}
template <bool WINDOW>
Variant variant_of(int dtype, int head_dim, int rows) {
  return dtype == KB200_DTYPE_FP32 ? variant_of<float, WINDOW>(head_dim, rows)
         : dtype == KB200_DTYPE_BF16 ? variant_of<__nv_bfloat16, WINDOW>(head_dim, rows) : variant_of<__half, WINDOW>(head_dim, rows);
}

}  // namespace

#ifdef KB200_WINDOW
CacheAttnVariant cache_attention_warp_window_variant(int dtype, int head_dim, int rows) { return variant_of<true>(dtype, head_dim, rows); }
}  // namespace kb200
#else
namespace {

// ---- host --------------------------------------------------------------------------------------

// 16-bit caches go to tiles of 128 rows on tcgen05 above this many rows of an item, above half of it where the items are fewer than half of the SMs.  (BF16, heads
// of 128, four to a key head, up to 8192 tokens.  32 sequences of 20, 32, 48 and 64 rows: 110, 121, 164, 151 us by warps; 127, 137, 127, 119 on tcgen05.  One sequence of
// 20, 32 and 64 rows: 28.2, 29.1, 34.2 us and 21.9, 22.3, 24.7.)
constexpr int kFewRows = 32;

Variant variant_for(const Cache& c, int rows, int tokens, bool many_items, bool window) {
  if (c.dtype != KB200_DTYPE_FP32 && c.view.head_dim <= 128 && rows > (many_items ? kFewRows : kFewRows / 2))
    return window ? cache_attention_tc_window_variant(c.dtype, c.view.head_dim, tokens) : cache_attention_tc_variant(c.dtype, c.view.head_dim, tokens);
  return window ? cache_attention_warp_window_variant(c.dtype, c.view.head_dim, rows) : variant_of<false>(c.dtype, c.view.head_dim, rows);
}
Variant variant_for(const Cache& c, int rows, int tokens, int heads, bool window) {
  return variant_for(c, tokens * (heads / c.view.kv_heads), tokens, 2 * (int64_t)rows * c.view.kv_heads >= c.sm_count, window);
}

// How a call is divided: a CTA per SM, but no more than have a tile for each of their warps.
struct Division {
  int parts, min_units, item_units;
  bool whole;
};
Division division_of(const Cache& c, const Variant& v, int rows, int tokens, int heads, int64_t most_keys) {
  const int64_t row_tiles = ((int64_t)tokens * (heads / c.view.kv_heads) + v.rows - 1) / v.rows;
  const int64_t tiles = std::min(most_keys, ((int64_t)c.view.max_pages << c.view.page_log2) + v.tile - 1) / v.tile;
  Division d{0, 1, 0, tiles <= v.groups};
  if (!d.whole) d.min_units = v.groups, d.item_units = v.item_units;
  const double units = (double)rows * c.view.kv_heads * row_tiles * (d.whole ? 1 : tiles + d.item_units);
  d.parts = (int)std::min<double>(std::ceil(units / d.min_units), (double)c.sm_count);
  return d;
}
uint64_t workspace_of(const Variant& v, const Division& d) {
  return d.whole ? 0 : (uint64_t)d.parts * (2 * v.part_floats * sizeof(float) + sizeof(CacheJoin));
}

constexpr int64_t kAllKeys = INT64_MAX;
// Keys of the tiles that an item may have (cache_items): those with the first keys, and a window's wherever it lies.
int64_t window_keys(const Variant& v, int tokens, int window, int sinks) {
  const int64_t front = ((int64_t)sinks + v.tile - 1) / v.tile, near = ((int64_t)window + tokens - 1 + v.tile - 2) / v.tile + 1;
  return (front + near) * v.tile;
}

// What a call with a window or with the logarithms of sums asks for beside (window 0: neither).
struct Beside {
  int window = 0, sinks = 0;
  const int32_t* places = nullptr;
  float* lse = nullptr;
  int64_t lse_stride[3] = {0, 0, 0};
};

}  // namespace

int cache_attention_prepare(Cache& c) {
  const EncodeFn encode = encode_fn();
  if (encode == nullptr) return fail(KB200_ERR_CUDA, "kb200_cache_create: the driver has no cuTensorMapEncodeTiled");
  const CacheView& v = c.view;
  const int page = 1 << v.page_log2, columns = 128 / c.element, tile = variant_for(c, 1, 1, true, false).tile;
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
  for (const int tokens : {1, kMaskAhead + 1})
    for (const int rows : {2, 4, 8, 12, 16, 32, 64})
      for (const bool window : {false, true}) {
        const Variant of = variant_for(c, rows, tokens, true, window);
        KB200_CUDA(cudaFuncSetAttribute(of.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, of.smem));
      }
  return KB200_OK;
}

namespace {

int attend(kb200_cache* handle, int layer, const kb200_rows* q, const kb200_rows* out, int rows, int tokens, const uint8_t* mask, const int64_t* mask_stride,
           const int32_t* counts, const int32_t* slots, float scale, const Beside& beside, void* workspace, uint64_t workspace_bytes, void* stream) {
  const bool window = beside.window > 0;
  if (handle == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: cache is null");
  const Cache& c = *cache_of(handle);
  if (layer < 0 || layer >= c.view.layers) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: layer %d of %d", layer, c.view.layers);
  if (q == nullptr || out == nullptr || q->heads != out->heads || !cache_attention_call_ok(c, rows, tokens, q->heads) || (slots == nullptr && rows > c.view.sequences))
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
  if (!(scale >= 1e-30f) || !(scale <= 1e30f)) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend: scale must be from 1e-30 to 1e30");
  const Variant v = variant_for(c, rows, tokens, q->heads, window);
  const Division d = division_of(c, v, rows, tokens, q->heads, window ? window_keys(v, tokens, beside.window, beside.sinks) : kAllKeys);
  const uint64_t need = workspace_of(v, d);
  if (need > 0 && (workspace == nullptr || !tc::aligned16(workspace) || workspace_bytes < need))
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
  p.joins = d.whole ? nullptr : static_cast<CacheJoin*>(workspace);
  p.partial = reinterpret_cast<float*>(static_cast<CacheJoin*>(workspace) + d.parts);
  p.partial_floats = v.part_floats;
  p.layer = layer;
  p.rows = rows;
  p.tokens = tokens;
  p.heads = q->heads;
  p.group = q->heads / c.view.kv_heads;
  p.parts = d.parts;
  p.min_units = d.min_units;
  p.item_units = d.item_units;
  p.whole = d.whole;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.q_fp32 = q->dtype != c.dtype;
  p.window = beside.window;
  p.sinks = beside.sinks;
  p.places = beside.places;
  p.lse = beside.lse;
  for (int i = 0; i < 3; ++i) p.lse_stride[i] = beside.lse_stride[i];
  KB200_CUDA(launch_kernel(true, v.kernel, dim3(d.parts), dim3(v.threads), v.smem, s, c.map, p));
  if (!d.whole) KB200_CUDA(launch_kernel(true, v.join, dim3(d.parts, std::max(1, v.rows / 8)), dim3(kJoinThreads), 0, s, p));
  return KB200_OK;
}

uint64_t workspace_for(const kb200_cache* handle, int rows, int tokens, int heads, int window, int sinks) {
  if (handle == nullptr) return 0;
  const Cache& c = *cache_of(handle);
  if (!cache_attention_call_ok(c, rows, tokens, heads) || rows == 0 || tokens == 0) return 0;
  const Variant v = variant_for(c, rows, tokens, heads, window > 0);
  return workspace_of(v, division_of(c, v, rows, tokens, heads, window > 0 ? window_keys(v, tokens, window, sinks) : kAllKeys));
}

}  // namespace
}  // namespace kb200

using namespace kb200;

KB200_EXPORT uint64_t kb200_cache_attend_workspace(const kb200_cache* handle, int rows, int tokens, int heads) { return workspace_for(handle, rows, tokens, heads, 0, 0); }

KB200_EXPORT int kb200_cache_attend(kb200_cache* handle, int layer, const kb200_rows* q, const kb200_rows* out, int rows, int tokens,
                                    const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale,
                                    void* workspace, uint64_t workspace_bytes, void* stream) {
  return attend(handle, layer, q, out, rows, tokens, mask, mask_stride, counts, slots, scale, Beside(), workspace, workspace_bytes, stream);
}

// (No window: one that all tokens are in.)
KB200_EXPORT uint64_t kb200_cache_attend_window_workspace(const kb200_cache* handle, int rows, int tokens, int heads, int window, int sinks) {
  if (window < 0 || sinks < 0) return 0;
  return workspace_for(handle, rows, tokens, heads, window == 0 ? INT_MAX : window, sinks);
}

KB200_EXPORT int kb200_cache_attend_window(kb200_cache* handle, int layer, const kb200_rows* q, const kb200_rows* out, int rows, int tokens,
                                           const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale,
                                           int window, int sinks, const int32_t* places, float* lse, const int64_t* lse_stride,
                                           void* workspace, uint64_t workspace_bytes, void* stream) {
  if (window < 0 || sinks < 0) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend_window: a window of %d tokens behind %d", window, sinks);
  if (lse != nullptr && lse_stride == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_attend_window: lse without strides");
  Beside beside;
  beside.window = window == 0 ? INT_MAX : window;
  beside.sinks = sinks;
  beside.places = places;
  beside.lse = lse;
  for (int i = 0; i < 3; ++i) beside.lse_stride[i] = lse != nullptr ? lse_stride[i] : 0;
  return attend(handle, layer, q, out, rows, tokens, mask, mask_stride, counts, slots, scale, beside, workspace, workspace_bytes, stream);
}
#endif
