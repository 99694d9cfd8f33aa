// What the kernels of the attention over a paged cache share: the call's parameters and how its work is divided.
#pragma once

#include "cache.h"

namespace kb200 {

struct CacheAttnParams {
  CacheView c;
  const void* q;
  void* out;
  int64_t q_stride[3], out_stride[3];      // batch row, token, head; elements
  const uint8_t* mask;                     // null: token t is seen by t and those behind it
  int64_t mask_stride[3];
  const int32_t *counts, *slots;
  struct CacheJoin* joins;                 // see below, as are these
  float* partial;
  int64_t partial_floats;                  // of one part
  int layer, rows, tokens, heads, group;
  int parts;                               // CTAs that share the work at most
  int min_units;                           // ... each this many units at least
  int item_units;                          // what beginning and ending an item costs
  float scale_log2;
  bool whole;                              // items are not divided: no parts
  bool q_fp32;                             // q is float32 where the cache is not
  // of kernels with a window (WINDOW below)
  int window, sinks;
  const int32_t* places;                   // null: token t stands t behind the committed ones
  float* lse;                              // or null
  int64_t lse_stride[3];
  bool committed;                          // (kOrCommitted, in the place of WINDOW) the rows are the last of the committed tokens
};
constexpr int kOrCommitted = 2;

// Work is counted in units: a tile of keys for a tile of query rows (the drafted tokens of a sequence times the heads that share a key head), and in front of an
// item's tiles a few for its beginning and end.  All units of a call, sequence by sequence, key head by key head, row tile by row tile, are divided into equal runs of neighbours, one
// per CTA, whatever the sequences' lengths are: a ragged batch keeps all SMs busy to the end.  A run that starts or ends inside an item (a
// row tile of a head of a sequence) leaves its part of the softmax in the workspace, at most two parts per CTA; the
// second launch joins them in the order of the keys.  Where no sequence can have more tiles than a CTA works on at once the units are whole items, and there is
// nothing to join.

// What CTA x leaves for CTA x of the second launch: the item that ends in its run and began before it.
struct CacheJoin {
  int b, head, row_tile, rows;             // rows 0: there is none
  int first, later;                        // the run that its first tile is in; 1: behind another item's, so that its part is that run's second
  int pad[2];
};

struct CacheItems {                        // of one batch row
  int slot, length, count;                 // committed and drafted tokens
  int end;                                 // keys
  int row_tiles, key_tiles;
  int64_t units;
};

#ifdef __CUDACC__
// A window: a row at position P sees the keys from P - window + 1 on, and the first `sinks`.  The tiles of an item are those with the first keys that it sees, and, behind
// a gap, those from the first key that its first row sees in its window.  (WINDOW is a parameter of the kernels, so that calls without one keep their registers.)
struct CacheGap {
  int front, gap;                          // tiles in front of it; tiles that are left out
  __device__ __forceinline__ int tile(int i) const { return i < front ? i : i + gap; }
};
// Of the rows from place `place` on.
template <int TILE>
__device__ __forceinline__ CacheGap gap_of(const CacheAttnParams& p, int length, int place) {
  const int begin = max(0, length + place - p.window + 1), front = (min(p.sinks, begin) + TILE - 1) / TILE;
  return CacheGap{front, max(0, begin / TILE - front)};
}
// Tokens that a tile of query rows has at most.
template <int ROWS>
__host__ __device__ __forceinline__ int tokens_of_tile(int group) { return ROWS % group == 0 ? ROWS / group : (ROWS + group - 2) / group + 1; }
// Tiles from the window's first key to the rows' last, wherever they lie.
template <int TILE>
__host__ __device__ __forceinline__ int64_t window_tiles(int window, int tokens) { return ((int64_t)window + tokens - 1 + TILE - 2) / TILE + 1; }

// The last place of an item's rows.
template <int ROWS>
__device__ __forceinline__ int last_place(const CacheAttnParams& p, int row_tile, int rows_here) {
  return p.mask != nullptr || p.places != nullptr ? p.tokens - 1 : (row_tile * ROWS + rows_here - 1) / p.group;
}
__device__ __forceinline__ int place_of(const CacheAttnParams& p, int b, int token) {
  return p.places == nullptr ? token : min(max(p.places[(int64_t)b * p.tokens + token], 0), p.tokens - 1);
}
__device__ __forceinline__ bool own_places(const CacheAttnParams& p) { return p.mask == nullptr && p.places == nullptr; }

template <int ROWS, int TILE, int WINDOW>
__device__ __forceinline__ CacheItems cache_items(const CacheAttnParams& p, int b) {
  CacheItems r{};
  const int slot = p.slots != nullptr ? p.slots[b] : b;
  int count = p.counts != nullptr ? p.counts[b] : p.tokens;
  if ((unsigned)slot >= (unsigned)p.c.sequences || count < 0 || count > p.tokens) {
    cache_fault(p.c, KB200_CACHE_BAD_INDEX);
    if ((unsigned)slot >= (unsigned)p.c.sequences) return r;
    count = min(max(count, 0), p.tokens);
  }
  const int64_t room = (int64_t)min(max(p.c.held[slot], 0), p.c.max_pages) << p.c.page_log2;
  int length = max(p.c.lengths[slot], 0);
  if constexpr (WINDOW == kOrCommitted) {
    if (p.committed) {
      if (count > length) cache_fault(p.c, KB200_CACHE_BAD_INDEX);
      count = min(count, length);
      length -= count;
    }
  }
  r.slot = slot;
  r.count = count;
  r.length = length;
  r.end = (int)min((int64_t)length + count, room);              // tokens without a page are left out
  if (count == 0) return r;
  if (r.end < length + count) cache_fault(p.c, KB200_CACHE_NO_ROOM);
  r.row_tiles = (count * p.group + ROWS - 1) / ROWS;
  r.key_tiles = max(1, (r.end + TILE - 1) / TILE);
  if constexpr (WINDOW == 1) {
    if (r.row_tiles > 1 && own_places(p)) {          // row tiles begin at keys of their own; all have as many tiles as any may have
      const int begin = max(0, length + count - p.window), front = (min(p.sinks, begin) + TILE - 1) / TILE;
      r.key_tiles = (int)min((int64_t)r.key_tiles, front + window_tiles<TILE>(p.window, tokens_of_tile<ROWS>(p.group)));
    } else {
      r.key_tiles = max(1, r.key_tiles - gap_of<TILE>(p, length, 0).gap);
    }
  }
  r.units = (int64_t)r.row_tiles * (p.whole ? 1 : r.key_tiles + p.item_units) * p.c.kv_heads;
  return r;
}

// Where a run is: an item (batch row, key head, row tile) and a key tile of it.
struct CacheCursor {
  int b, head, row_tile, tile;
  CacheItems it;
};
// The gap of the item at hand.
template <int ROWS, int TILE>
__device__ __forceinline__ CacheGap gap_of(const CacheAttnParams& p, const CacheCursor& u) {
  return gap_of<TILE>(p, u.it.length, u.it.row_tiles > 1 && own_places(p) ? u.row_tile * ROWS / p.group : 0);
}
// Keys in front of which a mask hides nothing from an item's rows: without one, those up to its first row's own.
template <int ROWS>
__device__ __forceinline__ int sure_keys(const CacheAttnParams& p, const CacheCursor& u) {
  return u.it.length + (p.mask == nullptr ? u.row_tile * ROWS / p.group + 1 : 0);
}
// To the next item.
template <int ROWS, int TILE, int WINDOW>
__device__ __forceinline__ void next_item(const CacheAttnParams& p, CacheCursor& u) {
  u.tile = 0;
  if (++u.row_tile < u.it.row_tiles) return;
  u.row_tile = 0;
  if (++u.head < p.c.kv_heads) return;
  u.head = 0;
  while (++u.b < p.rows) {
    u.it = cache_items<ROWS, TILE, WINDOW>(p, u.b);
    if (u.it.units > 0) return;
  }
}

struct CacheRun {
  int64_t all, lo, hi;             // units of the call, of this CTA
  int parts;                       // CTAs that have any
  CacheCursor at;
  int64_t left;                    // units from here on, the first `skip` of which are not tiles
  int skip;
  // The tiles of the item at hand that are in the run; 0: the run ends here.
  __device__ __forceinline__ int tiles(const CacheAttnParams& p) const {
    if (left <= skip) return 0;
    return p.whole ? at.it.key_tiles : (int)min(left - skip, (int64_t)at.it.key_tiles - at.tile);
  }
  template <int ROWS, int TILE, int WINDOW = false>
  __device__ __forceinline__ void pass(const CacheAttnParams& p, int tiles) {
    left -= p.whole ? 1 : skip + tiles;
    skip = p.item_units;
    if (left > 0) next_item<ROWS, TILE, WINDOW>(p, at);
  }
};
struct CacheRunShared {
  int64_t sums[32], rest;
  int b;
  CacheItems it;
};

// The run of CTA `part`, by all threads of a CTA of THREADS; false: it has none.
template <int ROWS, int TILE, int THREADS, int WINDOW = false>
__device__ __forceinline__ bool find_run(const CacheAttnParams& p, int part, CacheRunShared& shared, CacheRun* run) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool one_round = p.rows <= THREADS;
  int64_t base = 0, from = 0;
  CacheItems it{};
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 0 || !one_round) {
      base = 0;
      for (int b0 = 0; b0 < p.rows; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        if (b < p.rows) it = cache_items<ROWS, TILE, WINDOW>(p, b);
        else it.units = 0;
        int64_t sum = it.units;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int64_t below = __shfl_up_sync(0xffffffffu, sum, d);
          if (lane >= d) sum += below;
        }
        __syncthreads();
        if (lane == 31) shared.sums[warp] = sum;
        __syncthreads();
        int64_t before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
          before += w < warp ? shared.sums[w] : 0;
          total += shared.sums[w];
        }
        from = base + before + sum - it.units;
        if (pass == 1 && run->lo >= from && run->lo < from + it.units) shared.b = b, shared.rest = run->lo - from, shared.it = it;
        base += total;
      }
    } else if (run->lo >= from && run->lo < from + it.units) {
      shared.b = threadIdx.x, shared.rest = run->lo - from, shared.it = it;
    }
    if (pass == 0) {
      run->all = base;
      run->parts = (int)min((int64_t)p.parts, (base + p.min_units - 1) / p.min_units);
      if (part >= run->parts) return false;
      run->lo = base * part / run->parts;
      run->hi = base * (part + 1) / run->parts;
    }
  }
  __syncthreads();
  CacheCursor& at = run->at;
  at.b = shared.b;
  at.it = shared.it;
  int64_t rest = shared.rest;
  const int item = p.whole ? 1 : at.it.key_tiles + p.item_units;
  const int64_t per_head = (int64_t)at.it.row_tiles * item;
  at.head = (int)(rest / per_head);
  rest -= at.head * per_head;
  at.row_tile = (int)(rest / item);
  const int in_item = (int)(rest - (int64_t)at.row_tile * item);
  at.tile = max(0, in_item - p.item_units);
  run->skip = max(0, p.item_units - in_item);
  run->left = run->hi - run->lo;
  return true;
}

// By one thread of every CTA of the first launch.
template <int ROWS>
__device__ __forceinline__ void leave_join(const CacheAttnParams& p, bool any, const CacheRun& run) {
  if (p.joins == nullptr) return;
  CacheJoin j{};
  const CacheCursor& at = run.at;
  if (any && at.tile != 0 && at.it.key_tiles - at.tile <= run.hi - run.lo) {
    const int64_t first_tile = run.lo - at.tile;
    j.b = at.b, j.head = at.head, j.row_tile = at.row_tile;
    j.rows = min(ROWS, at.it.count * p.group - at.row_tile * ROWS);
    j.first = (int)(((first_tile + 1) * run.parts - 1) / run.all);
    j.later = run.all * j.first / run.parts < first_tile - p.item_units ? 1 : 0;
  }
  p.joins[blockIdx.x] = j;
}

// An item's row: the token and, of the heads that share its key head, the one.
struct CacheRow {
  int token, head;
};
template <int ROWS>
__device__ __forceinline__ CacheRow row_of(const CacheAttnParams& p, int row_tile, int head, int row) {
  const int r = row_tile * ROWS + row, token = r / p.group;
  return CacheRow{token, head * p.group + r - token * p.group};
}
template <int ROWS>
__device__ __forceinline__ CacheRow row_of(const CacheAttnParams& p, const CacheCursor& at, int row) { return row_of<ROWS>(p, at.row_tile, at.head, row); }
#endif

}  // namespace kb200
