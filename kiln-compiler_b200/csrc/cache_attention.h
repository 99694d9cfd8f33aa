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
  float* partial;                          // see below
  int64_t partial_floats;                  // of one part
  int layer, rows, tokens, heads, group;
  int parts;                               // CTAs that share the work at most
  int min_units;                           // ... each this many units at least
  float scale_log2;
  bool q_fp32;                             // q is float32 where the cache is not
};

// Work is counted in units: a tile of keys for a tile of query rows (the drafted tokens of a sequence times the heads that share a key head).  All units
// of a call, sequence by sequence, key head by key head, row tile by row tile, are divided into equal runs of neighbours, one
// per CTA, whatever the sequences' lengths are: a ragged batch keeps all SMs busy to the end.  A run that starts or ends inside an item (a
// row tile of a head of a sequence) leaves its part of the softmax in the workspace, at most two parts per CTA; the
// second launch joins them in the order of the keys.

struct CacheItems {                        // of one batch row
  int slot, length, count;                 // committed and drafted tokens
  int end;                                 // keys
  int row_tiles, key_tiles;
  int64_t units;
};

#ifdef __CUDACC__
template <int ROWS, int TILE>
__device__ __forceinline__ CacheItems cache_items(const CacheAttnParams& p, int b) {
  CacheItems r{};
  const int slot = p.slots != nullptr ? p.slots[b] : b;
  if ((unsigned)slot >= (unsigned)p.c.sequences) {
    cache_fault(p.c, KB200_CACHE_BAD_INDEX);
    return r;
  }
  int count = p.counts != nullptr ? p.counts[b] : p.tokens;
  if (count < 0 || count > p.tokens) {
    cache_fault(p.c, KB200_CACHE_BAD_INDEX);
    count = min(max(count, 0), p.tokens);
  }
  const int64_t room = (int64_t)min(max(p.c.held[slot], 0), p.c.max_pages) << p.c.page_log2;
  const int length = max(p.c.lengths[slot], 0);
  r.slot = slot;
  r.count = count;
  r.length = length;
  r.end = (int)min((int64_t)length + count, room);              // tokens without a page are left out
  if (count == 0) return r;
  if (r.end < length + count) cache_fault(p.c, KB200_CACHE_NO_ROOM);
  r.row_tiles = (count * p.group + ROWS - 1) / ROWS;
  r.key_tiles = max(1, (r.end + TILE - 1) / TILE);
  r.units = (int64_t)r.row_tiles * r.key_tiles * p.c.kv_heads;
  return r;
}
#endif

}  // namespace kb200
