// The pages of a K/V cache: forking, making room (with the copies that sharing asks for), freeing, compacting, writing new tokens and keeping
// the accepted ones.  State and rules: include/kb200.h.
//
// What bounds them: the bytes of the tokens that move.  The tables are small (4 bytes per page and sequence), so the work on them
// is all latency, and is done on the device so that a step of a serving loop needs no answer from the host and can be one graph.
// Nothing here depends on the order in which threads arrive: free pages are handed out by rank (a prefix sum), holders
// are counted with integer atomics, and the list of copies is the only thing in any order.
//
// Tables that belong together change in one launch: of one CTA where they are small, else of a single cluster, whose CTAs meet at the hardware barrier (all of them
// are resident by definition, so nothing can wait for a CTA that has not started); the tokens then move in a launch over the whole GPU.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>

#include <algorithm>
#include <new>

#include "cache.h"
#include "tc_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

constexpr int kCluster = 8;              // CTAs of a launch on the tables, the largest cluster that every GPU of the kind takes
constexpr int kTableThreads = 1024;
// One CTA up to here, whose barrier costs less than a cluster's: four beams of two prompts, forked and reserved, 17.4 us by clusters, 10.6 so; 96 pages compacted 21.4
// and 14.7; a step of 64 drafting sequences 53.3 and 49.9.  But 128 sequences, eight beams each, 73.4 and 81.4.  (16384 pages are 16 to a thread.)
constexpr int kFewPages = 16384, kFewSequences = 64;

// counters: how many copies, pages in use, new pages of all sequences, and per CTA of the cluster three counts of its pages
enum { kCopies = 0, kUsed, kWanted, kPerCta, kCounters = kPerCta + 3 * kCluster };

struct Scratch {
  int32_t *rows, *slot, *page_a, *page_b;
  int4* copies;
  int* counters;
};

// All threads of the launch meet; what they wrote is there.
template <bool ONE>
__device__ __forceinline__ void meet() {
  if constexpr (ONE) {
    __syncthreads();
  } else {
    tc::cluster_arrive();
    tc::cluster_wait();
  }
}

// Exclusive prefix sum over the block's threads; `total` for all.  Shared memory for a value per warp.
template <typename S>
__device__ __forceinline__ S block_scan(S value, S* shared, S* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  S sum = value;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const S below = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += below;
  }
  __syncthreads();                       // (the last call's values have been read)
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    S of_warp = lane < warps ? shared[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const S below = __shfl_up_sync(0xffffffffu, of_warp, d);
      if (lane >= d) of_warp += below;
    }
    if (lane < warps) shared[lane] = of_warp;
  }
  __syncthreads();
  *total = shared[warps - 1];
  return sum - value + (warp ? shared[warp - 1] : 0);
}

// ---- forking -----------------------------------------------------------------------------------
// All sequences change at once, so their rows are set aside first; the counts of holders go up for the new row and down for the old one,
// in any order.

__global__ void fork_stage_kernel(const CacheView c, const int32_t* sources, const Scratch to) {
  pdl_wait();
  pdl_launch_dependents();
  for (int s = blockIdx.x; s < c.sequences; s += gridDim.x) {
    int source = sources[s];
    if (source < -1 || source >= c.sequences) {
      if (threadIdx.x == 0) cache_fault(c, KB200_CACHE_BAD_INDEX);
      source = s;
    }
    const int held = source < 0 ? 0 : min(max(c.held[source], 0), c.max_pages);
    if (threadIdx.x == 0) {
      to.slot[s] = source;
      to.slot[c.sequences + s] = held;
      to.slot[2 * c.sequences + s] = source < 0 ? 0 : c.lengths[source];
    }
    if (source == s) continue;
    for (int k = threadIdx.x; k < held; k += blockDim.x) {
      const int page = c.table[(int64_t)source * c.max_pages + k];
      to.rows[(int64_t)s * c.max_pages + k] = page;
      if (cache_page_ok(c, page)) atomicAdd(c.refs + page, 1);
    }
    const int old = min(max(c.held[s], 0), c.max_pages);
    for (int k = threadIdx.x; k < old; k += blockDim.x) {
      const int page = c.table[(int64_t)s * c.max_pages + k];
      if (cache_page_ok(c, page)) atomicSub(c.refs + page, 1);
    }
  }
}

__global__ void fork_commit_kernel(const CacheView c, const Scratch from) {
  pdl_wait();
  pdl_launch_dependents();
  for (int s = blockIdx.x; s < c.sequences; s += gridDim.x) {
    if (from.slot[s] == s) continue;
    const int held = from.slot[c.sequences + s], old = min(max(c.held[s], 0), c.max_pages);
    __syncthreads();                     // (held[s] has been read)
    if (threadIdx.x == 0) {
      c.held[s] = held;
      c.lengths[s] = from.slot[2 * c.sequences + s];
    }
    for (int k = threadIdx.x; k < max(held, old); k += blockDim.x)
      c.table[(int64_t)s * c.max_pages + k] = k < held ? from.rows[(int64_t)s * c.max_pages + k] : -1;
  }
}

// Both in one launch of one CTA, a warp to a sequence.
__global__ void __launch_bounds__(kTableThreads) fork_small_kernel(const CacheView c, const int32_t* sources, const Scratch to) {
  __shared__ int source_of[kFewSequences], held_of[kFewSequences], length_of[kFewSequences];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  for (int s = threadIdx.x >> 5; s < c.sequences; s += kTableThreads / 32) {
    int source = sources[s];
    if (source < -1 || source >= c.sequences) {
      if (lane == 0) cache_fault(c, KB200_CACHE_BAD_INDEX);
      source = s;
    }
    const int held = source < 0 ? 0 : min(max(c.held[source], 0), c.max_pages), old = min(max(c.held[s], 0), c.max_pages);
    if (lane == 0) source_of[s] = source, held_of[s] = held, length_of[s] = source < 0 ? 0 : c.lengths[source];
    if (source == s) continue;
    for (int k = lane; k < max(held, old); k += 32) {
      const int page = k < held ? c.table[(int64_t)source * c.max_pages + k] : -1, gone = k < old ? c.table[(int64_t)s * c.max_pages + k] : -1;
      if (k < held) to.rows[(int64_t)s * c.max_pages + k] = page;
      if (page == gone) continue;
      if (cache_page_ok(c, page)) atomicAdd(c.refs + page, 1);
      if (cache_page_ok(c, gone)) atomicSub(c.refs + gone, 1);
    }
  }
  __syncthreads();
  for (int s = threadIdx.x >> 5; s < c.sequences; s += kTableThreads / 32) {
    if (source_of[s] == s) continue;
    const int held = held_of[s], old = min(max(c.held[s], 0), c.max_pages);
    for (int k = lane; k < max(held, old); k += 32) c.table[(int64_t)s * c.max_pages + k] = k < held ? to.rows[(int64_t)s * c.max_pages + k] : -1;
    __syncwarp();
    if (lane == 0) c.held[s] = held, c.lengths[s] = length_of[s];
  }
}

// ---- room for new tokens -----------------------------------------------------------------------

struct Span {
  int first, need, held;      // the pages that a sequence is going to write: first..need; it has `held`
  int rows;                   // committed tokens in the first of them
  bool bad, too_long;
};
__device__ __forceinline__ Span span_of(const CacheView& c, const int32_t* counts, int s) {
  const int count = counts[s], length = max(c.lengths[s], 0);
  const int64_t need = ((int64_t)length + max(count, 0) + (1 << c.page_log2) - 1) >> c.page_log2;
  Span r;
  r.first = length >> c.page_log2;
  r.rows = length & ((1 << c.page_log2) - 1);
  r.held = min(max(c.held[s], 0), c.max_pages);
  r.bad = count < 0;
  r.too_long = count > 0 && need > c.max_pages;
  r.need = count > 0 && !r.too_long ? (int)need : r.first;
  return r;
}

// A warp takes a sequence and its lanes the pages, so that both many sequences of a page each and a long prompt's hundreds of
// pages are a few rounds; a thread takes neighbouring pages where free ones are counted.
template <bool ONE>
__global__ void __launch_bounds__(kTableThreads) reserve_kernel(const CacheView c, const int32_t* counts, const Scratch w) {
  __shared__ int shared[32];
  __shared__ int64_t shared_wide[32];
  pdl_wait();
  pdl_launch_dependents();
  const int rank = ONE ? 0 : blockIdx.x, ranks = ONE ? 1 : gridDim.x, lane = threadIdx.x & 31;
  const int warp = rank * (kTableThreads / 32) + (threadIdx.x >> 5), warps = ranks * (kTableThreads / 32);
  int32_t* const wanted = w.slot;                          // [sequences]: new pages, then where the sequence's begin
  int32_t *const writers = w.page_a, *const lowest = w.page_b;
  const int part = (c.pages + ranks * kTableThreads - 1) / (ranks * kTableThreads);
  const int lo = min((rank * kTableThreads + (int)threadIdx.x) * part, c.pages), hi = min(lo + part, c.pages);

  // Everybody looks at all counts: nothing is done unless all are good.
  int faults = 0;
  for (int s = threadIdx.x; s < c.sequences; s += blockDim.x) {
    const Span r = span_of(c, counts, s);
    faults |= (r.bad ? KB200_CACHE_BAD_INDEX : 0) | (r.too_long ? KB200_CACHE_TOO_LONG : 0);
  }
  int free_mine = 0;
  for (int page = lo; page < hi; ++page) free_mine += c.refs[page] == 0;
  const int bad = __syncthreads_or(faults & KB200_CACHE_BAD_INDEX), too_long = __syncthreads_or(faults & KB200_CACHE_TOO_LONG);
  if (rank == 0 && threadIdx.x == 0) w.counters[kCopies] = 0;
  if (bad || too_long) {
    if (rank == 0 && threadIdx.x == 0) cache_fault(c, (bad ? KB200_CACHE_BAD_INDEX : 0) | (too_long ? KB200_CACHE_TOO_LONG : 0));
    return;
  }
  int free_here;
  const int free_below = block_scan(free_mine, shared, &free_here);
  if (threadIdx.x == 0) w.counters[kPerCta + rank] = free_here;

  // Shared pages that are going to be written: by how many, and by whom first.
  auto each_shared = [&](auto&& f) {
    bool any = false;
    for (int s = warp; s < c.sequences; s += warps) {
      const Span r = span_of(c, counts, s);
      for (int k = r.first + lane; k < min(r.need, r.held); k += 32) {
        const int page = c.table[(int64_t)s * c.max_pages + k];
        if (cache_page_ok(c, page) && c.refs[page] > 1) {
          f(page, s);
          any = true;
        }
      }
    }
    return any;
  };
  bool any = each_shared([&](int page, int) { writers[page] = 0, lowest[page] = INT_MAX; });
  if constexpr (ONE) any = __syncthreads_or(any);          // (a cluster meets in any case)
  else any = true;
  if (any) {
    if constexpr (!ONE) meet<ONE>();
    each_shared([&](int page, int s) { atomicAdd(writers + page, 1), atomicMin(lowest + page, s); });
    meet<ONE>();
  }
  // Which pages have to be new.
  for (int s = warp; s < c.sequences; s += warps) {
    const Span r = span_of(c, counts, s);
    int n = 0;
    for (int k = r.first + lane; k < r.need; k += 32) {
      bool fresh = true;
      if (k < r.held) {
        const int page = c.table[(int64_t)s * c.max_pages + k];
        if (cache_page_ok(c, page)) {
          const int refs = c.refs[page];
          fresh = refs > 1 && !(__ldcg(writers + page) == refs && __ldcg(lowest + page) == s);
        }
      }
      w.rows[(int64_t)s * c.max_pages + k] = fresh;
      n += fresh;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) wanted[s] = n;
  }
  meet<ONE>();
  // The first CTA says where every sequence's new pages begin.  (A table of 2^31 entries and more may ask for as many: summed in 64 bits.  Where a sum does not fit in
  // 32 it is beyond the free pages, and nobody uses it.)
  if (rank == 0) {
    int64_t base = 0;
    for (int s0 = 0; s0 < c.sequences; s0 += blockDim.x) {
      const int s = s0 + threadIdx.x;
      const int64_t n = s < c.sequences ? __ldcg(wanted + s) : 0;
      int64_t total;
      const int64_t before = block_scan(n, shared_wide, &total);
      if (s < c.sequences) wanted[s] = (int)min(base + before, (int64_t)INT_MAX);
      base += total;
    }
    if (threadIdx.x == 0) w.counters[kWanted] = (int)min(base, (int64_t)INT_MAX);
  }
  meet<ONE>();
  const int all = __ldcg(w.counters + kWanted);
  int free_before = free_below, free_all = 0;
  for (int r = 0; r < ranks; ++r) {
    const int n = __ldcg(w.counters + kPerCta + r);
    free_before += r < rank ? n : 0;
    free_all += n;
  }
  if (all > free_all) {
    if (rank == 0 && threadIdx.x == 0) cache_fault(c, KB200_CACHE_NO_PAGES);
    return;
  }
  // The free pages by rank (over the list of writers, which has been read).
  int32_t* const free_pages = w.page_a;
  for (int page = lo; page < hi && free_before < all; ++page)
    if (c.refs[page] == 0) free_pages[free_before++] = page;
  meet<ONE>();
  for (int s = warp; s < c.sequences; s += warps) {
    const Span r = span_of(c, counts, s);
    int next = __ldcg(wanted + s);
    for (int k0 = r.first; k0 < r.need; k0 += 32) {
      const int k = k0 + lane;
      const bool fresh = k < r.need && w.rows[(int64_t)s * c.max_pages + k] != 0;
      const unsigned all_fresh = __ballot_sync(0xffffffffu, fresh);
      if (fresh) {
        int32_t* const entry = c.table + (int64_t)s * c.max_pages + k;
        const int page = __ldcg(free_pages + next + __popc(all_fresh & ((1u << lane) - 1)));
        const int old = k < r.held ? *entry : -1;
        *entry = page;
        c.refs[page] = 1;
        if (cache_page_ok(c, old)) {
          atomicSub(c.refs + old, 1);
          if (k == r.first && r.rows > 0) w.copies[atomicAdd(w.counters + kCopies, 1)] = make_int4(old, page, r.rows, 0);
        } else if (k == r.first && r.rows > 0) {
          cache_fault(c, KB200_CACHE_BAD_INDEX);             // committed tokens whose page is gone (truncated into what was released)
        }
      }
      next += __popc(all_fresh);
    }
    __syncwarp();
    if (lane == 0 && r.need > r.held) c.held[s] = r.need;
  }
}

// The listed copies in all layers: a warp moves a page's rows of one layer, head and of K or V, which lie together, 4 KB in flight.
constexpr int kCopyThreads = 256;

__device__ __forceinline__ void copy_pages(const CacheView& c, const Scratch& w, int block, int blocks) {
  const int n = w.counters[kCopies];
  const int64_t planes = (int64_t)c.layers * 2 * c.kv_heads, units = n * planes;
  const int lane = threadIdx.x & 31, warps = blocks * (kCopyThreads / 32);
  const int64_t page_chunks = (int64_t)c.row_chunks << c.page_log2, half = (int64_t)c.pages * c.kv_heads;     // K or V of a layer, in (page, head)
  uint4* const pool = static_cast<uint4*>(c.pool);
  for (int64_t u = block * (kCopyThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    const int4 job = w.copies[u / planes];
    const int64_t plane = u % planes, of = plane / c.kv_heads * half + plane % c.kv_heads;
    const uint4* const from = pool + (of + (int64_t)job.x * c.kv_heads) * page_chunks;
    uint4* const to = pool + (of + (int64_t)job.y * c.kv_heads) * page_chunks;
    const int chunks = job.z * c.row_chunks;
    for (int i = lane; i < chunks; i += 32 * 8) {
      uint4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + 32 * j < chunks) v[j] = __ldcs(from + i + 32 * j);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + 32 * j < chunks) to[i + 32 * j] = v[j];
    }
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CacheView c, const Scratch w) {
  pdl_wait();
  pdl_launch_dependents();
  copy_pages(c, w, blockIdx.x, gridDim.x);
}

// ---- freeing -----------------------------------------------------------------------------------

constexpr int kSlotThreads = 128;

__global__ void __launch_bounds__(kSlotThreads) truncate_kernel(const CacheView c, const int32_t* lengths) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x * (kSlotThreads / 32) + (threadIdx.x >> 5);
  if (s >= c.sequences || lengths[s] < 0) return;
  cut(c, s, min(max(c.lengths[s], 0), lengths[s]));
}

// ---- accepted tokens ---------------------------------------------------------------------------

// Can a sequence's entries be followed?  By a warp, while nobody changes how many hold a page: what moves is committed by the answer that the moving launch got, since
// in the committing one other sequences give their pages back.
__device__ __forceinline__ int accept_faults(const CacheView& c, const int32_t* counts, const int32_t* kept, int width, int s) {
  const int lane = threadIdx.x & 31, n = counts[s];
  if (n < 0 || (kept != nullptr && n > width)) return KB200_CACHE_BAD_INDEX;
  if (n == 0) return 0;
  const int length = max(c.lengths[s], 0), held = min(max(c.held[s], 0), c.max_pages);
  const int64_t room = ((int64_t)held << c.page_log2) - length;           // tokens behind the committed ones that have pages
  if (kept == nullptr) return n <= room ? 0 : KB200_CACHE_NO_ROOM;
  const int32_t* const mine = kept + (int64_t)s * width;
  int faults = 0;
  bool moves = false;
  for (unsigned i = lane; i < (unsigned)n; i += 32) {
    const int at = mine[i], before = i > 0 ? mine[i - 1] : -1;
    faults |= at <= before ? KB200_CACHE_BAD_INDEX : at >= room ? KB200_CACHE_NO_ROOM : 0;
    moves = moves || at != (int)i;
  }
  if (__any_sync(0xffffffffu, moves))                                      // what is written has to be the sequence's own
    for (int k = (length >> c.page_log2) + lane; k < held && k <= (int)(((int64_t)length + n - 1) >> c.page_log2); k += 32) {
      const int page = c.table[(int64_t)s * c.max_pages + k];
      faults |= !cache_page_ok(c, page) ? KB200_CACHE_NO_ROOM : c.refs[page] > 1 ? KB200_CACHE_SHARED : 0;
    }
  return (int)__reduce_or_sync(0xffffffffu, (unsigned)faults);
}

// A warp moves one sequence's tokens in one layer, head and of K or V.  Row i comes from row kept[i] >= i: batches ascend, and a batch is
// read before any of it is written, so nothing is overwritten that is still to be read.
__global__ void __launch_bounds__(kCopyThreads) accept_move_kernel(const CacheView c, const int32_t* counts, const int32_t* kept, int width, int32_t* answers) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t planes = (int64_t)c.layers * 2 * c.kv_heads, units = planes * c.sequences;
  const int lane = threadIdx.x & 31, in_page = (1 << c.page_log2) - 1;
  uint4* const pool = static_cast<uint4*>(c.pool);
  for (int64_t u = (int64_t)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); u < units; u += (int64_t)gridDim.x * (kCopyThreads / 32)) {
    const int s = (int)(u / planes);
    const int n = counts[s], faults = accept_faults(c, counts, kept, width, s);
    if (lane == 0 && u % planes == 0) answers[s] = faults;
    if (n <= 0 || faults != 0) continue;
    const int64_t plane = u % planes, of = plane / c.kv_heads * c.pages;
    const int head = (int)(plane % c.kv_heads), length = max(c.lengths[s], 0);
    const int32_t *const mine = kept + (int64_t)s * width, *const row = c.table + (int64_t)s * c.max_pages;
    auto place = [&](int token, int chunk) -> uint4* {
      const int at = length + token, page = row[at >> c.page_log2];
      if (!cache_page_ok(c, page)) return nullptr;
      return pool + ((((of + page) * c.kv_heads + head) << c.page_log2) + (at & in_page)) * c.row_chunks + chunk;
    };
    // (by 2^20 tokens, whose chunks are a number of 32 bits; those of 2^25 are not)
    for (int first = 0; first < n; first += 1 << 20) {
      const int chunks = min(n - first, 1 << 20) * c.row_chunks;
      for (int i0 = 0; i0 < chunks; i0 += 32 * 4) {
        uint4 v[4];
        uint4* to[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + 32 * j + lane, chunk = i % c.row_chunks, token = first + i / c.row_chunks;
          to[j] = nullptr;
          if (i < chunks && mine[token] != token) {
            const uint4* const from = place(mine[token], chunk);
            if (from != nullptr) {
              v[j] = *from;
              to[j] = place(token, chunk);
            }
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (to[j] != nullptr) *to[j] = v[j];
        __syncwarp();
      }
    }
  }
}

// answers: of the moving launch; null: nothing moves, and a sequence's own numbers say all.
__global__ void __launch_bounds__(kSlotThreads) accept_commit_kernel(const CacheView c, const int32_t* counts, const int32_t* kept, int width, const int32_t* answers) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x * (kSlotThreads / 32) + (threadIdx.x >> 5);
  if (s >= c.sequences) return;
  const int faults = answers != nullptr ? answers[s] : accept_faults(c, counts, kept, width, s);
  if (faults != 0) {
    if ((threadIdx.x & 31) == 0) cache_fault(c, faults);
    return;
  }
  cut(c, s, max(c.lengths[s], 0) + counts[s]);
}

// ---- compacting --------------------------------------------------------------------------------

template <bool ONE>
__global__ void __launch_bounds__(kTableThreads) compact_kernel(const CacheView c, const Scratch w) {
  __shared__ int shared[32];
  pdl_wait();
  pdl_launch_dependents();
  const int rank = ONE ? 0 : blockIdx.x, ranks = ONE ? 1 : gridDim.x;
  const int part = (c.pages + ranks * kTableThreads - 1) / (ranks * kTableThreads);
  const int lo = min((rank * kTableThreads + (int)threadIdx.x) * part, c.pages), hi = min(lo + part, c.pages);
  int n = 0, used;
  for (int page = lo; page < hi; ++page) n += c.refs[page] != 0;
  block_scan(n, shared, &used);
  if constexpr (!ONE) {
    if (threadIdx.x == 0) w.counters[kPerCta + rank] = used;
    meet<ONE>();
    used = 0;
    for (int r = 0; r < ranks; ++r) used += __ldcg(w.counters + kPerCta + r);
  }
  // Pages in use behind the first `used`, and free ones among those: as many of one as of the other.
  int leave = 0, enter = 0, moves, enter_here;
  for (int page = lo; page < hi; ++page) {
    const bool in_use = c.refs[page] != 0;
    leave += in_use && page >= used;
    enter += !in_use && page < used;
  }
  int leave_at = block_scan(leave, shared, &moves), enter_at = block_scan(enter, shared, &enter_here);
  if constexpr (!ONE) {
    if (threadIdx.x == 0) w.counters[kPerCta + kCluster + rank] = moves, w.counters[kPerCta + 2 * kCluster + rank] = enter_here;
    meet<ONE>();
    moves = 0;
    for (int r = 0; r < ranks; ++r) {
      const int l = __ldcg(w.counters + kPerCta + kCluster + r), e = __ldcg(w.counters + kPerCta + 2 * kCluster + r);
      leave_at += r < rank ? l : 0;
      enter_at += r < rank ? e : 0;
      moves += l;
    }
  }
  int32_t *const leaving = w.page_a, *const entering = w.page_b;
  for (int page = lo; page < hi; ++page) {
    const bool in_use = c.refs[page] != 0;
    if (in_use && page >= used) leaving[leave_at++] = page;
    if (!in_use && page < used) entering[enter_at++] = page;
  }
  meet<ONE>();
  for (int i = rank * kTableThreads + threadIdx.x; i < moves; i += ranks * kTableThreads) {
    const int from = __ldcg(leaving + i), to = __ldcg(entering + i);
    w.copies[i] = make_int4(from, to, 1 << c.page_log2, 0);
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (rank == 0 && threadIdx.x == 0) w.counters[kCopies] = moves, w.counters[kUsed] = used;
}

// The tokens, and the tables' entries: where a page went is its rank among those that left.
__global__ void __launch_bounds__(kCopyThreads) compact_move_kernel(const CacheView c, const Scratch w) {
  pdl_wait();
  pdl_launch_dependents();
  const int moves = w.counters[kCopies], used = w.counters[kUsed];
  for (int s = blockIdx.x; s < c.sequences && moves > 0; s += gridDim.x) {
    const int held = min(max(c.held[s], 0), c.max_pages);
    for (int k = threadIdx.x; k < held; k += blockDim.x) {
      int32_t* const entry = c.table + (int64_t)s * c.max_pages + k;
      const int page = *entry;
      if (page < used || page >= c.pages) continue;
      int at = 0;                        // the last one that is not behind it
      for (int step = 1 << (31 - __clz(moves)); step > 0; step >>= 1)
        if (at + step < moves && w.page_a[at + step] <= page) at += step;
      if (w.page_a[at] == page) *entry = w.page_b[at];
    }
  }
  copy_pages(c, w, blockIdx.x, gridDim.x);
}

// ---- new tokens --------------------------------------------------------------------------------

struct AppendParams {
  const void *k, *v;
  int64_t k_stride[3], v_stride[3];
  const int32_t *counts, *slots;
  int rows, tokens, layer;
};

template <typename T>
__device__ __forceinline__ uint4 load_rounded(const float* from);
template <>
__device__ __forceinline__ uint4 load_rounded<__nv_bfloat16>(const float* from) {
  const float4 a = *reinterpret_cast<const float4*>(from), b = *reinterpret_cast<const float4*>(from + 4);
  const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w), __floats2bfloat162_rn(b.x, b.y),
                               __floats2bfloat162_rn(b.z, b.w)};
  return *reinterpret_cast<const uint4*>(h);
}
template <>
__device__ __forceinline__ uint4 load_rounded<__half>(const float* from) {
  const float4 a = *reinterpret_cast<const float4*>(from), b = *reinterpret_cast<const float4*>(from + 4);
  const __half2 h[4] = {__floats2half2_rn(a.x, a.y), __floats2half2_rn(a.z, a.w), __floats2half2_rn(b.x, b.y), __floats2half2_rn(b.z, b.w)};
  return *reinterpret_cast<const uint4*>(h);
}

// A CTA takes part of a batch row's tokens; a thread 16 bytes of the cache at a time, of K and of V.  T: the cache's type where the
// input is float32 and is rounded on the way (to nearest, ties to even, as a conversion by torch), float: copied as it is.
template <typename T>
__global__ void __launch_bounds__(kCopyThreads) append_kernel(const CacheView c, const AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr bool kRound = sizeof(T) == 2;
  uint4* const pool = static_cast<uint4*>(c.pool);
  const int64_t half = (int64_t)c.pages * c.kv_heads << c.page_log2;      // K's rows of a layer
  for (int b = blockIdx.y; b < p.rows; b += gridDim.y) {
    const int slot = p.slots != nullptr ? p.slots[b] : b;
    int count = p.counts != nullptr ? p.counts[b] : p.tokens;
    bool bad = slot < 0 || slot >= c.sequences;
    if (p.slots != nullptr) {              // a sequence that an earlier row names is that row's
      bool again = false;
      for (int i = threadIdx.x; i < b; i += blockDim.x) again = again || p.slots[i] == slot;
      bad = __syncthreads_or(again) || bad;
    }
    if (bad || count < 0 || count > p.tokens) {
      if (threadIdx.x == 0 && blockIdx.x == 0) cache_fault(c, KB200_CACHE_BAD_INDEX);
      count = bad ? 0 : min(max(count, 0), p.tokens);
    }
    if (count == 0) continue;
    const int length = max(c.lengths[slot], 0), held = min(max(c.held[slot], 0), c.max_pages);
    const int64_t chunks = (int64_t)count * c.kv_heads * c.row_chunks;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * blockDim.x) {
      const int chunk = (int)(i % c.row_chunks);
      const int64_t row = i / c.row_chunks;
      const int head = (int)(row % c.kv_heads), token = (int)(row / c.kv_heads);
      const int64_t at = (int64_t)length + token;
      const int page = (at >> c.page_log2) < held ? c.table[(int64_t)slot * c.max_pages + (at >> c.page_log2)] : -1;
      const int fault = !cache_page_ok(c, page) ? KB200_CACHE_NO_ROOM : c.refs[page] > 1 ? KB200_CACHE_SHARED : 0;
      if (fault != 0) {
        cache_fault(c, fault);
        continue;
      }
      const int64_t to = (cache_row(c, p.layer, 0, page, head) + (at & ((1 << c.page_log2) - 1))) * c.row_chunks + chunk;
      const int64_t from_k = b * p.k_stride[0] + token * p.k_stride[1] + head * p.k_stride[2];
      const int64_t from_v = b * p.v_stride[0] + token * p.v_stride[1] + head * p.v_stride[2];
      uint4 k, v;
      if constexpr (kRound) {
        k = load_rounded<T>(static_cast<const float*>(p.k) + from_k + chunk * 8);
        v = load_rounded<T>(static_cast<const float*>(p.v) + from_v + chunk * 8);
      } else {                             // (strides in 16-byte chunks here)
        k = static_cast<const uint4*>(p.k)[from_k + chunk];
        v = static_cast<const uint4*>(p.v)[from_v + chunk];
      }
      pool[to] = k;
      pool[to + half * c.row_chunks] = v;
    }
  }
}

__global__ void told_kernel(int* status, int bits) { atomicAnd(status, ~bits); }

// ---- host --------------------------------------------------------------------------------------

Scratch scratch_of(const Cache& c) { return Scratch{c.stage_rows, c.stage_slot, c.page_a, c.page_b, c.copies, c.counters}; }

// One CTA or one cluster.
bool few(const Cache& c) { return c.view.pages <= kFewPages && c.view.sequences <= kFewSequences; }
template <typename... KArgs, typename... Args>
cudaError_t launch_tables(const Cache& c, void (*one)(KArgs...), void (*cluster)(KArgs...), cudaStream_t s, Args&&... args) {
  if (few(c)) return launch_kernel(true, one, dim3(1), dim3(kTableThreads), 0, s, static_cast<KArgs>(args)...);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster);
  cfg.blockDim = dim3(kTableThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, cluster, static_cast<KArgs>(args)...);
}

int copy_grid(const Cache& c) { return c.sm_count * 8; }

bool rows_ok(const Cache& c, const kb200_rows* r, int heads) {
  if (r == nullptr || r->data == nullptr || !tc::aligned16(r->data) || r->heads != heads || (r->dtype != c.dtype && r->dtype != KB200_DTYPE_FP32)) return false;
  const int per16 = r->dtype == KB200_DTYPE_FP32 ? 4 : 8;
  for (const int64_t s : r->stride)
    if (s % per16 != 0) return false;
  return true;
}

}  // namespace
}  // namespace kb200

using namespace kb200;

namespace {
int page_log2_of(int tokens) {
  int log2 = 0;
  while ((1 << log2) < tokens && log2 < 9) ++log2;
  return log2;
}
}  // namespace

KB200_EXPORT int kb200_cache_check(const kb200_cache_desc* d) {
  if (d == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_create: no description");
  if (d->dtype < KB200_DTYPE_FP32 || d->dtype > KB200_DTYPE_FP16) return fail(KB200_ERR_ARGUMENT, "kb200_cache_create: unknown type %d", d->dtype);
  if (d->layers < 1 || d->sequences < 1 || d->max_pages < 1 || d->pages < 1 || d->kv_heads < 1)
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_create: layers, sequences, max_pages, pages and kv_heads must be positive");
  if (d->page_tokens < 8 || d->page_tokens > 256 || (1 << page_log2_of(d->page_tokens)) != d->page_tokens)
    return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: pages of %d tokens (8, 16, 32, 64, 128 or 256)", d->page_tokens);
  if (d->head_dim < 16 || d->head_dim > 256 || d->head_dim % 16 != 0)
    return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: heads of %d (a multiple of 16 up to 256)", d->head_dim);
  if ((int64_t)d->max_pages * d->page_tokens >= (1 << 30)) return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: sequences of 2^30 tokens or more");
  if (d->layers > (1 << 16) || d->kv_heads > (1 << 16) || d->sequences > (1 << 20) || d->pages > (1 << 29))
    return fail(KB200_ERR_UNSUPPORTED, "kb200_cache_create: more than 2^16 layers or heads, 2^20 sequences or 2^29 pages");
  const double bytes = 2.0 * d->layers * d->pages * (double)d->kv_heads * d->page_tokens * d->head_dim * (d->dtype == KB200_DTYPE_FP32 ? 4 : 2);
  if (d->pool == nullptr || d->table == nullptr || d->held == nullptr || d->lengths == nullptr || d->refs == nullptr)
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_create: a buffer is null");
  if (!tc::aligned16(d->pool)) return fail(KB200_ERR_ARGUMENT, "kb200_cache_create: the pool is not on 16 bytes");
  if (bytes > (double)d->pool_bytes)
    return fail(KB200_ERR_BOUNDS, "kb200_cache_create: the pool takes %.0f bytes, the buffer has %llu", bytes, (unsigned long long)d->pool_bytes);
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_create(const kb200_cache_desc* d, int device, kb200_cache** out) {
  if (out == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_create: out is null");
  *out = nullptr;
  const int checked = kb200_cache_check(d);
  if (checked != KB200_OK) return checked;
  const DeviceGuard guard(device);
  if (guard.error != cudaSuccess) return cuda_fail(guard.error, "cudaSetDevice");
  Cache* c = new (std::nothrow) Cache;
  if (c == nullptr) return fail(KB200_ERR_CUDA, "kb200_cache_create: out of host memory");
  c->device = device;
  c->dtype = d->dtype;
  c->element = d->dtype == KB200_DTYPE_FP32 ? 4 : 2;
  cudaDeviceGetAttribute(&c->sm_count, cudaDevAttrMultiProcessorCount, device);
  const int64_t S = d->sequences, copies = std::max<int64_t>(S, d->pages);
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t rows = up(S * d->max_pages * 4), slot = up(3 * S * 4), page = up((int64_t)d->pages * 4), list = up(copies * 16), words = up(kCounters * 4 + 4);
  const cudaError_t e = cudaMalloc(&c->scratch, (size_t)(rows + slot + 2 * page + list + words));
  if (e != cudaSuccess) {
    delete c;
    cudaGetLastError();
    return cuda_fail(e, "kb200_cache_create: cudaMalloc");
  }
  char* at = static_cast<char*>(c->scratch);
  c->copies = reinterpret_cast<int4*>(at);
  c->stage_rows = reinterpret_cast<int32_t*>(at += list);
  c->stage_slot = reinterpret_cast<int32_t*>(at += rows);
  c->page_a = reinterpret_cast<int32_t*>(at += slot);
  c->page_b = reinterpret_cast<int32_t*>(at += page);
  c->counters = reinterpret_cast<int*>(at += page);
  int* const status = c->counters + kCounters;
  cudaError_t z = cudaMemset(c->counters, 0, (size_t)words);
  if (z == cudaSuccess) z = cudaDeviceSynchronize();
  if (z != cudaSuccess) {
    cudaFree(c->scratch);
    delete c;
    return cuda_fail(z, "kb200_cache_create: cudaMemset");
  }
  c->view = CacheView{d->pool, d->table, d->held, d->lengths, d->refs, status, d->layers, d->sequences, d->max_pages, d->pages, d->kv_heads,
                      page_log2_of(d->page_tokens), d->head_dim, d->head_dim * c->element / 16};
  int prepared = cache_attention_prepare(*c);
  if (prepared == KB200_OK) prepared = cache_weigh_prepare(*c);
  if (prepared == KB200_OK) prepared = cache_verify_prepare(*c);
  if (prepared != KB200_OK) {
    cudaFree(c->scratch);
    delete c;
    return prepared;
  }
  *out = reinterpret_cast<kb200_cache*>(c);
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_fork(kb200_cache* handle, const int32_t* sources, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_fork");
  if (sources == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_fork: sources is null");
  if (few(c)) {
    KB200_CUDA(launch_kernel(true, fork_small_kernel, dim3(1), dim3(kTableThreads), 0, s, c.view, sources, scratch_of(c)));
    return KB200_OK;
  }
  const dim3 grid(std::min(c.view.sequences, 4 * c.sm_count));
  KB200_CUDA(launch_kernel(true, fork_stage_kernel, grid, dim3(kSlotThreads), 0, s, c.view, sources, scratch_of(c)));
  KB200_CUDA(launch_kernel(true, fork_commit_kernel, grid, dim3(kSlotThreads), 0, s, c.view, scratch_of(c)));
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_reserve(kb200_cache* handle, const int32_t* counts, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_reserve");
  if (counts == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_reserve: counts is null");
  KB200_CUDA(launch_tables(c, reserve_kernel<true>, reserve_kernel<false>, s, c.view, counts, scratch_of(c)));
  KB200_CUDA(launch_kernel(true, copy_pages_kernel, dim3(copy_grid(c)), dim3(kCopyThreads), 0, s, c.view, scratch_of(c)));
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_truncate(kb200_cache* handle, const int32_t* lengths, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_truncate");
  if (lengths == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_truncate: lengths is null");
  const int per = kSlotThreads / 32;
  KB200_CUDA(launch_kernel(true, truncate_kernel, dim3((c.view.sequences + per - 1) / per), dim3(kSlotThreads), 0, s, c.view, lengths));
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_compact(kb200_cache* handle, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_compact");
  KB200_CUDA(launch_tables(c, compact_kernel<true>, compact_kernel<false>, s, c.view, scratch_of(c)));
  KB200_CUDA(launch_kernel(true, compact_move_kernel, dim3(copy_grid(c)), dim3(kCopyThreads), 0, s, c.view, scratch_of(c)));
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_append(kb200_cache* handle, int layer, const kb200_rows* k, const kb200_rows* v, int rows, int tokens,
                                    const int32_t* counts, const int32_t* slots, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_append");
  if (layer < 0 || layer >= c.view.layers) return fail(KB200_ERR_ARGUMENT, "kb200_cache_append: layer %d of %d", layer, c.view.layers);
  if (rows < 0 || rows > (1 << 30) || tokens < 0 || (slots == nullptr && rows > c.view.sequences))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_append: %d rows of %d tokens for %d sequences", rows, tokens, c.view.sequences);
  if (rows == 0 || tokens == 0) return KB200_OK;
  if (!rows_ok(c, k, c.view.kv_heads) || !rows_ok(c, v, c.view.kv_heads) || k->dtype != v->dtype)
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_append: k and v must be [rows, tokens, %d, %d], both of the cache's type or float32, on 16 bytes",
                c.view.kv_heads, c.view.head_dim);
  AppendParams p{k->data, v->data, {}, {}, counts, slots, rows, tokens, layer};
  const bool rounded = k->dtype != c.dtype;
  const int unit = rounded ? 1 : 16 / c.element;
  for (int i = 0; i < 3; ++i) p.k_stride[i] = k->stride[i] / unit, p.v_stride[i] = v->stride[i] / unit;
  const int64_t chunks = (int64_t)tokens * c.view.kv_heads * c.view.row_chunks;
  const dim3 grid((unsigned)std::min<int64_t>((chunks + kCopyThreads - 1) / kCopyThreads, std::max(1, 16 * c.sm_count / rows)), (unsigned)std::min(rows, 65535));
  const auto kernel = !rounded ? append_kernel<float> : c.dtype == KB200_DTYPE_BF16 ? append_kernel<__nv_bfloat16> : append_kernel<__half>;
  KB200_CUDA(launch_kernel(true, kernel, grid, dim3(kCopyThreads), 0, s, c.view, p));
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_accept(kb200_cache* handle, const int32_t* counts, const int32_t* kept, int width, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_accept");
  if (counts == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_accept: counts is null");
  if (kept != nullptr && width < 0) return fail(KB200_ERR_ARGUMENT, "kb200_cache_accept: kept is %d wide", width);
  int32_t* const answers = kept != nullptr && width > 0 ? c.stage_slot : nullptr;
  if (answers != nullptr) {
    const int64_t units = c.planes() * c.view.sequences;
    const int grid = (int)std::min<int64_t>((units + kCopyThreads / 32 - 1) / (kCopyThreads / 32), copy_grid(c));
    KB200_CUDA(launch_kernel(true, accept_move_kernel, dim3(grid), dim3(kCopyThreads), 0, s, c.view, counts, kept, width, answers));
  }
  const int per = kSlotThreads / 32;
  KB200_CUDA(launch_kernel(true, accept_commit_kernel, dim3((c.view.sequences + per - 1) / per), dim3(kSlotThreads), 0, s, c.view, counts, kept, width, answers));
  return KB200_OK;
}

KB200_EXPORT int kb200_cache_status(kb200_cache* handle) {
  if (handle == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_status: cache is null");
  Cache& c = *cache_of(handle);
  const DeviceGuard guard(c.device);
  if (guard.error != cudaSuccess) return cuda_fail(guard.error, "kb200_cache_status");
  int word = 0;
  KB200_CUDA(cudaMemcpy(&word, c.view.status, sizeof(int), cudaMemcpyDeviceToHost));
  if (word == 0) return KB200_OK;
  // What has been read is cleared and nothing else (calls may be under way), and that is done before this returns: no stream of the caller's waits for this one.
  told_kernel<<<1, 1, 0, cudaStreamLegacy>>>(c.view.status, word);
  KB200_CUDA(cudaGetLastError());
  KB200_CUDA(cudaStreamSynchronize(cudaStreamLegacy));
  if (word & kCacheWaitFault) return fail(KB200_ERR_DEVICE_WAIT, "a bounded device-side wait of kb200_cache_attend ran out");
  return fail(word & KB200_CACHE_NO_PAGES ? KB200_ERR_PAGES : KB200_ERR_BOUNDS, "cache:%s%s%s%s%s%s",
              word & KB200_CACHE_NO_PAGES ? " fewer free pages than were to be reserved;" : "",
              word & KB200_CACHE_TOO_LONG ? " a sequence would need more than max_pages;" : "",
              word & KB200_CACHE_BAD_INDEX ? " an index or a count out of range;" : "",
              word & KB200_CACHE_NO_ROOM ? " tokens without a page;" : "",
              word & KB200_CACHE_SHARED ? " a write into a shared page;" : "", word & KB200_CACHE_BAD_VALUE ? " logits that are no distribution;" : "");
}

KB200_EXPORT void kb200_cache_destroy(kb200_cache* handle) {
  if (handle == nullptr) return;
  Cache* c = cache_of(handle);
  const DeviceGuard guard(c->device);
  cudaFree(c->scratch);
  delete c;
}
