// Tokens and pages that a sequence gives up before its end: pages that a sliding window has left (kb200_cache_release), and all but the heaviest
// tokens (kb200_cache_evict).  Rules: include/kb200.h.
//
// What bounds them: the release the latency of one pass over the tables, the eviction the bytes of the tokens that move, twice, in all layers.  Which tokens
// stay is chosen by a CTA per sequence, and the tokens move in a launch over the whole GPU.
#include <limits.h>

#include <algorithm>

#include "cache.h"
#include "tc_common.cuh"

#define KB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace kb200 {
namespace {

// ---- pages behind a window ---------------------------------------------------------------------

constexpr int kReleaseThreads = 256;

// A thread looks at an entry.  No token to come sees the tokens in front of length - window + 1, but for the first `sinks`; a page goes when all of its tokens are such.
__global__ void __launch_bounds__(kReleaseThreads) release_kernel(const CacheView c, int window, int sinks) {
  pdl_wait();
  pdl_launch_dependents();
  const int first = (int)(((int64_t)sinks + (1 << c.page_log2) - 1) >> c.page_log2);
  for (int s = blockIdx.y; s < c.sequences; s += gridDim.y) {
    const int hidden = max(c.lengths[s], 0) - window + 1;
    const int end = min(min(max(c.held[s], 0), c.max_pages), max(hidden, 0) >> c.page_log2);
    for (int k = first + blockIdx.x * kReleaseThreads + threadIdx.x; k < end; k += gridDim.x * kReleaseThreads) {
      int32_t* const entry = c.table + (int64_t)s * c.max_pages + k;
      const int page = *entry;
      if (cache_page_ok(c, page)) atomicSub(c.refs + page, 1);
      *entry = -1;
    }
  }
}

// ---- which tokens stay -------------------------------------------------------------------------

constexpr int kChooseThreads = 1024, kChooseWarps = kChooseThreads / 32;
constexpr int kBins = 2048;

struct EvictParams {
  const float* weights;
  float* out;
  int64_t weights_stride, out_stride;
  const int32_t* keep;
  int64_t* from;           // [sequences][width]: where the kept tokens are, a page's number times its tokens plus the token's in it
  float* staged;           // [sequences][width]: their weights
  int2* answers;           // [sequences]: how many tokens stay (-1: all, nothing moves), the first that moves
  int recent, sinks, width;
};

// Weights as integers in the same order: NaN above all, the two zeros alike.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of a warp's lanes up to each.
__device__ __forceinline__ int warp_sums(int x) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int below = __shfl_up_sync(0xffffffffu, x, d);
    if ((threadIdx.x & 31) >= d) x += below;
  }
  return x;
}

// A CTA takes a sequence.  The least rank that stays is found digit by digit (11, 11 and 10 bits from the top), by counting the candidates of each digit; of the tokens
// at that rank the first ones stay.  Then every kept token gets its place, 8192 tokens at a time: by ballots, how many stay of each 32, and sums of those.  The first 8192 weights are
// read once, eight to a thread (read again for every digit, with sums over the warps one by one, a sequence of 1000 took 9.2 us and one of 4096 14.7).
constexpr int kHeld = 8, kGroup = kHeld * kChooseThreads;

__global__ void __launch_bounds__(kChooseThreads, 1) evict_choose_kernel(const CacheView c, const EvictParams p) {
  __shared__ int bins[kBins];
  __shared__ int sums[kChooseWarps];
  __shared__ int2 counts[kHeld * kChooseWarps];
  __shared__ int2 group_counts;
  __shared__ int digit, above, in_digit, first_moved, faults;
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_page = (1 << c.page_log2) - 1;
  const float* const weights = p.weights + s * p.weights_stride;
  float* const out = p.out + s * p.out_stride;
  const int32_t* const row = c.table + (int64_t)s * c.max_pages;
  float w[kHeld];                                             // (asked for before the sequence's length is known)
#pragma unroll
  for (int k = 0; k < kHeld; ++k) w[k] = k * kChooseThreads + (int)threadIdx.x < p.width ? weights[k * kChooseThreads + threadIdx.x] : 0.0f;
  const int held = min(max(c.held[s], 0), c.max_pages), want = p.keep[s];
  int length = max(c.lengths[s], 0);
  const bool has_pages = (int64_t)length <= (int64_t)held << c.page_log2;
  if (!has_pages) length = held << c.page_log2;
  if (threadIdx.x == 0) first_moved = INT_MAX, faults = has_pages ? 0 : KB200_CACHE_NO_ROOM;
  if (has_pages && want >= 0 && want < length) {
    // What is written has to be the sequence's own (as far as anything moves): the first pages are looked at meanwhile.
    auto page_faults = [&](int k) {
      const int page = row[k];
      return !cache_page_ok(c, page) ? KB200_CACHE_NO_ROOM : c.refs[page] > 1 ? KB200_CACHE_SHARED : 0;
    };
    const int last_page = (want - 1) >> c.page_log2, my_page_faults = (int)threadIdx.x <= last_page ? page_faults(threadIdx.x) : 0;
    const int first = min(p.sinks, want), last = min(p.recent, want - first);
    const int lo = first, hi = length - last;                 // the candidates, of which `need` stay
    int need = want - first - last;
    uint32_t prefix = 0u;
    int shift = 32;
    bool all = need == 0;                                     // every candidate of this prefix and above stays (need 0: none)
    while (shift > 0 && !all) {
      const int bits = shift > 10 ? 11 : 10;
      bins[threadIdx.x] = bins[threadIdx.x + kChooseThreads] = 0;
      __syncthreads();
      auto count = [&](int j, float x) {
        const uint32_t r = rank_of(x);
        if (j >= lo && j < hi && (shift == 32 || r >> shift == prefix)) atomicAdd(&bins[r >> (shift - bits) & ((1u << bits) - 1)], 1);
      };
#pragma unroll
      for (int k = 0; k < kHeld; ++k) count(k * kChooseThreads + threadIdx.x, w[k]);
      for (int j = kGroup + threadIdx.x; j < hi; j += kChooseThreads) count(j, weights[j]);
      __syncthreads();
      // from the highest digit down: thread t has digits kBins - 1 - 2t and the one below
      const int d = kBins - 1 - 2 * threadIdx.x, a = bins[d], b = bins[d - 1], upto = warp_sums(a + b);
      if (lane == 31) sums[warp] = upto;
      __syncthreads();
      const int of_warps = warp_sums(sums[lane]), before = __shfl_sync(0xffffffffu, of_warps - sums[lane], warp) + upto - a - b;
      if (before < need && before + a >= need) digit = d, above = before, in_digit = a;
      else if (before + a < need && before + a + b >= need) digit = d - 1, above = before + a, in_digit = b;
      __syncthreads();
      need -= above;
      prefix = prefix << bits | (uint32_t)digit;
      shift -= bits;
      all = in_digit == need;
    }
    const uint32_t least = need == 0 ? 0xffffffffu : prefix << shift;
    const int ties = need == 0 ? 0 : all ? INT_MAX : need;
    int64_t* const kept = p.from + (int64_t)s * p.width;
    float* const staged = p.staged + (int64_t)s * p.width;
    const unsigned below = (1u << lane) - 1;
    const bool in_one = length <= kGroup;                     // the kept weights stay where they are until it is known that the tokens may move
    int places[kHeld], moved = INT_MAX, fault = 0;
    int2 base = make_int2(0, 0);                              // kept whatever the others are; at the least rank
    for (int j0 = 0; j0 < length; j0 += kGroup) {
      unsigned sure[kHeld], tied[kHeld];
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int j = j0 + k * kChooseThreads + threadIdx.x;
        if (j0 > 0) w[k] = j < length ? weights[j] : 0.0f;
        const uint32_t r = rank_of(w[k]);
        const bool in = j >= lo && j < hi;
        sure[k] = __ballot_sync(0xffffffffu, j < length && (!in || (all && need > 0 ? r >= least : r > least)));
        tied[k] = __ballot_sync(0xffffffffu, j < length && in && !all && r == least);
        if (lane == k) counts[k * kChooseWarps + warp] = make_int2(__popc(sure[k]), __popc(tied[k]));
      }
      __syncthreads();
      if (warp == 0) {
        int2 mine[kHeld], sum = make_int2(0, 0);              // a lane has eight in a row
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
          const int2 x = counts[lane * kHeld + k];
          mine[k] = sum;
          sum.x += x.x, sum.y += x.y;
        }
        const int x = warp_sums(sum.x), y = warp_sums(sum.y);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) counts[lane * kHeld + k] = make_int2(mine[k].x + x - sum.x, mine[k].y + y - sum.y);
        if (lane == 31) group_counts = make_int2(x, y);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int j = j0 + k * kChooseThreads + threadIdx.x;
        const int2 before = counts[k * kChooseWarps + warp];
        const int equal = base.y + before.y + __popc(tied[k] & below);
        places[k] = -1;
        if ((sure[k] >> lane & 1) != 0 || ((tied[k] >> lane & 1) != 0 && equal < ties)) {
          const int at = base.x + before.x + __popc(sure[k] & below) + min(equal, ties), page = row[j >> c.page_log2];
          kept[at] = ((int64_t)page << c.page_log2) + (j & in_page);
          places[k] = at;
          if (!in_one) staged[at] = w[k];
          if (at != j) moved = min(moved, at);
          fault |= cache_page_ok(c, page) ? 0 : KB200_CACHE_NO_ROOM;
        }
      }
      base.x += group_counts.x, base.y += group_counts.y;
      __syncthreads();
    }
    if (moved != INT_MAX) atomicMin(&first_moved, moved);
    if (fault != 0) atomicOr(&faults, fault);
    __syncthreads();
    if (first_moved != INT_MAX) {
      const int first_page = first_moved >> c.page_log2;
      int bad = (int)threadIdx.x >= first_page ? my_page_faults : 0;
      for (int k = threadIdx.x + kChooseThreads; k <= last_page; k += kChooseThreads) bad |= k >= first_page ? page_faults(k) : 0;
      if (bad != 0) atomicOr(&faults, bad);
    }
    __syncthreads();
    if (faults == 0) {
      if (threadIdx.x == 0) p.answers[s] = make_int2(want, first_moved);
      if (in_one) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (places[k] >= 0) out[places[k]] = w[k];
      }
      for (int i = threadIdx.x; i < p.width; i += kChooseThreads)
        if (!in_one || i >= want) out[i] = i < want ? staged[i] : 0.0f;
      return;
    }
  }
  if (threadIdx.x == 0) {
    if (faults != 0) cache_fault(c, faults);
    p.answers[s] = make_int2(-1, 0);
  }
  for (int i = threadIdx.x; i < p.width; i += kChooseThreads) out[i] = i < length ? weights[i] : 0.0f;
}

// ---- the tokens --------------------------------------------------------------------------------

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32, kMoveAtOnce = 16;

// A CTA takes one sequence's tokens in one layer, head and of K or V.  Token i comes from a place behind its own or from its own: batches ascend, and a batch
// is read before any of it is written, so nothing is overwritten that is still to be read.  A warp has up to 32 neighbouring tokens of a batch, whose places its lanes work out, one each, and moves
// up to 512 chunks of 16 bytes, 16 to a lane, all under way at once.  (With a place looked up for every chunk 157 us for 390 MB, 5.0 TB/s both ways.)
// And what is behind the kept tokens is given up, which no token moves into or out of.
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(const CacheView c, const EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_page = (1 << c.page_log2) - 1;
  for (int s = gridDim.x * warp + blockIdx.x; s < c.sequences; s += gridDim.x * kMoveWarps)
    if (p.answers[s].x >= 0) cut(c, s, p.answers[s].x);
  const int64_t planes = (int64_t)c.layers * 2 * c.kv_heads, units = planes * c.sequences;
  const int rows = min(32, 32 * kMoveAtOnce / c.row_chunks), chunks = rows * c.row_chunks;        // of a warp (row_chunks: 64 at most)
  const int reciprocal = ((1 << 20) + c.row_chunks - 1) / c.row_chunks;                           // chunk / row_chunks of up to 2048 = chunk * reciprocal >> 20
  uint4* const pool = static_cast<uint4*>(c.pool);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int s = (int)(u / planes);
    const int2 answer = p.answers[s];
    if (answer.x < 0 || answer.y >= answer.x) continue;
    const int64_t plane = u % planes;
    const int64_t half = plane / c.kv_heads * c.pages;          // K or V of a layer, in pages
    const int head = (int)(plane % c.kv_heads);
    const int32_t* const table = c.table + (int64_t)s * c.max_pages;
    const int64_t* const kept = p.from + (int64_t)s * p.width;
    auto place = [&](int64_t page, int at) { return ((((half + page) * c.kv_heads + head) << c.page_log2) + at) * c.row_chunks; };
    for (int token0 = answer.y; token0 < answer.x; token0 += kMoveWarps * rows) {
      const int token = token0 + warp * rows + lane, there = min(rows, answer.x - token0 - warp * rows);
      int64_t from = 0, to = 0;
      if (lane < there) {
        const int64_t slot = kept[token];
        from = place(slot >> c.page_log2, (int)(slot & in_page));
        to = place(table[token >> c.page_log2], token & in_page);
      }
      uint4 v[kMoveAtOnce];
      auto each = [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < kMoveAtOnce; ++j) {
          if (32 * j >= chunks) break;
          const int i = 32 * j + lane, r = i * reciprocal >> 20;
          f(j, r, i - r * c.row_chunks);
        }
      };
      each([&](int j, int r, int chunk) {
        const int64_t at = __shfl_sync(0xffffffffu, from, r & 31);
        if (r < there) v[j] = __ldcs(pool + at + chunk);
      });
      __syncthreads();
      each([&](int j, int r, int chunk) {
        const int64_t at = __shfl_sync(0xffffffffu, to, r & 31);
        if (r < there) pool[at + chunk] = v[j];
      });
    }
  }
}

// ---- host --------------------------------------------------------------------------------------

int64_t width_of(const Cache& c) { return (int64_t)c.view.max_pages << c.view.page_log2; }
int64_t up(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace kb200

using namespace kb200;

KB200_EXPORT int kb200_cache_release(kb200_cache* handle, int window, int sinks, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_release");
  if (window < 1 || sinks < 0) return fail(KB200_ERR_ARGUMENT, "kb200_cache_release: a window of %d tokens behind %d", window, sinks);
  const dim3 grid((unsigned)std::min((c.view.max_pages + kReleaseThreads - 1) / kReleaseThreads, 64), (unsigned)std::min(c.view.sequences, 65535));
  KB200_CUDA(launch_kernel(true, release_kernel, grid, dim3(kReleaseThreads), 0, s, c.view, window, sinks));
  return KB200_OK;
}

KB200_EXPORT uint64_t kb200_cache_evict_workspace(const kb200_cache* handle) {
  if (handle == nullptr) return 0;
  const Cache& c = *cache_of(handle);
  const int64_t n = c.view.sequences * width_of(c);
  return (uint64_t)(up(n * 8) + up(n * 4) + up((int64_t)c.view.sequences * 8));
}

KB200_EXPORT int kb200_cache_evict(kb200_cache* handle, const float* weights, int64_t weights_stride, const int32_t* keep, int recent, int sinks, float* out,
                                   int64_t out_stride, void* workspace, uint64_t workspace_bytes, void* stream) {
  KB200_CACHE_ENTER("kb200_cache_evict");
  if (weights == nullptr || keep == nullptr || out == nullptr) return fail(KB200_ERR_ARGUMENT, "kb200_cache_evict: weights, keep or out is null");
  if (recent < 0 || sinks < 0) return fail(KB200_ERR_ARGUMENT, "kb200_cache_evict: %d recent and %d first tokens", recent, sinks);
  const int64_t width = width_of(c), n = c.view.sequences * width;
  if (c.view.sequences > 1 && (weights_stride < width || out_stride < width))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_evict: rows of weights and out are %lld long", (long long)width);
  if (workspace == nullptr || !tc::aligned16(workspace) || workspace_bytes < kb200_cache_evict_workspace(handle))
    return fail(KB200_ERR_ARGUMENT, "kb200_cache_evict: a workspace of %llu bytes on 16 bytes is needed", (unsigned long long)kb200_cache_evict_workspace(handle));
  char* const at = static_cast<char*>(workspace);
  EvictParams p{weights, out, weights_stride, out_stride, keep, reinterpret_cast<int64_t*>(at), reinterpret_cast<float*>(at + up(n * 8)),
                reinterpret_cast<int2*>(at + up(n * 8) + up(n * 4)), recent, sinks, (int)width};
  KB200_CUDA(launch_kernel(true, evict_choose_kernel, dim3(c.view.sequences), dim3(kChooseThreads), 0, s, c.view, p));
  const int64_t units = c.planes() * c.view.sequences;
  KB200_CUDA(launch_kernel(true, evict_move_kernel, dim3((unsigned)std::min<int64_t>(units, 2 * c.sm_count)), dim3(kMoveThreads), 0, s, c.view, p));
  return KB200_OK;
}
