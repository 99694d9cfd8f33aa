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

// A CTA takes a sequence.  The least rank that stays is found digit by digit (11, 11 and 10 bits from the top), by counting the candidates of each digit; of the tokens
// at that rank the first ones stay.  Two sweeps then give every kept token its place: a warp has neighbouring tokens, so that its places begin behind those of the
// warps before it.
__global__ void __launch_bounds__(kChooseThreads) evict_choose_kernel(const CacheView c, const EvictParams p) {
  __shared__ int bins[kBins];
  __shared__ int sums[kChooseWarps];
  __shared__ int2 counts[kChooseWarps];
  __shared__ int digit, above, in_digit, first_moved, faults;
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_page = (1 << c.page_log2) - 1;
  const float* const weights = p.weights + s * p.weights_stride;
  float* const out = p.out + s * p.out_stride;
  const int32_t* const row = c.table + (int64_t)s * c.max_pages;
  const int held = min(max(c.held[s], 0), c.max_pages), want = p.keep[s];
  int length = max(c.lengths[s], 0);
  if (threadIdx.x == 0) first_moved = INT_MAX, faults = 0;
  if ((int64_t)length > (int64_t)held << c.page_log2) {
    if (threadIdx.x == 0) cache_fault(c, KB200_CACHE_NO_ROOM);
    length = held << c.page_log2;
  } else if (want >= 0 && want < length) {
    const int first = min(p.sinks, want), last = min(p.recent, want - first);
    const int lo = first, hi = length - last;                 // the candidates, of which `need` stay
    int need = want - first - last;
    uint32_t prefix = 0u;
    int shift = 32;
    bool all = need == 0;                                     // every candidate of this prefix and above stays (need 0: none)
    while (shift > 0 && !all) {
      const int bits = shift > 10 ? 11 : 10;
      for (int i = threadIdx.x; i < kBins; i += kChooseThreads) bins[i] = 0;
      __syncthreads();
      for (int j = lo + threadIdx.x; j < hi; j += kChooseThreads) {
        const uint32_t r = rank_of(weights[j]);
        if (shift == 32 || r >> shift == prefix) atomicAdd(&bins[r >> (shift - bits) & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      // from the highest digit down: thread t has digits kBins - 1 - 2t and the one below
      const int d = kBins - 1 - 2 * threadIdx.x, a = bins[d], b = bins[d - 1];
      int sum = a + b;
#pragma unroll
      for (int i = 1; i < 32; i *= 2) {
        const int below = __shfl_up_sync(0xffffffffu, sum, i);
        if (lane >= i) sum += below;
      }
      if (lane == 31) sums[warp] = sum;
      __syncthreads();
      int before = 0;
      for (int w = 0; w < warp; ++w) before += sums[w];
      before += sum - a - b;
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
    // Kept whatever the others are; kept if `ties` allow.
    auto sure = [&](int j, uint32_t r) { return j < lo || j >= hi || (all && need > 0 ? r >= least : r > least); };
    auto tied = [&](int j, uint32_t r) { return j >= lo && j < hi && !all && r == least; };
    const int part = (length + kChooseThreads - 1) / kChooseThreads * 32, from = min(warp * part, length), to = min(from + part, length);
    int2 mine = make_int2(0, 0);
    for (int j0 = from; j0 < to; j0 += 32) {
      const int j = j0 + lane;
      const uint32_t r = j < to ? rank_of(weights[j]) : 0u;
      mine.x += __popc(__ballot_sync(0xffffffffu, j < to && sure(j, r)));
      mine.y += __popc(__ballot_sync(0xffffffffu, j < to && tied(j, r)));
    }
    if (lane == 0) counts[warp] = mine;
    __syncthreads();
    int places = 0, equal = 0;
    for (int w = 0; w < warp; ++w) places += counts[w].x, equal += counts[w].y;
    places += min(equal, ties);
    int64_t* const kept = p.from + (int64_t)s * p.width;
    float* const staged = p.staged + (int64_t)s * p.width;
    const unsigned below = (1u << lane) - 1;
    int moved = INT_MAX, fault = 0;
    for (int j0 = from; j0 < to; j0 += 32) {
      const int j = j0 + lane;
      const float w = j < to ? weights[j] : 0.0f;
      const uint32_t r = rank_of(w);
      const bool is_tied = j < to && tied(j, r);
      const unsigned all_tied = __ballot_sync(0xffffffffu, is_tied);
      const bool stays = j < to && (sure(j, r) || (is_tied && equal + __popc(all_tied & below) < ties));
      const unsigned all_stay = __ballot_sync(0xffffffffu, stays);
      if (stays) {
        const int at = places + __popc(all_stay & below), page = row[j >> c.page_log2];
        kept[at] = ((int64_t)page << c.page_log2) + (j & in_page);
        staged[at] = w;
        if (at != j) moved = min(moved, at);
        fault |= cache_page_ok(c, page) ? 0 : KB200_CACHE_NO_ROOM;
      }
      places += __popc(all_stay);
      equal += __popc(all_tied);
    }
    if (moved != INT_MAX) atomicMin(&first_moved, moved);
    if (fault != 0) atomicOr(&faults, fault);
    __syncthreads();
    // What is written has to be the sequence's own.
    if (first_moved != INT_MAX)
      for (int k = (first_moved >> c.page_log2) + threadIdx.x; k <= (want - 1) >> c.page_log2; k += kChooseThreads) {
        const int page = row[k];
        const int bad = !cache_page_ok(c, page) ? KB200_CACHE_NO_ROOM : c.refs[page] > 1 ? KB200_CACHE_SHARED : 0;
        if (bad != 0) atomicOr(&faults, bad);
      }
    __syncthreads();
    if (faults == 0) {
      if (threadIdx.x == 0) p.answers[s] = make_int2(want, first_moved);
      for (int i = threadIdx.x; i < p.width; i += kChooseThreads) out[i] = i < want ? staged[i] : 0.0f;
      return;
    }
    if (threadIdx.x == 0) cache_fault(c, faults);
  }
  if (threadIdx.x == 0) p.answers[s] = make_int2(-1, 0);
  for (int i = threadIdx.x; i < p.width; i += kChooseThreads) out[i] = i < length ? weights[i] : 0.0f;
}

// ---- the tokens --------------------------------------------------------------------------------

constexpr int kMoveThreads = 256, kMoveAtOnce = 8;

// A CTA takes one sequence's tokens in one layer, head and of K or V.  Token i comes from a place behind its own or from its own: batches ascend, and a batch
// is read before any of it is written, so nothing is overwritten that is still to be read.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const CacheView c, const EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t planes = (int64_t)c.layers * 2 * c.kv_heads, units = planes * c.sequences;
  const int in_page = (1 << c.page_log2) - 1;
  uint4* const pool = static_cast<uint4*>(c.pool);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int s = (int)(u / planes);
    const int2 answer = p.answers[s];
    if (answer.x < 0 || answer.y >= answer.x) continue;
    const int64_t plane = u % planes;
    const int64_t half = plane / c.kv_heads * c.pages;          // K or V of a layer, in pages
    const int head = (int)(plane % c.kv_heads);
    const int32_t* const row = c.table + (int64_t)s * c.max_pages;
    const int64_t* const kept = p.from + (int64_t)s * p.width;
    auto place = [&](int64_t page, int at) { return pool + ((((half + page) * c.kv_heads + head) << c.page_log2) + at) * c.row_chunks; };
    const int64_t chunks = (int64_t)(answer.x - answer.y) * c.row_chunks;
    for (int64_t i0 = 0; i0 < chunks; i0 += kMoveThreads * kMoveAtOnce) {
      uint4 v[kMoveAtOnce];
      uint4* to[kMoveAtOnce];
      const int batch = (int)min((int64_t)(kMoveThreads * kMoveAtOnce), chunks - i0);
      const int token0 = answer.y + (int)(i0 / c.row_chunks), chunk0 = (int)(i0 % c.row_chunks);
#pragma unroll
      for (int j = 0; j < kMoveAtOnce; ++j) {
        const int i = threadIdx.x + kMoveThreads * j;
        to[j] = nullptr;
        if (i < batch) {
          const int ahead = (chunk0 + i) / c.row_chunks, chunk = chunk0 + i - ahead * c.row_chunks, token = token0 + ahead;
          const int64_t from = kept[token];
          v[j] = __ldcs(place(from >> c.page_log2, (int)(from & in_page)) + chunk);
          to[j] = place(row[token >> c.page_log2], token & in_page) + chunk;
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMoveAtOnce; ++j)
        if (to[j] != nullptr) *to[j] = v[j];
    }
  }
}

constexpr int kSlotThreads = 128;

__global__ void __launch_bounds__(kSlotThreads) evict_commit_kernel(const CacheView c, const EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x * (kSlotThreads / 32) + (threadIdx.x >> 5);
  if (s < c.sequences && p.answers[s].x >= 0) cut(c, s, p.answers[s].x);
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
  KB200_CUDA(launch_kernel(true, evict_move_kernel, dim3((unsigned)std::min<int64_t>(units, 16 * c.sm_count)), dim3(kMoveThreads), 0, s, c.view, p));
  const int per = kSlotThreads / 32;
  KB200_CUDA(launch_kernel(true, evict_commit_kernel, dim3((c.view.sequences + per - 1) / per), dim3(kSlotThreads), 0, s, c.view, p));
  return KB200_OK;
}
