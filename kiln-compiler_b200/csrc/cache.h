// The paged K/V cache: what its operations (cache.cu) and the attention over it (cache_attention.cu) share.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kb200_internal.h"

namespace kb200 {

// The cache as kernels see it.
struct CacheView {
  void* pool;
  int32_t *table, *held, *lengths, *refs;
  int* status;
  int layers, sequences, max_pages, pages, kv_heads, page_log2, head_dim;
  int row_chunks;          // 16-byte chunks of a token's row
};

constexpr int kCacheWaitFault = 1 << 16;      // a bounded wait of the attention ran out (beside kb200_cache_fault in the status word)

struct Cache {
  CacheView view;
  int dtype = 0;
  int device = 0;
  int sm_count = 148;
  int element = 2;         // bytes
  int64_t planes() const { return (int64_t)view.layers * 2 * view.kv_heads; }      // of a page
  // scratch of the operations that change the cache, one allocation
  void* scratch = nullptr;
  int32_t* stage_rows = nullptr;     // [sequences, max_pages]
  int32_t* stage_slot = nullptr;     // [3, sequences]
  int32_t* page_a = nullptr;         // [pages]
  int32_t* page_b = nullptr;         // [pages]
  int4* copies = nullptr;            // pages to copy: from, to, tokens
  int* counters = nullptr;           // see cache.cu
  CUtensorMap map;                   // the pool: elements of a row, rows of a page (head by head), pages of K and of V layer by layer
};

int cache_attention_prepare(Cache& c);       // (cache_attention.cu) the pool's map and the kernels' limits, on the current device

// This thread's device for the duration of a call.
struct DeviceGuard {
  int before = -1;
  cudaError_t error;
  explicit DeviceGuard(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
    else if (error == cudaSuccess) before = -1;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};

#ifdef __CUDACC__
__device__ __forceinline__ void cache_fault(const CacheView& c, int bits) { atomicOr(c.status, bits); }
__device__ __forceinline__ bool cache_page_ok(const CacheView& c, int page) { return (unsigned)page < (unsigned)c.pages; }
// The first of a page's rows: [layer, K or V, page, head]
__device__ __forceinline__ int64_t cache_row(const CacheView& c, int layer, int which, int page, int head) {
  return ((((int64_t)layer * 2 + which) * c.pages + page) * c.kv_heads + head) << c.page_log2;
}
#endif

}  // namespace kb200
