// Device code that the operators beside the programs share: vectors of rows in memory, conversions, who a row belongs
// to, where a position lies in the cache, status words.
#ifndef B2VM_OPERATORS_DEV_CUH_
#define B2VM_OPERATORS_DEV_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "operators.h"
#include "ptx.cuh"

namespace b2 {

template <typename T> __device__ __forceinline__ float ToF(T v);
template <> __device__ __forceinline__ float ToF<float>(float v) { return v; }
template <> __device__ __forceinline__ float ToF<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float ToF<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromF(float v);
template <> __device__ __forceinline__ float FromF<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromF<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromF<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V values next to each other, moved as one access.
template <typename T, int V> struct __align__(sizeof(T) * V) Vec { T v[V]; };

// The first fault a cache's calls meet stays in its status words.
__device__ __forceinline__ void cache_fault(uint32_t *status, uint32_t code, uint32_t seq, uint32_t where, uint32_t detail) {
  if (atomicCAS(status, 0u, code) == 0u) {
    status[1] = seq;
    status[2] = where;
    status[3] = detail;
  }
}

__device__ __forceinline__ Seq load_seq(const BatchView &b, uint64_t capacity, uint32_t i) {
  return MakeSeq(b.row_start[i], b.row_start[i + 1], b.length[i], b.n_rows, b.max_rows, capacity);
}
__device__ __forceinline__ uint64_t capacity_of(const CacheView &c, const BatchView &b) { return static_cast<uint64_t>(b.max_pages) * c.page_size; }

// Byte offset of position p's row (head 0) in the pages, -1 when its page does not exist (the fault is recorded). p must be
// below the sequence's length, which is at most max_pages x page_size.
__device__ __forceinline__ int64_t page_offset(const CacheView &c, const BatchView &b, uint32_t seq, uint32_t p, int64_t *scale_at) {
  const uint32_t e = c.by_page.quot(p), slot = p - e * c.page_size;
  const int32_t page = __ldg(b.pages + static_cast<int64_t>(seq) * b.pages_stride + e);
  if (static_cast<uint32_t>(page) >= c.n_pages) {
    cache_fault(c.status, kStBadPage, seq, e, static_cast<uint32_t>(page));
    return -1;
  }
  *scale_at = page * c.s_page + slot * c.s_slot;
  return page * c.page_bytes + slot * c.slot_bytes;
}

// The sequence that row i belongs to: the last b with row_start[b] <= i. One warp, 32 starts a step.
__device__ __forceinline__ uint32_t seq_of_row(const int32_t *row_start, uint32_t n_seqs, int32_t i) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t lo = 0, n = n_seqs;                            // among [lo, lo + n)
  while (n > 1u) {
    const uint32_t step = (n + 31u) / 32u, at = lo + lane * step;
    const bool below = lane * step < n && row_start[at] <= i;
    const uint32_t m = __ballot_sync(0xffffffffu, below);
    const uint32_t k = m ? 31u - __clz(m) : 0u;           // the last of the 32 that starts at or before i
    const uint32_t end = lo + n;
    lo += k * step;
    n = min(lo + step, end) - lo;
  }
  return lo;
}

}  // namespace b2
#endif
