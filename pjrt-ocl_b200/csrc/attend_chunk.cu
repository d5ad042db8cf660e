// Attention of many rows of each sequence over the paged cache: chunks of prompts.
//
// Simple form: a warp to a row of a head, one pass over the keys it sees.
#include "attend_common.cuh"

namespace b2 {
namespace {

__global__ void __launch_bounds__(256) b2_attend_rows(const __grid_constant__ AttendArgs a) {
  const uint64_t cap = capacity_of(a.c, a.b);
  const uint32_t tid = threadIdx.x;
  if (blockIdx.x == 0u) {
    for (uint32_t i = tid; i < a.b.n_seqs; i += 256u) {
      const Seq q = load_seq(a.b, cap, i);
      if (q.bad) cache_fault(a.c.status, kStBadBatch, i, static_cast<uint32_t>(q.bad), static_cast<uint32_t>(q.value));
    }
  }
  const uint64_t warps = static_cast<uint64_t>(gridDim.x) * 8u;
  for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * 8u + (tid >> 5); r < static_cast<uint64_t>(a.b.n_rows) * a.q_heads; r += warps) {
    const int32_t row = static_cast<int32_t>(r / a.q_heads);
    const uint32_t seq = seq_of_row(a.b.row_start, a.b.n_seqs, row);
    const Seq s = load_seq(a.b, cap, seq);
    if (row < s.first || row - s.first >= s.n) continue;
    attend_row_alone(a, seq, s, row - s.first, static_cast<uint32_t>(r % a.q_heads));
  }
}

}  // namespace

int PrepareAttendChunk() { return 0; }
size_t AttendChunkPartialBytes(uint32_t) { return 0; }
int LaunchAttendChunk(const AttendArgs &a, CUstream_st *stream) {
  b2_attend_rows<<<148 * 8, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace b2
