// What the operators beside the programs share between their C entry points (operators.cc), their checks
// (operators_check.cc, host only) and their kernels (rope.cu, paged_cache.cu, attend_step.cu, attend_chunk.cu).
#ifndef B2VM_OPERATORS_H_
#define B2VM_OPERATORS_H_

#include <stddef.h>
#include <stdint.h>

#include <string>

#include "../../include/b2vm.h"

#ifdef __CUDACC__
#define B2_HD __host__ __device__ __forceinline__
#else
#define B2_HD inline
#endif

struct CUstream_st;

namespace b2 {

constexpr uint32_t kStBadPage = 5, kStBadBatch = 6;   // b2_exec_status codes of the cache's calls
constexpr uint32_t kStTcTimeout = 4;

inline uint32_t TypeBytes(uint32_t dtype) { return dtype == B2_F32 ? 4u : dtype == B2_E4M3 ? 1u : 2u; }

// x / d and x % d for 0 <= x < 2^31 by a multiplication: m = ceil(2^(32 + s) / d) with 2^s >= d, so that the error of
// the product stays below 2^32 for such x.
struct FastDiv {
  uint32_t d = 1, m = 0, s = 0;     // m holds the multiplier less 2^32
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << s) < div) ++s;
    m = static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - div)) / div + 1);
  }
  B2_HD uint32_t quot(uint32_t x) const {
    const uint32_t hi = static_cast<uint32_t>((static_cast<uint64_t>(x) * m) >> 32);
    return static_cast<uint32_t>((static_cast<uint64_t>(hi) + x) >> s);
  }
};

struct RowsRef { uint8_t *p; int64_t row, head; };    // strides in elements

struct RopeArgs {
  RowsRef x[2], y[2], g[2];        // queries, keys: inputs, results, gradients of the results
  const void *w[2];
  float *dw[2];
  float *partial;                  // backward: [CTA][2][head_dim]
  const int32_t *pos;
  const double *turns;             // turns for each position: frequency / 2 pi
  float magnitude, eps;
  uint32_t n_rows, heads[2], hd, rot, interleaved, norm, weight_f32;
};

// The cache as the kernels see it.
struct CacheView {
  uint8_t *k, *v;
  float *ks, *vs;
  int64_t page_bytes, slot_bytes, head_bytes;         // of the pages
  int64_t s_page, s_slot, s_head;                     // of the scales, in elements
  uint32_t n_pages, page_size, heads, hd;
  FastDiv by_page;
  uint32_t *status;                // 4 words, the first one wins
};
struct BatchView {
  const int32_t *row_start, *length, *pages;
  int64_t pages_stride;
  uint32_t n_seqs, n_rows, max_rows, max_pages;
};

// A sequence of the batch, with what does not fit its bounds cut off (`bad` names it): n rows from `first`, `len` positions.
struct Seq {
  int32_t first, n, len;
  int32_t bad;                     // 0, or 1 + which value was cut: row_start, row_start's end, length, rows
  int32_t value;
};
B2_HD Seq MakeSeq(int32_t r0, int32_t r1, int32_t length, uint32_t n_rows, uint32_t max_rows, uint64_t capacity) {
  Seq s;
  s.first = r0; s.n = r1 - r0; s.len = length; s.bad = 0; s.value = 0;
  if (r0 < 0 || r1 < r0) { s.first = 0; s.n = 0; s.bad = 1; s.value = r0 < 0 ? r0 : r1; }
  else if (static_cast<uint32_t>(r1) > n_rows) { s.n = 0; s.bad = 2; s.value = r1; }
  else if (max_rows && static_cast<uint32_t>(s.n) > max_rows) { s.bad = 4; s.value = s.n; s.n = 0; }
  if (length < 0 || static_cast<uint64_t>(length) > capacity) { s.len = 0; s.n = 0; s.bad = 3; s.value = length; }
  return s;
}

struct AttendArgs {
  CacheView c;
  BatchView b;
  RowsRef q, o;
  float *lse;
  float *part;                     // results of parts of a tile's keys
  uint32_t *arrived;               // counters, zero at rest
  float scale_log2;                // softmax scale x log2(e)
  uint32_t q_heads, group, causal, window;
  FastDiv by_group;
  uint32_t bf16;                   // type of the rows
  uint32_t e4m3;
  uint64_t wait_budget_ns;         // of each wait on the tensor cores
};

// Keys that row i of a sequence sees: [lo, hi).
struct Span { int32_t lo, hi; };
B2_HD Span SeenBy(const Seq &s, int32_t i, uint32_t causal, uint32_t window) {
  Span r;
  r.lo = 0;
  r.hi = s.len;
  if (causal) {
    r.hi = s.len - s.n + i + 1;
    if (window && r.hi > 0 && static_cast<uint32_t>(r.hi) > window) r.lo = r.hi - static_cast<int32_t>(window);
  }
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}
// Keys that any of rows [i0, i1) sees.
B2_HD Span SeenByRows(const Seq &s, int32_t i0, int32_t i1, uint32_t causal, uint32_t window) {
  Span r;
  r.lo = SeenBy(s, i0, causal, window).lo;
  r.hi = SeenBy(s, i1 - 1, causal, window).hi;
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}

constexpr uint32_t kStepRows = 16;        // rows x group of a sequence that the single-token kernel takes
constexpr uint32_t kChunkRows = 256;      // rows x group of a tile of the chunk kernel
constexpr uint32_t kScratchCounters = 1024;

// ---- checks (operators_check.cc): the message, empty = fine ----
std::string CheckRopeDesc(const b2_rope_desc *d);
std::string CheckCacheDesc(const b2_cache_desc *d);
std::string CheckBatch(const b2_batch *b);
std::string CheckRows(const char *what, const b2_rows *r, uint32_t n_rows, uint32_t heads, uint32_t dtype);
// Results: their own rows and heads apart from each other, and apart from other rows (`same`: but for the very same ones). Both sets have been checked as rows.
std::string CheckResult(const char *what, const b2_rows *r, uint32_t n_rows, uint32_t heads, uint32_t head_dim, uint32_t dtype);
std::string CheckApart(const char *result, const b2_rows *y, uint32_t y_heads, const char *other, const b2_rows *x, uint32_t x_heads, uint32_t n_rows, uint32_t head_dim, uint32_t dtype,
                       bool same);
std::string CheckAttend(const b2_cache_desc &d, const b2_batch *b, const b2_rows *q, const b2_rows *o, float scale, int causal, uint32_t window, const void *lse);

// ---- launches; each returns a cudaError_t's value ----
int PrepareRope();                        // shared-memory attributes on the current device
int LaunchRope(const RopeArgs &a, uint32_t dtype, bool backward, uint32_t sms, CUstream_st *stream);
uint32_t RopeBackwardCtas(uint32_t sms);
int LaunchCacheMove(const CacheView &c, const BatchView &b, const RowsRef &k, const RowsRef &v, uint32_t dtype, uint32_t row_dtype, bool write, uint32_t sms, CUstream_st *stream);
int PrepareAttendStep();                  // (as PrepareRope)
int PrepareAttendChunk();
int LaunchAttendStep(const AttendArgs &a, uint32_t sms, CUstream_st *stream);
int LaunchAttendChunk(const AttendArgs &a, uint32_t sms, CUstream_st *stream);
size_t AttendStepPartialBytes(uint32_t sms);
size_t AttendChunkPartialBytes(uint32_t sms);

}  // namespace b2
#endif
