// What the operators' entry points refuse before anything reaches the device. Host only: no CUDA here.
#include <math.h>

#include <algorithm>

#include "operators.h"

namespace b2 {
namespace {

std::string N(uint64_t v) { return std::to_string(v); }
bool Float(uint32_t t) { return t == B2_F32 || t == B2_F16 || t == B2_BF16; }
bool Half(uint32_t t) { return t == B2_F16 || t == B2_BF16; }

// Rows by bytes: head h of row r is `width` bytes from at + r row + h head.
typedef __int128 Wide;               // (2^31 rows of strides up to 2^40)
struct Place {
  Wide at, row, head, lo, hi;        // [lo, hi): all of it
  int64_t n, heads, width;
  Place(const b2_rows &r, uint32_t rows, uint32_t h, uint32_t head_dim, uint32_t dtype) : n(rows), heads(h) {
    const int64_t e = TypeBytes(dtype);
    at = static_cast<Wide>(reinterpret_cast<uintptr_t>(r.data));
    row = rows > 1 ? static_cast<Wide>(r.row_stride) * e : 0;
    head = h > 1 ? static_cast<Wide>(r.head_stride) * e : 0;
    width = head_dim * e;
    const Wide far_row = row * (n - 1), far_head = head * (heads - 1);
    lo = at + std::min<Wide>(far_row, 0) + std::min<Wide>(far_head, 0);
    hi = at + std::max<Wide>(far_row, 0) + std::max<Wide>(far_head, 0) + width;
  }
};
Wide Abs(Wide x) { return x < 0 ? -x : x; }
// Whether |d - r row - h head| < width for some r in (-n, n) and h in [h0, h1]; `itself`: but for r = h = 0.
bool Meets(Wide d, Wide row, Wide head, int64_t n, int64_t h0, int64_t h1, int64_t width, bool itself) {
  for (int64_t h = h0; h <= h1; ++h) {
    const Wide rest = d - h * head, near = row ? std::max<Wide>(1 - n, std::min<Wide>(rest / row, n - 1)) : 0;
    for (Wide r = near - 1; r <= near + 1; ++r)
      if (Abs(r) < n && Abs(rest - r * row) < width && !(itself && r == 0 && h == 0)) return true;
  }
  return false;
}

}  // namespace

std::string CheckResult(const char *what, const b2_rows *r, uint32_t n_rows, uint32_t heads, uint32_t head_dim, uint32_t dtype) {
  if (n_rows == 0 || heads == 0) return "";
  const Place p(*r, n_rows, heads, head_dim, dtype);
  const bool by_rows = (heads == 1 || Abs(p.head) >= p.width) && (n_rows == 1 || Abs(p.row) >= Abs(p.head) * (p.heads - 1) + p.width);
  const bool by_heads = (n_rows == 1 || Abs(p.row) >= p.width) && (heads == 1 || Abs(p.head) >= Abs(p.row) * (p.n - 1) + p.width);
  if (by_rows || by_heads || !Meets(0, p.row, p.head, p.n, 0, p.heads - 1, p.width, true)) return "";
  return std::string(what) + ": rows or heads lie over each other";
}

std::string CheckApart(const char *result, const b2_rows *y, uint32_t y_heads, const char *other, const b2_rows *x, uint32_t x_heads, uint32_t n_rows, uint32_t head_dim,
                       uint32_t dtype, bool same) {
  if (n_rows == 0 || y_heads == 0 || x_heads == 0) return "";
  const Place p(*y, n_rows, y_heads, head_dim, dtype), q(*x, n_rows, x_heads, head_dim, dtype);
  if (p.hi <= q.lo || q.hi <= p.lo) return "";
  const bool rows_alike = p.row == q.row, heads_alike = p.head == q.head || y_heads == 1 || x_heads == 1;
  if (same && p.at == q.at && rows_alike && p.head == q.head) return "";
  // (rows of different strides in the same memory: taken to meet)
  if (rows_alike && heads_alike && !Meets(q.at - p.at, p.row, y_heads > 1 ? p.head : q.head, p.n, 1 - q.heads, p.heads - 1, p.width, false)) return "";
  return std::string(result) + " lies over " + other;
}

std::string CheckRopeDesc(const b2_rope_desc *d) {
  if (!d) return "null description";
  if (!Float(d->dtype)) return "rows of type " + N(d->dtype) + " (f32, f16 or bf16)";
  if (d->weight_dtype != B2_F32 && d->weight_dtype != d->dtype) return "weights are f32 or of the rows' type";
  if (d->head_dim == 0 || d->head_dim % 2 || d->head_dim > 256) return "head_dim " + N(d->head_dim) + " (even, 2 to 256)";
  if (d->rot_dim % 2 || d->rot_dim > d->head_dim) return "rot_dim " + N(d->rot_dim) + " (even, at most head_dim " + N(d->head_dim) + ")";
  if (d->q_heads > 65535 || d->k_heads > 65535 || d->q_heads + d->k_heads == 0) return "heads: 1 to 65535";
  if (d->norm && !(d->eps >= 0.0f && isfinite(d->eps))) return "eps must be finite and not negative";
  if (d->rot_dim && !d->frequencies) return "null frequencies";
  for (uint32_t i = 0; i < d->rot_dim / 2; ++i)
    if (!isfinite(d->frequencies[i])) return "frequency " + N(i) + " is not finite";
  if (d->rot_dim && !isfinite(static_cast<float>(d->magnitude))) return "magnitude must be finite in f32";
  return "";
}

std::string CheckCacheDesc(const b2_cache_desc *d) {
  if (!d) return "null description";
  if (!Half(d->dtype) && d->dtype != B2_E4M3) return "pages of type " + N(d->dtype) + " (f16, bf16 or e4m3)";
  if (!Float(d->row_dtype)) return "rows of type " + N(d->row_dtype) + " (f32, f16 or bf16)";
  if (Half(d->dtype) && d->row_dtype != B2_F32 && d->row_dtype != d->dtype) return "16-bit pages take rows of their own type or f32";
  if (d->heads == 0 || d->heads > 65535) return "heads: 1 to 65535";
  if (d->q_heads % d->heads || d->q_heads > 65535 || d->q_heads == 0) return "q_heads " + N(d->q_heads) + " is not a multiple of heads " + N(d->heads);
  if (d->head_dim == 0 || d->head_dim % 16 || d->head_dim > 128) return "head_dim " + N(d->head_dim) + " (a multiple of 16, at most 128)";
  if (d->page_size == 0 || d->page_size > 0x7fffffffu) return "page_size must be at least 1";
  if (d->n_pages == 0 || d->n_pages > 0x7fffffffu) return "n_pages must be at least 1";
  if (!d->k_pages || !d->v_pages) return "null pages";
  const int64_t e = TypeBytes(d->dtype);
  if (reinterpret_cast<uintptr_t>(d->k_pages) % 16 || reinterpret_cast<uintptr_t>(d->v_pages) % 16) return "pages must be 16-byte aligned";
  for (int64_t s : {d->page_stride, d->slot_stride, d->head_stride})
    if (s < 0 || s > (int64_t(1) << 48) || s * e % 16) return "strides of pages must be multiples of 16 bytes and not negative";
  // rows that lie over each other would be written over each other
  if ((d->heads > 1 && d->head_stride < d->head_dim) || (d->page_size > 1 && d->slot_stride < d->head_dim) || (d->n_pages > 1 && d->page_stride < d->head_dim))
    return "strides of pages are smaller than a row of " + N(d->head_dim) + " values";
  if (d->dtype == B2_E4M3) {
    if (!d->k_scales || !d->v_scales) return "e4m3 pages need scales";
    if (reinterpret_cast<uintptr_t>(d->k_scales) % 4 || reinterpret_cast<uintptr_t>(d->v_scales) % 4) return "scales must be 4-byte aligned";
    for (int64_t s : {d->scale_page_stride, d->scale_slot_stride, d->scale_head_stride})
      if (s < 0 || s > (int64_t(1) << 48)) return "strides of scales must not be negative";
    if ((d->heads > 1 && !d->scale_head_stride) || (d->page_size > 1 && !d->scale_slot_stride) || (d->n_pages > 1 && !d->scale_page_stride))
      return "scales of different rows share a place (a stride of 0)";
  }
  return "";
}

std::string CheckBatch(const b2_batch *b) {
  if (!b) return "null batch";
  if (b->n_seqs > (1u << 20)) return "n_seqs " + N(b->n_seqs) + " (at most 1048576)";
  if (b->n_rows > 0x7fffffffu) return "n_rows " + N(b->n_rows) + " (below 2^31)";
  if (b->n_seqs == 0 || b->n_rows == 0) return "";        // nothing to do
  if (!b->row_start || !b->length || (!b->pages && b->max_pages)) return "null row_start, length or pages";
  if (reinterpret_cast<uintptr_t>(b->row_start) % 4 || reinterpret_cast<uintptr_t>(b->length) % 4 || reinterpret_cast<uintptr_t>(b->pages) % 4)
    return "row_start, length and pages must be 4-byte aligned";
  if (b->pages_stride < 0 || b->pages_stride > (int64_t(1) << 40) || (b->n_seqs > 1 && static_cast<uint64_t>(b->pages_stride) < b->max_pages))
    return "pages_stride is smaller than max_pages " + N(b->max_pages);
  return "";
}

std::string CheckRows(const char *what, const b2_rows *r, uint32_t n_rows, uint32_t heads, uint32_t dtype) {
  if (n_rows == 0 || heads == 0) return "";
  const std::string w = what;
  if (!r || !r->data) return w + ": null rows";
  if (reinterpret_cast<uintptr_t>(r->data) % TypeBytes(dtype)) return w + ": not aligned to its type";
  const int64_t most = int64_t(1) << 40;
  if (r->row_stride < -most || r->row_stride > most || r->head_stride < -most || r->head_stride > most) return w + ": stride out of range";
  return "";
}

std::string CheckAttend(const b2_cache_desc &d, const b2_batch *b, const b2_rows *q, const b2_rows *o, float scale, int causal, uint32_t window, const void *lse) {
  std::string m = CheckBatch(b);
  if (!m.empty()) return m;
  if (d.row_dtype == B2_F32) return "attention of f32 rows (f16 or bf16)";
  if (!(scale > 0.0f && scale <= 1e38f)) return "scale must be positive and at most 1e38";
  if (window && !causal) return "a window needs causal";
  if (window > 0x7fffffffu) return "window " + N(window) + " (below 2^31)";
  if (reinterpret_cast<uintptr_t>(lse) % 4) return "lse must be 4-byte aligned";
  if ((m = CheckRows("q", q, b->n_rows, d.q_heads, d.row_dtype)).empty()) m = CheckRows("out", o, b->n_rows, d.q_heads, d.row_dtype);
  // (a sequence's rows x group are numbered in 31 bits)
  const uint64_t most = b->max_rows && b->max_rows < b->n_rows ? b->max_rows : b->n_rows;
  if (m.empty() && most * (d.q_heads / d.heads) > 0x7fffffffu) m = "rows of a sequence x q_heads / heads: " + N(most) + " x " + N(d.q_heads / d.heads) + " (below 2^31)";
  if (m.empty() && b->n_rows && q->data == o->data) m = "out lies over q (a row of q may be read after its result is there)";
  return m;
}

}  // namespace b2
