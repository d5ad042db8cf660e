// The host side of the operators beside the programs, checked without a device: what their entry points refuse, and the
// arithmetic that host and kernels share (operators.h), against its definitions. Prints what is wrong and exits 1.
#include <cmath>
#include <cstdio>
#include <limits>

#include "operators.h"

static int wrong = 0;
static void Say(const char *what, const std::string &got) {
  std::printf("%s: %s\n", what, got.c_str());
  ++wrong;
}
static void Refused(const char *what, const std::string &m, const char *part) {
  if (m.find(part) == std::string::npos || m.empty()) Say(what, m.empty() ? "not refused" : m);
}
static void Fine(const char *what, const std::string &m) {
  if (!m.empty()) Say(what, m);
}

static void Divisions() {
  for (uint64_t d : {1ull, 2ull, 3ull, 5ull, 7ull, 16ull, 24ull, 48ull, 100ull, 255ull, 4097ull, 65535ull, 1000003ull, 0x40000000ull, 0x40000001ull, 0x7fffffffull}) {
    const b2::FastDiv f(static_cast<uint32_t>(d));
    uint64_t x = 1;
    for (int i = 0; i < 20000; ++i) {
      x = x * 6364136223846793005ull + 1442695040888963407ull;
      uint32_t v = static_cast<uint32_t>(x >> 33);
      if (i % 4 == 1) v = static_cast<uint32_t>(v / d * d);                            // a multiple
      if (i % 4 == 2 && v / d) v = static_cast<uint32_t>(v / d * d - 1);
      if (i < 3) v = 0x7fffffffu - static_cast<uint32_t>(i);
      if (f.quot(v) != v / d) { Say("quotient", std::to_string(v) + " / " + std::to_string(d)); break; }
    }
  }
}

static void Sequences() {
  struct { int32_t r0, r1, len, bad, n, l; } cases[] = {
      {0, 4, 9, 0, 4, 9}, {0, 0, 0, 0, 0, 0}, {3, 10, 2, 0, 7, 2}, {-1, 4, 9, 1, 0, 9}, {5, 4, 9, 1, 0, 9}, {0, 101, 200, 2, 0, 200},
      {0, 21, 30, 4, 0, 30}, {0, 4, -1, 3, 0, 0}, {0, 4, 1025, 3, 0, 0}, {0, 4, std::numeric_limits<int32_t>::max(), 3, 0, 0},
      {std::numeric_limits<int32_t>::min(), std::numeric_limits<int32_t>::max(), 5, 1, 0, 5}, {0, std::numeric_limits<int32_t>::max(), 5, 2, 0, 5}};
  for (const auto &c : cases) {
    const b2::Seq s = b2::MakeSeq(c.r0, c.r1, c.len, 100, 20, 1024);
    if (s.bad != c.bad || s.n != c.n || s.len != c.l) Say("sequence", std::to_string(c.r0) + ".." + std::to_string(c.r1) + " of " + std::to_string(c.len));
  }
  // what a row sees, key by key
  for (int32_t n : {1, 3, 7})
    for (int32_t len : {0, 1, 3, 6, 12})
      for (uint32_t causal : {0u, 1u})
        for (uint32_t window : {0u, 1u, 4u, 50u}) {
          if (window && !causal) continue;
          const b2::Seq s = b2::MakeSeq(0, n, len, 100, 0, 1024);
          int32_t lo = len, hi = 0;
          for (int32_t i = 0; i < n; ++i) {
            const b2::Span sp = b2::SeenBy(s, i, causal, window);
            for (int32_t k = 0; k < len; ++k) {
              const int32_t at = len - n + i;
              const bool sees = !causal || (k <= at && (!window || k > at - static_cast<int32_t>(window)));
              if (sees != (k >= sp.lo && k < sp.hi)) Say("seen", std::to_string(n) + " " + std::to_string(len) + " row " + std::to_string(i) + " key " + std::to_string(k));
              if (sees) { lo = k < lo ? k : lo; hi = k + 1 > hi ? k + 1 : hi; }
            }
          }
          const b2::Span all = b2::SeenByRows(s, 0, n, causal, window);
          if (lo < hi && (all.lo > lo || all.hi < hi)) Say("seen by rows", std::to_string(n) + " " + std::to_string(len));
        }
}

static void Refusals() {
  const float inf = std::numeric_limits<float>::infinity(), nan = std::numeric_limits<float>::quiet_NaN();
  double f[4] = {1.0, 0.1, 0.01, 0.001};
  b2_rope_desc r = {};
  r.head_dim = 8; r.rot_dim = 8; r.q_heads = 2; r.k_heads = 1; r.dtype = B2_BF16; r.weight_dtype = B2_F32; r.eps = 1e-6f; r.magnitude = 1.0; r.frequencies = f;
  Fine("rope", b2::CheckRopeDesc(&r));
  Refused("no rope", b2::CheckRopeDesc(nullptr), "null");
  auto rope = [&](const char *part, auto change) { b2_rope_desc x = r; change(x); Refused(part, b2::CheckRopeDesc(&x), part); };
  rope("rows of type", [](b2_rope_desc &x) { x.dtype = B2_E4M3; });
  rope("weights are", [](b2_rope_desc &x) { x.weight_dtype = B2_F16; });
  rope("head_dim", [](b2_rope_desc &x) { x.head_dim = 0; });
  rope("head_dim", [](b2_rope_desc &x) { x.head_dim = 9; });
  rope("head_dim", [](b2_rope_desc &x) { x.head_dim = 258; });
  rope("rot_dim", [](b2_rope_desc &x) { x.rot_dim = 10; });
  rope("rot_dim", [](b2_rope_desc &x) { x.rot_dim = 7; });
  rope("heads", [](b2_rope_desc &x) { x.q_heads = x.k_heads = 0; });
  rope("heads", [](b2_rope_desc &x) { x.q_heads = 65536; });
  rope("eps", [=](b2_rope_desc &x) { x.norm = 1; x.eps = nan; });
  rope("eps", [=](b2_rope_desc &x) { x.norm = 1; x.eps = -1.0f; });
  rope("null frequencies", [](b2_rope_desc &x) { x.frequencies = nullptr; });
  rope("magnitude", [=](b2_rope_desc &x) { x.magnitude = inf; });
  f[3] = inf;
  Refused("frequency", b2::CheckRopeDesc(&r), "frequency 3");
  r.rot_dim = 6;                                          // (it is not one of these)
  Fine("rope of three pairs", b2::CheckRopeDesc(&r));

  alignas(16) char mem[64];
  b2_cache_desc c = {};
  c.dtype = B2_E4M3; c.row_dtype = B2_BF16; c.heads = 2; c.q_heads = 4; c.head_dim = 64; c.page_size = 16; c.n_pages = 4; c.k_pages = c.v_pages = mem;
  c.page_stride = 2048; c.slot_stride = 128; c.head_stride = 64;
  c.k_scales = c.v_scales = reinterpret_cast<float *>(mem); c.scale_page_stride = 32; c.scale_slot_stride = 2; c.scale_head_stride = 1;
  Fine("cache", b2::CheckCacheDesc(&c));
  Refused("no cache", b2::CheckCacheDesc(nullptr), "null");
  auto cache = [&](const char *part, auto change) { b2_cache_desc x = c; change(x); Refused(part, b2::CheckCacheDesc(&x), part); };
  cache("pages of type", [](b2_cache_desc &x) { x.dtype = B2_F32; });
  cache("rows of type", [](b2_cache_desc &x) { x.row_dtype = B2_E4M3; });
  cache("16-bit pages", [](b2_cache_desc &x) { x.dtype = B2_F16; });
  cache("heads", [](b2_cache_desc &x) { x.heads = 0; });
  cache("q_heads", [](b2_cache_desc &x) { x.q_heads = 3; });
  cache("q_heads", [](b2_cache_desc &x) { x.q_heads = 0; });
  cache("head_dim", [](b2_cache_desc &x) { x.head_dim = 72; });
  cache("head_dim", [](b2_cache_desc &x) { x.head_dim = 144; });
  cache("page_size", [](b2_cache_desc &x) { x.page_size = 0; });
  cache("n_pages", [](b2_cache_desc &x) { x.n_pages = 0x80000000u; });
  cache("null pages", [](b2_cache_desc &x) { x.v_pages = nullptr; });
  cache("16-byte aligned", [&](b2_cache_desc &x) { x.k_pages = mem + 8; });
  cache("multiples of 16 bytes", [](b2_cache_desc &x) { x.slot_stride = 136; });
  cache("not negative", [](b2_cache_desc &x) { x.page_stride = -2048; });
  cache("smaller than a row", [](b2_cache_desc &x) { x.head_stride = 48; });
  cache("need scales", [](b2_cache_desc &x) { x.v_scales = nullptr; });
  cache("4-byte aligned", [&](b2_cache_desc &x) { x.k_scales = reinterpret_cast<float *>(mem + 2); });
  cache("share a place", [](b2_cache_desc &x) { x.scale_slot_stride = 0; });
  cache("must not be negative", [](b2_cache_desc &x) { x.scale_head_stride = -1; });

  b2_batch b = {};
  b.n_seqs = 2; b.n_rows = 5; b.max_pages = 3; b.pages_stride = 3; b.row_start = b.length = b.pages = mem;
  Fine("batch", b2::CheckBatch(&b));
  Refused("no batch", b2::CheckBatch(nullptr), "null");
  auto batch = [&](const char *part, auto change) { b2_batch x = b; change(x); Refused(part, b2::CheckBatch(&x), part); };
  batch("n_seqs", [](b2_batch &x) { x.n_seqs = (1u << 20) + 1u; });
  batch("n_rows", [](b2_batch &x) { x.n_rows = 0x80000000u; });
  batch("null row_start", [](b2_batch &x) { x.length = nullptr; });
  batch("null row_start", [](b2_batch &x) { x.pages = nullptr; });
  batch("4-byte aligned", [&](b2_batch &x) { x.row_start = mem + 1; });
  batch("pages_stride", [](b2_batch &x) { x.pages_stride = 2; });
  batch("pages_stride", [](b2_batch &x) { x.n_seqs = 1; x.pages_stride = -1; });
  b2_batch none = {};
  Fine("batch of nothing", b2::CheckBatch(&none));

  alignas(16) char other[64];
  const b2_rows q = {mem, 256, 64}, o = {other, 256, 64};
  auto attend = [&](const b2_rows *qq, const b2_rows *oo, float scale, int causal, uint32_t window, const void *lse) { return b2::CheckAttend(c, &b, qq, oo, scale, causal, window, lse); };
  Fine("attend", attend(&q, &o, 0.125f, 1, 0, nullptr));
  Fine("attend, not causal", attend(&q, &o, 0.125f, 0, 0, mem));
  Refused("no q", attend(nullptr, &o, 0.125f, 1, 0, nullptr), "q: null");
  const b2_rows odd = {other + 1, 256, 64}, far = {other, (int64_t(1) << 41), 64}, nothing = {nullptr, 256, 64};
  Refused("no out", attend(&q, &nothing, 0.125f, 1, 0, nullptr), "out: null");
  Refused("odd out", attend(&q, &odd, 0.125f, 1, 0, nullptr), "out: not aligned");
  Refused("far out", attend(&q, &far, 0.125f, 1, 0, nullptr), "out: stride");
  Refused("out over q", attend(&q, &q, 0.125f, 1, 0, nullptr), "over q");
  for (float s : {0.0f, -1.0f, nan, inf, 3e38f}) Refused("scale", attend(&q, &o, s, 1, 0, nullptr), "scale");
  Refused("window", attend(&q, &o, 0.125f, 0, 5, nullptr), "needs causal");
  Refused("window", attend(&q, &o, 0.125f, 1, 0x80000000u, nullptr), "window");
  Refused("lse", attend(&q, &o, 0.125f, 1, 0, mem + 2), "lse");
  b2_batch many = b;
  many.n_rows = 0x40000000u;                              // (two heads to a cache head)
  Refused("2^31 rows x heads", b2::CheckAttend(c, &many, &q, &o, 0.125f, 1, 0, nullptr), "below 2^31");
  many.max_rows = 1000;
  Fine("of which a sequence has few", b2::CheckAttend(c, &many, &q, &o, 0.125f, 1, 0, nullptr));
  b2_cache_desc f32 = c;
  f32.row_dtype = B2_F32;
  Refused("f32 rows", b2::CheckAttend(f32, &b, &q, &o, 0.125f, 1, 0, nullptr), "f32 rows");
}

int main() {
  Divisions();
  Sequences();
  Refusals();
  return wrong ? 1 : 0;
}
