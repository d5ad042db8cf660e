// Attention of many rows of each sequence over the paged cache: chunks of prompts.
//
// The rows of a sequence times the query heads that share a cache head, row by row, are cut into tiles of 256: two slots of 128 rows,
// each a tensor-core tile, so that a block of 128 keys is fetched once for all of them. Per slot and block, with the scores in
// tensor memory:  S = Q K^T (128 x 128 x hd),  p = 2^(s scale log2 e - m) over the running maximum m,  O += P V (128 x hd x 128).
// O stays in tensor memory; it is rescaled in place only when a row's maximum grew by more than 2^8 since the one in use was set
// (p then stays below 256 and the result is mathematically the same). P overwrites the scores it came from. Two threads that have a row's maximum
// between them tell each other 16 bits that are not below theirs, and all of them only when a row of their warps may move: a maximum of thousands is off by
// dozens in 16 bits, and weights of f16 that are 2^-24 of what they should be are gone.
//
// Roles of a CTA: a warp to issue the products, four warps (8-bit pages: eight) that fill the ring of K and V blocks (and Q), eight softmax
// warps for each slot, two threads to a row with half of the keys each (one thread to a row: as fast with 128 values a head, 5 % slower
// with 64). The products of one slot run while the other slot's softmax does:
//   issue:    O0 += P0 V(j), S0 = Q0 K(j+1), O1 += P1 V(j), S1 = Q1 K(j+1), ..
// A product waits for P of its slot; a softmax for S, whose arrival says that everything issued before is done as well.
// The ring holds blocks in the 128-byte-swizzled layout that the tensor cores read, filled page by page: pages have any size, so a row
// of the cache is found by itself (one page number a row, looked up a block ahead).
// 8-bit pages: codes become f16 on their way into the ring. K's exactly, its scales go onto the scores, in f32; q is scaled by a power of two
// for each row to fit f16. V's, for bf16 rows, times their key's scale relative to a power of two above the scales of 16 keys side by side
// (rounded to 2^-11 of themselves, as the weights are), the power goes onto the weights; f16 rows' results are rounded no coarser than that
// themselves, so for them V is exact, too, and its scales go onto the weights before those are rounded. (A warp that reads 64 scales waits
// for 8 KB of them: 871 us instead of 782 for 2048 rows behind 14336 of 32 heads of 128 values, in a graph.) The codes of a block ahead wait in
// shared memory as they are, copied asynchronously (in registers: 1045 us).
//
// Work: one CTA to an SM. The tiles of the batch in a row, sequence by sequence and head by head, each weighed by the keys it sees and something for its
// beginning and end, are dealt to the CTAs in equal runs, whatever their number and lengths; a run that ends inside a tile ends between
// two blocks of its keys, and a second launch joins the parts. The filling warps walk the run; the others read what they need of a tile
// from shared memory. The ring runs on from tile to tile.
//
// Bound: the tensor cores, under the power cap. 2048 rows behind 14336 of 32 heads of 128 values, bf16: 474 us in a graph with L2 warm, 78 % of
// the rate that a large product sustains (without exponentials and copies it would be 356); 555 us one call after another with L2 cold, 67 %.
#include <type_traits>

#include "attend_common.cuh"
#include "tc_common.cuh"

namespace b2 {
namespace {

constexpr uint32_t kCkRows = 128, kCkKeys = 128;          // rows of a slot, keys of a block
constexpr uint32_t kSoftWarps = 16;
// What goes by the pages' type: filling warps (codes are converted by them), registers of a thread. Launched with as many as the threads divide the SM's by, the
// softmax warps take what the others give up; three of the last four warps only hold registers back.
template <bool Q8>
struct ChunkWarps {
  static constexpr uint32_t kLoad = Q8 ? 8 : 4, kThreads = (kSoftWarps + kLoad + 4) * 32;
  static constexpr int kLaunch = Q8 ? 72 : 80, kSoft = Q8 ? 80 : 96, kFill = Q8 ? 72 : 56, kIssue = 40;
  static_assert(4 * kSoft + static_cast<int>(kLoad) / 4 * kFill + kIssue == (5 + static_cast<int>(kLoad) / 4) * kLaunch, "the launch's registers");
  static_assert(kSoft > kLaunch && kFill <= kLaunch && kIssue < kLaunch, "raised or lowered (the other way round is no instruction)");
};
constexpr uint32_t kCkCols = 512;                         // tensor memory: S0, S1 (128 columns each), O0, O1
constexpr float kGrow = 8.0f;                             // log2 of the growth of a row maximum that forces a rescale
constexpr float kCkPScale = 64.0f;                        // 8-bit pages: p (below 2^8) on the largest scale stays below 2^14
// V's codes (at most 448) times their scale over a power above it are as large as f16 holds; with scales down to 2^-15 of the power, normal codes stay
// normal. What a power is above 16 keys for loses no bits as long as their scales are within that: no more than 2^14 (by their exponents) apart.
constexpr uint32_t kCkVLog = 7, kCkApart = 14;

template <bool BF, bool Q8, int HD>
struct ChunkShape {
  static constexpr uint32_t kHalf = 128u * 128u;          // 128 rows of 64 values
  static constexpr uint32_t kBlock = kHalf * (HD / 64);   // Q of a slot, K or V of a block
  static constexpr bool kExactV = Q8 && !BF;              // V's scales go onto the weights
  static constexpr uint32_t kStages = HD == 64 ? 8 : kExactV ? 3 : Q8 ? 4 : 5;
  // Q, the ring, codes of K and V of a block, scales of two blocks, what the softmax warps tell each other
  static constexpr uint32_t kQ = 0, kRing = 2 * kBlock, kCodes = kRing + kStages * kBlock, kScales = kCodes + (Q8 ? kBlock : 0u);
  static constexpr uint32_t kTops = kScales + (kExactV ? 2048u : Q8 ? 1024u : 0u), kShared = kTops + 1024u;
};
// A tile's part that a CTA works on: packed rows [r0, r0 + rows) of a sequence (row x group + head), blocks [b0, b1) of the `blocks` of keys from
// keys.lo that any of them sees.
struct Tile {
  uint32_t seq, head, r0, rows, blocks, b0, b1, part;     // part: 0 whole, else 1 + where its results go
  Seq s;
  Span keys;
};
// What a CTA tells the launch that joins: the tile whose first blocks end its run (no rows: none), and its blocks of the tile in which the run
// begins. Behind the parts in the scratch.
struct Join {
  Tile tile;
  uint32_t b0, b1;
};
constexpr size_t kPartFloats = kChunkRows * (128u + 2u);  // (room for a part of 128 values a row)
__device__ __forceinline__ Join *joins_of(const AttendArgs &a, uint32_t most) { return reinterpret_cast<Join *>(a.part + most * 2u * kPartFloats); }
struct ChunkShared {
  uint64_t q_full, q_free, full[8], empty[8], s_full[2], p_full[2], pv_done[2], scales_free[2][2];
  uint32_t tmem, failed;
  unsigned long long budget;                              // ns that a wait may take without a sign of life
  unsigned long long alive;                               // when a warp last said that it is working rows out again
  alignas(16) float v_ref[2][8];                          // 8-bit pages: powers of two above V's scales of two blocks, 16 keys each; negative: scales far apart
  // Keys of a block whose pages do not exist, a bit each; a block is filled at most four ahead of the one that the softmax warps are at.
  uint32_t absent[8][kCkKeys / 32u];
  Tile tile;                                              // no rows: the end
  union {
    unsigned long long find[30];                          // (before any row is looked at)
    int8_t q_exp[256];                                    // 8-bit pages: each row of q was scaled by 2^e
  };
};
template <bool BF, bool Q8, int HD>
constexpr uint32_t ChunkSmem() { return ChunkShape<BF, Q8, HD>::kShared + ((sizeof(ChunkShared) + 15u) & ~15u); }
constexpr bool ChunkFits(uint32_t bytes) { return bytes <= 227u * 1024u; }
static_assert(ChunkFits(ChunkSmem<true, false, 128>()) && ChunkFits(ChunkSmem<true, true, 128>()) && ChunkFits(ChunkSmem<false, true, 128>()) &&
                  ChunkFits(ChunkSmem<false, true, 64>()), "shared memory of an SM");

// Waits of limited time (as in tc_common.cuh): they end without success when another role has, or when the budget has gone by both since they began and
// since a warp last said that it works rows out again, which may take long.
__device__ __forceinline__ bool stuck(ChunkShared *S, unsigned long long t0) {
  const unsigned long long seen = *const_cast<volatile unsigned long long *>(&S->alive), now = globaltimer_ns();
  return now - max(t0, min(seen, now)) >= S->budget;
}
__device__ __forceinline__ bool wait_for(ChunkShared *S, uint64_t *bar, uint32_t parity) {
  if (mbar_try_wait_parity(bar, parity)) return true;
  volatile uint32_t *failed = &S->failed;
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
    if (*failed) return false;
    if (stuck(S, t0)) { *failed = 1u; return false; }
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait_parity(bar, parity)) return true;
  }
}
static __device__ __noinline__ bool wait_for_away(ChunkShared *S, uint64_t *bar, uint32_t parity) { return wait_for(S, bar, parity); }
// (a whole warp, in step)
__device__ __forceinline__ bool wait_together(ChunkShared *S, uint64_t *bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_try_wait_parity(bar, parity))) return true;
  volatile uint32_t *failed = &S->failed;
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
    if (__any_sync(0xffffffffu, *failed != 0u || stuck(S, t0))) {
      *failed = 1u;
      return false;
    }
    for (int i = 0; i < 32; ++i)
      if (__all_sync(0xffffffffu, mbar_try_wait_parity(bar, parity))) return true;
  }
}

// ---- how the work is dealt ----
typedef unsigned long long u64;
// Weights of a sequence's tiles (of one head): tile t weighs base + slope (t + 1), the last one less by `short_by`; in keys x group, and kTileCost blocks
// for what a tile costs beside its blocks.
constexpr uint32_t kTileCost = 3;
struct Weights {
  uint32_t tiles;
  u64 base, slope, short_by;
  __device__ __forceinline__ u64 before(u64 t) const { return t * base + slope * (t * (t + 1ull) / 2ull); }
  __device__ __forceinline__ u64 all() const { return tiles ? before(tiles) - short_by : 0ull; }
};
__device__ __forceinline__ Weights weights_of(const AttendArgs &a, const Seq &s) {
  Weights w;
  const u64 rows = static_cast<u64>(s.n) * a.group;
  w.tiles = static_cast<uint32_t>((rows + kChunkRows - 1u) / kChunkRows);
  const u64 past = s.len > s.n ? static_cast<u64>(s.len - s.n) : 0ull;
  u64 keys = static_cast<u64>(s.len);
  w.slope = 0ull;
  w.short_by = 0ull;
  if (a.causal && a.window) {
    keys = min(keys, static_cast<u64>(a.window) + kChunkRows / a.group);
  } else if (a.causal) {
    keys = past;
    w.slope = kChunkRows;
    w.short_by = w.tiles * static_cast<u64>(kChunkRows) - rows;
  }
  w.base = (keys + kTileCost * kCkKeys) * a.group;
  return w;
}
// The whole batch: weight of everything, CTAs that share it (a few blocks at least for each).
__device__ __forceinline__ u64 units_of_seq(const AttendArgs &a, uint64_t cap, uint32_t i) { return weights_of(a, load_seq(a.b, cap, i)).all() * a.c.heads; }
__device__ __forceinline__ uint32_t ctas_of(const AttendArgs &a, u64 all, uint32_t most) {
  const u64 n = all / (static_cast<u64>(kTileCost + 2u) * kCkKeys * a.group);
  return n < 1ull ? 1u : n > most ? most : static_cast<uint32_t>(n);
}
struct Runs {
  u64 each;
  uint32_t rest, ctas;
  __device__ __forceinline__ Runs(u64 all, uint32_t n) : each(all / n), rest(static_cast<uint32_t>(all - all / n * n)), ctas(n) {}
  __device__ __forceinline__ u64 begin(uint32_t cta) const { return each * cta + rest * cta / ctas; }     // (rest and cta are below the SMs)
};

// A place in the row of tiles.
struct Walk {
  uint32_t seq, head, index;
  Seq s;
  Weights w;
  u64 at;                                                 // weight before the tile
  __device__ __forceinline__ u64 weight() const { return w.base + w.slope * (index + 1ull) - (index + 1u == w.tiles ? w.short_by : 0ull); }
  // to the tile that holds unit x, of sequence `seq` whose units begin at x0
  __device__ __forceinline__ void seek(const AttendArgs &a, uint64_t cap, uint32_t b, u64 x0, u64 x) {
    seq = b;
    s = load_seq(a.b, cap, b);
    w = weights_of(a, s);
    const u64 one = w.all();
    head = static_cast<uint32_t>((x - x0) / one);
    at = x0 + head * one;
    uint32_t lo = 0, hi = w.tiles;                        // before(lo) <= x - at < before(hi)
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) / 2u;
      if (w.before(mid) <= x - at) lo = mid;
      else hi = mid;
    }
    index = lo;
    at += w.before(lo);
  }
  __device__ __forceinline__ bool next(const AttendArgs &a, uint64_t cap) {
    at += weight();
    if (++index < w.tiles) return true;
    index = 0;
    if (++head < a.c.heads) return true;
    head = 0;
    do {
      if (++seq >= a.b.n_seqs) return false;
      s = load_seq(a.b, cap, seq);
      w = weights_of(a, s);
    } while (w.tiles == 0u);
    return true;
  }
  // the tile's blocks that a run over units [x, y) has
  __device__ __forceinline__ void tile(const AttendArgs &a, u64 x, u64 y, Tile &t) const {
    t.seq = seq;
    t.head = head;
    t.s = s;
    t.r0 = index * kChunkRows;
    t.rows = min(t.r0 + kChunkRows, static_cast<uint32_t>(s.n) * a.group) - t.r0;
    t.keys = SeenByRows(s, static_cast<int32_t>(t.r0 / a.group), static_cast<int32_t>((t.r0 + t.rows - 1u) / a.group) + 1, a.causal, a.window);
    t.blocks = (static_cast<uint32_t>(t.keys.hi - t.keys.lo) + kCkKeys - 1u) / kCkKeys;
    t.b0 = block_at(t.blocks, x);
    t.b1 = block_at(t.blocks, y);
  }
  // the block at which a run that begins at unit x begins
  __device__ __forceinline__ uint32_t block_at(uint32_t blocks, u64 x) const {
    if (x <= at) return 0u;
    const u64 all = weight();
    return x - at >= all ? blocks : static_cast<uint32_t>((x - at) * blocks / all);
  }
};

__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {      // 16-byte chunk of a row of HD values
  return (chunk >> 3) * (128u * 128u) + row * 128u + (((chunk & 7u) ^ (row & 7u)) << 4);
}

// Rows that see nothing of the cache.
__device__ __forceinline__ void clear_rows(const AttendArgs &a, const Tile &t, uint32_t thread, uint32_t threads) {
  for (uint32_t i = thread; i < t.rows * a.c.hd; i += threads) {
    const uint32_t r = i / a.c.hd, d = i - r * a.c.hd, pr = t.r0 + r, tok = a.by_group.quot(pr), h = t.head * a.group + (pr - tok * a.group);
    const int32_t row = t.s.first + static_cast<int32_t>(tok);
    store_row_value(row_at(a.o, row, h) + 2u * d, 0.0f, a.bf16 != 0u);
    if (d == 0u && a.lse) a.lse[static_cast<int64_t>(row) * a.q_heads + h] = -INFINITY;
  }
}

// ---- the filling warps ----------------------------------------------------------------------
// Rows of q into shared memory, a 16-byte chunk to a thread. As they are they come by asynchronous copies (still under way on return).
template <bool BF, bool Q8, int HD>
static __device__ __forceinline__ void load_q(const AttendArgs &a, const Tile &t, uint32_t tid, uint32_t base, int8_t *q_exp) {
  using Sh = ChunkShape<BF, Q8, HD>;
  constexpr uint32_t QL = HD / 8, AT = ChunkWarps<Q8>::kLoad * 32u / QL;      // threads to a row, rows at once
  const bool vec = ((reinterpret_cast<uintptr_t>(a.q.p) & 15u) | ((a.q.row | a.q.head) & 7)) == 0;
  const uint32_t c = tid % QL, r0 = tid / QL, rows = t.rows > kCkRows ? 256u : 128u;
  const bool in_hd = c * 8u < a.c.hd;
  auto place = [&](uint32_t r) {
    const uint32_t pr = t.r0 + r, tok = a.by_group.quot(pr);
    return row_at(a.q, t.s.first + static_cast<int32_t>(tok), t.head * a.group + (pr - tok * a.group)) + 16u * c;
  };
  auto chunk = [&](uint32_t r) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < t.rows && in_hd) {
      const uint8_t *p = place(r);
      if (vec) {
        v = *reinterpret_cast<const uint4 *>(p);
      } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
        v = make_uint4(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16), h[4] | (static_cast<uint32_t>(h[5]) << 16),
                       h[6] | (static_cast<uint32_t>(h[7]) << 16));
      }
    }
    return v;
  };
  auto dst = [&](uint32_t r) { return base + Sh::kQ + (r >> 7) * Sh::kBlock + swizzled(r & 127u, c); };
  if (Q8 && BF) {
#pragma unroll 1
    for (uint32_t r = r0; r < rows; r += 4u * AT) {
      uint4 v[4];
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k) v[k] = chunk(r + k * AT);
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t ww[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(ww[i] << 16)), fabsf(__uint_as_float(ww[i] & 0xffff0000u))));
#pragma unroll
        for (uint32_t o = QL / 2u; o > 0u; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int ex = static_cast<int>(__float_as_uint(top) >> 23);
        const int e = ex == 0 || ex == 255 ? 0 : min(100, 127 + 14 - ex);      // (-113 and more)
        const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        if (c == 0u) q_exp[r + k * AT] = static_cast<int8_t>(e);
        auto h2 = [&](uint32_t x) { return cvt_f16x2(__uint_as_float(x & 0xffff0000u) * up, __uint_as_float(x << 16) * up); };
        sts_v4(dst(r + k * AT), make_uint4(h2(v[k].x), h2(v[k].y), h2(v[k].z), h2(v[k].w)));
      }
    }
  } else if (vec) {
#pragma unroll 4
    for (uint32_t r = r0; r < rows; r += AT) {
      const bool has = r < t.rows && in_hd;
      cp_async_16_zfill(dst(r), has ? place(r) : a.q.p, has ? 16u : 0u);
    }
  } else {
#pragma unroll 1
    for (uint32_t r = r0; r < rows; r += AT) sts_v4(dst(r), chunk(r));
  }
}

template <bool BF, bool Q8, int HD>
static __device__ __forceinline__ void chunk_load(const AttendArgs &a, Walk &wk, u64 x0, u64 x1, uint8_t *sm, ChunkShared *S) {
  using Sh = ChunkShape<BF, Q8, HD>;
  constexpr uint32_t NS = Sh::kStages;
  const uint64_t cap = capacity_of(a.c, a.b);
  const uint32_t tid = threadIdx.x - kSoftWarps * 32u, lane = tid & 31u, w = tid >> 5;
  const uint32_t base = smem_addr(sm);
  uint32_t it = 0;                                        // blocks filled so far: K, V, K, V, ..
  uint32_t used[2][2] = {{0u, 0u}, {0u, 0u}};             // 8-bit pages: how often each slot has used each place for scales
  Tile t = {};
  // the lane's key of a block: RW w + lane
  constexpr uint32_t RW = kCkKeys / ChunkWarps<Q8>::kLoad;
  int32_t page = -1;
  uint32_t slot = 0, entry = 0;
  bool live = false;
  auto look_ahead = [&](uint32_t j) {
    const int32_t p = t.keys.lo + static_cast<int32_t>(j * kCkKeys + RW * w + lane);
    live = j < t.b1 && p < t.keys.hi && lane < RW;
    if (live) {
      entry = a.c.by_page.quot(static_cast<uint32_t>(p));
      slot = static_cast<uint32_t>(p) - entry * a.c.page_size;
      page = __ldg(a.b.pages + static_cast<int64_t>(t.seq) * a.b.pages_stride + entry);
    }
  };
  // (the wait itself: 8-bit pages out of line, where the loop has the registers and not the code: 782 and 870 us for 796 and 908; 16-bit pages in line: 479 us
  // for 596)
  auto ready = [&](uint64_t *bar, uint32_t parity) {
    if constexpr (Q8) return mbar_try_wait_parity(bar, parity) || wait_for_away(S, bar, parity);
    else return wait_for(S, bar, parity);
  };
  // ---- K and V ----
  uint32_t absent = 0u;
  auto place = [&](int64_t &off, int64_t &soff) -> uint32_t {       // the lane's key; which lanes of the warp have one, and which have one without a page
    const bool lost = live && static_cast<uint32_t>(page) >= a.c.n_pages, ok = live && !lost;
    if (lost) cache_fault(a.c.status, kStBadPage, t.seq, entry, static_cast<uint32_t>(page));
    absent = __ballot_sync(0xffffffffu, lost);
    off = ok ? page * a.c.page_bytes + slot * a.c.slot_bytes + t.head * a.c.head_bytes : 0;
    soff = ok && Q8 ? page * a.c.s_page + slot * a.c.s_slot + t.head * a.c.s_head : 0;
    return __ballot_sync(0xffffffffu, ok);
  };
  auto say_absent = [&](uint32_t i) {                     // (with K of a block, item i of the ring)
    uint32_t *const to = S->absent[(i >> 1) & 7u];
    if (lane == 0u) {
      if (Q8) reinterpret_cast<uint16_t *>(to)[w] = static_cast<uint16_t>(absent);
      else to[w] = absent;
    }
  };
  auto room = [&](uint32_t i) { return ready(&S->empty[i % NS], ((i / NS) & 1u) ^ 1u); };
  auto done = [&](uint32_t i) {
    fence_proxy_async_smem();
    mbar_arrive(&S->full[i % NS]);
  };
  bool ok = true;
  constexpr uint32_t CH = Q8 ? HD / 16 : HD / 8, AT = 32u / CH, N = RW / AT;     // 16-byte chunks of a row; rows at once; loads of a thread
  const uint32_t sub = lane % CH, r1 = lane / CH;
  const bool in_hd = sub * 16u < a.c.hd * (Q8 ? 1u : 2u);
  auto copy = [&](const uint8_t *pages, uint32_t i, int64_t off, uint32_t mask) {
    const uint32_t dst = base + Sh::kRing + (i % NS) * Sh::kBlock;
    // (all 16 in a row are more code to fetch: 477 us instead of 464 in a graph; two at a time 479)
#pragma unroll 4
    for (uint32_t k = 0; k < N; ++k) {
      const uint32_t r = k * AT + r1;
      const int64_t o = __shfl_sync(0xffffffffu, off, r);
      const uint32_t bytes = ((mask >> r) & 1u) && in_hd ? 16u : 0u;
      cp_async_16_zfill(dst + swizzled(RW * w + r, sub), pages + (bytes ? o + 16 * sub : 0), bytes);
    }
    cp_async_commit();
  };
  // 8-bit pages: the thread's own 16 bytes of each of its rows wait as they are, K (v: 0) and V (1) of a block ahead
  const uint32_t codes = base + Sh::kCodes + tid * 16u;
  constexpr uint32_t kCodeRow = ChunkWarps<Q8>::kLoad * 512u;
  auto fetch = [&](const uint8_t *pages, uint32_t v, int64_t off, uint32_t mask) {
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
      const uint32_t r = k * AT + r1;
      const int64_t o = __shfl_sync(0xffffffffu, off, r);
      const uint32_t bytes = ((mask >> r) & 1u) && in_hd ? 16u : 0u;
      cp_async_16_zfill(codes + (v * N + k) * kCodeRow, pages + (bytes ? o + 16 * sub : 0), bytes);
    }
    cp_async_commit();
  };
  // the warp's keys of a block; V's times `mul`
  auto put = [&](uint32_t i, uint32_t v, float mul) {
    const uint32_t dst = base + Sh::kRing + (i % NS) * Sh::kBlock;
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
      const uint32_t r0 = k * AT + r1, r = RW * w + r0;
      const uint4 x = lds_v4(codes + (v * N + k) * kCodeRow);
      const uint32_t c[4] = {x.x, x.y, x.z, x.w};
      uint32_t h[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) h[q] = cvt_e4m3x2_f16x2(q & 1 ? c[q >> 1] >> 16 : c[q >> 1] & 0xffffu);
      if (v && !Sh::kExactV) {
        const float m = __shfl_sync(0xffffffffu, mul, r0);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[q]));
          h[q] = cvt_f16x2(f.y * m, f.x * m);
        }
      }
      // (the threads of a row's second 64 values the other way round: other banks)
      const uint4 h0 = make_uint4(h[0], h[1], h[2], h[3]), h1 = make_uint4(h[4], h[5], h[6], h[7]);
      const uint32_t late = HD == 128 ? sub >> 2 : 0u;
      sts_v4(dst + swizzled(r, 2u * sub + late), late ? h1 : h0);
      sts_v4(dst + swizzled(r, 2u * sub + (late ^ 1u)), late ? h0 : h1);
    }
  };
  uint32_t settled = 0;                                   // 16-bit pages: blocks that have landed and are said to have
  auto settle = [&](uint32_t n) {
    for (; settled < n; ++settled) done(settled);
  };
  uint32_t turn = 0;                                      // tiles so far
  for (bool more = true; ok; ++turn) {
    // ---- the next tile of the run that has blocks there ----
    bool found = false;
    while (more && !found) {
      more = wk.at < x1;
      if (!more) break;
      wk.tile(a, x0, x1, t);
      if (tid == 0u) {
        Join *const j = joins_of(a, gridDim.x) + blockIdx.x;
        if (wk.at < x0) { j->b0 = t.b0; j->b1 = t.b1; }
        if (t.b0 == 0u && t.b1 != 0u && t.b1 != t.blocks) j->tile = t;
      }
      // (rows that see no key are cleared by the CTA in whose run the tile begins)
      if (t.blocks == 0u) {
        if (wk.at >= x0) clear_rows(a, t, tid, ChunkWarps<Q8>::kLoad * 32u);
      }
      found = t.b0 < t.b1;
      t.part = t.b0 == 0u && t.b1 == t.blocks ? 0u : 1u + blockIdx.x * 2u + (t.b0 == 0u ? 1u : 0u);
      more = wk.next(a, cap);
    }
    if (!found) t.rows = 0u;
    const uint32_t slots = t.rows > kCkRows ? 2u : 1u;
    if (found) look_ahead(t.b0);
    bool q_there = false;
    auto q_to_all = [&]() {                               // Q and the tile, when the scores of the tile before are done
      q_there = true;
      ok = ok && __all_sync(0xffffffffu, ready(&S->q_free, (turn & 1u) ^ 1u));
      if (!ok) return;
      if (tid == 0u) S->tile = t;
      if (found) load_q<BF, Q8, HD>(a, t, tid, base, S->q_exp);
      cp_async_commit();
      cp_async_wait_all();
      fence_proxy_async_smem();
      mbar_arrive(&S->q_full);
    };
    if (!found) {
      if constexpr (!Q8) {
        cp_async_wait_all();
        settle(it);
      }
      q_to_all();
      break;
    }
    if constexpr (!Q8) {
      for (uint32_t j = t.b0; ok && j < t.b1; ++j) {
        int64_t off, soff;
        const uint32_t mask = place(off, soff);
        look_ahead(j + 1u);
#pragma unroll
        for (uint32_t v = 0; v < 2u; ++v) {
          // (a lane that gave up takes its warp with it)
          ok = __all_sync(0xffffffffu, ok && room(it));
          if (!ok) break;
          if (v == 0u) say_absent(it);
          copy(v ? a.c.v : a.c.k, it, off, mask);
          ++it;
          if (it > settled + 2u) { cp_async_wait<2>(); settle(it - 2u); }
        }
        if (ok && !q_there) {                             // (the products wait for these blocks and for Q)
          q_to_all();                                     // (waits for what is on the way)
          if (ok) settle(it);
        }
      }
    } else {
      int64_t off, soff;
      uint32_t mask = place(off, soff);
      fetch(a.c.k, 0u, off, mask);
      fetch(a.c.v, 1u, off, mask);
      float ksc = (mask >> lane) & 1u ? a.c.ks[soff] : 0.0f, vsc = (mask >> lane) & 1u ? a.c.vs[soff] : 0.0f;
      look_ahead(t.b0 + 1u);
      for (uint32_t j = t.b0; ok && j < t.b1; ++j) {
        const uint32_t buf = (it >> 1) & 1u;
        bool free = room(it);
        for (uint32_t s = 0; s < 2u; ++s) {
          uint32_t &n = used[s][buf];
          if (n) free = free && ready(&S->scales_free[s][buf], (n - 1u) & 1u);
          if (s < slots) ++n;
        }
        ok = __all_sync(0xffffffffu, free);
        if (!ok) break;
        say_absent(it);
        if (lane < RW) {
          float *const s = reinterpret_cast<float *>(sm + Sh::kScales + buf * 512u) + RW * w + lane;
          *s = ksc;
          if (Sh::kExactV) s[256] = vsc;
        }
        // V's power of two: above the scales of the warp's keys that are finite
        const uint32_t vb = lane < RW && (__float_as_uint(vsc) & 0x7fffffffu) < 0x7f800000u ? __float_as_uint(vsc) & 0x7fffffffu : 0u;
        const uint32_t most = __reduce_max_sync(0xffffffffu, vb), least = __reduce_min_sync(0xffffffffu, vb ? vb : 0x7f7fffffu);
        const float v_ref = power_above(__uint_as_float(most));
        if (lane == 0u) S->v_ref[buf][w] = most && (most >> 23) > (least >> 23) + kCkApart ? -v_ref : v_ref;
        cp_async_wait<1>();                               // (K's codes)
        put(it, 0u, 1.0f);
        done(it++);
        mask = place(off, soff);
        look_ahead(j + 2u);
        if (j + 1u < t.b1) fetch(a.c.k, 0u, off, mask);
        else cp_async_commit();                           // (nothing: zeros would meet the next tile's copies)
        ksc = (mask >> lane) & 1u ? a.c.ks[soff] : 0.0f;
        ok = __all_sync(0xffffffffu, room(it));
        if (!ok) break;
        cp_async_wait<1>();                               // (V's)
        put(it, 1u, vsc * __uint_as_float(((254u + kCkVLog) << 23) - __float_as_uint(v_ref)));
        done(it++);
        if (j + 1u < t.b1) fetch(a.c.v, 1u, off, mask);
        else cp_async_commit();
        vsc = (mask >> lane) & 1u ? a.c.vs[soff] : 0.0f;
        if (!q_there) q_to_all();
      }
    }
  }
  cp_async_wait_all();
  // the products have read what was filled last, and their arrivals on the ring's barriers are in
  if (ok && tid == 0u) {
    bool read = true;
    for (uint32_t k = 0; k < NS && read; ++k) read = ready(&S->empty[(it + k) % NS], (((it + k) / NS) & 1u) ^ 1u);
    ready(&S->q_free, (turn & 1u) ^ 1u);
  }
}

// ---- the issuing warp -----------------------------------------------------------------------
template <bool BF, bool Q8, int HD>
static __device__ __forceinline__ void chunk_products(uint8_t *sm, ChunkShared *S) {
  using Sh = ChunkShape<BF, Q8, HD>;
  constexpr uint32_t NS = Sh::kStages;
  const uint32_t base = smem_addr(sm), tmem = S->tmem;
  const uint32_t fmt = Q8 || !BF ? 0u : 1u;
  const uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kCkKeys >> 3) << 17) | ((kCkRows >> 4) << 24);
  const uint32_t idesc_o = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((static_cast<uint32_t>(HD) >> 3) << 17) | ((kCkRows >> 4) << 24);
  const uint64_t dq = tc_desc(base + Sh::kQ, 16u, 1024u), dk = tc_desc(base + Sh::kRing, 16u, 1024u), dv = tc_desc(base + Sh::kRing, Sh::kHalf, 1024u);
  const bool leader = elect_one_sync();
  auto scores = [&](uint32_t s, uint32_t st) {
    if (leader) {
#pragma unroll
      for (uint32_t k = 0; k < HD / 16u; ++k) {
        const uint64_t step = ((k >> 2) * Sh::kHalf + (k & 3u) * 32u) >> 4;
        tc_mma_f16(tmem + s * 128u, dq + ((s * Sh::kBlock) >> 4) + step, dk + ((st * Sh::kBlock) >> 4) + step, idesc_s, k ? 1u : 0u);
      }
      tc_commit(&S->s_full[s]);
    }
    __syncwarp();
  };
  auto values = [&](uint32_t s, uint32_t st, bool first) {
    if (leader) {
#pragma unroll
      for (uint32_t k = 0; k < kCkKeys / 16u; ++k)
        tc_mma_f16_ts(tmem + 256u + s * HD, tmem + s * 128u + 8u * k + (k >> 2) * 32u, dv + ((st * Sh::kBlock) >> 4) + k * (2048u >> 4), idesc_o, (!first || k) ? 1u : 0u);
    }
    __syncwarp();
  };
  auto release = [&](uint32_t st) {
    if (leader) tc_commit(&S->empty[st]);
    __syncwarp();
  };
  auto full = [&](uint32_t i) { return wait_together(S, &S->full[i % NS], (i / NS) & 1u); };
  uint32_t it = 0, n[2] = {0u, 0u};                       // the ring's blocks; each slot's blocks
  for (uint32_t turn = 0;; ++turn) {
    if (!wait_together(S, &S->q_full, turn & 1u)) return;
    const uint32_t rows = *const_cast<volatile uint32_t *>(&S->tile.rows);
    const uint32_t blocks = *const_cast<volatile uint32_t *>(&S->tile.b1) - *const_cast<volatile uint32_t *>(&S->tile.b0);
    if (rows == 0u) return;
    const uint32_t slots = rows > kCkRows ? 2u : 1u;
    if (!full(it)) return;
    tc_fence_after_sync();
    for (uint32_t s = 0; s < slots; ++s) scores(s, it % NS);
    release(it % NS);
    for (uint32_t j = 0; j < blocks; ++j, it += 2u) {
      const bool more = j + 1u < blocks;
      if (!more && leader) tc_commit(&S->q_free);         // (all of the tile's scores are on their way)
      __syncwarp();
      if (!full(it + 1u)) return;
      for (uint32_t s = 0; s < slots; ++s) {
        if (!wait_together(S, &S->p_full[s], n[s] & 1u)) return;
        ++n[s];
        tc_fence_after_sync();
        values(s, (it + 1u) % NS, j == 0u);
        if (s + 1u == slots) release((it + 1u) % NS);
        if (more) {
          if (s == 0u && !full(it + 2u)) return;
          tc_fence_after_sync();
          scores(s, (it + 2u) % NS);
          if (s + 1u == slots) release((it + 2u) % NS);
        } else {
          if (leader) tc_commit(&S->pv_done[s]);
          __syncwarp();
        }
      }
    }
  }
}

// ---- the softmax warps ----------------------------------------------------------------------
// The largest of three; a NaN wins.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The bits below bit n (none below 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int32_t n) { return static_cast<uint32_t>((1ull << max(0, min(32, n))) - 1ull); }
constexpr uint16_t kLeft = 0xffffu;
// x as the next bf16 that is not below it (its bits).
__device__ __forceinline__ uint32_t rounded_up(float x) {
  const uint32_t u = __float_as_uint(x);
  return (x > 0.0f ? u + 0xffffu : u) >> 16;              // (NaN and what is below 0: cut off)
}
// and x again, from that and its lower half.
__device__ __forceinline__ float from_halves(uint32_t up, uint32_t low) {
  return __uint_as_float((up << 16 | low) - (low != 0u && !(up & 0x8000u) ? 0x10000u : 0u));
}
template <bool BF, bool Q8, int HD>
static __device__ __forceinline__ void chunk_rows(const AttendArgs &a, uint8_t *sm, ChunkShared *S) {
  using Sh = ChunkShape<BF, Q8, HD>;
  const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31u, s = w >> 3, half = (w >> 2) & 1u, q4 = w & 3u;
  const uint32_t r = s * kCkRows + 32u * q4 + lane;       // the thread's row, of whose keys it has columns 64 half .. + 63
  const uint32_t row_addr = S->tmem + ((32u * q4) << 16), s_addr = row_addr + s * 128u, o_addr = row_addr + 256u + s * HD + half * (HD / 2);
  const int pair = 1 + static_cast<int>(s * 4u + q4);     // the two warps of 32 rows
  uint16_t *top_s = reinterpret_cast<uint16_t *>(sm + Sh::kTops) + s * 256u + 32u * q4 + lane;      // [slot][half][row]
  float *sum_s = reinterpret_cast<float *>(sm + Sh::kTops + s * 512u + (lane >> 4) * 256u + 64u * q4) + (lane & 15u);      // (in the same two warps' bytes)
  uint32_t g = 0, n = 0, mine = 0;                        // blocks of all tiles; the slot's blocks and tiles
  // A warp whose wait ran out meets the other of its pair once more, which may have got through: at the exchange of the maxima, where kLeft (no NaN that a
  // maximum gives) tells it to leave as well, or at its own end.
  auto leave = [&]() {
    top_s[half * 128u] = kLeft;
    bar_sync(pair, 64);
  };
#pragma unroll 1
  for (uint32_t turn = 0;; ++turn) {
    if (!wait_together(S, &S->q_full, turn & 1u)) return leave();
    const Tile &t = S->tile;
    const uint32_t rows = t.rows, seq = t.seq, part_at = t.part, r0 = t.r0, t_head = t.head;
    const int32_t keys_lo = t.keys.lo, keys_hi = t.keys.hi;
    const uint32_t b0 = t.b0, b1 = t.b1;
    const Seq ts = t.s;
    const int32_t e = Q8 && BF ? S->q_exp[r] : 0;
    __syncwarp();
    if (lane == 0u) mbar_arrive(&S->q_free);
    if (rows == 0u) return leave();
    if (s * kCkRows >= rows) {                            // the other slot's alone
      g += b1 - b0;
      continue;
    }
    const bool has = r < rows;
    const uint32_t pr = r0 + r, tok = a.by_group.quot(pr), head = t_head * a.group + (pr - tok * a.group);
    const Span sp = has ? SeenBy(ts, static_cast<int32_t>(tok), a.causal, a.window) : Span{0, 0};
    const float sl2 = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    float m_used = -INFINITY, l = 0.0f, v_ref = 0.0f;
    bool redo = false;
#pragma unroll 1
    for (uint32_t j = b0; j < b1; ++j, ++g, ++n) {
      if (!wait_together(S, &S->s_full[s], n & 1u)) return leave();
      tc_fence_after_sync();
      const int32_t j0 = keys_lo + static_cast<int32_t>(j * kCkKeys);
      const int32_t lo = sp.lo - j0, hi = sp.hi - j0;     // columns [lo, hi) of the block are seen
      const bool whole = __all_sync(0xffffffffu, lo <= 0 && hi >= static_cast<int32_t>(kCkKeys) && S->absent[g & 7u][lane & 3u] == 0u);
      // 1: the row's maximum. The scores are read twice: half of a row's in registers at once leave too few for the rest
      const int32_t lo_h = lo - 64 * static_cast<int32_t>(half), hi_h = hi - 64 * static_cast<int32_t>(half);
      const float *ks = reinterpret_cast<const float *>(sm + Sh::kScales + (g & 1u) * 512u) + 64u * half;
      auto scores = [&](int c, uint32_t (&x)[32]) {
        __syncwarp();
        tc_ld32(s_addr + 64u * half + 32u * c, x);
        tc_wait_ld();
        if (Q8) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4 *>(ks + 32 * c + i);
            x[i] = __float_as_uint(__uint_as_float(x[i]) * k4.x); x[i + 1] = __float_as_uint(__uint_as_float(x[i + 1]) * k4.y);
            x[i + 2] = __float_as_uint(__uint_as_float(x[i + 2]) * k4.z); x[i + 3] = __float_as_uint(__uint_as_float(x[i + 3]) * k4.w);
          }
        }
        if (!whole) {
          const uint32_t hide = S->absent[g & 7u][2u * half + c] | below(lo_h - 32 * c) | ~below(hi_h - 32 * c);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((hide >> i) & 1u) x[i] = 0xff800000u;
        }
      };
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t x[32];
        scores(c, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) m4[i & 3] = max3_nan(m4[i & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 16]));
      }
      const float own = max3_nan(m4[0], m4[1], max3_nan(m4[2], m4[3], m4[2]));
      const uint32_t own_up = rounded_up(own);
      top_s[half * 128u] = static_cast<uint16_t>(own_up);
      bar_sync(pair, 64);
      const uint32_t other_up = top_s[(half ^ 1u) * 128u];
      float mx = max3_nan(__uint_as_float(own_up << 16), __uint_as_float(other_up << 16), -INFINITY) * sl2;
      bool grow = !(mx <= m_used + kGrow);                // (a NaN as well)
      float top = v_ref, vv[8];
      if (Q8) {
        const float4 va = *reinterpret_cast<const float4 *>(S->v_ref[g & 1u]), vb = *reinterpret_cast<const float4 *>(S->v_ref[g & 1u] + 4);
        vv[0] = va.x; vv[1] = va.y; vv[2] = va.z; vv[3] = va.w; vv[4] = vb.x; vv[5] = vb.y; vv[6] = vb.z; vv[7] = vb.w;
        if (whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(vv[k]));
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool seen = hi > 16 * k && lo < 16 * k + 16;
            top = seen ? fmaxf(top, fabsf(vv[k])) : top;
            // scales far apart, and some of the tile's keys not seen by the row: they may have set the power
            redo = redo || (seen && vv[k] < 0.0f && (lo > 16 * k || hi < min(16 * k + 16, keys_hi - j0)));
          }
        }
        grow = grow || top > v_ref;
      }
      // (the two warps agree: they have the same rows, and the same of all this)
      const bool move = __any_sync(0xffffffffu, grow);
      float alpha = 1.0f;
      if (move) {
        if (other_up == kLeft) return;                    // (all lanes)
        bar_sync(pair, 64);
        top_s[half * 128u] = static_cast<uint16_t>(__float_as_uint(own));
        bar_sync(pair, 64);
        mx = max3_nan(own, from_halves(other_up, top_s[(half ^ 1u) * 128u]), -INFINITY) * sl2;
        if (mx > m_used + kGrow) {
          alpha = m_used == -INFINITY ? 0.0f : fast_ex2(m_used - mx);
          l *= alpha;
          m_used = mx;
        }
        if (Q8 && top > v_ref) {
          alpha *= v_ref / top;                           // (a power of two, or 0 at first)
          v_ref = top;
        }
      }
      float v_mul[4] = {1.0f, 1.0f, 1.0f, 1.0f};          // of 16 columns each (exact V: the same for all, beside each one's scale)
      if (Q8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {                     // (columns that the row does not see may have a larger power)
          const float own = Sh::kExactV ? 1.0f : fabsf(half ? vv[4 + k] : vv[k]);
          v_mul[k] = v_ref > 0.0f ? own * __uint_as_float((254u << 23) - __float_as_uint(v_ref)) * kCkPScale : 0.0f;
          if (!Sh::kExactV) v_mul[k] = fminf(v_mul[k], kCkPScale);
        }
      }
      if (j > b0 && move) {                               // (these scores came after the products before them: O is at rest)
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < HD / 2; c0 += 16u) {
          uint32_t y[16];
          __syncwarp();
          tc_ld16(o_addr + c0, y);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
          tc_st16(o_addr + c0, y);
        }
      }
      // 2: the weights, over the scores
      const float neg = m_used == -INFINITY ? 0.0f : -m_used;
      const u64 sl2_2 = pack_f32x2(sl2, sl2), neg_2 = pack_f32x2(neg, neg);
      u64 sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t x[32], pk[16];
        scores(c, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float e0, e1;
          unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), sl2_2, neg_2), e0, e1);
          e0 = fast_ex2(e0);
          e1 = fast_ex2(e1);
          sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(e0, e1));
          if (Q8) {
            float f0 = v_mul[2 * c + (i >> 3)], f1 = f0;
            if (Sh::kExactV) {
              // (a scale that the row does not see may be anything)
              const float2 v2 = *reinterpret_cast<const float2 *>(ks + 256 + 32 * c + 2 * i);
              f0 *= whole || (32 * c + 2 * i >= lo_h && 32 * c + 2 * i < hi_h) ? v2.x : 0.0f;
              f1 *= whole || (32 * c + 2 * i + 1 >= lo_h && 32 * c + 2 * i + 1 < hi_h) ? v2.y : 0.0f;
            }
            e0 *= f0;
            e1 *= f1;
          }
          pk[i] = BF && !Q8 ? cvt_bf16x2(e1, e0) : cvt_f16x2(e1, e0);
        }
        __syncwarp();
        tc_st16(s_addr + 64u * half + 16u * c, pk);         // (over scores that were read)
      }
      tc_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0u) {
        mbar_arrive(&S->p_full[s]);
        if (Q8) mbar_arrive(&S->scales_free[s][g & 1u]);
      }
      float a0, a1;
      unpack_f32x2(add_f32x2(sum[0], sum[1]), a0, a1);
      l += a0 + a1;
    }
    // ---- the result: half of the row's values each ----
    bar_sync(pair, 64);                                   // (the other's maximum has been read)
    if (half) *sum_s = l;
    bar_sync(pair, 64);
    if (!half) {
      l += *sum_s;
      *sum_s = l;
    }
    bar_sync(pair, 64);
    if (half) l = *sum_s;
    bar_sync(pair, 64);                                   // (and the sum)
    if (!wait_together(S, &S->pv_done[s], mine & 1u)) return leave();
    ++mine;
    tc_fence_after_sync();
    const bool split = part_at != 0u;
    float *part = a.part + static_cast<size_t>(split ? part_at - 1u : 0u) * (kChunkRows * (HD + 2u));
    const bool none = m_used == -INFINITY && l == 0.0f;
    float mul = split ? 1.0f : none ? 0.0f : 1.0f / l;
    if (Q8) mul *= v_ref * (Sh::kExactV ? 1.0f / kCkPScale : 1.0f / (kCkPScale * (1u << kCkVLog)));
    if (redo && split) mul = __int_as_float(0x7fc00000);  // (for the launch that joins)
    const uint32_t d0 = half * (HD / 2);
    uint8_t *out = has ? row_at(a.o, ts.first + static_cast<int32_t>(tok), head) + 2u * d0 : a.o.p;
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15u) == 0u, wide = (reinterpret_cast<uintptr_t>(out) & 31u) == 0u;
    bool fine = true;
#pragma unroll 1
    for (uint32_t c0 = 0; c0 < HD / 2; c0 += 32u) {
      uint32_t x[32];
      __syncwarp();
      tc_ld32(o_addr + c0, x);
      tc_wait_ld();
      if (!has) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float v = __uint_as_float(x[i]) * mul;
        x[i] = __float_as_uint(v);
        fine = fine && isfinite(v);
      }
      if (split) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) stg_v8(part + r * HD + d0 + c0 + i, x + i);
        continue;
      }
      if (wide) {                                         // whole sectors: a row is 32-byte aligned, and so is its end
        uint32_t h[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) h[k] = BF ? cvt_bf16x2(__uint_as_float(x[2 * k + 1]), __uint_as_float(x[2 * k])) : cvt_f16x2(__uint_as_float(x[2 * k + 1]), __uint_as_float(x[2 * k]));
        if (d0 + c0 < a.c.hd) stg_v8(out + 2u * c0, h);
        if (d0 + c0 + 16u < a.c.hd) stg_v8(out + 2u * c0 + 32u, h + 8);
        continue;
      }
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        if (d0 + c0 + i >= a.c.hd) break;
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float u = __uint_as_float(x[i + 2 * k]), v = __uint_as_float(x[i + 2 * k + 1]);
          h[k] = BF ? cvt_bf16x2(v, u) : cvt_f16x2(v, u);
        }
        uint8_t *p = out + 2u * (c0 + i);
        if (vec) {
          *reinterpret_cast<uint4 *>(p) = make_uint4(h[0], h[1], h[2], h[3]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            reinterpret_cast<uint16_t *>(p)[2 * k] = static_cast<uint16_t>(h[k]);
            reinterpret_cast<uint16_t *>(p)[2 * k + 1] = static_cast<uint16_t>(h[k] >> 16);
          }
        }
      }
    }
    tc_fence_before_sync();
    if (has && split && !half) {
      part[kChunkRows * HD + r] = m_used;
      part[kChunkRows * HD + kChunkRows + r] = l;
    } else if (has && !split && !half && a.lse) {
      a.lse[static_cast<int64_t>(ts.first + static_cast<int32_t>(tok)) * a.q_heads + head] = (m_used + log2f(l)) * 0.69314718055994531f;
    }
    redo = has && !split && (redo || (!fine && isfinite(l) && (sp.lo > keys_lo || sp.hi < keys_hi)));      // (a sum that is not finite has met such a score: the result is right)
    for (uint32_t again = __ballot_sync(0xffffffffu, redo); again; again &= again - 1u) {      // (rows of this warp, one after another, its half of the values)
      const uint32_t k = __ffs(again) - 1u, q = r0 + s * kCkRows + 32u * q4 + k;
      __syncwarp();
      attend_row_alone(a, seq, ts, static_cast<int32_t>(q / a.group), t_head * a.group + q % a.group, d0, HD / 2, &S->alive);
    }
  }
}

template <bool BF, bool Q8, int HD>
__global__ void __launch_bounds__(ChunkWarps<Q8>::kThreads, 1) b2_attend_chunk(const __grid_constant__ AttendArgs a) {
  using Sh = ChunkShape<BF, Q8, HD>;
  constexpr uint32_t kLoadWarps = ChunkWarps<Q8>::kLoad, kCkThreads = ChunkWarps<Q8>::kThreads;
  extern __shared__ __align__(1024) uint8_t sm[];
  ChunkShared *S = reinterpret_cast<ChunkShared *>(sm + Sh::kShared);
  const uint32_t tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint64_t cap = capacity_of(a.c, a.b);
  if (blockIdx.x == 0u) {
    for (uint32_t i = tid; i < a.b.n_seqs; i += kCkThreads) {
      const Seq q = load_seq(a.b, cap, i);
      if (q.bad) cache_fault(a.c.status, kStBadBatch, i, static_cast<uint32_t>(q.bad), static_cast<uint32_t>(q.value));
    }
  }
  if (tid == 0u) {                                        // (what is there is of the call before)
    Join *const j = joins_of(a, gridDim.x) + blockIdx.x;
    j->tile.rows = 0u;
    j->b0 = j->b1 = 0u;
  }
  u64 all = 0ull;
  for (uint32_t i = tid; i < a.b.n_seqs; i += kCkThreads) all += units_of_seq(a, cap, i);
  all = warp_reduce(all, [](u64 x, u64 y) { return x + y; });
  if ((tid & 31u) == 0u) S->find[w] = all;
  __syncthreads();
  all = 0ull;
  for (uint32_t i = 0; i < kCkThreads / 32u; ++i) all += S->find[i];
  const uint32_t ctas = ctas_of(a, all, gridDim.x);
  if (all == 0ull || blockIdx.x >= ctas) return;
  const Runs runs(all, ctas);
  const u64 x0 = runs.begin(blockIdx.x), x1 = runs.begin(blockIdx.x + 1u);
  uint32_t seq;
  u64 before;
  if (!find_unit<kCkThreads>(a.b.n_seqs, x0, S->find, [&](uint32_t i) { return units_of_seq(a, cap, i); }, seq, before)) return;
  if (tid == 0u) {
    mbar_init(&S->q_full, kLoadWarps * 32u);
    mbar_init(&S->q_free, 1u + kSoftWarps);
    for (uint32_t i = 0; i < Sh::kStages; ++i) { mbar_init(&S->full[i], kLoadWarps * 32u); mbar_init(&S->empty[i], 1u); }
    for (uint32_t s = 0; s < 2u; ++s) {
      mbar_init(&S->s_full[s], 1u); mbar_init(&S->p_full[s], 8u); mbar_init(&S->pv_done[s], 1u);
      for (uint32_t i = 0; i < 2u; ++i) mbar_init(&S->scales_free[s][i], 8u);
    }
    S->failed = 0u;
    S->budget = a.wait_budget_ns;
    S->alive = 0ull;
    fence_mbar_init();
  }
  if (w == kSoftWarps + kLoadWarps) {
    __syncwarp();
    tmem_alloc(&S->tmem, kCkCols);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (w < kSoftWarps) {
    more_registers<ChunkWarps<Q8>::kSoft>();
    chunk_rows<BF, Q8, HD>(a, sm, S);
  } else if (w < kSoftWarps + kLoadWarps) {
    if constexpr (!Q8) fewer_registers<ChunkWarps<Q8>::kFill>();
    Walk wk;
    wk.seek(a, cap, seq, before, x0);
    chunk_load<BF, Q8, HD>(a, wk, x0, x1, sm, S);
  } else {
    fewer_registers<ChunkWarps<Q8>::kIssue>();
    if (w == kSoftWarps + kLoadWarps) chunk_products<BF, Q8, HD>(sm, S);
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  const bool gave_up = S->failed != 0u;
  if (gave_up) {                                          // products of other roles may still be landing: give them time
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 50000ull) nanosleep_ns(1000);
    if (tid == 0u) cache_fault(a.c.status, kStTcTimeout, seq, blockIdx.x, 0u);
  }
  if (w == kSoftWarps + kLoadWarps) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(S->tmem, kCkCols);
  }
}

// Tiles that lie in the runs of several CTAs (registers for two CTAs to an SM: with fewer the row's loop spills, 42 us instead of 40 for 128 rows behind
// 4000 keys): a warp to a row, the parts in their order. For each CTA whose run ends inside a tile that it began,
// a CTA of 32 rows at a time. (What to join was written down by the launch before: worked out here again, with 64-bit quotients in every warp, it
// was 37 us for 2048 rows behind 14336 of 32 heads of 128 values.)
constexpr uint32_t kJoinThreads = 256, kJoinRows = 32, kMostRuns = 1024;
template <int HD>
__global__ void __launch_bounds__(kJoinThreads, 2) b2_attend_join(const __grid_constant__ AttendArgs a, uint32_t most) {
  const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31u, begun = blockIdx.x / (kChunkRows / kJoinRows);
  const Join *const joins = joins_of(a, most);
  if (joins[begun].tile.rows <= (blockIdx.x % (kChunkRows / kJoinRows)) * kJoinRows) return;
  const Tile t = joins[begun].tile;
  constexpr uint32_t kPart = kChunkRows * (HD + 2u);
  __shared__ uint32_t part_s[kMostRuns], n_parts;
  if (w == 0u) {
    uint32_t n = 1u;
    if (lane == 0u) part_s[0] = begun * 2u + 1u;
    for (uint32_t c0 = begun + 1u; c0 < most; c0 += 32u) {
      const uint32_t c = c0 + lane, lo = c < most ? joins[c].b0 : 0u, hi = c < most ? joins[c].b1 : 0u;
      const uint32_t end = __ballot_sync(0xffffffffu, hi == t.blocks), upto = end ? 2u << (__ffs(end) - 1u) : 0u;      // (lanes up to the one with the last block)
      const bool has = lo < hi && (upto == 0u || ((upto - 1u) >> lane) & 1u);
      const uint32_t m = __ballot_sync(0xffffffffu, has);
      if (has) part_s[n + __popc(m & ((1u << lane) - 1u))] = c * 2u;
      n += __popc(m);
      if (end) break;
    }
    if (lane == 0u) n_parts = n;
  }
  __syncthreads();
  const uint32_t parts = n_parts, first = (blockIdx.x % (kChunkRows / kJoinRows)) * kJoinRows;
  // a warp's rows: first + w, + 8, + 16, + 24, side by side
  constexpr uint32_t kWarps = kJoinThreads / 32u, kRows = kJoinRows / kWarps, V = HD / 32;
  if (first + w >= t.rows) return;
  float mm[kRows], ll[kRows], o[kRows][V] = {};
#pragma unroll
  for (uint32_t q = 0; q < kRows; ++q) { mm[q] = -INFINITY; ll[q] = 0.0f; }
  auto row_of = [&](uint32_t q) { return min(first + w + q * kWarps, t.rows - 1u); };       // (rows that are not there: the last one again, not stored)
  for (uint32_t k = lane; k < parts; k += 32u) {
    const float *p = a.part + static_cast<size_t>(part_s[k]) * kPart + kChunkRows * HD;
#pragma unroll
    for (uint32_t q = 0; q < kRows; ++q) mm[q] = fmaxf(mm[q], p[row_of(q)]);
  }
#pragma unroll
  for (uint32_t q = 0; q < kRows; ++q) mm[q] = warp_reduce(mm[q], [](float u, float v) { return fmaxf(u, v); });
  for (uint32_t k0 = 0; k0 < parts; k0 += 32u) {
    float f[kRows] = {};
    if (k0 + lane < parts) {
      const float *p = a.part + static_cast<size_t>(part_s[k0 + lane]) * kPart + kChunkRows * HD;
#pragma unroll
      for (uint32_t q = 0; q < kRows; ++q) {
        const uint32_t r = row_of(q);
        f[q] = p[r] == mm[q] ? 1.0f : fast_ex2(p[r] - mm[q]);
        ll[q] += p[kChunkRows + r] * f[q];
      }
    }
    const uint32_t n = min(32u, parts - k0);
#pragma unroll 2
    for (uint32_t k = 0; k < n; ++k) {
      const float *p = a.part + static_cast<size_t>(part_s[k0 + k]) * kPart + lane * V;
#pragma unroll
      for (uint32_t q = 0; q < kRows; ++q) {
        const float fk = __shfl_sync(0xffffffffu, f[q], k);
        const Vec<float, V> x = *reinterpret_cast<const Vec<float, V> *>(p + row_of(q) * HD);
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) o[q][i] += x.v[i] * fk;
      }
    }
  }
#pragma unroll 1
  for (uint32_t q = 0; q < kRows; ++q) {
    const uint32_t r = first + w + q * kWarps;
    if (r >= t.rows) break;
    const uint32_t pr = t.r0 + r, tok = a.by_group.quot(pr), head = t.head * a.group + (pr - tok * a.group), d = lane * V;
    const int32_t row = t.s.first + static_cast<int32_t>(tok);
    float m = mm[0], sum = ll[0], x[V];
#pragma unroll
    for (uint32_t k = 0; k < kRows; ++k)
      if (k == q) {
        m = mm[k];
        sum = ll[k];
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) x[i] = o[k][i];
      }
    sum = warp_reduce(sum, [](float u, float v) { return u + v; });
    const float inv = m == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
    bool fine = true;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
      x[i] *= inv;
      fine = fine && isfinite(x[i]);
    }
    uint8_t *p = row_at(a.o, row, head) + 2u * d;
    if (d < a.c.hd) {
#pragma unroll
      for (uint32_t i = 0; i < V; i += 2) {
        const uint32_t h = a.bf16 ? cvt_bf16x2(x[i + 1], x[i]) : cvt_f16x2(x[i + 1], x[i]);
        if ((reinterpret_cast<uintptr_t>(p) & 3u) == 0u) {
          reinterpret_cast<uint32_t *>(p)[i / 2u] = h;
        } else {
          reinterpret_cast<uint16_t *>(p)[i] = static_cast<uint16_t>(h);
          reinterpret_cast<uint16_t *>(p)[i + 1] = static_cast<uint16_t>(h >> 16);
        }
      }
    }
    if (lane == 0u && a.lse) a.lse[static_cast<int64_t>(row) * a.q_heads + head] = (m + log2f(sum)) * 0.69314718055994531f;
    const Span sp = SeenBy(t.s, static_cast<int32_t>(tok), a.causal, a.window);
    if (__any_sync(0xffffffffu, !fine) && isfinite(sum) && (sp.lo > t.keys.lo || sp.hi < t.keys.hi)) {
      __syncwarp();
      attend_row_alone(a, t.seq, t.s, static_cast<int32_t>(tok), head, 0u, HD, nullptr);
    }
  }
}

template <bool BF, bool Q8, int HD>
int Launch(const AttendArgs &a, uint32_t sms, cudaStream_t stream) {
  if (sms > kMostRuns) sms = kMostRuns;
  b2_attend_chunk<BF, Q8, HD><<<sms, ChunkWarps<Q8>::kThreads, ChunkSmem<BF, Q8, HD>(), stream>>>(a);
  if (sms > 1u) b2_attend_join<HD><<<(sms - 1u) * (kChunkRows / kJoinRows), kJoinThreads, 0, stream>>>(a, sms);
  return static_cast<int>(cudaGetLastError());
}
template <bool BF, bool Q8, int HD>
cudaError_t Attr() {
  return cudaFuncSetAttribute(b2_attend_chunk<BF, Q8, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(ChunkSmem<BF, Q8, HD>()));
}

}  // namespace

int PrepareAttendChunk() {
  for (cudaError_t e : {Attr<true, false, 64>(), Attr<true, false, 128>(), Attr<false, false, 64>(), Attr<false, false, 128>(), Attr<true, true, 64>(), Attr<true, true, 128>(),
                        Attr<false, true, 64>(), Attr<false, true, 128>()})
    if (e != cudaSuccess) return static_cast<int>(e);
  return 0;
}
size_t AttendChunkPartialBytes(uint32_t sms) { return static_cast<size_t>(sms) * (2u * kPartFloats * sizeof(float) + sizeof(Join)); }

int LaunchAttendChunk(const AttendArgs &a, uint32_t sms, CUstream_st *stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool big = a.c.hd > 64u;
  if (a.e4m3) {
    if (a.bf16) return big ? Launch<true, true, 128>(a, sms, s) : Launch<true, true, 64>(a, sms, s);
    return big ? Launch<false, true, 128>(a, sms, s) : Launch<false, true, 64>(a, sms, s);
  }
  if (a.bf16) return big ? Launch<true, false, 128>(a, sms, s) : Launch<true, false, 64>(a, sms, s);
  return big ? Launch<false, false, 128>(a, sms, s) : Launch<false, false, 64>(a, sms, s);
}

}  // namespace b2
