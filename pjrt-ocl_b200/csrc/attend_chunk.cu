// Attention of many rows of each sequence over the paged cache: chunks of prompts.
//
// The rows of a sequence times the query heads that share a cache head, row by row, are cut into tiles of 256: two slots of 128 rows,
// each a tensor-core tile, so that a block of 128 keys is fetched once for all of them. Per slot and block, with the scores in
// tensor memory:  S = Q K^T (128 x 128 x hd),  p = 2^(s scale log2 e - m) over the running maximum m,  O += P V (128 x hd x 128).
// O stays in tensor memory; it is rescaled in place only when a row's maximum grew by more than 2^8 since the one in use was set
// (p then stays below 256 and the result is mathematically the same). P overwrites the scores it came from.
//
// Roles of a CTA: a warp to issue the products, four warps that fill the ring of K and V blocks (and Q), four softmax warps for each
// slot, one thread to a row. The products of one slot run while the other slot's softmax does:
//   issue:    O0 += P0 V(j), S0 = Q0 K(j+1), O1 += P1 V(j), S1 = Q1 K(j+1), ..
// A product waits for P of its slot; a softmax for S, whose arrival says that everything issued before is done as well.
// The ring holds blocks in the 128-byte-swizzled layout that the tensor cores read, filled page by page: pages have any size, so a row
// of the cache is found by itself (one page number a row, looked up a block ahead).
// 8-bit pages: codes become f16 on their way into the ring (exact), q is scaled by a power of two for each row to fit f16, a key's scale
// goes onto its scores and a value's onto p (see attend_step.cu).
//
// Few tiles: the keys of a tile are split over as many CTAs as there are SMs for, and a second launch joins their results.
#include "attend_common.cuh"
#include "tc_common.cuh"

namespace b2 {
namespace {

constexpr uint32_t kCkRows = 128, kCkKeys = 128;          // rows of a slot, keys of a block
constexpr uint32_t kSoftWarps = 8, kLoadWarps = 4, kCkThreads = (kSoftWarps + kLoadWarps + 4) * 32;     // (three of the last four warps only hold registers back)
// Registers of a thread: launched with 128 each, the softmax warps take those that the others give up (2 x 184 + 88 + 56 = 4 x 128).
constexpr int kSoftRegs = 184, kLoadRegs = 88, kIssueRegs = 56;
constexpr uint32_t kCkCols = 512;                         // tensor memory: S0, S1 (128 columns each), O0, O1
constexpr float kGrow = 8.0f;                             // log2 of the growth of a row maximum that forces a rescale
constexpr float kCkPScale = 64.0f;                        // 8-bit pages: p (below 2^8) on the largest scale stays below 2^14
constexpr unsigned long long kBudget = 2000000000ull;     // ns that a wait may take

template <int HD>
struct ChunkShape {
  static constexpr uint32_t kHalf = 128u * 128u;          // 128 rows of 64 values
  static constexpr uint32_t kBlock = kHalf * (HD / 64);   // Q of a slot, K or V of a block
  static constexpr uint32_t kStages = HD == 128 ? 5 : 8;
  static constexpr uint32_t kQ = 0, kRing = 2 * kBlock, kScales = kRing + kStages * kBlock, kShared = kScales + 2u * 1024u;      // scales of two blocks: K's, V's
};
struct ChunkShared {
  uint64_t q_full, full[8], empty[8], s_full[2], p_full[2], pv_done[2], scales_free[2];
  uint32_t tmem, failed;
  uint32_t redo[8];
  union {
    unsigned long long find[kCkThreads / 32 + 2];         // (before any row is looked at)
    int8_t q_exp[256];                                    // 8-bit pages: each row of q was scaled by 2^e
  };
};
template <int HD>
constexpr uint32_t ChunkSmem() { return ChunkShape<HD>::kShared + ((sizeof(ChunkShared) + 15u) & ~15u); }
static_assert(ChunkSmem<128>() <= 227u * 1024u && ChunkSmem<64>() <= 227u * 1024u, "shared memory of an SM");

// A tile of rows: packed rows [r0, r0 + rows) of sequence `seq` (row x group + head), and the blocks of keys that any of them sees.
struct Tile {
  uint32_t seq, r0, rows;
  Seq s;
  Span keys;
  uint32_t blocks;
};
__device__ __forceinline__ Tile make_tile(const AttendArgs &a, uint64_t cap, uint32_t seq, uint32_t index) {
  Tile t;
  t.seq = seq;
  t.s = load_seq(a.b, cap, seq);
  t.r0 = index * kChunkRows;
  t.rows = min(t.r0 + kChunkRows, static_cast<uint32_t>(t.s.n) * a.group) - t.r0;
  t.keys = SeenByRows(t.s, static_cast<int32_t>(t.r0 / a.group), static_cast<int32_t>((t.r0 + t.rows - 1u) / a.group) + 1, a.causal, a.window);
  t.blocks = (static_cast<uint32_t>(t.keys.hi - t.keys.lo) + kCkKeys - 1u) / kCkKeys;
  return t;
}
__device__ __forceinline__ unsigned long long tiles_of_seq(const AttendArgs &a, uint64_t cap, uint32_t i) {
  const Seq s = load_seq(a.b, cap, i);
  return (static_cast<unsigned long long>(s.n) * a.group + kChunkRows - 1u) / kChunkRows;
}
// The work of a CTA: which tile, cache head, part of the tile's blocks. Tiles with the most keys (a sequence's last) come first.
struct Work { uint32_t tile, head, split, item; };
__device__ __forceinline__ Work work_of(const AttendArgs &a, uint32_t index, uint32_t splits) {
  Work w;
  w.split = index % splits;
  w.item = index / splits;
  w.head = w.item % a.c.heads;
  w.tile = a.tiles - 1u - w.item / a.c.heads;
  return w;
}
// Blocks [b0, b1) of a split, and how many splits have any.
__device__ __forceinline__ void split_of(uint32_t blocks, uint32_t splits, uint32_t split, uint32_t &b0, uint32_t &b1, uint32_t &used) {
  const uint32_t per = (blocks + splits - 1u) / splits;
  b0 = min(blocks, split * per);
  b1 = min(blocks, b0 + per);
  used = per ? (blocks + per - 1u) / per : 0u;
}

__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {      // 16-byte chunk of a row of HD values
  return (chunk >> 3) * (128u * 128u) + row * 128u + (((chunk & 7u) ^ (row & 7u)) << 4);
}

// ---- the filling warps ----------------------------------------------------------------------
template <bool BF, bool Q8, int HD>
static __device__ __forceinline__ void chunk_load(const AttendArgs &a, const Tile &t, uint32_t head, uint32_t b0, uint32_t b1, uint8_t *sm, ChunkShared *S) {
  using Sh = ChunkShape<HD>;
  constexpr uint32_t NS = Sh::kStages;
  volatile uint32_t *failed = &S->failed;
  const uint32_t tid = threadIdx.x - kSoftWarps * 32u, lane = tid & 31u, w = tid >> 5;
  const uint32_t base = smem_addr(sm);
  uint32_t it = 0;                                        // blocks filled so far: K, V, K, V, ..
  // the lane's key of a block: 32 w + lane
  int32_t page = -1;
  uint32_t slot = 0, entry = 0;
  bool live = false;
  auto look_ahead = [&](uint32_t j) {
    const int32_t p = t.keys.lo + static_cast<int32_t>(j * kCkKeys + 32u * w + lane);
    live = j < b1 && p < t.keys.hi;
    if (live) {
      entry = a.c.by_page.quot(static_cast<uint32_t>(p));
      slot = static_cast<uint32_t>(p) - entry * a.c.page_size;
      page = __ldg(a.b.pages + static_cast<int64_t>(t.seq) * a.b.pages_stride + entry);
    }
  };
  look_ahead(b0);
  // ---- Q: a thread to a row of each slot ----
  const bool vec = ((reinterpret_cast<uintptr_t>(a.q.p) & 15u) | ((a.q.row | a.q.head) & 7)) == 0;
#pragma unroll 1
  for (uint32_t s = 0; s < 2u; ++s) {
    const uint32_t r = s * kCkRows + tid;
    if (s * kCkRows >= t.rows) break;
    const bool has = r < t.rows;
    const uint32_t pr = t.r0 + r, tok = pr / a.group;
    const uint8_t *p = has ? row_at(a.q, t.s.first + static_cast<int32_t>(tok), head * a.group + (pr - tok * a.group)) : a.q.p;
    auto chunk = [&](uint32_t c) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (has && c * 8u < a.c.hd) {
        if (vec) {
          v = *reinterpret_cast<const uint4 *>(p + 16u * c);
        } else {
          const uint16_t *h = reinterpret_cast<const uint16_t *>(p) + 8u * c;
          v = make_uint4(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16), h[4] | (static_cast<uint32_t>(h[5]) << 16),
                         h[6] | (static_cast<uint32_t>(h[7]) << 16));
        }
      }
      return v;
    };
    const uint32_t dst = base + Sh::kQ + s * Sh::kBlock;
    if (Q8 && BF) {
      float top = 0.0f;
#pragma unroll 4
      for (uint32_t c = 0; c < HD / 8; ++c) {
        const uint4 v = chunk(c);
        const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(ww[i] << 16)), fabsf(__uint_as_float(ww[i] & 0xffff0000u))));
      }
      const int ex = static_cast<int>(__float_as_uint(top) >> 23);
      const int e = ex == 0 || ex == 255 ? 0 : max(-100, min(100, 127 + 14 - ex));
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      S->q_exp[r] = static_cast<int8_t>(e);
#pragma unroll 4
      for (uint32_t c = 0; c < HD / 8; ++c) {
        uint4 v = chunk(c);
        auto h2 = [&](uint32_t x) { return cvt_f16x2(__uint_as_float(x & 0xffff0000u) * up, __uint_as_float(x << 16) * up); };
        v.x = h2(v.x); v.y = h2(v.y); v.z = h2(v.z); v.w = h2(v.w);
        sts_v4(dst + swizzled(tid, c), v);
      }
    } else {
#pragma unroll 4
      for (uint32_t c = 0; c < HD / 8; ++c) sts_v4(dst + swizzled(tid, c), chunk(c));
    }
  }
  fence_proxy_async_smem();
  mbar_arrive(&S->q_full);
  // ---- K and V ----
  auto place = [&](int64_t &off, int64_t &soff) -> uint32_t {       // the lane's key; which lanes of the warp have one
    bool ok = live;
    if (ok && static_cast<uint32_t>(page) >= a.c.n_pages) {
      cache_fault(a.c.status, kStBadPage, t.seq, entry, static_cast<uint32_t>(page));
      ok = false;
    }
    off = ok ? page * a.c.page_bytes + slot * a.c.slot_bytes + head * a.c.head_bytes : 0;
    soff = ok && Q8 ? page * a.c.s_page + slot * a.c.s_slot + head * a.c.s_head : 0;
    return __ballot_sync(0xffffffffu, ok);
  };
  auto room = [&](uint32_t i) { return tc_wait(&S->empty[i % NS], ((i / NS) & 1u) ^ 1u, failed, kBudget); };
  auto done = [&](uint32_t i) {
    fence_proxy_async_smem();
    mbar_arrive(&S->full[i % NS]);
  };
  bool ok = true;
  if constexpr (!Q8) {
    constexpr uint32_t CH = HD / 8, AT = 32u / CH;        // chunks of a row; rows at once
    const uint32_t sub = lane % CH, r1 = lane / CH;
    const bool in_hd = sub * 8u < a.c.hd;
    auto copy = [&](const uint8_t *pages, uint32_t i, int64_t off, uint32_t mask) {
      const uint32_t dst = base + Sh::kRing + (i % NS) * Sh::kBlock;
#pragma unroll
      for (uint32_t k = 0; k < 32u / AT; ++k) {
        const uint32_t r = k * AT + r1;
        const int64_t o = __shfl_sync(0xffffffffu, off, r);
        const uint32_t bytes = ((mask >> r) & 1u) && in_hd ? 16u : 0u;
        cp_async_16_zfill(dst + swizzled(32u * w + r, sub), pages + (bytes ? o + 16 * sub : 0), bytes);
      }
      cp_async_commit();
    };
    for (uint32_t j = b0; ok && j < b1; ++j) {
      int64_t off, soff;
      const uint32_t mask = place(off, soff);
      look_ahead(j + 1u);
#pragma unroll
      for (uint32_t v = 0; v < 2u; ++v) {
        // (a lane that gave up takes its warp with it)
        ok = __all_sync(0xffffffffu, ok && room(it));
        if (!ok) break;
        copy(v ? a.c.v : a.c.k, it, off, mask);
        if (it >= 2u) { cp_async_wait<2>(); done(it - 2u); }
        ++it;
      }
    }
    cp_async_wait_all();
    if (ok) {
      if (it >= 2u) done(it - 2u);
      if (it >= 1u) done(it - 1u);
    }
  } else {
    constexpr uint32_t CH = HD / 16, AT = 32u / CH, N = 32u / AT;     // 16-code chunks of a row; rows at once; loads of a thread
    const uint32_t sub = lane % CH, r1 = lane / CH;
    const bool in_hd = sub * 16u < a.c.hd;
    uint4 kw[N], vw[N];
    float ksc = 0.0f, vsc = 0.0f;
    auto fetch = [&](const uint8_t *pages, int64_t off, uint32_t mask, uint4 (&x)[N]) {
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) {
        const uint32_t r = k * AT + r1;
        const int64_t o = __shfl_sync(0xffffffffu, off, r);
        x[k] = make_uint4(0u, 0u, 0u, 0u);
        if (((mask >> r) & 1u) && in_hd) x[k] = ldg_v4(pages + o + 16 * sub);
      }
    };
    auto put = [&](uint32_t i, const uint4 (&x)[N], float scale) {
      // (block i / 2's place for scales; the softmax is done with those of the block two before)
      const uint32_t dst = base + Sh::kRing + (i % NS) * Sh::kBlock;
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) {
        const uint32_t r = 32u * w + k * AT + r1;
        const uint32_t c[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
        uint32_t h[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) { h[2 * q] = cvt_e4m3x2_f16x2(c[q] & 0xffffu); h[2 * q + 1] = cvt_e4m3x2_f16x2(c[q] >> 16); }
        sts_v4(dst + swizzled(r, 2u * sub), make_uint4(h[0], h[1], h[2], h[3]));
        sts_v4(dst + swizzled(r, 2u * sub + 1u), make_uint4(h[4], h[5], h[6], h[7]));
      }
      *reinterpret_cast<float *>(sm + Sh::kScales + (i & 3u) * 512u + (32u * w + lane) * 4u) = scale;
    };
    int64_t off, soff;
    uint32_t mask = place(off, soff);
    fetch(a.c.k, off, mask, kw);
    ksc = (mask >> lane) & 1u ? a.c.ks[soff] : 0.0f;
    for (uint32_t j = b0; ok && j < b1; ++j) {
      fetch(a.c.v, off, mask, vw);
      vsc = (mask >> lane) & 1u ? a.c.vs[soff] : 0.0f;
      look_ahead(j + 1u);
      const uint32_t n = j - b0;
      ok = __all_sync(0xffffffffu, room(it) && tc_wait(&S->scales_free[n & 1u], ((n >> 1) & 1u) ^ 1u, failed, kBudget));
      if (!ok) break;
      put(it, kw, ksc);
      done(it++);
      mask = place(off, soff);
      fetch(a.c.k, off, mask, kw);
      ksc = (mask >> lane) & 1u ? a.c.ks[soff] : 0.0f;
      ok = __all_sync(0xffffffffu, room(it));
      if (!ok) break;
      put(it, vw, vsc);
      done(it++);
    }
  }
  // the products have read what was filled last, and their arrivals on the ring's barriers are in
  if (ok && tid == 0u) tc_drain(S->empty, NS, it, failed, kBudget);
}

// ---- the issuing warp -----------------------------------------------------------------------
template <bool F16, int HD>
static __device__ __forceinline__ void chunk_products(uint32_t blocks, uint32_t slots, uint8_t *sm, ChunkShared *S) {
  using Sh = ChunkShape<HD>;
  constexpr uint32_t NS = Sh::kStages;
  volatile uint32_t *failed = &S->failed;
  const uint32_t base = smem_addr(sm), tmem = S->tmem;
  const uint32_t fmt = F16 ? 0u : 1u;
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
        tc_mma_f16_ts(tmem + 256u + s * HD, tmem + s * 128u + 8u * k, dv + ((st * Sh::kBlock) >> 4) + k * (2048u >> 4), idesc_o, (!first || k) ? 1u : 0u);
    }
    __syncwarp();
  };
  auto release = [&](uint32_t st) {
    if (leader) tc_commit(&S->empty[st]);
    __syncwarp();
  };
  uint32_t it = 0;
  bool ok = tc_wait_uniform(&S->q_full, 0u, failed, kBudget) && tc_wait_uniform(&S->full[0], 0u, failed, kBudget);
  if (!ok) return;
  tc_fence_after_sync();
  for (uint32_t s = 0; s < slots; ++s) scores(s, 0u);
  release(0u);
  ++it;
  for (uint32_t j = 0; j < blocks; ++j) {
    const uint32_t sv = it % NS, pv = (it / NS) & 1u, sk = (it + 1u) % NS, pk = ((it + 1u) / NS) & 1u;
    const bool more = j + 1u < blocks;
    ok = tc_wait_uniform(&S->full[sv], pv, failed, kBudget);
    for (uint32_t s = 0; ok && s < slots; ++s) {
      ok = tc_wait_uniform(&S->p_full[s], j & 1u, failed, kBudget);
      if (!ok) break;
      tc_fence_after_sync();
      values(s, sv, j == 0u);
      if (s + 1u == slots) release(sv);
      if (more) {
        if (s == 0u) ok = tc_wait_uniform(&S->full[sk], pk, failed, kBudget);
        if (!ok) break;
        tc_fence_after_sync();
        scores(s, sk);
        if (s + 1u == slots) release(sk);
      } else {
        if (leader) tc_commit(&S->pv_done[s]);
        __syncwarp();
      }
    }
    if (!ok) return;
    it += 2u;
  }
}

// ---- the softmax warps ----------------------------------------------------------------------
// One block's scores of a row: their maximum and, for 8-bit pages, the largest scale among the keys that the row sees.
template <bool BF, bool Q8, int HD>
static __device__ __forceinline__ void chunk_rows(const AttendArgs &a, const Tile &t, const Work &wk, uint32_t b0, uint32_t b1, uint8_t *sm, ChunkShared *S) {
  using Sh = ChunkShape<HD>;
  constexpr uint32_t NS = Sh::kStages;
  volatile uint32_t *failed = &S->failed;
  const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31u, s = w >> 2, q4 = w & 3u;
  if (s * kCkRows >= t.rows) return;
  const uint32_t r = s * kCkRows + 32u * q4 + lane;
  const bool has = r < t.rows;
  const uint32_t pr = t.r0 + r, tok = pr / a.group, head = wk.head * a.group + (pr - tok * a.group);
  Span sp = has ? SeenBy(t.s, static_cast<int32_t>(tok), a.causal, a.window) : Span{0, 0};
  const uint32_t s_addr = S->tmem + ((32u * q4) << 16) + s * 128u, o_addr = S->tmem + ((32u * q4) << 16) + 256u + s * HD;
  float sl2 = a.scale_log2;
  if (Q8 && BF) {
    if (!tc_wait_uniform(&S->q_full, 0u, failed, kBudget)) return;
    sl2 *= __uint_as_float(static_cast<uint32_t>(127 - S->q_exp[r]) << 23);
  }
  float m_used = -INFINITY, l = 0.0f, v_ref = 0.0f;
  uint32_t it = 0;                                        // the ring's blocks: K of block j is 2 j, V 2 j + 1
#pragma unroll 1
  for (uint32_t j = b0; j < b1; ++j, it += 2u) {
    if (!tc_wait_uniform(&S->s_full[s], (j - b0) & 1u, failed, kBudget)) return;
    const float *ks = reinterpret_cast<const float *>(sm + Sh::kScales + (it & 3u) * 512u);
    const float *vs = ks + 128;
    if (Q8 && !tc_wait_uniform(&S->full[(it + 1u) % NS], ((it + 1u) / NS) & 1u, failed, kBudget)) return;      // (the values' scales)
    tc_fence_after_sync();
    const int32_t j0 = t.keys.lo + static_cast<int32_t>(j * kCkKeys);
    const int32_t lo = sp.lo - j0, hi = sp.hi - j0;       // columns [lo, hi) are seen
    const bool whole = __all_sync(0xffffffffu, lo <= 0 && hi >= static_cast<int32_t>(kCkKeys));
    // 1: the row's scores into registers, and their maximum
    uint32_t x[4][32];
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) tc_ld32(s_addr + 32u * c, x[c]);
    tc_wait_ld();
    float mx = -INFINITY, v_top = 0.0f;
    if (Q8) {
#pragma unroll
      for (int i = 0; i < 128; i += 4) {
        const float4 k4 = *reinterpret_cast<const float4 *>(ks + i), v4 = *reinterpret_cast<const float4 *>(vs + i);
        const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, vv[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[i >> 5][(i & 31) + e] = __float_as_uint(__uint_as_float(x[i >> 5][(i & 31) + e]) * kk[e]);
          const bool seen = whole || (i + e >= lo && i + e < hi);
          v_top = fmaxf(v_top, seen ? vv[e] : 0.0f);
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 128; ++i)
        if (i < lo || i >= hi) x[i >> 5][i & 31] = 0xff800000u;
    }
    {
      float m4[4] = {mx, mx, mx, mx};
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        m4[i & 1] = max3(m4[i & 1], __uint_as_float(x[0][i]), __uint_as_float(x[1][i]));
        m4[2 + (i & 1)] = max3(m4[2 + (i & 1)], __uint_as_float(x[2][i]), __uint_as_float(x[3][i]));
      }
      mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    }
    mx *= sl2;
    bool grow = mx > m_used + kGrow;
    float alpha = 1.0f, v_mul = 1.0f;
    if (grow) {
      alpha = m_used == -INFINITY ? 0.0f : fast_ex2(m_used - mx);
      l *= alpha;
      m_used = mx;
    }
    if (Q8) {
      const float ref = power_above(v_top);
      if (ref > v_ref) {
        alpha *= v_ref / ref;
        v_ref = ref;
        grow = true;
      }
      v_mul = kCkPScale / v_ref;
    }
    if (j > b0 && __any_sync(0xffffffffu, grow)) {        // (these scores came after the products before them: O is at rest)
#pragma unroll 1
      for (uint32_t c0 = 0; c0 < HD; c0 += 16u) {
        uint32_t y[16];
        __syncwarp();
        tc_ld16(o_addr + c0, y);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
        tc_st16(o_addr + c0, y);
      }
      tc_wait_st();
    }
    // 2: the weights, over the scores they came from
    const float neg = m_used == -INFINITY ? 0.0f : -m_used;
    const unsigned long long sl2_2 = pack_f32x2(sl2, sl2), neg_2 = pack_f32x2(neg, neg);
    unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float e0, e1;
        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])), sl2_2, neg_2), e0, e1);
        e0 = fast_ex2(e0);
        e1 = fast_ex2(e1);
        sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(e0, e1));
        if (Q8) {
          const float2 v2 = *reinterpret_cast<const float2 *>(vs + 32 * c + 2 * i);
          e0 = e0 == 0.0f ? 0.0f : e0 * (v2.x * v_mul);
          e1 = e1 == 0.0f ? 0.0f : e1 * (v2.y * v_mul);
        }
        pk[i] = BF && !Q8 ? cvt_bf16x2(e1, e0) : cvt_f16x2(e1, e0);
      }
      __syncwarp();
      tc_st16(s_addr + 16u * c, pk);
    }
    tc_wait_st();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0u) {
      mbar_arrive(&S->p_full[s]);
      if (Q8) mbar_arrive(&S->scales_free[(j - b0) & 1u]);
    }
    float a0, a1;
    unpack_f32x2(add_f32x2(sum[0], sum[1]), a0, a1);
    l += a0 + a1;
  }
  // ---- the result ----
  if (!tc_wait_uniform(&S->pv_done[s], 0u, failed, kBudget)) return;
  tc_fence_after_sync();
  const bool split = a.splits > 1u;
  float *part = a.part + static_cast<size_t>(wk.item * a.splits + wk.split) * (kChunkRows * (HD + 2u));
  const bool none = m_used == -INFINITY && l == 0.0f;
  float mul = split ? 1.0f : none ? 0.0f : 1.0f / l;
  if (Q8) mul *= v_ref * (1.0f / kCkPScale);
  uint8_t *out = has ? row_at(a.o, t.s.first + static_cast<int32_t>(tok), head) : a.o.p;
  const bool vec = (reinterpret_cast<uintptr_t>(out) & 15u) == 0u;
  bool fine = true;
#pragma unroll 1
  for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
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
      for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4 *>(part + r * HD + c0 + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      continue;
    }
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      if (c0 + i >= a.c.hd) break;
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = __uint_as_float(x[i + 2 * e]), v = __uint_as_float(x[i + 2 * e + 1]);
        h[e] = BF ? cvt_bf16x2(v, u) : cvt_f16x2(v, u);
      }
      uint8_t *p = out + 2u * (c0 + i);
      if (vec) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(h[0], h[1], h[2], h[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          reinterpret_cast<uint16_t *>(p)[2 * e] = static_cast<uint16_t>(h[e]);
          reinterpret_cast<uint16_t *>(p)[2 * e + 1] = static_cast<uint16_t>(h[e] >> 16);
        }
      }
    }
  }
  tc_fence_before_sync();
  if (!has) return;
  if (split) {
    part[kChunkRows * HD + r] = m_used;
    part[kChunkRows * HD + kChunkRows + r] = l;
  } else {
    if (a.lse) a.lse[static_cast<int64_t>(t.s.first + static_cast<int32_t>(tok)) * a.q_heads + head] = (m_used + log2f(l)) * 0.69314718055994531f;
    if (!fine && (sp.lo > t.keys.lo || sp.hi < t.keys.hi)) atomicOr(&S->redo[r >> 5], 1u << (r & 31u));
  }
}

// Rows that see nothing of the cache.
__device__ __forceinline__ void clear_rows(const AttendArgs &a, const Tile &t, uint32_t head, uint32_t threads) {
  for (uint32_t i = threadIdx.x; i < t.rows * a.c.hd; i += threads) {
    const uint32_t r = i / a.c.hd, d = i - r * a.c.hd, pr = t.r0 + r, tok = pr / a.group, h = head * a.group + (pr - tok * a.group);
    const int32_t row = t.s.first + static_cast<int32_t>(tok);
    store_row_value(row_at(a.o, row, h) + 2u * d, 0.0f, a.bf16 != 0u);
    if (d == 0u && a.lse) a.lse[static_cast<int64_t>(row) * a.q_heads + h] = -INFINITY;
  }
}

template <bool BF, bool Q8, int HD>
__global__ void __launch_bounds__(kCkThreads, 1) b2_attend_chunk(const __grid_constant__ AttendArgs a) {
  using Sh = ChunkShape<HD>;
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
  const Work wk = work_of(a, blockIdx.x, a.splits);
  uint32_t seq;
  unsigned long long before;
  if (!find_unit<kCkThreads>(a.b.n_seqs, wk.tile, S->find, [&](uint32_t i) { return tiles_of_seq(a, cap, i); }, seq, before)) return;
  const Tile t = make_tile(a, cap, seq, static_cast<uint32_t>(wk.tile - before));
  if (t.blocks == 0u) {
    if (wk.split == 0u) clear_rows(a, t, wk.head, kCkThreads);
    return;
  }
  uint32_t b0, b1, used;
  split_of(t.blocks, a.splits, wk.split, b0, b1, used);
  if (b0 >= b1) return;
  if (tid == 0u) {
    mbar_init(&S->q_full, kLoadWarps * 32u);
    for (uint32_t i = 0; i < Sh::kStages; ++i) { mbar_init(&S->full[i], kLoadWarps * 32u); mbar_init(&S->empty[i], 1u); }
    for (uint32_t s = 0; s < 2u; ++s) { mbar_init(&S->s_full[s], 1u); mbar_init(&S->p_full[s], 4u); mbar_init(&S->pv_done[s], 1u); mbar_init(&S->scales_free[s], t.rows > kCkRows ? 8u : 4u); }
    S->failed = 0u;
    for (uint32_t i = 0; i < 8u; ++i) S->redo[i] = 0u;
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
    more_registers<kSoftRegs>();
    chunk_rows<BF, Q8, HD>(a, t, wk, b0, b1, sm, S);
  } else if (w < kSoftWarps + kLoadWarps) {
    fewer_registers<kLoadRegs>();
    chunk_load<BF, Q8, HD>(a, t, wk.head, b0, b1, sm, S);
  } else {
    fewer_registers<kIssueRegs>();
    if (w == kSoftWarps + kLoadWarps) chunk_products<Q8 || !BF, HD>(b1 - b0, t.rows > kCkRows ? 2u : 1u, sm, S);
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  const bool gave_up = S->failed != 0u;
  if (gave_up) {                                          // products of other roles may still be landing: give them time
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 50000ull) nanosleep_ns(1000);
    if (tid == 0u) cache_fault(a.c.status, kStTcTimeout, t.seq, wk.tile, 0u);
  }
  if (w == kSoftWarps + kLoadWarps) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(S->tmem, kCkCols);
  }
  if (gave_up || a.splits > 1u) return;
  for (uint32_t r = w; r < t.rows; r += kCkThreads / 32u)
    if ((S->redo[r >> 5] >> (r & 31u)) & 1u) attend_row_alone(a, t.seq, t.s, static_cast<int32_t>((t.r0 + r) / a.group), wk.head * a.group + (t.r0 + r) % a.group);
}

// Tiles whose keys were split: a warp to a row, the parts in their order.
constexpr uint32_t kJoinThreads = 256, kJoinRows = 32;    // rows of a CTA
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) b2_attend_join(const __grid_constant__ AttendArgs a) {
  __shared__ unsigned long long find[kJoinThreads / 32 + 2];
  const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint64_t cap = capacity_of(a.c, a.b);
  const Work wk = work_of(a, blockIdx.x / (kChunkRows / kJoinRows), 1u);
  uint32_t seq;
  unsigned long long before;
  if (!find_unit<kJoinThreads>(a.b.n_seqs, wk.tile, find, [&](uint32_t i) { return tiles_of_seq(a, cap, i); }, seq, before)) return;
  const Tile t = make_tile(a, cap, seq, static_cast<uint32_t>(wk.tile - before));
  uint32_t b0, b1, used;
  split_of(t.blocks, a.splits, 0u, b0, b1, used);
  if (used == 0u) return;                                 // (rows without keys are cleared already)
  const uint32_t first = (blockIdx.x % (kChunkRows / kJoinRows)) * kJoinRows;
  const float *part = a.part + static_cast<size_t>(wk.item) * a.splits * (kChunkRows * (HD + 2u));
  for (uint32_t r = first + w; r < min(t.rows, first + kJoinRows); r += kJoinThreads / 32u) {
    const uint32_t pr = t.r0 + r, tok = pr / a.group, head = wk.head * a.group + (pr - tok * a.group), d = lane * (HD / 32);
    const int32_t row = t.s.first + static_cast<int32_t>(tok);
    float mm = -INFINITY, ll = 0.0f, x[HD / 32] = {};
    for (uint32_t k = 0; k < used; ++k) mm = fmaxf(mm, part[static_cast<size_t>(k) * (kChunkRows * (HD + 2u)) + kChunkRows * HD + r]);
#pragma unroll 4
    for (uint32_t k = 0; k < used; ++k) {
      const float *p = part + static_cast<size_t>(k) * (kChunkRows * (HD + 2u));
      const float mk = p[kChunkRows * HD + r], f = mk == mm ? 1.0f : fast_ex2(mk - mm);
      ll += p[kChunkRows * HD + kChunkRows + r] * f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) x[i] += p[r * HD + d + i] * f;
    }
    const float inv = mm == -INFINITY && ll == 0.0f ? 0.0f : 1.0f / ll;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const float v = x[i] * inv;
      fine = fine && isfinite(v);
      if (d + i < a.c.hd) store_row_value(row_at(a.o, row, head) + 2u * (d + i), v, a.bf16 != 0u);
    }
    if (lane == 0u && a.lse) a.lse[static_cast<int64_t>(row) * a.q_heads + head] = (mm + log2f(ll)) * 0.69314718055994531f;
    const Span sp = SeenBy(t.s, static_cast<int32_t>(tok), a.causal, a.window);
    if (__any_sync(0xffffffffu, !fine) && (sp.lo > t.keys.lo || sp.hi < t.keys.hi)) {
      __syncwarp();
      attend_row_alone(a, t.seq, t.s, static_cast<int32_t>(tok), head);
    }
  }
}

template <bool BF, bool Q8, int HD>
int Launch(const AttendArgs &a, cudaStream_t stream) {
  const uint32_t items = a.tiles * a.c.heads;
  b2_attend_chunk<BF, Q8, HD><<<items * a.splits, kCkThreads, ChunkSmem<HD>(), stream>>>(a);
  if (a.splits > 1u) b2_attend_join<HD><<<items * (kChunkRows / kJoinRows), kJoinThreads, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
template <bool BF, bool Q8, int HD>
cudaError_t Attr() {
  return cudaFuncSetAttribute(b2_attend_chunk<BF, Q8, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(ChunkSmem<HD>()));
}

}  // namespace

int PrepareAttendChunk() {
  for (cudaError_t e : {Attr<true, false, 64>(), Attr<true, false, 128>(), Attr<false, false, 64>(), Attr<false, false, 128>(), Attr<true, true, 64>(), Attr<true, true, 128>(),
                        Attr<false, true, 64>(), Attr<false, true, 128>()})
    if (e != cudaSuccess) return static_cast<int>(e);
  return 0;
}
size_t AttendChunkPartialBytes(uint32_t sms) { return static_cast<size_t>(sms) * kChunkRows * (128u + 2u) * sizeof(float); }

int LaunchAttendChunk(const AttendArgs &a, CUstream_st *stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool big = a.c.hd > 64u;
  if (a.e4m3) {
    if (a.bf16) return big ? Launch<true, true, 128>(a, s) : Launch<true, true, 64>(a, s);
    return big ? Launch<false, true, 128>(a, s) : Launch<false, true, 64>(a, s);
  }
  if (a.bf16) return big ? Launch<true, false, 128>(a, s) : Launch<true, false, 64>(a, s);
  return big ? Launch<false, false, 128>(a, s) : Launch<false, false, 64>(a, s);
}

}  // namespace b2
