// Attention of a few rows of each sequence over the paged cache: decode steps. rows x (query heads to a cache head) <= 16.
//
// One pass over the keys with a running maximum m and sum l of the softmax (base 2): for a tile of keys s = k q^T scale log2 e,
// p = 2^(s - m), l += sum p, o += v^T p; where a row's scores outgrow m by more than 2^8, m moves and l and o are scaled by
// 2^(m_old - m). The result is o / l.
//
// Bound: HBM, K and V of every visible key read once.
// Work: a cache head of a sequence is an item, cut into tiles of 16 or 32 keys. The tiles of the whole batch in a row, with some for
// what an item costs beside its tiles, are dealt to the CTAs in equal runs, whatever the lengths. A CTA's warps take
// its tiles in turn, each through two stages of its own (K and V of a tile, 8 KB, by 16-byte asynchronous copies, page by page): no barrier
// stands between tiles. At an item's end the warps' (m, l, o) are joined through the stage each has free; an item that is split between
// CTAs leaves partial results, and the CTA that comes last joins them in the CTAs' order.
// Products: warp-level, 16 x 8 x 16, with the keys (then the values' head_dim) as the 16 rows and the rows of q that share a cache head as the 8
// columns, so that a decode step of up to 8 heads to a cache head wastes nothing (as the 16 rows they would be half padding at best: twice the
// products, scores and registers; 32 x 8 bits x 128: 1240 instructions a tile, 283 us for 64 sequences of 200 to 16000 tokens). Scores become the
// second product's operand by a transposition of 8 x 8 fragments.
// 8-bit pages: codes are exact in f16, so the products are f16 x f16 whatever the rows' type. q of type bf16 is scaled by a power of
// two for each row so that its largest value is near 2^14 (f16 then holds what bf16 held to 2^-38 of that); a key's scale goes onto its
// scores, a value's onto p, relative to a power of two not below any scale that the row has seen (p v's factor stays in f16's normal range).
// p is split into two 16-bit values (p and what rounding left), since the second product costs little here (64 sequences of 200 to 16000
// tokens, f16 rows, 8-bit pages: 116 us, 113 without it; 16-bit pages: no difference); the result is then only rounded once, as it is
// stored. Only bf16 rows over 8-bit pages do without: p in f16 is eight times finer than their results.
#include "attend_common.cuh"

namespace b2 {
namespace {

constexpr uint32_t kStages = 2;
// CTAs to an SM: of three warps four, so that one's joins lie under the others' loads.
constexpr uint32_t PerSm(int warps) { return warps == 3 ? 4u : 1u; }
constexpr float kPHead = 6.0f;           // 8-bit pages: p (below 2^8) on the largest scale stays below 2^14
constexpr float kGrow = 8.0f;            // log2 of the growth of a row maximum that moves it
constexpr uint32_t kItemTiles = 8;       // what an item costs beside its tiles, in tiles

template <bool Q8, int HD, int NR, int NW>
struct StepShape {
  static constexpr int KT = (Q8 || HD == 64) ? 32 : 16;       // keys of a tile
  static constexpr int CH = HD * (Q8 ? 1 : 2) / 16;           // 16-byte chunks of a row
  static constexpr int kBytes = KT * CH * 16;                 // K (or V) of a tile
  static constexpr int kScales = Q8 ? 2 * KT * 4 : 0;
  static constexpr int kStage = 2 * kBytes + kScales;
  static constexpr int kRing = NW * static_cast<int>(kStages) * kStage;
  static constexpr int kQ = 8 * NR * HD * 2;                    // q of an item
  static constexpr int kSmem = kRing + 2 * kQ;
};
// Chunk of a row in shared memory: eight rows of the same chunk lie in different banks.
template <int CH>
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t c) {
  return (row * CH + (CH >= 8 ? (c ^ (row & 7u)) : (c ^ ((row >> 1) & 3u)))) * 16u;
}
// The transposed 8 x 8 fragment of 16-bit values.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float lds_f32(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}

template <int NW>
struct StepShared {
  static constexpr uint32_t kStepWarps = NW;
  float m[kStepWarps][16], l[kStepWarps][16];
  unsigned long long sum[2][kStepWarps], find[kStepWarps + 2];
  uint32_t at[kStepWarps];         // the stage each warp left its result in
  uint32_t last, redo[2];          // redo by turns: an item's rows to be worked out again
};

// An item: cache head h of sequence b, `nt` tiles of keys from `lo`.
template <int KT>
struct Walk {
  uint32_t b, h;
  Seq s;
  Span keys;
  uint32_t nt;
  __device__ __forceinline__ void load(const AttendArgs &a, uint64_t cap) {
    s = load_seq(a.b, cap, b);
    keys = s.n > 0 ? SeenByRows(s, 0, s.n, a.causal, a.window) : Span{0, 0};
    nt = s.n > 0 ? max(1u, (static_cast<uint32_t>(keys.hi - keys.lo) + KT - 1u) / KT) : 0u;
  }
  // false behind the last item
  __device__ __forceinline__ bool next(const AttendArgs &a, uint64_t cap) {
    if (++h < a.c.heads) return true;
    h = 0;
    do {
      if (++b >= a.b.n_seqs) return false;
      load(a, cap);
    } while (nt == 0u);
    return true;
  }
};

// NR: groups of 8 rows. NW: warps of a CTA.
template <bool BF, bool Q8, int HD, int NR, int NW>
__global__ void __launch_bounds__(NW * 32, PerSm(NW)) b2_attend_step(const __grid_constant__ AttendArgs a) {
  using Sh = StepShape<Q8, HD, NR, NW>;
  constexpr uint32_t kStepWarps = NW, kStepThreads = NW * 32;
  constexpr int KT = Sh::KT, CH = Sh::CH, MT = KT / 16;
  constexpr uint32_t kPitch = NR == 1 ? HD + 4 : HD;          // of a result's rows in a stage
  static_assert(2 * Sh::kBytes >= 8 * NR * static_cast<int>(kPitch) * 4, "a stage holds a warp's result");
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ StepShared<NW> S;
  const uint32_t tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u, quad = lane >> 2, t4 = lane & 3u;
  const uint64_t cap = capacity_of(a.c, a.b);
  // ---- how much work there is, and where this CTA's run of it begins ----
  auto units_of = [&](uint32_t i, uint32_t &items) -> unsigned long long {
    Walk<KT> x;
    x.b = i; x.h = 0;
    x.load(a, cap);
    if (x.s.bad && blockIdx.x == 0u) cache_fault(a.c.status, kStBadBatch, i, static_cast<uint32_t>(x.s.bad), static_cast<uint32_t>(x.s.value));
    items = x.nt ? a.c.heads : 0u;
    return x.nt ? static_cast<unsigned long long>(x.nt + kItemTiles) * a.c.heads : 0ull;
  };
  // Up to 128 sequences: every warp looks at all of them, four to a lane, and waits for no other. More: the CTA together.
  const bool few = a.b.n_seqs <= 128u;
  unsigned long long mine = 0, many = 0, u4[4] = {0, 0, 0, 0};
  if (few) {
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k) {
      uint32_t items = 0;
      if (lane * 4u + k < a.b.n_seqs) u4[k] = units_of(lane * 4u + k, items);
      mine += u4[k];
      many += items;
    }
  } else {
    for (uint32_t i = tid; i < a.b.n_seqs; i += kStepThreads) {
      uint32_t items;
      mine += units_of(i, items);
      many += items;
    }
  }
  auto add = [](unsigned long long x, unsigned long long y) { return x + y; };
  unsigned long long U = warp_reduce(mine, add), items = warp_reduce(many, add);
  if (tid == 0u) S.redo[0] = 0u;
  if (!few) {
    if (lane == 0u) { S.sum[0][w] = U; S.sum[1][w] = items; }
    __syncthreads();
    U = items = 0;
#pragma unroll
    for (uint32_t i = 0; i < kStepWarps; ++i) { U += S.sum[0][i]; items += S.sum[1][i]; }
  }
  if (U == 0ull) return;
  // As many CTAs as give each warp a tile; but items of up to four tiles for each of a CTA's warps are not split for that (300 keys, 8 heads:
  // joining two or three CTAs' results takes longer than another round of tiles).
  const unsigned long long tiles = U - items * kItemTiles;
  unsigned long long G = tiles / kStepWarps;
  if (G > items && tiles <= items * 4ull * kStepWarps) G = items;
  G = G < 1ull ? 1ull : G > gridDim.x ? gridDim.x : G;
  if (blockIdx.x >= G) return;
  const unsigned long long u0 = U * blockIdx.x / G, u1 = U * (blockIdx.x + 1ull) / G;
  Walk<KT> cw;                                            // the item being worked on
  unsigned long long x0;                                  // its place: kItemTiles units, then its tiles
  if (few) {
    unsigned long long x = mine;
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const uint32_t from = __ffs(__ballot_sync(0xffffffffu, x > u0)) - 1u;     // the lane that has it
    x -= mine;
    uint32_t k = 0;
#pragma unroll
    for (uint32_t i = 0; i < 3u; ++i)
      if (k == i && x + u4[i] <= u0) { x += u4[i]; ++k; }
    x0 = __shfl_sync(0xffffffffu, x, from);
    cw.b = __shfl_sync(0xffffffffu, lane * 4u + k, from);
  } else {
    uint32_t ignored;
    if (!find_unit<kStepThreads>(a.b.n_seqs, u0, S.find, [&](uint32_t i) { return units_of(i, ignored); }, cw.b, x0)) return;
  }
  cw.load(a, cap);
  const uint32_t per = cw.nt + kItemTiles;
  cw.h = static_cast<uint32_t>((u0 - x0) / per);
  x0 += static_cast<unsigned long long>(cw.h) * per;
  // tiles [t_begin, t_end) of the item are this CTA's
  auto tile_at = [](unsigned long long u, unsigned long long x, uint32_t nt) -> uint32_t {
    return u <= x + kItemTiles ? 0u : static_cast<uint32_t>(min(static_cast<unsigned long long>(nt), u - x - kItemTiles));
  };
  uint32_t t_begin = tile_at(u0, x0, cw.nt), t_end = tile_at(u1, x0, cw.nt);
  if (t_begin >= t_end) return;                           // (a run that is shorter than what an item costs beside its tiles)

  // ---- the warp's copies: its tiles are w, w + NW, .. of the CTA's ----
  uint8_t *const ring = sm + w * (kStages * Sh::kStage);
  const uint32_t ring_s = smem_addr(ring);
  Walk<KT> pw = cw;                                       // the item of the next tile to fetch
  uint32_t p_tile = t_begin + w, p_end = t_end;           // its tile there, and the end of the CTA's tiles there
  unsigned long long px = x0;
  bool p_more = true;
  uint32_t issued = 0;
  int32_t page = -1;                                      // page number of the lane's key in that tile
  uint32_t key_slot = 0, key_entry = 0;
  bool key_live = false;
  uint32_t keys_next = 0u;                                // which keys of the tile fetched last are there, a bit each
  constexpr uint32_t kAllKeys = KT == 32 ? 0xffffffffu : (1u << (KT & 31)) - 1u;
  auto look_ahead = [&]() {                               // the next tile's place, and its keys' pages on the way
    while (p_more && p_tile >= p_end) {
      p_tile -= p_end;
      px += pw.nt + kItemTiles;
      p_more = px + kItemTiles < u1 && pw.next(a, cap);
      p_end = p_more ? tile_at(u1, px, pw.nt) : 0u;
    }
    if (!p_more) return;
    const int32_t j = pw.keys.lo + static_cast<int32_t>(p_tile) * KT + static_cast<int32_t>(lane);
    key_live = lane < KT && j < pw.keys.hi;
    if (key_live) {
      key_entry = a.c.by_page.quot(static_cast<uint32_t>(j));
      key_slot = static_cast<uint32_t>(j) - key_entry * a.c.page_size;
      page = __ldg(a.b.pages + static_cast<int64_t>(pw.b) * a.b.pages_stride + key_entry);
    }
  };
  auto issue = [&]() {
    if (p_more) {
      const uint32_t st = ring_s + (issued % kStages) * Sh::kStage;
      bool live = key_live;
      if (live && static_cast<uint32_t>(page) >= a.c.n_pages) {
        cache_fault(a.c.status, kStBadPage, pw.b, key_entry, static_cast<uint32_t>(page));
        live = false;
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, live);
      keys_next = mask;
      constexpr int kAtOnce = 32 / CH;
      const uint32_t sub = lane % CH, r0 = lane / CH;
      const bool in_hd = sub * 16u < a.c.hd * (Q8 ? 1u : 2u);
      const int64_t head_at = pw.h * a.c.head_bytes + sub * 16u;
      const uint32_t entry0 = __shfl_sync(0xffffffffu, key_entry, 0);
      if (mask == kAllKeys && __all_sync(0xffffffffu, lane >= KT || key_entry == entry0)) {     // a whole tile in one page
        int64_t o = __shfl_sync(0xffffffffu, page, 0) * a.c.page_bytes + (__shfl_sync(0xffffffffu, key_slot, 0) + r0) * a.c.slot_bytes + head_at;
        if (!in_hd) o = 0;
        const int64_t step = in_hd ? kAtOnce * a.c.slot_bytes : 0;
        const uint32_t bytes = in_hd ? 16u : 0u;
        const uint8_t *kp = a.c.k + o, *vp = a.c.v + o;
#pragma unroll
        for (int i = 0; i < KT / kAtOnce; ++i, kp += step, vp += step) {
          const uint32_t dst = st + chunk_at<CH>(i * kAtOnce + r0, sub);
          cp_async_16_zfill(dst, kp, bytes);
          cp_async_16_zfill(dst + Sh::kBytes, vp, bytes);
        }
      } else {
        const int64_t off = live ? page * a.c.page_bytes + key_slot * a.c.slot_bytes : 0;
#pragma unroll
        for (int i = 0; i < KT / kAtOnce; ++i) {
          const uint32_t r = i * kAtOnce + r0;
          const int64_t o = __shfl_sync(0xffffffffu, off, r);
          const uint32_t bytes = ((mask >> r) & 1u) && in_hd ? 16u : 0u;       // else zeros
          const int64_t at = bytes ? o + head_at : 0;
          const uint32_t dst = st + chunk_at<CH>(r, sub);
          cp_async_16_zfill(dst, a.c.k + at, bytes);
          cp_async_16_zfill(dst + Sh::kBytes, a.c.v + at, bytes);
        }
      }
      if (Q8) {
        const int64_t so = live ? page * a.c.s_page + key_slot * a.c.s_slot + pw.h * a.c.s_head : 0;
        const uint32_t dst = st + 2u * Sh::kBytes + lane * 4u;
        cp_async_4_zfill(dst, a.c.ks + so, live ? 4u : 0u);
        cp_async_4_zfill(dst + KT * 4u, a.c.vs + so, live ? 4u : 0u);
      }
      p_tile += kStepWarps;
    }
    cp_async_commit();
    ++issued;
    look_ahead();
  };
  // q of an item: [16 rows][HD], rows and values that are not there as zeros
  const uint32_t q_s = smem_addr(sm + Sh::kRing);
  const bool q_vec = ((reinterpret_cast<uintptr_t>(a.q.p) & 15u) | ((a.q.row | a.q.head) & 7)) == 0;
  auto fetch_q = [&](const Walk<KT> &x, uint32_t buf) {
    constexpr uint32_t QC = HD / 8;
    const uint32_t rows = static_cast<uint32_t>(x.s.n) * a.group;
    for (uint32_t i = tid; i < 8u * NR * QC; i += kStepThreads) {
      const uint32_t r = i / QC, c = i - r * QC, tok = r / a.group;
      const bool live = r < rows && c * 8u < a.c.hd;
      const uint8_t *p = live ? row_at(a.q, x.s.first + static_cast<int32_t>(tok), x.h * a.group + (r - tok * a.group)) + 16u * c : a.q.p;
      const uint32_t dst = q_s + buf * Sh::kQ + chunk_at<QC>(r, c);
      if (q_vec) {
        cp_async_16_zfill(dst, p, live ? 16u : 0u);
      } else {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        const uint16_t *e = reinterpret_cast<const uint16_t *>(p);
        if (live) v = make_uint4(e[0] | (static_cast<uint32_t>(e[1]) << 16), e[2] | (static_cast<uint32_t>(e[3]) << 16), e[4] | (static_cast<uint32_t>(e[5]) << 16), e[6] | (static_cast<uint32_t>(e[7]) << 16));
        sts_v4(dst, v);
      }
    }
  };
  look_ahead();
  fetch_q(cw, 0u);
  cp_async_commit();
  issue();
  cp_async_wait<1>();
  __syncthreads();

  uint32_t taken = 0, turn = 0;                           // tiles that the warp has worked on; items so far
  uint32_t w_tile = t_begin + w;                          // the warp's next tile, in the item
  Walk<KT> nw = cw;                                       // the item after
  for (;;) {
    const unsigned long long nx = x0 + cw.nt + kItemTiles;
    bool more = nx + kItemTiles < u1;                     // (a tile of the next item lies in the CTA's run)
    if (more) more = nw.next(a, cap);
    const uint32_t rows = static_cast<uint32_t>(cw.s.n) * a.group;
    const bool any = w_tile < t_end;
    // this thread's rows (columns of the products): 8 g + 2 t4 + e
    Span sp[NR][2];
    // the maximum in use; the exponent that weights are relative to; 8-bit pages: a power of two above the scales that the row has seen
    float sl2[NR][2], m[NR][2], ref[NR][2], l[NR][2], v_ref[NR][2];
    uint32_t qf[NR][HD / 16][2];
    float o[NR][HD / 16][4];
    int32_t full_lo = 0, full_hi = 0x7fffffff;            // keys that all rows see
    if (any) {
#pragma unroll
      for (int g = 0; g < NR; ++g) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) { o[g][i][0] = 0.0f; o[g][i][1] = 0.0f; o[g][i][2] = 0.0f; o[g][i][3] = 0.0f; }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = 8u * g + 2u * t4 + e;
          sp[g][e] = r < rows ? SeenBy(cw.s, static_cast<int32_t>(r / a.group), a.causal, a.window) : Span{0, 0};
          sl2[g][e] = a.scale_log2; m[g][e] = ref[g][e] = -INFINITY; l[g][e] = 0.0f; v_ref[g][e] = power_above(0.0f);
        }
        const uint32_t qb = q_s + (turn & 1u) * Sh::kQ;
        if constexpr (!Q8) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ks += 2) {
            uint32_t b[4];
            ldmatrix_x4(b, qb + chunk_at<HD / 8>(8u * g + (lane & 7u), ks * 2 + (lane >> 3)));
            qf[g][ks][0] = b[0]; qf[g][ks][1] = b[1]; qf[g][ks + 1][0] = b[2]; qf[g][ks + 1][1] = b[3];
          }
        } else {
          float top = 0.0f;
#pragma unroll
          for (int seg = 0; seg < HD / 32; ++seg) {       // eight values side by side: those of product 2 seg first (as K's codes lie)
            const uint4 v = lds_v4(qb + chunk_at<HD / 8>(8u * g + quad, seg * 4 + t4));
            qf[g][2 * seg][0] = v.x; qf[g][2 * seg][1] = v.y; qf[g][2 * seg + 1][0] = v.z; qf[g][2 * seg + 1][1] = v.w;
            if (BF) {
              const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(ww[i] << 16)), fabsf(__uint_as_float(ww[i] & 0xffff0000u))));
            }
          }
          if (BF) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e brings the largest to [2^14, 2^15); rows of zeros, and of what is not finite, stay as they are
            const int ex = static_cast<int>(__float_as_uint(top) >> 23);
            const int e = ex == 0 || ex == 255 ? 0 : min(100, 127 + 14 - ex);      // (-113 and more)
            const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
              for (int i = 0; i < 2; ++i) qf[g][ks][i] = cvt_f16x2(__uint_as_float(qf[g][ks][i] & 0xffff0000u) * up, __uint_as_float(qf[g][ks][i] << 16) * up);
            sl2[g][0] *= __shfl_sync(0xffffffffu, down, 8u * t4);
            sl2[g][1] *= __shfl_sync(0xffffffffu, down, 8u * t4 + 4u);
          }
        }
      }
      if (cw.s.n > 0) {
        full_lo = SeenBy(cw.s, cw.s.n - 1, a.causal, a.window).lo;
        full_hi = SeenBy(cw.s, 0, a.causal, a.window).hi;
      }
    }
    if (more) fetch_q(nw, (turn + 1u) & 1u);              // (on the way with the next tile's copies)
    for (; w_tile < t_end; w_tile += kStepWarps, ++taken) {
      cp_async_wait_all();
      __syncwarp();
      const uint32_t there = keys_next;
      issue();                                            // into the other stage
      const uint32_t st = ring_s + (taken % kStages) * Sh::kStage;
      const int32_t j0 = cw.keys.lo + static_cast<int32_t>(w_tile) * KT;
      float s[NR][MT][4];
#pragma unroll
      for (int g = 0; g < NR; ++g)
#pragma unroll
        for (int t = 0; t < MT; ++t) { s[g][t][0] = 0.0f; s[g][t][1] = 0.0f; s[g][t][2] = 0.0f; s[g][t][3] = 0.0f; }
      if constexpr (!Q8) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t x[4];
            ldmatrix_x4(x, st + chunk_at<CH>(t * 16 + (lane & 15u), ks * 2 + (lane >> 4)));
#pragma unroll
            for (int g = 0; g < NR; ++g) {
              if (BF) mma_bf16_16816(s[g][t], x, qf[g][ks][0], qf[g][ks][1]);
              else mma_f16_16816(s[g][t], x, qf[g][ks][0], qf[g][ks][1]);
            }
          }
      } else {
#pragma unroll
        for (int seg = 0; seg < HD / 32; ++seg)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            // eight codes each of keys `quad` and `quad` + 8, those of product 2 seg first
            uint2 c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(c[i].x), "=r"(c[i].y) : "r"(st + chunk_at<CH>(t * 16 + i * 8 + quad, seg * 2 + (t4 >> 1)) + (t4 & 1u) * 8u) : "memory");
            const uint32_t x0f[4] = {cvt_e4m3x2_f16x2(c[0].x & 0xffffu), cvt_e4m3x2_f16x2(c[1].x & 0xffffu), cvt_e4m3x2_f16x2(c[0].x >> 16), cvt_e4m3x2_f16x2(c[1].x >> 16)};
            const uint32_t x1f[4] = {cvt_e4m3x2_f16x2(c[0].y & 0xffffu), cvt_e4m3x2_f16x2(c[1].y & 0xffffu), cvt_e4m3x2_f16x2(c[0].y >> 16), cvt_e4m3x2_f16x2(c[1].y >> 16)};
#pragma unroll
            for (int g = 0; g < NR; ++g) {
              mma_f16_16816(s[g][t], x0f, qf[g][2 * seg][0], qf[g][2 * seg][1]);
              mma_f16_16816(s[g][t], x1f, qf[g][2 * seg + 1][0], qf[g][2 * seg + 1][1]);
            }
          }
      }
      // keys that the row does not see, or that have no page, at -inf; the thread's keys: 16 t + quad, + 8
      const bool whole = j0 >= full_lo && j0 + KT <= full_hi && there == kAllKeys;
      float vs[MT][2], top[NR][2], v_top[NR][2];
#pragma unroll
      for (int g = 0; g < NR; ++g) { top[g][0] = top[g][1] = -INFINITY; v_top[g][0] = v_top[g][1] = 0.0f; }
      if (Q8) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float ksc = lds_f32(st + 2u * Sh::kBytes + (t * 16 + i * 8 + quad) * 4u);
            vs[t][i] = lds_f32(st + 2u * Sh::kBytes + (KT + t * 16 + i * 8 + quad) * 4u);
#pragma unroll
            for (int g = 0; g < NR; ++g) { s[g][t][2 * i] *= ksc; s[g][t][2 * i + 1] *= ksc; }
          }
      }
      if (whole) {
        if (Q8) {
          float x = 0.0f;
#pragma unroll
          for (int t = 0; t < MT; ++t) x = fmaxf(x, fmaxf(vs[t][0], vs[t][1]));
#pragma unroll
          for (int g = 0; g < NR; ++g) v_top[g][0] = v_top[g][1] = x;
        }
      } else {
#pragma unroll
        for (int g = 0; g < NR; ++g)
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int32_t j = j0 + t * 16 + static_cast<int32_t>(quad) + 8 * (c >> 1);
              const int e = c & 1;
              const bool seen = j >= sp[g][e].lo && j < sp[g][e].hi && ((there >> (t * 16 + quad + 8 * (c >> 1))) & 1u);
              s[g][t][c] = seen ? s[g][t][c] : -INFINITY;
              if (Q8) v_top[g][e] = fmaxf(v_top[g][e], seen ? vs[t][c >> 1] : 0.0f);
            }
      }
      // (a NaN is dropped here; the sum of the weights finds it)
      bool grow = false;
#pragma unroll
      for (int g = 0; g < NR; ++g) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          top[g][0] = max3(top[g][0], s[g][t][0], s[g][t][2]);
          top[g][1] = max3(top[g][1], s[g][t][1], s[g][t][3]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) grow = grow || top[g][e] * sl2[g][e] > m[g][e] + kGrow || (Q8 && v_top[g][e] >= v_ref[g][e]);
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int g = 0; g < NR; ++g) {
          float corr[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[g][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            x *= sl2[g][e];
            if (x > m[g][e] + kGrow) m[g][e] = x;
            if (Q8) {
              float v = v_top[g][e];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
              v_ref[g][e] = fmaxf(v_ref[g][e], power_above(v));
            }
            // p = 2^(s - ref); 8-bit pages: 2^6 / v_ref times as large, so that p times a value's scale is what f16 holds best
            const float r = m[g][e] == -INFINITY ? -INFINITY : Q8 ? m[g][e] - kPHead + static_cast<float>(static_cast<int>(__float_as_uint(v_ref[g][e]) >> 23) - 127) : m[g][e];
            corr[e] = r == ref[g][e] ? 1.0f : ref[g][e] == -INFINITY ? 0.0f : fast_ex2(ref[g][e] - r);
            ref[g][e] = r;
            l[g][e] *= corr[e];
          }
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) { o[g][i][0] *= corr[0]; o[g][i][1] *= corr[1]; o[g][i][2] *= corr[0]; o[g][i][3] *= corr[1]; }
        }
      }
      uint32_t pb[NR][MT][2], pl[NR][MT][2];
#pragma unroll
      for (int g = 0; g < NR; ++g) {
        const float neg[2] = {ref[g][0] == -INFINITY ? 0.0f : -ref[g][0], ref[g][1] == -INFINITY ? 0.0f : -ref[g][1]};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int e = c & 1;
            const float p = fast_ex2(fmaf(s[g][t][c], sl2[g][e], neg[e]));
            l[g][e] += p;
            s[g][t][c] = p;
          }
          if (Q8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) s[g][t][c] = !whole && s[g][t][c] == 0.0f ? 0.0f : s[g][t][c] * vs[t][c >> 1];     // (a scale that the row does not see may be anything)
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float lo = s[g][t][2 * i], hi = s[g][t][2 * i + 1];
            if (BF && !Q8) {
              const uint32_t r = cvt_bf16x2(hi, lo);
              pb[g][t][i] = transposed(r);
              pl[g][t][i] = transposed(cvt_bf16x2(hi - __uint_as_float(r & 0xffff0000u), lo - __uint_as_float(r << 16)));
            } else {
              const uint32_t r = cvt_f16x2(hi, lo);
              pb[g][t][i] = transposed(r);
              if (!BF) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
                pl[g][t][i] = transposed(cvt_f16x2(hi - f.y, lo - f.x));
              }
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) {
        if constexpr (!Q8) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t x[4];
            ldmatrix_x4_trans(x, st + Sh::kBytes + chunk_at<CH>(t * 16 + (lane >> 4) * 8 + (lane & 7u), n * 2 + ((lane >> 3) & 1u)));
#pragma unroll
            for (int g = 0; g < NR; ++g) {
              if (BF) {
                mma_bf16_16816(o[g][n], x, pb[g][t][0], pb[g][t][1]);
                mma_bf16_16816(o[g][n], x, pl[g][t][0], pl[g][t][1]);
              } else {
                mma_f16_16816(o[g][n], x, pb[g][t][0], pb[g][t][1]);
                mma_f16_16816(o[g][n], x, pl[g][t][0], pl[g][t][1]);
              }
            }
          }
        } else {
          // Transposed by pairs of codes: a register holds values 2 quad and 2 quad + 1 of two keys; the even ones are rows 0 to 7 of the
          // product, the odd ones 8 to 15. All 32 keys come at once.
          uint32_t b[4];
          ldmatrix_x4_trans(b, st + Sh::kBytes + chunk_at<CH>(lane, n));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const uint32_t c0 = __byte_perm(b[2 * t], 0u, 0x3120), c1 = __byte_perm(b[2 * t + 1], 0u, 0x3120);
            const uint32_t x[4] = {cvt_e4m3x2_f16x2(c0 & 0xffffu), cvt_e4m3x2_f16x2(c0 >> 16), cvt_e4m3x2_f16x2(c1 & 0xffffu), cvt_e4m3x2_f16x2(c1 >> 16)};
#pragma unroll
            for (int g = 0; g < NR; ++g) {
              mma_f16_16816(o[g][n], x, pb[g][t][0], pb[g][t][1]);
              if (!BF) mma_f16_16816(o[g][n], x, pl[g][t][0], pl[g][t][1]);
            }
          }
        }
      }
      __syncwarp();                                       // the stage is read: it may be filled again
    }
    // ---- the warps' results into the stage each has free ----
    float *slot = reinterpret_cast<float *>(ring + (issued % kStages) * Sh::kStage);
    if (any) {
#pragma unroll
      for (int g = 0; g < NR; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = 8u * g + 2u * t4 + e;
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[g][e] += __shfl_xor_sync(0xffffffffu, l[g][e], d);
          if (quad == 0u) { S.m[w][r] = ref[g][e]; S.l[w][r] = l[g][e]; }
          if (r < rows) {
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
              const float lo = o[g][n][e], hi = o[g][n][2 + e];
              if (Q8) {
                *reinterpret_cast<float2 *>(slot + r * kPitch + n * 16 + 2u * quad) = make_float2(lo, hi);
              } else {
                slot[r * kPitch + n * 16 + quad] = lo;
                slot[r * kPitch + n * 16 + 8u + quad] = hi;
              }
            }
          }
        }
    } else if (lane < 16u) {
      S.m[w][lane] = -INFINITY;
      S.l[w][lane] = 0.0f;
    }
    if (lane == 0u) S.at[w] = (w * kStages + issued % kStages) * Sh::kStage;
    if (!any) {                                           // the next item's q is there (a tile's wait came after it)
      cp_async_commit();
      cp_async_wait_all();
    }
    __syncthreads();
    if (tid == 0u) S.redo[(turn + 1u) & 1u] = 0u;         // the next item's (everybody is done with the one before)
    const bool whole = t_begin == 0u && t_end == cw.nt;
    // partial results: [CTA][first or last item][16 rows][HD + 2]
    constexpr uint32_t kPart = 16u * (HD + 2u);
    float *part = a.part + (static_cast<size_t>(blockIdx.x) * 2u + (t_begin == 0u ? 1u : 0u)) * kPart;
    auto finish = [&](uint32_t r, uint32_t d, float4 x, float mm, float ll) {
      const uint32_t tok = r / a.group, head = cw.h * a.group + (r - tok * a.group);
      const int32_t row = cw.s.first + static_cast<int32_t>(tok);
      const float inv = mm == -INFINITY && ll == 0.0f ? 0.0f : 1.0f / ll;
      x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
      if (d < a.c.hd) {
        uint8_t *p = row_at(a.o, row, head) + 2u * d;
        if ((reinterpret_cast<uintptr_t>(p) & 7u) == 0u) {
          *reinterpret_cast<uint2 *>(p) = BF ? make_uint2(cvt_bf16x2(x.y, x.x), cvt_bf16x2(x.w, x.z)) : make_uint2(cvt_f16x2(x.y, x.x), cvt_f16x2(x.w, x.z));
        } else {
          store_row_value(p, x.x, BF); store_row_value(p + 2, x.y, BF); store_row_value(p + 4, x.z, BF); store_row_value(p + 6, x.w, BF);
        }
        if (cw.s.n > 1 && isfinite(ll) && !(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w))) atomicOr(&S.redo[turn & 1u], 1u << r);
      }
      if (d == 0u && a.lse) a.lse[static_cast<int64_t>(row) * a.q_heads + head] = (mm + log2f(ll)) * 0.69314718055994531f;
    };
    for (uint32_t i = tid; i < rows * (HD / 4); i += kStepThreads) {
      const uint32_t r = i / (HD / 4), d = (i - r * (HD / 4)) * 4u;
      float mm = -INFINITY, ll = 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < kStepWarps; ++k) mm = fmaxf(mm, S.m[k][r]);
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (uint32_t k = 0; k < kStepWarps; ++k) {
        // a warp without a tile of this item has left nothing in its stage; one without a key that the row sees has zeros there
        if (S.m[k][r] == -INFINITY && S.l[k][r] == 0.0f) continue;
        const float f = S.m[k][r] == mm ? 1.0f : fast_ex2(S.m[k][r] - mm);
        const float4 y = *reinterpret_cast<const float4 *>(sm + S.at[k] + (r * kPitch + d) * 4u);
        ll += S.l[k][r] * f;
        x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
      }
      if (whole) {
        finish(r, d, x, mm, ll);
      } else {
        *reinterpret_cast<float4 *>(part + r * HD + d) = x;
        if (d == 0u) { part[16u * HD + r] = mm; part[16u * HD + 16u + r] = ll; }
      }
    }
    __syncthreads();                                      // the stages may be filled again
    bool joined = whole;
    // A part of an item. Its CTAs: those whose runs hold its first and its last tile, and all between. One warp goes on with it, the others with
    // the next item; but of many parts all warps join what the last CTA finds.
    const unsigned long long t0 = x0 + kItemTiles, t1 = t0 + cw.nt;
    const uint32_t c0 = whole ? 0u : static_cast<uint32_t>(((t0 + 1ull) * G - 1ull) / U), c1 = whole ? 0u : static_cast<uint32_t>((t1 * G - 1ull) / U);
    const bool together = c1 - c0 >= 4u;
    if (!whole && (together || w == turn % kStepWarps)) {
      uint32_t last = 0u;
      if (together ? tid == 0u : lane == 0u) {
        __threadfence();
        last = atomicAdd(a.arrived + c0, 1u) == c1 - c0 ? 1u : 0u;
        if (last) a.arrived[c0] = 0u;                     // at rest again: nobody else comes
        __threadfence();
      }
      if (together) {
        if (tid == 0u) S.last = last;
        __syncthreads();
        last = S.last;
      } else {
        last = __shfl_sync(0xffffffffu, last, 0);
        __syncwarp();
      }
      if (last) {
        joined = true;
        for (uint32_t i = together ? tid : lane; i < rows * (HD / 4); i += together ? kStepThreads : 32u) {
          const uint32_t r = i / (HD / 4), d = (i - r * (HD / 4)) * 4u;
          float mm = -INFINITY, ll = 0.0f;
          auto of = [&](uint32_t c) { return a.part + (static_cast<size_t>(c) * 2u + (c == c0 ? 1u : 0u)) * kPart; };
#pragma unroll 8
          for (uint32_t c = c0; c <= c1; ++c) mm = fmaxf(mm, __ldcg(of(c) + 16u * HD + r));
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
          for (uint32_t c = c0; c <= c1; ++c) {
            const float *p = of(c);
            const float mc = __ldcg(p + 16u * HD + r), lc = __ldcg(p + 16u * HD + 16u + r);
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(p + r * HD + d));
            const float f = mc == mm ? 1.0f : fast_ex2(mc - mm);
            ll += lc * f;
            x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
          }
          finish(r, d, x, mm, ll);
        }
        if (together) __syncthreads();
        else __syncwarp();
      }
    }
    const uint32_t redo = joined ? *reinterpret_cast<volatile uint32_t *>(&S.redo[turn & 1u]) : 0u;
    if (redo) {
      const bool all = whole || together;                 // (else one warp is here)
      for (uint32_t r = all ? w : 0u; r < rows; r += all ? kStepWarps : 1u)
        if ((redo >> r) & 1u) attend_row_alone(a, cw.b, cw.s, static_cast<int32_t>(r / a.group), cw.h * a.group + r % a.group, 0u, HD, nullptr);
    }
    if (!more) break;
    w_tile -= t_end;                                      // (the warps take the CTA's tiles in turn, across items)
    x0 = nx;
    cw = nw;
    t_begin = 0;
    t_end = tile_at(u1, x0, cw.nt);
    ++turn;
  }
  cp_async_wait_all();
}

template <bool BF, bool Q8, int HD, int NR, int NW>
int Launch(const AttendArgs &a, uint32_t sms, cudaStream_t stream) {
  b2_attend_step<BF, Q8, HD, NR, NW><<<sms * PerSm(NW), NW * 32, StepShape<Q8, HD, NR, NW>::kSmem, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
template <bool BF, bool Q8, int HD, int NR, int NW>
cudaError_t Attr() {
  return cudaFuncSetAttribute(b2_attend_step<BF, Q8, HD, NR, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, StepShape<Q8, HD, NR, NW>::kSmem);
}
// 9 to 16 rows: CTAs of eight warps, whose threads may have 255 registers (with twelve warps and 168, 500 bytes of them were spilled: 32 sequences
// of 4000 to 8000 tokens, 16 heads to each of 4 cache heads, 8-bit pages: 81 us, 111 so).
// Up to 8 rows: items (sequences x cache heads) for no more than the SMs go to CTAs of twelve warps, of which few share an item (8 heads of 131000 keys,
// bf16: 90 us, 137 with CTAs of three); more items to CTAs of three, which lose less at an item's end (64 sequences of 200 to 16000 tokens, 8 heads, 8-bit
// pages: 110 us, 120 with CTAs of six).
template <bool BF, bool Q8, int HD>
int Choose(const AttendArgs &a, uint32_t sms, cudaStream_t s) {
  if (a.b.max_rows * a.group > 8u) return Launch<BF, Q8, HD, 2, 8>(a, sms, s);
  return static_cast<uint64_t>(a.b.n_seqs) * a.c.heads <= sms ? Launch<BF, Q8, HD, 1, 12>(a, sms, s) : Launch<BF, Q8, HD, 1, 3>(a, sms, s);
}
template <bool BF, bool Q8>
int Dim(const AttendArgs &a, uint32_t sms, cudaStream_t s) { return a.c.hd > 64u ? Choose<BF, Q8, 128>(a, sms, s) : Choose<BF, Q8, 64>(a, sms, s); }
template <bool BF, bool Q8>
cudaError_t Attrs() {
  for (cudaError_t e : {Attr<BF, Q8, 64, 2, 8>(), Attr<BF, Q8, 64, 1, 12>(), Attr<BF, Q8, 64, 1, 3>(), Attr<BF, Q8, 128, 2, 8>(), Attr<BF, Q8, 128, 1, 12>(), Attr<BF, Q8, 128, 1, 3>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace

int PrepareAttendStep() {
  for (cudaError_t e : {Attrs<true, false>(), Attrs<false, false>(), Attrs<true, true>(), Attrs<false, true>()})
    if (e != cudaSuccess) return static_cast<int>(e);
  return 0;
}
size_t AttendStepPartialBytes(uint32_t sms) { return static_cast<size_t>(sms) * PerSm(3) * 2u * 16u * (128u + 2u) * sizeof(float); }

int LaunchAttendStep(const AttendArgs &a, uint32_t sms, CUstream_st *stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a.e4m3) return a.bf16 ? Dim<true, true>(a, sms, s) : Dim<false, true>(a, sms, s);
  return a.bf16 ? Dim<true, false>(a, sms, s) : Dim<false, false>(a, sms, s);
}

}  // namespace b2
