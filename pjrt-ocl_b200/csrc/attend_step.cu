// Attention of a few rows of each sequence over the paged cache: decode steps. rows x (query heads to a cache head) <= 16.
//
// One pass over the keys with the running maximum m and sum l of the softmax (base 2): for a tile of keys s = q k^T scale log2 e,
// m' = max(m, s), p = 2^(s - m'), l = l 2^(m - m') + sum p, o = o 2^(m - m') + p v; the result is o / l.
//
// Bound: HBM, K and V of every visible key read once. The query heads that share a cache head are the rows of one 16-row
// product (m16n8k16 warp-level products: at most 16 multiplications to a byte, far from any tensor rate, and their results come in
// registers, where the softmax wants them).
// Work: a cache head of a sequence is an item, cut into tiles of 16 or 32 keys. All tiles of the batch in a row are dealt to the CTAs in
// equal runs (one CTA to an SM), whatever the lengths; a CTA's eight warps take its tiles in turn, each with a ring of three
// stages of its own (K and V of a tile, 8 KB, by 16-byte asynchronous copies, page by page), so that a warp always has two tiles on
// the way and no barrier stands between tiles. At an item's end the warps' (m, l, o) are joined through the stage each has free; an
// item that is split between CTAs leaves partial results, and the CTA that comes last joins them in the CTAs' order.
// 8-bit pages: codes are exact in f16, so the products are f16 x f16 whatever the rows' type. q of type bf16 is scaled by a power of
// two for each row so that its largest value is near 2^14 (f16 then holds what bf16 held to 2^-38 of that); a key's scale goes onto its
// scores, a value's onto p, relative to a power of two not below any scale so far (p v's factor stays in f16's normal range).
// bf16 pages: p is split into two bf16 values (p and what rounding left), since the second product costs nothing here; the result is
// then only rounded once, as it is stored.
#include "attend_common.cuh"

namespace b2 {
namespace {

constexpr uint32_t kStepWarps = 8, kStepThreads = kStepWarps * 32, kStages = 3;
constexpr float kPScale = 16384.0f;      // 8-bit pages: p = 1 on the largest scale, in f16

template <bool Q8, int HD>
struct StepShape {
  static constexpr int KT = (Q8 || HD == 64) ? 32 : 16;       // keys of a tile
  static constexpr int CH = HD * (Q8 ? 1 : 2) / 16;           // 16-byte chunks of a row
  static constexpr int kBytes = KT * CH * 16;                 // K (or V) of a tile
  static constexpr int kScales = Q8 ? 2 * KT * 4 : 0;
  static constexpr int kStage = 2 * kBytes + kScales;
  static constexpr int kSmem = static_cast<int>(kStepWarps * kStages) * kStage;
  static_assert(2 * kBytes >= 16 * HD * 4, "a stage holds a warp's result");
};
// Chunk of a row in shared memory: eight rows of the same chunk lie in different banks.
template <int CH>
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t c) {
  return (row * CH + (CH >= 8 ? (c ^ (row & 7u)) : (c ^ ((row >> 1) & 3u)))) * 16u;
}

struct StepShared {
  float m[kStepWarps][16], l[kStepWarps][16];
  unsigned long long sum[kStepWarps], scan[kStepWarps];
  unsigned long long total;
  uint32_t found_seq;
  unsigned long long found_base;
  uint32_t last, redo[2];           // by turns: an item's rows to be worked out again
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
  __device__ __forceinline__ void next(const AttendArgs &a, uint64_t cap) {
    if (++h < a.c.heads) return;
    h = 0;
    do {
      ++b;
      if (b >= a.b.n_seqs) { nt = 0xffffffffu; return; }      // (nobody walks beyond the last item)
      load(a, cap);
    } while (nt == 0u);
  }
};

template <bool BF, bool Q8, int HD>
__global__ void __launch_bounds__(kStepThreads, 1) b2_attend_step(const __grid_constant__ AttendArgs a) {
  using Sh = StepShape<Q8, HD>;
  constexpr int KT = Sh::KT, CH = Sh::CH, NT = KT / 8;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ StepShared S;
  const uint32_t tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u, quad = lane >> 2, t4 = lane & 3u;
  const uint64_t cap = capacity_of(a.c, a.b);
  // ---- how many tiles there are, and where this CTA's run of them begins ----
  auto tiles_of = [&](uint32_t i) -> unsigned long long {
    Walk<KT> x;
    x.b = i; x.h = 0;
    x.load(a, cap);
    if (x.s.bad && blockIdx.x == 0u) cache_fault(a.c.status, kStBadBatch, i, static_cast<uint32_t>(x.s.bad), static_cast<uint32_t>(x.s.value));
    return static_cast<unsigned long long>(x.nt) * a.c.heads;
  };
  unsigned long long mine = 0;
  for (uint32_t i = tid; i < a.b.n_seqs; i += kStepThreads) mine += tiles_of(i);
  const unsigned long long sum = warp_reduce(mine, [](unsigned long long x, unsigned long long y) { return x + y; });
  if (lane == 0u) S.sum[w] = sum;
  if (tid == 0u) S.redo[0] = 0u;
  __syncthreads();
  unsigned long long U = 0;
#pragma unroll
  for (uint32_t i = 0; i < kStepWarps; ++i) U += S.sum[i];
  if (U == 0ull) return;
  // every CTA that takes part has a tile for each of its warps, where there are as many
  unsigned long long G = U / kStepWarps;
  G = G < 1ull ? 1ull : G > gridDim.x ? gridDim.x : G;
  if (blockIdx.x >= G) return;
  const unsigned long long u0 = U * blockIdx.x / G, u1 = U * (blockIdx.x + 1ull) / G;
  {
    unsigned long long run = 0;
    for (uint32_t i0 = 0; i0 < a.b.n_seqs; i0 += kStepThreads) {
      const uint32_t i = i0 + tid;
      const unsigned long long v = i < a.b.n_seqs ? (a.b.n_seqs <= kStepThreads ? mine : tiles_of(i)) : 0ull;
      unsigned long long x = v;
#pragma unroll
      for (uint32_t o = 1; o < 32u; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31u) S.scan[w] = x;
      __syncthreads();
      unsigned long long before = run;
      for (uint32_t k = 0; k < kStepWarps; ++k) {
        if (k < w) before += S.scan[k];
        run += S.scan[k];
      }
      if (before + x > u0 && before + x - v <= u0) {
        S.found_seq = i;
        S.found_base = before + x - v;
      }
      if (run > u0) break;                                // (the same for all threads)
    }
    __syncthreads();
  }
  Walk<KT> cw;                                            // the item being worked on
  cw.b = S.found_seq;
  cw.load(a, cap);
  cw.h = static_cast<uint32_t>((u0 - S.found_base) / cw.nt);
  uint32_t t_begin = static_cast<uint32_t>((u0 - S.found_base) - static_cast<unsigned long long>(cw.h) * cw.nt);

  // ---- the warp's copies: its tiles are w, w + 8, .. of the CTA's ----
  uint8_t *const ring = sm + w * (kStages * Sh::kStage);
  const uint32_t ring_s = smem_addr(ring);
  Walk<KT> pw = cw;                                       // the item of the next tile to fetch
  unsigned long long pt = static_cast<unsigned long long>(t_begin) + w;     // its tile in that item
  unsigned long long p_left = u1 - u0 > w ? (u1 - u0 - w + kStepWarps - 1ull) / kStepWarps : 0ull;    // tiles still to fetch
  uint32_t issued = 0;
  int32_t page = -1;                                      // page number of the lane's key in that tile
  uint32_t key_slot = 0, key_entry = 0;
  bool key_live = false;
  auto look_ahead = [&]() {                               // the next tile's place, and its keys' pages on the way
    if (p_left == 0ull) return;
    while (pt >= pw.nt) { pt -= pw.nt; pw.next(a, cap); }
    const int32_t j = pw.keys.lo + static_cast<int32_t>(pt) * KT + static_cast<int32_t>(lane);
    key_live = lane < KT && j < pw.keys.hi;
    if (key_live) {
      key_entry = a.c.by_page.quot(static_cast<uint32_t>(j));
      key_slot = static_cast<uint32_t>(j) - key_entry * a.c.page_size;
      page = __ldg(a.b.pages + static_cast<int64_t>(pw.b) * a.b.pages_stride + key_entry);
    }
  };
  auto issue = [&]() {
    if (p_left != 0ull) {
      const uint32_t st = ring_s + (issued % kStages) * Sh::kStage;
      int64_t off = 0;
      bool live = key_live;
      if (live && static_cast<uint32_t>(page) >= a.c.n_pages) {
        cache_fault(a.c.status, kStBadPage, pw.b, key_entry, static_cast<uint32_t>(page));
        live = false;
      }
      if (live) off = page * a.c.page_bytes + key_slot * a.c.slot_bytes + pw.h * a.c.head_bytes;
      const uint32_t mask = __ballot_sync(0xffffffffu, live);
      constexpr int kRowsAtOnce = 32 / CH;
      const uint32_t sub = lane % CH, r0 = lane / CH;
      const bool in_hd = sub * 16u < a.c.hd * (Q8 ? 1u : 2u);
#pragma unroll
      for (int i = 0; i < KT / kRowsAtOnce; ++i) {
        const uint32_t r = i * kRowsAtOnce + r0;
        const int64_t o = __shfl_sync(0xffffffffu, off, r);
        const uint32_t bytes = ((mask >> r) & 1u) && in_hd ? 16u : 0u;         // else zeros
        const int64_t at = bytes ? o + sub * 16u : 0;
        const uint32_t dst = st + chunk_at<CH>(r, sub);
        cp_async_16_zfill(dst, a.c.k + at, bytes);
        cp_async_16_zfill(dst + Sh::kBytes, a.c.v + at, bytes);
      }
      if (Q8) {
        const int64_t so = live ? page * a.c.s_page + key_slot * a.c.s_slot + pw.h * a.c.s_head : 0;
        const uint32_t dst = st + 2u * Sh::kBytes + lane * 4u;
        cp_async_4_zfill(dst, a.c.ks + so, live ? 4u : 0u);
        cp_async_4_zfill(dst + KT * 4u, a.c.vs + so, live ? 4u : 0u);
      }
      --p_left;
      pt += kStepWarps;
    }
    cp_async_commit();
    ++issued;
    look_ahead();
  };
  look_ahead();
  issue();
  issue();

  uint32_t taken = 0, turn = 0;                           // tiles that the warp has worked on; items so far
  unsigned long long u = u0;
  unsigned long long wu = u0 + w;                         // the warp's next tile among all
  while (u < u1) {
    const uint32_t t_end = static_cast<uint32_t>(min(static_cast<unsigned long long>(cw.nt), t_begin + (u1 - u)));
    const unsigned long long u_end = u + (t_end - t_begin);
    const uint32_t rows = static_cast<uint32_t>(cw.s.n) * a.group;
    // this thread's rows of the products: quad and quad + 8
    Span sp[2];
    float sl2[2] = {a.scale_log2, a.scale_log2};
    uint32_t qf[HD / 16][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[HD / 8][4];
    const bool any = wu < u_end;
    if (any) {
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) { o[i][0] = 0.0f; o[i][1] = 0.0f; o[i][2] = 0.0f; o[i][3] = 0.0f; }
      float top[2] = {0.0f, 0.0f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t r = quad + 8u * half, tok = r / a.group;
        const bool live = r < rows;
        sp[half] = live ? SeenBy(cw.s, static_cast<int32_t>(tok), a.causal, a.window) : Span{0, 0};
        const uint8_t *p = live ? row_at(a.q, cw.s.first + static_cast<int32_t>(tok), cw.h * a.group + (r - tok * a.group)) : a.q.p;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int b8 = 0; b8 < 2; ++b8) {
            // 8-bit pages: a thread's values of two products lie side by side (see the K operand below)
            const uint32_t d = Q8 ? (ks >> 1) * 32u + 8u * t4 + 4u * (ks & 1) + 2u * b8 : ks * 16u + 2u * t4 + 8u * b8;
            uint32_t v = 0u;
            if (live && d < a.c.hd) v = *reinterpret_cast<const uint16_t *>(p + 2u * d) | (static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(p + 2u * d + 2u)) << 16);
            qf[ks][half + 2 * b8] = v;
            if (Q8 && BF) top[half] = fmaxf(top[half], fmaxf(fabsf(__uint_as_float(v << 16)), fabsf(__uint_as_float(v & 0xffff0000u))));
          }
      }
      if (Q8 && BF) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          // 2^e brings the largest to [2^14, 2^15); rows of zeros, and of what is not finite, stay as they are
          const int ex = static_cast<int>(__float_as_uint(x) >> 23);
          const int e = ex == 0 || ex == 255 ? 0 : max(-100, min(100, 127 + 14 - ex));
          const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          sl2[half] = a.scale_log2 * down;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
            for (int b8 = 0; b8 < 2; ++b8) {
              const uint32_t v = qf[ks][half + 2 * b8];
              qf[ks][half + 2 * b8] = cvt_f16x2(__uint_as_float(v & 0xffff0000u) * up, __uint_as_float(v << 16) * up);
            }
        }
      }
    }
    float v_ref[2] = {0.0f, 0.0f};                        // 8-bit pages: power of two not below the scales that the row has seen, 0 = none yet
    for (; wu < u_end; wu += kStepWarps, ++taken) {
      cp_async_wait<1>();
      __syncwarp();
      issue();                                            // into the stage before last
      const uint32_t st = ring_s + (taken % kStages) * Sh::kStage;
      const int32_t j0 = cw.keys.lo + static_cast<int32_t>(t_begin + static_cast<uint32_t>(wu - u)) * KT;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) { s[n][0] = 0.0f; s[n][1] = 0.0f; s[n][2] = 0.0f; s[n][3] = 0.0f; }
      if constexpr (!Q8) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            uint32_t b[4];
            ldmatrix_x4(b, st + chunk_at<CH>(np * 16 + (lane >> 4) * 8 + (lane & 7u), ks * 2 + ((lane >> 3) & 1u)));
            if (BF) { mma_bf16_16816(s[2 * np], qf[ks], b[0], b[1]); mma_bf16_16816(s[2 * np + 1], qf[ks], b[2], b[3]); }
            else { mma_f16_16816(s[2 * np], qf[ks], b[0], b[1]); mma_f16_16816(s[2 * np + 1], qf[ks], b[2], b[3]); }
          }
      } else {
#pragma unroll
        for (int seg = 0; seg < HD / 32; ++seg)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            // eight codes of key `quad`, those of product 2 seg first; the order along d is Q's
            uint2 c;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(c.x), "=r"(c.y) : "r"(st + chunk_at<CH>(n * 8 + quad, seg * 2 + (t4 >> 1)) + (t4 & 1u) * 8u) : "memory");
            mma_f16_16816(s[n], qf[2 * seg], cvt_e4m3x2_f16x2(c.x & 0xffffu), cvt_e4m3x2_f16x2(c.x >> 16));
            mma_f16_16816(s[n], qf[2 * seg + 1], cvt_e4m3x2_f16x2(c.y & 0xffffu), cvt_e4m3x2_f16x2(c.y >> 16));
          }
      }
      // scores in the log2 domain, keys that the row does not see at -inf
      float mx[2] = {-INFINITY, -INFINITY}, v_top[2] = {0.0f, 0.0f};
      float2 vs2[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 ks2 = make_float2(1.0f, 1.0f);
        if (Q8) {
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ks2.x), "=f"(ks2.y) : "r"(st + 2u * Sh::kBytes + (n * 8 + 2u * t4) * 4u) : "memory");
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(vs2[n].x), "=f"(vs2[n].y) : "r"(st + 2u * Sh::kBytes + (KT + n * 8 + 2u * t4) * 4u) : "memory");
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int32_t j = j0 + n * 8 + static_cast<int32_t>(2u * t4) + (c & 1);
          const float x = s[n][c] * (Q8 ? sl2[c >> 1] * ((c & 1) ? ks2.y : ks2.x) : sl2[c >> 1]);
          const bool seen = j >= sp[c >> 1].lo && j < sp[c >> 1].hi;
          s[n][c] = seen ? x : -INFINITY;
          if (Q8) v_top[c >> 1] = fmaxf(v_top[c >> 1], seen ? ((c & 1) ? vs2[n].y : vs2[n].x) : 0.0f);
          // (a NaN must not be lost here: fmaxf would drop it, and the sum below finds it again)
          mx[c >> 1] = fmaxf(mx[c >> 1], s[n][c]);
        }
      }
      float corr[2];
      bool moved = false;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
        const float m2 = fmaxf(m[half], mx[half]);
        corr[half] = m[half] == m2 ? 1.0f : m[half] == -INFINITY ? 0.0f : fast_ex2(m[half] - m2);
        moved = moved || corr[half] != 1.0f;
        m[half] = m2;
        l[half] *= corr[half];
      }
      float v_mul[2] = {1.0f, 1.0f};
      if (Q8) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = fmaxf(v_top[half], __shfl_xor_sync(0xffffffffu, v_top[half], 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          const float ref = __uint_as_float(min(250u, max(4u, (__float_as_uint(x) >> 23) + 1u)) << 23);
          if (ref > v_ref[half]) {
            corr[half] *= v_ref[half] / ref;              // (a power of two, or 0 at first)
            moved = true;
            v_ref[half] = ref;
          }
          v_mul[half] = kPScale / v_ref[half];
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) { o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1]; }
      }
      const float neg[2] = {m[0] == -INFINITY ? 0.0f : -m[0], m[1] == -INFINITY ? 0.0f : -m[1]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float p = fast_ex2(s[n][c] + neg[c >> 1]);
          l[c >> 1] += p;
          s[n][c] = Q8 ? (p == 0.0f ? 0.0f : p * (((c & 1) ? vs2[n].y : vs2[n].x) * v_mul[c >> 1])) : p;
        }
      }
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk) {
        const float(&x)[4] = s[2 * kk];
        const float(&y)[4] = s[2 * kk + 1];
        uint32_t pa[4], pl[4];
        if (BF && !Q8) {
          pa[0] = cvt_bf16x2(x[1], x[0]); pa[1] = cvt_bf16x2(x[3], x[2]); pa[2] = cvt_bf16x2(y[1], y[0]); pa[3] = cvt_bf16x2(y[3], y[2]);
          auto left = [](float hi, float lo, uint32_t r) { return cvt_bf16x2(hi - __uint_as_float(r & 0xffff0000u), lo - __uint_as_float(r << 16)); };
          pl[0] = left(x[1], x[0], pa[0]); pl[1] = left(x[3], x[2], pa[1]); pl[2] = left(y[1], y[0], pa[2]); pl[3] = left(y[3], y[2], pa[3]);
        } else {
          pa[0] = cvt_f16x2(x[1], x[0]); pa[1] = cvt_f16x2(x[3], x[2]); pa[2] = cvt_f16x2(y[1], y[0]); pa[3] = cvt_f16x2(y[3], y[2]);
        }
#pragma unroll
        for (int n2 = 0; n2 < HD / 16; ++n2) {
          uint32_t b[4];
          if constexpr (!Q8) {
            ldmatrix_x4_trans(b, st + Sh::kBytes + chunk_at<CH>(kk * 16 + ((lane >> 3) & 1u) * 8 + (lane & 7u), n2 * 2 + (lane >> 4)));
            if (BF) {
              mma_bf16_16816(o[2 * n2], pa, b[0], b[1]); mma_bf16_16816(o[2 * n2 + 1], pa, b[2], b[3]);
              mma_bf16_16816(o[2 * n2], pl, b[0], b[1]); mma_bf16_16816(o[2 * n2 + 1], pl, b[2], b[3]);
            } else {
              mma_f16_16816(o[2 * n2], pa, b[0], b[1]); mma_f16_16816(o[2 * n2 + 1], pa, b[2], b[3]);
            }
          } else if (kk == 0) {
            // Transposed by pairs of codes: a register holds d = 2 quad and 2 quad + 1 of two keys; split, the even and the odd values of
            // the 16 are one column tile each. Both halves of the 32 keys come at once.
            ldmatrix_x4_trans(b, st + Sh::kBytes + chunk_at<CH>((lane >> 3) * 8 + (lane & 7u), n2));
            uint32_t pb[4];
            const float(&x2)[4] = s[NT > 2 ? 2 : 0];
            const float(&y2)[4] = s[NT > 2 ? 3 : 1];
            pb[0] = cvt_f16x2(x2[1], x2[0]); pb[1] = cvt_f16x2(x2[3], x2[2]); pb[2] = cvt_f16x2(y2[1], y2[0]); pb[3] = cvt_f16x2(y2[3], y2[2]);
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
              const uint32_t c0 = __byte_perm(b[2 * k2], 0u, 0x3120), c1 = __byte_perm(b[2 * k2 + 1], 0u, 0x3120);
              mma_f16_16816(o[2 * n2], k2 ? pb : pa, cvt_e4m3x2_f16x2(c0 & 0xffffu), cvt_e4m3x2_f16x2(c1 & 0xffffu));
              mma_f16_16816(o[2 * n2 + 1], k2 ? pb : pa, cvt_e4m3x2_f16x2(c0 >> 16), cvt_e4m3x2_f16x2(c1 >> 16));
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
      for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        const uint32_t r = quad + 8u * half;
        if (t4 == 0u) { S.m[w][r] = m[half]; S.l[w][r] = l[half]; }
        const float mul = Q8 ? v_ref[half] * (1.0f / kPScale) : 1.0f;
        if (r < rows) {
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            const float x0 = o[2 * i][2 * half] * mul, x1 = o[2 * i][2 * half + 1] * mul, y0 = o[2 * i + 1][2 * half] * mul, y1 = o[2 * i + 1][2 * half + 1] * mul;
            if (Q8) {
              *reinterpret_cast<float4 *>(slot + r * HD + i * 16 + 4u * t4) = make_float4(x0, y0, x1, y1);
            } else {
              *reinterpret_cast<float2 *>(slot + r * HD + i * 16 + 2u * t4) = make_float2(x0, x1);
              *reinterpret_cast<float2 *>(slot + r * HD + i * 16 + 8u + 2u * t4) = make_float2(y0, y1);
            }
          }
        }
      }
    } else if (lane < 16u) {
      S.m[w][lane] = -INFINITY;
      S.l[w][lane] = 0.0f;
    }
    // where each warp's stage is: all warps have issued the same number or one less; the number is left beside m
    if (lane == 0u) S.scan[w] = issued % kStages;
    __syncthreads();
    if (tid == 0u) S.redo[(turn + 1u) & 1u] = 0u;         // the next item's (everybody is done with the one before)
    const bool whole = t_begin == 0u && t_end == cw.nt;
    const unsigned long long item0 = u - t_begin, item1 = item0 + cw.nt;      // the item's tiles among all
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
        if (cw.s.n > 1 && !(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w))) atomicOr(&S.redo[turn & 1u], 1u << r);
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
        const float4 y = *reinterpret_cast<const float4 *>(sm + k * (kStages * Sh::kStage) + S.scan[k] * Sh::kStage + (r * HD + d) * 4u);
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
    if (!whole) {
      // the item's CTAs: those whose runs hold its first and its last tile, and all between
      const uint32_t c0 = static_cast<uint32_t>(((item0 + 1ull) * G - 1ull) / U), c1 = static_cast<uint32_t>((item1 * G - 1ull) / U);
      __threadfence();
      __syncthreads();
      if (tid == 0u) {
        const uint32_t old = atomicAdd(a.arrived + c0, 1u);
        S.last = old == c1 - c0 ? 1u : 0u;
        if (S.last) a.arrived[c0] = 0u;                   // at rest again: nobody else comes
      }
      __syncthreads();
      if (S.last) {
        __threadfence();
        for (uint32_t i = tid; i < rows * (HD / 4); i += kStepThreads) {
          const uint32_t r = i / (HD / 4), d = (i - r * (HD / 4)) * 4u;
          float mm = -INFINITY, ll = 0.0f;
          auto of = [&](uint32_t c) { return a.part + (static_cast<size_t>(c) * 2u + (c == c0 ? 1u : 0u)) * kPart; };
          for (uint32_t c = c0; c <= c1; ++c) mm = fmaxf(mm, __ldcg(of(c) + 16u * HD + r));
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
      }
    }
    __syncthreads();                                      // the stages may be filled again
    const uint32_t redo = S.redo[turn & 1u];
    if (redo && (whole || S.last)) {
      for (uint32_t r = w; r < rows; r += kStepWarps)
        if ((redo >> r) & 1u) attend_row_alone(a, cw.b, cw.s, static_cast<int32_t>(r / a.group), cw.h * a.group + r % a.group);
    }
    u = u_end;
    ++turn;
    t_begin = 0;
    if (u < u1) cw.next(a, cap);
  }
  cp_async_wait_all();
}

template <bool BF, bool Q8, int HD>
int Launch(const AttendArgs &a, uint32_t sms, cudaStream_t stream) {
  b2_attend_step<BF, Q8, HD><<<sms, kStepThreads, StepShape<Q8, HD>::kSmem, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
template <bool BF, bool Q8, int HD>
cudaError_t Attr() {
  return cudaFuncSetAttribute(b2_attend_step<BF, Q8, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, StepShape<Q8, HD>::kSmem);
}

}  // namespace

int PrepareAttendStep() {
  for (cudaError_t e : {Attr<true, false, 64>(), Attr<true, false, 128>(), Attr<false, false, 64>(), Attr<false, false, 128>(), Attr<true, true, 64>(), Attr<true, true, 128>(),
                        Attr<false, true, 64>(), Attr<false, true, 128>()})
    if (e != cudaSuccess) return static_cast<int>(e);
  return 0;
}
size_t AttendStepPartialBytes(uint32_t sms) { return static_cast<size_t>(sms) * 2u * 16u * (128u + 2u) * sizeof(float); }

int LaunchAttendStep(const AttendArgs &a, uint32_t sms, CUstream_st *stream) {
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
