// A batch's rows of K and V into the pages of a cache, quantised to e4m3 where the pages are, and back out of them.
//
// e4m3: s = max|x| / 448, code = x / s to the nearest, both as IEEE divisions, so that the codes are those of the definition to
// the bit. The largest magnitude is taken over the values' bit patterns, where NaN is above infinity: a row that holds either
// gets a scale that is not finite and reads back as NaN throughout.
//
// Bound: HBM, each row read and written once. A CTA takes some tokens at a time: its warps look up which sequence each belongs
// to (32 starts at a time) and where its position lies, all tokens' lookups at once; then threads move the tokens' 2 x heads
// rows, 8 values to a thread, two rows' worth of loads in flight each.
#include "operators_dev.cuh"

namespace b2 {
namespace {

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;
constexpr uint32_t kMoveTokens = 16;

template <typename R>
__device__ __forceinline__ void load8(const R *p, bool vec, float (&x)[8]) {
  if (vec) {
    constexpr int W = 16 / sizeof(R);
#pragma unroll
    for (int j = 0; j < 8 / W; ++j) {
      const Vec<R, W> a = reinterpret_cast<const Vec<R, W> *>(p)[j];
#pragma unroll
      for (int i = 0; i < W; ++i) x[j * W + i] = ToF(a.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ToF(p[i]);
  }
}
template <typename R>
__device__ __forceinline__ void store8(R *p, bool vec, const float (&x)[8]) {
  if (vec) {
    constexpr int W = 16 / sizeof(R);
#pragma unroll
    for (int j = 0; j < 8 / W; ++j) {
      Vec<R, W> a;
#pragma unroll
      for (int i = 0; i < W; ++i) a.v[i] = FromF<R>(x[j * W + i]);
      reinterpret_cast<Vec<R, W> *>(p)[j] = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = FromF<R>(x[i]);
  }
}

struct MoveShape {
  uint32_t tokens, lanes;          // tokens of a CTA at a time, threads to a row (a power of two)
  uint32_t vec[2];                 // rows of K, V: 16-byte accesses
  FastDiv by_heads;
};

// R: type of the rows, P: of the pages.
template <typename R, typename P, bool WRITE>
__global__ void __launch_bounds__(kMoveThreads) b2_cache_move(const __grid_constant__ CacheView c, const __grid_constant__ BatchView b, const __grid_constant__ RowsRef kr,
                                                              const __grid_constant__ RowsRef vr, const __grid_constant__ MoveShape s) {
  constexpr bool Q8 = sizeof(P) == 1;
  __shared__ int64_t at_s[kMoveTokens], scale_s[kMoveTokens];     // -1: nothing there, -2: the row is nobody's
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint64_t cap = capacity_of(c, b);
  const uint32_t sub = tid & (s.lanes - 1u), slot0 = tid / s.lanes, slots = kMoveThreads / s.lanes;
  const bool has = sub * 8u < c.hd;
  if (blockIdx.x == 0u) {                                 // batches that do not fit are named even where they have no row
    for (uint32_t i = tid; i < b.n_seqs; i += kMoveThreads) {
      const Seq q = load_seq(b, cap, i);
      if (q.bad) cache_fault(c.status, kStBadBatch, i, static_cast<uint32_t>(q.bad), static_cast<uint32_t>(q.value));
    }
  }
  for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * s.tokens; base < b.n_rows; base += static_cast<uint64_t>(gridDim.x) * s.tokens) {
    const uint32_t tok0 = static_cast<uint32_t>(base), n_tok = min(tok0 + s.tokens, b.n_rows) - tok0;
    __syncthreads();                                      // the places before have been used
    for (uint32_t t = warp; t < n_tok; t += kMoveWarps) {
      const int32_t i = static_cast<int32_t>(tok0 + t);
      const uint32_t q = seq_of_row(b.row_start, b.n_seqs, i);
      if (lane == 0u) {
        const Seq sq = load_seq(b, cap, q);
        int64_t at = -2, sc = 0;
        if (i >= sq.first && i - sq.first < sq.n) {
          const int32_t p = sq.len - sq.n + (i - sq.first);
          at = p >= 0 ? page_offset(c, b, q, static_cast<uint32_t>(p), &sc) : -1;
        }
        at_s[t] = at;
        scale_s[t] = sc;
      }
    }
    __syncthreads();
    const uint32_t rows = n_tok * 2u * c.heads;
    for (uint32_t r0 = 0; r0 < rows; r0 += 2u * slots) {
      float x[2][8];
      int64_t at[2];
      uint32_t tok[2], h[2], kv[2];
      float scale[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t r = r0 + static_cast<uint32_t>(j) * slots + slot0;
        const uint32_t th = s.by_heads.quot(r);           // token and K or V; the heads run fastest
        h[j] = r - th * c.heads; kv[j] = th & 1u; tok[j] = th >> 1;
        at[j] = r < rows ? at_s[tok[j]] : -2;
        scale[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
        if (at[j] < 0) continue;
        if (WRITE) {
          const RowsRef &rr = kv[j] ? vr : kr;
          if (has) load8(reinterpret_cast<const R *>(rr.p) + static_cast<int64_t>(base + tok[j]) * rr.row + static_cast<int64_t>(h[j]) * rr.head + sub * 8u, s.vec[kv[j]] != 0u, x[j]);
        } else {
          const uint8_t *p = (kv[j] ? c.v : c.k) + at[j] + h[j] * c.head_bytes + sub * 8u * sizeof(P);
          if constexpr (Q8) {
            scale[j] = (kv[j] ? c.vs : c.ks)[scale_s[tok[j]] + h[j] * c.s_head];
            if (has) {
              const uint2 w = *reinterpret_cast<const uint2 *>(p);
              const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(ww[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
                const float2 f = __half22float2(__half2(hr));
                x[j][2 * i] = f.x;
                x[j][2 * i + 1] = f.y;
              }
            }
          } else if (has) {
            load8(reinterpret_cast<const P *>(p), true, x[j]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (WRITE) {
          if constexpr (Q8) {
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[j][i]) & 0x7fffffffu);
            for (uint32_t o = s.lanes >> 1; o > 0u; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float sc = __fdiv_rn(__uint_as_float(m), 448.0f);
            if (at[j] >= 0) {
              if (has) {
                uint32_t w[2] = {0u, 0u};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float v = sc == 0.0f ? 0.0f : __fdiv_rn(x[j][i], sc);
                  w[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3)) << (8 * (i & 3));
                }
                *reinterpret_cast<uint2 *>((kv[j] ? c.v : c.k) + at[j] + h[j] * c.head_bytes + sub * 8u) = make_uint2(w[0], w[1]);
              }
              if (sub == 0u) (kv[j] ? c.vs : c.ks)[scale_s[tok[j]] + h[j] * c.s_head] = sc;
            }
          } else if (at[j] >= 0 && has) {
            store8(reinterpret_cast<P *>((kv[j] ? c.v : c.k) + at[j] + h[j] * c.head_bytes) + sub * 8u, true, x[j]);
          }
        } else if (at[j] != -2 && has) {                  // (a position that is not there reads as zeros)
          if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = at[j] < 0 ? 0.0f : x[j][i] * scale[j];
          }
          const RowsRef &rr = kv[j] ? vr : kr;
          store8(reinterpret_cast<R *>(rr.p) + static_cast<int64_t>(base + tok[j]) * rr.row + static_cast<int64_t>(h[j]) * rr.head + sub * 8u, s.vec[kv[j]] != 0u, x[j]);
        }
      }
    }
  }
}

template <typename R, typename P>
int Launch(const CacheView &c, const BatchView &b, const RowsRef &k, const RowsRef &v, bool write, uint32_t sms, cudaStream_t stream) {
  MoveShape s;
  s.lanes = 1;
  while (s.lanes * 8u < c.hd) s.lanes *= 2u;
  const uint32_t rounds = b.n_rows / (sms * 16u);         // (as in rope.cu: few tokens spread over the SMs, many share their lookups)
  s.tokens = rounds < 1u ? 1u : rounds > kMoveTokens ? kMoveTokens : rounds;
  constexpr int64_t W = 16 / sizeof(R);
  const RowsRef *r[2] = {&k, &v};
  for (int t = 0; t < 2; ++t)
    s.vec[t] = reinterpret_cast<uintptr_t>(r[t]->p) % 16 == 0 && r[t]->row % W == 0 && (c.heads == 1u || r[t]->head % W == 0) ? 1u : 0u;
  s.by_heads = FastDiv(c.heads);
  uint32_t ctas = (b.n_rows + s.tokens - 1u) / s.tokens;
  if (ctas > sms * 8u) ctas = sms * 8u;
  if (write) b2_cache_move<R, P, true><<<ctas, kMoveThreads, 0, stream>>>(c, b, k, v, s);
  else b2_cache_move<R, P, false><<<ctas, kMoveThreads, 0, stream>>>(c, b, k, v, s);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int LaunchCacheMove(const CacheView &c, const BatchView &b, const RowsRef &k, const RowsRef &v, uint32_t dtype, uint32_t row_dtype, bool write, uint32_t sms, CUstream_st *stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == B2_E4M3) {
    if (row_dtype == B2_F32) return Launch<float, __nv_fp8_e4m3>(c, b, k, v, write, sms, st);
    return row_dtype == B2_BF16 ? Launch<__nv_bfloat16, __nv_fp8_e4m3>(c, b, k, v, write, sms, st) : Launch<__half, __nv_fp8_e4m3>(c, b, k, v, write, sms, st);
  }
  if (dtype == B2_BF16) return row_dtype == B2_F32 ? Launch<float, __nv_bfloat16>(c, b, k, v, write, sms, st) : Launch<__nv_bfloat16, __nv_bfloat16>(c, b, k, v, write, sms, st);
  return row_dtype == B2_F32 ? Launch<float, __half>(c, b, k, v, write, sms, st) : Launch<__half, __half>(c, b, k, v, write, sms, st);
}

}  // namespace b2
