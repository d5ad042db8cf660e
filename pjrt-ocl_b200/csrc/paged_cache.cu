// A batch's rows of K and V into the pages of a cache, quantised to e4m3 where the pages are, and back out of them.
//
// e4m3: s = max|x| / 448, code = x / s to the nearest, both as IEEE divisions, so that the codes are those of the definition to
// the bit. The largest magnitude is taken over the values' bit patterns, where NaN is above infinity: a row that holds either
// gets a scale that is not finite and reads back as NaN throughout.
//
// Bound: HBM, each row read and written once. A warp takes a token (few tokens: a part of its rows): it looks up the token's sequence, 32 starts
// at a time, and where its position lies, while the rows of the token before are on the way, and moves the 2 x heads rows, 8 values to a
// thread, four rows of each group of threads in flight. No barrier anywhere.
#include "operators_dev.cuh"

namespace b2 {
namespace {

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;
constexpr int kAtOnce = 4;                                // rows in flight to each group of threads

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
  uint32_t lanes;                  // threads to a row, a power of two
  uint32_t split;                  // warps to a token
  uint32_t vec[2];                 // rows of K, V: 16-byte accesses
};

// Where a row of the batch lies in the cache: byte offset of its place (-1: it has none, -2: the row is nobody's) and of its scales.
struct Place { int64_t at, scale; };
__device__ __forceinline__ Place place_of(const CacheView &c, const BatchView &b, uint64_t cap, uint32_t i) {
  Place p = {-2, 0};
  if (i >= b.n_rows) return p;
  const uint32_t q = seq_of_row(b.row_start, b.n_seqs, static_cast<int32_t>(i));
  const Seq s = load_seq(b, cap, q);
  const int32_t k = static_cast<int32_t>(i) - s.first;
  if (k >= 0 && k < s.n) {
    const int32_t pos = s.len - s.n + k;
    p.at = pos >= 0 ? page_offset(c, b, q, static_cast<uint32_t>(pos), &p.scale) : -1;
  }
  return p;
}

// Codes of eight values with scale s. x / s correctly rounded: with the correctly rounded reciprocal r of s, q = x r and q + (x - q s) r is (Markstein,
// 1990), as long as nothing leaves the normal range; else by the division itself.
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float s) {
  uint32_t w[4];
  float v[8];
  if (s > 1.0e-27f && s < 1.0e27f) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = x[i] * r;
      v[i] = fmaf(fmaf(-q, s, x[i]), r, q);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s == 0.0f ? 0.0f : __fdiv_rn(x[i], s);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// R: type of the rows, P: of the pages.
template <typename R, typename P, bool WRITE>
__global__ void __launch_bounds__(kMoveThreads) b2_cache_move(const __grid_constant__ CacheView c, const __grid_constant__ BatchView b, const __grid_constant__ RowsRef kr,
                                                              const __grid_constant__ RowsRef vr, const __grid_constant__ MoveShape s) {
  constexpr bool Q8 = sizeof(P) == 1;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint64_t cap = capacity_of(c, b);
  const uint32_t sub = lane & (s.lanes - 1u), group = lane / s.lanes, groups = 32u / s.lanes;
  const bool has = sub * 8u < c.hd;
  if (blockIdx.x == 0u) {                                 // batches that do not fit are named even where they have no row
    for (uint32_t i = tid; i < b.n_seqs; i += kMoveThreads) {
      const Seq q = load_seq(b, cap, i);
      if (q.bad) cache_fault(c.status, kStBadBatch, i, static_cast<uint32_t>(q.bad), static_cast<uint32_t>(q.value));
    }
  }
  const uint32_t warps = gridDim.x * kMoveWarps, me = blockIdx.x * kMoveWarps + warp, rows = 2u * c.heads;
  const uint32_t step = warps / s.split, first_row = (me % s.split) * groups + group, row_step = s.split * groups;
  uint32_t tok = me / s.split;
  if (tok >= step) return;                                // (warps that a split leaves over)
  Place now = place_of(c, b, cap, tok);
  for (; tok < b.n_rows; ) {
    const uint32_t next = b.n_rows - tok > step ? tok + step : b.n_rows;
    Place after = {-2, 0};
    for (uint32_t r0 = first_row; r0 - group < rows; r0 += kAtOnce * row_step) {
      float x[kAtOnce][8], scale[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const uint32_t r = r0 + static_cast<uint32_t>(j) * row_step, kv = r >= c.heads ? 1u : 0u, h = r - kv * c.heads;
        scale[j] = 0.0f;
        if (r < rows && now.at >= 0) {
          if (WRITE) {
            const RowsRef &rr = kv ? vr : kr;
            if (has) load8(reinterpret_cast<const R *>(rr.p) + static_cast<int64_t>(tok) * rr.row + static_cast<int64_t>(h) * rr.head + sub * 8u, s.vec[kv] != 0u, x[j]);
          } else {
            const uint8_t *p = (kv ? c.v : c.k) + now.at + h * c.head_bytes + sub * 8u * sizeof(P);
            if constexpr (Q8) {
              scale[j] = (kv ? c.vs : c.ks)[now.scale + h * c.s_head];
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
        if (!(r < rows && now.at >= 0 && has)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
        }
      }
      if (r0 == first_row) after = place_of(c, b, cap, next);      // (under the loads' flight)
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const uint32_t r = r0 + static_cast<uint32_t>(j) * row_step, kv = r >= c.heads ? 1u : 0u, h = r - kv * c.heads;
        if (WRITE) {
          if constexpr (Q8) {
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[j][i]) & 0x7fffffffu);
            for (uint32_t o = s.lanes >> 1; o > 0u; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float sc = __fdiv_rn(__uint_as_float(m), 448.0f);
            if (r < rows && now.at >= 0) {
              if (has) *reinterpret_cast<uint2 *>((kv ? c.v : c.k) + now.at + h * c.head_bytes + sub * 8u) = codes_of(x[j], sc);
              if (sub == 0u) (kv ? c.vs : c.ks)[now.scale + h * c.s_head] = sc;
            }
          } else if (r < rows && now.at >= 0 && has) {
            store8(reinterpret_cast<P *>((kv ? c.v : c.k) + now.at + h * c.head_bytes) + sub * 8u, true, x[j]);
          }
        } else if (r < rows && now.at != -2 && has) {     // (a position that is not there reads as zeros)
          if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = now.at < 0 ? 0.0f : x[j][i] * scale[j];
          }
          const RowsRef &rr = kv ? vr : kr;
          store8(reinterpret_cast<R *>(rr.p) + static_cast<int64_t>(tok) * rr.row + static_cast<int64_t>(h) * rr.head + sub * 8u, s.vec[kv] != 0u, x[j]);
        }
      }
    }
    tok = next;
    now = after;
  }
}

template <typename R, typename P>
int Launch(const CacheView &c, const BatchView &b, const RowsRef &k, const RowsRef &v, bool write, uint32_t sms, cudaStream_t stream) {
  MoveShape s;
  s.lanes = 1;
  while (s.lanes * 8u < c.hd) s.lanes *= 2u;
  // Few tokens: a CTA's warps share one, as far as it has rows for them.
  s.split = 1;
  while (s.split < kMoveWarps && static_cast<uint64_t>(b.n_rows) * s.split < sms * 8u && 2u * c.heads * s.lanes > s.split * 32u) s.split *= 2u;
  constexpr int64_t W = 16 / sizeof(R);
  const RowsRef *r[2] = {&k, &v};
  for (int t = 0; t < 2; ++t)
    s.vec[t] = reinterpret_cast<uintptr_t>(r[t]->p) % 16 == 0 && r[t]->row % W == 0 && (c.heads == 1u || r[t]->head % W == 0) ? 1u : 0u;
  const uint64_t want = (static_cast<uint64_t>(b.n_rows) * s.split + kMoveWarps - 1u) / kMoveWarps;
  const uint32_t ctas = want > sms * 8u ? sms * 8u : static_cast<uint32_t>(want);
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
