// A batch's rows of K and V into the pages of a cache, quantised to e4m3 where the pages are, and back out of them.
//
// e4m3: s = max|x| / 448, code = x / s to the nearest, both as IEEE divisions, so that the codes are those of the definition to
// the bit. The largest magnitude is taken over the values' bit patterns, where NaN is above infinity: a row that holds either
// gets a scale that is not finite and reads back as NaN throughout.
//
// Bound: HBM, each row read and written once. A warp takes a token (few tokens: a part of its rows): it looks up the token's sequence, 32 starts
// at a time, and where its position lies, while the rows of the token before are on the way, and moves the 2 x heads rows, 8 values to a
// thread, four rows of each group of threads in flight. No barrier anywhere.
#include <type_traits>

#include "operators_dev.cuh"

namespace b2 {
namespace {

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;
constexpr int kAtOnce = 4;                                // rows in flight to each group of threads

// Eight values of a row as they come, in words.
template <typename R, bool VEC>
__device__ __forceinline__ void load8(const R *p, uint32_t (&w)[2 * sizeof(R)]) {
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(R)) / 2; ++j) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[j];
      w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
    }
  } else if constexpr (sizeof(R) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
  } else {
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
  }
}
template <typename R, bool VEC>
__device__ __forceinline__ void store8(R *p, const uint32_t (&w)[2 * sizeof(R)]) {
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(R)) / 2; ++j) reinterpret_cast<uint4 *>(p)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  } else if constexpr (sizeof(R) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<uint32_t *>(p)[i] = w[i];
  } else {
    uint16_t *h = reinterpret_cast<uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) { h[2 * i] = static_cast<uint16_t>(w[i]); h[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16); }
  }
}
template <typename R>
__device__ __forceinline__ void widen8(const uint32_t (&w)[2 * sizeof(R)], float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(R) == 4) x[i] = __uint_as_float(w[i]);
    else if constexpr (std::is_same<R, __nv_bfloat16>::value) x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else x[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
  }
}
template <typename R>
__device__ __forceinline__ void narrow8(const float (&x)[8], uint32_t (&w)[2 * sizeof(R)]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(2 * sizeof(R)); ++i) {
    if constexpr (sizeof(R) == 4) w[i] = __float_as_uint(x[i]);
    else if constexpr (std::is_same<R, __nv_bfloat16>::value) w[i] = cvt_bf16x2(x[2 * i + 1], x[2 * i]);
    else w[i] = cvt_f16x2(x[2 * i + 1], x[2 * i]);
  }
}
// The largest magnitude of a row whose eight values each of `lanes` threads have; by bit patterns, so that a NaN is largest.
template <typename R>
__device__ __forceinline__ float largest(const uint32_t (&w)[2 * sizeof(R)], uint32_t lanes) {
  uint32_t m = 0u;
  if constexpr (sizeof(R) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
    for (uint32_t o = lanes >> 1; o > 0u; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return __uint_as_float(m);
  } else {                                                // two at a time
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    for (uint32_t o = lanes >> 1; o > 0u; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<R, __nv_bfloat16>::value) return __uint_as_float(m << 16);
    else return __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
  }
}

struct MoveShape {
  uint32_t lanes;                  // threads to a row, a power of two
  uint32_t split;                  // warps to a token
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

// One of a token's K and V: rows of `heads` heads from row (a thread's eight values) to page or back.
template <typename R, typename P, bool WRITE, bool VEC, typename F>
__device__ __forceinline__ void move_rows(const CacheView &c, const MoveShape &s, R *row, int64_t row_head, uint8_t *page, float *scales, const Place &at, uint32_t first, uint32_t group,
                                          uint32_t step, uint32_t sub, bool has, F under) {
  constexpr bool Q8 = sizeof(P) == 1;
  constexpr int WR = 2 * sizeof(R);
  row += sub * 8u;
  page += at.at + sub * 8u * sizeof(P);
  scales += at.scale;
  for (uint32_t h0 = first; h0 - group < c.heads; h0 += kAtOnce * step) {
    uint32_t w[kAtOnce][WR];
    uint2 code[kAtOnce];
    float scale[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const uint32_t h = h0 + static_cast<uint32_t>(j) * step;
      const bool live = h < c.heads && at.at >= 0 && has;
      code[j] = make_uint2(0u, 0u);
      scale[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < WR; ++i) w[j][i] = 0u;
      if (!live) continue;
      if constexpr (WRITE) {
        load8<R, VEC>(row + static_cast<int64_t>(h) * row_head, w[j]);
      } else if constexpr (Q8) {
        code[j] = *reinterpret_cast<const uint2 *>(page + h * c.head_bytes);
        scale[j] = scales[h * c.s_head];
      } else {
        uint32_t pw[2 * sizeof(P)];
        load8<P, true>(reinterpret_cast<const P *>(page + h * c.head_bytes), pw);
        if constexpr (std::is_same<R, P>::value) {
#pragma unroll
          for (int i = 0; i < WR; ++i) w[j][i] = pw[i];
        } else {
          float x[8];
          widen8<P>(pw, x);
          narrow8<R>(x, w[j]);
        }
      }
    }
    under(h0 == first);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const uint32_t h = h0 + static_cast<uint32_t>(j) * step;
      if constexpr (WRITE) {
        float x[8];
        if constexpr (Q8) {
          const float sc = __fdiv_rn(largest<R>(w[j], s.lanes), 448.0f);
          if (h < c.heads && at.at >= 0) {
            widen8<R>(w[j], x);
            if (has) *reinterpret_cast<uint2 *>(page + h * c.head_bytes) = codes_of(x, sc);
            if (sub == 0u) scales[h * c.s_head] = sc;
          }
        } else if (h < c.heads && at.at >= 0 && has) {
          if constexpr (std::is_same<R, P>::value) {
            store8<P, true>(reinterpret_cast<P *>(page + h * c.head_bytes), w[j]);
          } else {
            uint32_t pw[2 * sizeof(P)];
            widen8<R>(w[j], x);
            narrow8<P>(x, pw);
            store8<P, true>(reinterpret_cast<P *>(page + h * c.head_bytes), pw);
          }
        }
      } else if (h < c.heads && at.at != -2 && has) {     // (a position that is not there reads as zeros)
        if constexpr (Q8) {
          float x[8];
          const uint32_t ww[2] = {code[j].x, code[j].y};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(ww[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
            const float2 f = __half22float2(__half2(hr));
            x[2 * i] = f.x * scale[j];
            x[2 * i + 1] = f.y * scale[j];
          }
          narrow8<R>(x, w[j]);
        }
        store8<R, VEC>(row + static_cast<int64_t>(h) * row_head, w[j]);
      }
    }
  }
}

// R: type of the rows, P: of the pages. VEC: rows of 16-byte accesses.
template <typename R, typename P, bool WRITE, bool VEC>
__global__ void __launch_bounds__(kMoveThreads) b2_cache_move(const __grid_constant__ CacheView c, const __grid_constant__ BatchView b, const __grid_constant__ RowsRef kr,
                                                              const __grid_constant__ RowsRef vr, const __grid_constant__ MoveShape s) {
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
  const uint32_t warps = gridDim.x * kMoveWarps, me = blockIdx.x * kMoveWarps + warp;
  const uint32_t step = warps / s.split, first = (me % s.split) * groups + group, head_step = s.split * groups;
  uint32_t tok = me / s.split;
  Place now = place_of(c, b, cap, tok);
  while (tok < b.n_rows) {
    const uint32_t next = b.n_rows - tok > step ? tok + step : b.n_rows;
    Place after = {-2, 0};
    move_rows<R, P, WRITE, VEC>(c, s, reinterpret_cast<R *>(kr.p) + static_cast<int64_t>(tok) * kr.row, kr.head, c.k, c.ks, now, first, group, head_step, sub, has,
                                [&](bool once) { if (once) after = place_of(c, b, cap, next); });      // (under the loads' flight)
    move_rows<R, P, WRITE, VEC>(c, s, reinterpret_cast<R *>(vr.p) + static_cast<int64_t>(tok) * vr.row, vr.head, c.v, c.vs, now, first, group, head_step, sub, has, [](bool) {});
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
  while (s.split < kMoveWarps && static_cast<uint64_t>(b.n_rows) * s.split < sms * 8u && c.heads * s.lanes > s.split * 32u) s.split *= 2u;
  constexpr int64_t W = 16 / sizeof(R);
  bool vec = true;
  for (const RowsRef *r : {&k, &v}) vec = vec && reinterpret_cast<uintptr_t>(r->p) % 16 == 0 && r->row % W == 0 && (c.heads == 1u || r->head % W == 0);
  const uint64_t want = (static_cast<uint64_t>(b.n_rows) * s.split + kMoveWarps - 1u) / kMoveWarps;
  const uint32_t ctas = want > sms * 8u ? sms * 8u : static_cast<uint32_t>(want);
  if (write) {
    if (vec) b2_cache_move<R, P, true, true><<<ctas, kMoveThreads, 0, stream>>>(c, b, k, v, s);
    else b2_cache_move<R, P, true, false><<<ctas, kMoveThreads, 0, stream>>>(c, b, k, v, s);
  } else {
    if (vec) b2_cache_move<R, P, false, true><<<ctas, kMoveThreads, 0, stream>>>(c, b, k, v, s);
    else b2_cache_move<R, P, false, false><<<ctas, kMoveThreads, 0, stream>>>(c, b, k, v, s);
  }
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
