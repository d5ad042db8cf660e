// A batch's rows of K and V into the pages of a cache, quantised to e4m3 where the pages are, and back out of them.
//
// e4m3: s = max|x| / 448, code = x / s to the nearest, both as IEEE divisions, so that the codes are those of the definition to
// the bit. The largest magnitude is taken over the values' bit patterns, where NaN is above infinity: a row that holds either
// gets a scale that is not finite and reads back as NaN throughout.
//
// Bound: HBM, each row read and written once. A warp takes a token (few tokens: a part of its rows): it looks up the token's sequence, 32 starts
// at a time, and where its position lies, while the rows of the token before are on the way, and moves the 2 x heads rows, 8 values
// each of both halves of a row to a thread, a row of K and one of V in flight to each group of threads. No barrier anywhere.
// Measured, bf16 rows and e4m3 pages of 128 values: written 27 us (53 % of the copy rate; 2.8 instructions of 4 a cycle go to maxima, quotients and
// conversions), read back 39 us (80 %).
#include <type_traits>

#include "operators_dev.cuh"

namespace b2 {
namespace {

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;
constexpr int kPer = 8;                                   // values side by side of a thread, which has two such parts of a row

// A thread's values of a row as they come, in words.
template <typename R, bool VEC>
__device__ __forceinline__ void load_row(const R *p, uint32_t (&w)[kPer * sizeof(R) / 4]) {
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < kPer * static_cast<int>(sizeof(R)) / 16; ++j) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[j];
      w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
    }
  } else if constexpr (sizeof(R) == 4) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
  } else {
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
  }
}
template <typename R, bool VEC>
__device__ __forceinline__ void store_row(R *p, const uint32_t (&w)[kPer * sizeof(R) / 4]) {
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < kPer * static_cast<int>(sizeof(R)) / 16; ++j) reinterpret_cast<uint4 *>(p)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  } else if constexpr (sizeof(R) == 4) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) reinterpret_cast<uint32_t *>(p)[i] = w[i];
  } else {
    uint16_t *h = reinterpret_cast<uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) { h[2 * i] = static_cast<uint16_t>(w[i]); h[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16); }
  }
}
template <typename R>
__device__ __forceinline__ void widen(const uint32_t (&w)[kPer * sizeof(R) / 4], float (&x)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if constexpr (sizeof(R) == 4) x[i] = __uint_as_float(w[i]);
    else if constexpr (std::is_same<R, __nv_bfloat16>::value) x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else x[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
  }
}
template <typename R>
__device__ __forceinline__ void narrow(const float (&x)[kPer], uint32_t (&w)[kPer * sizeof(R) / 4]) {
#pragma unroll
  for (int i = 0; i < kPer * static_cast<int>(sizeof(R)) / 4; ++i) {
    if constexpr (sizeof(R) == 4) w[i] = __float_as_uint(x[i]);
    else if constexpr (std::is_same<R, __nv_bfloat16>::value) w[i] = cvt_bf16x2(x[2 * i + 1], x[2 * i]);
    else w[i] = cvt_f16x2(x[2 * i + 1], x[2 * i]);
  }
}
// The largest magnitude of a row that `lanes` threads have between them; by bit patterns, so that a NaN is largest.
template <typename R>
__device__ __forceinline__ float largest(const uint32_t (&w)[2][kPer * sizeof(R) / 4], uint32_t lanes) {
  uint32_t m = 0u;
  if constexpr (sizeof(R) == 4) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) m = max(m, max(w[0][i] & 0x7fffffffu, w[1][i] & 0x7fffffffu));
    for (uint32_t o = lanes >> 1; o > 0u; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return __uint_as_float(m);
  } else {                                                // two at a time
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) m = __vmaxu2(m, __vmaxu2(w[0][i] & 0x7fff7fffu, w[1][i] & 0x7fff7fffu));
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

// x / s correctly rounded, r the correctly rounded reciprocal of s: q = x r, then q + (x - q s) r (Markstein, 1990), as long as nothing leaves the normal
// range: s between 1e-27 and 1e27 and x / s at most 448 (a quotient that does is far below the smallest code).
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, s, x), r, q);
}
__device__ __forceinline__ bool plain_scale(float s) { return s > 1.0e-27f && s < 1.0e27f; }
__device__ __forceinline__ float scale_of(float largest) {
  return plain_scale(largest) ? quotient(largest, 448.0f, 1.0f / 448.0f) : __fdiv_rn(largest, 448.0f);
}
__device__ __forceinline__ uint2 codes_of(const float (&x)[kPer], float s, bool plain, float r) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i) {
    float2 v;
    if (plain) v = make_float2(quotient(x[2 * i], s, r), quotient(x[2 * i + 1], s, r));
    else v = s == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(__fdiv_rn(x[2 * i], s), __fdiv_rn(x[2 * i + 1], s));
    w[i >> 1] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3)) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

// A row of the batch (a thread's two parts of it) into its page.
template <typename R, typename P>
__device__ __forceinline__ void to_page(const uint32_t (&w)[2][kPer * sizeof(R) / 4], uint8_t *page, uint32_t far, float *scale, bool live, const bool (&has)[2], uint32_t sub, uint32_t lanes) {
  float x[kPer];
  if constexpr (sizeof(P) == 1) {
    const float sc = scale_of(largest<R>(w, lanes));
    if (live) {
      const bool plain = plain_scale(sc);
      const float r = plain ? __frcp_rn(sc) : 0.0f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        widen<R>(w[q], x);
        if (has[q]) *reinterpret_cast<uint2 *>(page + q * far) = codes_of(x, sc, plain, r);
      }
      if (sub == 0u) *scale = sc;
    }
  } else if (live) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (!has[q]) continue;
      if constexpr (std::is_same<R, P>::value) {
        store_row<P, true>(reinterpret_cast<P *>(page + q * far), w[q]);
      } else {
        uint32_t pw[kPer * sizeof(P) / 4];
        widen<R>(w[q], x);
        narrow<P>(x, pw);
        store_row<P, true>(reinterpret_cast<P *>(page + q * far), pw);
      }
    }
  }
}
template <typename R, typename P, bool VEC>
__device__ __forceinline__ void to_row(const uint32_t (&w)[kPer * sizeof(P) / 4], float scale, R *row) {
  if constexpr (std::is_same<R, P>::value) {
    store_row<R, VEC>(row, w);
  } else {
    float x[kPer];
    if constexpr (sizeof(P) == 1) {
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) {
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
        const float2 f = __half22float2(__half2(hr));
        x[2 * i] = f.x * scale;
        x[2 * i + 1] = f.y * scale;
      }
    } else {
      widen<P>(w, x);
    }
    uint32_t o[kPer * sizeof(R) / 4];
    narrow<R>(x, o);
    store_row<R, VEC>(row, o);
  }
}
// A thread's part in a page: codes or 16-bit values.
template <typename P>
__device__ __forceinline__ void load_page(const uint8_t *p, uint32_t (&w)[kPer * sizeof(P) / 4]) {
  if constexpr (sizeof(P) == 1) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
}

// R: type of the rows, P: of the pages. VEC: rows of 16-byte accesses.
template <typename R, typename P, bool WRITE, bool VEC>
__global__ void __launch_bounds__(kMoveThreads, 4) b2_cache_move(const __grid_constant__ CacheView c, const __grid_constant__ BatchView b, const __grid_constant__ RowsRef kr,
                                                              const __grid_constant__ RowsRef vr, const __grid_constant__ MoveShape s) {
  using From = typename std::conditional<WRITE, R, P>::type;
  constexpr int WF = kPer * sizeof(From) / 4;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint64_t cap = capacity_of(c, b);
  const uint32_t sub = lane & (s.lanes - 1u), group = lane / s.lanes, groups = 32u / s.lanes;
  const bool has[2] = {sub * kPer < c.hd, (sub + s.lanes) * kPer < c.hd};
  const uint32_t far_row = s.lanes * kPer, far_page = far_row * sizeof(P);       // to the second part
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
    R *rows[2] = {reinterpret_cast<R *>(kr.p) + static_cast<int64_t>(tok) * kr.row + sub * kPer, reinterpret_cast<R *>(vr.p) + static_cast<int64_t>(tok) * vr.row + sub * kPer};
    const int64_t row_head[2] = {kr.head, vr.head};
    uint8_t *pages[2] = {c.k + now.at + sub * kPer * sizeof(P), c.v + now.at + sub * kPer * sizeof(P)};
    float *scales[2] = {c.ks + now.scale, c.vs + now.scale};
    for (uint32_t h = first; h - group < c.heads; h += head_step) {
      uint32_t w[2][2][WF];
      float scale[2] = {0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < WF; ++i) w[t][q][i] = 0u;
          if (h < c.heads && now.at >= 0 && has[q]) {     // (a position that is not there reads as zeros)
            if constexpr (WRITE) {
              load_row<R, VEC>(rows[t] + static_cast<int64_t>(h) * row_head[t] + q * far_row, w[t][q]);
            } else {
              load_page<P>(pages[t] + h * c.head_bytes + q * far_page, w[t][q]);
              if (sizeof(P) == 1 && q == 0) scale[t] = scales[t][h * c.s_head];
            }
          }
        }
      if (h == first) after = place_of(c, b, cap, next);    // (under the loads' flight)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (WRITE) {
          to_page<R, P>(w[t], pages[t] + h * c.head_bytes, far_page, scales[t] + h * c.s_head, h < c.heads && now.at >= 0, has, sub, s.lanes);
        } else if (h < c.heads && now.at != -2) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (has[q]) to_row<R, P, VEC>(w[t][q], scale[t], rows[t] + static_cast<int64_t>(h) * row_head[t] + q * far_row);
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
  while (s.lanes * 2u * kPer < c.hd) s.lanes *= 2u;
  // Few tokens: a CTA's warps share one, as far as it has rows for them.
  s.split = 1;
  while (s.split < kMoveWarps && static_cast<uint64_t>(b.n_rows) * s.split < sms * 8u && c.heads * s.lanes > s.split * 32u) s.split *= 2u;
  constexpr int64_t W = 16 / sizeof(R);
  bool vec = true;
  for (const RowsRef *r : {&k, &v}) vec = vec && reinterpret_cast<uintptr_t>(r->p) % 16 == 0 && r->row % W == 0 && (c.heads == 1u || r->head % W == 0);
  const uint64_t want = (static_cast<uint64_t>(b.n_rows) * s.split + kMoveWarps - 1u) / kMoveWarps;
  const uint32_t ctas = want > sms * 4u ? sms * 4u : static_cast<uint32_t>(want);
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
