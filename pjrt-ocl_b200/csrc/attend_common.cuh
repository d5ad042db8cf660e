// What both attention kernels over a paged cache use.
#ifndef B2VM_ATTEND_COMMON_CUH_
#define B2VM_ATTEND_COMMON_CUH_

#include "operators_dev.cuh"

namespace b2 {

// A warpgroup's registers, by the thread: all four warps of it execute these.
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 32 bytes at once, 32-byte aligned.
__device__ __forceinline__ void stg_v8(void *p, const uint32_t *w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// Two e4m3 values as two f16 (exact).
__device__ __forceinline__ uint32_t cvt_e4m3x2_f16x2(uint32_t lo16) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(lo16));
  return r;
}

// A power of two above a scale, from 2^-80 (below which a value's last bits, then the value, are lost) to 2^104 (above which its product overflows).
__device__ __forceinline__ float power_above(float x) { return __uint_as_float(min(231u, max(47u, (__float_as_uint(x) >> 23) + 1u)) << 23); }

// A value of the rows' type (16 bits) as f32.
__device__ __forceinline__ float row_value(const uint8_t *p, bool bf16) {
  const uint16_t w = *reinterpret_cast<const uint16_t *>(p);
  return bf16 ? __uint_as_float(static_cast<uint32_t>(w) << 16) : __half2float(__ushort_as_half(w));
}
__device__ __forceinline__ void store_row_value(uint8_t *p, float v, bool bf16) {
  *reinterpret_cast<uint16_t *>(p) = bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ uint8_t *row_at(const RowsRef &r, int32_t row, uint32_t head) {
  return r.p + 2 * (static_cast<int64_t>(row) * r.row + static_cast<int64_t>(head) * r.head);
}

// One row of the result by itself, over the keys that it sees and no others, by one warp. A product over a tile of keys gives a
// key that a row does not see the weight 0, and 0 times a NaN or an infinity is a NaN: where a tile's result is not finite, the
// rows that do not see all of its keys are worked out here again. Slow, and only reached by caches whose V holds such values, or
// 8-bit pages whose scales are further apart than a tile's product holds. (Keys one after another: four at once would take registers from the chunk
// kernel's loops, whose 8-bit chunk went from 784 to 797 us.)
// (of its values [v0, v0 + nv), and lse with the first; `alive`: where others see that it goes on, or null)
static __device__ __noinline__ void attend_row_alone(const AttendArgs &a, uint32_t seq, const Seq s, int32_t i, uint32_t head, uint32_t v0, uint32_t nv,
                                                     volatile unsigned long long *alive) {
  const uint32_t lane = threadIdx.x & 31u, h = head / a.group, d0 = lane * 4u;
  const bool has = d0 < a.c.hd, bf = a.bf16 != 0u;
  const Span sp = SeenBy(s, i, a.causal, a.window);
  float q[4] = {0.0f, 0.0f, 0.0f, 0.0f}, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
  if (has) {
    const uint8_t *p = row_at(a.q, s.first + i, head) + 2u * d0;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = row_value(p + 2 * k, bf) * a.scale_log2;
  }
  auto four = [&](const uint8_t *p, float scale, float (&x)[4]) {
    if (!has) { x[0] = x[1] = x[2] = x[3] = 0.0f; return; }
    if (a.e4m3) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(p + d0);
      const uint32_t lo = cvt_e4m3x2_f16x2(w & 0xffffu), hi = cvt_e4m3x2_f16x2(w >> 16);
      const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), v = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
      x[0] = u.x * scale; x[1] = u.y * scale; x[2] = v.x * scale; x[3] = v.y * scale;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = row_value(p + 2u * (d0 + k), bf);
    }
  };
  for (int32_t j0 = sp.lo; j0 < sp.hi; j0 += 32) {
    int64_t at = -1, sc = 0;
    if (j0 + static_cast<int32_t>(lane) < sp.hi) at = page_offset(a.c, a.b, seq, static_cast<uint32_t>(j0) + lane, &sc);
    const int32_t n = min(32, sp.hi - j0);
    if (alive && lane == 0u) *alive = globaltimer_ns();
    float mine = -INFINITY;                               // the score of the lane's key
#pragma unroll 1
    for (int32_t j = 0; j < n; ++j) {
      const int64_t o = __shfl_sync(0xffffffffu, at, j), so = __shfl_sync(0xffffffffu, sc, j);
      if (o < 0) continue;
      float x[4];
      four(a.c.k + o + h * a.c.head_bytes, a.e4m3 ? a.c.ks[so + h * a.c.s_head] : 1.0f, x);
      const float sum = warp_reduce(q[0] * x[0] + q[1] * x[1] + q[2] * x[2] + q[3] * x[3], [](float u, float v) { return u + v; });
      if (static_cast<int32_t>(lane) == j) mine = sum;
    }
    const float m2 = fmaxf(m, warp_reduce(mine, [](float u, float v) { return fmaxf(u, v); }));
    const float c = m == -INFINITY ? 0.0f : exp2f(m - m2), p = mine == -INFINITY ? 0.0f : exp2f(mine - m2);     // (a NaN loses in the maximum and stays in p)
    l = l * c + warp_reduce(p, [](float u, float v) { return u + v; });
    m = m2;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] *= c;
#pragma unroll 1
    for (int32_t j = 0; j < n; ++j) {
      const int64_t o = __shfl_sync(0xffffffffu, at, j), so = __shfl_sync(0xffffffffu, sc, j);
      const float pj = __shfl_sync(0xffffffffu, p, j);
      if (o < 0) continue;
      float x[4];
      four(a.c.v + o + h * a.c.head_bytes, a.e4m3 ? a.c.vs[so + h * a.c.s_head] : 1.0f, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += pj * x[k];
    }
  }
  const bool none = m == -INFINITY && l == 0.0f;
  if (has && d0 >= v0 && d0 < v0 + nv) {
    uint8_t *p = row_at(a.o, s.first + i, head) + 2u * d0;
#pragma unroll
    for (int k = 0; k < 4; ++k) store_row_value(p + 2 * k, none ? 0.0f : acc[k] / l, bf);
  }
  if (lane == 0u && v0 == 0u && a.lse) a.lse[static_cast<int64_t>(s.first + i) * a.q_heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// The sequence b whose units hold unit `target` of all sequences' units in a row, and the number of those before b's; false where
// there are not that many. of(b): the units of sequence b. All threads of the CTA; `sh` has room for THREADS / 32 + 2 words.
template <uint32_t THREADS, typename F>
__device__ __forceinline__ bool find_unit(uint32_t n_seqs, unsigned long long target, unsigned long long *sh, F of, uint32_t &seq, unsigned long long &before) {
  constexpr uint32_t W = THREADS / 32u;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, w = tid >> 5;
  unsigned long long run = 0;
  bool found = false;
  for (uint32_t i0 = 0; i0 < n_seqs && !found; i0 += THREADS) {
    const uint32_t i = i0 + tid;
    const unsigned long long v = i < n_seqs ? of(i) : 0ull;
    unsigned long long x = v;
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31u) sh[w] = x;
    __syncthreads();
    unsigned long long mine = run;
    for (uint32_t k = 0; k < W; ++k) {
      if (k < w) mine += sh[k];
      run += sh[k];
    }
    if (v != 0ull && mine + x > target && mine + x - v <= target) {
      sh[W] = i;
      sh[W + 1u] = mine + x - v;
    }
    found = run > target;                                 // (the same for all threads)
  }
  __syncthreads();
  if (!found) return false;
  seq = static_cast<uint32_t>(sh[W]);
  before = sh[W + 1u];
  return true;
}

}  // namespace b2
#endif
