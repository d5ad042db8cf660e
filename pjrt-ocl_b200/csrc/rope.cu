// Rotary positions with the norms of queries and keys in the same pass, and its backward pass.
//
// A row x of hd values (one token, one head):  r = 1 / sqrt(mean x^2 + eps),  y = x r w;  pairs (a, b) of the first rot values
// turn by t = position f_i:  (a', b') = m (a cos t - b sin t, a sin t + b cos t).  Backward, with g = R^T dy and h = w g:
//   dx = r h - x r^3 / hd sum(h x),   dw = sum over rows and heads of g x r.
//
// Bound: HBM. Every row is read once and written once (backward: x and dy read, dx written).
// A warp takes a token (few tokens: a part of its heads). It works out the token's angles once, in 64-bit turns (position x turns, less the
// nearest whole number; sine and cosine of the rest in f32. Quotient and product are off by 2^-53 each: 2^-52 of the angle, 2^-25 at 2^27 and 2^-21 at 2^31;
// the rest as f32 by 2^-26 turns, 2^-23.3; f32's sine by some 2^-24), and keeps those of its pairs in registers for all
// heads. A row belongs to up to 32 threads; a thread holds V pairs of it, both halves of each, so that neither layout needs an exchange
// between threads: the half layout is two V-wide accesses rot/2 apart, the neighbouring one two that touch. What lies behind
// rot is treated the same with no angle. V is as wide as the addresses, strides and rot allow up to 16 bytes. The next rows are on the
// way while a row is worked on. No barrier stands between tokens.
// Gradients of the weights are summed in registers over a token's heads, in shared memory over a warp's tokens, joined once a CTA, and a second
// small launch adds the CTAs' sums in their order, so that a result does not change from call to call.
// Measured, 40 heads of 128 bf16 values with norms: 16384 tokens forward 69 us (74 % of the copy rate; 2.95 instructions of 4 a cycle), 8192
// backward 72 (54 %; the sums of a row stand between its loads and stores). With a register copy of the next row instead of the ring
// the backward pass took 80.
#include "operators_dev.cuh"

namespace b2 {
namespace {

constexpr int kRopeThreads = 256, kRopeWarps = kRopeThreads / 32;
constexpr uint32_t kRopeBackPerSm = 2, kRopePerSm = 3;
constexpr uint32_t kRing = 4;                             // stages of a warp's ring

struct RopeShape {
  uint32_t split;         // warps to a token
  uint32_t lanes;         // threads to a row, a power of two
  uint32_t units;         // V-pair units of a row
  uint32_t rot_units;     // of these turned
  uint32_t ring_at;       // bytes of shared memory before the rings
};

// First elements of the two V-wide accesses of unit u.
template <int V>
__device__ __forceinline__ void unit_at(const RopeArgs &a, const RopeShape &s, uint32_t u, uint32_t &e0, uint32_t &e1) {
  if (u < s.rot_units) {
    if (a.interleaved) { e0 = 2u * V * u; e1 = e0 + V; }
    else { e0 = V * u; e1 = e0 + a.rot / 2u; }
  } else {
    e0 = a.rot + V * (u - s.rot_units);
    e1 = e0 + (a.hd - a.rot) / 2u;
  }
}
// Pair i of a unit in its 2 V values: half layout (i, V + i), neighbours (2 i, 2 i + 1).
template <int V>
__device__ __forceinline__ void turn(float (&y)[2 * V], const float2 (&cs)[V], bool inter, float sign) {
  if (inter) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float p = y[2 * i], q = y[2 * i + 1], sn = sign * cs[i].y;
      y[2 * i] = p * cs[i].x - q * sn;
      y[2 * i + 1] = p * sn + q * cs[i].x;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float p = y[i], q = y[V + i], sn = sign * cs[i].y;
      y[i] = p * cs[i].x - q * sn;
      y[V + i] = p * sn + q * cs[i].x;
    }
  }
}
// The two accesses of a unit as they come: V values each, in 32-bit words (one value of 16 bits: in the low half).
template <typename T, int V> struct Raw {
  static constexpr int W = V * sizeof(T) >= 4 ? V * static_cast<int>(sizeof(T)) / 4 : 1;
  uint32_t a[W], b[W];
};
template <int BYTES>
__device__ __forceinline__ void load_words(const void *p, uint32_t *w) {
  if constexpr (BYTES == 16) {
    const uint4 v = *static_cast<const uint4 *>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *static_cast<const uint2 *>(p);
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (BYTES == 4) {
    w[0] = *static_cast<const uint32_t *>(p);
  } else {
    w[0] = *static_cast<const uint16_t *>(p);
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_unit(const T *p, uint32_t e0, uint32_t e1, Raw<T, V> &x) {
  load_words<V * sizeof(T)>(p + e0, x.a);
  load_words<V * sizeof(T)>(p + e1, x.b);
}
template <typename T> __device__ __forceinline__ float value_of(const uint32_t *w, int i);
template <> __device__ __forceinline__ float value_of<float>(const uint32_t *w, int i) { return __uint_as_float(w[i]); }
template <> __device__ __forceinline__ float value_of<__nv_bfloat16>(const uint32_t *w, int i) { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
template <> __device__ __forceinline__ float value_of<__half>(const uint32_t *w, int i) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
}
template <typename T, int V>
__device__ __forceinline__ void widen(const Raw<T, V> &r, float (&x)[2 * V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) { x[i] = value_of<T>(r.a, i); x[V + i] = value_of<T>(r.b, i); }
}
template <typename T, int V>
__device__ __forceinline__ void store_unit(T *p, uint32_t e0, uint32_t e1, const float (&x)[2 * V]) {
  Vec<T, V> a, b;
#pragma unroll
  for (int i = 0; i < V; ++i) { a.v[i] = FromF<T>(x[i]); b.v[i] = FromF<T>(x[V + i]); }
  *reinterpret_cast<Vec<T, V> *>(p + e0) = a;
  *reinterpret_cast<Vec<T, V> *>(p + e1) = b;
}
__device__ __forceinline__ float row_sum(float v, uint32_t lanes) {
  for (uint32_t o = lanes >> 1; o > 0u; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// U: units of a row that a thread may have (rows of more than 32 units).
template <typename T, int V, int U, bool BACK>
__global__ void __launch_bounds__(kRopeThreads, BACK ? kRopeBackPerSm : kRopePerSm) b2_rope(const __grid_constant__ RopeArgs a, const __grid_constant__ RopeShape s) {
  extern __shared__ __align__(16) uint8_t sm[];           // weights [2][hd], then the warps' angles [warps][rot / 2]
  float *w_s = reinterpret_cast<float *>(sm);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, half = a.rot / 2u;
  float2 *cs_s = reinterpret_cast<float2 *>(w_s + 2u * a.hd) + warp * half;
  const uint32_t at_once = 32u / s.lanes, slot = lane / s.lanes, sub = lane & (s.lanes - 1u);
  if (a.norm) {
    for (uint32_t i = tid; i < 2u * a.hd; i += kRopeThreads) {
      const uint32_t t = i >= a.hd ? 1u : 0u, e = i - t * a.hd;
      const void *w = a.w[t];
      w_s[i] = !w ? 1.0f : a.weight_f32 ? static_cast<const float *>(w)[e] : ToF(static_cast<const T *>(w)[e]);
    }
    __syncthreads();
  }
  uint32_t e0[U], e1[U];
  bool has[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = sub + static_cast<uint32_t>(k) * s.lanes;
    has[k] = u < s.units;
    unit_at<V>(a, s, has[k] ? u : 0u, e0[k], e1[k]);
  }
  // sums of the weights' gradients, of a token in registers, of the warp's tokens in shared memory: [warps][2][U][2 V][32]
  const bool sums = BACK && a.partial;
  float *acc_s = reinterpret_cast<float *>(sm) + 2u * a.hd + 2u * kRopeWarps * half + (warp * 2u * U * 2 * V) * 32u + lane;
  if (sums) {
#pragma unroll
    for (int i = 0; i < 4 * U * V; ++i) acc_s[i * 32] = 0.0f;
  }
  const float inv_hd = 1.0f / static_cast<float>(a.hd);
  const bool inter = a.interleaved != 0u;
  const uint32_t me = blockIdx.x * kRopeWarps + warp, step = gridDim.x * kRopeWarps / s.split, part = me % s.split;
  const uint32_t stride = s.split * at_once, first = part * at_once + slot;       // the warp's heads
  const bool some[2] = {part * at_once < a.heads[0], part * at_once < a.heads[1]};
  auto token_after = [&](uint32_t tok) { return a.n_rows - tok > step ? tok + step : a.n_rows; };
  // The warp's next rows: a unit's two accesses of x and, backward, of the gradient. Of 16 bytes they come through a ring of stages of each thread's own
  // in shared memory, three on the way while one is worked on; narrower ones straight into registers.
  constexpr bool RING = V * sizeof(T) == 16;
  constexpr uint32_t kTensors = BACK ? 2 : 1;
  Raw<T, V> xr[U], gr[U];
  uint32_t p_tok = me / s.split, p_t = some[0] ? 0u : 1u, p_head = first, issued = 0, taken = 0;
  const uint32_t ring = smem_addr(sm) + s.ring_at + warp * (kRing * kTensors * 2u * U * 512u) + lane * 16u;
  auto issue = [&]() {
    if (p_tok < a.n_rows) {
      const bool live = p_head < (p_t ? a.heads[1] : a.heads[0]);
      const RowsRef &xo = p_t ? a.x[1] : a.x[0], &go = p_t ? a.g[1] : a.g[0];
      const T *xp = reinterpret_cast<const T *>(xo.p) + (static_cast<int64_t>(p_tok) * xo.row + static_cast<int64_t>(p_head) * xo.head);
      const T *gp = reinterpret_cast<const T *>(go.p) + (static_cast<int64_t>(p_tok) * go.row + static_cast<int64_t>(p_head) * go.head);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool here = live && has[k];
        if constexpr (RING) {
          const uint32_t dst = ring + ((issued % kRing) * U + k) * kTensors * 1024u, bytes = here ? 16u : 0u;       // (what is not there is 0)
          if (!BACK || a.norm) {
            cp_async_16_zfill(dst, here ? xp + e0[k] : reinterpret_cast<const T *>(xo.p), bytes);
            cp_async_16_zfill(dst + 512u, here ? xp + e1[k] : reinterpret_cast<const T *>(xo.p), bytes);
          }
          if (BACK) {
            cp_async_16_zfill(dst + 1024u, here ? gp + e0[k] : reinterpret_cast<const T *>(go.p), bytes);
            cp_async_16_zfill(dst + 1536u, here ? gp + e1[k] : reinterpret_cast<const T *>(go.p), bytes);
          }
        } else if (here) {
          if (!BACK || a.norm) load_unit<T, V>(xp, e0[k], e1[k], xr[k]);
          if (BACK) load_unit<T, V>(gp, e0[k], e1[k], gr[k]);
        } else {
#pragma unroll
          for (int i = 0; i < Raw<T, V>::W; ++i) { xr[k].a[i] = xr[k].b[i] = 0u; gr[k].a[i] = gr[k].b[i] = 0u; }
        }
      }
      p_head += stride;
      if (p_head - slot >= (p_t ? a.heads[1] : a.heads[0])) {      // the other tensor, or the next token
        p_head = first;
        if (p_t == 0u && some[1]) {
          p_t = 1u;
        } else {
          p_t = some[0] ? 0u : 1u;
          p_tok = token_after(p_tok);
        }
      }
    }
    if constexpr (RING) cp_async_commit();
    ++issued;
  };
  if constexpr (RING) {
    for (uint32_t i = 0; i + 1u < kRing; ++i) issue();
  } else {
    issue();
  }
  uint32_t tok = me / s.split;
  int32_t pos_next = half && tok < a.n_rows ? a.pos[tok] : 0;
  while (tok < a.n_rows) {
    const uint32_t next = token_after(tok);
    // ---- the angles of the token ----
    float2 cs[U][V];
    if (half) {
      __syncwarp();                                       // (those of the token before are in registers)
      const double pos = static_cast<double>(pos_next);
      if (next < a.n_rows) pos_next = a.pos[next];
      for (uint32_t f = lane; f < half; f += 32u) {
        double t = pos * a.turns[f];
        t -= rint(t);
        float sn, cn;
        sincospif(2.0f * static_cast<float>(t), &sn, &cn);
        cs_s[f] = make_float2(cn * a.magnitude, sn * a.magnitude);
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint32_t u = sub + static_cast<uint32_t>(k) * s.lanes;
#pragma unroll
        for (int i = 0; i < V; ++i) cs[k][i] = u < s.rot_units ? cs_s[V * u + i] : make_float2(1.0f, 0.0f);
      }
    }
#pragma unroll
    for (uint32_t t = 0; t < 2u; ++t) {                   // queries, keys
      const uint32_t heads = a.heads[t];
      float w[U][2 * V];
      if (a.norm) {
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) { w[k][i] = w_s[t * a.hd + e0[k] + i]; w[k][V + i] = w_s[t * a.hd + e1[k] + i]; }
      }
      float acc[U][2 * V];
      if (BACK) {
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) acc[k][i] = 0.0f;
      }
      T *yp = reinterpret_cast<T *>(a.y[t].p) + (static_cast<int64_t>(tok) * a.y[t].row + static_cast<int64_t>(first) * a.y[t].head);
      const int64_t ys = stride * a.y[t].head;
      for (uint32_t head = first; head - slot < heads; head += stride) {
        const bool live = head < heads;
        float x[U][2 * V], y[U][2 * V];
        if constexpr (RING) {
          cp_async_wait<kRing - 2>();
          const uint32_t src = ring + (taken % kRing) * U * kTensors * 1024u;
#pragma unroll
          for (int k = 0; k < U; ++k) {
            auto part_of = [&](uint32_t at, uint32_t *w) {
              const uint4 v = lds_v4(src + k * kTensors * 1024u + at);
              w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            };
            if (!BACK || a.norm) { part_of(0u, xr[k].a); part_of(512u, xr[k].b); }
            if (BACK) { part_of(1024u, gr[k].a); part_of(1536u, gr[k].b); }
          }
          ++taken;
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (!BACK || a.norm) widen(xr[k], x[k]);
          if (BACK) widen(gr[k], y[k]);
        }
        issue();
        float r = 1.0f;
        if (a.norm) {
          float ss[2] = {0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < U; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) { ss[0] += x[k][i] * x[k][i]; ss[1] += x[k][V + i] * x[k][V + i]; }
          const float sum = row_sum(ss[0] + ss[1], s.lanes);
          r = live ? rsqrtf(sum * inv_hd + a.eps) : 0.0f;       // (no row: adds nothing to the weights' gradients)
        }
        if (!BACK) {
#pragma unroll
          for (int k = 0; k < U; ++k) {
            if (a.norm) {
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) x[k][i] *= r * w[k][i];
            }
            if (half) turn<V>(x[k], cs[k], inter, 1.0f);
            if (live && has[k]) store_unit<T, V>(yp, e0[k], e1[k], x[k]);
          }
        } else {
          float hx[2] = {0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < U; ++k) {
            if (half) turn<V>(y[k], cs[k], inter, -1.0f);
            if (a.norm) {
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) {
                acc[k][i] += y[k][i] * (x[k][i] * r);
                y[k][i] *= w[k][i];
                hx[i >= V] += y[k][i] * x[k][i];
              }
            }
          }
          if (a.norm) {
            const float c = row_sum(hx[0] + hx[1], s.lanes) * inv_hd * r * r * r;
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) y[k][i] = r * y[k][i] - c * x[k][i];
          }
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (live && has[k]) store_unit<T, V>(yp, e0[k], e1[k], y[k]);
        }
        yp += ys;
      }
      if (sums) {
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) acc_s[((t * U + k) * 2 * V + i) * 32] += acc[k][i];
      }
    }
    tok = next;
  }
  if (!sums) return;
  // ---- gradients of the weights: lanes of the same unit, then warps, then CTAs ----
  float *red = reinterpret_cast<float *>(sm) + 2u * a.hd + 2u * kRopeWarps * half;        // [warps][2][hd], over the warps' sums
  static_assert(U * 2 * V * 32 >= 256, "room for a warp's rows");
  float v[2][U][2 * V];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) {
        v[t][k][i] = acc_s[((t * U + k) * 2 * V + i) * 32];
        for (uint32_t o = s.lanes; o < 32u; o <<= 1) v[t][k][i] += __shfl_xor_sync(0xffffffffu, v[t][k][i], o);
      }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i)
        if (slot == 0u && has[k]) red[(warp * 2u + t) * a.hd + (i < V ? e0[k] + i : e1[k] + i - V)] = v[t][k][i];
  __syncthreads();
  const uint32_t cols = 2u * a.hd;
  for (uint32_t i = tid; i < cols; i += kRopeThreads) {
    float v = 0.0f;
#pragma unroll
    for (int wp = 0; wp < kRopeWarps; ++wp) v += red[wp * cols + i];
    a.partial[static_cast<size_t>(blockIdx.x) * cols + i] = v;
  }
}

// The CTAs' sums in their order: 32 columns to a CTA, its warps a part of them each.
constexpr uint32_t kSumWarps = 32;
__global__ void __launch_bounds__(kSumWarps * 32) b2_rope_weights(const __grid_constant__ RopeArgs a, uint32_t ctas) {
  __shared__ float red[kSumWarps][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, cols = 2u * a.hd, c = blockIdx.x * 32u + lane;
  const uint32_t per = (ctas + kSumWarps - 1u) / kSumWarps, b1 = min(ctas, (warp + 1u) * per);
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < cols) {
    const float *p = a.partial + c;
    uint32_t b = warp * per;
    for (; b + 8u <= b1; b += 8u) {
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = p[static_cast<size_t>(b + i) * cols];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i & 3] += q[i];
    }
    for (; b < b1; ++b) v[0] += p[static_cast<size_t>(b) * cols];
  }
  red[warp][lane] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  if (warp == 0u && c < cols) {
    float sum = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kSumWarps; ++k) sum += red[k][lane];
    const uint32_t t = c >= a.hd ? 1u : 0u;
    if (a.dw[t]) a.dw[t][c - t * a.hd] = sum;
  }
}

uint32_t Pow2AtLeast(uint32_t v) {
  uint32_t p = 1;
  while (p < v) p *= 2;
  return p;
}

template <typename T, int V, int U, bool BACK>
int Launch(const RopeArgs &a, uint32_t sms, cudaStream_t stream) {
  RopeShape s;
  s.units = a.hd / 2u / V;
  s.rot_units = a.rot / 2u / V;
  s.lanes = Pow2AtLeast(s.units) < 32u ? Pow2AtLeast(s.units) : 32u;
  // Few tokens: a CTA's warps share one, as far as it has heads for them.
  s.split = 1;
  const uint32_t heads = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
  while (s.split < static_cast<uint32_t>(kRopeWarps) && static_cast<uint64_t>(a.n_rows) * s.split < sms * 8u && heads * s.lanes > s.split * 32u) s.split *= 2u;
  const uint64_t want = (static_cast<uint64_t>(a.n_rows) * s.split + kRopeWarps - 1u) / kRopeWarps;
  const uint32_t most = (BACK ? kRopeBackPerSm : kRopePerSm) * sms;
  const uint32_t ctas = want < 1u ? 1u : want > most ? most : static_cast<uint32_t>(want);
  size_t smem = sizeof(float) * 2u * a.hd + sizeof(float2) * kRopeWarps * (a.rot / 2u);
  if (BACK && a.partial) smem += sizeof(float) * kRopeWarps * 2u * U * 2 * V * 32u;
  smem = (smem + 15u) & ~size_t(15);
  s.ring_at = static_cast<uint32_t>(smem);
  if (V * sizeof(T) == 16) smem += kRopeWarps * kRing * (BACK ? 2u : 1u) * 2u * U * 512u;       // 107 KB at most in all
  b2_rope<T, V, U, BACK><<<ctas, kRopeThreads, smem, stream>>>(a, s);
  if (BACK && a.partial) b2_rope_weights<<<(2u * a.hd + 31u) / 32u, kSumWarps * 32u, 0, stream>>>(a, ctas);
  return static_cast<int>(cudaGetLastError());
}

// The widest access that every address of the call allows.
template <typename T>
uint32_t Width(const RopeArgs &a, bool backward) {
  uint32_t v = 16u / sizeof(T);
  const uint32_t half = a.rot / 2u, rest = (a.hd - a.rot) / 2u;
  while (v > 1u && (half % v || rest % v)) v /= 2u;
  auto fit = [&](const RowsRef &r, uint32_t heads) {
    if (!heads || !r.p) return;
    while (v > 1u && (reinterpret_cast<uintptr_t>(r.p) % (v * sizeof(T)) || r.row % static_cast<int64_t>(v) || (heads > 1u && r.head % static_cast<int64_t>(v)))) v /= 2u;
  };
  for (int t = 0; t < 2; ++t) {
    if (!backward || a.norm) fit(a.x[t], a.heads[t]);
    fit(a.y[t], a.heads[t]);
    if (backward) fit(a.g[t], a.heads[t]);
  }
  return v;
}

template <typename T, bool BACK>
int Dispatch(const RopeArgs &a, uint32_t sms, cudaStream_t stream) {
  const uint32_t v = Width<T>(a, BACK);
  if constexpr (sizeof(T) == 2) {
    if (v == 8u) return Launch<T, 8, 1, BACK>(a, sms, stream);
  }
  if (v >= 4u) return Launch<T, 4, 1, BACK>(a, sms, stream);
  return Launch<T, 1, 4, BACK>(a, sms, stream);
}

}  // namespace

namespace {
constexpr int kRopeSmem = 110 * 1024;                     // more than any shape takes
template <typename T, int V, int U>
cudaError_t Attr() {
  const cudaError_t e = cudaFuncSetAttribute(b2_rope<T, V, U, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRopeSmem);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(b2_rope<T, V, U, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRopeSmem);
}
}  // namespace
int PrepareRope() {
  for (cudaError_t e : {Attr<float, 4, 1>(), Attr<__half, 8, 1>(), Attr<__nv_bfloat16, 8, 1>()})
    if (e != cudaSuccess) return static_cast<int>(e);
  return 0;
}
uint32_t RopeBackwardCtas(uint32_t sms) { return kRopeBackPerSm * sms; }

int LaunchRope(const RopeArgs &a, uint32_t dtype, bool backward, uint32_t sms, CUstream_st *stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (backward) {
    if (dtype == B2_F32) return Dispatch<float, true>(a, sms, s);
    return dtype == B2_BF16 ? Dispatch<__nv_bfloat16, true>(a, sms, s) : Dispatch<__half, true>(a, sms, s);
  }
  if (dtype == B2_F32) return Dispatch<float, false>(a, sms, s);
  return dtype == B2_BF16 ? Dispatch<__nv_bfloat16, false>(a, sms, s) : Dispatch<__half, false>(a, sms, s);
}

}  // namespace b2
