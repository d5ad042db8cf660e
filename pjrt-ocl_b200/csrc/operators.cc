// C entry points of the operators beside the programs (include/b2vm.h): handles, checks, argument blocks. Nothing here
// waits or allocates but the create calls and b2_cache_status; nothing throws out of an entry.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <exception>
#include <mutex>
#include <new>
#include <string>

#include "operators.h"

struct b2_scratch {
  int device = 0;
  uint32_t sms = 0;
  uint8_t *mem = nullptr;          // counters, then partial results
  size_t bytes = 0;
};
struct b2_rope {
  int device = 0;
  uint32_t sms = 0;
  b2_rope_desc desc{};
  double *turns = nullptr;
};
struct b2_cache {
  int device = 0;
  uint32_t sms = 0;
  b2_cache_desc desc{};
  b2::CacheView view{};
  uint64_t wait_budget_ns = 2000000000ull;      // (set while other threads' calls read it)
};

namespace {

constexpr size_t kCounterBytes = b2::kScratchCounters * sizeof(uint32_t);

b2_status Say(char *err, size_t cap, b2_status st, const std::string &m) {
  if (err && cap) std::snprintf(err, cap, "%s", m.c_str());
  return st;
}
b2_status CudaFail(char *err, size_t cap, const char *what, cudaError_t e, b2_status st = B2_INTERNAL) {
  cudaGetLastError();
  return Say(err, cap, st, std::string(what) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
}

// The device of a handle, current for the length of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    e_ = cudaGetDevice(&prev_);
    if (e_ == cudaSuccess && prev_ != device && (e_ = cudaSetDevice(device)) == cudaSuccess) moved_ = true;
  }
  ~OnDevice() { if (moved_) cudaSetDevice(prev_); }
  OnDevice(const OnDevice &) = delete;
  OnDevice &operator=(const OnDevice &) = delete;
  cudaError_t error() const { return e_; }

 private:
  int prev_ = 0;
  bool moved_ = false;
  cudaError_t e_ = cudaSuccess;
};

// The body of an entry: nothing is thrown into C.
template <typename F>
b2_status Entry(const char *name, char *err, size_t cap, F body) {
  try {
    return body();
  } catch (const std::bad_alloc &) {
    return Say(err, cap, B2_RESOURCE_EXHAUSTED, std::string(name) + ": out of host memory");
  } catch (const std::exception &x) {
    return Say(err, cap, B2_INTERNAL, std::string(name) + ": " + x.what());
  } catch (...) {
    return Say(err, cap, B2_INTERNAL, std::string(name) + ": failed");
  }
}
b2_status Refuse(const char *name, char *err, size_t cap, const std::string &m, b2_status st = B2_INVALID_ARGUMENT) {
  return Say(err, cap, st, std::string(name) + ": " + m);
}

b2::RowsRef Ref(const b2_rows *r) {
  if (!r) return b2::RowsRef{nullptr, 0, 0};
  return b2::RowsRef{static_cast<uint8_t *>(r->data), r->row_stride, r->head_stride};
}
b2::BatchView View(const b2_batch *b) {
  b2::BatchView v;
  v.row_start = static_cast<const int32_t *>(b->row_start);
  v.length = static_cast<const int32_t *>(b->length);
  v.pages = static_cast<const int32_t *>(b->pages);
  v.pages_stride = b->pages_stride;
  v.n_seqs = b->n_seqs; v.n_rows = b->n_rows; v.max_rows = b->max_rows; v.max_pages = b->max_pages;
  return v;
}

// What the handles of a device have in common, made with the first of them and kept: the kernels' attributes, and a stream on which the contents of
// a new handle are settled without waiting for anything else on the device. The device is current.
cudaError_t OfDevice(int device, cudaStream_t *stream) {
  static std::mutex lock;
  static cudaStream_t streams[64] = {};
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> held(lock);
  if (!streams[device]) {
    for (int e : {b2::PrepareRope(), b2::PrepareAttendStep(), b2::PrepareAttendChunk()})
      if (e) return static_cast<cudaError_t>(e);
    const cudaError_t e = cudaStreamCreateWithFlags(&streams[device], cudaStreamNonBlocking);
    if (e != cudaSuccess) return e;
  }
  *stream = streams[device];
  return cudaSuccess;
}
b2_status Kind(cudaError_t e) { return e == cudaErrorMemoryAllocation ? B2_RESOURCE_EXHAUSTED : B2_INTERNAL; }

// Memory of a handle that goes. Waits for what uses it; a capture that is under way on some stream stays as it is.
void Release(void *p) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  cudaFree(p);
  cudaThreadExchangeStreamCaptureMode(&mode);
  cudaGetLastError();
}

// What every create call needs of a runtime.
template <typename H>
b2_status OfRuntime(const char *name, b2_runtime *rt, H *h, char *err, size_t cap) {
  if (!rt) return Refuse(name, err, cap, "null runtime");
  b2_device_info info;
  const b2_status st = b2_runtime_info(rt, &info);
  if (st != B2_OK) return Refuse(name, err, cap, "no device", st);
  h->device = info.device_ordinal;
  h->sms = info.sm_count;
  return B2_OK;
}

b2_status Move(const char *name, b2_cache *c, const b2_batch *batch, const b2_rows *k, const b2_rows *v, void *stream, bool write, char *err, size_t cap) {
  if (!c) return Refuse(name, err, cap, "null cache");
  std::string m = b2::CheckBatch(batch);
  if (m.empty()) m = b2::CheckRows("k", k, batch->n_rows, c->desc.heads, c->desc.row_dtype);
  if (m.empty()) m = b2::CheckRows("v", v, batch->n_rows, c->desc.heads, c->desc.row_dtype);
  if (m.empty() && !write) {
    const b2_cache_desc &d = c->desc;
    if ((m = b2::CheckResult("k", k, batch->n_rows, d.heads, d.head_dim, d.row_dtype)).empty()) m = b2::CheckResult("v", v, batch->n_rows, d.heads, d.head_dim, d.row_dtype);
  }
  if (!m.empty()) return Refuse(name, err, cap, m);
  if (!batch->n_seqs || !batch->n_rows) return B2_OK;
  OnDevice on(c->device);
  cudaError_t e = on.error();
  if (e == cudaSuccess)
    e = static_cast<cudaError_t>(b2::LaunchCacheMove(c->view, View(batch), Ref(k), Ref(v), c->desc.dtype, c->desc.row_dtype, write, c->sms, static_cast<cudaStream_t>(stream)));
  return e == cudaSuccess ? B2_OK : CudaFail(err, cap, name, e);
}

}  // namespace

extern "C" {

// ---- scratch -------------------------------------------------------------------------------
b2_status b2_scratch_create(b2_runtime *rt, b2_scratch **out, char *err, size_t err_cap) {
  return Entry("b2_scratch_create", err, err_cap, [&]() -> b2_status {
    if (!out) return Refuse("b2_scratch_create", err, err_cap, "null result");
    *out = nullptr;
    b2_scratch s;
    const b2_status st = OfRuntime("b2_scratch_create", rt, &s, err, err_cap);
    if (st != B2_OK) return st;
    OnDevice on(s.device);
    const size_t uses[3] = {sizeof(float) * 2 * 256 * b2::RopeBackwardCtas(s.sms), b2::AttendStepPartialBytes(s.sms), b2::AttendChunkPartialBytes(s.sms)};
    s.bytes = kCounterBytes + std::max(uses[0], std::max(uses[1], uses[2]));
    cudaStream_t own = nullptr;
    cudaError_t e = on.error();
    if (e == cudaSuccess) e = OfDevice(s.device, &own);
    if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void **>(&s.mem), s.bytes);
    if (e != cudaSuccess) return CudaFail(err, err_cap, "b2_scratch_create", e, Kind(e));
    e = cudaMemsetAsync(s.mem, 0, kCounterBytes, own);
    if (e == cudaSuccess) e = cudaStreamSynchronize(own);
    b2_scratch *h = e == cudaSuccess ? new (std::nothrow) b2_scratch(s) : nullptr;
    if (!h) {
      cudaFree(s.mem);
      return e != cudaSuccess ? CudaFail(err, err_cap, "b2_scratch_create", e) : Refuse("b2_scratch_create", err, err_cap, "out of host memory", B2_RESOURCE_EXHAUSTED);
    }
    *out = h;
    return B2_OK;
  });
}
void b2_scratch_destroy(b2_scratch *s) {
  if (!s) return;
  OnDevice on(s->device);
  Release(s->mem);
  delete s;
}

// ---- rotary positions ------------------------------------------------------------------------
b2_status b2_rope_frequencies(uint32_t rot_dim, double base, int scaling, double factor, double original_length, double slow, double fast, double *out,
                              size_t out_cap, char *err, size_t err_cap) {
  return Entry("b2_rope_frequencies", err, err_cap, [&]() -> b2_status {
    const char *name = "b2_rope_frequencies";
    if (rot_dim % 2 || rot_dim > 256) return Refuse(name, err, err_cap, "rot_dim " + std::to_string(rot_dim) + " (even, at most 256)");
    if (out_cap < rot_dim / 2 || (!out && rot_dim)) return Refuse(name, err, err_cap, "room for " + std::to_string(rot_dim / 2) + " values is needed");
    if (!(base > 0.0) || !std::isfinite(base)) return Refuse(name, err, err_cap, "base must be positive");
    if (scaling < B2_ROPE_PLAIN || scaling > B2_ROPE_PARTS) return Refuse(name, err, err_cap, "unknown scaling " + std::to_string(scaling));
    if (scaling != B2_ROPE_PLAIN && (!(factor > 0.0) || !std::isfinite(factor))) return Refuse(name, err, err_cap, "factor must be positive");
    if (scaling == B2_ROPE_PARTS && (!(original_length > 0.0) || !std::isfinite(original_length) || !std::isfinite(slow) || !std::isfinite(fast) || !(fast > slow)))
      return Refuse(name, err, err_cap, "needs original_length > 0 and fast > slow");
    const double b = scaling == B2_ROPE_STRETCH && rot_dim > 2 ? base * std::pow(factor, static_cast<double>(rot_dim) / (rot_dim - 2)) : base;
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
      double f = std::pow(b, -2.0 * i / rot_dim);
      if (scaling == B2_ROPE_LINEAR) f /= factor;
      if (scaling == B2_ROPE_PARTS) {
        double keep = (original_length * f / (2.0 * 3.14159265358979323846) - slow) / (fast - slow);
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        f *= keep + (1.0 - keep) / factor;
      }
      out[i] = f;
    }
    return B2_OK;
  });
}

b2_status b2_rope_create(b2_runtime *rt, const b2_rope_desc *desc, b2_rope **out, char *err, size_t err_cap) {
  return Entry("b2_rope_create", err, err_cap, [&]() -> b2_status {
    const char *name = "b2_rope_create";
    if (!out) return Refuse(name, err, err_cap, "null result");
    *out = nullptr;
    const std::string m = b2::CheckRopeDesc(desc);
    if (!m.empty()) return Refuse(name, err, err_cap, m);
    b2_rope r;
    const b2_status st = OfRuntime(name, rt, &r, err, err_cap);
    if (st != B2_OK) return st;
    r.desc = *desc;
    r.desc.frequencies = nullptr;
    double turns[128];
    for (uint32_t i = 0; i < desc->rot_dim / 2; ++i) turns[i] = desc->frequencies[i] / (2.0 * 3.14159265358979323846);
    OnDevice on(r.device);
    cudaStream_t own = nullptr;
    cudaError_t e = on.error();
    if (e == cudaSuccess) e = OfDevice(r.device, &own);
    if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void **>(&r.turns), sizeof turns);
    if (e != cudaSuccess) return CudaFail(err, err_cap, name, e, Kind(e));
    e = cudaMemcpyAsync(r.turns, turns, sizeof(double) * (desc->rot_dim / 2), cudaMemcpyHostToDevice, own);
    if (e == cudaSuccess) e = cudaStreamSynchronize(own);
    b2_rope *h = e == cudaSuccess ? new (std::nothrow) b2_rope(r) : nullptr;
    if (!h) {
      cudaFree(r.turns);
      return e != cudaSuccess ? CudaFail(err, err_cap, name, e) : Refuse(name, err, err_cap, "out of host memory", B2_RESOURCE_EXHAUSTED);
    }
    *out = h;
    return B2_OK;
  });
}
void b2_rope_destroy(b2_rope *r) {
  if (!r) return;
  OnDevice on(r->device);
  Release(r->turns);
  delete r;
}

static b2_status RopeCall(const char *name, const b2_rope *r, b2_scratch *scratch, bool backward, uint32_t n_rows, const void *positions, const b2_rows *const (&x)[2],
                          const void *const (&w)[2], const b2_rows *const (&g)[2], const b2_rows *const (&y)[2], void *const (&dw)[2], void *stream, char *err, size_t cap) {
  if (!r) return Refuse(name, err, cap, "null rope");
  const b2_rope_desc &d = r->desc;
  if (n_rows > 0x7fffffffu) return Refuse(name, err, cap, "n_rows " + std::to_string(n_rows) + " (below 2^31)");
  if (n_rows && !positions && d.rot_dim) return Refuse(name, err, cap, "null positions");
  if (reinterpret_cast<uintptr_t>(positions) % 4) return Refuse(name, err, cap, "positions must be 4-byte aligned");
  b2::RopeArgs a;
  std::memset(static_cast<void *>(&a), 0, sizeof a);
  const uint32_t heads[2] = {d.q_heads, d.k_heads};
  const char *const of[2] = {"q", "k"};
  const bool need_x = !backward || d.norm;
  bool any_dw = false;
  for (int t = 0; t < 2; ++t) {
    std::string m;
    if (need_x) m = b2::CheckRows(of[t], x[t], n_rows, heads[t], d.dtype);
    if (m.empty()) m = b2::CheckRows(backward ? "gradient of an input" : "result", y[t], n_rows, heads[t], d.dtype);
    if (m.empty() && backward) m = b2::CheckRows("gradient of a result", g[t], n_rows, heads[t], d.dtype);
    const size_t wa = d.weight_dtype == B2_F32 ? 4 : 2;
    if (m.empty() && reinterpret_cast<uintptr_t>(w[t]) % wa) m = "weights must be aligned to their type";
    if (m.empty() && reinterpret_cast<uintptr_t>(dw[t]) % 4) m = "gradients of weights must be 4-byte aligned";
    if (m.empty() && dw[t] && !d.norm) m = "gradients of weights without a norm";
    if (!m.empty()) return Refuse(name, err, cap, m);
    if (need_x) a.x[t] = Ref(x[t]);
    a.y[t] = Ref(y[t]);
    a.g[t] = Ref(g[t]);
    a.w[t] = w[t];
    a.dw[t] = heads[t] ? static_cast<float *>(dw[t]) : nullptr;
    if (dw[t] && !heads[t]) return Refuse(name, err, cap, "gradients of weights of no heads");
    a.heads[t] = heads[t];
    any_dw = any_dw || a.dw[t];
  }
  for (int t = 0; t < 2; ++t) {
    const char *const result = backward ? "gradient of an input" : "result";
    std::string m = b2::CheckResult(result, y[t], n_rows, heads[t], d.head_dim, d.dtype);
    for (int u = 0; u < 2 && m.empty(); ++u) {
      if (need_x) m = b2::CheckApart(result, y[t], heads[t], of[u], x[u], heads[u], n_rows, d.head_dim, d.dtype, t == u);
      if (m.empty() && backward) m = b2::CheckApart(result, y[t], heads[t], "gradient of a result", g[u], heads[u], n_rows, d.head_dim, d.dtype, t == u);
    }
    if (m.empty() && t) m = b2::CheckApart(result, y[1], heads[1], "the other result", y[0], heads[0], n_rows, d.head_dim, d.dtype, false);
    if (!m.empty()) return Refuse(name, err, cap, m);
  }
  if (any_dw) {
    if (!scratch) return Refuse(name, err, cap, "gradients of weights need a scratch");
    if (scratch->device != r->device) return Refuse(name, err, cap, "the scratch is another device's");
    a.partial = reinterpret_cast<float *>(scratch->mem + kCounterBytes);
  }
  if (!n_rows && !any_dw) return B2_OK;
  a.pos = static_cast<const int32_t *>(positions);
  a.turns = r->turns;
  a.magnitude = static_cast<float>(d.magnitude);
  a.eps = d.eps;
  a.n_rows = n_rows; a.hd = d.head_dim; a.rot = d.rot_dim; a.interleaved = d.interleaved ? 1u : 0u; a.norm = d.norm ? 1u : 0u;
  a.weight_f32 = d.weight_dtype == B2_F32 ? 1u : 0u;
  OnDevice on(r->device);
  cudaError_t e = on.error();
  if (e == cudaSuccess) e = static_cast<cudaError_t>(b2::LaunchRope(a, d.dtype, backward, r->sms, static_cast<cudaStream_t>(stream)));
  return e == cudaSuccess ? B2_OK : CudaFail(err, cap, name, e);
}

b2_status b2_rope_apply(const b2_rope *rope, uint32_t n_rows, const void *positions, const b2_rows *q, const b2_rows *k, const void *q_weight, const void *k_weight,
                        const b2_rows *q_out, const b2_rows *k_out, void *cuda_stream, char *err, size_t err_cap) {
  return Entry("b2_rope_apply", err, err_cap, [&]() -> b2_status {
    return RopeCall("b2_rope_apply", rope, nullptr, false, n_rows, positions, {q, k}, {q_weight, k_weight}, {nullptr, nullptr}, {q_out, k_out}, {nullptr, nullptr}, cuda_stream,
                    err, err_cap);
  });
}
b2_status b2_rope_apply_backward(const b2_rope *rope, b2_scratch *scratch, uint32_t n_rows, const void *positions, const b2_rows *q, const b2_rows *k, const void *q_weight,
                                 const void *k_weight, const b2_rows *dq_out, const b2_rows *dk_out, const b2_rows *dq, const b2_rows *dk, void *dq_weight, void *dk_weight,
                                 void *cuda_stream, char *err, size_t err_cap) {
  return Entry("b2_rope_apply_backward", err, err_cap, [&]() -> b2_status {
    return RopeCall("b2_rope_apply_backward", rope, scratch, true, n_rows, positions, {q, k}, {q_weight, k_weight}, {dq_out, dk_out}, {dq, dk}, {dq_weight, dk_weight},
                    cuda_stream, err, err_cap);
  });
}

// ---- the paged cache -------------------------------------------------------------------------
b2_status b2_cache_create(b2_runtime *rt, const b2_cache_desc *desc, b2_cache **out, char *err, size_t err_cap) {
  return Entry("b2_cache_create", err, err_cap, [&]() -> b2_status {
    const char *name = "b2_cache_create";
    if (!out) return Refuse(name, err, err_cap, "null result");
    *out = nullptr;
    const std::string m = b2::CheckCacheDesc(desc);
    if (!m.empty()) return Refuse(name, err, err_cap, m);
    b2_cache c;
    const b2_status st = OfRuntime(name, rt, &c, err, err_cap);
    if (st != B2_OK) return st;
    c.desc = *desc;
    b2::CacheView &v = c.view;
    const int64_t e = b2::TypeBytes(desc->dtype);
    v.k = static_cast<uint8_t *>(desc->k_pages); v.v = static_cast<uint8_t *>(desc->v_pages);
    v.ks = desc->k_scales; v.vs = desc->v_scales;
    v.page_bytes = desc->page_stride * e; v.slot_bytes = desc->slot_stride * e; v.head_bytes = desc->head_stride * e;
    v.s_page = desc->scale_page_stride; v.s_slot = desc->scale_slot_stride; v.s_head = desc->scale_head_stride;
    v.n_pages = desc->n_pages; v.page_size = desc->page_size; v.heads = desc->heads; v.hd = desc->head_dim;
    v.by_page = b2::FastDiv(desc->page_size);
    OnDevice on(c.device);
    cudaStream_t own = nullptr;
    cudaError_t ce = on.error();
    if (ce == cudaSuccess) ce = OfDevice(c.device, &own);
    if (ce == cudaSuccess) ce = cudaMalloc(reinterpret_cast<void **>(&v.status), 4 * sizeof(uint32_t));
    if (ce != cudaSuccess) return CudaFail(err, err_cap, name, ce, Kind(ce));
    ce = cudaMemsetAsync(v.status, 0, 4 * sizeof(uint32_t), own);
    if (ce == cudaSuccess) ce = cudaStreamSynchronize(own);
    b2_cache *h = ce == cudaSuccess ? new (std::nothrow) b2_cache(c) : nullptr;
    if (!h) {
      cudaFree(v.status);
      return ce != cudaSuccess ? CudaFail(err, err_cap, name, ce) : Refuse(name, err, err_cap, "out of host memory", B2_RESOURCE_EXHAUSTED);
    }
    *out = h;
    return B2_OK;
  });
}
void b2_cache_destroy(b2_cache *c) {
  if (!c) return;
  OnDevice on(c->device);
  Release(c->view.status);
  delete c;
}

void b2_cache_set_wait_budget_ns(b2_cache *cache, uint64_t ns) {
  if (cache) __atomic_store_n(&cache->wait_budget_ns, ns, __ATOMIC_RELAXED);
}

b2_status b2_cache_write(b2_cache *cache, const b2_batch *batch, const b2_rows *k, const b2_rows *v, void *cuda_stream, char *err, size_t err_cap) {
  return Entry("b2_cache_write", err, err_cap, [&]() -> b2_status { return Move("b2_cache_write", cache, batch, k, v, cuda_stream, true, err, err_cap); });
}
b2_status b2_cache_read(b2_cache *cache, const b2_batch *batch, const b2_rows *k, const b2_rows *v, void *cuda_stream, char *err, size_t err_cap) {
  return Entry("b2_cache_read", err, err_cap, [&]() -> b2_status { return Move("b2_cache_read", cache, batch, k, v, cuda_stream, false, err, err_cap); });
}

b2_status b2_cache_attend(b2_cache *cache, b2_scratch *scratch, const b2_batch *batch, const b2_rows *q, float scale, int causal, uint32_t window, const b2_rows *out,
                          void *lse, void *cuda_stream, char *err, size_t err_cap) {
  return Entry("b2_cache_attend", err, err_cap, [&]() -> b2_status {
    const char *name = "b2_cache_attend";
    if (!cache) return Refuse(name, err, err_cap, "null cache");
    const b2_cache_desc &d = cache->desc;
    std::string m = b2::CheckAttend(d, batch, q, out, scale, causal, window, lse);
    if (m.empty()) m = b2::CheckResult("out", out, batch->n_rows, d.q_heads, d.head_dim, d.row_dtype);
    if (m.empty()) m = b2::CheckApart("out", out, d.q_heads, "q (a row of q may be read after its result is there)", q, d.q_heads, batch->n_rows, d.head_dim, d.row_dtype, false);
    if (!m.empty()) return Refuse(name, err, err_cap, m, d.row_dtype == B2_F32 && b2::CheckBatch(batch).empty() ? B2_UNIMPLEMENTED : B2_INVALID_ARGUMENT);
    if (!scratch) return Refuse(name, err, err_cap, "null scratch");
    if (scratch->device != cache->device) return Refuse(name, err, err_cap, "the scratch is another device's");
    if (!batch->n_seqs || !batch->n_rows) return B2_OK;
    b2::AttendArgs a;
    std::memset(static_cast<void *>(&a), 0, sizeof a);
    a.c = cache->view;
    a.b = View(batch);
    if (!a.b.max_rows || a.b.max_rows > a.b.n_rows) a.b.max_rows = a.b.n_rows;
    a.q = Ref(q);
    a.o = Ref(out);
    a.lse = static_cast<float *>(lse);
    a.arrived = reinterpret_cast<uint32_t *>(scratch->mem);
    a.part = reinterpret_cast<float *>(scratch->mem + kCounterBytes);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.q_heads = d.q_heads;
    a.group = d.q_heads / d.heads;
    a.by_group = b2::FastDiv(a.group);
    a.causal = causal ? 1u : 0u;
    a.window = window;
    a.bf16 = d.row_dtype == B2_BF16 ? 1u : 0u;
    a.e4m3 = d.dtype == B2_E4M3 ? 1u : 0u;
    a.wait_budget_ns = __atomic_load_n(&cache->wait_budget_ns, __ATOMIC_RELAXED);
    OnDevice on(cache->device);
    cudaError_t e = on.error();
    if (e == cudaSuccess) {
      // Up to 16 rows (rows x heads that share a cache head) are one tile of warp-level products, bound by the cache's
      // bytes; more are the tensor cores'.
      if (static_cast<uint64_t>(a.b.max_rows) * a.group <= b2::kStepRows) {
        e = static_cast<cudaError_t>(b2::LaunchAttendStep(a, cache->sms, static_cast<cudaStream_t>(cuda_stream)));
      } else {
        e = static_cast<cudaError_t>(b2::LaunchAttendChunk(a, cache->sms, static_cast<cudaStream_t>(cuda_stream)));
      }
    }
    return e == cudaSuccess ? B2_OK : CudaFail(err, err_cap, name, e);
  });
}

b2_status b2_cache_status(b2_cache *cache, b2_exec_status *out, char *err, size_t err_cap) {
  return Entry("b2_cache_status", err, err_cap, [&]() -> b2_status {
    const char *name = "b2_cache_status";
    if (!cache || !out) return Refuse(name, err, err_cap, "null argument");
    std::memset(out, 0, sizeof *out);
    OnDevice on(cache->device);
    uint32_t w[4] = {0, 0, 0, 0};
    cudaError_t e = on.error();
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(w, cache->view.status, sizeof w, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && w[0]) {
      e = cudaMemset(cache->view.status, 0, sizeof w);
      if (e == cudaSuccess) e = cudaDeviceSynchronize();
    }
    if (e != cudaSuccess) return CudaFail(err, err_cap, name, e);
    out->code = w[0]; out->lane = w[1]; out->where = w[2]; out->detail = w[3];
    switch (w[0]) {
      case 0: return B2_OK;
      case b2::kStBadPage:
        return Refuse(name, err, err_cap, "sequence " + std::to_string(w[1]) + " names page " + std::to_string(static_cast<int32_t>(w[3])) + " (entry " + std::to_string(w[2]) + ") of " +
                                              std::to_string(cache->desc.n_pages));
      case b2::kStBadBatch:
        return Refuse(name, err, err_cap, "sequence " + std::to_string(w[1]) + " does not fit the batch's bounds (value " + std::to_string(static_cast<int32_t>(w[3])) + ")");
      default:
        return Refuse(name, err, err_cap, "a wait on the tensor cores ran out", B2_DEADLINE_EXCEEDED);
    }
  });
}

}  // extern "C"
