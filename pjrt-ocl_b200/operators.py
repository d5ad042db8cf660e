"""The operators beside the programs (include/b2vm.h): rotary positions with the norms of queries and keys, a paged
cache of keys and values, and the attention of new rows over it. No counterpart in the reference.

Device buffers are the caller's: a torch tensor, whose type, size and device are checked, or an address (`data_ptr()`, or
what `Runtime.AllocDevice` gave), which is taken as it is; rows x heads x head_dim tensors as `Rows`. Calls are enqueued on `stream` (0 = the default stream of the runtime's
device) and not waited for; a refusal raises the same errors as the rest of the package.
"""
from __future__ import annotations

import ctypes
import operator
import threading

from .runtime import _ERRCAP, InvalidArgument, Runtime, _check, _errbuf, _ExecStatus, lib

DTYPES = {"f32": 0, "f16": 6, "bf16": 7, "e4m3": 8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
_TORCH = {"torch.float32": "f32", "torch.float16": "f16", "torch.bfloat16": "bf16"}
SCALINGS = {"plain": 0, "linear": 1, "stretch": 2, "parts": 3}

_vp, _u32, _i64 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int64


class _RowsC(ctypes.Structure):
    _fields_ = [("data", _vp), ("row_stride", _i64), ("head_stride", _i64)]


class _RopeDesc(ctypes.Structure):
    _fields_ = [("head_dim", _u32), ("rot_dim", _u32), ("q_heads", _u32), ("k_heads", _u32), ("dtype", _u32), ("weight_dtype", _u32),
                ("interleaved", _u32), ("norm", _u32), ("eps", ctypes.c_float), ("magnitude", ctypes.c_double),
                ("frequencies", ctypes.POINTER(ctypes.c_double))]


class _CacheDesc(ctypes.Structure):
    _fields_ = [("dtype", _u32), ("row_dtype", _u32), ("heads", _u32), ("q_heads", _u32), ("head_dim", _u32), ("page_size", _u32), ("n_pages", _u32),
                ("k_pages", _vp), ("v_pages", _vp), ("page_stride", _i64), ("slot_stride", _i64), ("head_stride", _i64),
                ("k_scales", _vp), ("v_scales", _vp), ("scale_page_stride", _i64), ("scale_slot_stride", _i64), ("scale_head_stride", _i64)]


class _BatchC(ctypes.Structure):
    _fields_ = [("n_seqs", _u32), ("n_rows", _u32), ("max_rows", _u32), ("max_pages", _u32), ("pages_stride", _i64),
                ("row_start", _vp), ("length", _vp), ("pages", _vp)]


class _Local(threading.local):
    """A thread's buffer for messages: what a call writes there is read before the thread makes another."""

    def __init__(self):
        self.err = _errbuf()


_local = _Local()


def _dtype(name: str) -> int:
    if name not in DTYPES:
        raise InvalidArgument(f"unknown type {name!r} (one of {', '.join(DTYPES)})")
    return DTYPES[name]


_NAMES = {"i32": "torch.int32", "f32": "torch.float32", "f16": "torch.float16", "bf16": "torch.bfloat16"}


def _address(what: str, x, dtype: str, n: int, device) -> int:
    """The address of `n` values of a type: an address already, None (0), or a tensor that has them without gaps."""
    if type(x) is int:
        return x
    if x is None:
        return 0
    if not hasattr(x, "data_ptr"):
        return operator.index(x)
    if str(x.dtype) != _NAMES[dtype]:
        raise InvalidArgument(f"{what}: of type {x.dtype}, want {_NAMES[dtype]}")
    if not x.is_cuda or (device is not None and x.device.index != device):
        raise InvalidArgument(f"{what}: on {x.device}, the runtime is on {'a device' if device is None else device}")
    if not x.is_contiguous() or x.numel() < n:
        raise InvalidArgument(f"{what}: {list(x.shape)} of strides {list(x.stride())}, want {n} values without gaps")
    return x.data_ptr()


class Rows:
    """rows x heads x head_dim on the device, the last axis without gaps; strides in elements (default: no gaps)."""

    __slots__ = ("ptr", "dtype", "shape", "device", "_ref", "_keep", "_kind")

    def __init__(self, ptr: int, dtype: str, shape, strides=None, device=None):
        n, heads, dim = (int(x) for x in shape)
        _dtype(dtype)
        strides = (heads * dim, dim) if strides is None else tuple(int(x) for x in strides)
        self.ptr, self.dtype, self.shape, self.device = int(ptr), dtype, (n, heads, dim), device
        self._keep = _RowsC(self.ptr, strides[0], strides[1])
        self._ref = ctypes.byref(self._keep)
        self._kind = (dtype, heads, dim)

    @staticmethod
    def Of(tensor) -> "Rows":
        """A torch tensor [rows, heads, head_dim] (a view will do, if its last axis has stride 1). The tensor must live
        as long as calls that use it are under way."""
        dt = _TORCH.get(str(tensor.dtype))
        if dt is None:
            raise InvalidArgument(f"rows of type {tensor.dtype} (f32, f16 or bf16)")
        if tensor.dim() != 3:
            raise InvalidArgument(f"rows are [rows, heads, head_dim]: got {tuple(tensor.shape)}")
        if not tensor.is_cuda:
            raise InvalidArgument("rows must be in device memory")
        if tensor.shape[2] > 1 and tensor.stride(2) != 1:
            raise InvalidArgument("the last axis of rows must have stride 1")
        return Rows(tensor.data_ptr(), dt, tensor.shape, tensor.stride()[:2], tensor.device.index)


def _rows(what: str, r, device: int, n: int, kind: tuple):
    """The C struct of rows that fit a call: (type, heads, head_dim) are `kind`, at least n rows."""
    if r is None:
        if n and kind[1]:
            raise InvalidArgument(f"{what}: missing")
        return None
    if r._kind != kind or r.shape[0] < n:
        raise InvalidArgument(f"{what}: {r.dtype}{list(r.shape)}, want {kind[0]}[{n} or more, {kind[1]}, {kind[2]}]")
    if r.device is not None and r.device != device:
        raise InvalidArgument(f"{what}: on device {r.device}, the runtime is on {device}")
    return r._ref


class Scratch:
    """Room for partial results. Calls that share one run one after another."""

    def __init__(self, rt: Runtime, handle):
        self._rt, self._h = rt, handle

    @staticmethod
    def Create(rt: Runtime) -> "Scratch":
        h, err = ctypes.c_void_p(), _errbuf()
        _check(lib().b2_scratch_create(rt._h, ctypes.byref(h), err, _ERRCAP), err)
        return Scratch(rt, h)

    def close(self):
        if self._h:
            lib().b2_scratch_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:      # noqa: BLE001
            pass


def RopeFrequencies(rot_dim: int, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0, original_length: float = 0.0,
                    slow: float = 1.0, fast: float = 32.0) -> list:
    """Radians for each position of each pair: base^(-2i/rot_dim), in one of the forms for longer contexts."""
    if scaling not in SCALINGS:
        raise InvalidArgument(f"unknown scaling {scaling!r} (one of {', '.join(SCALINGS)})")
    n = max(0, int(rot_dim)) // 2
    out, err = (ctypes.c_double * max(1, n))(), _errbuf()
    _check(lib().b2_rope_frequencies(int(rot_dim), base, SCALINGS[scaling], factor, original_length, slow, fast, out, n, err, _ERRCAP), err)
    return list(out[:n])


class Rope:
    """Rotary positions of one layer's queries and keys, with their norms where asked."""

    def __init__(self, rt: Runtime, handle, desc: dict):
        self._rt, self._h, self.desc = rt, handle, desc
        self._dev = rt.device_ordinal
        self._dim, self._wt = desc["head_dim"], desc["weight_dtype"]
        self._q, self._k = ((desc["dtype"], desc[heads], desc["head_dim"]) for heads in ("q_heads", "k_heads"))
        self._apply, self._back = lib().b2_rope_apply, lib().b2_rope_apply_backward

    @staticmethod
    def Create(rt: Runtime, head_dim: int, q_heads: int, k_heads: int, dtype: str, rot_dim=None, frequencies=None, interleaved: bool = False,
               norm: bool = False, eps: float = 1e-6, weight_dtype: str = "f32", magnitude: float = 1.0) -> "Rope":
        rot_dim = head_dim if rot_dim is None else rot_dim
        f = RopeFrequencies(rot_dim) if frequencies is None else [float(x) for x in frequencies]
        if len(f) != rot_dim // 2:
            raise InvalidArgument(f"{len(f)} frequencies, want rot_dim / 2 = {rot_dim // 2}")
        arr = (ctypes.c_double * max(1, len(f)))(*f)
        d = _RopeDesc(head_dim, rot_dim, q_heads, k_heads, _dtype(dtype), _dtype(weight_dtype), int(interleaved), int(norm), eps, magnitude, arr)
        h, err = ctypes.c_void_p(), _errbuf()
        _check(lib().b2_rope_create(rt._h if rt is not None else None, ctypes.byref(d), ctypes.byref(h), err, _ERRCAP), err)
        return Rope(rt, h, {"head_dim": head_dim, "q_heads": q_heads, "k_heads": k_heads, "dtype": dtype, "norm": bool(norm), "weight_dtype": weight_dtype})

    def Apply(self, n_rows: int, positions, q, k, q_out, k_out, q_weight=0, k_weight=0, stream: int = 0) -> None:
        """`positions`: int32 [n_rows]; weights: head_dim values each, or 0 (ones)."""
        dev, qk, kk, err = self._dev, self._q, self._k, _local.err
        if not type(positions) is type(q_weight) is type(k_weight) is int:      # (small calls' time is Python's)
            positions = _address("positions", positions, "i32", n_rows, dev)
            q_weight, k_weight = (_address(what, t, self._wt, self._dim, dev) for what, t in (("q_weight", q_weight), ("k_weight", k_weight)))
        st = self._apply(self._h, n_rows, positions, _rows("q", q, dev, n_rows, qk), _rows("k", k, dev, n_rows, kk), q_weight, k_weight,
                         _rows("q_out", q_out, dev, n_rows, qk), _rows("k_out", k_out, dev, n_rows, kk), stream, err, _ERRCAP)
        if st:
            _check(st, err)

    def ApplyBackward(self, n_rows: int, positions, q, k, dq_out, dk_out, dq, dk, q_weight=0, k_weight=0, dq_weight=0, dk_weight=0,
                      scratch: Scratch = None, stream: int = 0) -> None:
        """Gradients; q and k (the inputs of Apply) are needed with norm only, `scratch` for those of the weights."""
        dev, qk, kk, err = self._dev, self._q, self._k, _local.err
        norm = self.desc["norm"]
        x = [None if r is None and not norm else _rows(what, r, dev, n_rows, kind) for what, r, kind in (("q", q, qk), ("k", k, kk))]
        w = [_address(what, t, self._wt, self._dim, dev) for what, t in (("q_weight", q_weight), ("k_weight", k_weight))]
        dw = [_address(what, t, "f32", self._dim, dev) for what, t in (("dq_weight", dq_weight), ("dk_weight", dk_weight))]
        st = self._back(self._h, scratch._h if scratch is not None else None, n_rows, _address("positions", positions, "i32", n_rows, dev), x[0], x[1], w[0], w[1],
                        _rows("dq_out", dq_out, dev, n_rows, qk), _rows("dk_out", dk_out, dev, n_rows, kk),
                        _rows("dq", dq, dev, n_rows, qk), _rows("dk", dk, dev, n_rows, kk), dw[0], dw[1], stream, err, _ERRCAP)
        if st:
            _check(st, err)

    def close(self):
        if self._h:
            lib().b2_rope_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:      # noqa: BLE001
            pass


class Batch:
    """Sequences of a batch: int32 row_start[n_seqs + 1], length[n_seqs] and pages[n_seqs][pages_stride] on the device (tensors are
    kept), and the bounds that the host knows (see b2_batch)."""

    __slots__ = ("_keep", "_ref", "n_rows", "_device", "_tensors")

    def __init__(self, n_seqs: int, row_start, length, pages, max_pages: int, n_rows: int, max_rows: int = 0, pages_stride=None):
        for what, v in (("n_seqs", n_seqs), ("max_pages", max_pages), ("n_rows", n_rows), ("max_rows", max_rows)):
            if not 0 <= v <= 0xFFFFFFFF:
                raise InvalidArgument(f"{what} {v} is out of range")
        self._tensors = [t for t in (row_start, length, pages) if hasattr(t, "data_ptr")]
        self._device = self._tensors[0].device.index if self._tensors and self._tensors[0].is_cuda else None
        if pages_stride is None:
            pages_stride = pages.shape[1] if hasattr(pages, "data_ptr") and pages.dim() == 2 else max_pages
        row_start, length, pages = (_address(what, t, "i32", n, self._device) for what, t, n in (
            ("row_start", row_start, n_seqs + 1), ("length", length, n_seqs), ("pages", pages, (n_seqs - 1) * pages_stride + max_pages if n_seqs else 0)))
        self._keep = _BatchC(n_seqs, n_rows, max_rows, max_pages, pages_stride, row_start, length, pages)
        self._ref = ctypes.byref(self._keep)
        self.n_rows = n_rows


class PagedCache:
    """A view of the caller's pages of keys and values ([page, slot, head, head_dim] unless strides say otherwise)."""

    def __init__(self, rt: Runtime, handle, desc: dict):
        self._rt, self._h, self.desc = rt, handle, desc
        self._dev = rt.device_ordinal
        self._kv, self._q = ((desc["row_dtype"], desc[heads], desc["head_dim"]) for heads in ("heads", "q_heads"))
        self._scale = desc["head_dim"] ** -0.5
        self._write, self._read, self._attend = lib().b2_cache_write, lib().b2_cache_read, lib().b2_cache_attend

    @staticmethod
    def Create(rt: Runtime, dtype: str, row_dtype: str, heads: int, head_dim: int, page_size: int, n_pages: int, k_pages: int, v_pages: int, q_heads=None,
               strides=None, k_scales: int = 0, v_scales: int = 0, scale_strides=None) -> "PagedCache":
        """`strides` / `scale_strides`: (page, slot, head) in elements."""
        q_heads = heads if q_heads is None else q_heads
        s = (page_size * heads * head_dim, heads * head_dim, head_dim) if strides is None else strides
        ss = (page_size * heads, heads, 1) if scale_strides is None else scale_strides
        d = _CacheDesc(_dtype(dtype), _dtype(row_dtype), heads, q_heads, head_dim, page_size, n_pages, k_pages, v_pages, *s, k_scales, v_scales, *ss)
        h, err = ctypes.c_void_p(), _errbuf()
        _check(lib().b2_cache_create(rt._h if rt is not None else None, ctypes.byref(d), ctypes.byref(h), err, _ERRCAP), err)
        return PagedCache(rt, h, {"dtype": dtype, "row_dtype": row_dtype, "heads": heads, "q_heads": q_heads, "head_dim": head_dim})

    def _batch(self, batch: Batch):
        if batch._device not in (None, self._dev):
            raise InvalidArgument(f"batch: on device {batch._device}, the runtime is on {self._dev}")
        return batch._ref

    def Write(self, batch: Batch, k: Rows, v: Rows, stream: int = 0) -> None:
        n, err = batch.n_rows, _local.err
        st = self._write(self._h, self._batch(batch), _rows("k", k, self._dev, n, self._kv), _rows("v", v, self._dev, n, self._kv), stream, err, _ERRCAP)
        if st:
            _check(st, err)

    def Read(self, batch: Batch, k: Rows, v: Rows, stream: int = 0) -> None:
        n, err = batch.n_rows, _local.err
        st = self._read(self._h, self._batch(batch), _rows("k", k, self._dev, n, self._kv), _rows("v", v, self._dev, n, self._kv), stream, err, _ERRCAP)
        if st:
            _check(st, err)

    def Attend(self, batch: Batch, q: Rows, out: Rows, scratch: Scratch, scale=None, causal: bool = True, window: int = 0, lse=0, stream: int = 0) -> None:
        """`scale` defaults to 1 / sqrt(head_dim); `lse`: f32 [n_rows][q_heads], or 0."""
        if not 0 <= window <= 0xFFFFFFFF:
            raise InvalidArgument(f"window {window} is out of range")
        n, err = batch.n_rows, _local.err
        st = self._attend(self._h, scratch._h if scratch is not None else None, self._batch(batch), _rows("q", q, self._dev, n, self._q), self._scale if scale is None else scale,
                          1 if causal else 0, window, _rows("out", out, self._dev, n, self._q), _address("lse", lse, "f32", n * self._q[1], self._dev), stream, err, _ERRCAP)
        if st:
            _check(st, err)

    def set_wait_budget_ns(self, ns: int) -> None:
        """Of each of attention's waits on the tensor cores, for the calls that follow (default 2e9)."""
        lib().b2_cache_set_wait_budget_ns(self._h, ns)

    def Status(self) -> dict:
        """Waits for the device; raises what this cache's calls met since the last report."""
        st, err = _ExecStatus(), _errbuf()
        _check(lib().b2_cache_status(self._h, ctypes.byref(st), err, _ERRCAP), err)
        return {"code": st.code, "lane": st.lane, "where": st.where, "detail": st.detail}

    def close(self):
        if self._h:
            lib().b2_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:      # noqa: BLE001
            pass
