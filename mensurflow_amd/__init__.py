"""mensurflow_amd -- an MI355X (gfx950) backend for mensurflow's fp32 BLAS hot path.

The product is two native libraries built in-tree (``mensurflow_amd/build.py``):

* ``_lib/libmfr_rocm.so``: hand-written HIP kernels behind the C ABI of
  ``include/mfr_rocm.h`` (fp32-MFMA GEMM with a fused epilogue, HBM-bound gemv, softmax,
  where, bias+gelu, argmax, strided copy; for serving in 8 bits, RMS norm, conversion to e4m3 with
  block scales, and products of such matrices);
* ``_lib/libmensurflow.so``: the C++17 host layer that plugs those kernels into mensurflow's
  ``Backend``/``Dispatcher`` API as the ``rocm`` device.

This Python module is a thin driver over the C ABI (device buffers, streams, events and the
compute entry points), used by the tests and ``bench.py``. It has no CPU fallback: without the
library, or without a gfx950 device, every call raises.
"""
from __future__ import annotations

import ctypes
import threading
from dataclasses import dataclass

import numpy as np

from . import abi
from .abi import (ACT_GELU_ERF, ACT_GELU_TANH, ACT_NONE, ACT_SILU, F8GemmDesc,  # noqa: F401
                  GemmDesc, RmsNormDesc)

__all__ = [
    "ACT_NONE", "ACT_GELU_TANH", "ACT_GELU_ERF", "GemmDesc", "device_count", "device_info",
    "Stream", "DeviceArray", "Event", "sgemm", "gemm", "gemm_batched", "sgemv", "matvec", "dot",
    "bias_act", "where", "where_nd", "elementwise", "softmax", "argmax", "strided_copy", "fill", "attention",
    "attention_fused", "attention_composed", "gemm_plan",
    "ACT_SILU", "F8Matrix", "F8GemmDesc", "RmsNormDesc", "quantize_f8", "rms_norm_desc",
    "rms_norm_run", "rms_norm", "rms_norm_f8", "f8gemm_desc", "f8gemm", "f8gemm_plan", "gemm_f8",
    "gemm_f8_gated",
]


def device_count() -> int:
    """Usable gfx950 devices (0 without a driver or device)."""
    lib = abi.load()
    n = ctypes.c_int(0)
    abi.check(lib.mfr_get_device_count(ctypes.byref(n)), "mfr_get_device_count")
    return n.value


@dataclass
class DeviceInfo:
    name: str
    memory_bytes: int
    compute_units: int
    clock_khz: int


def device_info(device: int = 0) -> DeviceInfo:
    lib = abi.load()
    name = ctypes.create_string_buffer(256)
    mem = ctypes.c_size_t(0)
    cus = ctypes.c_int(0)
    clk = ctypes.c_int(0)
    abi.check(lib.mfr_get_device_info(device, name, 256, ctypes.byref(mem), ctypes.byref(cus),
                                      ctypes.byref(clk)), "mfr_get_device_info")
    return DeviceInfo(name.value.decode(), mem.value, cus.value, clk.value)


class Stream:
    """An mfr_stream_t: one HIP stream on one device with its kernel workspace.

    The stream keeps the device memory of arrays released on it for its later allocations.
    Kernels and copies on one stream run in order, so work on a new array that takes a released
    block is queued after every use of the old array, and neither the release nor the allocation
    waits for the device (hipFree waits for the whole device; hipMalloc of a large block costs
    tens of microseconds). Blocks come in size classes (powers of two below 1 MiB, at least
    512 B; multiples of 2 MiB above); idle blocks are kept up to 1/8 of the device's memory
    (at least 1 GiB), past that a released block is freed. An array used by work queued on
    another stream must be released only after that work is done, as before."""

    _SMALL = 1 << 20
    _LARGE_STEP = 2 << 20

    def __init__(self, device: int = 0):
        handle = ctypes.c_void_p()
        abi.check(abi.load().mfr_stream_create(device, ctypes.byref(handle)), "mfr_stream_create")
        self._adopt(handle, device)

    def _adopt(self, handle, device: int) -> None:
        lib = abi.load()
        self.device = device
        self.handle = handle
        self._scratch: dict = {}
        self._idle: dict = {}
        self._idle_bytes = 0
        self._pool_lock = threading.Lock()   # host threads may share a stream
        mem = ctypes.c_size_t(0)
        lib.mfr_get_device_info(device, None, 0, ctypes.byref(mem), None, None)
        self._idle_limit = max(mem.value // 8, 1 << 30)

    @classmethod
    def wrap(cls, hip_stream: int, device: int = 0) -> "Stream":
        """A Stream over a HIP stream that another library owns (its handle as an integer, 0 for
        the default stream): kernels order with that library's work (mfr_stream_wrap). The HIP
        stream stays its owner's."""
        lib = abi.load()
        out = cls.__new__(cls)
        out.handle = None
        handle = ctypes.c_void_p()
        abi.check(lib.mfr_stream_wrap(device, ctypes.c_void_p(hip_stream or None),
                                      ctypes.byref(handle)), "mfr_stream_wrap")
        out._adopt(handle, device)
        return out

    @classmethod
    def size_class(cls, nbytes: int) -> int:
        if nbytes >= cls._SMALL:
            return (nbytes + cls._LARGE_STEP - 1) // cls._LARGE_STEP * cls._LARGE_STEP
        size = 512
        while size < nbytes:
            size *= 2
        return size

    def _take(self, size: int) -> int:
        """A device block of `size` bytes (a size class): an idle one, else a new allocation."""
        with self._pool_lock:
            blocks = self._idle.get(size)
            if blocks:
                self._idle_bytes -= size
                return blocks.pop()
        lib = abi.load()
        ptr = ctypes.c_void_p()
        if lib.mfr_malloc(self.device, size, ctypes.byref(ptr)) != abi.MFR_OK:
            self.release_idle()
            abi.check(lib.mfr_malloc(self.device, size, ctypes.byref(ptr)), "mfr_malloc")
        return ptr.value or 0

    def _give(self, size: int, ptr: int) -> None:
        with self._pool_lock:
            if self.handle is not None and self._idle_bytes + size <= self._idle_limit:
                self._idle.setdefault(size, []).append(ptr)
                self._idle_bytes += size
                return
        if self.handle is not None:
            self.synchronize()
        abi.check(abi.load().mfr_free(self.device, ptr), "mfr_free")

    def release_idle(self) -> None:
        """Free the idle blocks (after the work queued on the stream is done)."""
        if not self._idle:
            return
        if self.handle is not None:
            self.synchronize()
        lib = abi.load()
        with self._pool_lock:
            idle, self._idle, self._idle_bytes = self._idle, {}, 0
        for blocks in idle.values():
            for ptr in blocks:
                abi.check(lib.mfr_free(self.device, ptr), "mfr_free")

    def scratch(self, tag, shape, dtype=np.float32) -> "DeviceArray":
        """A device array of `shape` for temporaries of work queued on this stream. Each tag
        keeps one allocation between calls, replaced by a larger one when a call needs more.
        Work on one stream runs in order, so the temporaries of an earlier call are no longer
        read when later work on this stream writes them. The contents are whatever the last
        user of the tag left there."""
        dtype = np.dtype(dtype)
        nbytes = int(np.prod(shape, dtype=np.int64)) * dtype.itemsize
        held = self._scratch.get(tag)
        if held is None or held.nbytes_alloc < nbytes:
            if held is not None:
                held.close()
            held = DeviceArray((max(nbytes, 1),), np.uint8, self)
            self._scratch[tag] = held
        return DeviceArray(shape, dtype, self, _base=held, _ptr=held._ptr)

    def synchronize(self) -> None:
        abi.check(abi.load().mfr_stream_sync(self.handle), "mfr_stream_sync")

    def hip_stream(self) -> int:
        return abi.load().mfr_stream_handle(self.handle) or 0

    def close(self) -> None:
        for held in self._scratch.values():
            held.close()
        self._scratch.clear()
        self.release_idle()
        if self.handle is not None and self.handle.value:
            abi.check(abi.load().mfr_stream_destroy(self.handle), "mfr_stream_destroy")
        self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Event:
    def __init__(self):
        handle = ctypes.c_void_p()
        abi.check(abi.load().mfr_event_create(ctypes.byref(handle)), "mfr_event_create")
        self.handle = handle

    def record(self, stream: Stream) -> None:
        abi.check(abi.load().mfr_event_record(self.handle, stream.handle), "mfr_event_record")

    def elapsed_ms(self, end: "Event") -> float:
        ms = ctypes.c_float(0.0)
        abi.check(abi.load().mfr_event_elapsed_ms(self.handle, end.handle, ctypes.byref(ms)),
                  "mfr_event_elapsed_ms")
        return ms.value

    def __del__(self):
        try:
            if self.handle is not None and self.handle.value:
                abi.load().mfr_event_destroy(self.handle)
            self.handle = None
        except Exception:
            pass


class DeviceArray:
    """A contiguous device allocation viewed with numpy-style shape and element strides.

    Views (``transpose``, ``T``, ``view``, ``slice_rows``) share the allocation; the owner frees
    it when it is garbage collected or closed.
    """

    def __init__(self, shape, dtype=np.float32, stream: Stream | None = None, *, _base=None,
                 _offset=0, _strides=None, _ptr=None):
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        self.stream = stream
        self._base = _base
        self.offset = int(_offset)  # elements from the allocation start
        if _strides is None:
            strides, step = [], 1
            for s in reversed(self.shape):
                strides.append(step)
                step *= s
            _strides = tuple(reversed(strides))
        self.strides = tuple(int(s) for s in _strides)
        if _base is None:
            nbytes = int(np.prod(self.shape, dtype=np.int64)) * self.dtype.itemsize
            if stream is not None and stream.handle is not None and nbytes > 0:
                # A block of the stream's pool, returned to it by close().
                self.nbytes_alloc = Stream.size_class(nbytes)
                self._ptr = stream._take(self.nbytes_alloc)
                self._device = stream.device
            else:
                self.nbytes_alloc = nbytes
                ptr = ctypes.c_void_p()
                dev = stream.device if stream is not None else 0
                abi.check(abi.load().mfr_malloc(dev, nbytes, ctypes.byref(ptr)), "mfr_malloc")
                self._ptr = ptr.value or 0
                self._device = dev
            self._pooled = self._ptr != 0 and stream is not None and stream.handle is not None
        else:
            self._ptr = _ptr
            self._device = _base._device

    # -- construction --------------------------------------------------------------------------
    @classmethod
    def from_numpy(cls, array: np.ndarray, stream: Stream) -> "DeviceArray":
        host = np.ascontiguousarray(array)
        out = cls(host.shape, host.dtype, stream)
        out.upload(host)
        return out

    @classmethod
    def empty(cls, shape, stream: Stream, dtype=np.float32) -> "DeviceArray":
        return cls(shape, dtype, stream)

    @classmethod
    def wrap(cls, ptr: int, shape, stream: Stream, dtype=np.float32, strides=None) -> "DeviceArray":
        """A view of memory that another library owns on the stream's device, `ptr` the address of
        its first element, `strides` in elements (contiguous if None). Nothing frees it here; it
        has to outlive the work queued on it."""
        owner = cls.__new__(cls)
        owner._base, owner._ptr, owner._device = None, 0, stream.device
        return cls(shape, dtype, stream, _base=owner, _strides=strides, _ptr=int(ptr))

    # -- data movement ---------------------------------------------------------------------------
    @property
    def ptr(self) -> int:
        """Device address of the first element of this view."""
        return self._ptr + self.offset * self.dtype.itemsize

    @property
    def size(self) -> int:
        return int(np.prod(self.shape, dtype=np.int64))

    def is_contiguous(self) -> bool:
        step = 1
        for s, st in zip(reversed(self.shape), reversed(self.strides)):
            if s != 1 and st != step:
                return False
            step *= s
        return True

    def upload(self, host: np.ndarray) -> None:
        if not self.is_contiguous():
            raise ValueError("upload needs a contiguous view")
        host = np.ascontiguousarray(host, dtype=self.dtype)
        if host.shape != self.shape:
            raise ValueError(f"upload: host shape {host.shape} differs from {self.shape}")
        abi.check(abi.load().mfr_memcpy_h2d(self.stream.handle, self.ptr, host.ctypes.data,
                                            host.nbytes), "mfr_memcpy_h2d")

    def numpy(self) -> np.ndarray:
        """Copy to the host (waits for queued work), following strides for views."""
        if self.is_contiguous():
            out = np.empty(self.shape, dtype=self.dtype)
            abi.check(abi.load().mfr_memcpy_d2h(self.stream.handle, out.ctypes.data, self.ptr,
                                                out.nbytes), "mfr_memcpy_d2h")
            return out
        packed = strided_copy(self)
        return packed.numpy()

    # -- views -------------------------------------------------------------------------------------
    def _view(self, shape, strides, offset) -> "DeviceArray":
        base = self._base if self._base is not None else self
        v = DeviceArray(shape, self.dtype, self.stream, _base=base, _offset=offset,
                        _strides=strides, _ptr=self._ptr)
        return v

    def transpose(self, d0=-2, d1=-1) -> "DeviceArray":
        nd = len(self.shape)
        d0 %= nd
        d1 %= nd
        shape = list(self.shape)
        strides = list(self.strides)
        shape[d0], shape[d1] = shape[d1], shape[d0]
        strides[d0], strides[d1] = strides[d1], strides[d0]
        return self._view(shape, strides, self.offset)

    @property
    def T(self) -> "DeviceArray":
        return self.transpose(-2, -1)

    def view(self, shape) -> "DeviceArray":
        if not self.is_contiguous():
            raise ValueError("view: the array is not contiguous")
        shape = list(shape)
        if -1 in shape:
            i = shape.index(-1)
            rest = int(np.prod([s for j, s in enumerate(shape) if j != i], dtype=np.int64))
            shape[i] = self.size // rest
        if int(np.prod(shape, dtype=np.int64)) != self.size:
            raise ValueError(f"view: cannot view {self.shape} as {tuple(shape)}")
        strides, step = [], 1
        for s in reversed(shape):
            strides.append(step)
            step *= s
        return self._view(shape, tuple(reversed(strides)), self.offset)

    def expand(self, shape) -> "DeviceArray":
        shape = tuple(int(s) for s in shape)
        lead = len(shape) - len(self.shape)
        strides = [0] * lead
        for i, (s, st) in enumerate(zip(self.shape, self.strides)):
            want = shape[lead + i]
            if s == want:
                strides.append(st)
            elif s == 1:
                strides.append(0)
            else:
                raise ValueError(f"cannot expand {self.shape} to {shape}")
        return self._view(shape, strides, self.offset)

    def slice(self, dim, start, end) -> "DeviceArray":
        shape = list(self.shape)
        shape[dim] = end - start
        return self._view(shape, self.strides, self.offset + start * self.strides[dim])

    def close(self) -> None:
        if self._base is None and self._ptr:
            ptr, self._ptr = self._ptr, 0
            if self._pooled and self.stream.handle is not None:
                # Later users of the block are queued after the work still using this array.
                self.stream._give(self.nbytes_alloc, ptr)
                return
            # Kernels queued on the stream may still read or write this memory.
            if self.stream is not None and self.stream.handle is not None:
                self.stream.synchronize()
            abi.check(abi.load().mfr_free(self._device, ptr), "mfr_free")

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- compute entry points -------------------------------------------------------------------------


def _ptr_or_none(arr):
    return None if arr is None else arr.ptr


def sgemm(stream: Stream, desc: GemmDesc) -> None:
    """mfr_sgemm on a filled descriptor."""
    abi.check(abi.load().mfr_sgemm(stream.handle, ctypes.byref(desc)), "mfr_sgemm")


def _fill_batch(field, values, dims):
    for i in range(dims):
        field[i] = int(values[i])


def gemm_batched(a: DeviceArray, b: DeviceArray, c: DeviceArray, *, alpha=1.0,
                 c0: DeviceArray | None = None, beta=0.0, bias: DeviceArray | None = None,
                 act=ACT_NONE, tile=0, stage=0, splits=0, causal=False) -> None:
    """c[...] = act(alpha*a@b + beta*c0 + bias) over the leading (batch) dimensions.

    a is [..., m, k], b is [..., k, n] (any strides with a unit stride in one matrix dimension;
    batch strides may be 0), c and c0 are [..., m, n] with unit column stride. The batch shapes
    must already agree (expand them first). tile is an abi.TILE_* value, stage an abi.STAGE_*
    value (copy operands that 16-byte loads cannot read into an aligned workspace first), splits
    the number of depth ranges (0 = automatic, 1 = none; split-K, abi.MAX_SPLITS at most).
    causal: c[..., i, j] = -inf wherever j > i (abi.GEMM_CAUSAL, attention's scores); only the
    panel path takes it, NotImplementedError elsewhere.
    """
    sgemm(c.stream, _gemm_desc(a, b, c, alpha, c0, beta, bias, act, tile, stage, splits,
                               causal))


def gemm_plan(a: DeviceArray, b: DeviceArray, c: DeviceArray, *, tile=0, stage=0, splits=0,
              c0: DeviceArray | None = None, beta=0.0,
              causal=False) -> tuple[int, int, int, int]:
    """(tile, stage, splits, regions) that gemm_batched(a, b, c, ...) would run with
    (mfr_sgemm_plan): AUTO resolved to a fixed tile, stage reported as STAGE_ALWAYS (operands
    copied first) or STAGE_NEVER, splits the depth ranges (1 = no split) -- both of the main
    region -- and regions the output rectangles launched separately (more than 1 when AUTO peels
    edge strips). Raises as gemm_batched would for a point that cannot run."""
    d = _gemm_desc(a, b, c, 1.0, c0, beta, None, ACT_NONE, tile, stage, splits, causal)
    t, st, sp, rg = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
    abi.check(abi.load().mfr_sgemm_plan(c.stream.device, ctypes.byref(d), ctypes.byref(t),
                                        ctypes.byref(st), ctypes.byref(sp), ctypes.byref(rg)),
              "mfr_sgemm_plan")
    return t.value, st.value, sp.value, rg.value


def _gemm_desc(a, b, c, alpha, c0, beta, bias, act, tile, stage, splits=0,
               causal=False) -> GemmDesc:
    m, k = a.shape[-2:]
    k2, n = b.shape[-2:]
    if k != k2:
        raise ValueError(f"inner dimensions differ: {a.shape} x {b.shape}")
    batch = c.shape[:-2]
    dims = len(batch)
    if dims > abi.MAX_BATCH_DIMS:
        raise ValueError("too many batch dimensions")
    for t in (a, b) + ((c0,) if c0 is not None else ()):
        if t.shape[:-2] != batch:
            raise ValueError(f"batch shapes differ: {t.shape} vs {c.shape}")
    if c.strides[-1] != 1 or (c0 is not None and c0.strides[-1] != 1):
        raise ValueError("c and c0 need a unit column stride")
    d = GemmDesc()
    d.m, d.n, d.k = m, n, k
    d.batch_dims = dims
    d.act = act
    _fill_batch(d.batch, batch, dims)
    d.a = a.ptr
    d.a_rs, d.a_cs = a.strides[-2], a.strides[-1]
    _fill_batch(d.a_bs, a.strides[:-2], dims)
    d.b = b.ptr
    d.b_rs, d.b_cs = b.strides[-2], b.strides[-1]
    _fill_batch(d.b_bs, b.strides[:-2], dims)
    d.c = c.ptr
    d.c_rs = c.strides[-2]
    _fill_batch(d.c_bs, c.strides[:-2], dims)
    if c0 is not None:
        d.c0 = c0.ptr
        d.c0_rs = c0.strides[-2]
        _fill_batch(d.c0_bs, c0.strides[:-2], dims)
    d.bias = _ptr_or_none(bias)
    d.alpha = alpha
    d.beta = beta
    d.tile = tile
    d.stage = stage
    d.splits = splits
    d.flags = abi.GEMM_CAUSAL if causal else 0
    return d


def gemm(a: DeviceArray, b: DeviceArray, *, alpha=1.0, c0: DeviceArray | None = None, beta=0.0,
         trans_a=False, trans_b=False, bias: DeviceArray | None = None, act=ACT_NONE,
         out: DeviceArray | None = None, tile=0, stage=0, splits=0) -> DeviceArray:
    """mensurflow::gemm's semantics (plus the fused bias/activation): a new [m, n] result."""
    left = a.T if trans_a else a
    right = b.T if trans_b else b
    m, n = left.shape[-2], right.shape[-1]
    if out is None:
        out = DeviceArray.empty((m, n), a.stream)
    gemm_batched(left, right, out, alpha=alpha, c0=c0, beta=beta, bias=bias, act=act, tile=tile,
                 stage=stage, splits=splits)
    return out


def sgemv(a: DeviceArray, x: DeviceArray, *, alpha=1.0, y0: DeviceArray | None = None, beta=0.0,
          trans=False, out: DeviceArray | None = None) -> DeviceArray:
    rows, cols = a.shape
    if a.strides[1] != 1:
        raise ValueError("gemv needs a row-major matrix (unit column stride)")
    n_out = cols if trans else rows
    if out is None:
        out = DeviceArray.empty((n_out,), a.stream)
    abi.check(abi.load().mfr_sgemv(a.stream.handle, 1 if trans else 0, rows, cols, alpha, a.ptr,
                                   a.strides[0], x.ptr, beta, _ptr_or_none(y0), out.ptr),
              "mfr_sgemv")
    return out


def matvec(a: DeviceArray, x: DeviceArray, out: DeviceArray | None = None) -> DeviceArray:
    m, k = a.shape
    if out is None:
        out = DeviceArray.empty((m,), a.stream)
    abi.check(abi.load().mfr_smatvec(a.stream.handle, m, k, a.ptr, a.strides[0], x.ptr, out.ptr),
              "mfr_smatvec")
    return out


def dot(x: DeviceArray, y: DeviceArray, out: DeviceArray | None = None) -> DeviceArray:
    """mensurflow::dot (src/ops/blas.cpp:41-68) through mfr_sdot: sum of x[i] * y[i] over two
    contiguous vectors of equal length, the products and their sum in double, rounded once; a
    0-d array."""
    if x.size != y.size:
        raise ValueError(f"dot: lengths differ ({x.size} and {y.size})")
    if out is None:
        out = DeviceArray.empty((), x.stream)
    abi.check(abi.load().mfr_sdot(x.stream.handle, x.size, x.ptr, y.ptr, out.ptr), "mfr_sdot")
    return out


def bias_act(x: DeviceArray, bias: DeviceArray | None, act=ACT_NONE,
             out: DeviceArray | None = None) -> DeviceArray:
    rows, cols = (x.shape if len(x.shape) == 2 else (1, x.size))
    if out is None:
        out = DeviceArray.empty(x.shape, x.stream)
    abi.check(abi.load().mfr_bias_act(x.stream.handle, x.ptr, _ptr_or_none(bias), out.ptr, rows,
                                      cols, act), "mfr_bias_act")
    return out


def where(cond: DeviceArray, x: DeviceArray, y: DeviceArray,
          out: DeviceArray | None = None) -> DeviceArray:
    if out is None:
        out = DeviceArray.empty(x.shape, x.stream)
    abi.check(abi.load().mfr_where(x.stream.handle, cond.ptr, x.ptr, y.ptr, out.ptr, x.size),
              "mfr_where")
    return out


def where_nd(cond: DeviceArray, x: DeviceArray, y: DeviceArray,
             out: DeviceArray | None = None) -> DeviceArray:
    """out = cond ? x : y with each operand read through its own strides (mfr_where_nd): cond,
    x and y are views of out's shape, expanded (stride 0) where they broadcast."""
    shape = out.shape if out is not None else x.shape
    for t in (cond, x, y):
        if t.shape != shape:
            raise ValueError(f"where_nd: operand shape {t.shape} differs from {shape}")
    if out is None:
        out = DeviceArray.empty(shape, x.stream)
    nd = len(shape)
    arr = ctypes.c_int64 * max(nd, 1)
    abi.check(abi.load().mfr_where_nd(x.stream.handle, nd, arr(*shape), cond.ptr,
                                      arr(*cond.strides), x.ptr, arr(*x.strides), y.ptr,
                                      arr(*y.strides), out.ptr), "mfr_where_nd")
    return out


def elementwise(op: int, a: DeviceArray, b: DeviceArray | None = None, alpha=1.0,
                out: DeviceArray | None = None) -> DeviceArray:
    """out = a + b (abi.EW_ADD), a - b (abi.EW_SUB), a * b (abi.EW_MUL) or alpha * a
    (abi.EW_SCAL, b unused) over contiguous arrays of a's size (mfr_elementwise)."""
    if out is None:
        out = DeviceArray.empty(a.shape, a.stream)
    b_ptr = None if b is None else b.ptr
    abi.check(abi.load().mfr_elementwise(a.stream.handle, op, a.ptr, b_ptr, alpha, out.ptr,
                                         a.size), "mfr_elementwise")
    return out


def softmax(x: DeviceArray, axis=-1, out: DeviceArray | None = None) -> DeviceArray:
    shape = x.shape if x.shape else (1,)
    axis %= len(shape)
    outer = int(np.prod(shape[:axis], dtype=np.int64))
    length = int(shape[axis])
    inner = int(np.prod(shape[axis + 1:], dtype=np.int64))
    if out is None:
        out = DeviceArray.empty(x.shape, x.stream)
    abi.check(abi.load().mfr_softmax(x.stream.handle, x.ptr, out.ptr, outer, length, inner),
              "mfr_softmax")
    return out


def argmax(x: DeviceArray, out: DeviceArray | None = None) -> DeviceArray:
    width = x.shape[-1]
    rows = x.size // width if width else int(np.prod(x.shape[:-1], dtype=np.int64))
    if out is None:
        out = DeviceArray.empty(x.shape[:-1], x.stream, np.int64)
    abi.check(abi.load().mfr_argmax(x.stream.handle, x.ptr, out.ptr, rows, width), "mfr_argmax")
    return out


def strided_copy(x: DeviceArray, out: DeviceArray | None = None) -> DeviceArray:
    if out is None:
        out = DeviceArray.empty(x.shape, x.stream, x.dtype)
    nd = len(x.shape)
    shape = (ctypes.c_int64 * max(nd, 1))(*x.shape)
    strides = (ctypes.c_int64 * max(nd, 1))(*x.strides)
    abi.check(abi.load().mfr_strided_copy(x.stream.handle, x.ptr, out.ptr, x.dtype.itemsize, nd,
                                          shape, strides), "mfr_strided_copy")
    return out


def fill(x: DeviceArray, value) -> None:
    bits = np.array([value], dtype=x.dtype).view(
        {1: np.uint8, 2: np.uint16, 4: np.uint32, 8: np.uint64}[x.dtype.itemsize])[0]
    abi.check(abi.load().mfr_fill(x.stream.handle, x.ptr, x.dtype.itemsize, x.size, int(bits)),
              "mfr_fill")


# ---- 8-bit matrices -------------------------------------------------------------------------------


@dataclass
class F8Matrix:
    """An e4m3 matrix with block scales (mfr_f8_matrix): `values` a uint8 array [rows, cols] whose
    rows are contiguous and 16 bytes aligned, `scales` a float32 array [rows or row blocks,
    column blocks of 128] of any strides, `block_rows` 1 (activations) or 128 (weights)."""
    values: DeviceArray
    scales: DeviceArray
    block_rows: int = 1

    @classmethod
    def empty(cls, rows: int, cols: int, stream: Stream, block_rows: int = 1) -> "F8Matrix":
        """Room for [rows, cols], laid out as mfr_f8gemm reads it best: rows padded to 16 bytes, from
        1024 on to 128 (a block's bytes are a cache line then); scales of rows stored [blocks,
        rows]."""
        if block_rows not in (1, abi.F8_BLOCK):
            raise ValueError(f"F8Matrix: block_rows must be 1 or {abi.F8_BLOCK}, got {block_rows}")
        if rows < 0 or cols < 0:
            raise ValueError(f"F8Matrix: negative dimension in {(rows, cols)}")
        blocks = -(-cols // abi.F8_BLOCK)
        unit = 128 if cols >= 1024 else 16
        values = DeviceArray.empty((rows, -(-cols // unit) * unit), stream, np.uint8)
        if block_rows == 1:
            scales = DeviceArray.empty((blocks, rows), stream).T
        else:
            scales = DeviceArray.empty((-(-rows // block_rows), blocks), stream)
        return cls(values.slice(1, 0, cols), scales, block_rows)

    @property
    def shape(self):
        return self.values.shape

    @property
    def stream(self) -> Stream:
        return self.values.stream


def _f8_desc(m: F8Matrix | None, what: str) -> abi.F8Desc:
    d = abi.F8Desc()
    d.block_rows = 1
    if m is None:
        return d
    rows, cols = m.values.shape
    blocks = (-(-rows // m.block_rows) if m.block_rows > 0 else rows, -(-cols // abi.F8_BLOCK))
    if m.values.dtype.itemsize != 1 or m.scales.dtype != np.float32:
        raise ValueError(f"{what}: values of one byte and float32 scales are needed")
    if m.scales.shape != blocks:
        raise ValueError(f"{what}: scales {m.scales.shape}, {blocks} are needed")
    if cols > 1 and m.values.strides[1] != 1:
        raise ValueError(f"{what}: rows need unit stride")
    d.values = m.values.ptr
    d.rs = m.values.strides[0] if rows > 1 else -(-cols // 16) * 16
    d.scales, (d.scales_rs, d.scales_cs) = m.scales.ptr, m.scales.strides
    d.block_rows = m.block_rows
    return d


def _rows_of(t: DeviceArray | None, shape, what: str) -> tuple:
    """(address, row stride) of a float32 matrix of unit column stride; (None, 0) for None."""
    if t is None:
        return None, 0
    if t.dtype != np.float32 or t.shape != tuple(shape):
        raise ValueError(f"{what}: {t.dtype} {t.shape}, float32 {tuple(shape)} is needed")
    if shape[1] > 1 and t.strides[1] != 1:
        raise ValueError(f"{what}: rows need unit stride")
    # The stride of a single row says nothing.
    return t.ptr, t.strides[0] if shape[0] > 1 else max(t.strides[0], shape[1])


def _arrays_of(what: str, *operands) -> tuple:
    """The arrays of operands that are arrays, F8Matrix or None (not given); refuses those of more
    than one device."""
    arrays = tuple(a for t in operands if t is not None
                   for a in ((t.values, t.scales) if isinstance(t, F8Matrix) else (t,)))
    if len({a.stream.device for a in arrays}) > 1:
        raise ValueError(f"{what}: operands of different devices")
    return arrays


def _same_device(what: str, stream: Stream, desc) -> None:
    if desc.held and desc.held[0].stream.device != stream.device:
        raise ValueError(f"{what}: a stream of another device than the operands'")


def _vector_of(t: DeviceArray | None, length: int, what: str):
    if t is None:
        return None
    if t.dtype != np.float32 or t.shape != (length,) or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous float32 vector of {length} is needed")
    return t.ptr


def quantize_f8(x: DeviceArray, block_rows: int = 1, out: F8Matrix | None = None) -> F8Matrix:
    """x [rows, cols] as e4m3 with a scale per block of block_rows x 128 (mfr_f8_quantize): 1 for
    activations, 128 for weights."""
    rows, cols = x.shape
    ptr, rs = _rows_of(x, (rows, cols), "quantize_f8: x")
    if out is None:
        out = F8Matrix.empty(rows, cols, x.stream, block_rows)
    if out.shape != x.shape or out.block_rows != block_rows:
        raise ValueError(f"quantize_f8: out is {out.shape} with block_rows {out.block_rows}")
    _arrays_of("quantize_f8", x, out)
    d = _f8_desc(out, "quantize_f8: out")
    abi.check(abi.load().mfr_f8_quantize(x.stream.handle, rows, cols, ptr, rs, ctypes.byref(d)),
              "mfr_f8_quantize")
    return out


def rms_norm_desc(x: DeviceArray, weight: DeviceArray | None = None, *,
                  residual: DeviceArray | None = None, eps: float = 1e-6,
                  summed: DeviceArray | None = None, out: DeviceArray | None = None,
                  out_f8: F8Matrix | None = None) -> RmsNormDesc:
    """The descriptor of one rms_norm over the rows of x [rows, cols], to be filled once and run
    many times (rms_norm_run): t = x + residual to `summed`, t / rms(t) * weight to `out` (fp32)
    and `out_f8` (8 bits), whichever are given. The descriptor keeps the arrays that it points to
    (`held`)."""
    rows, cols = x.shape
    d = RmsNormDesc()
    d.held = _arrays_of("rms_norm", x, weight, residual, summed, out, out_f8)
    d.rows, d.cols, d.eps = rows, cols, eps
    d.x, d.x_rs = _rows_of(x, x.shape, "rms_norm: x")
    d.residual, d.residual_rs = _rows_of(residual, x.shape, "rms_norm: residual")
    d.sum, d.sum_rs = _rows_of(summed, x.shape, "rms_norm: summed")
    d.out, d.out_rs = _rows_of(out, x.shape, "rms_norm: out")
    d.weight = _vector_of(weight, cols, "rms_norm: weight")
    if out_f8 is not None and out_f8.shape != x.shape:
        raise ValueError(f"rms_norm: out_f8 is {out_f8.shape}, x {x.shape}")
    d.out_f8 = _f8_desc(out_f8, "rms_norm: out_f8")
    return d


def rms_norm_run(stream: Stream, desc: RmsNormDesc) -> None:
    """mfr_rms_norm on a filled descriptor."""
    _same_device("rms_norm", stream, desc)
    abi.check(abi.load().mfr_rms_norm(stream.handle, ctypes.byref(desc)), "mfr_rms_norm")


def rms_norm(x: DeviceArray, weight: DeviceArray | None = None, *,
             residual: DeviceArray | None = None, eps: float = 1e-6,
             summed: DeviceArray | None = None, out: DeviceArray | None = None) -> DeviceArray:
    """(x + residual) / rms * weight over the last dimension of a matrix, in fp32; x + residual is
    written to `summed` where that is given (it may be x or residual)."""
    if out is None:
        out = DeviceArray.empty(x.shape, x.stream)
    rms_norm_run(x.stream, rms_norm_desc(x, weight, residual=residual, eps=eps, summed=summed,
                                         out=out))
    return out


def rms_norm_f8(x: DeviceArray, weight: DeviceArray | None = None, *,
                residual: DeviceArray | None = None, eps: float = 1e-6,
                summed: DeviceArray | None = None, out: F8Matrix | None = None) -> F8Matrix:
    """rms_norm with its result in 8 bits, a scale per row and 128 columns: what gemm_f8 reads."""
    if out is None:
        out = F8Matrix.empty(*x.shape, x.stream)
    rms_norm_run(x.stream, rms_norm_desc(x, weight, residual=residual, eps=eps, summed=summed,
                                         out_f8=out))
    return out


def f8gemm_desc(a: F8Matrix, b: F8Matrix, *, up: F8Matrix | None = None, act=ACT_NONE,
                c0: DeviceArray | None = None, beta=0.0, bias: DeviceArray | None = None,
                out: DeviceArray | None = None, out_f8: F8Matrix | None = None) -> F8GemmDesc:
    """The descriptor of one product of 8-bit matrices (mfr_f8gemm_desc), to be filled once and run
    many times (f8gemm): a [m, k] with a scale per row, b and up [n, k] with 128 x 128 blocks; the
    result goes to `out` (fp32), `out_f8` (8 bits) or both. The descriptor keeps the arrays that it
    points to (`held`)."""
    (m, k), n = a.shape, b.shape[0]
    for w in (b, up):
        if w is not None and w.shape != (n, k):
            raise ValueError(f"f8gemm: a is {a.shape}, a weight {w.shape}")
    if out_f8 is not None and out_f8.shape != (m, n):
        raise ValueError(f"f8gemm: out_f8 is {out_f8.shape}, {(m, n)} is needed")
    d = F8GemmDesc()
    d.held = _arrays_of("f8gemm", a, b, up, c0, bias, out, out_f8)
    d.m, d.n, d.k = m, n, k
    d.a, d.b, d.up = _f8_desc(a, "f8gemm: a"), _f8_desc(b, "f8gemm: b"), _f8_desc(up, "f8gemm: up")
    d.c, d.c_rs = _rows_of(out, (m, n), "f8gemm: out")
    d.c0, d.c0_rs = _rows_of(c0, (m, n), "f8gemm: c0")
    d.bias = _vector_of(bias, n, "f8gemm: bias")
    d.out_f8 = _f8_desc(out_f8, "f8gemm: out_f8")
    d.beta, d.act = beta, act
    return d


def f8gemm(stream: Stream, desc: F8GemmDesc) -> None:
    """mfr_f8gemm on a filled descriptor."""
    _same_device("f8gemm", stream, desc)
    abi.check(abi.load().mfr_f8gemm(stream.handle, ctypes.byref(desc)), "mfr_f8gemm")


def f8gemm_plan(stream: Stream, desc: F8GemmDesc) -> tuple[int, int, int, int]:
    """(form, splits, regions, workspace) that f8gemm(stream, desc) would run with
    (mfr_f8gemm_plan): abi.F8_* and the ranges of the depth (1: whole) of the main part, the parts of
    the outputs that run by themselves, and the bytes of the stream's workspace that it takes."""
    _same_device("f8gemm_plan", stream, desc)
    form, splits, regions = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
    workspace = ctypes.c_size_t()
    abi.check(abi.load().mfr_f8gemm_plan(stream.device, ctypes.byref(desc), ctypes.byref(form),
                                         ctypes.byref(splits), ctypes.byref(regions),
                                         ctypes.byref(workspace)), "mfr_f8gemm_plan")
    return form.value, splits.value, regions.value, workspace.value


def gemm_f8(a: F8Matrix, b: F8Matrix, *, c0: DeviceArray | None = None, beta=0.0,
            bias: DeviceArray | None = None, act=ACT_NONE, out: DeviceArray | None = None,
            out_f8: F8Matrix | None = None):
    """act(a b^T + beta c0 + bias) of 8-bit matrices, b [n, k] as weights are stored: a new fp32
    array, or `out` and / or `out_f8` where they are given. Returns out_f8 where only that is."""
    if out is None and out_f8 is None:
        out = DeviceArray.empty((a.shape[0], b.shape[0]), a.stream)
    f8gemm(a.stream, f8gemm_desc(a, b, act=act, c0=c0, beta=beta, bias=bias, out=out,
                                 out_f8=out_f8))
    return out if out is not None else out_f8


def gemm_f8_gated(a: F8Matrix, gate: F8Matrix, up: F8Matrix, *, act=ACT_SILU,
                  out: DeviceArray | None = None, out_f8: F8Matrix | None = None):
    """act(a gate^T) * (a up^T), both projections in one kernel: in 8 bits for the next product (a
    new F8Matrix), or to `out` (fp32) and / or `out_f8` where they are given. Returns out_f8 where
    that is given or made, else out. A call of at most 64 rows that is captured into a
    graph is faster with both: the sums then need no workspace, which a captured call does not
    take."""
    if out is None and out_f8 is None:
        out_f8 = F8Matrix.empty(a.shape[0], gate.shape[0], a.stream)
    f8gemm(a.stream, f8gemm_desc(a, gate, up=up, act=act, out=out, out_f8=out_f8))
    return out_f8 if out_f8 is not None else out


def attention_fused(q: DeviceArray, k: DeviceArray, v: DeviceArray,
                    mask: DeviceArray | None = None, causal: bool = False, scale: float = 0.0,
                    out: DeviceArray | None = None) -> DeviceArray:
    """mfr_attention: the whole op in one kernel (online softmax, no score matrix). q [..., Lq, D],
    k and v [..., Lk, D] with equal batch shapes (stride 0 for broadcast), D a multiple of 16 up to
    128;
    mask a uint8 array broadcastable to [..., Lq, Lk]. Raises NotImplementedError for layouts
    the kernel does not take."""
    lq, depth = q.shape[-2:]
    lk = k.shape[-2]
    batch = q.shape[:-2]
    dims = len(batch)
    if dims > abi.MAX_BATCH_DIMS:
        raise ValueError("too many batch dimensions")
    if k.shape != batch + (lk, depth) or v.shape != batch + (lk, depth):
        raise ValueError(f"attention: q {q.shape}, k {k.shape}, v {v.shape} do not agree")
    for t in (q, k, v):
        if t.strides[-1] != 1:
            raise NotImplementedError("attention: fused kernel needs unit stride along d")
    if out is None:
        out = DeviceArray.empty(batch + (lq, depth), q.stream)
    d = abi.AttentionDesc()
    d.lq, d.lk, d.d = lq, lk, depth
    d.batch_dims = dims
    d.causal = 1 if causal else 0
    _fill_batch(d.batch, batch, dims)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        setattr(d, name, t.ptr)
        setattr(d, name + "_rs", t.strides[-2])
        _fill_batch(getattr(d, name + "_bs"), t.strides[:-2], dims)
    if mask is not None:
        full = mask.expand(batch + (lq, lk))
        d.mask = full.ptr
        d.mask_rs, d.mask_cs = full.strides[-2], full.strides[-1]
        _fill_batch(d.mask_bs, full.strides[:-2], dims)
    d.scale = scale
    abi.check(abi.load().mfr_attention(q.stream.handle, ctypes.byref(d)), "mfr_attention")
    return out


def attention(q: DeviceArray, k: DeviceArray, v: DeviceArray, mask: DeviceArray | None = None,
              causal: bool = False, scale: float = 0.0, fused: bool | None = None) -> DeviceArray:
    """mensurflow::attention (src/ops/attention.cpp:48-98). fused=None runs the fused kernel
    (attention_fused) when it takes the layout and the composition otherwise; True only the
    fused kernel; False only the composition."""
    if fused is not False:
        try:
            return attention_fused(q, k, v, mask=mask, causal=causal, scale=scale)
        except NotImplementedError:
            if fused:
                raise
    return attention_composed(q, k, v, mask=mask, causal=causal, scale=scale)


def attention_composed(q: DeviceArray, k: DeviceArray, v: DeviceArray,
                       mask: DeviceArray | None = None, causal: bool = False,
                       scale: float = 0.0) -> DeviceArray:
    """mensurflow::attention's composition on the device (src/ops/attention.cpp:48-98): scores =
    gemm_batched(q, k^T, alpha=scale), where(mask, scores, -inf) with the mask and the -inf
    scalar read through broadcast views (mfr_where_nd; mensurflow::where packs them to the
    scores' shape), the causal mask the same way, softmax over the keys, gemm_batched(weights,
    v). The causal mask is the scores GEMM's own (causal=True: the same bits as the where over
    the lower triangle, without the pass over the scores) where the GEMM takes it, the where
    otherwise. q [..., Lq, D], k [..., Lk, D], v [..., Lk, Dv] with equal batch shapes; mask a
    Bool (uint8) array broadcastable to [..., Lq, Lk]. Every array is on q's stream; the scores
    are that stream's scratch array, reused by later calls."""
    stream = q.stream
    lq, depth = q.shape[-2:]
    lk = k.shape[-2]
    batch = q.shape[:-2]
    if scale == 0.0:
        scale = float(np.float32(1.0 / np.sqrt(depth))) if depth > 0 else 1.0
    scores = stream.scratch("attention.scores", batch + (lq, lk))
    causal_done = False
    if causal:
        try:
            gemm_batched(q, k.transpose(-2, -1), scores, alpha=scale, causal=True)
            causal_done = True
        except NotImplementedError:
            pass
    if not causal_done:
        gemm_batched(q, k.transpose(-2, -1), scores, alpha=scale)
    minus_inf = None

    def masked(keep: DeviceArray) -> DeviceArray:
        nonlocal minus_inf
        if minus_inf is None:
            minus_inf = stream.scratch("attention.scalar", (1,))
            fill(minus_inf, -np.inf)
        return where_nd(keep.expand(scores.shape), scores, minus_inf.expand(scores.shape),
                        out=scores)

    if mask is not None:
        masked(mask)
    if causal and not causal_done:
        # The [Lq, Lk] lower triangle, kept on the stream until a call needs another shape.
        lower = stream._scratch.get("attention.causal")
        if lower is None or lower.shape != (lq, lk):
            if lower is not None:
                lower.close()
            lower = DeviceArray.from_numpy(np.tril(np.ones((lq, lk), dtype=np.uint8)), stream)
            stream._scratch["attention.causal"] = lower
        masked(lower)
    weights = softmax(scores, axis=-1, out=scores)
    out = DeviceArray.empty(batch + (lq, v.shape[-1]), stream)
    gemm_batched(weights, v, out)
    return out
