"""CudaBackend: the reference's device-plugin interface, implemented on B200.

The reference routes every non-CPU tensor operation to the abstract
``MetalBackend`` (include/vectorcore/metal_backend.hpp:13-56). ``CudaBackend``
offers the same methods with the same argument meaning -- element counts,
shapes, strides, ``[outer, length, inner]`` axis splits -- and returns
``CudaStorage`` objects (the counterpart of ``Storage``,
include/vectorcore/storage.hpp:11-27), plus the fused entry points the CUDA
device adds (backward rules, sum_to_shape, softmax family, cross-entropy).
All calls go through the C ABI (include/vc_cuda.h); failures raise the
reference's exception types and nothing falls back to the CPU.
"""
from __future__ import annotations

import ctypes
import threading

import numpy as np

from . import _abi
from ._abi import ADD, DIV, MUL, SUB  # noqa: F401  (re-exported op codes)
from ._abi import EXP, LOG, NEG, RELU, RELU_GRAD, SIGMOID  # noqa: F401
from ._abi import REDUCE_ARGMAX, REDUCE_MAX, REDUCE_MEAN, REDUCE_SUM  # noqa: F401

_F32 = 4
_FLOAT32, _INT64, _INT8 = np.dtype(np.float32), np.dtype(np.int64), np.dtype(np.int8)


class CudaStorage:
    """Device buffer from the stream-ordered pool plus the in-place
    modification counter shared by every view (storage.hpp:22-23).

    ``dtype`` is float32 except for the int64 index / target buffers the
    fused kernels use and the int8 values of 8-bit matrices."""

    __slots__ = ("ptr", "size", "dtype", "version", "__weakref__")

    def __init__(self, elements: int, dtype=np.float32):
        self.dtype = np.dtype(dtype)
        self.size = int(elements)
        self.version = 0
        self.ptr = _abi.alloc(max(self.size, 1) * self.dtype.itemsize)

    @classmethod
    def borrow(cls, ptr: int, elements: int, dtype=_FLOAT32) -> "CudaStorage":
        """A storage over device memory that somebody else owns (another
        library's tensor, part of a larger buffer): nothing is allocated, and
        nothing is freed when it goes. The owner keeps the memory until the
        work enqueued on it is done."""
        s = _Borrowed.__new__(_Borrowed)
        s.ptr, s.size, s.dtype, s.version = ptr, elements, np.dtype(dtype), 0
        return s

    @property
    def nbytes(self) -> int:
        return self.size * self.dtype.itemsize

    def bump_version(self) -> None:
        self.version += 1

    def __del__(self):
        ptr, self.ptr = getattr(self, "ptr", 0), 0
        if ptr:
            try:
                _abi.lib.vc_cuda_free(ctypes.c_void_p(ptr))
            except Exception:  # interpreter shutdown
                pass

    def device(self) -> str:
        return "cuda"


class _Borrowed(CudaStorage):
    __slots__ = ()

    def __del__(self):
        pass


def _p(x):
    """Raw device address of a storage (or None)."""
    return None if x is None else ctypes.c_void_p(x.ptr)


def _at(x, elements, dtype, what):
    """Raw device address of a storage that has to hold `elements` of `dtype`
    (None stays None)."""
    if x is None:
        return None
    if x.dtype is not dtype and x.dtype != dtype:
        raise ValueError(f"{what} is {x.dtype}, not {dtype}")
    if x.size < elements:
        raise IndexError(f"{what} has {x.size} elements, {elements} are needed")
    return x.ptr


def _span(rows, cols, stride):
    """Elements from the first of `rows` rows to the end of the last."""
    if rows < 0 or cols < 0 or stride < 0:
        raise ValueError("sizes and strides are not negative")
    return (rows - 1) * stride + cols if rows else 0


def q8_pitch(cols: int) -> int:
    """Bytes between the rows of an 8-bit matrix with `cols` columns: rows
    start on 16-byte boundaries."""
    return (cols + 15) // 16 * 16


class PinnedBuffer:
    """Page-locked host memory (vc_cuda_host_alloc) viewed as a numpy array:
    the host side of the asynchronous transfers."""

    def __init__(self, elements: int, dtype=np.float32):
        self.dtype = np.dtype(dtype)
        self.size = int(elements)
        ptr = ctypes.c_void_p()
        _abi.call("vc_cuda_host_alloc", ctypes.c_size_t(max(self.size, 1) * self.dtype.itemsize), ctypes.byref(ptr))
        self.ptr = ptr.value
        buf = (ctypes.c_char * (self.size * self.dtype.itemsize)).from_address(self.ptr)
        self.array = np.frombuffer(buf, dtype=self.dtype, count=self.size)

    @property
    def nbytes(self) -> int:
        return self.size * self.dtype.itemsize

    def close(self) -> None:
        ptr, self.ptr = getattr(self, "ptr", 0), 0
        if ptr:
            self.array = None
            _abi.lib.vc_cuda_host_free(ctypes.c_void_p(ptr))

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown
            pass


class CudaGraph:
    """A replayable capture of the library stream's work (vc_cuda_graph_*).
    The pool blocks allocated while capturing stay reserved for the graph
    until close(); storages returned by the captured calls are rewritten by
    every replay."""

    def __init__(self, handle: int):
        self._h = ctypes.c_void_p(handle)

    def launch(self) -> None:
        if not self._h.value:
            raise RuntimeError("CudaGraph: launch after close()")
        _abi.call("vc_cuda_graph_launch", self._h)

    @property
    def nodes(self) -> int:
        n = ctypes.c_size_t(0)
        _abi.call("vc_cuda_graph_nodes", self._h, ctypes.byref(n))
        return int(n.value)

    def close(self) -> None:
        if self._h.value:
            _abi.call("vc_cuda_graph_destroy", self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class CudaBackend:
    _instance = None
    _lock = threading.Lock()

    @classmethod
    def instance(cls) -> "CudaBackend":
        with cls._lock:
            if cls._instance is None:
                cls._instance = cls()
            return cls._instance

    # ---- device ---------------------------------------------------------------
    def available(self) -> bool:
        return _abi.available()

    def device_name(self) -> str:
        return _abi.device_name() if self.available() else "unavailable"

    def last_error(self) -> str:
        return _abi.last_error()

    def synchronize(self) -> None:
        _abi.synchronize()

    def use_stream(self, handle: int | None) -> None:
        """Enqueue on the stream with this raw handle from now on (another
        library's, e.g. torch.cuda.Stream.cuda_stream; 0 is the default
        stream). None goes back to the device's own stream. Call it again
        whenever the owner works on another stream: what is enqueued on two
        streams is not ordered, except by this call, which waits for the
        stream it leaves."""
        # NULL restores the own stream in the C ABI; 1 is cudaStreamLegacy
        _abi.call("vc_cuda_set_stream", ctypes.c_void_p(None if handle is None else handle or 1))

    def capture(self, fn):
        """Run fn() under stream capture; returns (CudaGraph, fn's result).
        The captured work is NOT executed by the capture itself: launch the
        graph to run it."""
        _abi.call("vc_cuda_graph_begin")
        try:
            result = fn()
        except BaseException:
            h = ctypes.c_void_p(0)
            try:
                _abi.call("vc_cuda_graph_end", ctypes.byref(h))
            finally:
                if h.value:
                    _abi.call("vc_cuda_graph_destroy", h)
            raise
        h = ctypes.c_void_p(0)
        _abi.call("vc_cuda_graph_end", ctypes.byref(h))
        return CudaGraph(h.value), result

    # ---- memory ---------------------------------------------------------------
    def allocate(self, elements: int, dtype=np.float32) -> CudaStorage:
        return CudaStorage(elements, dtype)

    def upload(self, values: np.ndarray, dtype=None) -> CudaStorage:
        """Copy to the device as float32, or int64 where the values are that;
        `dtype` keeps another type (np.int8: the values of an 8-bit matrix)."""
        values = np.ascontiguousarray(values, dtype)
        if dtype is None and values.dtype not in (np.float32, np.int64):
            values = values.astype(np.float32)
        s = CudaStorage(values.size, values.dtype)
        _abi.call("vc_cuda_upload", ctypes.c_void_p(s.ptr), values.ctypes.data_as(ctypes.c_void_p),
                  ctypes.c_size_t(values.nbytes))
        return s

    def download(self, source: CudaStorage, elements: int | None = None) -> np.ndarray:
        n = source.size if elements is None else int(elements)
        if n > source.size:
            raise IndexError("download exceeds storage")
        out = np.empty(n, source.dtype)
        _abi.call("vc_cuda_download", out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(source.ptr),
                  ctypes.c_size_t(out.nbytes))
        return out

    # ---- asynchronous transfers (vc_cuda_upload_async & co.) --------------------
    def upload_async(self, dst: CudaStorage, src: PinnedBuffer, nbytes: int | None = None) -> int:
        """Copy a pinned host buffer into dst on the upload copy stream; later
        work waits for it only after transfer_wait(ticket)."""
        nb = src.nbytes if nbytes is None else int(nbytes)
        if nb > dst.nbytes or nb > src.nbytes:
            raise IndexError("upload_async exceeds a buffer")
        t = ctypes.c_uint64(0)
        _abi.call("vc_cuda_upload_async", ctypes.c_void_p(dst.ptr), ctypes.c_void_p(src.ptr), ctypes.c_size_t(nb),
                  ctypes.byref(t))
        return int(t.value)

    def download_async(self, dst: PinnedBuffer, src: CudaStorage, nbytes: int | None = None) -> int:
        """Copy src into a pinned host buffer on the download copy stream,
        after the work enqueued so far; read dst after transfer_sync(ticket)."""
        nb = src.nbytes if nbytes is None else int(nbytes)
        if nb > dst.nbytes or nb > src.nbytes:
            raise IndexError("download_async exceeds a buffer")
        t = ctypes.c_uint64(0)
        _abi.call("vc_cuda_download_async", ctypes.c_void_p(dst.ptr), ctypes.c_void_p(src.ptr),
                  ctypes.c_size_t(nb), ctypes.byref(t))
        return int(t.value)

    def transfer_wait(self, ticket: int) -> None:
        _abi.call("vc_cuda_transfer_wait", ctypes.c_uint64(ticket))

    def transfer_sync(self, ticket: int) -> None:
        _abi.call("vc_cuda_transfer_sync", ctypes.c_uint64(ticket))

    # ---- MetalBackend methods ---------------------------------------------------
    def binary(self, a, a_shape, a_strides, b, b_shape, b_strides, out_shape, op) -> CudaStorage:
        out = CudaStorage(int(np.prod(out_shape, dtype=np.int64)))
        sa, ra = _abi.shape_arg(a_shape)
        sb, rb = _abi.shape_arg(b_shape)
        so, ro = _abi.shape_arg(out_shape)
        ta = _abi.shape_arg(a_strides)[0] if a_strides is not None else None
        tb = _abi.shape_arg(b_strides)[0] if b_strides is not None else None
        _abi.call("vc_cuda_binary", op, _p(a), sa, ta, ra, _p(b), sb, tb, rb, _p(out), so, ro)
        return out

    def binary_scalar(self, a, count, scalar, op, scalar_first=False) -> CudaStorage:
        out = CudaStorage(count)
        _abi.call("vc_cuda_binary_scalar", op, _p(a), ctypes.c_float(scalar), int(scalar_first), _p(out),
                  ctypes.c_size_t(count))
        return out

    def unary(self, inp, count, op) -> CudaStorage:
        out = CudaStorage(count)
        _abi.call("vc_cuda_unary", op, _p(inp), _p(out), ctypes.c_size_t(count))
        return out

    def reduce_sum(self, inp, count) -> CudaStorage:
        out = CudaStorage(1)
        _abi.call("vc_cuda_reduce_all", REDUCE_SUM, _p(inp), ctypes.c_size_t(count), _p(out), None)
        return out

    def reduce_all(self, inp, count, op, want_index=False):
        out = CudaStorage(1)
        idx = CudaStorage(1, np.int64) if want_index else None
        _abi.call("vc_cuda_reduce_all", op, _p(inp), ctypes.c_size_t(count), _p(out), _p(idx))
        return (out, idx) if want_index else out

    def reduce_axis(self, inp, outer, length, inner, op, want_index=False):
        """SUM / MEAN / MAX values, or ARGMAX as float indices (the
        reference's convention); want_index also returns int64 indices."""
        out = CudaStorage(outer * inner)
        idx = CudaStorage(outer * inner, np.int64) if want_index else None
        _abi.call("vc_cuda_reduce_axis", op, _p(inp), ctypes.c_size_t(outer), ctypes.c_size_t(length),
                  ctypes.c_size_t(inner), _p(out), _p(idx))
        return (out, idx) if want_index else out

    def scatter_axis(self, values, indices, outer, length, inner) -> CudaStorage:
        out = CudaStorage(outer * length * inner)
        f32 = indices if indices.dtype == np.float32 else None
        i64 = indices if indices.dtype == np.int64 else None
        _abi.call("vc_cuda_scatter_axis", _p(values), _p(f32), _p(i64), _p(out), ctypes.c_size_t(outer),
                  ctypes.c_size_t(length), ctypes.c_size_t(inner))
        return out

    def axpy_inplace(self, target, source, count, alpha) -> None:
        _abi.call("vc_cuda_axpy", _p(target), _p(source), ctypes.c_size_t(count), ctypes.c_float(alpha))

    def matmul(self, a, b, m, k, n, a_offsets, b_offsets, trans_a=False, trans_b=False) -> CudaStorage:
        if len(a_offsets) != len(b_offsets) or not a_offsets:
            raise ValueError("matmul needs one A and B offset per batch")
        batch = len(a_offsets)
        out = CudaStorage(batch * m * n)
        ao = (ctypes.c_size_t * batch)(*[int(v) for v in a_offsets])
        bo = (ctypes.c_size_t * batch)(*[int(v) for v in b_offsets])
        _abi.call("vc_cuda_matmul", _p(a), _p(b), _p(out), ctypes.c_size_t(m), ctypes.c_size_t(k),
                  ctypes.c_size_t(n), ao, bo, ctypes.c_size_t(batch), int(trans_a), int(trans_b))
        return out

    def transpose_last2(self, inp, batch, rows, cols) -> CudaStorage:
        out = CudaStorage(batch * rows * cols)
        _abi.call("vc_cuda_transpose_last2", _p(inp), _p(out), ctypes.c_size_t(batch), ctypes.c_size_t(rows),
                  ctypes.c_size_t(cols))
        return out

    # ---- fused entry points of the CUDA device ---------------------------------------
    def fill(self, count, value) -> CudaStorage:
        out = CudaStorage(count)
        _abi.call("vc_cuda_fill", _p(out), ctypes.c_size_t(count), ctypes.c_float(value))
        return out

    def copy(self, src: CudaStorage) -> CudaStorage:
        out = CudaStorage(src.size, src.dtype)
        _abi.call("vc_cuda_copy", _p(out), _p(src), ctypes.c_size_t(src.nbytes))
        return out

    def unary_backward(self, op, x, y, g, count) -> CudaStorage:
        out = CudaStorage(count)
        _abi.call("vc_cuda_unary_backward", op, _p(x), _p(y), _p(g), _p(out), ctypes.c_size_t(count))
        return out

    def broadcast_to(self, value, v_shape, t_shape) -> CudaStorage:
        out = CudaStorage(int(np.prod(t_shape, dtype=np.int64)))
        sv, rv = _abi.shape_arg(v_shape)
        st, rt = _abi.shape_arg(t_shape)
        _abi.call("vc_cuda_broadcast_to", _p(value), sv, rv, _p(out), st, rt)
        return out

    def sum_to_shape(self, g, g_shape, t_shape) -> CudaStorage:
        out = CudaStorage(int(np.prod(t_shape, dtype=np.int64)))
        sg, rg = _abi.shape_arg(g_shape)
        st, rt = _abi.shape_arg(t_shape)
        _abi.call("vc_cuda_sum_to_shape", _p(g), sg, rg, _p(out), st, rt)
        return out

    def binary_backward(self, op, a, a_shape, b, b_shape, g, g_shape, need_a=True, need_b=True):
        da = CudaStorage(int(np.prod(a_shape, dtype=np.int64))) if need_a else None
        db = CudaStorage(int(np.prod(b_shape, dtype=np.int64))) if need_b else None
        sa, ra = _abi.shape_arg(a_shape)
        sb, rb = _abi.shape_arg(b_shape)
        sg, rg = _abi.shape_arg(g_shape)
        _abi.call("vc_cuda_binary_backward", op, _p(a), sa, ra, _p(b), sb, rb, _p(g), sg, rg, _p(da), _p(db))
        return da, db

    def reduce_axis_backward(self, op, g, indices, outer, length, inner) -> CudaStorage:
        out = CudaStorage(outer * length * inner)
        _abi.call("vc_cuda_reduce_axis_backward", op, _p(g), _p(indices), _p(out), ctypes.c_size_t(outer),
                  ctypes.c_size_t(length), ctypes.c_size_t(inner))
        return out

    def softmax(self, x, outer, length, inner, log=False, stats=True):
        y = CudaStorage(outer * length * inner)
        m = CudaStorage(outer * inner) if stats else None
        s = CudaStorage(outer * inner) if stats else None
        _abi.call("vc_cuda_log_softmax" if log else "vc_cuda_softmax", _p(x), _p(y), _p(m), _p(s),
                  ctypes.c_size_t(outer), ctypes.c_size_t(length), ctypes.c_size_t(inner))
        return y, m, s

    def softmax_backward(self, x, m, s, g, outer, length, inner, log=False) -> CudaStorage:
        dx = CudaStorage(outer * length * inner)
        _abi.call("vc_cuda_log_softmax_backward" if log else "vc_cuda_softmax_backward", _p(x), _p(m), _p(s),
                  _p(g), _p(dx), ctypes.c_size_t(outer), ctypes.c_size_t(length), ctypes.c_size_t(inner))
        return dx

    def cross_entropy(self, logits, targets, batch, classes, batch_total=0):
        loss = CudaStorage(1)
        m = CudaStorage(batch)
        s = CudaStorage(batch)
        part = CudaStorage(1, np.float64)
        _abi.call("vc_cuda_cross_entropy", _p(logits), _p(targets), ctypes.c_size_t(batch),
                  ctypes.c_size_t(classes), ctypes.c_size_t(batch_total), _p(loss), _p(m), _p(s), _p(part))
        return loss, m, s, part

    def cross_entropy_backward(self, logits, targets, m, s, upstream, batch, classes, batch_total=0):
        dx = CudaStorage(batch * classes)
        _abi.call("vc_cuda_cross_entropy_backward", _p(logits), _p(targets), _p(m), _p(s), _p(upstream),
                  ctypes.c_size_t(batch), ctypes.c_size_t(classes), ctypes.c_size_t(batch_total), _p(dx))
        return dx

    # ---- fused chain relu(x + b).sum() (one launch each way) ----------------
    def bias_relu_sum(self, x, b, rows, cols):
        """loss storage (1 element) = relu(x + b).sum() for x [rows, cols], b [cols]."""
        loss = CudaStorage(1)
        _abi.call("vc_cuda_bias_relu_sum", _p(x), _p(b), ctypes.c_size_t(rows), ctypes.c_size_t(cols), _p(loss),
                  None)
        return loss

    def bias_relu_sum_backward(self, x, b, upstream, rows, cols):
        """(dx, db) of relu(x + b).sum() given the upstream scalar gradient."""
        dx = CudaStorage(rows * cols)
        db = CudaStorage(cols)
        _abi.call("vc_cuda_bias_relu_sum_backward", _p(x), _p(b), _p(upstream), ctypes.c_size_t(rows),
                  ctypes.c_size_t(cols), _p(dx), _p(db), None)
        return dx, db

    # ---- language-model operators: norm, 8-bit product, sampling --------------
    # `out` takes the storages to write (a loop that must not allocate);
    # without it they come from the pool like every other result.
    def rms_norm(self, x, weight, rows, cols, eps=1e-6, residual=None, x_stride=None, residual_stride=None,
                 out=None):
        """(y, h, rstd) of h = x + residual, rstd = 1 / sqrt(mean(h^2) + eps),
        y = h * rstd * weight, row by row. Without a residual h is x, and the
        h returned is None unless `out` has a storage for it."""
        xs = cols if x_stride is None else x_stride
        rs = cols if residual_stride is None else residual_stride
        n = _span(rows, cols, cols)
        if out is None:
            out = (CudaStorage(n), CudaStorage(n) if residual is not None else None, CudaStorage(rows))
        y, h, rstd = out
        _abi.call("vc_cuda_rms_norm", _at(x, _span(rows, cols, xs), _FLOAT32, "x"), xs,
                  _at(residual, _span(rows, cols, rs), _FLOAT32, "residual"), rs, _at(weight, cols, _FLOAT32, "weight"),
                  rows, cols, eps, _at(h, n, _FLOAT32, "h"), _at(y, n, _FLOAT32, "y"),
                  _at(rstd, rows, _FLOAT32, "rstd"))
        return out

    def rms_norm_backward(self, h, weight, rstd, gy, rows, cols, gh=None, need_w=True, out=None):
        """(dh, dw) for the upstream gradients gy of y and gh of h (None:
        zero); dh is the gradient of x and of the residual alike."""
        n = _span(rows, cols, cols)
        if out is None:
            out = (CudaStorage(n), CudaStorage(cols) if need_w else None)
        dh, dw = out
        _abi.call("vc_cuda_rms_norm_backward", _at(h, n, _FLOAT32, "h"), _at(weight, cols, _FLOAT32, "weight"),
                  _at(rstd, rows, _FLOAT32, "rstd"), _at(gy, n, _FLOAT32, "gy"), _at(gh, n, _FLOAT32, "gh"), rows, cols,
                  _at(dh, n, _FLOAT32, "dh"), _at(dw, cols, _FLOAT32, "dw"))
        return out

    def rms_norm_q8(self, x, weight, rows, cols, eps=1e-6, residual=None, x_stride=None, residual_stride=None,
                    out=None):
        """(q, scale, h): rms_norm with y as an 8-bit matrix, its rows
        q8_pitch(cols) bytes apart."""
        xs = cols if x_stride is None else x_stride
        rs = cols if residual_stride is None else residual_stride
        n, pitch = _span(rows, cols, cols), q8_pitch(cols)
        if out is None:
            out = (CudaStorage(rows * pitch, _INT8), CudaStorage(rows), CudaStorage(n) if residual is not None else None)
        q, scale, h = out
        _abi.call("vc_cuda_rms_norm_q8", _at(x, _span(rows, cols, xs), _FLOAT32, "x"), xs,
                  _at(residual, _span(rows, cols, rs), _FLOAT32, "residual"), rs, _at(weight, cols, _FLOAT32, "weight"),
                  rows, cols, eps, _at(h, n, _FLOAT32, "h"), _at(q, rows * pitch, _INT8, "q"), pitch,
                  _at(scale, rows, _FLOAT32, "scale"))
        return out

    def quantize_q8(self, x, rows, cols, x_stride=None, out=None):
        """(q, scale): the rows of x as an 8-bit matrix, rows q8_pitch(cols)
        bytes apart."""
        xs, pitch = cols if x_stride is None else x_stride, q8_pitch(cols)
        need = _span(rows, cols, xs)
        if out is None:
            out = (CudaStorage(rows * pitch, _INT8), CudaStorage(rows))
        q, scale = out
        _abi.call("vc_cuda_quantize_q8", _at(x, need, _FLOAT32, "x"), xs, rows, cols, _at(q, rows * pitch, _INT8, "q"),
                  pitch, _at(scale, rows, _FLOAT32, "scale"))
        return out

    def matmul_q8(self, a, a_scale, b, b_scale, m, n, k, bias=None, a_pitch=None, b_pitch=None, out=None):
        """out [m, n] = (a b^T) * a_scale * b_scale (+ bias) for 8-bit matrices
        a [m, k] and b [n, k], rows q8_pitch(k) bytes apart by default."""
        ap = q8_pitch(k) if a_pitch is None else a_pitch
        bp = q8_pitch(k) if b_pitch is None else b_pitch
        na, nb = _span(m, k, ap), _span(n, k, bp)
        if out is None:
            out = CudaStorage(m * n)
        _abi.call("vc_cuda_matmul_q8", _at(a, na, _INT8, "a"), ap, _at(a_scale, m, _FLOAT32, "a_scale"),
                  _at(b, nb, _INT8, "b"), bp, _at(b_scale, n, _FLOAT32, "b_scale"), _at(bias, n, _FLOAT32, "bias"), m, n, k,
                  _at(out, m * n, _FLOAT32, "out"))
        return out

    def sample(self, logits, noise, rows, vocab, temperature=None, top_k=None, top_p=None, min_p=None,
               row_stride=None, noise_stride=None, out=None):
        """(token int64, logprob) of each row of logits [rows, vocab]; noise
        holds standard-exponential random numbers, the settings a value for
        each row (top_k int64) or None for off."""
        ls = vocab if row_stride is None else row_stride
        ns = vocab if noise_stride is None else noise_stride
        nl, nn = _span(rows, vocab, ls), _span(rows, vocab, ns)
        if out is None:
            out = (CudaStorage(rows, _INT64), CudaStorage(rows))
        token, logprob = out
        _abi.call("vc_cuda_sample", _at(logits, nl, _FLOAT32, "logits"), ls, _at(noise, nn, _FLOAT32, "noise"), ns,
                  _at(temperature, rows, _FLOAT32, "temperature"), _at(top_k, rows, _INT64, "top_k"),
                  _at(top_p, rows, _FLOAT32, "top_p"), _at(min_p, rows, _FLOAT32, "min_p"), rows, vocab,
                  _at(token, rows, _INT64, "token"), _at(logprob, rows, _FLOAT32, "logprob"))
        return out
