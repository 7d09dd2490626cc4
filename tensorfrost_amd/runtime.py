"""Python face of the device runtime: buffers of 32-bit words, JIT kernels, events, primitives.

Everything here is a thin, typed view of the C ABI in include/tfhip.h; it holds no compute of its
own. Buffers follow the reference's memory model: flat arrays of 32-bit words whose element kind
(float32 / int32 / uint32 / bool-as-word) is only a reinterpretation
(TensorFrost/Backend/CodeGen/Generators.cpp:406-426; upload coercions as
TensorFrost/Frontend/Python/PyTensorMemory.cpp:21-63: f64->f32, i64->i32, u64->u32, bool->u32).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import TFHipError, call

REDUCE_SUM, REDUCE_MAX, REDUCE_MIN = 0, 1, 2
_REDUCE_OPS = {"sum": REDUCE_SUM, "max": REDUCE_MAX, "min": REDUCE_MIN}

_initialized = False


def initialize(device: int = 0) -> None:
    """Binds the library to one GPU (idempotent)."""
    global _initialized
    call("tfhip_init", device)
    _initialized = True


def shutdown() -> None:
    global _initialized
    call("tfhip_shutdown")
    _initialized = False


def device_info() -> dict:
    name = C.create_string_buffer(256)
    cus, mem = C.c_int(0), C.c_size_t(0)
    call("tfhip_device_info", name, 256, C.byref(cus), C.byref(mem))
    return {"name": name.value.decode(), "compute_units": cus.value, "hbm_bytes": mem.value}


def synchronize() -> None:
    call("tfhip_sync")


def _coerce(arr: np.ndarray) -> np.ndarray:
    """Host array -> contiguous array of a 32-bit element kind, as the reference's upload does."""
    arr = np.asarray(arr)
    k = arr.dtype.kind
    if k == "f":
        arr = arr.astype(np.float32, copy=False)
    elif k == "i":
        arr = arr.astype(np.int32, copy=False)
    elif k == "u":
        arr = arr.astype(np.uint32, copy=False)
    elif k == "b":
        arr = arr.astype(np.uint32)
    else:
        raise TypeError(f"unsupported dtype {arr.dtype}")
    return np.ascontiguousarray(arr)


class DeviceView:
    """`n_words` 32-bit words of device memory that something else owns (DeviceBuffer.view)."""

    def __init__(self, ptr: int, n_words: int):
        self.ptr = ptr
        self.n_words = n_words

    def write(self, arr, offset_words: int = 0) -> None:
        arr = _coerce(arr)
        if offset_words + arr.size > self.n_words:
            raise ValueError("write past the end of the buffer")
        call("tfhip_h2d", self.ptr, offset_words, arr.ctypes.data, arr.size)

    def numpy(self, dtype=np.float32, shape=None, offset_words: int = 0) -> np.ndarray:
        dtype = np.dtype(dtype)
        if dtype.itemsize != 4:
            raise TypeError("buffers hold 32-bit words")
        count = self.n_words - offset_words if shape is None else int(np.prod(shape))
        if offset_words + count > self.n_words:
            raise ValueError("read past the end of the buffer")
        out = np.empty(count, dtype=dtype)
        call("tfhip_d2h", out.ctypes.data, self.ptr, offset_words, count)
        return out if shape is None else out.reshape(shape)

    def fill(self, word: int) -> None:
        call("tfhip_fill_u32", self.ptr, word & 0xFFFFFFFF, self.n_words)

    def free(self) -> None:
        """Lets go of the address; the memory stays its owner's."""
        self.ptr = None


class DeviceBuffer(DeviceView):
    """An owned device allocation of `n_words` 32-bit words."""

    def __init__(self, n_words: int):
        if n_words <= 0:
            raise ValueError("Trying to allocate a tensor with size 0")
        ptr = C.c_void_p()
        call("tfhip_malloc", C.byref(ptr), n_words)
        super().__init__(ptr.value, int(n_words))

    @classmethod
    def from_numpy(cls, arr) -> "DeviceBuffer":
        arr = _coerce(arr)
        buf = cls(arr.size)
        buf.write(arr)
        return buf

    @staticmethod
    def view(ptr: int, n_words: int) -> DeviceView:
        """A buffer over memory of the library's device that something else owns (a tensor of another library): never freed from here.
        The library's work runs on its own stream, so what fills or reads that memory elsewhere has to be waited for."""
        if not ptr or ptr & 3 or n_words <= 0:
            raise ValueError("a view needs a 4-byte aligned device address and at least one word")
        return DeviceView(ptr, n_words)

    def free(self) -> None:
        if self.ptr:
            ptr, self.ptr = self.ptr, None  # the memory is gone even when the call reports an earlier kernel's error
            call("tfhip_free", ptr)

    def __del__(self):
        try:
            if getattr(self, "ptr", None) and _initialized:
                self.free()
        except Exception:
            pass


class Event:
    def __init__(self):
        h = C.c_void_p()
        call("tfhip_event_create", C.byref(h))
        self.handle = h.value

    def record(self) -> None:
        call("tfhip_event_record", self.handle)

    def elapsed_ms(self, stop: "Event") -> float:
        ms = C.c_float()
        call("tfhip_event_elapsed_ms", self.handle, stop.handle, C.byref(ms))
        return ms.value

    def __del__(self):
        try:
            if getattr(self, "handle", None):
                _lib.load().tfhip_event_destroy(self.handle)
        except Exception:
            pass


class Graph:
    """Everything issued inside the `with` block is recorded instead of run; launch() then enqueues it at once.

        g = Graph()
        with g:
            sort_kv(...)
        g.launch()

    Host copies, synchronize() and free are refused while recording; the recorded work keeps using the same buffers.
    """

    def __init__(self):
        self.handle = None

    def __enter__(self):
        call("tfhip_graph_begin")
        return self

    def __exit__(self, exc_type, exc, tb):
        if exc_type is not None:
            _lib.load().tfhip_graph_end(None)  # abandon the recording, keep the original error
            return False
        h = C.c_void_p()
        call("tfhip_graph_end", C.byref(h))
        self.handle = h.value
        return False

    @property
    def nodes(self) -> int:
        n = C.c_size_t()
        call("tfhip_graph_node_count", self.handle, C.byref(n))
        return n.value

    def launch(self) -> None:
        call("tfhip_graph_launch", self.handle)

    def destroy(self) -> None:
        if self.handle:
            call("tfhip_graph_destroy", self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class Kernel:
    """A hiprtc-compiled `extern "C" __global__` function (buffers..., vars struct)."""

    def __init__(self, source: str, name: str, options: str = ""):
        h = C.c_void_p()
        call("tfhip_module_compile", source.encode(), name.encode(), options.encode(), C.byref(h))
        self.handle = h.value
        self.name = name

    def launch(self, grid: int, block, buffers, variables=()) -> None:
        bx, by, bz = (list(block) + [1, 1])[:3]
        ptrs = (C.c_void_p * max(1, len(buffers)))(*[b.ptr if isinstance(b, DeviceView) else b for b in buffers])
        words = np.asarray(list(variables), dtype=np.uint32)
        vars_arr = (C.c_uint32 * max(1, len(words)))(*[int(w) for w in words])
        call("tfhip_launch", self.handle, grid, bx, by, bz, ptrs, len(buffers), vars_arr, len(words))

    def __del__(self):
        try:
            if getattr(self, "handle", None):
                _lib.load().tfhip_module_unload(self.handle)
        except Exception:
            pass


# ---- primitives ---------------------------------------------------------------------------------

def reduce_rows(op: str, x: DeviceBuffer, out: DeviceBuffer, rows: int, cols: int) -> None:
    """out[r] = op over the last axis of the [rows, cols] fp32 matrix in x."""
    call("tfhip_reduce_rows_f32", _REDUCE_OPS[op], x.ptr, out.ptr, rows, cols)


def reduce_cols(op: str, x: DeviceBuffer, out: DeviceBuffer, rows: int, cols: int) -> None:
    """out[c] = op over axis 0 of the [rows, cols] fp32 matrix in x."""
    call("tfhip_reduce_cols_f32", _REDUCE_OPS[op], x.ptr, out.ptr, rows, cols)


def reduce_cols_slabs(op: str, x: DeviceBuffer, out: DeviceBuffer, rows: int, cols: int, rows_per_slab: int) -> None:
    """out[s, c] = op over rows [s*rows_per_slab, (s+1)*rows_per_slab) of column c."""
    call("tfhip_reduce_cols_slabs_f32", _REDUCE_OPS[op], x.ptr, out.ptr, rows, cols, rows_per_slab)


def softmax_rows(x: DeviceBuffer, y: DeviceBuffer, rows: int, cols: int, row_max: DeviceBuffer = None, row_sum: DeviceBuffer = None) -> None:
    """y = softmax of every row of x[rows, cols]; with row_max and row_sum also the rows' maxima and sums of exp(x - max)."""
    if row_max is None and row_sum is None:
        call("tfhip_softmax_rows_f32", x.ptr, y.ptr, rows, cols)
    else:
        call("tfhip_softmax_rows_stats_f32", x.ptr, y.ptr, row_max.ptr if row_max else None, row_sum.ptr if row_sum else None, rows, cols)


def log_softmax_rows(x: DeviceBuffer, y: DeviceBuffer, rows: int, cols: int, row_max: DeviceBuffer = None, row_sum: DeviceBuffer = None) -> None:
    """y = (x - max) - log(sum(exp(x - max))) along every row of x[rows, cols]; with row_max and row_sum also those two."""
    if row_max is None and row_sum is None:
        call("tfhip_log_softmax_rows_f32", x.ptr, y.ptr, rows, cols)
    else:
        call("tfhip_log_softmax_rows_stats_f32", x.ptr, y.ptr, row_max.ptr if row_max else None, row_sum.ptr if row_sum else None, rows, cols)


def scan_inclusive(x: DeviceBuffer, out: DeviceBuffer, n: int, dtype=np.uint32) -> None:
    """out[i] = x[0] + ... + x[i]; dtype picks the u32 / i32 / f32 entry point."""
    kind = np.dtype(dtype).kind
    name = {"u": "tfhip_scan_inclusive_u32", "i": "tfhip_scan_inclusive_i32", "f": "tfhip_scan_inclusive_f32"}[kind]
    call(name, x.ptr, out.ptr, n)


def sgemm_batched(layout: str, a: DeviceBuffer, b: DeviceBuffer, c: DeviceBuffer, m: int, n: int, k: int, batch: int,
                  stride_a: int, stride_b: int, stride_c: int) -> None:
    """`batch` products in one launch; a stride of 0 shares that operand across the batch."""
    call("tfhip_sgemm_batched", {"nn": 0, "nt": 1, "tn": 2}[layout], a.ptr, b.ptr, c.ptr, m, n, k, batch, stride_a, stride_b, stride_c)


def scan_inclusive_cols(x: DeviceBuffer, out: DeviceBuffer, batch: int, rows: int, cols: int, dtype=np.uint32) -> None:
    """Prefix sums down the columns of `batch` row-major [rows, cols] matrices."""
    name = "tfhip_scan_inclusive_cols_f32" if np.dtype(dtype).kind == "f" else "tfhip_scan_inclusive_cols_u32"
    call(name, x.ptr, out.ptr, batch, rows, cols)


def scan_inclusive_rows(x: DeviceBuffer, out: DeviceBuffer, rows: int, cols: int, dtype=np.uint32) -> None:
    """Prefix sums along the last axis of a row-major [rows, cols] matrix, every row on its own."""
    name = "tfhip_scan_inclusive_rows_f32" if np.dtype(dtype).kind == "f" else "tfhip_scan_inclusive_rows_u32"
    call(name, x.ptr, out.ptr, rows, cols)


_KEY_KINDS = {"u": 0, "i": 1, "f": 2}


def radix_sort_kv(keys: DeviceBuffer, vals, keys_out: DeviceBuffer, vals_out, n: int, key_dtype=np.uint32,
                  keys_tmp: DeviceBuffer | None = None, vals_tmp: DeviceBuffer | None = None) -> None:
    """Stable ascending key(/payload) sort; vals / vals_out may be None for a keys-only sort."""
    p = lambda b: b.ptr if b is not None else None
    call("tfhip_radix_sort_kv", _KEY_KINDS[np.dtype(key_dtype).kind], keys.ptr, p(vals), keys_out.ptr, p(vals_out), p(keys_tmp), p(vals_tmp), n)


_EPILOGUES = {None: 0, "bias_relu": 1, "bias": 2, "mask_positive": 3}


def sgemm(layout: str, a: DeviceBuffer, b: DeviceBuffer, c: DeviceBuffer, m: int, n: int, k: int, epilogue=None, aux=None) -> None:
    """C[m,n] = op(A) op(B); layout 'nn' (A[m,k] B[k,n]), 'nt' (A[m,k] B[n,k]) or 'tn' (A[k,m] B[k,n]).
    epilogue: None | 'bias' | 'bias_relu' (aux = bias[n]) | 'mask_positive' (aux[m,n]: keep where aux > 0)."""
    if epilogue is None:
        call({"nn": "tfhip_sgemm_nn", "nt": "tfhip_sgemm_nt", "tn": "tfhip_sgemm_tn"}[layout], a.ptr, b.ptr, c.ptr, m, n, k)
    else:
        call("tfhip_sgemm_fused", {"nn": 0, "nt": 1, "tn": 2}[layout], a.ptr, b.ptr, c.ptr, m, n, k, _EPILOGUES[epilogue], aux.ptr if aux is not None else None)


def _words(buf: DeviceView | None, n_words: int, name: str):
    """The address of a buffer that has to hold at least n_words; None stays None. A buffer that was freed is an error, not None:
    the calls read a null pointer as one that was not given."""
    if buf is None:
        return None
    if buf.ptr is None:
        raise ValueError(f"{name} has been freed")
    if buf.n_words < n_words:
        raise ValueError(f"{name} holds {buf.n_words} words, {n_words} are needed")
    return buf.ptr


def layer_norm_rows(x: DeviceView, weight: DeviceView | None, bias: DeviceView | None, y: DeviceView, rows: int, cols: int, eps: float = 1e-5,
                    mean: DeviceView | None = None, rstd: DeviceView | None = None) -> None:
    """y = (x - mean) * rstd * weight + bias along every row of x[rows, cols]; mean and rstd receive the rows' statistics,
    which layer_norm_rows_backward takes. weight / bias None: 1 / 0. x may be y."""
    n = rows * cols
    call("tfhip_layer_norm_rows_f32", _words(x, n, "x"), _words(weight, cols, "weight"), _words(bias, cols, "bias"), _words(y, n, "y"), _words(mean, rows, "mean"),
         _words(rstd, rows, "rstd"), rows, cols, eps)


def layer_norm_rows_backward(x: DeviceView, dy: DeviceView, weight: DeviceView | None, mean: DeviceView, rstd: DeviceView, rows: int, cols: int,
                             dx: DeviceView | None = None, dweight: DeviceView | None = None, dbias: DeviceView | None = None) -> None:
    """The gradients of layer_norm_rows from the upstream gradient dy; any of dx, dweight, dbias that is given. dx may be
    x or dy."""
    n = rows * cols
    call("tfhip_layer_norm_rows_backward_f32", _words(x, n, "x"), _words(dy, n, "dy"), _words(weight, cols, "weight"), _words(mean, rows, "mean"), _words(rstd, rows, "rstd"),
         _words(dx, n, "dx"), _words(dweight, cols, "dweight"), _words(dbias, cols, "dbias"), rows, cols)


def embedding_rows(tokens: DeviceView, table: DeviceView, out: DeviceView, n: int, vocab: int, cols: int, scale: float = 1.0) -> None:
    """out[i] = scale * table[tokens[i]] for n int32 tokens; zeros for a token outside [0, vocab)."""
    call("tfhip_embedding_rows_f32", _words(tokens, n, "tokens"), _words(table, vocab * cols, "table"), _words(out, n * cols, "out"), n, vocab, cols, scale)


def embedding_rows_backward(tokens: DeviceView, dy: DeviceView, dtable: DeviceView, n: int, vocab: int, cols: int, scale: float = 1.0) -> None:
    """dtable[v] = scale * the sum of dy[i] over the positions with tokens[i] == v; every row of dtable is written."""
    call("tfhip_embedding_rows_backward_f32", _words(tokens, n, "tokens"), _words(dy, n * cols, "dy"), _words(dtable, vocab * cols, "dtable"), n, vocab, cols, scale)


NEWTON_SCHULZ_QUINTIC = (3.4445, -4.7750, 2.0315)  # drives singular values into about 0.7 .. 1.2 within five steps


def newton_schulz(g: DeviceView, out: DeviceView, rows: int, cols: int, steps: int = 5, batch: int = 1, coefficients=NEWTON_SCHULZ_QUINTIC, eps: float = 1e-7) -> None:
    """Orthogonalises `batch` matrices [rows, cols] by `steps` Newton-Schulz products. coefficients: (a, b, c) of every
    step, or one such triple per step. g may be out."""
    if not 1 <= steps <= 64:  # before there is a triple for each of them, and before the number becomes one of 32 bits
        raise ValueError(f"{steps} Newton-Schulz steps (1 to 64 are taken)")
    triples = np.asarray(coefficients, dtype=np.float32)
    if triples.ndim == 1:
        triples = np.tile(triples, (steps, 1))
    if triples.shape != (steps, 3):
        raise ValueError(f"{steps} steps need three coefficients, or {steps} x 3; got an array of shape {triples.shape}")
    triples = np.ascontiguousarray(triples)
    n = batch * rows * cols
    call("tfhip_newton_schulz_f32", _words(g, n, "g"), _words(out, n, "out"), batch, rows, cols, steps, triples.ctypes.data_as(C.POINTER(C.c_float)), eps)


__all__ = [
    "initialize", "shutdown", "device_info", "synchronize", "DeviceBuffer", "DeviceView", "Event", "Kernel",
    "reduce_rows", "reduce_cols", "reduce_cols_slabs", "softmax_rows", "log_softmax_rows", "scan_inclusive", "radix_sort_kv", "sgemm",
    "layer_norm_rows", "layer_norm_rows_backward", "embedding_rows", "embedding_rows_backward", "newton_schulz", "NEWTON_SCHULZ_QUINTIC", "TFHipError",
]
