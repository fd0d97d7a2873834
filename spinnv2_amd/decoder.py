"""Operators of a decoder layer in 8 bits (include/spkv2_decoder.h) from Python.

    rmsnorm_i8      residual + root-mean-square norm -> int8 rows with scales
    quantize_i8     rows -> int8 rows with scales
    dequantize_i8   int8 rows -> values
    matmul_i8       int8 rows x int8 weights, a scale for each row and channel
    KvCache         a paged int8 key/value cache: write, read
    attention       attention of new tokens to a KvCache

No counterpart in the reference.  A tensor is anything with ``data_ptr()``,
``shape``, ``stride()`` and ``dtype`` on the GPU: a torch tensor (import torch
before this library is loaded, so that both use one HIP runtime) or a
`DeviceArray`, which needs no torch.  Calls enqueue on ``stream`` (a
hipStream_t as a number, torch's ``Stream.cuda_stream``; 0 is the default
stream), return without waiting, and write into tensors of the caller's: keep
every tensor of a call until its work is done.  Shapes and types that do not
fit raise ValueError, numbers past the C types' ranges struct.error, what the
library refuses raises RuntimeError_.
"""

from __future__ import annotations

import ctypes
import math
import struct

import numpy as np

from .runtime import DeviceBuffer, _check, load_library

_FP32, _INT8, _FP16, _BF16, _INT32, _INT64 = 1, 2, 3, 4, 101, 102
#: dtype -> the library's code; torch's own dtype objects join at first sight
_CODES = {"float32": _FP32, "float16": _FP16, "bfloat16": _BF16, "int8": _INT8, "int32": _INT32, "int64": _INT64}
_FLOATS = (_FP32, _FP16, _BF16)
_FP32S, _INT8S, _INT32S, _INT64S = (_FP32,), (_INT8,), (_INT32,), (_INT64,)

_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class _RmsNorm(ctypes.Structure):
    _fields_ = [("x", _P), ("residual", _P), ("weight", _P), ("residual_out", _P), ("q", _P), ("scale", _P),
                ("rows", _I64), ("cols", _I64), ("x_stride", _I64), ("residual_stride", _I64),
                ("residual_out_stride", _I64), ("q_stride", _I64), ("dtype", _I32), ("weight_dtype", _I32),
                ("norm", _I32), ("eps", _F)]


class _Dequantize(ctypes.Structure):
    _fields_ = [("q", _P), ("scale", _P), ("out", _P), ("rows", _I64), ("cols", _I64), ("q_stride", _I64),
                ("out_stride", _I64), ("dtype", _I32), ("reserved", _I32)]


class _Matmul(ctypes.Structure):
    _fields_ = [("a", _P), ("b", _P), ("a_scale", _P), ("b_scale", _P), ("bias", _P), ("out", _P),
                ("m", _I64), ("n", _I64), ("k", _I64), ("a_stride", _I64), ("b_stride", _I64), ("out_stride", _I64),
                ("dtype", _I32), ("reserved", _I32)]


class _Cache(ctypes.Structure):
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("pages", _I64), ("kv_heads", _I32),
                ("page_size", _I32), ("head_dim", _I32), ("reserved", _I32)]


class _Write(ctypes.Structure):
    _fields_ = [("k", _P), ("v", _P), ("slots", _P), ("tokens", _I64), ("k_stride", _I64), ("v_stride", _I64),
                ("dtype", _I32), ("reserved", _I32)]


class _Read(ctypes.Structure):
    _fields_ = [("table", _P), ("first", _P), ("offsets", _P), ("k", _P), ("v", _P), ("tokens", _I64),
                ("k_stride", _I64), ("v_stride", _I64), ("sequences", _I32), ("table_width", _I32), ("dtype", _I32),
                ("reserved", _I32)]


class _Attention(ctypes.Structure):
    _fields_ = [("q", _P), ("out", _P), ("table", _P), ("lengths", _P), ("offsets", _P), ("workspace", _P),
                ("workspace_size", ctypes.c_size_t), ("queries", _I64), ("q_stride", _I64), ("out_stride", _I64),
                ("max_queries", _I64), ("max_length", _I64), ("sequences", _I32), ("table_width", _I32), ("heads", _I32),
                ("dtype", _I32), ("causal", _I32), ("window", _I32), ("scale", _F), ("reserved", _I32)]


_LETTERS = {_P: "P", _I32: "i", _I64: "q", _F: "f", ctypes.c_size_t: "N"}


def _packer(cls):
    """The function that lays a Structure's fields out as bytes, which a call
    takes as the struct's address: a fifth of the time that setting a
    Structure's fields takes (norm's 18: 0.5 against 2.4 us)."""
    s = struct.Struct("@" + "".join(_LETTERS[kind] for _, kind in cls._fields_))
    assert s.size == ctypes.sizeof(cls)
    return s.pack


_pack_norm, _pack_dequantize, _pack_matmul = _packer(_RmsNorm), _packer(_Dequantize), _packer(_Matmul)
_pack_write, _pack_read, _pack_attention = _packer(_Write), _packer(_Read), _packer(_Attention)


class DeviceArray:
    """A tensor in a `DeviceBuffer`, for callers without torch.

    ``dtype`` is one of float32, float16, bfloat16, int8, int32, int64;
    bfloat16 values come and go as float32 arrays.  ``at`` elements from the
    buffer's start; ``strides`` in elements, none below zero (default:
    contiguous).
    """

    is_cuda = True

    def __init__(self, shape, dtype: str, *, buffer: DeviceBuffer | None = None, at: int = 0, strides=None) -> None:
        if dtype not in _CODES:
            raise ValueError(f"unknown dtype {dtype!r}")
        self.shape, self.dtype = tuple(int(d) for d in shape), dtype
        self.strides = tuple(strides) if strides else tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))
        self.itemsize = 2 if dtype == "bfloat16" else np.dtype(dtype).itemsize
        self.at = at
        extent = 1 + sum((d - 1) * s for d, s in zip(self.shape, self.strides)) if math.prod(self.shape) else 0
        if buffer is None:
            buffer = DeviceBuffer(max(16, (at + extent) * self.itemsize))
        if at < 0 or min(self.strides, default=0) < 0 or (at + extent) * self.itemsize > buffer.nbytes:
            raise ValueError("the array does not fit its buffer")
        self.buffer = buffer

    @classmethod
    def of(cls, values: np.ndarray, dtype: str | None = None) -> "DeviceArray":
        """A contiguous array of these values, in `dtype` (default: theirs)."""
        a = cls(values.shape, dtype or str(values.dtype))
        a.upload(values)
        return a

    def data_ptr(self) -> int:
        return self.buffer.ptr.value + self.at * self.itemsize

    def stride(self) -> tuple:
        return self.strides

    def _whole(self) -> np.ndarray:
        raw = np.empty(self.buffer.nbytes, np.uint8)
        _check(self.buffer.lib, self.buffer.lib.spkv2_device_memcpy_d2h(raw.ctypes.data, self.buffer.ptr, raw.nbytes), "d2h")
        return raw

    def _view(self, raw: np.ndarray) -> np.ndarray:
        kind = np.dtype(np.uint16 if self.dtype == "bfloat16" else self.dtype)
        flat = raw[: raw.nbytes // kind.itemsize * kind.itemsize].view(kind)[self.at:]
        return np.lib.stride_tricks.as_strided(flat, self.shape, [s * kind.itemsize for s in self.strides])

    def upload(self, values) -> None:
        """Writes the values, rounded to the array's type; what lies between strided rows stays."""
        values = np.broadcast_to(np.asarray(values), self.shape)
        raw = self._whole()
        self._view(raw)[...] = to_bfloat16(values) if self.dtype == "bfloat16" else values.astype(self.dtype)
        self.buffer.upload(raw)

    def download(self) -> np.ndarray:
        a = self._view(self._whole()).copy()
        return (a.astype(np.uint32) << 16).view(np.float32) if self.dtype == "bfloat16" else a


def to_bfloat16(values) -> np.ndarray:
    """float32 values rounded to the nearest bfloat16, ties to even, as its 16 bits."""
    f = np.ascontiguousarray(values, np.float32)
    u = f.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7FC0), r)


def _code(t) -> int:
    """The library's code of a tensor's dtype; torch's dtype objects join _CODES here."""
    code = _CODES.get(t.dtype)
    if code is None:
        code = _CODES.get(str(t.dtype).replace("torch.", ""))
        if code is None:
            raise ValueError(f"unsupported dtype {t.dtype}")
        _CODES[t.dtype] = code
    return code


def _fail(name: str, why: str):
    raise ValueError(f"{name}: {why}")


def _refuse(name: str, t, codes, shape) -> None:
    """Says which of a tensor's type, shape and place does not fit; nothing
    where its dtype object was only met for the first time."""
    if _code(t) not in codes:
        _fail(name, f"unexpected dtype {t.dtype}")
    if t.shape != shape:
        _fail(name, f"shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_cuda:
        _fail(name, "not on the GPU")


def _rows(name: str, t, codes, shape) -> int:
    """A 2-d tensor's row stride, its type and shape checked."""
    if t.shape != shape or _CODES.get(t.dtype) not in codes or not t.is_cuda:
        _refuse(name, t, codes, shape)
    row, step = t.stride()
    if step != 1 and shape[1] > 1:
        _fail(name, "its last axis is not contiguous")
    return row


def _vector(name: str, t, codes, n: int) -> int:
    """A contiguous vector's address, its type and length checked."""
    if t.shape != (n,) or _CODES.get(t.dtype) not in codes or not t.is_cuda:
        _refuse(name, t, codes, (n,))
    if t.stride() != (1,) and n > 1:
        _fail(name, "not contiguous")
    return t.data_ptr()


def _heads(name: str, t, codes, shape) -> int:
    """A [tokens, heads, dim] tensor's token stride: the heads have to lie one after the other."""
    if t.shape != shape or _CODES.get(t.dtype) not in codes or not t.is_cuda:
        _refuse(name, t, codes, shape)
    row, head, step = t.stride()
    if step != 1 or (head != shape[2] and shape[1] > 1):
        _fail(name, "its heads are not contiguous")
    return row


def _table(t) -> tuple:
    """(sequences, width) of a page table."""
    shape = t.shape
    if len(shape) != 2:
        _fail("table", "not two-dimensional")
    if _rows("table", t, _INT32S, shape) != shape[1] and shape[0] > 1:
        _fail("table", "not contiguous")
    return shape


def rmsnorm_i8(x, weight, q, scale, *, residual=None, residual_out=None, eps: float = 1e-6, stream: int = 0) -> None:
    """h = x + residual; q, scale = int8 rows of h * weight / sqrt(mean(h^2) + eps).

    x [rows, cols] in float32, float16 or bfloat16, residual and residual_out
    (where h is stored; it may be x or residual) of the same type; weight
    [cols] of that type or float32, or None; q int8, scale [rows] float32.
    """
    _norm_rows(x, weight, q, scale, residual, residual_out, 1, eps, stream)


def quantize_i8(x, q, scale, *, stream: int = 0) -> None:
    """q, scale = int8 rows of x."""
    _norm_rows(x, None, q, scale, None, None, 0, 0.0, stream)


def _norm_rows(x, weight, q, scale, residual, residual_out, norm, eps, stream) -> None:
    shape, code = x.shape, _code(x)
    if len(shape) != 2:
        _fail("x", "not two-dimensional")
    rows, cols = shape
    w = w_code = r = r_stride = h = h_stride = 0
    if weight is not None:
        w, w_code = _vector("weight", weight, (code, _FP32), cols), _CODES[weight.dtype]
    if residual is not None:
        r_stride, r = _rows("residual", residual, (code,), shape), residual.data_ptr()
    if residual_out is not None:
        h_stride, h = _rows("residual_out", residual_out, (code,), shape), residual_out.data_ptr()
    a = _pack_norm(x.data_ptr(), r, w, h, q.data_ptr(), _vector("scale", scale, _FP32S, rows), rows, cols,
                   _rows("x", x, _FLOATS, shape), r_stride, h_stride, _rows("q", q, _INT8S, shape), code, w_code, norm, eps)
    lib = load_library()
    if code := lib.spkv2_mi355x_rmsnorm_i8(a, stream):
        _check(lib, code, "rmsnorm_i8")


def dequantize_i8(q, scale, out, *, stream: int = 0) -> None:
    """out = q * scale, row by row; out float32, float16 or bfloat16."""
    shape = q.shape
    if len(shape) != 2:
        _fail("q", "not two-dimensional")
    rows, cols = shape
    a = _pack_dequantize(q.data_ptr(), _vector("scale", scale, _FP32S, rows), out.data_ptr(), rows, cols,
                         _rows("q", q, _INT8S, shape), _rows("out", out, _FLOATS, shape), _code(out), 0)
    lib = load_library()
    if code := lib.spkv2_mi355x_dequantize_i8(a, stream):
        _check(lib, code, "dequantize_i8")


def matmul_i8(a, a_scale, b, b_scale, out, *, bias=None, stream: int = 0) -> None:
    """out[m, n] = a_scale[m] b_scale[n] sum_k a[m, k] b[n, k] + bias[n].

    a [m, k] and b [n, k] int8, the scales and bias float32, out [m, n]
    float32, float16 or bfloat16.
    """
    if len(a.shape) != 2 or len(b.shape) != 2:
        _fail("a, b", "not two-dimensional")
    (m, k), n = a.shape, b.shape[0]
    g = _pack_matmul(a.data_ptr(), b.data_ptr(), _vector("a_scale", a_scale, _FP32S, m), _vector("b_scale", b_scale, _FP32S, n),
                     0 if bias is None else _vector("bias", bias, _FP32S, n), out.data_ptr(), m, n, k,
                     _rows("a", a, _INT8S, (m, k)), _rows("b", b, _INT8S, (n, k)), _rows("out", out, _FLOATS, (m, n)),
                     _code(out), 0)
    lib = load_library()
    if code := lib.spkv2_mi355x_matmul_i8(g, stream):
        _check(lib, code, "matmul_i8")


class KvCache:
    """A paged int8 cache over the caller's buffers.

    k, v: int8 [pages, kv_heads, page_size, head_dim], k_scale, v_scale:
    float32 [pages, kv_heads, page_size], contiguous.  Token i of a sequence is
    row i % page_size of page table[i // page_size], its slot that page *
    page_size + row.
    """

    def __init__(self, k, v, k_scale, v_scale) -> None:
        if len(k.shape) != 4:
            _fail("k", "not [pages, kv_heads, page_size, head_dim]")
        self.pages, self.kv_heads, self.page_size, self.head_dim = (int(d) for d in k.shape)
        for name, t, code, shape in (("k", k, _INT8, tuple(k.shape)), ("v", v, _INT8, tuple(k.shape)),
                                     ("k_scale", k_scale, _FP32, tuple(k.shape)[:3]),
                                     ("v_scale", v_scale, _FP32, tuple(k.shape)[:3])):
            if _code(t) != code or tuple(t.shape) != shape or not t.is_cuda:
                _fail(name, f"expected {shape} of another type or place")
            if not _contiguous(t):
                _fail(name, "not contiguous")
        self.buffers = (k, v, k_scale, v_scale)  # held as long as the cache is
        self._c = _Cache(*(t.data_ptr() for t in self.buffers), self.pages, self.kv_heads, self.page_size, self.head_dim, 0)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, head_dim: int) -> "KvCache":
        """A cache in memory of its own; what it holds is not set."""
        shape = (pages, kv_heads, page_size, head_dim)
        return cls(DeviceArray(shape, "int8"), DeviceArray(shape, "int8"), DeviceArray(shape[:3], "float32"),
                   DeviceArray(shape[:3], "float32"))

    def write(self, k, v, slots, *, stream: int = 0) -> None:
        """Quantises k and v [tokens, kv_heads, head_dim] into the slots (int64
        [tokens]; negative ones, and those past the cache, are not written)."""
        shape = (k.shape[0], self.kv_heads, self.head_dim)
        code = _code(k)
        a = _pack_write(k.data_ptr(), v.data_ptr(), _vector("slots", slots, _INT64S, shape[0]), shape[0],
                        _heads("k", k, _FLOATS, shape), _heads("v", v, (code,), shape), code, 0)
        lib = load_library()
        if code := lib.spkv2_mi355x_kv_write_i8(self._ref, a, stream):
            _check(lib, code, "kv_write_i8")

    def read(self, table, first, offsets, k, v, *, stream: int = 0) -> None:
        """Reads tokens first[s] .. of each sequence s into rows offsets[s] ..
        offsets[s + 1] of k and v.  table int32 [sequences, width], first int32
        [sequences] or None, offsets int32 [sequences + 1]."""
        shape = (k.shape[0], self.kv_heads, self.head_dim)
        seqs, width = _table(table)
        code = _code(k)
        a = _pack_read(table.data_ptr(), 0 if first is None else _vector("first", first, _INT32S, seqs),
                       _vector("offsets", offsets, _INT32S, seqs + 1), k.data_ptr(), v.data_ptr(), shape[0],
                       _heads("k", k, _FLOATS, shape), _heads("v", v, (code,), shape), seqs, width, code, 0)
        lib = load_library()
        if code := lib.spkv2_mi355x_kv_read_i8(self._ref, a, stream):
            _check(lib, code, "kv_read_i8")


def attention_workspace(sequences: int, queries: int, heads: int, cache: KvCache, *, max_queries: int, max_length: int) -> int:
    """Bytes of workspace that `attention` needs at these sizes (0: none)."""
    a = _Attention(queries=queries, max_queries=max_queries, max_length=max_length, sequences=sequences, heads=heads,
                   dtype=_FP32)
    size = ctypes.c_size_t()
    lib = load_library()
    _check(lib, lib.spkv2_mi355x_attention_i8_workspace(cache._ref, ctypes.byref(a), ctypes.byref(size)), "attention_i8_workspace")
    return size.value


def attention(q, cache: KvCache, table, lengths, offsets, out, *, max_queries: int, max_length: int, causal: bool = True,
              window: int = 0, scale: float | None = None, workspace=None, stream: int = 0) -> None:
    """out = softmax(scale q k^T) v over each sequence's cached tokens.

    q, out [queries, heads, head_dim]; sequence s has rows offsets[s] ..
    offsets[s + 1] of them and lengths[s] cached tokens, found through its row
    of table.  Causal: query i of n is token lengths[s] - n + i and reads the
    tokens up to itself, the last `window` of them where window > 0; otherwise
    (an encoder's states) each query reads all.  A query that has nothing to
    read gets zeros.  max_queries and max_length bound the sequences' counts and
    lengths; workspace: a buffer of attention_workspace() bytes; scale: 1 /
    sqrt(head_dim) by default.
    """
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.head_dim:
        _fail("q", f"shape {tuple(shape)}, expected [queries, heads, {cache.head_dim}]")
    seqs, width = _table(table)
    code = _code(q)
    size = at = 0
    if workspace is not None:
        size = math.prod(workspace.shape)
        if _code_size(workspace) != 1 or not workspace.is_cuda:
            _fail("workspace", "not bytes on the GPU")
        if workspace.stride() != (1,) and not _contiguous(workspace):
            _fail("workspace", "not contiguous")
        at = workspace.data_ptr() if size else 0
    a = _pack_attention(q.data_ptr(), out.data_ptr(), table.data_ptr(), _vector("lengths", lengths, _INT32S, seqs),
                        _vector("offsets", offsets, _INT32S, seqs + 1), at, size, shape[0], _heads("q", q, _FLOATS, shape),
                        _heads("out", out, (code,), shape), max_queries, max_length, seqs, width, shape[1], code, 1 if causal else 0,
                        window, cache.head_dim ** -0.5 if scale is None else scale, 0)
    lib = load_library()
    if code := lib.spkv2_mi355x_attention_i8(cache._ref, a, stream):
        _check(lib, code, "attention_i8")


def _contiguous(t) -> bool:
    """Whether a tensor's elements lie one after the other; an axis of one element may have any stride."""
    step = 1
    for n, stride in zip(reversed(t.shape), reversed(t.stride())):
        if n != 1 and stride != step:
            return False
        step *= n
    return True


def _code_size(t) -> int:
    return t.itemsize if hasattr(t, "itemsize") else t.element_size()
