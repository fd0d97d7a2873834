// The decoder layer's calls for Python: tensors' attributes checked and laid out
// as the C entry points' arguments (include/spkv2_decoder.h).
//
// A call of a few tokens is bound by the host.  A tensor checked from Python,
// its numbers packed there too, costs 0.5 us, from here 0.3, which its five
// attributes are themselves: a product's call without its launch took 2.7 us and
// takes 1.5, 4 rows of 2048 normed and read back 14.3 us and 12.1, one token of
// 4 sequences rotated into the cache and read back 17.9 us and 14.0.
//
// A tensor is anything with data_ptr(), shape, stride(), dtype and is_cuda.
// Nothing is kept between calls but the entry points' addresses.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>

#include "spkv2_decoder.h"

namespace {

// Types as spinnv2_amd.decoder numbers them
enum Code { kFp32 = 1, kInt8 = 2, kFp16 = 3, kBf16 = 4, kInt32 = 101, kInt64 = 102, kF8 = 103 };
constexpr unsigned bit(int code) { return code < 32 ? 1u << code : 1u << (code - 101 + 8); }
constexpr unsigned kFloats = bit(kFp32) | bit(kFp16) | bit(kBf16);

// An owned reference
struct Ref {
    PyObject *o;
    explicit Ref(PyObject *p) : o(p) {}
    Ref(const Ref &) = delete;
    Ref &operator=(const Ref &) = delete;
    ~Ref() { Py_XDECREF(o); }
    explicit operator bool() const { return o != nullptr; }
};

// Set by bind(), which spinnv2_amd.decoder calls once
PyObject *codes, *code_of, *range_error;  // dtype -> code; what adds one or refuses it; struct.error
PyObject *s_shape, *s_dtype, *s_is_cuda, *s_stride, *s_data_ptr;
struct Entries {
    int (*rotate)(const Spkv2KvCacheI8 *, const Spkv2Rotate *, void *);
    int (*rows)(const Spkv2RowsF8 *, void *);
    int (*dequantize)(const Spkv2DequantizeF8 *, void *);
    int (*matmul)(const Spkv2MatmulF8 *, void *);
    int (*experts)(const Spkv2MatmulF8Experts *, void *);
    int (*sort)(const Spkv2SortTokens *, void *);
    int (*combine)(const Spkv2Combine *, void *);
    int (*kv_write)(const Spkv2KvCacheI8 *, const Spkv2KvWrite *, void *);
    int (*kv_read)(const Spkv2KvCacheI8 *, const Spkv2KvRead *, void *);
} entries;

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const char *name, const char *why) {
    PyErr_Format(PyExc_ValueError, "%s: %s", name, why);
    throw Refused{};
}

int64_t number(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (PyErr_ExceptionMatches(PyExc_OverflowError)) {
            PyErr_Clear();
            PyErr_SetString(range_error, "a number does not fit 64 bits");
        }
        throw Refused{};
    }
    return v;
}
int32_t small_number(PyObject *o) {
    const int64_t v = number(o);
    if (v != static_cast<int32_t>(v)) {
        PyErr_SetString(range_error, "a number does not fit 32 bits");
        throw Refused{};
    }
    return static_cast<int32_t>(v);
}
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{};
    return static_cast<float>(v);
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused{};
    return v;
}
void *address(PyObject *o) { return reinterpret_cast<void *>(number(o)); }
// as ctypes takes a void pointer: a number, None, or a c_void_p
void *handle(PyObject *o) {
    if (o == Py_None) return nullptr;
    if (PyIndex_Check(o)) return address(o);
    Ref value(PyObject_GetAttrString(o, "value"));
    if (!value) throw Refused{};
    return value.o == Py_None ? nullptr : address(value.o);
}

constexpr int kMostAxes = 3;
struct Tensor {
    PyObject *o;
    const char *name;
    int axes;
    int64_t shape[kMostAxes], stride[kMostAxes];
    int code;
    char *p;
};

// n numbers of a tuple (or what can be made one)
int numbers(PyObject *o, int64_t (&v)[kMostAxes]) {
    Ref made(PyTuple_Check(o) ? nullptr : PySequence_Tuple(o));
    PyObject *t = made ? made.o : o;
    if (!PyTuple_Check(t)) throw Refused{};
    const Py_ssize_t n = PyTuple_GET_SIZE(t);
    for (Py_ssize_t i = 0; i < n && i < kMostAxes; i++) v[i] = number(PyTuple_GET_ITEM(t, i));
    return static_cast<int>(n);
}

// shape and type, which other tensors' are held against
Tensor first_look(PyObject *o, const char *name, int axes, const char *kind) {
    Tensor t{o, name, axes, {}, {}, 0, nullptr};
    Ref shape(PyObject_GetAttr(o, s_shape));
    if (!shape) throw Refused{};
    if (numbers(shape.o, t.shape) != axes) refuse(name, kind);
    Ref dtype(PyObject_GetAttr(o, s_dtype));
    if (!dtype) throw Refused{};
    PyObject *code = PyDict_GetItemWithError(codes, dtype.o);
    if (code) {
        t.code = static_cast<int>(PyLong_AsLong(code));
    } else {
        if (PyErr_Occurred()) throw Refused{};
        Ref found(PyObject_CallFunctionObjArgs(code_of, o, nullptr));
        if (!found) throw Refused{};
        t.code = static_cast<int>(PyLong_AsLong(found.o));
    }
    return t;
}
// the rest of it, its type and shape (-1: any) checked
Tensor &settle(Tensor &t, unsigned allowed, const int64_t *shape) {
    if (!(bit(t.code) & allowed)) {
        Ref dtype(PyObject_GetAttr(t.o, s_dtype));
        if (dtype) PyErr_Format(PyExc_ValueError, "%s: unexpected dtype %S", t.name, dtype.o);
        throw Refused{};
    }
    for (int i = 0; i < t.axes; i++)
        if (t.shape[i] != shape[i]) {
            Ref is(PyObject_GetAttr(t.o, s_shape));
            if (is) PyErr_Format(PyExc_ValueError, "%s: shape %S, expected %lld along axis %d", t.name, is.o, static_cast<long long>(shape[i]), i);
            throw Refused{};
        }
    Ref cuda(PyObject_GetAttr(t.o, s_is_cuda));
    if (!cuda) throw Refused{};
    if (!truth(cuda.o)) refuse(t.name, "not on the GPU");
    Ref stride(PyObject_CallMethodNoArgs(t.o, s_stride));
    if (!stride) throw Refused{};
    if (numbers(stride.o, t.stride) != t.axes) refuse(t.name, "a stride for each axis is missing");
    Ref p(PyObject_CallMethodNoArgs(t.o, s_data_ptr));
    if (!p) throw Refused{};
    t.p = static_cast<char *>(address(p.o));
    return t;
}

Tensor &rows_settled(Tensor &t, unsigned allowed, int64_t rows, int64_t cols) {
    const int64_t shape[] = {rows, cols};
    settle(t, allowed, shape);
    if (t.stride[1] != 1 && cols > 1) refuse(t.name, "its last axis is not contiguous");
    return t;
}
// [rows, cols], rows any distance apart
Tensor rows_of(PyObject *o, const char *name, unsigned allowed, int64_t rows, int64_t cols) {
    Tensor t = first_look(o, name, 2, "not two-dimensional");
    return rows_settled(t, allowed, rows, cols);
}
// [rows, cols], contiguous
Tensor matrix(PyObject *o, const char *name, unsigned allowed, int64_t rows, int64_t cols) {
    Tensor t = rows_of(o, name, allowed, rows, cols);
    if (t.stride[0] != cols && rows > 1) refuse(name, "not contiguous");
    return t;
}
// [n], contiguous
Tensor &vector_settled(Tensor &t, unsigned allowed, int64_t n) {
    settle(t, allowed, &n);
    if (t.stride[0] != 1 && n > 1) refuse(t.name, "not contiguous");
    return t;
}
Tensor vector(PyObject *o, const char *name, unsigned allowed, int64_t n) {
    Tensor t = first_look(o, name, 1, "not one-dimensional");
    return vector_settled(t, allowed, n);
}
// [tokens, heads, dim], heads one after the other
Tensor &heads_settled(Tensor &t, unsigned allowed, int64_t tokens, int64_t heads, int64_t dim) {
    const int64_t shape[] = {tokens, heads, dim};
    settle(t, allowed, shape);
    if (t.stride[2] != 1 || (t.stride[1] != dim && heads > 1)) refuse(t.name, "its heads are not contiguous");
    return t;
}
Tensor heads_of(PyObject *o, const char *name, unsigned allowed, int64_t tokens, int64_t heads, int64_t dim) {
    Tensor t = first_look(o, name, 3, "not [tokens, heads, head_dim]");
    return heads_settled(t, allowed, tokens, heads, dim);
}

bool given(PyObject *o) { return o != Py_None; }
int64_t blocks(int64_t n) { return (n + SPKV2_F8_BLOCK - 1) / SPKV2_F8_BLOCK; }
template <typename T>
T *as(const Tensor &t) {
    return reinterpret_cast<T *>(t.p);
}
int32_t as_int32(int64_t v) {
    if (v != static_cast<int32_t>(v)) {
        PyErr_SetString(range_error, "a size does not fit 32 bits");
        throw Refused{};
    }
    return static_cast<int32_t>(v);
}

// The library's answer, as a number; COUNT arguments
template <int COUNT, typename F>
PyObject *guarded(Py_ssize_t count, F &&f) {
    if (count != COUNT) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", COUNT, count);
        return nullptr;
    }
    if (!codes) {
        PyErr_SetString(PyExc_RuntimeError, "bind() was not called");
        return nullptr;
    }
    try {
        return PyLong_FromLong(f());
    } catch (const Refused &) {
        return nullptr;
    }
}
// without the interpreter's lock, as other threads may wait for it while a launch waits for its queue
template <typename F>
int unlocked(F &&f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = f();
    Py_END_ALLOW_THREADS return rc;
}

// (q, k, positions, frequencies, q_out, k_out, axes, norm, q_weight, k_weight, eps, interleaved, cache, kv_heads, head_dim, v, slots, stream):
// cache the address of its struct or None, with its heads
PyObject *rotate(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<18>(count, [&]() -> int {
        Spkv2Rotate g{};
        const bool has_q = given(a[0]), has_k = given(a[1]);
        if (!has_q && !has_k) refuse("q, k", "neither is there");
        Tensor x = first_look(has_q ? a[0] : a[1], has_q ? "q" : "k", 3, "not [tokens, heads, head_dim]");
        const int64_t tokens = x.shape[0], dim = x.shape[2];
        g.tokens = tokens;
        g.head_dim = as_int32(dim);
        g.dtype = x.code;
        heads_settled(x, kFloats, tokens, x.shape[1], dim);
        const unsigned same = bit(x.code);
        if (has_q) {
            if (!given(a[4])) refuse("q_out", "queries without an output");
            const Tensor out = heads_of(a[4], "q_out", same, tokens, x.shape[1], dim);
            g.heads = as_int32(x.shape[1]);
            g.q = x.p, g.q_stride = x.stride[0];
            g.q_out = out.p, g.q_out_stride = out.stride[0];
        }
        const bool cached = given(a[12]);
        if (has_k) {
            Tensor k = x;
            if (has_q) {
                k = first_look(a[1], "k", 3, "not [tokens, kv_heads, head_dim]");
                heads_settled(k, same, tokens, k.shape[1], dim);
            }
            g.kv_heads = as_int32(k.shape[1]);
            g.k = k.p, g.k_stride = k.stride[0];
            if (given(a[5])) {
                const Tensor out = heads_of(a[5], "k_out", same, tokens, k.shape[1], dim);
                g.k_out = out.p, g.k_out_stride = out.stride[0];
            } else if (!cached) {
                refuse("k_out", "keys without an output or a cache");
            }
        }
        if (cached) {
            if (!has_k || !given(a[15]) || !given(a[16])) refuse("cache", "keys, values or slots are missing");
            if (number(a[13]) != g.kv_heads || number(a[14]) != dim) refuse("k", "the cache has other heads");
            const Tensor v = heads_of(a[15], "v", same, tokens, g.kv_heads, dim);
            g.v = v.p, g.v_stride = v.stride[0];
            g.slots = as<int64_t>(vector(a[16], "slots", bit(kInt64), tokens));
        }
        g.norm = truth(a[7]);
        if (g.norm) {
            if (given(a[8])) {
                const Tensor w = vector(a[8], "q_weight", same | bit(kFp32), dim);
                g.q_weight = w.p, g.weight_dtype = w.code;
            }
            if (given(a[9])) {
                const Tensor w = vector(a[9], "k_weight", same | bit(kFp32), dim);
                if (g.weight_dtype && g.weight_dtype != w.code) refuse("k_weight", "the weights are of different types");
                g.k_weight = w.p, g.weight_dtype = w.code;
            }
        }
        g.eps = real(a[10]);
        Tensor f = first_look(a[3], "frequencies", 1, "not one-dimensional");
        g.frequencies = as<float>(vector_settled(f, bit(kFp32), f.shape[0]));
        g.pairs = as_int32(f.shape[0]);
        Ref shape(PyObject_GetAttr(a[2], s_shape));
        if (!shape) throw Refused{};
        const Py_ssize_t axes = PyObject_Size(shape.o);
        if (axes == 1) {
            g.positions = as<int32_t>(vector(a[2], "positions", bit(kInt32), tokens));
            g.axes = 1, g.position_stride = 1;
        } else {
            Tensor p = first_look(a[2], "positions", 2, "not [tokens] or [tokens, axes]");
            g.positions = as<int32_t>(rows_settled(p, bit(kInt32), tokens, p.shape[1]));
            g.axes = as_int32(p.shape[1]), g.position_stride = p.stride[0];
        }
        if (given(a[6])) g.axis = as<int32_t>(vector(a[6], "axes", bit(kInt32), g.pairs));
        g.interleaved = truth(a[11]);
        const auto *cache = cached ? static_cast<const Spkv2KvCacheI8 *>(address(a[12])) : nullptr;
        void *stream = handle(a[17]);
        return unlocked([&] { return entries.rotate(cache, &g, stream); });
    });
}

// (kind, x, weight, q, scale, residual, residual_out, eps, stream)
PyObject *rows_f8(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<9>(count, [&]() -> int {
        Spkv2RowsF8 g{};
        g.kind = small_number(a[0]);
        Tensor q = first_look(a[3], "q", 2, "not two-dimensional");
        g.rows = q.shape[0], g.cols = q.shape[1];
        rows_settled(q, bit(kF8), g.rows, g.cols);
        g.q = as<uint8_t>(q), g.q_stride = q.stride[0];
        const Tensor x = rows_of(a[1], "x", kFloats, g.rows, g.kind == SPKV2_F8_GATE ? 2 * g.cols : g.cols);
        g.x = x.p, g.x_stride = x.stride[0], g.dtype = x.code;
        if (given(a[2])) {
            const Tensor w = vector(a[2], "weight", bit(x.code) | bit(kFp32), g.cols);
            g.weight = w.p, g.weight_dtype = w.code;
        }
        if (given(a[5])) {
            const Tensor r = rows_of(a[5], "residual", bit(x.code), g.rows, g.cols);
            g.residual = r.p, g.residual_stride = r.stride[0];
        }
        if (given(a[6])) {
            const Tensor r = rows_of(a[6], "residual_out", bit(x.code), g.rows, g.cols);
            g.residual_out = r.p, g.residual_out_stride = r.stride[0];
        }
        const Tensor s = rows_of(a[4], "scale", bit(kFp32), g.rows, blocks(g.cols));
        g.scale = as<float>(s), g.scale_stride = s.stride[0];
        g.eps = real(a[7]);
        void *stream = handle(a[8]);
        return unlocked([&] { return entries.rows(&g, stream); });
    });
}

// (q, scale, out, stream)
PyObject *dequantize_f8(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<4>(count, [&]() -> int {
        Spkv2DequantizeF8 g{};
        Tensor q = first_look(a[0], "q", 2, "not two-dimensional");
        g.rows = q.shape[0], g.cols = q.shape[1];
        g.q = as<uint8_t>(rows_settled(q, bit(kF8), g.rows, g.cols)), g.q_stride = q.stride[0];
        const Tensor s = rows_of(a[1], "scale", bit(kFp32), g.rows, blocks(g.cols));
        g.scale = as<float>(s), g.scale_stride = s.stride[0];
        const Tensor out = rows_of(a[2], "out", kFloats, g.rows, g.cols);
        g.out = out.p, g.out_stride = out.stride[0], g.dtype = out.code;
        void *stream = handle(a[3]);
        return unlocked([&] { return entries.dequantize(&g, stream); });
    });
}

// (a, a_scale, b, b_scale, out, bias, stream)
PyObject *matmul_f8(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<7>(count, [&]() -> int {
        Spkv2MatmulF8 g{};
        Tensor x = first_look(a[0], "a", 2, "not two-dimensional"), w = first_look(a[2], "b", 2, "not two-dimensional");
        g.m = x.shape[0], g.k = x.shape[1], g.n = w.shape[0];
        g.a = as<uint8_t>(rows_settled(x, bit(kF8), g.m, g.k)), g.a_stride = x.stride[0];
        g.b = as<uint8_t>(rows_settled(w, bit(kF8), g.n, g.k)), g.b_stride = w.stride[0];
        const Tensor sa = rows_of(a[1], "a_scale", bit(kFp32), g.m, blocks(g.k)), sb = rows_of(a[3], "b_scale", bit(kFp32), blocks(g.n), blocks(g.k));
        g.a_scale = as<float>(sa), g.a_scale_stride = sa.stride[0];
        g.b_scale = as<float>(sb), g.b_scale_stride = sb.stride[0];
        const Tensor out = rows_of(a[4], "out", kFloats, g.m, g.n);
        g.out = out.p, g.out_stride = out.stride[0], g.dtype = out.code;
        if (given(a[5])) g.bias = as<float>(vector(a[5], "bias", bit(kFp32), g.n));
        void *stream = handle(a[6]);
        return unlocked([&] { return entries.matmul(&g, stream); });
    });
}

// [experts, rows, cols], experts and rows any distance apart
Tensor weights(PyObject *o, const char *name, unsigned allowed, int64_t experts, int64_t rows, int64_t cols) {
    Tensor t = first_look(o, name, 3, "not three-dimensional");
    const int64_t shape[] = {experts, rows, cols};
    settle(t, allowed, shape);
    if (t.stride[2] != 1 && cols > 1) refuse(name, "its last axis is not contiguous");
    return t;
}

// (a, a_scale, b, b_scale, offsets, out, order, per_token, bias, stream)
PyObject *matmul_f8_experts(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<10>(count, [&]() -> int {
        Spkv2MatmulF8Experts e{};
        Spkv2MatmulF8 &g = e.product;
        Tensor x = first_look(a[0], "a", 2, "not two-dimensional"), out = first_look(a[5], "out", 2, "not two-dimensional");
        const Tensor look = first_look(a[2], "b", 3, "not three-dimensional");
        e.a_rows = x.shape[0], g.k = x.shape[1], g.m = out.shape[0], g.n = look.shape[1];
        e.experts = as_int32(look.shape[0]);
        g.a = as<uint8_t>(rows_settled(x, bit(kF8), e.a_rows, g.k)), g.a_stride = x.stride[0];
        const Tensor w = weights(a[2], "b", bit(kF8), e.experts, g.n, g.k), sb = weights(a[3], "b_scale", bit(kFp32), e.experts, blocks(g.n), blocks(g.k));
        g.b = as<uint8_t>(w), e.b_expert_stride = w.stride[0], g.b_stride = w.stride[1];
        g.b_scale = as<float>(sb), e.b_scale_expert_stride = sb.stride[0], g.b_scale_stride = sb.stride[1];
        const Tensor sa = rows_of(a[1], "a_scale", bit(kFp32), e.a_rows, blocks(g.k));
        g.a_scale = as<float>(sa), g.a_scale_stride = sa.stride[0];
        rows_settled(out, kFloats, g.m, g.n);
        g.out = out.p, g.out_stride = out.stride[0], g.dtype = out.code;
        e.offsets = as<int32_t>(vector(a[4], "offsets", bit(kInt32), e.experts + int64_t(1)));
        if (given(a[6])) e.order = as<int32_t>(vector(a[6], "order", bit(kInt32), g.m));
        e.per_token = small_number(a[7]);
        if (given(a[8])) g.bias = as<float>(matrix(a[8], "bias", bit(kFp32), e.experts, g.n));
        void *stream = handle(a[9]);
        return unlocked([&] { return entries.experts(&e, stream); });
    });
}

// (experts, offsets, order, place, stream)
PyObject *sort_tokens(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<5>(count, [&]() -> int {
        Spkv2SortTokens g{};
        Tensor ids = first_look(a[0], "experts", 2, "not two-dimensional");
        g.tokens = ids.shape[0], g.per_token = as_int32(ids.shape[1]);
        ids = matrix(a[0], "experts", bit(kInt32) | bit(kInt64), g.tokens, g.per_token);
        g.ids = ids.p, g.wide_ids = ids.code == kInt64;
        Tensor offsets = first_look(a[1], "offsets", 1, "not one-dimensional");
        g.offsets = as<int32_t>(vector_settled(offsets, bit(kInt32), offsets.shape[0]));
        g.experts = as_int32(offsets.shape[0] - 1);
        g.order = as<int32_t>(vector(a[2], "order", bit(kInt32), g.tokens * g.per_token));
        g.place = as<int32_t>(matrix(a[3], "place", bit(kInt32), g.tokens, g.per_token));
        void *stream = handle(a[4]);
        return unlocked([&] { return entries.sort(&g, stream); });
    });
}

// (y, place, weights, out, residual, stream)
PyObject *combine(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<6>(count, [&]() -> int {
        Spkv2Combine g{};
        Tensor y = first_look(a[0], "y", 2, "not two-dimensional"), place = first_look(a[1], "place", 2, "not two-dimensional");
        g.rows = y.shape[0], g.cols = y.shape[1], g.dtype = y.code;
        g.y = rows_settled(y, kFloats, g.rows, g.cols).p, g.y_stride = y.stride[0];
        g.tokens = place.shape[0], g.per_token = as_int32(place.shape[1]);
        rows_settled(place, bit(kInt32), g.tokens, g.per_token);
        if (place.stride[0] != g.per_token && g.tokens > 1) refuse("place", "not contiguous");
        g.place = as<int32_t>(place);
        g.weights = as<float>(matrix(a[2], "weights", bit(kFp32), g.tokens, g.per_token));
        const Tensor out = rows_of(a[3], "out", bit(y.code), g.tokens, g.cols);
        g.out = out.p, g.out_stride = out.stride[0];
        if (given(a[4])) {
            const Tensor r = rows_of(a[4], "residual", bit(y.code), g.tokens, g.cols);
            g.residual = r.p, g.residual_stride = r.stride[0];
        }
        void *stream = handle(a[5]);
        return unlocked([&] { return entries.combine(&g, stream); });
    });
}

// (cache, kv_heads, head_dim, k, v, slots, stream): cache the address of its struct
PyObject *kv_write(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<7>(count, [&]() -> int {
        Spkv2KvWrite g{};
        const int64_t heads = number(a[1]), dim = number(a[2]);
        Tensor k = first_look(a[3], "k", 3, "not [tokens, kv_heads, head_dim]");
        g.tokens = k.shape[0], g.dtype = k.code;
        g.k = heads_settled(k, kFloats, g.tokens, heads, dim).p, g.k_stride = k.stride[0];
        const Tensor v = heads_of(a[4], "v", bit(k.code), g.tokens, heads, dim);
        g.v = v.p, g.v_stride = v.stride[0];
        g.slots = as<int64_t>(vector(a[5], "slots", bit(kInt64), g.tokens));
        const auto *cache = static_cast<const Spkv2KvCacheI8 *>(address(a[0]));
        void *stream = handle(a[6]);
        return unlocked([&] { return entries.kv_write(cache, &g, stream); });
    });
}

// (cache, kv_heads, head_dim, table, first, offsets, k, v, stream)
PyObject *kv_read(PyObject *, PyObject *const *a, Py_ssize_t count) {
    return guarded<9>(count, [&]() -> int {
        Spkv2KvRead g{};
        const int64_t heads = number(a[1]), dim = number(a[2]);
        Tensor table = first_look(a[3], "table", 2, "not two-dimensional");
        const int64_t sequences = table.shape[0];
        rows_settled(table, bit(kInt32), sequences, table.shape[1]);
        if (table.stride[0] != table.shape[1] && sequences > 1) refuse("table", "not contiguous");
        g.table = as<int32_t>(table);
        g.sequences = as_int32(sequences), g.table_width = as_int32(table.shape[1]);
        if (given(a[4])) g.first = as<int32_t>(vector(a[4], "first", bit(kInt32), sequences));
        g.offsets = as<int32_t>(vector(a[5], "offsets", bit(kInt32), sequences + 1));
        Tensor k = first_look(a[6], "k", 3, "not [tokens, kv_heads, head_dim]");
        g.tokens = k.shape[0], g.dtype = k.code;
        g.k = heads_settled(k, kFloats, g.tokens, heads, dim).p, g.k_stride = k.stride[0];
        const Tensor v = heads_of(a[7], "v", bit(k.code), g.tokens, heads, dim);
        g.v = v.p, g.v_stride = v.stride[0];
        const auto *cache = static_cast<const Spkv2KvCacheI8 *>(address(a[0]));
        void *stream = handle(a[8]);
        return unlocked([&] { return entries.kv_read(cache, &g, stream); });
    });
}

// (codes, code_of, range_error, addresses): the dict of types, what looks one up that it lacks, struct.error, the entry
// points' addresses in the order of Entries
PyObject *bind(PyObject *, PyObject *args) {
    PyObject *d, *f, *r, *list;
    if (!PyArg_ParseTuple(args, "O!OOO!", &PyDict_Type, &d, &f, &r, &PyTuple_Type, &list)) return nullptr;
    void *p[9];
    static_assert(sizeof(p) == sizeof(entries), "an address for each entry");
    if (PyTuple_GET_SIZE(list) != 9) {
        PyErr_SetString(PyExc_TypeError, "expected nine addresses");
        return nullptr;
    }
    for (int i = 0; i < 9; i++) {
        p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(list, i));
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is 0");
            return nullptr;
        }
    }
    __builtin_memcpy(&entries, p, sizeof(p));
    Py_INCREF(d), Py_INCREF(f), Py_INCREF(r);
    Py_XDECREF(codes), Py_XDECREF(code_of), Py_XDECREF(range_error);
    codes = d, code_of = f, range_error = r;
    Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<rotate>("rotate"),
                         method<rows_f8>("rows_f8"),
                         method<dequantize_f8>("dequantize_f8"),
                         method<matmul_f8>("matmul_f8"),
                         method<matmul_f8_experts>("matmul_f8_experts"),
                         method<sort_tokens>("sort_tokens"),
                         method<combine>("combine"),
                         method<kv_write>("kv_write"),
                         method<kv_read>("kv_read"),
                         {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decoder_calls() {
    s_shape = PyUnicode_InternFromString("shape");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_stride = PyUnicode_InternFromString("stride");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    if (!s_shape || !s_dtype || !s_is_cuda || !s_stride || !s_data_ptr) return nullptr;
    return PyModule_Create(&module);
}
