// Native call path of the Python operators: one C function per operator that checks its tensors,
// allocates the output when the caller gave none, and calls the C ABI on the current stream.
//
// A decode step is a few hundred calls of 2-8 us of device work each, so what a call costs on the
// host is what an eager step takes.  Through ctypes a call cost 9.7 us (14.1 with an allocated
// output) on the B200 box's host: 3.2 us for the Stream object behind torch.cuda.current_stream(),
// 2.5 for torch.empty, about 2 for ctypes' eleven conversions, the rest attribute reads.  Here the
// stream, the pointers and the shapes are read from the C++ objects and the driver's launch (2 us)
// is what is left.  The library's functions come from the handle that _lib.py opened, so that there
// is one library whatever path it was loaded from.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <dlfcn.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>

#include "../../include/miori_b200.h"

namespace {

constexpr int MAX_ARGS = 15;
PyObject* g_error = nullptr;  // _lib.MioriError

#define MIORI_ENTRIES(X)                                                                         \
    X(last_error) X(gemv4) X(gemv8) X(dequant4_rowmajor) X(dequant8_rowmajor) X(dequant4_cache)  \
    X(cache_bytes) X(gemm_bf16_cache_ws) X(gemm_bf16_strided) X(gemv_bf16_cache) X(linear4)      \
    X(rmsnorm) X(post_norm_add) X(silu_mul) X(embed8) X(argmax) X(gemv4_rmsnorm)                 \
    X(gemv8_rmsnorm) X(gemv4_silu) X(gemv4_post_norm_add) X(gemv4_rmsnorm_silu) X(page_slots)    \
    X(rope_kv) X(attention_paged) X(attention_prompt) X(quant_fp8) X(gemm_fp8) X(moe4) X(moe_fp8)

struct Abi {
#define X(name) decltype(&miori_##name) name;
    MIORI_ENTRIES(X)
#undef X
} abi;

struct Failed {};  // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Failed();
}

// Arguments of a METH_FASTCALL | METH_KEYWORDS call by position: v[i] is null where none was given.
struct Args {
    PyObject* v[MAX_ARGS] = {};
    Args(const char* fn, const char* const* names, int count, int required, PyObject* const* args, Py_ssize_t n,
         PyObject* kw) {
        if (n > count) raise(PyExc_TypeError, "%s() takes at most %d arguments (%zd given)", fn, count, n);
        for (Py_ssize_t i = 0; i < n; ++i) v[i] = args[i];
        const Py_ssize_t nk = kw ? PyTuple_GET_SIZE(kw) : 0;
        for (Py_ssize_t k = 0; k < nk; ++k) {
            Py_ssize_t len = 0;
            const char* key = PyUnicode_AsUTF8AndSize(PyTuple_GET_ITEM(kw, k), &len);
            if (!key) throw Failed();
            int at = -1;
            for (int i = 0; i < count; ++i)
                if (names[i][0] == key[0] && std::strcmp(names[i], key) == 0) { at = i; break; }
            if (at < 0) raise(PyExc_TypeError, "%s() got an unexpected keyword argument '%s'", fn, key);
            if (v[at]) raise(PyExc_TypeError, "%s() got multiple values for argument '%s'", fn, key);
            v[at] = args[n + k];
        }
        for (int i = 0; i < required; ++i)
            if (!v[i]) raise(PyExc_TypeError, "%s() missing required argument '%s'", fn, names[i]);
    }
    bool given(int i) const { return v[i] && v[i] != Py_None; }
    const at::Tensor& tensor(int i) const {
        if (!v[i] || !THPVariable_Check(v[i])) raise(PyExc_TypeError, "argument %d: a tensor is expected", i + 1);
        return THPVariable_Unpack(v[i]);
    }
    uint32_t u32(int i, uint32_t dflt) const {
        if (!v[i]) return dflt;
        const unsigned long r = PyLong_AsUnsignedLongMask(v[i]);
        if (r == (unsigned long)-1 && PyErr_Occurred()) throw Failed();
        return (uint32_t)r;
    }
    float f32(int i) const {
        if (PyFloat_CheckExact(v[i])) return (float)PyFloat_AS_DOUBLE(v[i]);
        PyObject* f = PyNumber_Float(v[i]);  // whatever float() takes
        if (!f) throw Failed();
        const double d = PyFloat_AS_DOUBLE(f);
        Py_DECREF(f);
        return (float)d;
    }
};

void need_cuda(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts) {
        if (!t->is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
        if (!t->is_contiguous()) raise(PyExc_ValueError, "miori_b200 ops need contiguous tensors");
    }
}
void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }
at::Tensor empty(at::IntArrayRef shape, at::ScalarType dt, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(shape, dt, like.device(), std::nullopt));
}
at::ScalarType out_type(uint32_t flags) { return flags & MIORI_OUT_BF16 ? at::kBFloat16 : at::kFloat; }

// The output: the caller's object (returned as it is) or a new tensor.
struct Out {
    PyObject* given = nullptr;
    at::Tensor made;
    void* ptr() const { return given ? THPVariable_Unpack(given).data_ptr() : made.data_ptr(); }
    PyObject* result() {
        if (given) return Py_NewRef(given);
        return THPVariable_Wrap(std::move(made));
    }
};
// Memory of the caller's that a kernel writes: on a GPU or pinned, contiguous, large enough.
void need_room(const at::Tensor& t, const char* what, size_t bytes) {
    if (!t.is_cuda() && !t.is_pinned()) raise(PyExc_ValueError, "%s: a CUDA tensor is expected", what);
    if (!t.is_contiguous()) raise(PyExc_ValueError, "%s: a contiguous tensor is expected", what);
    if ((size_t)t.numel() * t.element_size() < bytes)
        raise(PyExc_ValueError, "%s: %zu bytes needed, the tensor has %zu", what, bytes, (size_t)t.numel() * t.element_size());
}
// `need`: what the kernel writes, where that is not the type of a new tensor.
Out output(const Args& a, int i, at::IntArrayRef shape, at::ScalarType dt, const at::Tensor& like,
           at::ScalarType need = at::ScalarType::Undefined) {
    Out o;
    if (a.given(i)) {
        size_t bytes = c10::elementSize(need == at::ScalarType::Undefined ? dt : need);
        for (const int64_t n : shape) bytes *= (size_t)n;
        need_room(a.tensor(i), "out", bytes);
        o.given = a.v[i];
    } else {
        o.made = empty(shape, dt, like);
    }
    return o;
}

// Call into the library without the interpreter lock (a launch may block on a full queue).  The arguments
// are evaluated before, under the lock: reading a tensor's pointer may throw.
template <class... P, class... A>
void call(int (*fn)(P...), A... args) {
    PyThreadState* ts = PyEval_SaveThread();
    const int rc = fn(static_cast<P>(args)...);
    PyEval_RestoreThread(ts);
    if (rc != MIORI_OK) {
        PyObject* exc = PyObject_CallFunction(g_error, "is", rc, abi.last_error());
        if (exc) {
            PyErr_SetObject(g_error, exc);
            Py_DECREF(exc);
        }
        throw Failed();
    }
}

template <class F>
PyObject* guarded(F body) {
    try {
        return body();
    } catch (const Failed&) {
    } catch (...) {  // torch's own, as its operators raise them: out of memory, no storage, a missing dimension
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

#define OP(name, required, ...)                                                                    \
    const char* const name##_names[] = {__VA_ARGS__};                                              \
    PyObject* name##_body(const Args& a);                                                          \
    PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {            \
        constexpr int count = sizeof(name##_names) / sizeof(char*);                                \
        static_assert(count <= MAX_ARGS, "");                                                      \
        return guarded([&] { return name##_body(Args(#name, name##_names, count, required, args, n, kw)); }); \
    }                                                                                              \
    PyObject* name##_body(const Args& a)

// Rows and columns of the activations: [K] counts as [1][K].
void rows_of(const at::Tensor& x, int64_t& M, int64_t& K) {
    if (x.dim() == 1) {
        M = 1, K = x.size(0);
    } else if (x.dim() == 2) {
        M = x.size(0), K = x.size(1);
    } else {
        raise(PyExc_ValueError, "activations of one or two dimensions expected");
    }
}
void check_words(const at::Tensor& q, int64_t per_word, int64_t K) {
    if (q.size(1) * per_word != K)
        raise(PyExc_ValueError, "q has %lld words per row, expected %lld", (long long)q.size(1), (long long)(K / per_word));
}

PyObject* gemv(const Args& a, decltype(abi.gemv4) fn, int64_t per_word) {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &x = a.tensor(3);
    need_cuda({&q, &s, &b, &x});
    int64_t M, K;
    rows_of(x, M, K);
    check_words(q, per_word, K);
    const int64_t N = q.size(0);
    const uint32_t group = a.u32(4, 32), flags = a.u32(5, 0);
    Out y = output(a, 6, {M, N}, out_type(flags), x);
    call(fn, q.data_ptr(), s.data_ptr(), b.data_ptr(), x.data_ptr(), y.ptr(), N, K, M, group, flags, stream());
    return y.result();
}
OP(gemv4, 4, "q", "s", "b", "x", "group", "flags", "out") { return gemv(a, abi.gemv4, 8); }
OP(gemv8, 4, "q", "s", "b", "x", "group", "flags", "out") { return gemv(a, abi.gemv8, 4); }

PyObject* dequant(const Args& a, decltype(abi.dequant4_rowmajor) fn, int64_t per_word, bool flat) {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2);
    need_cuda({&q, &s, &b});
    const int64_t N = q.size(0), K = q.size(1) * per_word;
    const uint32_t group = a.u32(3, 32);
    const int64_t flat_shape[1] = {(int64_t)(abi.cache_bytes(N, K) / 2)}, shape[2] = {N, K};
    Out o = output(a, 4, flat ? at::IntArrayRef(flat_shape) : at::IntArrayRef(shape), at::kBFloat16, q);
    call(fn, q.data_ptr(), s.data_ptr(), b.data_ptr(), o.ptr(), N, K, group, stream());
    return o.result();
}
OP(dequant4_rowmajor, 3, "q", "s", "b", "group", "out") { return dequant(a, abi.dequant4_rowmajor, 8, false); }
OP(dequant8_rowmajor, 3, "q", "s", "b", "group", "out") { return dequant(a, abi.dequant8_rowmajor, 4, false); }
OP(dequant4_cache, 3, "q", "s", "b", "group", "out") { return dequant(a, abi.dequant4_cache, 8, true); }

// Pointer and bytes of an optional workspace tensor.
void workspace(const Args& a, int i, void*& p, size_t& bytes) {
    p = nullptr, bytes = 0;
    if (!a.given(i)) return;
    const at::Tensor& w = a.tensor(i);
    need_room(w, "workspace", 0);
    p = w.data_ptr();
    bytes = (size_t)w.numel() * w.element_size();
}

OP(gemm_bf16_cache, 3, "A", "cache", "N", "flags", "out", "workspace") {
    const at::Tensor &A = a.tensor(0), &cache = a.tensor(1);
    need_cuda({&A, &cache});
    if (A.dim() != 2) raise(PyExc_ValueError, "gemm_bf16_cache: A [M][K] expected");
    const int64_t M = A.size(0), K = A.size(1), N = a.u32(2, 0);
    const uint32_t flags = a.u32(3, 0);
    Out c = output(a, 4, {M, N}, out_type(flags), A);
    void* wp;
    size_t wb;
    workspace(a, 5, wp, wb);
    call(abi.gemm_bf16_cache_ws, A.data_ptr(), cache.data_ptr(), c.ptr(), M, N, K, flags, wp, wb, stream());
    return c.result();
}

OP(gemm_bf16_strided, 2, "A", "B", "flags", "out") {
    const at::Tensor &A = a.tensor(0), &B = a.tensor(1);
    if (!A.is_cuda() || !B.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    if (A.scalar_type() != at::kBFloat16 || B.scalar_type() != at::kBFloat16)
        raise(PyExc_TypeError, "gemm_bf16_strided: bf16 operands expected");
    if (A.dim() != 2 || B.dim() != 2 || B.size(1) != A.size(1) || A.stride(1) != 1 || B.stride(1) != 1)
        raise(PyExc_ValueError, "gemm_bf16_strided: A [M][K] and B [N][K] with contiguous rows expected");
    const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
    const uint32_t flags = a.u32(2, 0);
    const at::ScalarType dt = out_type(flags);
    Out o;  // rows of a caller's output may lie apart
    if (a.given(3)) a.tensor(3), o.given = a.v[3];
    else o.made = empty({M, N}, dt, A);
    const at::Tensor& c = o.given ? THPVariable_Unpack(o.given) : o.made;
    if (!c.is_cuda() && !c.is_pinned()) raise(PyExc_ValueError, "out: a CUDA tensor is expected");
    if (c.scalar_type() != dt || c.dim() != 2 || c.size(0) != M || c.size(1) != N || c.stride(1) != 1)
        raise(PyExc_ValueError, "gemm_bf16_strided: bad output tensor");
    call(abi.gemm_bf16_strided, A.data_ptr(), A.stride(0), B.data_ptr(), B.stride(0), c.data_ptr(), c.stride(0), M, N,
         K, flags, stream());
    return o.result();
}

OP(gemv_bf16_cache, 3, "x", "cache", "N", "flags", "out") {
    const at::Tensor &x = a.tensor(0), &cache = a.tensor(1);
    need_cuda({&x, &cache});
    if (x.dim() != 2) raise(PyExc_ValueError, "gemv_bf16_cache: x [M][K] expected");
    const int64_t M = x.size(0), K = x.size(1), N = a.u32(2, 0);
    const uint32_t flags = a.u32(3, 0);
    Out y = output(a, 4, {M, N}, out_type(flags), x);
    call(abi.gemv_bf16_cache, x.data_ptr(), cache.data_ptr(), y.ptr(), M, N, K, flags, stream());
    return y.result();
}

OP(linear4, 5, "q", "s", "b", "cache", "x", "group", "flags", "out", "workspace") {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &x = a.tensor(4);
    need_cuda({&q, &s, &b, &x});
    if (x.dim() != 2) raise(PyExc_ValueError, "linear4: x [M][K] expected");
    const int64_t M = x.size(0), K = x.size(1), N = q.size(0);
    const void* cache = a.given(3) ? a.tensor(3).data_ptr() : nullptr;
    const uint32_t group = a.u32(5, 32), flags = a.u32(6, 0);
    Out y = output(a, 7, {M, N}, at::kFloat, x, out_type(flags));
    void* wp;
    size_t wb;
    workspace(a, 8, wp, wb);
    call(abi.linear4, q.data_ptr(), s.data_ptr(), b.data_ptr(), cache, x.data_ptr(), y.ptr(), N, K, M, group, flags,
         wp, wb, stream());
    return y.result();
}

OP(rmsnorm, 3, "x", "gamma", "eps", "flags", "out") {
    const at::Tensor &x = a.tensor(0), &gamma = a.tensor(1);
    need_cuda({&x, &gamma});
    if (x.dim() != 2) raise(PyExc_ValueError, "rmsnorm: x [rows][n] expected");
    const int64_t rows = x.size(0), n = x.size(1);
    const float eps = a.f32(2);
    const uint32_t flags = a.u32(3, 0);
    Out y = output(a, 4, {rows, n}, at::kBFloat16, x);
    call(abi.rmsnorm, x.data_ptr(), gamma.data_ptr(), y.ptr(), rows, n, eps, flags, stream());
    return y.result();
}

OP(post_norm_add, 4, "x", "src", "gamma", "eps", "flags", "out") {
    const at::Tensor &x = a.tensor(0), &src = a.tensor(1), &gamma = a.tensor(2);
    need_cuda({&x, &src, &gamma});
    if (x.dim() != 2) raise(PyExc_ValueError, "post_norm_add: x [rows][n] expected");
    const int64_t rows = x.size(0), n = x.size(1);
    const float eps = a.f32(3);
    const uint32_t flags = a.u32(4, 0);
    Out o = output(a, 5, {rows, n}, x.scalar_type(), x, at::kFloat);
    call(abi.post_norm_add, x.data_ptr(), src.data_ptr(), gamma.data_ptr(), o.ptr(), rows, n, eps, flags, stream());
    return o.result();
}

OP(silu_mul, 2, "gate", "up", "flags", "out") {
    const at::Tensor &gate = a.tensor(0), &up = a.tensor(1);
    need_cuda({&gate, &up});
    const uint32_t flags = a.u32(2, 0);
    Out o = output(a, 3, gate.sizes(), at::kBFloat16, gate);
    call(abi.silu_mul, gate.data_ptr(), up.data_ptr(), o.ptr(), gate.numel(), flags, stream());
    return o.result();
}

OP(embed8, 4, "q", "s", "b", "tokens", "group", "flags", "out") {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &tokens = a.tensor(3);
    need_cuda({&q, &s, &b, &tokens});
    const int64_t rows = q.size(0), K = q.size(1) * 4, T = tokens.numel();
    const uint32_t group = a.u32(4, 32), flags = a.u32(5, 0);
    Out o = output(a, 6, {T, K}, at::kBFloat16, q);
    call(abi.embed8, q.data_ptr(), s.data_ptr(), b.data_ptr(), tokens.data_ptr(), o.ptr(), T, rows, K, group, flags,
         stream());
    return o.result();
}

OP(argmax, 1, "v", "flags") {
    const at::Tensor& v = a.tensor(0);
    need_cuda({&v});
    const uint32_t flags = a.u32(1, 0) | (v.scalar_type() == at::kBFloat16 ? MIORI_OUT_BF16 : 0u);
    at::Tensor idx = empty({1}, at::kInt, v), val = empty({1}, at::kFloat, v);
    call(abi.argmax, v.data_ptr(), v.numel(), flags, idx.data_ptr(), val.data_ptr(), stream());
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw Failed();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(idx)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(val)));
    return pair;
}

void need_f32(const at::Tensor& x) {
    if (x.scalar_type() != at::kFloat) raise(PyExc_TypeError, "the fused norm takes fp32 activations");
}
PyObject* gemv_rmsnorm(const Args& a, decltype(abi.gemv4_rmsnorm) fn) {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &x = a.tensor(3), &gamma = a.tensor(4);
    need_cuda({&q, &s, &b, &x, &gamma});
    need_f32(x);
    int64_t M, K;
    rows_of(x, M, K);
    const int64_t N = q.size(0);
    const float eps = a.f32(5);
    const uint32_t group = a.u32(6, 32), flags = a.u32(7, 0);
    Out y = output(a, 8, {M, N}, out_type(flags), x);
    call(fn, q.data_ptr(), s.data_ptr(), b.data_ptr(), x.data_ptr(), gamma.data_ptr(), eps, y.ptr(), N, K, M, group,
         flags, stream());
    return y.result();
}
OP(gemv4_rmsnorm, 6, "q", "s", "b", "x", "gamma", "eps", "group", "flags", "out") { return gemv_rmsnorm(a, abi.gemv4_rmsnorm); }
OP(gemv8_rmsnorm, 6, "q", "s", "b", "x", "gamma", "eps", "group", "flags", "out") { return gemv_rmsnorm(a, abi.gemv8_rmsnorm); }

OP(gemv4_silu, 4, "q", "s", "b", "x", "group", "flags", "out") {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &x = a.tensor(3);
    need_cuda({&q, &s, &b, &x});
    int64_t M, K;
    rows_of(x, M, K);
    check_words(q, 8, K);
    const int64_t N = q.size(0);
    const uint32_t group = a.u32(4, 32), flags = a.u32(5, 0);
    Out y = output(a, 6, {M, N / 2}, at::kBFloat16, x);
    call(abi.gemv4_silu, q.data_ptr(), s.data_ptr(), b.data_ptr(), x.data_ptr(), y.ptr(), N, K, M, group, flags,
         stream());
    return y.result();
}

OP(gemv4_post_norm_add, 8, "q", "s", "b", "x", "residual", "gamma", "eps", "counter", "group", "flags", "out") {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &x = a.tensor(3), &residual = a.tensor(4),
                     &gamma = a.tensor(5), &counter = a.tensor(7);
    need_cuda({&q, &s, &b, &x, &residual, &gamma, &counter});
    int64_t M, K;
    rows_of(x, M, K);
    check_words(q, 8, K);
    const int64_t N = q.size(0);
    if (residual.scalar_type() != at::kFloat || residual.numel() != M * N)
        raise(PyExc_ValueError, "residual: fp32 [M][N] expected");
    const float eps = a.f32(6);
    const uint32_t group = a.u32(8, 32), flags = a.u32(9, 0);
    Out o = output(a, 10, {M, N}, at::kFloat, x);
    call(abi.gemv4_post_norm_add, q.data_ptr(), s.data_ptr(), b.data_ptr(), x.data_ptr(), residual.data_ptr(),
         gamma.data_ptr(), eps, counter.data_ptr(), o.ptr(), N, K, M, group, flags, stream());
    return o.result();
}

OP(gemv4_rmsnorm_silu, 6, "q", "s", "b", "x", "gamma", "eps", "group", "flags", "out") {
    const at::Tensor &q = a.tensor(0), &s = a.tensor(1), &b = a.tensor(2), &x = a.tensor(3), &gamma = a.tensor(4);
    need_cuda({&q, &s, &b, &x, &gamma});
    need_f32(x);
    int64_t M, K;
    rows_of(x, M, K);
    const int64_t N = q.size(0);
    const float eps = a.f32(5);
    const uint32_t group = a.u32(6, 32), flags = a.u32(7, 0);
    Out y = output(a, 8, {M, N / 2}, at::kBFloat16, x);
    call(abi.gemv4_rmsnorm_silu, q.data_ptr(), s.data_ptr(), b.data_ptr(), x.data_ptr(), gamma.data_ptr(), eps,
         y.ptr(), N, K, M, group, flags, stream());
    return y.result();
}

// Whole numbers of a step's plan: int32, on the GPU, contiguous.
const int32_t* ints(const at::Tensor& t, const char* what, int64_t numel) {
    if (!t.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    if (t.scalar_type() != at::kInt) raise(PyExc_TypeError, "%s: an int32 tensor is expected", what);
    if (!t.is_contiguous()) raise(PyExc_ValueError, "miori_b200 ops need contiguous tensors");
    if (numel >= 0 && t.numel() != numel) raise(PyExc_ValueError, "%s: %lld numbers expected, got %lld", what, (long long)numel, (long long)t.numel());
    return static_cast<const int32_t*>(t.data_ptr());
}
// A bf16 tensor of `dims` dimensions whose last one is contiguous; the others lie as they like.
void need_heads(const at::Tensor& t, const char* what, int64_t dims) {
    if (!t.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    if (t.scalar_type() != at::kBFloat16) raise(PyExc_TypeError, "%s: a bf16 tensor is expected", what);
    if (t.dim() != dims) raise(PyExc_ValueError, "%s: %lld dimensions expected, got %lld", what, (long long)dims, (long long)t.dim());
    if (t.size(dims - 1) != 1 && t.stride(dims - 1) != 1) raise(PyExc_ValueError, "%s: the last dimension must be contiguous", what);
}
// A stride, or where there is only one step to take any that passes the library's checks.
int64_t step(const at::Tensor& t, int64_t d) { return t.size(d) == 1 ? t.size(t.dim() - 1) : t.stride(d); }

// A contiguous piece of `whole` as a tensor of its own (several small outputs of one allocation: each of its own costs a microsecond).
at::Tensor piece(const at::Tensor& whole, int64_t offset, int64_t numel) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({numel});
    return t;
}
PyObject* tuple_of(std::initializer_list<at::Tensor*> ts) {
    PyObject* all = PyTuple_New((Py_ssize_t)ts.size());
    if (!all) throw Failed();
    Py_ssize_t i = 0;
    for (at::Tensor* t : ts) PyTuple_SET_ITEM(all, i++, THPVariable_Wrap(std::move(*t)));
    return all;
}

OP(page_slots, 7, "held", "new", "table", "pool", "taken", "page", "tokens", "flags") {
    const at::Tensor &held = a.tensor(0), &fresh = a.tensor(1), &table = a.tensor(2), &pool = a.tensor(3), &taken = a.tensor(4);
    const int64_t R = held.numel();
    const int32_t *hp = ints(held, "held", -1), *fp = ints(fresh, "new", R), *tp = ints(table, "table", -1), *pp = ints(pool, "pool", -1),
                  *kp = ints(taken, "taken", 1);
    if (table.dim() != 2 || table.size(0) != R) raise(PyExc_ValueError, "table: [%lld][width] expected", (long long)R);
    const uint32_t page = a.u32(5, 0), T = a.u32(6, 0), flags = a.u32(7, 0);
    auto room = [](int64_t n) { return (n + 3) / 4 * 4; };  // pieces begin on 16-byte boundaries
    const int64_t at_positions = room(T), at_cu = at_positions + room(T), at_after = at_cu + room(R + 1), at_taken = at_after + room(R);
    const at::Tensor whole = empty({at_taken + 1}, at::kInt, held);
    at::Tensor slots = piece(whole, 0, T), positions = piece(whole, at_positions, T), cu = piece(whole, at_cu, R + 1), after = piece(whole, at_after, R),
               taken_after = piece(whole, at_taken, 1);
    auto out = [](at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
    call(abi.page_slots, hp, fp, const_cast<int32_t*>(tp), pp, kp, out(slots), out(positions), out(cu), out(after), out(taken_after), R,
         table.size(1), page, pool.numel(), T, flags, stream());
    return tuple_of({&slots, &positions, &cu, &after, &taken_after});
}

OP(rope_kv, 7, "qkv", "turns", "positions", "slots", "k_cache", "v_cache", "heads", "axes", "gamma_q", "gamma_k", "eps", "flags", "out") {
    const at::Tensor &qkv = a.tensor(0), &turns = a.tensor(1), &positions = a.tensor(2), &slots = a.tensor(3), &k = a.tensor(4), &v = a.tensor(5);
    if (!qkv.is_cuda() || !turns.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    const bool fp32 = qkv.scalar_type() == at::kFloat;
    if (!fp32 && qkv.scalar_type() != at::kBFloat16) raise(PyExc_TypeError, "qkv: an fp32 or bf16 tensor is expected");
    if (turns.scalar_type() != at::kLong || !turns.is_contiguous()) raise(PyExc_TypeError, "turns: a contiguous int64 tensor is expected");
    need_heads(k, "k_cache", 4);
    need_heads(v, "v_cache", 4);
    if (k.sizes() != v.sizes()) raise(PyExc_ValueError, "k_cache and v_cache differ in shape");
    if (qkv.dim() != 2 || (qkv.size(1) != 1 && qkv.stride(1) != 1)) raise(PyExc_ValueError, "qkv: [tokens][columns] with contiguous rows expected");
    const int64_t T = qkv.size(0), G = k.size(1), D = k.size(3), H = a.u32(6, 0), half = turns.numel();
    if (qkv.size(1) != (H + 2 * G) * D)
        raise(PyExc_ValueError, "qkv: %lld columns expected for %lld + 2 * %lld heads of %lld, got %lld", (long long)((H + 2 * G) * D), (long long)H, (long long)G,
              (long long)D, (long long)qkv.size(1));
    if (positions.dim() > 2 || positions.dim() < 1 || positions.size(positions.dim() - 1) != T) raise(PyExc_ValueError, "positions: [tokens] or [axes][tokens] expected");
    const int64_t A = positions.dim() == 2 ? positions.size(0) : 1;
    const int32_t *pp = ints(positions, "positions", -1), *sp = ints(slots, "slots", T), *ap = a.given(7) ? ints(a.tensor(7), "axes", half) : nullptr;
    auto gamma = [&](int i, const char* what) -> const void* {
        if (!a.given(i)) return nullptr;
        need_heads(a.tensor(i), what, 1);
        if (a.tensor(i).numel() != D) raise(PyExc_ValueError, "%s: %lld weights expected", what, (long long)D);
        return a.tensor(i).data_ptr();
    };
    const void *gq = gamma(8, "gamma_q"), *gk = gamma(9, "gamma_k");
    const float eps = a.given(10) ? a.f32(10) : 0.0f;
    const uint32_t flags = (a.u32(11, 0) & ~MIORI_ROPE_F32) | (fp32 ? MIORI_ROPE_F32 : 0u);
    const int64_t strides[6] = {step(k, 0), step(k, 1), step(k, 2), step(v, 0), step(v, 1), step(v, 2)};
    Out o = output(a, 12, {T, H, D}, at::kBFloat16, qkv);
    call(abi.rope_kv, qkv.data_ptr(), T == 1 ? qkv.size(1) : qkv.stride(0), static_cast<const uint64_t*>(turns.data_ptr()), ap, pp, sp, gq, gk, eps, o.ptr(),
         k.data_ptr(), v.data_ptr(), strides, T, H, G, D, 2 * half, A, k.size(0), k.size(2), flags, stream());
    return o.result();
}

// scale given, or 1 / sqrt(dim)
float scale_of(const Args& a, int i, int64_t D) { return a.given(i) ? a.f32(i) : 1.0f / std::sqrt((float)D); }
// The output of q's shape: strided views of the caller's are fine.
Out heads_out(const Args& a, int i, const at::Tensor& q) {
    Out o;
    if (!a.given(i)) {
        o.made = empty(q.sizes(), at::kBFloat16, q);
        return o;
    }
    need_heads(a.tensor(i), "out", 3);
    if (a.tensor(i).sizes() != q.sizes()) raise(PyExc_ValueError, "out: the shape of q is expected");
    o.given = a.v[i];
    return o;
}

OP(attention_paged, 7, "q", "k_cache", "v_cache", "table", "lens", "cu", "max_new", "scale", "flags", "out", "workspace") {
    const at::Tensor &q = a.tensor(0), &k = a.tensor(1), &v = a.tensor(2), &table = a.tensor(3), &lens = a.tensor(4), &cu = a.tensor(5);
    need_heads(q, "q", 3);
    need_heads(k, "k_cache", 4);
    need_heads(v, "v_cache", 4);
    if (k.sizes() != v.sizes()) raise(PyExc_ValueError, "k_cache and v_cache differ in shape");
    const int64_t T = q.size(0), H = q.size(1), D = q.size(2), G = k.size(1), R = lens.numel();
    if (k.size(3) != D) raise(PyExc_ValueError, "heads of q and of the cache differ in size");
    const int32_t *tp = ints(table, "table", -1), *lp = ints(lens, "lens", -1), *cp = ints(cu, "cu", R + 1);
    if (table.dim() != 2 || table.size(0) != R) raise(PyExc_ValueError, "table: [%lld][width] expected", (long long)R);
    const uint32_t max_new = a.u32(6, 0), flags = a.u32(8, 0);
    const float scale = scale_of(a, 7, D);
    Out o = heads_out(a, 9, q);
    const at::Tensor& out = o.given ? THPVariable_Unpack(o.given) : o.made;
    void* wp;
    size_t wb;
    workspace(a, 10, wp, wb);
    const int64_t strides[10] = {step(q, 0), step(q, 1), step(out, 0), step(out, 1), step(k, 0), step(k, 1), step(k, 2), step(v, 0), step(v, 1), step(v, 2)};
    call(abi.attention_paged, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), strides, tp, lp, cp, R, T, table.size(1), k.size(0), k.size(2), H, G, D,
         max_new, scale, flags, wp, wb, stream());
    return o.result();
}

OP(attention_prompt, 4, "q", "k", "v", "cu", "cu_k", "scale", "flags", "out", "workspace") {
    const at::Tensor &q = a.tensor(0), &k = a.tensor(1), &v = a.tensor(2), &cu = a.tensor(3);
    need_heads(q, "q", 3);
    need_heads(k, "k", 3);
    need_heads(v, "v", 3);
    if (k.sizes() != v.sizes()) raise(PyExc_ValueError, "k and v differ in shape");
    const int64_t T = q.size(0), H = q.size(1), D = q.size(2), G = k.size(1), R = cu.numel() - 1;
    if (k.size(2) != D) raise(PyExc_ValueError, "heads of q and of k differ in size");
    if (!a.given(4) && k.size(0) != T) raise(PyExc_ValueError, "k: %lld rows expected, as q has (or give cu_k)", (long long)T);
    const int32_t *cp = ints(cu, "cu", -1), *kp = a.given(4) ? ints(a.tensor(4), "cu_k", R + 1) : nullptr;
    const float scale = scale_of(a, 5, D);
    const uint32_t flags = a.u32(6, 0);
    Out o = heads_out(a, 7, q);
    const at::Tensor& out = o.given ? THPVariable_Unpack(o.given) : o.made;
    void* wp;
    size_t wb;
    workspace(a, 8, wp, wb);
    const int64_t strides[8] = {step(q, 0), step(q, 1), step(out, 0), step(out, 1), step(k, 0), step(k, 1), step(v, 0), step(v, 1)};
    call(abi.attention_prompt, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), strides, cp, kp, R, T, k.size(0), H, G, D, scale, flags, wp, wb, stream());
    return o.result();
}

// An optional argument for the next function; one that is not on a GPU is refused, or taken where it is pinned, by its own check.
const at::Tensor* or_first(const Args& a, int i) { return a.given(i) && a.tensor(i).is_cuda() ? &a.tensor(i) : &a.tensor(0); }
// A call on a device that need not be the current one, on its current stream.
void* stream(c10::Device d) { return (void*)c10::cuda::getCurrentCUDAStream(d.index()).stream(); }
template <class... P, class... A>
void call_on(c10::Device d, int (*fn)(P...), A... args) {
    const c10::cuda::CUDAGuard guard(d);
    call(fn, args...);
}
// The device of these tensors, which have to share one.
c10::Device device_of(std::initializer_list<const at::Tensor*> ts) {
    const c10::Device d = (*ts.begin())->device();
    for (const at::Tensor* t : ts)
        if (t->device() != d) raise(PyExc_ValueError, "tensors of one device are expected, got some of %s and of %s", d.str().c_str(), t->device().str().c_str());
    return d;
}

// A matrix of 8-bit floating point: rows may lie apart, on 16-byte boundaries (the library checks those).
void need_fp8(const at::Tensor& t, const char* what, int64_t dims) {
    if (!t.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    if (t.scalar_type() != at::kFloat8_e4m3fn) raise(PyExc_TypeError, "%s: a float8_e4m3fn tensor is expected", what);
    if (t.dim() != dims) raise(PyExc_ValueError, "%s: %lld dimensions expected, got %lld", what, (long long)dims, (long long)t.dim());
    if (t.size(dims - 1) != 1 && t.stride(dims - 1) != 1) raise(PyExc_ValueError, "%s: the last dimension must be contiguous", what);
}
// Scales [rows][cols] fp32 of any strides.
void need_scales(const at::Tensor& t, const char* what, int64_t rows, int64_t cols) {
    if (!t.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    if (t.scalar_type() != at::kFloat) raise(PyExc_TypeError, "%s: an fp32 tensor is expected", what);
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols) raise(PyExc_ValueError, "%s: [%lld][%lld] expected", what, (long long)rows, (long long)cols);
}
// The pitch of a matrix's rows; that of a single one is of no account.
int64_t pitch(const at::Tensor& t, int64_t unit) { return t.size(0) == 1 ? (t.size(1) + unit - 1) / unit * unit : t.stride(0); }
int64_t blocks(int64_t n) { return (n + 127) / 128; }
// Sizes that the library counts in 32 bits.
void need_u32(const char* fn, std::initializer_list<int64_t> sizes) {
    for (const int64_t n : sizes)
        if (n > 0x7FFFFFFF) raise(PyExc_ValueError, "%s: a size of %lld", fn, (long long)n);
}

OP(quant_fp8, 1, "x", "tile", "flags", "out", "scales") {
    const at::Tensor& x = a.tensor(0);
    if (!x.is_cuda()) raise(PyExc_ValueError, "miori_b200 ops need CUDA tensors (there is no CPU path)");
    const bool fp32 = x.scalar_type() == at::kFloat;
    if (!fp32 && x.scalar_type() != at::kBFloat16) raise(PyExc_TypeError, "x: an fp32 or bf16 tensor is expected");
    if (x.dim() != 2 || (x.size(1) != 1 && x.stride(1) != 1)) raise(PyExc_ValueError, "x: [rows][K] with contiguous rows expected");
    const int64_t R = x.size(0), K = x.size(1), tile = a.u32(1, 1);
    if (tile != 1 && tile != 128) raise(PyExc_ValueError, "tile: 1 or 128 rows expected, got %lld", (long long)tile);
    need_u32("quant_fp8", {R, K});
    const int64_t row_blocks = (R + tile - 1) / tile;
    const uint32_t flags = (a.u32(2, 0) & ~MIORI_QUANT_F32) | (fp32 ? MIORI_QUANT_F32 : 0u);
    at::Tensor q, s;
    const c10::Device on = device_of({&x, or_first(a, 3), or_first(a, 4)});
    const int64_t pitch_made = (K + 15) / 16 * 16, k_blocks = blocks(K);  // rows of new codes begin on 16-byte boundaries
    if (a.given(3)) {
        q = a.tensor(3);
        need_fp8(q, "out", 2);
        if (q.size(0) != R || q.size(1) != K) raise(PyExc_ValueError, "out: the shape of x is expected");
    } else {
        q = empty({R, pitch_made}, at::kFloat8_e4m3fn, x);
        q.unsafeGetTensorImpl()->set_sizes_and_strides(std::vector<int64_t>{R, K}, std::vector<int64_t>{pitch_made, 1});
    }
    if (a.given(4)) {
        s = a.tensor(4);
        need_scales(s, "scales", row_blocks, k_blocks);
    } else {
        s = empty({row_blocks, k_blocks}, at::kFloat, x);
    }
    call_on(on, abi.quant_fp8, x.data_ptr(), R == 1 ? K : x.stride(0), q.data_ptr(), pitch(q, 16), static_cast<float*>(s.data_ptr()), s.stride(0), s.stride(1), R, K, tile,
         flags, stream(on));
    return tuple_of({&q, &s});
}

OP(gemm_fp8, 4, "a", "sa", "w", "sw", "flags", "out") {
    const at::Tensor &x = a.tensor(0), &sa = a.tensor(1), &w = a.tensor(2), &sw = a.tensor(3);
    need_fp8(x, "a", 2);
    need_fp8(w, "w", 2);
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    if (w.size(1) != K) raise(PyExc_ValueError, "w: rows of %lld expected, as a has, got %lld", (long long)K, (long long)w.size(1));
    need_u32("gemm_fp8", {M, N, K});
    need_scales(sa, "sa", M, blocks(K));
    need_scales(sw, "sw", blocks(N), blocks(K));
    const uint32_t flags = a.u32(4, 0);
    const at::ScalarType dt = out_type(flags);
    const c10::Device on = device_of({&x, &sa, &w, &sw, or_first(a, 5)});
    Out o;  // rows of a caller's output may lie apart
    if (a.given(5)) a.tensor(5), o.given = a.v[5];
    else o.made = empty({M, N}, dt, x);
    const at::Tensor& c = o.given ? THPVariable_Unpack(o.given) : o.made;
    if (!c.is_cuda()) raise(PyExc_ValueError, "out: a CUDA tensor is expected");
    if (c.scalar_type() != dt || c.dim() != 2 || c.size(0) != M || c.size(1) != N || (N != 1 && c.stride(1) != 1))
        raise(PyExc_ValueError, "out: [%lld][%lld] of the output's type with contiguous rows expected", (long long)M, (long long)N);
    call_on(on, abi.gemm_fp8, x.data_ptr(), pitch(x, 16), static_cast<const float*>(sa.data_ptr()), sa.stride(0), sa.stride(1), w.data_ptr(), pitch(w, 16),
         static_cast<const float*>(sw.data_ptr()), sw.stride(0), sw.stride(1), c.data_ptr(), M == 1 ? N : c.stride(0), M, N, K, flags, stream(on));
    return o.result();
}

// What both layers of experts are called with beside their weights.
struct Layer {
    int64_t T, H, E;
    const float* bias = nullptr;
    void* workspace;
    size_t bytes;
};
Layer layer(const Args& a, int x_at, int workspace_at, int bias_at) {
    const at::Tensor &x = a.tensor(x_at), &router = a.tensor(x_at + 1);
    need_cuda({&x, &router});
    if (x.scalar_type() != at::kBFloat16 || router.scalar_type() != at::kBFloat16) raise(PyExc_TypeError, "x and router: bf16 tensors are expected");
    Layer l;
    rows_of(x, l.T, l.H);
    if (router.dim() != 2 || router.size(1) != l.H) raise(PyExc_ValueError, "router: [experts][%lld] expected", (long long)l.H);
    l.E = router.size(0);
    need_u32("moe", {l.T, l.H, l.E});
    if (a.given(bias_at)) {
        const at::Tensor& b = a.tensor(bias_at);
        need_cuda({&b});
        if (b.scalar_type() != at::kFloat || b.numel() != l.E) raise(PyExc_ValueError, "bias: fp32, one an expert, expected");
        l.bias = static_cast<const float*>(b.data_ptr());
    }
    if (!a.given(workspace_at)) raise(PyExc_TypeError, "workspace: a tensor is expected (moe_workspace)");
    workspace(a, workspace_at, l.workspace, l.bytes);
    return l;
}
// A tensor of the experts' weights: contiguous, of this type and shape.
const void* weights(const at::Tensor& t, const char* what, at::ScalarType dt, int64_t E, int64_t rows, int64_t cols) {
    need_cuda({&t});
    if (t.scalar_type() != dt) raise(PyExc_TypeError, "%s: a tensor of another type is expected", what);
    if (t.dim() != 3 || t.size(0) != E || t.size(1) != rows || t.size(2) != cols)
        raise(PyExc_ValueError, "%s: [%lld][%lld][%lld] expected", what, (long long)E, (long long)rows, (long long)cols);
    return t.data_ptr();
}
int64_t ff_of(const at::Tensor& up, const char* what) {
    if (up.dim() != 3 || up.size(1) % 2) raise(PyExc_ValueError, "%s: [experts][2 ff][..] expected", what);
    need_u32("moe", {up.size(1)});
    return up.size(1) / 2;
}

OP(moe4, 10, "x", "router", "q_up", "s_up", "b_up", "q_down", "s_down", "b_down", "top", "workspace", "bias", "group", "factor", "flags", "out") {
    const Layer l = layer(a, 0, 9, 10);
    const int64_t F = ff_of(a.tensor(2), "q_up"), group = a.u32(11, 32);
    if (group != 32 && group != 64) raise(PyExc_ValueError, "group must be 32 or 64, got %lld", (long long)group);
    if (l.H % 128 || F % 128) raise(PyExc_ValueError, "hidden and ff are multiples of 128, got %lld and %lld", (long long)l.H, (long long)F);
    const void *qu = weights(a.tensor(2), "q_up", at::kInt, l.E, 2 * F, l.H / 8), *su = weights(a.tensor(3), "s_up", at::kBFloat16, l.E, 2 * F, l.H / group),
               *bu = weights(a.tensor(4), "b_up", at::kBFloat16, l.E, 2 * F, l.H / group), *qd = weights(a.tensor(5), "q_down", at::kInt, l.E, l.H, F / 8),
               *sd = weights(a.tensor(6), "s_down", at::kBFloat16, l.E, l.H, F / group), *bd = weights(a.tensor(7), "b_down", at::kBFloat16, l.E, l.H, F / group);
    const uint32_t top = a.u32(8, 0), flags = a.u32(13, 0);
    const c10::Device on = device_of({&a.tensor(0), &a.tensor(1), &a.tensor(2), &a.tensor(3), &a.tensor(4), &a.tensor(5), &a.tensor(6), &a.tensor(7), &a.tensor(9),
                                             or_first(a, 10), or_first(a, 14)});
    const float factor = a.given(12) ? a.f32(12) : 1.0f;
    Out o = output(a, 14, {l.T, l.H}, out_type(flags), a.tensor(0));
    call_on(on, abi.moe4, a.tensor(0).data_ptr(), a.tensor(1).data_ptr(), l.bias, qu, su, bu, qd, sd, bd, o.ptr(), l.T, l.E, top, l.H, F, group, factor, flags, l.workspace,
         l.bytes, stream(on));
    return o.result();
}

OP(moe_fp8, 8, "x", "router", "w_up", "s_up", "w_down", "s_down", "top", "workspace", "bias", "factor", "flags", "out") {
    const Layer l = layer(a, 0, 7, 8);
    const int64_t F = ff_of(a.tensor(2), "w_up");
    const void *wu = weights(a.tensor(2), "w_up", at::kFloat8_e4m3fn, l.E, 2 * F, l.H), *su = weights(a.tensor(3), "s_up", at::kFloat, l.E, blocks(2 * F), blocks(l.H)),
               *wd = weights(a.tensor(4), "w_down", at::kFloat8_e4m3fn, l.E, l.H, F), *sd = weights(a.tensor(5), "s_down", at::kFloat, l.E, blocks(l.H), blocks(F));
    const uint32_t top = a.u32(6, 0), flags = a.u32(10, 0);
    const c10::Device on = device_of({&a.tensor(0), &a.tensor(1), &a.tensor(2), &a.tensor(3), &a.tensor(4), &a.tensor(5), &a.tensor(7),
                                             or_first(a, 8), or_first(a, 11)});
    const float factor = a.given(9) ? a.f32(9) : 1.0f;
    Out o = output(a, 11, {l.T, l.H}, out_type(flags), a.tensor(0));
    call_on(on, abi.moe_fp8, a.tensor(0).data_ptr(), a.tensor(1).data_ptr(), l.bias, wu, static_cast<const float*>(su), wd, static_cast<const float*>(sd), o.ptr(), l.T, l.E,
         top, l.H, F, factor, flags, l.workspace, l.bytes, stream(on));
    return o.result();
}

// bind(handle, error): take the library's functions from the handle that ctypes opened.
PyObject* py_bind(PyObject*, PyObject* args) {
    unsigned long long h = 0;
    PyObject* err = nullptr;
    if (!PyArg_ParseTuple(args, "KO", &h, &err)) return nullptr;
#define X(name)                                                                                    \
    abi.name = reinterpret_cast<decltype(abi.name)>(dlsym(reinterpret_cast<void*>(h), "miori_" #name)); \
    if (!abi.name) return PyErr_Format(PyExc_ImportError, "miori_" #name " is missing from the library");
    MIORI_ENTRIES(X)
#undef X
    Py_XSETREF(g_error, Py_NewRef(err));
    Py_RETURN_NONE;
}

#define FAST(name, signature, text)                                                                \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_##name)),            \
     METH_FASTCALL | METH_KEYWORDS, #name "(" signature ")\n--\n\n" text}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, "bind(handle, error)\n--\n\nTake the C ABI from an open library handle."},
    FAST(gemv4, "q, s, b, x, group=32, flags=0, out=None",
         "y[M][N] for packed 4-bit weights q[N][K/8] (int32 words), s/b[N][K/group] bf16."),
    FAST(gemv8, "q, s, b, x, group=32, flags=0, out=None", "y[M][N] for packed 8-bit weights q[N][K/4] (int32 words)."),
    FAST(dequant4_rowmajor, "q, s, b, group=32, out=None", "bf16 [N][K] of packed 4-bit weights."),
    FAST(dequant8_rowmajor, "q, s, b, group=32, out=None", "bf16 [N][K] of packed 8-bit weights."),
    FAST(dequant4_cache, "q, s, b, group=32, out=None",
         "Layout-opaque bf16 cache for gemm_bf16_cache (returned as a flat bf16 tensor)."),
    FAST(gemm_bf16_cache, "A, cache, N, flags=0, out=None, workspace=None",
         "C[M][N] = A[M][K] x cache(N,K)^T on the tcgen05 tensor cores (split-K if a workspace tensor is\n"
         "given and the shape has few output tiles)."),
    FAST(gemm_bf16_strided, "A, B, flags=0, out=None",
         "C[M][N] = A[M][K] x B[N][K]^T for bf16 operands whose rows may be strided (views of larger\n"
         "tensors, last dimension contiguous); `out` may be a strided view too."),
    FAST(gemv_bf16_cache, "x, cache, N, flags=0, out=None",
         "y[M][N] = x[M][K] (bf16) against the bf16 cache, M <= 32: the narrow-batch kernel."),
    FAST(linear4, "q, s, b, cache, x, group=32, flags=0, out=None, workspace=None",
         "Projection dispatch: packed-weight GEMV up to four rows, the bf16 cache above (narrow-batch\n"
         "kernel or tensor-core GEMM by shape; lib.miori_linear4_route tells which)."),
    FAST(rmsnorm, "x, gamma, eps, flags=0, out=None",
         "bf16(x * rsqrt(mean(x^2) + eps) * gamma): x fp32 [rows][n], gamma bf16 [n]."),
    FAST(post_norm_add, "x, src, gamma, eps, flags=0, out=None",
         "x + src * rsqrt(mean(src^2) + eps) * gamma, fp32 [rows][n]; gamma bf16 [n]."),
    FAST(silu_mul, "gate, up, flags=0, out=None", "bf16(gate / (1 + exp(-gate)) * up), fp32 inputs of the same shape."),
    FAST(embed8, "q, s, b, tokens, group=32, flags=0, out=None",
         "Rows tokens[t] of the 8-bit table q [rows][K/4] dequantized to bf16 [T][K]."),
    FAST(argmax, "v, flags=0",
         "(index, value) tensors of the largest element of a 1-D fp32 or bf16 vector; ties: lowest index."),
    FAST(gemv4_rmsnorm, "q, s, b, x, gamma, eps, group=32, flags=0, out=None",
         "gemv4 over bf16(rmsnorm(x) * gamma) with the norm fused into the kernel's activation staging."),
    FAST(gemv8_rmsnorm, "q, s, b, x, gamma, eps, group=32, flags=0, out=None",
         "gemv8 over bf16(rmsnorm(x) * gamma) with the norm fused into the kernel's activation staging."),
    FAST(gemv4_silu, "q, s, b, x, group=32, flags=0, out=None",
         "bf16(silu(gate) * up) [M][N/2] for the fused gate + up weights q [N][K/8] (gate rows first):\n"
         "gemv4 with silu_mul as its epilogue."),
    FAST(gemv4_post_norm_add, "q, s, b, x, residual, gamma, eps, counter, group=32, flags=0, out=None",
         "residual + v * rsqrt(mean(v^2) + eps) * gamma for v = gemv4(x), fp32 [M][N], M <= 4: gemv4 with\n"
         "post_norm_add as its epilogue.  `counter`: a zeroed int32 tensor of one element, left zero."),
    FAST(gemv4_rmsnorm_silu, "q, s, b, x, gamma, eps, group=32, flags=0, out=None",
         "bf16(silu(gate) * up) [M][N/2] of the fused gate + up weights applied to bf16(rmsnorm(x) * gamma),\n"
         "x fp32 [M][K], M <= 4: one launch for the norm, both projections and the activation."),
    FAST(page_slots, "held, new, table, pool, taken, page, tokens, flags=0",
         "(slots, positions, cu, held_after, taken_after) of a step in which request r adds new[r] tokens to its held[r]:\n"
         "new pages come from pool[taken:] and are written into table [requests][width]; all int32.  slots and positions\n"
         "have `tokens` rows; rows without a token, or without a page for it, get slot -1."),
    FAST(rope_kv, "qkv, turns, positions, slots, k_cache, v_cache, heads, axes=None, gamma_q=None, gamma_k=None, eps=0.0, flags=0, out=None",
         "q [T][heads][dim] bf16 of qkv [T][(heads + 2 kv_heads) * dim] (fp32 or bf16): q and k heads normed (gamma) and turned\n"
         "by their positions [T] or [axes][T]; k and v written into slots[t] of the caches [pages][kv_heads][page][dim].\n"
         "turns, axes: see rope_turns.  flags: ROPE_ADJACENT, LAUNCH_PDL."),
    FAST(attention_paged, "q, k_cache, v_cache, table, lens, cu, max_new, scale=None, flags=0, out=None, workspace=None",
         "Causal attention of the packed tokens q [T][heads][dim] (request r: rows cu[r] to cu[r + 1] - 1, its newest) over the\n"
         "pages of each request, lens[r] positions; bf16.  max_new: the most tokens of a request.  workspace:\n"
         "attention_workspace(), lets SMs share a request.  flags: ATTENTION_FULL, LAUNCH_PDL."),
    FAST(attention_prompt, "q, k, v, cu, cu_k=None, scale=None, flags=0, out=None, workspace=None",
         "Causal attention of packed prompts: q [T][heads][dim], k and v [T][kv_heads][dim] bf16, prompt r being rows cu[r] to\n"
         "cu[r + 1] - 1 (keys: cu_k, where they are others').  workspace, flags: as attention_paged."),
    FAST(quant_fp8, "x, tile=1, flags=0, out=None, scales=None",
         "(q, scales) of x [rows][K] fp32 or bf16: q float8_e4m3fn, scales fp32 [rows / tile][K / 128] (both rounded up), a scale for\n"
         "each block of 128 along K of one row (tile=1: activations) or of 128 rows (tile=128: weights)."),
    FAST(gemm_fp8, "a, sa, w, sw, flags=0, out=None",
         "C[M][N] (fp32, OUT_BF16: bf16) of a [M][K] and w [N][K] float8_e4m3fn, with the scales of quant_fp8(tile=1) and\n"
         "quant_fp8(tile=128); rows may lie apart, on 16-byte boundaries."),
    FAST(moe4, "x, router, q_up, s_up, b_up, q_down, s_down, b_down, top, workspace, bias=None, group=32, factor=1.0, flags=0, out=None",
         "A layer of experts for up to 32 tokens, x [T][H] bf16 -> [T][H] fp32 (OUT_BF16: bf16): router [E][H] bf16, packed 4-bit\n"
         "weights [E][2 F][H] (gate rows first) and [E][H][F].  Each token's `top` experts by softmax (MOE_SIGMOID: sigmoid) + bias;\n"
         "MOE_NORM: their weights sum to one.  workspace: moe_workspace()."),
    FAST(moe_fp8, "x, router, w_up, s_up, w_down, s_down, top, workspace, bias=None, factor=1.0, flags=0, out=None",
         "moe4 with float8_e4m3fn weights [E][2 F][H] and [E][H][F] and their scales for each 128 x 128."),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "Native call path of the operators, " MIORI_TORCH_TAG, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
