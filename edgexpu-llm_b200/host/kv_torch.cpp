/*
 * kv_torch.cpp -- the paged cache's calls (edgexpu_cuda_kv_*, edgexpu_cuda_qk_norm_rope_dev) on torch
 * tensors: a CPython module that checks the tensors, makes the outputs and passes addresses and torch's
 * current stream to the C ABI.  A decode step makes these calls once a layer, and in Python the checks
 * alone took longer than the kernels (12 us a call; 5 here).  kv.py is the interface to it.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <initializer_list>
#include <sstream>

#include "../../include/edgexpu_cuda.h"

namespace {

PyObject *g_error = nullptr;  // EdgexpuError

// A Python exception is set; unwinds to the module's entry.
struct Raised {};

[[noreturn]] void wrong(PyObject *o, at::ScalarType dtype, std::initializer_list<int64_t> shape, const char *what, const char *kind) {
    std::ostringstream s;
    s << what << ": expected a " << kind << " CUDA tensor of " << dtype << ", shape (";
    for (const int64_t n : shape) s << n << ", ";
    s << "); got ";
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        s << t.scalar_type() << " " << t.sizes() << " on " << t.device();
    } else {
        s << Py_TYPE(o)->tp_name;
    }
    PyErr_SetString(PyExc_ValueError, s.str().c_str());
    throw Raised();
}

const at::Tensor &tensor(PyObject *o, const char *what) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_ValueError, "%s: expected a tensor, got %s", what, Py_TYPE(o)->tp_name);
        throw Raised();
    }
    return THPVariable_Unpack(o);
}

bool has_shape(const at::Tensor &t, std::initializer_list<int64_t> shape) { return t.sizes() == at::IntArrayRef(shape); }

// Address of a contiguous CUDA tensor of this type and shape.
template <typename T = void>
T *need(PyObject *o, at::ScalarType dtype, std::initializer_list<int64_t> shape, const char *what) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() == dtype && t.is_cuda() && has_shape(t, shape) && t.is_contiguous()) return static_cast<T *>(t.data_ptr());
    }
    wrong(o, dtype, shape, what, "contiguous");
}
int32_t *need_ints(PyObject *o, int64_t n, const char *what) { return need<int32_t>(o, at::kInt, {n}, what); }
template <typename T>
T *need_or_null(PyObject *o, at::ScalarType dtype, std::initializer_list<int64_t> shape, const char *what) {
    return o == Py_None ? nullptr : need<T>(o, dtype, shape, what);
}

int64_t number(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}
int small(PyObject *o) {
    const int64_t v = number(o);
    if (v < INT32_MIN || v > INT32_MAX) {
        PyErr_SetString(PyExc_ValueError, "a number does not fit 32 bits");
        throw Raised();
    }
    return static_cast<int>(v);
}
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return static_cast<float>(v);
}

int length(const at::Tensor &t, const char *what) {
    if (t.dim() < 1 || t.size(0) > INT32_MAX) {
        PyErr_Format(PyExc_ValueError, "%s: expected rows", what);
        throw Raised();
    }
    return static_cast<int>(t.size(0));
}

const edgexpu_cuda_kv_cache *cache_of(PyObject *o) {
    void *p = PyLong_AsVoidPtr(o);
    if (p == nullptr && PyErr_Occurred()) throw Raised();
    return static_cast<const edgexpu_cuda_kv_cache *>(p);
}
at::ScalarType type_of(const edgexpu_cuda_kv_cache *c) { return c->type == EDGEXPU_CUDA_TYPE_F16 ? at::kHalf : at::kBFloat16; }

void *stream_of(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.is_cuda() ? t.device().index() : -1).stream(); }

void done(int ok) {
    if (ok) return;
    PyErr_SetString(g_error != nullptr ? g_error : PyExc_RuntimeError, edgexpu_cuda_last_error());
    throw Raised();
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const at::Tensor &like) {
    return at::Tensor(at::detail::empty_cuda(shape, dtype, like.device(), c10::nullopt));
}

// (cache, seqs, n_new, missing or None) -> pos
PyObject *append(PyObject *const *a) {
    const auto *c = cache_of(a[0]);
    const at::Tensor &seqs = tensor(a[1], "seqs");
    const int n = length(seqs, "seqs");
    const int32_t *ps = need_ints(a[1], n, "seqs"), *pn = need_ints(a[2], n, "n_new");
    int32_t *missing = need_or_null<int32_t>(a[3], at::kInt, {1}, "missing");
    at::Tensor pos = empty({n}, at::kInt, seqs);
    done(edgexpu_cuda_kv_append_dev(c, ps, pn, n, pos.data_ptr<int32_t>(), missing, stream_of(seqs)));
    return THPVariable_Wrap(pos);
}

// (cache, src, dst)
template <int (*CALL)(const edgexpu_cuda_kv_cache *, const int32_t *, const int32_t *, int, void *)>
PyObject *pairs(PyObject *const *a) {
    const at::Tensor &src = tensor(a[1], "src");
    const int n = length(src, "src");
    const int32_t *ps = need_ints(a[1], n, "src"), *pd = need_ints(a[2], n, "dst");
    done(CALL(cache_of(a[0]), ps, pd, n, stream_of(src)));
    Py_RETURN_NONE;
}

// (cache, seqs, keep or None)
PyObject *free_(PyObject *const *a) {
    const at::Tensor &seqs = tensor(a[1], "seqs");
    const int n = length(seqs, "seqs");
    const int32_t *ps = need_ints(a[1], n, "seqs"), *pk = need_or_null<int32_t>(a[2], at::kInt, {n}, "keep");
    done(edgexpu_cuda_kv_free_dev(cache_of(a[0]), ps, pk, n, stream_of(seqs)));
    Py_RETURN_NONE;
}

// (cache, a tensor on its device) -> the pages in use
PyObject *compact(PyObject *const *a) {
    const at::Tensor &like = tensor(a[1], "table");
    at::Tensor live = empty({}, at::kInt, like);
    done(edgexpu_cuda_kv_compact_dev(cache_of(a[0]), live.data_ptr<int32_t>(), stream_of(like)));
    return THPVariable_Wrap(live);
}

// fp32 CUDA rows, contiguous each; *stride: floats from one to the next
const float *rows_of(PyObject *o, int64_t n, int64_t width, const char *what, int64_t *stride) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() == at::kFloat && t.is_cuda() && has_shape(t, {n, width}) && t.stride(1) == 1) {
            *stride = n > 1 ? t.stride(0) : width;  // the distance to a second row may be anything
            return static_cast<const float *>(t.data_ptr());
        }
    }
    wrong(o, at::kFloat, {n, width}, what, "row-contiguous");
}

// (cache, layer, q, k, v, seqs, pos, n_heads, q_norm, k_norm, eps, rope, pairing, out or None) -> out
PyObject *qk_norm_rope(PyObject *const *a) {
    const auto *c = cache_of(a[0]);
    const at::Tensor &q = tensor(a[2], "q");
    const int n = length(q, "q"), heads = small(a[7]);
    const int64_t dim = c->head_dim, narrow = c->n_kv * dim;
    int64_t qs, ks, vs;
    const float *pq = rows_of(a[2], n, heads * dim, "q", &qs), *pk = rows_of(a[3], n, narrow, "k", &ks),
                *pv = rows_of(a[4], n, narrow, "v", &vs);
    const int32_t *ps = need_ints(a[5], n, "seqs"), *pp = need_ints(a[6], n, "pos");
    const float *qw = need_or_null<float>(a[8], at::kFloat, {dim}, "q_norm"), *kw = need_or_null<float>(a[9], at::kFloat, {dim}, "k_norm");
    const float *rope = nullptr;
    int positions = 0, turned = 0;
    if (a[11] != Py_None) {
        const at::Tensor &r = tensor(a[11], "rope");
        positions = length(r, "rope");
        turned = r.dim() == 2 ? static_cast<int>(r.size(1)) : 0;
        rope = need<float>(a[11], at::kFloat, {positions, turned}, "rope");
    }
    at::Tensor out;
    void *po;
    if (a[13] == Py_None) {
        out = empty({n, heads, dim}, type_of(c), q);
        po = out.data_ptr();
    } else {
        po = need<void>(a[13], type_of(c), {n, heads, dim}, "out");
    }
    done(edgexpu_cuda_qk_norm_rope_dev(c, small(a[1]), pq, pk, pv, qs, ks, vs, n, heads, qw, kw, real(a[10]), rope, positions, turned,
                                       small(a[12]), ps, pp, po, stream_of(q)));
    if (a[13] == Py_None) return THPVariable_Wrap(out);
    Py_INCREF(a[13]);
    return a[13];
}

// (cache, layer, q, seqs, q_start or None, shared_seq, shared_len, max_len or None, scale or None, out or None, fp32 out) -> out
PyObject *attention(PyObject *const *a) {
    const auto *c = cache_of(a[0]);
    const at::Tensor &q = tensor(a[2], "q"), &seqs = tensor(a[3], "seqs");
    const int tokens = length(q, "q"), batch = length(seqs, "seqs");
    const int64_t dim = c->head_dim, heads = q.dim() == 3 ? q.size(1) : 0;
    if (heads < 1 || heads > INT32_MAX) wrong(a[2], type_of(c), {tokens, c->n_kv, dim}, "q", "contiguous");
    const void *pq = need<void>(a[2], type_of(c), {tokens, heads, dim}, "q");
    const int32_t *ps = need_ints(a[3], batch, "seqs");
    const int32_t *start = need_or_null<int32_t>(a[4], at::kInt, {batch + 1LL}, "q_start");
    const int shared_seq = small(a[5]), shared_len = small(a[6]), max_len = a[7] == Py_None ? c->max_pages * c->page_size : small(a[7]);
    const float scale = a[8] == Py_None ? 1.0f / sqrtf(static_cast<float>(dim)) : real(a[8]);
    at::Tensor out;
    if (a[9] == Py_None) {
        out = empty({tokens, heads, dim}, PyObject_IsTrue(a[10]) == 1 ? at::kFloat : type_of(c), q);
    } else {
        out = tensor(a[9], "out");
        need<void>(a[9], out.scalar_type() == at::kFloat ? at::kFloat : type_of(c), {tokens, heads, dim}, "out");
    }
    const size_t size = edgexpu_cuda_kv_attention_work_bytes(c, batch, tokens, static_cast<int>(heads), shared_len, max_len);
    at::Tensor work;
    if (size > 0) work = empty({static_cast<int64_t>(size)}, at::kByte, q);
    done(edgexpu_cuda_kv_attention_dev(c, small(a[1]), pq, ps, start, batch, tokens, static_cast<int>(heads), shared_seq, shared_len, max_len,
                                       scale, out.data_ptr(), out.scalar_type() == at::kFloat ? EDGEXPU_CUDA_TYPE_F32 : c->type,
                                       size > 0 ? work.data_ptr() : nullptr, size, stream_of(q)));
    if (a[9] == Py_None) return THPVariable_Wrap(out);
    Py_INCREF(a[9]);
    return a[9];
}

// A module function: N arguments, and no C++ exception past it.
template <int N, PyObject *(*CALL)(PyObject *const *)>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    try {
        return CALL(args);
    } catch (const Raised &) {
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown failure");
    }
    return nullptr;
}

PyObject *set_error(PyObject *const *a) {
    Py_INCREF(a[0]);
    Py_XDECREF(g_error);
    g_error = a[0];
    Py_RETURN_NONE;
}

template <int N, PyObject *(*CALL)(PyObject *const *)>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<N, CALL>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<1, set_error>("set_error"),
                           method<4, append>("append"),
                           method<3, pairs<edgexpu_cuda_kv_fork_dev>>("fork"),
                           method<3, free_>("free"),
                           method<3, pairs<edgexpu_cuda_kv_copy_dev>>("copy"),
                           method<2, compact>("compact"),
                           method<14, qk_norm_rope>("qk_norm_rope"),
                           method<11, attention>("attention"),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kv_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_torch(void) { return PyModule_Create(&g_module); }
