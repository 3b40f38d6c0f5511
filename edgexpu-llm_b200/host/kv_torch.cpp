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

// kv.py's descriptor: the library's, and the CUDA device that the cache is on.
struct Cache : edgexpu_cuda_kv_cache {
    int device;
};
static_assert(sizeof(Cache) == sizeof(edgexpu_cuda_kv_cache) + 8, "the device follows the library's fields");

[[noreturn]] void wrong(PyObject *o, const Cache *c, at::ScalarType dtype, std::initializer_list<int64_t> shape, const char *what, const char *kind) {
    std::ostringstream s;
    s << what << ": expected a " << kind << " tensor of " << dtype << ", shape (";
    for (const int64_t n : shape) s << n << ", ";
    s << ") on cuda:" << c->device << "; got ";
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
bool beside(const at::Tensor &t, const Cache *c) { return t.is_cuda() && t.device().index() == c->device; }

// Address of a contiguous tensor of this type and shape on the cache's device.
template <typename T = void>
T *need(PyObject *o, const Cache *c, at::ScalarType dtype, std::initializer_list<int64_t> shape, const char *what) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() == dtype && beside(t, c) && has_shape(t, shape) && t.is_contiguous()) return static_cast<T *>(t.data_ptr());
    }
    wrong(o, c, dtype, shape, what, "contiguous");
}
int32_t *need_ints(PyObject *o, const Cache *c, int64_t n, const char *what) { return need<int32_t>(o, c, at::kInt, {n}, what); }
template <typename T>
T *need_or_null(PyObject *o, const Cache *c, at::ScalarType dtype, std::initializer_list<int64_t> shape, const char *what) {
    return o == Py_None ? nullptr : need<T>(o, c, dtype, shape, what);
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

// The cache at this address, which is on the library's device (of a library that is not bound the call itself tells).
const Cache *cache_of(PyObject *o) {
    const auto *c = static_cast<const Cache *>(PyLong_AsVoidPtr(o));
    if (c == nullptr) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no cache");
        throw Raised();
    }
    const int bound = edgexpu_cuda_device();
    if (bound >= 0 && bound != c->device) {
        PyErr_Format(PyExc_ValueError, "the cache is on cuda:%d, the library on cuda:%d", c->device, bound);
        throw Raised();
    }
    return c;
}
at::ScalarType type_of(const Cache *c) { return c->type == EDGEXPU_CUDA_TYPE_F16 ? at::kHalf : at::kBFloat16; }

void *stream_of(const Cache *c) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(c->device)).stream(); }

void done(int ok) {
    if (ok) return;
    PyErr_SetString(g_error != nullptr ? g_error : PyExc_RuntimeError, edgexpu_cuda_last_error());
    throw Raised();
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const Cache *c) {
    return at::Tensor(at::detail::empty_cuda(shape, dtype, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(c->device)), c10::nullopt));
}

// (cache, seqs, n_new, missing or None) -> pos
PyObject *append(PyObject *const *a) {
    const Cache *c = cache_of(a[0]);
    const int n = length(tensor(a[1], "seqs"), "seqs");
    const int32_t *ps = need_ints(a[1], c, n, "seqs"), *pn = need_ints(a[2], c, n, "n_new");
    int32_t *missing = need_or_null<int32_t>(a[3], c, at::kInt, {1}, "missing");
    at::Tensor pos = empty({n}, at::kInt, c);
    done(edgexpu_cuda_kv_append_dev(c, ps, pn, n, pos.data_ptr<int32_t>(), missing, stream_of(c)));
    return THPVariable_Wrap(pos);
}

// (cache, src, dst)
template <int (*CALL)(const edgexpu_cuda_kv_cache *, const int32_t *, const int32_t *, int, void *)>
PyObject *pairs(PyObject *const *a) {
    const Cache *c = cache_of(a[0]);
    const int n = length(tensor(a[1], "src"), "src");
    const int32_t *ps = need_ints(a[1], c, n, "src"), *pd = need_ints(a[2], c, n, "dst");
    done(CALL(c, ps, pd, n, stream_of(c)));
    Py_RETURN_NONE;
}

// (cache, seqs, keep or None)
PyObject *free_(PyObject *const *a) {
    const Cache *c = cache_of(a[0]);
    const int n = length(tensor(a[1], "seqs"), "seqs");
    const int32_t *ps = need_ints(a[1], c, n, "seqs"), *pk = need_or_null<int32_t>(a[2], c, at::kInt, {n}, "keep");
    done(edgexpu_cuda_kv_free_dev(c, ps, pk, n, stream_of(c)));
    Py_RETURN_NONE;
}

// (cache) -> the pages in use
PyObject *compact(PyObject *const *a) {
    const Cache *c = cache_of(a[0]);
    at::Tensor live = empty({}, at::kInt, c);
    done(edgexpu_cuda_kv_compact_dev(c, live.data_ptr<int32_t>(), stream_of(c)));
    return THPVariable_Wrap(live);
}

// fp32 rows on the cache's device, contiguous each; *stride: floats from one to the next
const float *rows_of(PyObject *o, const Cache *c, int64_t n, int64_t width, const char *what, int64_t *stride) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() == at::kFloat && beside(t, c) && has_shape(t, {n, width}) && t.stride(1) == 1) {
            *stride = n > 1 ? t.stride(0) : width;  // the distance to a second row may be anything
            return static_cast<const float *>(t.data_ptr());
        }
    }
    wrong(o, c, at::kFloat, {n, width}, what, "row-contiguous");
}

// (cache, layer, q, k, v, seqs, pos, n_heads, q_norm, k_norm, eps, rope, pairing, out or None) -> out
PyObject *qk_norm_rope(PyObject *const *a) {
    const Cache *c = cache_of(a[0]);
    const int n = length(tensor(a[2], "q"), "q"), heads = small(a[7]);
    const int64_t dim = c->head_dim, narrow = c->n_kv * dim;
    int64_t qs, ks, vs;
    const float *pq = rows_of(a[2], c, n, heads * dim, "q", &qs), *pk = rows_of(a[3], c, n, narrow, "k", &ks),
                *pv = rows_of(a[4], c, n, narrow, "v", &vs);
    const int32_t *ps = need_ints(a[5], c, n, "seqs"), *pp = need_ints(a[6], c, n, "pos");
    const float *qw = need_or_null<float>(a[8], c, at::kFloat, {dim}, "q_norm"), *kw = need_or_null<float>(a[9], c, at::kFloat, {dim}, "k_norm");
    const float *rope = nullptr;
    int positions = 0, turned = 0;
    if (a[11] != Py_None) {
        const at::Tensor &r = tensor(a[11], "rope");
        positions = length(r, "rope");
        turned = r.dim() == 2 ? static_cast<int>(r.size(1)) : 0;
        rope = need<float>(a[11], c, at::kFloat, {positions, turned}, "rope");
    }
    at::Tensor out;
    void *po;
    if (a[13] == Py_None) {
        out = empty({n, heads, dim}, type_of(c), c);
        po = out.data_ptr();
    } else {
        po = need<void>(a[13], c, type_of(c), {n, heads, dim}, "out");
    }
    done(edgexpu_cuda_qk_norm_rope_dev(c, small(a[1]), pq, pk, pv, qs, ks, vs, n, heads, qw, kw, real(a[10]), rope, positions, turned,
                                       small(a[12]), ps, pp, po, stream_of(c)));
    if (a[13] == Py_None) return THPVariable_Wrap(out);
    Py_INCREF(a[13]);
    return a[13];
}

// (cache, layer, q, seqs, q_start or None, shared_seq, shared_len, max_len or None, scale or None, out or None, fp32 out) -> out
PyObject *attention(PyObject *const *a) {
    const Cache *c = cache_of(a[0]);
    const at::Tensor &q = tensor(a[2], "q");
    const int tokens = length(q, "q"), batch = length(tensor(a[3], "seqs"), "seqs");
    const int64_t dim = c->head_dim, heads = q.dim() == 3 ? q.size(1) : 0;
    if (heads < 1 || heads > INT32_MAX) wrong(a[2], c, type_of(c), {tokens, c->n_kv, dim}, "q", "contiguous");
    const void *pq = need<void>(a[2], c, type_of(c), {tokens, heads, dim}, "q");
    const int32_t *ps = need_ints(a[3], c, batch, "seqs");
    const int32_t *start = need_or_null<int32_t>(a[4], c, at::kInt, {batch + 1LL}, "q_start");
    const int shared_seq = small(a[5]), shared_len = small(a[6]), max_len = a[7] == Py_None ? c->max_pages * c->page_size : small(a[7]);
    const float scale = a[8] == Py_None ? 1.0f / sqrtf(static_cast<float>(dim)) : real(a[8]);
    at::Tensor out;
    if (a[9] == Py_None) {
        out = empty({tokens, heads, dim}, PyObject_IsTrue(a[10]) == 1 ? at::kFloat : type_of(c), c);
    } else {
        out = tensor(a[9], "out");
        need<void>(a[9], c, out.scalar_type() == at::kFloat ? at::kFloat : type_of(c), {tokens, heads, dim}, "out");
    }
    const size_t size = edgexpu_cuda_kv_attention_work_bytes(c, batch, tokens, static_cast<int>(heads), shared_len, max_len);
    at::Tensor work;
    if (size > 0) work = empty({static_cast<int64_t>(size)}, at::kByte, c);
    done(edgexpu_cuda_kv_attention_dev(c, small(a[1]), pq, ps, start, batch, tokens, static_cast<int>(heads), shared_seq, shared_len, max_len,
                                       scale, out.data_ptr(), out.scalar_type() == at::kFloat ? EDGEXPU_CUDA_TYPE_F32 : c->type,
                                       size > 0 ? work.data_ptr() : nullptr, size, stream_of(c)));
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
                           method<1, compact>("compact"),
                           method<14, qk_norm_rope>("qk_norm_rope"),
                           method<11, attention>("attention"),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kv_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_torch(void) { return PyModule_Create(&g_module); }
