// The Python front of calls on torch CUDA tensors, in native code.
//
// A decode linear is done on the GPU in 2 to 5 us, and its launch takes the host 2.5; the checks, the new output tensor and the ctypes call take Python 5 more
// (256 x 1024, one row of x: 7.4 us a call, of them new_empty 1.8 and ctypes 0.7; with this module 4.0). Here the whole call is one method of this module.
//
// A method takes the plain case only: an ordinary strided, contiguous CUDA tensor (or parameter) with the weight's type, row length and device, while nothing
// intercepts torch calls (function and dispatch modes, functorch transforms, tracing). For everything else, wrong arguments among it, it returns None
// before it has done anything, and the caller goes on with the general code in ops.py, which knows the errors. Python.h's and torch's headers are all
// this needs; the kernels are reached through the addresses of the C ABI's functions that bind() is given.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty_cuda_dispatch.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace {

using Linear = int (*)(const void* w, const void* x, int64_t m, const float* bias, float* y, int mem, void* stream);
using Backward = int (*)(const void* w, const float* g, int64_t m, float* gx, int mem, void* stream);
using Dequantize = int (*)(const void* w, float* dst, int mem, void* stream);
using Quantize = int (*)(int device, const float* x, int64_t count, void* out, int mem, void* stream);
constexpr int MEM_DEVICE = 1;

Linear g_linear = nullptr, g_linear_bf16 = nullptr;
Backward g_backward = nullptr;
Dequantize g_dequantize = nullptr;
Quantize g_quantize = nullptr;
PyObject* g_check = nullptr;   // raises what a status code stands for
PyObject* g_weight = nullptr;  // the class of weights
PyObject *s_addr = nullptr, *s_dims = nullptr, *s_device = nullptr;

PyObject* not_plain() { Py_RETURN_NONE; }

// Nothing stands between a torch call and its kernel.
bool undisturbed() {
    using c10::DispatchKey;
    constexpr c10::DispatchKeySet taken({DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::PythonDispatcher, DispatchKey::PreDispatch, DispatchKey::Tracer,
                                         DispatchKey::Functionalize, DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::FuncTorchDynamicLayerBackMode,
                                         DispatchKey::FuncTorchVmapMode, DispatchKey::FuncTorchBatched, DispatchKey::VmapMode, DispatchKey::Batched});
    return !c10::impl::tls_local_dispatch_key_set().included_.has_any(taken) && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
           at::impl::PythonTorchFunctionTLS::stack_len() == 0;
}

// The tensor behind a plain CUDA tensor or parameter, or null.
const at::Tensor* plain(PyObject* obj, at::ScalarType type) {
    using c10::DispatchKey;
    if (!THPVariable_CheckExact(obj)) {
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(obj);
    constexpr c10::DispatchKeySet special({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize, DispatchKey::Batched,
                                           DispatchKey::Conjugate, DispatchKey::Negative, DispatchKey::ZeroTensor});
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.scalar_type() != type || t.dim() < 1 || t.key_set().has_any(special) || !t.is_contiguous()) {
        return nullptr;
    }
    return &t;
}

struct Weight {
    void* handle;
    int64_t n, k;
    int device;
};

bool attribute(PyObject* obj, PyObject* name, int64_t& out) {
    PyObject* v = PyObject_GetAttr(obj, name);
    if (v == nullptr) {
        PyErr_Clear();
        return false;
    }
    const bool is_int = PyLong_Check(v);
    out = is_int ? PyLong_AsLongLong(v) : 0;
    Py_DECREF(v);
    if (PyErr_Occurred() != nullptr) {
        PyErr_Clear();
        return false;
    }
    return is_int;
}

bool weight_of(PyObject* obj, Weight& w) {
    if ((PyObject*)Py_TYPE(obj) != g_weight) {
        return false;
    }
    int64_t addr = 0, device = 0;
    if (!attribute(obj, s_addr, addr) || addr == 0 || !attribute(obj, s_device, device)) {
        return false;
    }
    PyObject* dims = PyObject_GetAttr(obj, s_dims);
    if (dims == nullptr) {
        PyErr_Clear();
        return false;
    }
    bool ok = PyTuple_Check(dims) && PyTuple_GET_SIZE(dims) == 2 && PyLong_Check(PyTuple_GET_ITEM(dims, 0)) && PyLong_Check(PyTuple_GET_ITEM(dims, 1));
    if (ok) {
        w = Weight{(void*)addr, PyLong_AsLongLong(PyTuple_GET_ITEM(dims, 0)), PyLong_AsLongLong(PyTuple_GET_ITEM(dims, 1)), (int)device};
        ok = w.n > 0 && w.k > 0;
    }
    Py_DECREF(dims);
    return ok;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

at::Tensor empty_like_rows(const at::Tensor& x, int64_t last, at::ScalarType type) {
    at::DimVector sizes(x.sizes());
    sizes.back() = last;
    return at::cuda::empty(sizes, x.options().dtype(type));
}

// y, or the exception of a status code.
PyObject* finish(int rc, PyObject* y) {
    if (rc == 0) {
        return y;
    }
    Py_XDECREF(y);
    PyObject* code = PyLong_FromLong(rc);
    PyObject* none = code != nullptr ? PyObject_CallOneArg(g_check, code) : nullptr;
    Py_XDECREF(code);
    if (none != nullptr) {
        Py_DECREF(none);
        PyErr_SetString(PyExc_RuntimeError, "a call of the library failed");
    }
    return nullptr;
}

template <typename F>
PyObject* guarded(F body) {
    try {
        return body();
    } catch (const c10::OutOfMemoryError& e) {  // the general code raises torch's own
        (void)e;
        return not_plain();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject* product(PyObject* const* args, Py_ssize_t count, at::ScalarType type, Linear fn) {
    return guarded([&]() -> PyObject* {
        Weight w;
        if (count != 3 || !weight_of(args[1], w) || !undisturbed()) {
            return not_plain();
        }
        const at::Tensor* const x = plain(args[0], type);
        if (x == nullptr || x->sizes().back() != w.k || x->get_device() != w.device) {
            return not_plain();
        }
        const float* bias = nullptr;
        if (args[2] != Py_None) {
            const at::Tensor* const b = plain(args[2], at::kFloat);
            if (b == nullptr || b->numel() != w.n || b->get_device() != w.device) {
                return not_plain();
            }
            bias = (const float*)b->const_data_ptr();
        }
        at::Tensor y = empty_like_rows(*x, w.n, at::kFloat);
        const void* const xp = x->const_data_ptr();
        float* const yp = (float*)y.mutable_data_ptr();
        const int64_t m = x->numel() / w.k;
        void* const stream = stream_of(w.device);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = fn(w.handle, xp, m, bias, yp, MEM_DEVICE, stream);
        Py_END_ALLOW_THREADS;
        return finish(rc, rc == 0 ? THPVariable_Wrap(std::move(y)) : nullptr);
    });
}

PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t count) { return product(args, count, at::kFloat, g_linear); }
PyObject* linear_bf16(PyObject*, PyObject* const* args, Py_ssize_t count) { return product(args, count, at::kBFloat16, g_linear_bf16); }

PyObject* backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        Weight w;
        if (count != 2 || !weight_of(args[1], w) || !undisturbed()) {
            return not_plain();
        }
        const at::Tensor* const g = plain(args[0], at::kFloat);
        if (g == nullptr || g->sizes().back() != w.n || g->get_device() != w.device) {
            return not_plain();
        }
        at::Tensor gx = empty_like_rows(*g, w.k, at::kFloat);
        const float* const gp = (const float*)g->const_data_ptr();
        float* const xp = (float*)gx.mutable_data_ptr();
        const int64_t m = g->numel() / w.n;
        void* const stream = stream_of(w.device);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = g_backward(w.handle, gp, m, xp, MEM_DEVICE, stream);
        Py_END_ALLOW_THREADS;
        return finish(rc, rc == 0 ? THPVariable_Wrap(std::move(gx)) : nullptr);
    });
}

PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t count) {  // weight, out
    return guarded([&]() -> PyObject* {
        Weight w;
        if (count != 2 || !weight_of(args[0], w) || !undisturbed()) {
            return not_plain();
        }
        const at::Tensor* const out = plain(args[1], at::kFloat);
        if (out == nullptr || out->numel() < w.n * w.k || out->get_device() != w.device) {
            return not_plain();
        }
        float* const to = (float*)out->mutable_data_ptr();
        void* const stream = stream_of(w.device);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = g_dequantize(w.handle, to, MEM_DEVICE, stream);
        Py_END_ALLOW_THREADS;
        return finish(rc, rc == 0 ? Py_NewRef(args[1]) : nullptr);
    });
}

PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        if (count != 1 || !undisturbed()) {
            return not_plain();
        }
        const at::Tensor* const x = plain(args[0], at::kFloat);
        if (x == nullptr || x->numel() == 0 || x->sizes().back() % 32 != 0) {
            return not_plain();
        }
        const int device = (int)x->get_device();
        at::Tensor out = at::cuda::empty({x->numel() / 32 * 34}, x->options().dtype(at::kByte));
        const float* const xp = (const float*)x->const_data_ptr();
        void* const to = out.mutable_data_ptr();
        const int64_t n = x->numel();
        void* const stream = stream_of(device);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = g_quantize(device, xp, n, to, MEM_DEVICE, stream);
        Py_END_ALLOW_THREADS;
        return finish(rc, rc == 0 ? THPVariable_Wrap(std::move(out)) : nullptr);
    });
}

// ---- the operators of paged decoding: the same for their plain calls, with outputs of their own (a rotation of queries and keys from Python 21 us a call, from here 5) ----
using RopeApply = int (*)(const void* r, int elem, int count, const void* const* x, void* const* y, const int* heads, int head_dim, const int64_t* strides, int64_t batch,
                          int64_t seq, const void* positions, int position_bytes, int64_t position_batch_stride, int64_t position_stride, int64_t offset, int inverse, void* stream);
using Append = int (*)(const void* p, const void* rope, int elem, int heads, const void* q, const void* k, const void* v, void* q_out, const int64_t* strides, int64_t tokens,
                       const int32_t* tables, int64_t table_stride, int64_t table_width, const int32_t* starts, const int32_t* lengths, int sequences, int64_t prefix_length,
                       int fill, void* stream);
using AttentionBytes = int (*)(const void* p, int elem, int heads, int64_t tokens, int64_t sequences, int64_t prefix_length, int64_t* nbytes);
using Attention = int (*)(const void* p, int elem, int heads, const void* q, void* out, const int64_t* strides, int64_t tokens, const int32_t* tables, int64_t table_stride,
                          int64_t table_width, const int32_t* starts, const int32_t* lengths, int sequences, const int32_t* prefix, int64_t prefix_width, int64_t prefix_length,
                          float scale, int fill, void* workspace, int64_t workspace_bytes, void* stream);
using VerifyBytes = int (*)(int64_t sequences, int64_t drafts, int64_t vocab, int logits, int64_t* nbytes);
using Verify = int (*)(int device, int elem, const void* target, int64_t target_stride, int64_t target_row_stride, const int32_t* drafts, const float* draft_probs,
                       int64_t draft_stride, int64_t draft_row_stride, const float* uniforms, const int32_t* counts, int64_t sequences, int64_t drafts_most, int64_t vocab,
                       int logits, double temperature, int32_t* accepted, int32_t* tokens, void* workspace, int64_t workspace_bytes, void* stream);
RopeApply g_rope_apply = nullptr;
Append g_append = nullptr;
AttentionBytes g_attention_bytes = nullptr;
Attention g_attention = nullptr;
VerifyBytes g_verify_bytes = nullptr;
Verify g_verify = nullptr;
PyObject *g_rope = nullptr, *g_pages = nullptr, *g_batch = nullptr;  // the classes
PyObject *s_plain_device = nullptr, *s_kv_heads = nullptr, *s_head_dim = nullptr, *s_code = nullptr, *s_rows = nullptr, *s_ahead = nullptr;

// The tensor behind a plain CUDA tensor on `device` (-1: any) whose last axis is in one piece, or null.
const at::Tensor* plain_strided(PyObject* obj, int64_t dims, int64_t device) {
    using c10::DispatchKey;
    if (!THPVariable_CheckExact(obj)) {
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(obj);
    constexpr c10::DispatchKeySet special({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize, DispatchKey::Batched,
                                           DispatchKey::Conjugate, DispatchKey::Negative, DispatchKey::ZeroTensor});
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.dim() != dims || t.key_set().has_any(special) || (device >= 0 && t.get_device() != device) ||
        t.numel() == 0 || t.stride(-1) != 1) {
        return nullptr;
    }
    return &t;
}

// The library's element type, -1 for others.
int elem_of(const at::Tensor& t) {
    const at::ScalarType s = t.scalar_type();
    return s == at::kFloat ? 0 : (s == at::kHalf ? 1 : (s == at::kBFloat16 ? 2 : -1));
}

at::Tensor like(const at::Tensor& x) { return at::cuda::empty(x.sizes(), x.options()); }

// An int32 tensor of that shape in one piece, or null.
const at::Tensor* whole(PyObject* obj, at::IntArrayRef shape, int64_t device) {
    const at::Tensor* const t = plain(obj, at::kInt);
    return t != nullptr && t->get_device() == device && t->sizes() == shape ? t : nullptr;
}

PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t count) {  // rope, tensor or pair, positions, inverse
    return guarded([&]() -> PyObject* {
        int64_t addr = 0, device = 0;
        if (count != 4 || (PyObject*)Py_TYPE(args[0]) != g_rope || !attribute(args[0], s_addr, addr) || addr == 0 || !attribute(args[0], s_plain_device, device) || !undisturbed()) {
            return not_plain();
        }
        const bool pair = PyTuple_Check(args[1]);
        const Py_ssize_t n = pair ? PyTuple_GET_SIZE(args[1]) : 1;
        if (n < 1 || n > 2) {
            return not_plain();
        }
        const at::Tensor* x[2] = {nullptr, nullptr};
        int heads[2] = {0, 0};
        int64_t dims = 0;
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject* const obj = pair ? PyTuple_GET_ITEM(args[1], i) : args[1];
            x[i] = plain_strided(obj, 3, device);
            if (x[i] == nullptr) {
                x[i] = plain_strided(obj, 4, device);
            }
            if (x[i] == nullptr || elem_of(*x[i]) < 0 || x[i]->scalar_type() != x[0]->scalar_type() || x[i]->dim() != x[0]->dim()) {
                return not_plain();
            }
            dims = x[i]->dim();
            for (int64_t d = 0; d < dims; d++) {
                if (d != dims - 2 && x[i]->size(d) != x[0]->size(d)) {
                    return not_plain();
                }
            }
            heads[i] = (int)x[i]->size(dims - 2);
        }
        const int64_t batch = dims == 4 ? x[0]->size(0) : 1, seq = x[0]->size(dims - 3);
        const void* at = nullptr;
        int bytes = 0;
        int64_t pb = 0, pt = 0, offset = 0;
        if (PyLong_CheckExact(args[2])) {
            offset = PyLong_AsLongLong(args[2]);
            if (PyErr_Occurred() != nullptr) {
                PyErr_Clear();
                return not_plain();
            }
        } else {
            const at::Tensor* p = plain(args[2], at::kInt);
            bytes = 4;
            if (p == nullptr) {
                p = plain(args[2], at::kLong);
                bytes = 8;
            }
            if (p == nullptr || p->get_device() != device || p->size(-1) != seq || !(p->dim() == 1 || (dims == 4 && p->dim() == 2 && p->size(0) == batch))) {
                return not_plain();
            }
            at = p->const_data_ptr();
            pt = 1;
            pb = p->dim() == 2 ? seq : 0;
        }
        const int inverse = PyObject_IsTrue(args[3]);
        at::Tensor y[2];
        const void* xp[2];
        void* yp[2];
        int64_t strides[12];
        for (Py_ssize_t i = 0; i < n; i++) {
            y[i] = like(*x[i]);
            xp[i] = x[i]->const_data_ptr();
            yp[i] = y[i].mutable_data_ptr();
            const at::Tensor* const of[2] = {x[i], &y[i]};
            for (int j = 0; j < 2; j++) {
                int64_t* const s = strides + 6 * i + 3 * j;
                s[0] = dims == 4 ? of[j]->stride(0) : 0;
                s[1] = of[j]->stride(dims - 3);
                s[2] = of[j]->stride(dims - 2);
            }
        }
        const int elem = elem_of(*x[0]), hd = (int)x[0]->size(-1);
        void* const stream = stream_of((int)device);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = g_rope_apply((const void*)addr, elem, (int)n, xp, yp, heads, hd, strides, batch, seq, at, bytes, pb, pt, offset, inverse, stream);
        Py_END_ALLOW_THREADS;
        if (rc != 0) {
            return finish(rc, nullptr);
        }
        PyObject* first = THPVariable_Wrap(std::move(y[0]));
        if (!pair) {
            return first;
        }
        return n == 2 ? Py_BuildValue("(NN)", first, THPVariable_Wrap(std::move(y[1]))) : Py_BuildValue("(N)", first);
    });
}

struct Pages {
    const void* handle;
    int64_t device, kv_heads, head_dim, code;
};
bool pages_of(PyObject* obj, Pages& p) {
    int64_t addr = 0;
    if ((PyObject*)Py_TYPE(obj) != g_pages || !attribute(obj, s_addr, addr) || addr == 0 || !attribute(obj, s_plain_device, p.device) || !attribute(obj, s_kv_heads, p.kv_heads) ||
        !attribute(obj, s_head_dim, p.head_dim) || !attribute(obj, s_code, p.code)) {
        return false;
    }
    p.handle = (const void*)addr;
    return true;
}
// The numbers that a PagedBatch keeps: tables, their stride and width, starts, lengths, sequences; prefix, its pages, its keys.
bool batch_of(PyObject* obj, int64_t device, int64_t (&v)[9]) {
    int64_t on = 0;
    if ((PyObject*)Py_TYPE(obj) != g_batch || !attribute(obj, s_plain_device, on) || on != device) {
        return false;
    }
    PyObject* const lists[2] = {PyObject_GetAttr(obj, s_rows), PyObject_GetAttr(obj, s_ahead)};
    bool ok = true;
    int at = 0;
    for (int i = 0; i < 2; i++) {
        const int want = i == 0 ? 6 : 3;
        ok = ok && lists[i] != nullptr && PyTuple_Check(lists[i]) && PyTuple_GET_SIZE(lists[i]) == want;
        for (int j = 0; j < want && ok; j++) {
            PyObject* const n = PyTuple_GET_ITEM(lists[i], j);
            v[at++] = n == Py_None ? 0 : PyLong_AsLongLong(n);
        }
        Py_XDECREF(lists[i]);
    }
    if (PyErr_Occurred() != nullptr) {
        PyErr_Clear();
        return false;
    }
    return ok;
}

PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t count) {  // pages, q, k, v, batch, rope or None
    return guarded([&]() -> PyObject* {
        Pages p;
        int64_t b[9], rope_addr = 0, rope_device = 0;
        if (count != 6 || !pages_of(args[0], p) || !batch_of(args[4], p.device, b) || !undisturbed()) {
            return not_plain();
        }
        if (args[5] != Py_None && ((PyObject*)Py_TYPE(args[5]) != g_rope || !attribute(args[5], s_addr, rope_addr) || rope_addr == 0 ||
                                   !attribute(args[5], s_plain_device, rope_device) || rope_device != p.device)) {
            return not_plain();
        }
        const at::Tensor *const q = plain_strided(args[1], 3, p.device), *const k = plain_strided(args[2], 3, p.device), *const v = plain_strided(args[3], 3, p.device);
        if (q == nullptr || k == nullptr || v == nullptr) {
            return not_plain();
        }
        const int elem = elem_of(*k);
        if (elem < 0 || (elem != 0 && elem != p.code) || elem_of(*q) != elem || elem_of(*v) != elem || k->size(1) != p.kv_heads || k->size(2) != p.head_dim ||
            v->sizes() != k->sizes() || q->size(0) != k->size(0) || q->size(2) != p.head_dim) {
            return not_plain();
        }
        at::Tensor y = like(*q);
        const int64_t strides[8] = {q->stride(0), q->stride(1), k->stride(0), k->stride(1), v->stride(0), v->stride(1), y.stride(0), y.stride(1)};
        const void *const qp = q->const_data_ptr(), *const kp = k->const_data_ptr(), *const vp = v->const_data_ptr();
        void *const yp = y.mutable_data_ptr(), *const stream = stream_of((int)p.device);
        const int heads = (int)q->size(1);
        const int64_t tokens = q->size(0);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = g_append(p.handle, (const void*)rope_addr, elem, heads, qp, kp, vp, yp, strides, tokens, (const int32_t*)b[0], b[1], b[2], (const int32_t*)b[3], (const int32_t*)b[4],
                      (int)b[5], b[8], 1, stream);
        Py_END_ALLOW_THREADS;
        return finish(rc, rc == 0 ? THPVariable_Wrap(std::move(y)) : nullptr);
    });
}

PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t count) {  // pages, q, batch, scale
    return guarded([&]() -> PyObject* {
        Pages p;
        int64_t b[9];
        if (count != 4 || !pages_of(args[0], p) || !PyFloat_CheckExact(args[3]) || !batch_of(args[2], p.device, b) || !undisturbed()) {
            return not_plain();
        }
        const at::Tensor* const q = plain_strided(args[1], 3, p.device);
        if (q == nullptr) {
            return not_plain();
        }
        const int elem = elem_of(*q), heads = (int)q->size(1);
        const int64_t tokens = q->size(0);
        if (elem < 0 || (elem != 0 && elem != p.code) || q->size(2) != p.head_dim || heads % p.kv_heads != 0) {
            return not_plain();
        }
        int64_t need = 0;
        int rc = g_attention_bytes(p.handle, elem, heads, tokens, b[5], b[8], &need);
        if (rc != 0) {
            return finish(rc, nullptr);
        }
        at::Tensor y = like(*q), space;
        if (need > 0) {
            space = at::cuda::empty({need}, q->options().dtype(at::kByte));
        }
        const int64_t strides[4] = {q->stride(0), q->stride(1), y.stride(0), y.stride(1)};
        const void* const qp = q->const_data_ptr();
        void *const yp = y.mutable_data_ptr(), *const sp = need > 0 ? space.mutable_data_ptr() : nullptr, *const stream = stream_of((int)p.device);
        const float scale = (float)PyFloat_AS_DOUBLE(args[3]);
        Py_BEGIN_ALLOW_THREADS;
        rc = g_attention(p.handle, elem, heads, qp, yp, strides, tokens, (const int32_t*)b[0], b[1], b[2], (const int32_t*)b[3], (const int32_t*)b[4], (int)b[5],
                         (const int32_t*)b[6], b[7], b[8], scale, 1, sp, need, stream);
        Py_END_ALLOW_THREADS;
        return finish(rc, rc == 0 ? THPVariable_Wrap(std::move(y)) : nullptr);
    });
}

PyObject* verify(PyObject*, PyObject* const* args, Py_ssize_t count) {  // target, drafts, uniforms, draft_probs, counts, temperature
    return guarded([&]() -> PyObject* {
        if (count != 6 || !undisturbed()) {
            return not_plain();
        }
        const at::Tensor* const x = plain_strided(args[0], 3, -1);
        if (x == nullptr || elem_of(*x) < 0 || x->size(1) < 2) {
            return not_plain();
        }
        const int64_t device = x->get_device(), n = x->size(0), rows = x->size(1), vocab = x->size(2);
        const bool logits = args[5] != Py_None;
        if (logits && !PyFloat_CheckExact(args[5])) {
            return not_plain();
        }
        const double temperature = logits ? PyFloat_AS_DOUBLE(args[5]) : 0.0;
        const at::Tensor* const drafts = whole(args[1], {n, rows - 1}, device);
        const at::Tensor* const u = plain(args[2], at::kFloat);
        const at::Tensor* q = nullptr;
        const at::Tensor* counts = nullptr;
        if (drafts == nullptr || u == nullptr || u->get_device() != device || u->sizes() != at::IntArrayRef({n, rows})) {
            return not_plain();
        }
        if (args[3] != Py_None) {
            q = plain_strided(args[3], 3, device);
            if (q == nullptr || q->scalar_type() != at::kFloat || q->sizes() != at::IntArrayRef({n, rows - 1, vocab})) {
                return not_plain();
            }
        }
        if (args[4] != Py_None) {
            counts = whole(args[4], {n}, device);
            if (counts == nullptr) {
                return not_plain();
            }
        }
        int64_t need = 0;
        int rc = g_verify_bytes(n, rows - 1, vocab, logits, &need);
        if (rc != 0) {
            return finish(rc, nullptr);
        }
        const at::TensorOptions options = x->options().dtype(at::kInt);
        at::Tensor accepted = at::cuda::empty({n}, options), tokens = at::cuda::empty({n, rows}, options), space;
        if (need > 0) {
            space = at::cuda::empty({need}, options.dtype(at::kByte));
        }
        const void* const xp = x->const_data_ptr();
        const int64_t xb = x->stride(0), xr = x->stride(1), qb = q != nullptr ? q->stride(0) : 0, qr = q != nullptr ? q->stride(1) : 0;
        const int32_t *const dp = (const int32_t*)drafts->const_data_ptr(), *const cp = counts != nullptr ? (const int32_t*)counts->const_data_ptr() : nullptr;
        const float *const up = (const float*)u->const_data_ptr(), *const qp = q != nullptr ? (const float*)q->const_data_ptr() : nullptr;
        int32_t *const ap = (int32_t*)accepted.mutable_data_ptr(), *const tp = (int32_t*)tokens.mutable_data_ptr();
        void *const sp = need > 0 ? space.mutable_data_ptr() : nullptr, *const stream = stream_of((int)device);
        const int elem = elem_of(*x);
        Py_BEGIN_ALLOW_THREADS;
        rc = g_verify((int)device, elem, xp, xb, xr, dp, qp, qb, qr, up, cp, n, rows - 1, vocab, logits, temperature, ap, tp, sp, need, stream);
        Py_END_ALLOW_THREADS;
        if (rc != 0) {
            return finish(rc, nullptr);
        }
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(accepted)), THPVariable_Wrap(std::move(tokens)));
    });
}

// bind_paged(Rope, PagedCache, PagedBatch, addresses of jq_rope_apply, jq_pages_append, jq_pages_attention_bytes, jq_pages_attention, jq_verify_bytes, jq_verify_drafts)
PyObject* bind_paged(PyObject*, PyObject* args) {
    PyObject *r, *p, *b;
    unsigned long long f[6];
    if (!PyArg_ParseTuple(args, "OOOKKKKKK", &r, &p, &b, &f[0], &f[1], &f[2], &f[3], &f[4], &f[5])) {
        return nullptr;
    }
    Py_XSETREF(g_rope, Py_NewRef(r));
    Py_XSETREF(g_pages, Py_NewRef(p));
    Py_XSETREF(g_batch, Py_NewRef(b));
    g_rope_apply = (RopeApply)f[0];
    g_append = (Append)f[1];
    g_attention_bytes = (AttentionBytes)f[2];
    g_attention = (Attention)f[3];
    g_verify_bytes = (VerifyBytes)f[4];
    g_verify = (Verify)f[5];
    Py_RETURN_NONE;
}

// bind(weight class, check, addresses of jq_linear_f32, jq_linear_bf16, jq_linear_backward_f32, jq_dequantize, jq_quantize_q8_0)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *weight, *check;
    unsigned long long f[5];
    if (!PyArg_ParseTuple(args, "OOKKKKK", &weight, &check, &f[0], &f[1], &f[2], &f[3], &f[4])) {
        return nullptr;
    }
    Py_XSETREF(g_weight, Py_NewRef(weight));
    Py_XSETREF(g_check, Py_NewRef(check));
    g_linear = (Linear)f[0];
    g_linear_bf16 = (Linear)f[1];
    g_backward = (Backward)f[2];
    g_dequantize = (Dequantize)f[3];
    g_quantize = (Quantize)f[4];
    Py_RETURN_NONE;
}

PyMethodDef METHODS[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
    {"linear_bf16", (PyCFunction)(void (*)(void))linear_bf16, METH_FASTCALL, nullptr},
    {"backward", (PyCFunction)(void (*)(void))backward, METH_FASTCALL, nullptr},
    {"dequantize", (PyCFunction)(void (*)(void))dequantize, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)(void))quantize, METH_FASTCALL, nullptr},
    {"bind_paged", bind_paged, METH_VARARGS, nullptr},
    {"rope", (PyCFunction)(void (*)(void))rope, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
    {"verify", (PyCFunction)(void (*)(void))verify, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front(void) {
    s_addr = PyUnicode_InternFromString("_addr");
    s_dims = PyUnicode_InternFromString("_dims");
    s_device = PyUnicode_InternFromString("_device");
    s_plain_device = PyUnicode_InternFromString("device");
    s_kv_heads = PyUnicode_InternFromString("kv_heads");
    s_head_dim = PyUnicode_InternFromString("head_dim");
    s_code = PyUnicode_InternFromString("_code");
    s_rows = PyUnicode_InternFromString("_rows");
    s_ahead = PyUnicode_InternFromString("_ahead");
    for (PyObject* name : {s_addr, s_dims, s_device, s_plain_device, s_kv_heads, s_head_dim, s_code, s_rows, s_ahead}) {
        if (name == nullptr) {
            return nullptr;
        }
    }
    return PyModule_Create(&MODULE);
}
