// CPython side of the call path (module lumen_b200._host): reads tensors' pointers, shapes and strides and calls the C
// ABI without ctypes structures in between. A call of a compiled function or of an attention / GEMM entry is host work
// of a few microseconds in front of kernels that may take less: descriptors built attribute by attribute in Python took
// 2 us each, three times a kernel launch.
//
// Tensors are duck-typed as everywhere in the package: anything with data_ptr(), shape, stride() and dtype.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <structmember.h>

#include <algorithm>
#include <deque>
#include <new>
#include <unordered_map>
#include <vector>

#include "../../include/lumen_b200.h"

namespace {

struct Names {
    PyObject *dtype, *shape, *stride, *data_ptr, *is_cuda, *is_contiguous, *get_device;
} names;
PyObject* code_of = nullptr;     // dict: dtype object or name -> lb_dtype code, filled as dtypes are met
PyObject* code_miss = nullptr;   // callable(dtype) -> code, for the first meeting
PyObject* raise_error = nullptr; // callable(status): raises the library's error
PyObject* raw_stream = nullptr;     // callable(device index) -> torch's current stream handle, or None
PyObject* current_stream = nullptr; // callable() -> the caller's current stream handle

bool dtype_code(PyObject* t, int32_t* out) {
    PyObject* d = PyObject_GetAttr(t, names.dtype);
    if (!d) return false;
    PyObject* c = PyDict_GetItemWithError(code_of, d);  // borrowed
    if (c) {
        *out = (int32_t)PyLong_AsLong(c);
        Py_DECREF(d);
        return true;
    }
    if (PyErr_Occurred()) {
        Py_DECREF(d);
        return false;
    }
    PyObject* made = PyObject_CallOneArg(code_miss, d);
    bool ok = made && PyDict_SetItem(code_of, d, made) == 0;
    if (ok) *out = (int32_t)PyLong_AsLong(made);
    Py_XDECREF(made);
    Py_DECREF(d);
    return ok;
}

bool read_pointer(PyObject* t, void** out) {
    PyObject* p = PyObject_CallMethodNoArgs(t, names.data_ptr);
    if (!p) return false;
    *out = PyLong_AsVoidPtr(p);
    Py_DECREF(p);
    return !PyErr_Occurred();
}

// A sequence of at most LB_MAX_RANK integers (a tuple, as torch and this package give it, or what another framework does).
// Steals the reference.
bool read_longs(PyObject* tuple, int64_t* out, int32_t* count, const char* what) {
    bool ok = false;
    if (tuple && !PyTuple_Check(tuple)) Py_SETREF(tuple, PySequence_Tuple(tuple));
    if (tuple && PyTuple_GET_SIZE(tuple) <= LB_MAX_RANK) {
        *count = (int32_t)PyTuple_GET_SIZE(tuple);
        ok = true;
        for (int32_t k = 0; k < *count; k++) out[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, k));
        if (PyErr_Occurred()) ok = false;
    } else if (tuple) {
        PyErr_Format(PyExc_TypeError, "a tensor's %s must be at most %d integers", what, LB_MAX_RANK);
    }
    Py_XDECREF(tuple);
    return ok;
}

bool truth(PyObject* b, bool* out) {  // steals b
    if (!b) return false;
    int v = PyObject_IsTrue(b);
    Py_DECREF(b);
    *out = v == 1;
    return v >= 0;
}

bool describe_view(PyObject* t, lb_tensor* out) {
    int32_t strides = 0;
    if (!dtype_code(t, &out->dtype) || !read_pointer(t, &out->ptr)) return false;
    if (!read_longs(PyObject_GetAttr(t, names.shape), out->shape, &out->rank, "shape")) return false;
    if (!read_longs(PyObject_CallMethodNoArgs(t, names.stride), out->stride, &strides, "stride")) return false;
    if (strides != out->rank) {
        PyErr_SetString(PyExc_TypeError, "a tensor needs as many strides as dimensions");
        return false;
    }
    return true;
}

bool describe(PyObject* t, lb_tensor* out) {
    PyObject* cuda = PyObject_GetAttr(t, names.is_cuda);
    bool on_gpu = true;
    if (!cuda) PyErr_Clear();  // a tensor type without the attribute answers for itself
    else if (!truth(cuda, &on_gpu)) return false;
    if (!on_gpu) {
        PyErr_SetString(PyExc_ValueError, "expected a CUDA tensor");
        return false;
    }
    return describe_view(t, out);
}

PyObject* finish(int status) {
    if (status == LB_OK) Py_RETURN_NONE;
    PyObject* r = PyObject_CallFunction(raise_error, "i", status);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "the library reported an error");
    return nullptr;
}

bool wants(Py_ssize_t got, Py_ssize_t want) {
    if (got == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return false;
}

// setup(codes, miss, raise, current_stream, raw_stream)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 5)) return nullptr;
    Py_XSETREF(code_of, Py_NewRef(a[0]));
    Py_XSETREF(code_miss, Py_NewRef(a[1]));
    Py_XSETREF(raise_error, Py_NewRef(a[2]));
    Py_XSETREF(current_stream, Py_NewRef(a[3]));
    Py_XSETREF(raw_stream, Py_NewRef(a[4]));
    Py_RETURN_NONE;
}

bool attn_desc(PyObject* const* a, lb_attn_desc* d) {
    d->scale = (float)PyFloat_AsDouble(a[0]);
    d->causal = (int32_t)PyLong_AsLong(a[1]);
    d->causal_offset = PyLong_AsLongLong(a[2]);
    return !PyErr_Occurred();
}

// attention_fwd(scale, causal, offset, q, k, v, o, lse, stream)
PyObject* attention_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    lb_attn_desc d;
    lb_tensor t[5];
    if (!wants(n, 9) || !attn_desc(a, &d)) return nullptr;
    for (int k = 0; k < 5; k++)
        if (!describe(a[3 + k], &t[k])) return nullptr;
    void* stream = PyLong_AsVoidPtr(a[8]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_attention_fwd(&d, &t[0], &t[1], &t[2], &t[3], &t[4], stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// attention_bwd_scratch_bytes(scale, causal, offset, q, k)
PyObject* attention_bwd_scratch_bytes(PyObject*, PyObject* const* a, Py_ssize_t n) {
    lb_attn_desc d;
    lb_tensor q, k;
    if (!wants(n, 5) || !attn_desc(a, &d) || !describe(a[3], &q) || !describe(a[4], &k)) return nullptr;
    return PyLong_FromSize_t(lb_attention_bwd_scratch_bytes(&d, &q, &k));
}

// attention_bwd(scale, causal, offset, q, k, v, o, dO, lse, delta, dq_accum or None, dq, dk, dv, scratch pointer, scratch bytes, stream)
PyObject* attention_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    lb_attn_desc d;
    lb_tensor t[11];
    if (!wants(n, 17) || !attn_desc(a, &d)) return nullptr;
    const bool atomic = a[10] != Py_None;
    for (int k = 0; k < 11; k++)
        if ((k != 7 || atomic) && !describe(a[3 + k], &t[k])) return nullptr;
    void* scratch = PyLong_AsVoidPtr(a[14]);
    const size_t bytes = PyLong_AsSize_t(a[15]);
    void* stream = PyLong_AsVoidPtr(a[16]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = atomic ? lb_attention_bwd_atomic(&d, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], &t[7], &t[8], &t[9], &t[10], stream)
                : lb_attention_bwd_scratch(&d, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], &t[8], &t[9], &t[10], scratch, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// gemm(a, b, out, aux or None, epilogue, kernel, scratch pointer, scratch bytes, stream)
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    lb_tensor ta, tb;
    lb_gemm_out out = {};
    lb_gemm_cfg cfg = {};
    if (!wants(n, 9) || !describe(a[0], &ta) || !describe(a[1], &tb) || !describe(a[2], &out.product)) return nullptr;
    if (a[3] != Py_None && !describe(a[3], &out.aux)) return nullptr;
    out.epilogue = (int32_t)PyLong_AsLong(a[4]);
    cfg.kernel = (int32_t)PyLong_AsLong(a[5]);
    cfg.scratch = PyLong_AsVoidPtr(a[6]);
    cfg.scratch_bytes = (size_t)PyLong_AsUnsignedLongLong(a[7]);
    void* stream = PyLong_AsVoidPtr(a[8]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_gemm(&ta, &tb, &out, &cfg, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// ---- operators of a decoder layer's step ----------------------------------------------------------------------------
// These look where a tensor lives: kernels launched on the current device do not read another one's memory.
struct Here {
    int device = -1;
    bool known = false;
    bool current(int* out) {
        if (!known && lb_get_device(&device) != LB_OK) device = -1;  // no GPU: the call itself says so
        known = true;
        *out = device;
        return device >= 0;
    }
    bool is(long at) {  // sets a Python error where it is not
        int now;
        if (at < 0) PyErr_SetString(PyExc_ValueError, "expected a CUDA tensor");
        else if (current(&now) && at != now) PyErr_Format(PyExc_ValueError, "a tensor is on GPU %ld, the current one is GPU %d", at, now);
        else return true;
        return false;
    }
};

// DLPack's exchange table of C functions, as an array type offers it in `__dlpack_c_exchange_api__` (DLPack 1.3, torch 2.11): one call reads all of a tensor
// in 30 ns, where its methods and attributes take 350.
struct DlTensor {
    void* data;
    int32_t device_type, device_id, ndim;
    uint8_t code, bits;
    uint16_t lanes;
    int64_t *shape, *strides;
    uint64_t byte_offset;
};
struct DlTable {
    uint32_t major, minor;
    void *previous, *allocate, *from_object, *to_object;
    int (*read)(void* object, DlTensor* out);  // may be null
    void* current_stream;
};
constexpr int kDlCuda = 2;

// The table of an object's type, or null; the type met last is remembered (and kept alive).
const DlTable* dl_table(PyObject* t) {
    static PyObject* type = nullptr;
    static const DlTable* table = nullptr;
    if ((PyObject*)Py_TYPE(t) == type) return table;
    PyObject* capsule = PyObject_GetAttrString((PyObject*)Py_TYPE(t), "__dlpack_c_exchange_api__");
    const DlTable* found = nullptr;
    if (capsule && PyCapsule_IsValid(capsule, "dlpack_exchange_api")) {
        found = (const DlTable*)PyCapsule_GetPointer(capsule, "dlpack_exchange_api");
        if (found->major != 1 || !found->read) found = nullptr;
    }
    PyErr_Clear();
    Py_XDECREF(capsule);
    Py_XSETREF(type, Py_NewRef((PyObject*)Py_TYPE(t)));
    return table = found;
}
int dl_dtype(const DlTensor& d) {
    static const struct { uint8_t code, bits; int dtype; } known[] = {{4, 16, LB_BF16}, {2, 32, LB_F32}, {2, 16, LB_F16}, {0, 64, LB_I64}, {0, 32, LB_I32}, {1, 8, LB_U8}};
    for (auto& k : known)
        if (k.code == d.code && k.bits == d.bits && d.lanes == 1) return k.dtype;
    return -1;
}
// 1: read; 0: the tensor has to be asked in the ordinary way; -1: a Python error
int read_dl(PyObject* t, lb_tensor* out, Here& here) {
    const DlTable* table = dl_table(t);
    if (!table) return 0;
    DlTensor d = {};
    if (table->read(t, &d) != 0) {
        PyErr_Clear();
        return 0;
    }
    const int dtype = dl_dtype(d);
    if (dtype < 0 || d.ndim > LB_MAX_RANK) return 0;
    if (!here.is(d.device_type == kDlCuda ? d.device_id : -1)) return -1;
    out->ptr = (char*)d.data + d.byte_offset, out->dtype = dtype, out->rank = d.ndim;
    int64_t step = 1;
    for (int k = d.ndim; k-- > 0; step *= d.shape[k]) out->shape[k] = d.shape[k], out->stride[k] = d.strides ? d.strides[k] : step;
    return out->ptr || step == 0;  // (a wrapper around other tensors has elements and no memory: its own methods have the say)
}
bool describe_here(PyObject* t, lb_tensor* out, Here& here) {
    if (const int read = read_dl(t, out, here)) return read > 0;
    PyObject* g = PyObject_CallMethodNoArgs(t, names.get_device);
    if (!g) {  // the package's own tensors do not say
        if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return false;
        PyErr_Clear();
        return describe(t, out);
    }
    const long at = PyLong_AsLong(g);
    Py_DECREF(g);
    return !(at == -1 && PyErr_Occurred()) && here.is(at) && describe_view(t, out);
}

// A call's workspace, from `take(bytes)` where it needs any; held until the call's kernels are queued.
struct Scratch {
    PyObject* held = nullptr;
    void* ptr = nullptr;
    ~Scratch() { Py_XDECREF(held); }
    bool get(PyObject* take, size_t bytes) {
        if (!bytes) return true;
        held = PyObject_CallFunction(take, "n", (Py_ssize_t)bytes);
        return held && read_pointer(held, &ptr);
    }
};

// qk_norm_rope(eps, interleaved, q, k, cos, sin, positions, q_weight, k_weight, q_out, k_out, stream), None where the ABI takes a null
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 12)) return nullptr;
    lb_rope_desc d = {(float)PyFloat_AsDouble(a[0]), (int32_t)PyLong_AsLong(a[1])};
    lb_tensor t[9];
    const lb_tensor* p[9];
    Here here;
    for (int k = 0; k < 9; k++) {
        p[k] = a[2 + k] == Py_None ? nullptr : &t[k];
        if (p[k] && !describe_here(a[2 + k], &t[k], here)) return nullptr;
    }
    void* stream = PyLong_AsVoidPtr(a[11]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_qk_norm_rope(&d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// qk_norm_rope_bwd(eps, interleaved, d_q_out, d_k_out, q, k, cos, sin, positions, q_weight, k_weight, d_q, d_k, d_q_weight, d_k_weight, take, stream)
PyObject* qk_norm_rope_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 17)) return nullptr;
    lb_rope_desc d = {(float)PyFloat_AsDouble(a[0]), (int32_t)PyLong_AsLong(a[1])};
    lb_tensor t[13];
    const lb_tensor* p[13];
    Here here;
    for (int k = 0; k < 13; k++) {
        p[k] = a[2 + k] == Py_None ? nullptr : &t[k];
        if (p[k] && !describe_here(a[2 + k], &t[k], here)) return nullptr;
    }
    void* stream = PyLong_AsVoidPtr(a[16]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t dim = p[2] && t[2].rank == 4 ? t[2].shape[3] : 0;
    const size_t bytes = (p[7] || p[8]) && dim > 0 && dim <= 4096 ? lb_qk_norm_rope_bwd_scratch_bytes((int)dim) : 0;
    Scratch scratch;
    if (!scratch.get(a[15], bytes)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_qk_norm_rope_bwd(&d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], p[10], p[11], p[12], scratch.ptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// gated_mlp_fwd(activation, x, w_gate_up, w_down, residual, y, gate_up, h, take, stream)
PyObject* gated_mlp_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 10)) return nullptr;
    const int act = (int)PyLong_AsLong(a[0]);
    lb_tensor t[7];
    const lb_tensor* p[7];
    Here here;
    for (int k = 0; k < 7; k++) {
        p[k] = a[1 + k] == Py_None ? nullptr : &t[k];
        if (p[k] && !describe_here(a[1 + k], &t[k], here)) return nullptr;
    }
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    size_t bytes = 0;
    int rc = lb_gated_mlp_fwd_scratch_bytes(act, p[0], p[1], p[2], p[4], p[5], p[6], &bytes);
    if (rc != LB_OK) return finish(rc);
    Scratch scratch;
    if (!scratch.get(a[8], bytes)) return nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_gated_mlp_fwd(act, p[0], p[1], p[2], p[3], p[4], p[5], p[6], scratch.ptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// gated_mlp_bwd(activation, d_y, x, w_gate_up, w_down, gate_up, h, d_x, d_w_gate_up, d_w_down, take, stream)
PyObject* gated_mlp_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 12)) return nullptr;
    const int act = (int)PyLong_AsLong(a[0]);
    lb_tensor t[9];
    Here here;
    for (int k = 0; k < 9; k++)
        if (!describe_here(a[1 + k], &t[k], here)) return nullptr;
    void* stream = PyLong_AsVoidPtr(a[11]);
    if (PyErr_Occurred()) return nullptr;
    size_t bytes = 0;
    int rc = lb_gated_mlp_bwd_scratch_bytes(act, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], &t[7], &t[8], &bytes);
    if (rc != LB_OK) return finish(rc);
    Scratch scratch;
    if (!scratch.get(a[10], bytes)) return nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_gated_mlp_bwd(act, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], &t[7], &t[8], scratch.ptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// linear_cross_entropy(reduction, ignore_index, x, weight, targets, loss, lse, take, stream)
PyObject* linear_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 9)) return nullptr;
    lb_loss_desc d = {(int32_t)PyLong_AsLong(a[0]), 0, PyLong_AsLongLong(a[1])};
    void* stream = PyLong_AsVoidPtr(a[8]);
    if (PyErr_Occurred()) return nullptr;
    lb_tensor t[5];
    Here here;
    for (int k = 0; k < 5; k++)
        if (!describe_here(a[2 + k], &t[k], here)) return nullptr;
    size_t bytes = 0;
    int rc = lb_linear_cross_entropy_scratch_bytes(&d, &t[0], &t[1], &t[2], &bytes);
    if (rc != LB_OK) return finish(rc);
    Scratch scratch;
    if (!scratch.get(a[7], bytes)) return nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_linear_cross_entropy(&d, &t[0], &t[1], &t[2], &t[3], &t[4], scratch.ptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// linear_cross_entropy_bwd(reduction, ignore_index, d_loss or None, x, weight, targets, lse, d_x, d_weight, take, stream)
PyObject* linear_cross_entropy_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 11)) return nullptr;
    lb_loss_desc d = {(int32_t)PyLong_AsLong(a[0]), 0, PyLong_AsLongLong(a[1])};
    void* stream = PyLong_AsVoidPtr(a[10]);
    if (PyErr_Occurred()) return nullptr;
    lb_tensor t[7];
    Here here;
    for (int k = 0; k < 7; k++)
        if ((k || a[2] != Py_None) && !describe_here(a[2 + k], &t[k], here)) return nullptr;
    size_t bytes = 0;
    int rc = lb_linear_cross_entropy_bwd_scratch_bytes(&d, &t[1], &t[2], &t[3], &t[5], &t[6], &bytes);
    if (rc != LB_OK) return finish(rc);
    Scratch scratch;
    if (!scratch.get(a[9], bytes)) return nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_linear_cross_entropy_bwd(&d, a[2] == Py_None ? nullptr : &t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], scratch.ptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// The tensors of a sequence; `gaps`: None stands for a tensor that there is not, which has no memory.
bool describe_all(PyObject* sequence, std::vector<lb_tensor>& out, Here& here, bool gaps) {
    PyObject* all = PySequence_Fast(sequence, "expected a sequence of tensors");
    if (!all) return false;
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(all);
    bool ok = count <= INT32_MAX;
    if (!ok) PyErr_SetString(PyExc_ValueError, "too many tensors");
    try {
        if (ok) out.resize((size_t)count);
    } catch (const std::bad_alloc&) {
        Py_DECREF(all);
        PyErr_NoMemory();
        return false;
    }
    for (Py_ssize_t i = 0; ok && i < count; i++) {
        PyObject* t = PySequence_Fast_GET_ITEM(all, i);
        if (gaps && t == Py_None) out[i] = lb_tensor{};
        else ok = describe_here(t, &out[i], here);
    }
    Py_DECREF(all);
    return ok;
}

// clip_grad_norm(tensors, outputs or None (in place), max_norm or None (the norm alone), norm, take, stream); sequences of tensors
PyObject* clip_grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 6)) return nullptr;
    const bool clips = a[2] != Py_None;
    const double most = clips ? PyFloat_AsDouble(a[2]) : 0.0;
    void* stream = PyLong_AsVoidPtr(a[5]);
    if (PyErr_Occurred()) return nullptr;
    std::vector<lb_tensor> t[2];
    lb_tensor norm;
    Here here;
    for (int k = 0; k < 2; k++)
        if (a[k] != Py_None && !describe_all(a[k], t[k], here, false)) return nullptr;
    if (a[1] != Py_None && t[0].size() != t[1].size()) {
        PyErr_Format(PyExc_ValueError, "%zu tensors and %zu results", t[0].size(), t[1].size());
        return nullptr;
    }
    if (!describe_here(a[3], &norm, here)) return nullptr;
    const int count = (int)t[0].size();
    const size_t bytes = lb_grad_norm_scratch_bytes(count);
    Scratch scratch;
    if (!scratch.get(a[4], bytes)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = clips ? lb_clip_grad_norm(t[0].data(), a[1] == Py_None ? t[0].data() : t[1].data(), count, most, &norm, scratch.ptr, bytes, stream)
               : lb_grad_norm(t[0].data(), count, &norm, scratch.ptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters (these three: sequences or None), step, lr (numbers or tensors),
//            beta1, beta2, eps, weight_decay, norm or None, max_norm, stream)
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 16)) return nullptr;
    lb_adamw_desc d = {};
    const bool counted = PyLong_Check(a[7]), fixed = PyFloat_Check(a[8]) || PyLong_Check(a[8]);
    if (counted) d.step = PyLong_AsLongLong(a[7]);
    if (fixed) d.lr = PyFloat_AsDouble(a[8]);
    d.beta1 = PyFloat_AsDouble(a[9]), d.beta2 = PyFloat_AsDouble(a[10]), d.eps = PyFloat_AsDouble(a[11]), d.weight_decay = PyFloat_AsDouble(a[12]);
    d.max_norm = a[13] == Py_None ? 0.0 : PyFloat_AsDouble(a[14]);
    void* stream = PyLong_AsVoidPtr(a[15]);
    if (PyErr_Occurred()) return nullptr;
    std::vector<lb_tensor> t[7];
    Here here;
    for (int k = 0; k < 7; k++) {
        if (k >= 4 && a[k] == Py_None) continue;
        if (!describe_all(a[k], t[k], here, k == 6)) return nullptr;
        if (t[k].size() != t[0].size()) {
            static const char* const what[] = {"", "gradients", "first moments", "second moments", "scales of first moments", "scales of second moments", "float32 copies"};
            PyErr_Format(PyExc_ValueError, "%zu parameters and %zu %s", t[0].size(), t[k].size(), what[k]);
            return nullptr;
        }
    }
    lb_tensor step, lr, norm;
    if ((!counted && !describe_here(a[7], &step, here)) || (!fixed && !describe_here(a[8], &lr, here)) || (a[13] != Py_None && !describe_here(a[13], &norm, here))) return nullptr;
    auto list = [&](int k) { return a[k] == Py_None ? nullptr : t[k].data(); };
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_adamw_step(&d, t[0].data(), t[1].data(), t[2].data(), t[3].data(), list(4), list(5), list(6), (int)t[0].size(), counted ? nullptr : &step,
                       fixed ? nullptr : &lr, a[13] == Py_None ? nullptr : &norm, stream);
    Py_END_ALLOW_THREADS
    return finish(rc);
}

// ---- the calls of one compiled function -----------------------------------------------------------------------------
// The signatures a `lumen_b200.compile`d function has met whose arguments are all tensors, by a hash of the arguments' types,
// dtypes and shapes and of the device: a call costs the same with one signature as with thousands (a cache that grows by a token a
// call). `call(args, stream, device)` finds the one that `args` match, runs its plan and returns its results; it returns None
// when the call needs the general path (an unknown signature, host or strided or foreign arguments).
struct Arg {
    PyObject* type;   // exact type
    PyObject* dtype;  // the dtype attribute
    int32_t rank;
    int64_t shape[LB_MAX_RANK];
};
struct Entry {
    std::vector<Arg> args;  // owns its references
    std::vector<char> torch;  // by argument: a torch tensor, which has to be on the GPU and contiguous
    long device;            // the GPU that the plan's workspace and results live on (-1: the process has one)
    const lb_plan* plan;
    void* workspace;
    std::vector<void*> outputs;
    PyObject *signature, *returned, *keep;  // keep: the last call's arguments, alive until the next call
};
struct CallTable {
    PyObject_HEAD
    std::deque<Entry>* entries;  // references stay valid while other threads add signatures
    std::unordered_multimap<uint64_t, Entry*>* index;
    std::vector<PyObject*>* types;  // the argument types of the entries (held by them): anything else is not looked up
    PyObject* latest;  // the signature object of the latest call
};

void drop(Entry& e) {
    for (Arg& a : e.args) Py_XDECREF(a.type), Py_XDECREF(a.dtype);
    Py_XDECREF(e.signature), Py_XDECREF(e.returned), Py_XDECREF(e.keep);
}
PyObject* table_new(PyTypeObject* type, PyObject*, PyObject*) {
    CallTable* t = (CallTable*)type->tp_alloc(type, 0);
    if (!t) return nullptr;
    t->entries = new (std::nothrow) std::deque<Entry>();
    t->index = new (std::nothrow) std::unordered_multimap<uint64_t, Entry*>();
    t->types = new (std::nothrow) std::vector<PyObject*>();
    t->latest = Py_NewRef(Py_None);
    if (!t->entries || !t->index || !t->types) {
        Py_DECREF(t);
        return PyErr_NoMemory();
    }
    return (PyObject*)t;
}
int table_traverse(CallTable* t, visitproc visit, void* arg) {
    if (t->entries)
        for (Entry& e : *t->entries) {
            Py_VISIT(e.signature);
            Py_VISIT(e.returned);
            Py_VISIT(e.keep);
        }
    Py_VISIT(t->latest);
    return 0;
}
int table_clear(CallTable* t) {
    std::deque<Entry> gone;
    if (t->index) t->index->clear();
    if (t->types) t->types->clear();
    if (t->entries) gone.swap(*t->entries);
    for (Entry& e : gone) drop(e);
    Py_CLEAR(t->latest);
    return 0;
}
void table_dealloc(CallTable* t) {
    PyObject_GC_UnTrack(t);
    table_clear(t);
    delete t->entries;
    delete t->index;
    delete t->types;
    Py_TYPE(t)->tp_free((PyObject*)t);
}

// What a call's argument is looked up by; the references are the caller's (`dtype` is new, `type` borrowed).
bool read_arg(PyObject* x, Arg* out) {
    out->type = (PyObject*)Py_TYPE(x);
    out->dtype = PyObject_GetAttr(x, names.dtype);
    return out->dtype && read_longs(PyObject_GetAttr(x, names.shape), out->shape, &out->rank, "shape");
}
bool hash_args(const Arg* args, size_t count, long device, uint64_t* out) {
    uint64_t h = (uint64_t)device + 0x9e3779b97f4a7c15ull;
    auto mix = [&](uint64_t v) { h = (h ^ v) * 0xff51afd7ed558ccdull, h ^= h >> 32; };
    for (size_t k = 0; k < count; k++) {
        const Py_hash_t d = PyObject_Hash(args[k].dtype);
        if (d == -1 && PyErr_Occurred()) return false;
        mix((uint64_t)(uintptr_t)args[k].type), mix((uint64_t)d), mix((uint64_t)args[k].rank);
        for (int32_t r = 0; r < args[k].rank; r++) mix((uint64_t)args[k].shape[r]);
    }
    *out = h;
    return true;
}

// add(args, torch_flags, device, plan handle, workspace pointer, output pointers, signature, returned)
PyObject* table_add(CallTable* t, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 8)) return nullptr;
    if (!PyTuple_Check(a[0]) || !PyTuple_Check(a[1]) || !PyTuple_Check(a[5]) || PyTuple_GET_SIZE(a[0]) != PyTuple_GET_SIZE(a[1])) {
        PyErr_SetString(PyExc_TypeError, "add: tuples of arguments, flags and output pointers");
        return nullptr;
    }
    Entry e = {};
    try {
        e.device = PyLong_AsLong(a[2]);
        e.plan = (const lb_plan*)PyLong_AsVoidPtr(a[3]);
        e.workspace = PyLong_AsVoidPtr(a[4]);
        for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(a[5]); k++) e.outputs.push_back(PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[5], k)));
        bool ok = !PyErr_Occurred();
        for (Py_ssize_t k = 0; ok && k < PyTuple_GET_SIZE(a[0]); k++) {
            e.args.push_back(Arg{});
            ok = read_arg(PyTuple_GET_ITEM(a[0], k), &e.args.back());
            Py_XINCREF(e.args.back().type);
            e.torch.push_back(PyTuple_GET_ITEM(a[1], k) == Py_True);
        }
        uint64_t h = 0;
        if (!ok || !hash_args(e.args.data(), e.args.size(), e.device, &h)) {
            drop(e);
            return nullptr;
        }
        for (const Arg& arg : e.args)
            if (std::find(t->types->begin(), t->types->end(), arg.type) == t->types->end()) t->types->push_back(arg.type);
        t->entries->push_back(e);
        e = {};  // the table's now
        Entry& kept = t->entries->back();
        kept.signature = Py_NewRef(a[6]), kept.returned = Py_NewRef(a[7]);
        t->index->emplace(h, &kept);
    } catch (const std::bad_alloc&) {
        drop(e);
        return PyErr_NoMemory();
    }
    Py_RETURN_NONE;
}

bool same_args(const Arg* got, const Entry& e) {
    for (size_t k = 0; k < e.args.size(); k++) {
        const Arg& want = e.args[k];
        if (got[k].type != want.type || got[k].rank != want.rank) return false;
        for (int32_t r = 0; r < want.rank; r++)
            if (got[k].shape[r] != want.shape[r]) return false;
        if (got[k].dtype != want.dtype) {
            const int same = PyObject_RichCompareBool(got[k].dtype, want.dtype, Py_EQ);
            if (same < 0) PyErr_Clear();
            if (same <= 0) return false;
        }
    }
    return true;
}
// 1: the torch tensor can be read where it is; 0: it cannot (on the host, strided, on another GPU); -1: a Python error
int in_place(PyObject* x, long device) {
    bool yes = false;
    if (!truth(PyObject_GetAttr(x, names.is_cuda), &yes)) return -1;
    if (!yes) return 0;
    if (!truth(PyObject_CallMethodNoArgs(x, names.is_contiguous), &yes)) return -1;
    if (!yes) return 0;
    if (device >= 0) {
        PyObject* g = PyObject_CallMethodNoArgs(x, names.get_device);
        if (!g) return -1;
        const long at = PyLong_AsLong(g);
        Py_DECREF(g);
        if (at != device) return PyErr_Occurred() ? -1 : 0;
    }
    return 1;
}

// The entry that the arguments match, or null (with a Python error set where reading one failed).
Entry* find(CallTable* t, PyObject* args, long device) {
    constexpr Py_ssize_t kMost = 64;
    const Py_ssize_t count = PyTuple_GET_SIZE(args);
    if (count > kMost) return nullptr;
    for (Py_ssize_t k = 0; k < count; k++)
        if (std::find(t->types->begin(), t->types->end(), (PyObject*)Py_TYPE(PyTuple_GET_ITEM(args, k))) == t->types->end()) return nullptr;
    Arg got[kMost];
    Py_ssize_t read = 0;
    bool ok = true;
    for (; ok && read < count; read++) ok = read_arg(PyTuple_GET_ITEM(args, read), &got[read]);
    Entry* found = nullptr;
    uint64_t h = 0;
    if (ok && hash_args(got, (size_t)count, device, &h)) {
        auto range = t->index->equal_range(h);
        for (auto it = range.first; it != range.second && !found; ++it)
            if ((Py_ssize_t)it->second->args.size() == count && it->second->device == device && same_args(got, *it->second)) found = it->second;
    }
    for (Py_ssize_t k = 0; k < read; k++) Py_XDECREF(got[k].dtype);
    return found;
}

// call(args, stream, device): stream 0 means the caller's current stream; `device`: the current device's index, on which the
// signature's memory and the arguments have to be (< 0: the process sees one GPU only)
PyObject* table_call(CallTable* t, PyObject* const* a, Py_ssize_t n) {
    if (!wants(n, 3)) return nullptr;
    PyObject* args = a[0];
    if (!PyTuple_Check(args)) {
        PyErr_SetString(PyExc_TypeError, "call: a tuple of arguments");
        return nullptr;
    }
    void* stream = PyLong_AsVoidPtr(a[1]);
    const long device = PyLong_AsLong(a[2]);
    if (PyErr_Occurred()) return nullptr;
    Entry* entry = find(t, args, device);
    if (!entry) {
        if (PyErr_Occurred()) return nullptr;
        Py_RETURN_NONE;
    }
    Entry& e = *entry;
    PyObject *returned = Py_NewRef(e.returned), *signature = Py_NewRef(e.signature);  // hold the plan and its memory
    const Py_ssize_t count = PyTuple_GET_SIZE(args);
    void* pointers[64];
    int usable = 1;
    bool torch = false;
    for (Py_ssize_t k = 0; usable == 1 && k < count; k++) {
        PyObject* x = PyTuple_GET_ITEM(args, k);
        if (e.torch[k]) torch = true, usable = in_place(x, device);
        if (usable == 1 && !read_pointer(x, &pointers[k])) usable = -1;
    }
    if (usable == 1 && !stream) {
        PyObject* s = torch && raw_stream != Py_None ? PyObject_CallFunction(raw_stream, "l", device < 0 ? 0L : device)
                                                     : PyObject_CallNoArgs(current_stream);
        if (s) stream = PyLong_AsVoidPtr(s);
        Py_XDECREF(s);
        if (PyErr_Occurred()) usable = -1;
    }
    if (usable != 1) {
        Py_DECREF(returned);
        Py_DECREF(signature);
        if (usable < 0) return nullptr;
        Py_RETURN_NONE;
    }
    PyObject* before = e.keep;
    e.keep = Py_NewRef(args);
    const lb_plan* plan = e.plan;
    void* workspace = e.workspace;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lb_plan_run(plan, workspace, pointers, (int)count, e.outputs.data(), (int)e.outputs.size(), 0, -1, stream);
    Py_END_ALLOW_THREADS
    Py_XDECREF(before);
    Py_XSETREF(t->latest, signature);
    if (rc != LB_OK) {
        Py_DECREF(returned);
        return finish(rc);
    }
    return returned;
}

PyMethodDef table_methods[] = {
    {"add", (PyCFunction)(void (*)(void))table_add, METH_FASTCALL, "adds a signature"},
    {"call", (PyCFunction)(void (*)(void))table_call, METH_FASTCALL, "runs the matching signature's plan, or returns None"},
    {nullptr, nullptr, 0, nullptr},
};
PyMemberDef table_members[] = {
    {"latest", T_OBJECT, offsetof(CallTable, latest), 0, "the signature object of the latest call"},
    {nullptr, 0, 0, 0, nullptr},
};
PyTypeObject table_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

PyMethodDef methods[] = {
    {"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, "dtype codes and callbacks"},
    {"attention_fwd", (PyCFunction)(void (*)(void))attention_fwd, METH_FASTCALL, "lb_attention_fwd on tensors"},
    {"attention_bwd", (PyCFunction)(void (*)(void))attention_bwd, METH_FASTCALL, "lb_attention_bwd_scratch / lb_attention_bwd_atomic on tensors"},
    {"attention_bwd_scratch_bytes", (PyCFunction)(void (*)(void))attention_bwd_scratch_bytes, METH_FASTCALL, "lb_attention_bwd_scratch_bytes of tensors"},
    {"gemm", (PyCFunction)(void (*)(void))gemm, METH_FASTCALL, "lb_gemm on tensors"},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, "lb_qk_norm_rope on tensors"},
    {"qk_norm_rope_bwd", (PyCFunction)(void (*)(void))qk_norm_rope_bwd, METH_FASTCALL, "lb_qk_norm_rope_bwd on tensors"},
    {"gated_mlp_fwd", (PyCFunction)(void (*)(void))gated_mlp_fwd, METH_FASTCALL, "lb_gated_mlp_fwd on tensors"},
    {"gated_mlp_bwd", (PyCFunction)(void (*)(void))gated_mlp_bwd, METH_FASTCALL, "lb_gated_mlp_bwd on tensors"},
    {"linear_cross_entropy", (PyCFunction)(void (*)(void))linear_cross_entropy, METH_FASTCALL, "lb_linear_cross_entropy on tensors"},
    {"linear_cross_entropy_bwd", (PyCFunction)(void (*)(void))linear_cross_entropy_bwd, METH_FASTCALL, "lb_linear_cross_entropy_bwd on tensors"},
    {"adamw_step", (PyCFunction)(void (*)(void))adamw_step, METH_FASTCALL, "lb_adamw_step on sequences of tensors"},
    {"clip_grad_norm", (PyCFunction)(void (*)(void))clip_grad_norm, METH_FASTCALL, "lb_grad_norm / lb_clip_grad_norm on sequences of tensors"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_host", "the call path of lumen_b200 over the C ABI", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    names.dtype = PyUnicode_InternFromString("dtype");
    names.shape = PyUnicode_InternFromString("shape");
    names.stride = PyUnicode_InternFromString("stride");
    names.data_ptr = PyUnicode_InternFromString("data_ptr");
    names.is_cuda = PyUnicode_InternFromString("is_cuda");
    names.is_contiguous = PyUnicode_InternFromString("is_contiguous");
    names.get_device = PyUnicode_InternFromString("get_device");
    table_type.tp_name = "lumen_b200._host.CallTable";
    table_type.tp_basicsize = sizeof(CallTable);
    table_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_GC;
    table_type.tp_new = table_new;
    table_type.tp_dealloc = (destructor)table_dealloc;
    table_type.tp_traverse = (traverseproc)table_traverse;
    table_type.tp_clear = (inquiry)table_clear;
    table_type.tp_methods = table_methods;
    table_type.tp_members = table_members;
    if (PyType_Ready(&table_type) < 0) return nullptr;
    PyObject* m = PyModule_Create(&module_def);
    if (!m) return nullptr;
    Py_INCREF(&table_type);
    if (PyModule_AddObject(m, "CallTable", (PyObject*)&table_type) < 0) {
        Py_DECREF(&table_type);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
