// The host path of gomlx_amd.nn in native code: argument checks, output allocation and the call into the C ABI for the
// operators of a decode loop.  In Python these steps took 11 us per call with its launch (attribute look-ups, ctypes conversions, one
// Tensor method call per property), longer than the kernels of a small projection; here 5 us.
//
// Every function returns None when it does not recognise its arguments or the library reports an error; gomlx_amd.nn then
// goes through the same call step by step in Python, which raises the exception that belongs to it.  The library's entry
// points come in as addresses (bind), so that whatever library _lib.py has loaded is the one that runs.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <limits>

#include "../../include/gomlx_hipq.h"

namespace {

struct Entry {
    decltype(&gq_qdense_check) check;
    decltype(&gq_qdense_f32) dense_f32;
    decltype(&gq_qdense_bf16) dense_bf16;
    decltype(&gq_qdense_block_f32) block_f32;
    decltype(&gq_qdense_block_bf16) block_bf16;
    decltype(&gq_qdense_gated_f32) gated_f32;
    decltype(&gq_qdense_gated_bf16) gated_bf16;
    decltype(&gq_qdense_f32_batch) batch_f32;
    decltype(&gq_qdense_norm_f32_batch) norm_batch_f32;
    decltype(&gq_qdense_norm_bf16_batch) norm_batch_bf16;
    decltype(&gq_dequantize) dequantize;
    decltype(&gq_embedding_lookup) lookup;
    decltype(&gq_bytes_per_block) bytes_per_block;
    decltype(&gq_values_per_block) values_per_block;
    decltype(&gq_qk_norm_rope) rope;
    decltype(&gq_kv_append) kv_append;
    decltype(&gq_kv_read) kv_read;
    decltype(&gq_kv_attention) kv_attention;
    decltype(&gq_kv_evict) kv_evict;
    decltype(&gq_draft_tree) draft_tree;
    decltype(&gq_kv_tree_attention) tree_attention;
    decltype(&gq_sample) sample;
    decltype(&gq_kv_accept) kv_accept;
} g;
constexpr int kEntries = 23;
bool g_bound = false;
PyTypeObject *g_activation = nullptr;  // nn.Activation
PyObject *s_scheme, *s_ggml_type, *s_gain, *s_epsilon, *s_scale_offset;

// activation.Type.ToBackend by the numeric value of nn.Activation
constexpr int kBackendAct[13] = {GQ_ACT_NONE, GQ_ACT_RELU, GQ_ACT_NONE, GQ_ACT_NONE, GQ_ACT_NONE, GQ_ACT_NONE, GQ_ACT_SILU,
                                 GQ_ACT_HARDSWISH, GQ_ACT_SILU, GQ_ACT_TANH, GQ_ACT_GELU, GQ_ACT_GELU, GQ_ACT_NONE};
constexpr long kSchemeGGML = 2;

bool to_long(PyObject *o, long &v) {
    if (!PyLong_Check(o)) return false;  // (IntEnum members are ints)
    v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return v >= INT_MIN && v <= INT_MAX;
}
bool attr_long(PyObject *o, PyObject *name, long &v) {
    PyObject *a = PyObject_GetAttr(o, name);
    if (!a) { PyErr_Clear(); return false; }
    const bool ok = to_long(a, v);
    Py_DECREF(a);
    return ok;
}
bool attr_double(PyObject *o, PyObject *name, double &v) {
    PyObject *a = PyObject_GetAttr(o, name);
    if (!a) { PyErr_Clear(); return false; }
    v = PyFloat_Check(a) || PyLong_Check(a) ? PyFloat_AsDouble(a) : -1.0;
    const bool ok = (PyFloat_Check(a) || PyLong_Check(a)) && !PyErr_Occurred();
    PyErr_Clear();
    Py_DECREF(a);
    return ok;
}
bool ggml_type_of(PyObject *quant, int &type) {
    long scheme, t;
    if (quant == Py_None || !attr_long(quant, s_scheme, scheme) || scheme != kSchemeGGML || !attr_long(quant, s_ggml_type, t)) return false;
    type = (int)t;
    return true;
}
// A member of nn.Activation itself: a bare number or a member of another enumeration says nothing about which function is meant.
bool backend_act(PyObject *act, int &v) {
    long a;
    if (Py_TYPE(act) != g_activation || !to_long(act, a) || a < 0 || a >= 13) return false;
    v = kBackendAct[a];
    return true;
}

// A plain contiguous GPU tensor, borrowed; null otherwise.
const at::Tensor *gpu_tensor(PyObject *o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && t.is_contiguous() ? &t : nullptr;
}
// An optional vector of n floats: 1 = given, 0 = None, -1 = not that.
int vector_of(PyObject *o, int64_t n, const float *&p) {
    p = nullptr;
    if (o == Py_None) return 0;
    const at::Tensor *t = gpu_tensor(o);
    if (!t || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != n) return -1;
    p = static_cast<const float *>(t->const_data_ptr());
    return 1;
}

struct Norm {
    gq_rmsnorm d;
    bool given = false;
    PyObject *gain = nullptr;  // owned: keeps the vector alive over the launch
    ~Norm() { Py_XDECREF(gain); }
    bool read(PyObject *o, int64_t K) {
        if (o == Py_None) return true;
        double eps, off;
        gain = PyObject_GetAttr(o, s_gain);
        if (!gain) { PyErr_Clear(); return false; }
        if (vector_of(gain, K, d.dGain) < 0 || !attr_double(o, s_epsilon, eps) || !attr_double(o, s_scale_offset, off)) return false;
        d.eps = (float)eps;
        d.gain_offset = (float)off;
        given = true;
        return true;
    }
    const gq_rmsnorm *ptr() const { return given ? &d : nullptr; }
};

// x [batch..., K] and W [N, bytes] of a GGML type: what nn checks before a dense call.
struct Operands {
    const at::Tensor *x, *w;
    int64_t M, K, N;
    bool bf16;
    bool read(PyObject *xo, PyObject *wo, int type, int act, int64_t bias_len) {
        x = gpu_tensor(xo);
        w = gpu_tensor(wo);
        if (!x || !w || w->scalar_type() != at::kByte || w->dim() != 2 || x->dim() < 1) return false;
        if (x->scalar_type() != at::kFloat && x->scalar_type() != at::kBFloat16) return false;
        bf16 = x->scalar_type() == at::kBFloat16;
        N = w->size(0);
        const int64_t k_in = x->size(-1);
        M = k_in ? x->numel() / k_in : 0;
        return g.check(type, bf16 ? GQ_BF16 : GQ_F32, M, k_in, N, w->size(1), bias_len, act, &K) == GQ_OK;
    }
    at::Tensor output() const {
        if (x->dim() == 2) return at::empty({x->size(0), N}, x->options().dtype(at::kFloat).requires_grad(false));
        std::vector<int64_t> shape(x->sizes().begin(), x->sizes().end());
        shape.back() = N;
        return at::empty(shape, x->options().dtype(at::kFloat).requires_grad(false));
    }
};
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

PyObject *none() { Py_RETURN_NONE; }
template <class F> int without_gil(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}
// An exception of torch (out of memory, say) is left to the Python path, which meets it again in its own terms.
template <class F> PyObject *guarded(F f) {
    if (!g_bound) return none();
    try {
        return f();
    } catch (...) {
        return none();
    }
}

// dense(x, weights, quant, bias, activation, norm, residual)
PyObject *dense(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int type, act;
        Operands o;
        Norm norm;
        if (n != 7 || !ggml_type_of(a[2], type) || !backend_act(a[4], act)) return none();
        const at::Tensor *w = gpu_tensor(a[1]);
        const float *bias, *residual = nullptr;
        if (!w || w->dim() != 2 || vector_of(a[3], w->size(0), bias) < 0) return none();
        if (!o.read(a[0], a[1], type, act, bias ? w->size(0) : -1) || !norm.read(a[5], o.K)) return none();
        at::Tensor y = o.output();
        if (a[6] != Py_None) {
            const at::Tensor *r = gpu_tensor(a[6]);
            if (!r || r->scalar_type() != at::kFloat || r->sizes() != y.sizes()) return none();
            residual = static_cast<const float *>(r->const_data_ptr());
        }
        const void *x = o.x->const_data_ptr(), *wp = o.w->const_data_ptr();
        float *yp = static_cast<float *>(y.mutable_data_ptr());
        void *s = stream_of(*o.x);
        const int rc = without_gil([&] {
            if (norm.given || residual)
                return o.bf16 ? g.block_bf16(type, static_cast<const uint16_t *>(x), o.M, o.K, norm.ptr(), wp, o.N, bias, act, residual, yp, s)
                              : g.block_f32(type, static_cast<const float *>(x), o.M, o.K, norm.ptr(), wp, o.N, bias, act, residual, yp, s);
            return o.bf16 ? g.dense_bf16(type, static_cast<const uint16_t *>(x), o.M, o.K, wp, o.N, bias, act, yp, s)
                          : g.dense_f32(type, static_cast<const float *>(x), o.M, o.K, wp, o.N, bias, act, yp, s);
        });
        return rc == GQ_OK ? THPVariable_Wrap(std::move(y)) : none();
    });
}

// gated(x, w_gate, w_up, quant, activation, bias_gate, bias_up, norm)
PyObject *gated(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int type, act;
        Operands o;
        Norm norm;
        if (n != 8 || !ggml_type_of(a[3], type) || !backend_act(a[4], act)) return none();
        const at::Tensor *up = gpu_tensor(a[2]);
        if (!o.read(a[0], a[1], type, act, -1) || !up || up->scalar_type() != at::kByte || up->sizes() != o.w->sizes()) return none();
        const float *bg, *bu;
        if (vector_of(a[5], o.N, bg) < 0 || vector_of(a[6], o.N, bu) < 0 || !norm.read(a[7], o.K)) return none();
        at::Tensor y = o.output();
        const void *x = o.x->const_data_ptr(), *wg = o.w->const_data_ptr(), *wu = up->const_data_ptr();
        float *yp = static_cast<float *>(y.mutable_data_ptr());
        void *s = stream_of(*o.x);
        const int rc = without_gil([&] {
            return o.bf16 ? g.gated_bf16(type, static_cast<const uint16_t *>(x), o.M, o.K, norm.ptr(), wg, bg, wu, bu, o.N, act, yp, s)
                          : g.gated_f32(type, static_cast<const float *>(x), o.M, o.K, norm.ptr(), wg, bg, wu, bu, o.N, act, yp, s);
        });
        return rc == GQ_OK ? THPVariable_Wrap(std::move(y)) : none();
    });
}

// batch(problems, norm): up to eight (x, weights, quant, bias, activation | None) tuples
PyObject *batch(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 2 || !(PyList_Check(a[0]) || PyTuple_Check(a[0]))) return none();
        const Py_ssize_t count = PySequence_Fast_GET_SIZE(a[0]);
        if (count < 1 || count > 8) return none();
        gq_dense_desc d[8];
        at::Tensor y[8];
        Operands o;
        bool bf16 = false;
        for (Py_ssize_t i = 0; i < count; i++) {
            PyObject *p = PySequence_Fast_GET_ITEM(a[0], i);
            int type, act = GQ_ACT_NONE;
            if (!PyTuple_Check(p) || PyTuple_GET_SIZE(p) != 5 || !ggml_type_of(PyTuple_GET_ITEM(p, 2), type)) return none();
            if (PyTuple_GET_ITEM(p, 4) != Py_None && !backend_act(PyTuple_GET_ITEM(p, 4), act)) return none();
            const float *bias;
            if (!o.read(PyTuple_GET_ITEM(p, 0), PyTuple_GET_ITEM(p, 1), type, act, -1) || vector_of(PyTuple_GET_ITEM(p, 3), o.N, bias) < 0) return none();
            if (i == 0) bf16 = o.bf16;
            if (o.bf16 != bf16 || (bf16 && a[1] == Py_None)) return none();
            y[i] = o.output();
            d[i] = gq_dense_desc{type, act, static_cast<const float *>(o.x->const_data_ptr()), o.M, o.K, o.w->const_data_ptr(), o.N, bias,
                                 static_cast<float *>(y[i].mutable_data_ptr())};
        }
        PyObject *p0 = PySequence_Fast_GET_ITEM(a[0], 0);
        const at::Tensor &x0 = THPVariable_Unpack(PyTuple_GET_ITEM(p0, 0));
        Norm norm;
        if (!norm.read(a[1], d[0].K)) return none();
        void *s = stream_of(x0);
        const int rc = without_gil([&] {
            if (!norm.given) return g.batch_f32((int)count, d, s);
            return bf16 ? g.norm_batch_bf16((int)count, d, &norm.d, s) : g.norm_batch_f32((int)count, d, &norm.d, s);
        });
        if (rc != GQ_OK) return none();
        PyObject *out = PyList_New(count);
        if (!out) return nullptr;
        for (Py_ssize_t i = 0; i < count; i++) PyList_SET_ITEM(out, i, THPVariable_Wrap(std::move(y[i])));
        return out;
    });
}

bool row_values(const at::Tensor &w, int type, int64_t &K) {
    const int bpb = g.bytes_per_block(type);
    if (w.scalar_type() != at::kByte || w.dim() != 2 || bpb <= 0 || w.size(1) % bpb) return false;
    K = w.size(1) / bpb * g.values_per_block(type);
    return true;
}

// dequantize(weights, ggml_type)
PyObject *dequantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        long type;
        int64_t K;
        const at::Tensor *w = n == 2 ? gpu_tensor(a[0]) : nullptr;
        if (!w || !to_long(a[1], type) || !row_values(*w, (int)type, K)) return none();
        at::Tensor y = at::empty({w->size(0), K}, w->options().dtype(at::kFloat).requires_grad(false));
        float *yp = static_cast<float *>(y.mutable_data_ptr());
        const void *wp = w->const_data_ptr();
        void *s = stream_of(*w);
        const int rc = without_gil([&] { return g.dequantize((int)type, wp, w->size(0), K, yp, s); });
        return rc == GQ_OK ? THPVariable_Wrap(std::move(y)) : none();
    });
}

// gather(table, indices int32 [batch..., 1], quant).  The kernel reports an index out of range in pinned host memory, which
// is read once the stream has drained: no clearing kernel and no copy back (28.4 -> 16.1 us for 512 rows of 4096 values).
PyObject *gather(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int type;
        int64_t K;
        if (n != 3 || !ggml_type_of(a[2], type)) return none();
        const at::Tensor *t = gpu_tensor(a[0]), *idx = gpu_tensor(a[1]);
        if (!t || !idx || !row_values(*t, type, K) || idx->scalar_type() != at::kInt || idx->dim() < 1 || idx->size(-1) != 1 || idx->numel() < 1)
            return none();
        std::vector<int64_t> shape(idx->sizes().begin(), idx->sizes().end());
        shape.back() = K;
        at::Tensor y = at::empty(shape, t->options().dtype(at::kFloat).requires_grad(false));
        at::Tensor flag = at::empty({1}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
        int32_t *fp = flag.mutable_data_ptr<int32_t>();
        *fp = 0;
        float *yp = static_cast<float *>(y.mutable_data_ptr());
        const void *tp = t->const_data_ptr();
        const int32_t *ip = idx->const_data_ptr<int32_t>();
        const hipStream_t s = static_cast<hipStream_t>(stream_of(*t));
        const int rc = without_gil([&] {
            const int r = g.lookup(type, tp, t->size(0), K, ip, idx->numel(), yp, fp, s);
            return r == GQ_OK && hipStreamSynchronize(s) != hipSuccess ? (int)GQ_ERR_HIP : r;
        });
        return rc == GQ_OK && *static_cast<volatile int32_t *>(fp) == 0 ? THPVariable_Wrap(std::move(y)) : none();
    });
}

// ---- rotation, the 4-bit cache and attention over it --------------------------------------------------------------------

bool to_i64(PyObject *o, int64_t &v) {
    if (!PyLong_Check(o)) return false;
    v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}
int element_type(at::ScalarType t) { return t == at::kFloat ? GQ_F32 : t == at::kBFloat16 ? GQ_BF16 : -1; }
bool head_dim_served(int64_t d) { return d == 64 || d == 128 || d == 256; }

// [rows, heads, values], the values side by side
struct HeadRows {
    const at::Tensor *t = nullptr;
    gq_head_rows d;
    bool read(PyObject *o) {
        if (!THPVariable_CheckExact(o)) return false;
        t = &THPVariable_Unpack(o);
        if (!t->is_cuda() || t->dim() != 3 || t->layout() != at::kStrided || element_type(t->scalar_type()) < 0 || t->stride(2) != 1) return false;
        d = gq_head_rows{t->const_data_ptr(), t->stride(0), t->stride(1)};
        return true;
    }
};

const int32_t *int32_vector(PyObject *o, int64_t n, c10::DeviceIndex device) {
    const at::Tensor *t = gpu_tensor(o);
    return t && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->get_device() == device ? t->const_data_ptr<int32_t>() : nullptr;
}

// What nn._kv_desc checks; empty calls are left to it.
struct Cache {
    gq_kv_cache d;
    const at::Tensor *t = nullptr;
    float *accounts = nullptr;
    bool read(PyObject *cache, PyObject *table, PyObject *lengths, PyObject *starts, PyObject *max_new, int64_t rows, PyObject *weights) {
        t = gpu_tensor(cache);
        if (!t || t->scalar_type() != at::kByte || t->dim() != 4 || t->size(3) % 36 || !head_dim_served(t->size(3) / 36) || t->numel() == 0) return false;
        if (!THPVariable_CheckExact(table) || !THPVariable_CheckExact(lengths)) return false;
        const at::Tensor &pt = THPVariable_Unpack(table), &ln = THPVariable_Unpack(lengths);
        const c10::DeviceIndex device = t->get_device();
        if (ln.dim() != 1 || ln.size(0) < 1 || !pt.is_cuda() || pt.get_device() != device || pt.scalar_type() != at::kInt || pt.dim() != 2 || pt.size(0) != ln.size(0) ||
            pt.size(1) < 1 || pt.size(1) > INT_MAX || (pt.size(1) > 1 && pt.stride(1) != 1))
            return false;
        d = gq_kv_cache{t->mutable_data_ptr(), t->size(0), (int)t->size(1), (int)(t->size(3) / 36), (int)(32 * t->size(2)), (int)pt.size(1), pt.const_data_ptr<int32_t>(),
                        ln.size(0) < 2 ? std::max(pt.stride(0), pt.size(1)) : pt.stride(0), int32_vector(lengths, ln.size(0), device), nullptr, ln.size(0), rows, 1};
        if (!d.dLengths || rows < 1 || !to_i64(max_new, d.max_new) || d.max_new < 1) return false;
        if (starts != Py_None) {
            if (!(d.dStarts = int32_vector(starts, d.seqs + 1, device))) return false;
        } else if (d.max_new != 1 || rows != d.seqs) {
            return false;
        }
        if (weights != Py_None) {
            const at::Tensor *w = gpu_tensor(weights);
            if (!w || w->get_device() != device || w->scalar_type() != at::kFloat || w->dim() != 3 || w->size(0) != d.pages || w->size(1) != d.kv_heads || w->size(2) != d.page_tokens)
                return false;
            accounts = static_cast<float *>(w->mutable_data_ptr());
        }
        return true;
    }
};

// (past the dispatcher, which costs 0.4 us a tensor: norms and rotation of one row, whose call the host bounds, 6.7 -> 5.5 us)
at::Tensor fresh(const at::Tensor &like, at::IntArrayRef shape, at::ScalarType type) { return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt)); }

PyObject *pair(at::Tensor &&a, at::Tensor &&b) {
    PyObject *out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(b)));
    return out;
}

// qk_norm_rope(q, k, positions, cos, sin, q_norm, k_norm, interleaved, dtype)
PyObject *qk_norm_rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        HeadRows q, k;
        Norm qn, kn;
        if (n != 9 || !q.read(a[0]) || !k.read(a[1]) || !PyBool_Check(a[7])) return none();
        const int64_t rows = q.t->size(0), dim = q.t->size(2);
        const c10::DeviceIndex device = q.t->get_device();
        const at::Tensor *cos = gpu_tensor(a[3]), *sin = gpu_tensor(a[4]);
        if (!head_dim_served(dim) || k.t->scalar_type() != q.t->scalar_type() || k.t->size(0) != rows || k.t->size(2) != dim || k.t->get_device() != device || !cos || !sin ||
            cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->get_device() != device ||
            sin->get_device() != device || q.t->size(1) > INT_MAX || k.t->size(1) > INT_MAX || cos->size(1) > dim)
            return none();
        at::ScalarType type = q.t->scalar_type();
        if (a[8] != Py_None) {
            if (!THPDtype_Check(a[8])) return none();
            type = reinterpret_cast<THPDtype *>(a[8])->scalar_type;
        }
        const int32_t *pos = int32_vector(a[2], rows, device);
        if (element_type(type) < 0 || !pos || !qn.read(a[5], dim) || !kn.read(a[6], dim)) return none();
        at::Tensor qo = fresh(*q.t, q.t->sizes(), type), ko = fresh(*q.t, k.t->sizes(), type);
        const float *cp = cos->const_data_ptr<float>(), *sp = sin->const_data_ptr<float>();
        void *qp = qo.mutable_data_ptr(), *kp = ko.mutable_data_ptr(), *s = stream_of(*q.t);
        const int rc = without_gil([&] {
            return g.rope(element_type(q.t->scalar_type()), &q.d, (int)q.t->size(1), &k.d, (int)k.t->size(1), (int)dim, rows, pos, cp, sp, cos->size(0), (int)(2 * cos->size(1)),
                          a[7] == Py_True, qn.ptr(), kn.ptr(), element_type(type), qp, kp, s);
        });
        return rc == GQ_OK ? pair(std::move(qo), std::move(ko)) : none();
    });
}

// kv_append(cache, k, v, page_table, lengths, starts, max_new, weights): True where it is done
PyObject *kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        HeadRows k, v;
        Cache c;
        if (n != 8 || !k.read(a[1]) || !v.read(a[2]) || !c.read(a[0], a[3], a[4], a[5], a[6], k.t->size(0), a[7])) return none();
        if (k.t->sizes() != v.t->sizes() || k.t->scalar_type() != v.t->scalar_type() || k.t->size(1) != c.d.kv_heads || k.t->size(2) != c.d.head_dim ||
            k.t->get_device() != c.t->get_device() || v.t->get_device() != c.t->get_device())
            return none();
        void *s = stream_of(*c.t);
        const int rc = without_gil([&] { return g.kv_append(&c.d, element_type(k.t->scalar_type()), &k.d, &v.d, c.accounts, s); });
        if (rc != GQ_OK) return none();
        Py_RETURN_TRUE;
    });
}

// kv_read(cache, page_table, lengths, starts, max_new, rows)
PyObject *kv_read(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Cache c;
        int64_t rows;
        if (n != 6) return none();
        if (a[5] == Py_None) {
            if (a[3] != Py_None || !THPVariable_CheckExact(a[2]) || THPVariable_Unpack(a[2]).dim() != 1) return none();
            rows = THPVariable_Unpack(a[2]).size(0);
        } else if (!to_i64(a[5], rows)) {
            return none();
        }
        if (!c.read(a[0], a[1], a[2], a[3], a[4], rows, Py_None)) return none();
        at::Tensor k = fresh(*c.t, {rows, c.d.kv_heads, c.d.head_dim}, at::kHalf), v = fresh(*c.t, {rows, c.d.kv_heads, c.d.head_dim}, at::kHalf);
        uint16_t *kp = static_cast<uint16_t *>(k.mutable_data_ptr()), *vp = static_cast<uint16_t *>(v.mutable_data_ptr());
        void *s = stream_of(*c.t);
        const int rc = without_gil([&] { return g.kv_read(&c.d, kp, vp, s); });
        return rc == GQ_OK ? pair(std::move(k), std::move(v)) : none();
    });
}

// cached_attention(q, cache, page_table, lengths, starts, max_new, scale | None, window, weights)
PyObject *cached_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        HeadRows q;
        Cache c;
        int64_t window;
        if (n != 9 || !q.read(a[0]) || !c.read(a[1], a[2], a[3], a[4], a[5], q.t->size(0), a[8]) || !to_i64(a[7], window)) return none();
        if (q.t->size(2) != c.d.head_dim || q.t->size(1) < 1 || q.t->size(1) % c.d.kv_heads || q.t->size(1) > INT_MAX || q.t->get_device() != c.t->get_device()) return none();
        double scale;
        if (a[6] == Py_None) scale = 1.0 / std::sqrt((double)c.d.head_dim);
        else if (PyFloat_Check(a[6])) scale = PyFloat_AS_DOUBLE(a[6]);
        else return none();
        at::Tensor out = fresh(*q.t, q.t->sizes(), q.t->scalar_type());
        void *op = out.mutable_data_ptr(), *s = stream_of(*c.t);
        const int rc = without_gil([&] { return g.kv_attention(&c.d, element_type(q.t->scalar_type()), &q.d, (int)q.t->size(1), (float)scale, window, c.accounts, op, s); });
        return rc == GQ_OK ? THPVariable_Wrap(std::move(out)) : none();
    });
}

// kv_evict(cache, weights, page_table, lengths, keep, recent)
PyObject *kv_evict(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Cache c;
        int64_t keep, recent;
        if (n != 6 || a[1] == Py_None || !THPVariable_CheckExact(a[3]) || THPVariable_Unpack(a[3]).dim() != 1 || !to_i64(a[4], keep) || !to_i64(a[5], recent)) return none();
        PyObject *one = PyLong_FromLong(1);  // (a small number: shared)
        const bool ok = c.read(a[0], a[2], a[3], Py_None, one, THPVariable_Unpack(a[3]).size(0), a[1]);
        Py_DECREF(one);
        if (!ok || keep < 1 || recent < 0 || recent > keep) return none();
        at::Tensor kept = fresh(*c.t, {c.d.seqs, c.d.kv_heads, keep}, at::kInt), left = fresh(*c.t, {c.d.seqs}, at::kInt);
        int32_t *kp = kept.mutable_data_ptr<int32_t>(), *lp = left.mutable_data_ptr<int32_t>();
        void *s = stream_of(*c.t);
        const int rc = without_gil([&] { return g.kv_evict(&c.d, c.accounts, keep, recent, kp, lp, s); });
        return rc == GQ_OK ? pair(std::move(kept), std::move(left)) : none();
    });
}

// ---- decoding with drafted tokens ------------------------------------------------------------------------------------------

// draft_tree(parents, first, starts, max_new)
PyObject *draft_tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int64_t most;
        if (n != 4 || !THPVariable_CheckExact(a[0]) || !THPVariable_CheckExact(a[1]) || !to_i64(a[3], most) || most < 1 || most > INT_MAX) return none();
        const at::Tensor &up = THPVariable_Unpack(a[0]), &fi = THPVariable_Unpack(a[1]);
        if (!up.is_cuda() || up.dim() != 1 || fi.dim() != 1 || up.size(0) < 1 || fi.size(0) < 1) return none();
        const int64_t rows = up.size(0), seqs = fi.size(0), words = (most + 31) / 32;
        const c10::DeviceIndex device = up.get_device();
        const int32_t *pp = int32_vector(a[0], rows, device), *fp = int32_vector(a[1], seqs, device), *sp = nullptr;
        if (!pp || !fp || (a[2] == Py_None ? rows != seqs || most != 1 : !(sp = int32_vector(a[2], seqs + 1, device)))) return none();
        at::Tensor tree = fresh(up, {rows, words}, at::kInt), positions = fresh(up, {rows}, at::kInt);
        int32_t *tp = tree.mutable_data_ptr<int32_t>(), *op = positions.mutable_data_ptr<int32_t>();
        void *s = stream_of(up);
        const int rc = without_gil([&] { return g.draft_tree(pp, fp, sp, seqs, rows, most, tp, words, op, s); });
        return rc == GQ_OK ? pair(std::move(tree), std::move(positions)) : none();
    });
}

// tree_attention(q, cache, page_table, lengths, tree, starts, max_new, scale | None, window)
PyObject *tree_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        HeadRows q;
        Cache c;
        int64_t window;
        if (n != 9 || !q.read(a[0]) || !c.read(a[1], a[2], a[3], a[5], a[6], q.t->size(0), Py_None) || !to_i64(a[8], window)) return none();
        if (q.t->size(2) != c.d.head_dim || q.t->size(1) < 1 || q.t->size(1) % c.d.kv_heads || q.t->size(1) > INT_MAX || q.t->get_device() != c.t->get_device()) return none();
        const at::Tensor *t = gpu_tensor(a[4]);
        if (!t || t->scalar_type() != at::kInt || t->dim() != 2 || t->size(0) != c.d.rows || t->size(1) < 1 || t->get_device() != c.t->get_device()) return none();
        double scale;
        if (a[7] == Py_None) scale = 1.0 / std::sqrt((double)c.d.head_dim);
        else if (PyFloat_Check(a[7])) scale = PyFloat_AS_DOUBLE(a[7]);
        else return none();
        at::Tensor out = fresh(*q.t, q.t->sizes(), q.t->scalar_type());
        const int32_t *tp = t->const_data_ptr<int32_t>();
        void *op = out.mutable_data_ptr(), *s = stream_of(*c.t);
        const int rc = without_gil([&] {
            return g.tree_attention(&c.d, element_type(q.t->scalar_type()), &q.d, (int)q.t->size(1), (float)scale, window, tp, t->size(1), op, s);
        });
        return rc == GQ_OK ? THPVariable_Wrap(std::move(out)) : none();
    });
}

// One setting of `sample`: a number in its range, or a vector with one for each row.
template <class T> bool setting(PyObject *o, at::ScalarType type, int64_t rows, c10::DeviceIndex device, double most, double &value, const T *&vector) {
    if (PyFloat_Check(o)) value = PyFloat_AS_DOUBLE(o);
    else if (PyLong_Check(o)) {
        int64_t v;
        if (!to_i64(o, v)) return false;
        value = (double)v;
    } else {
        const at::Tensor *t = gpu_tensor(o);
        if (!t || t->scalar_type() != type || t->dim() != 1 || t->size(0) != rows || t->get_device() != device) return false;
        vector = t->const_data_ptr<T>();
        return true;
    }
    return value >= 0.0 && value <= most;
}

// sample(logits, uniform, temperature, top_k, top_p, min_p, probabilities)
PyObject *sample(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 7 || !THPVariable_CheckExact(a[0]) || !PyBool_Check(a[6])) return none();
        const at::Tensor &x = THPVariable_Unpack(a[0]);
        if (!x.is_cuda() || x.layout() != at::kStrided || x.dim() != 2 || x.size(0) < 1 || x.size(1) < 1 || element_type(x.scalar_type()) < 0 || (x.size(1) > 1 && x.stride(1) != 1)) return none();
        const int64_t rows = x.size(0);
        const c10::DeviceIndex device = x.get_device();
        const at::Tensor *u = gpu_tensor(a[1]);
        if (!u || u->scalar_type() != at::kFloat || u->dim() != 1 || u->size(0) != rows || u->get_device() != device) return none();
        gq_sampling d{};
        double k = 0.0;
        const double any = std::numeric_limits<double>::infinity();
        if (PyFloat_Check(a[3]) || !setting(a[2], at::kFloat, rows, device, any, d.temperature, d.dTemperature) || !setting(a[3], at::kInt, rows, device, 2147483647.0, k, d.dTopK) ||
            !setting(a[4], at::kFloat, rows, device, 1.0, d.top_p, d.dTopP) || !setting(a[5], at::kFloat, rows, device, 1.0, d.min_p, d.dMinP))
            return none();
        d.top_k = (int64_t)k;
        at::Tensor tokens = fresh(x, {rows}, at::kInt), shares;
        int32_t *tp = tokens.mutable_data_ptr<int32_t>();
        float *sp = nullptr;
        if (a[6] == Py_True) {
            shares = fresh(x, {rows}, at::kFloat);
            sp = shares.mutable_data_ptr<float>();
        }
        const void *xp = x.const_data_ptr();
        const float *up = u->const_data_ptr<float>();
        void *s = stream_of(x);
        const int rc = without_gil([&] { return g.sample(element_type(x.scalar_type()), xp, rows, x.size(1), x.stride(0), up, &d, tp, sp, s); });
        if (rc != GQ_OK) return none();
        return sp ? pair(std::move(tokens), std::move(shares)) : THPVariable_Wrap(std::move(tokens));
    });
}

// kv_accept(cache, page_table, lengths, parents, tokens, sampled, starts, max_new, weights)
PyObject *kv_accept(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Cache c;
        if (n != 9 || !THPVariable_CheckExact(a[3]) || THPVariable_Unpack(a[3]).dim() != 1 || !c.read(a[0], a[1], a[2], a[6], a[7], THPVariable_Unpack(a[3]).size(0), a[8])) return none();
        const c10::DeviceIndex device = c.t->get_device();
        const int32_t *in[3];
        for (int i = 0; i < 3; i++)
            if (!(in[i] = int32_vector(a[3 + i], c.d.rows, device))) return none();
        at::Tensor path = fresh(*c.t, {c.d.seqs, c.d.max_new}, at::kInt), token = fresh(*c.t, {c.d.seqs}, at::kInt), left = fresh(*c.t, {c.d.seqs}, at::kInt);
        int32_t *pp = path.mutable_data_ptr<int32_t>(), *tp = token.mutable_data_ptr<int32_t>(), *lp = left.mutable_data_ptr<int32_t>();
        void *s = stream_of(*c.t);
        const int rc = without_gil([&] { return g.kv_accept(&c.d, in[0], in[1], in[2], c.accounts, pp, c.d.max_new, tp, lp, s); });
        if (rc != GQ_OK) return none();
        PyObject *out = PyTuple_New(3);
        if (!out) return nullptr;
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(path)));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(token)));
        PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(left)));
        return out;
    });
}

// bind(Activation, address, ...): the enumeration of nn.py, the entry points in the order of Entry
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != kEntries + 1 || !PyType_Check(a[0])) { PyErr_Format(PyExc_TypeError, "bind takes a type and %d addresses", kEntries); return nullptr; }
    void *p[kEntries];
    for (int i = 0; i < kEntries; i++) {
        p[i] = PyLong_AsVoidPtr(a[i + 1]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
            return nullptr;
        }
    }
    static_assert(sizeof(Entry) == sizeof p, "one pointer per entry point");
    std::memcpy(static_cast<void *>(&g), p, sizeof p);
    Py_INCREF(a[0]);
    Py_XDECREF(reinterpret_cast<PyObject *>(g_activation));
    g_activation = reinterpret_cast<PyTypeObject *>(a[0]);
    g_bound = true;
    return none();
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"dense", (PyCFunction)(void (*)(void))dense, METH_FASTCALL, nullptr},
    {"gated", (PyCFunction)(void (*)(void))gated, METH_FASTCALL, nullptr},
    {"batch", (PyCFunction)(void (*)(void))batch, METH_FASTCALL, nullptr},
    {"dequantize", (PyCFunction)(void (*)(void))dequantize, METH_FASTCALL, nullptr},
    {"gather", (PyCFunction)(void (*)(void))gather, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, nullptr},
    {"kv_append", (PyCFunction)(void (*)(void))kv_append, METH_FASTCALL, nullptr},
    {"kv_read", (PyCFunction)(void (*)(void))kv_read, METH_FASTCALL, nullptr},
    {"cached_attention", (PyCFunction)(void (*)(void))cached_attention, METH_FASTCALL, nullptr},
    {"kv_evict", (PyCFunction)(void (*)(void))kv_evict, METH_FASTCALL, nullptr},
    {"draft_tree", (PyCFunction)(void (*)(void))draft_tree, METH_FASTCALL, nullptr},
    {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
    {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, nullptr},
    {"kv_accept", (PyCFunction)(void (*)(void))kv_accept, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
    s_scheme = PyUnicode_InternFromString("scheme");
    s_ggml_type = PyUnicode_InternFromString("ggml_type");
    s_gain = PyUnicode_InternFromString("gain");
    s_epsilon = PyUnicode_InternFromString("epsilon");
    s_scale_offset = PyUnicode_InternFromString("scale_offset");
    return PyModule_Create(&module);
}
