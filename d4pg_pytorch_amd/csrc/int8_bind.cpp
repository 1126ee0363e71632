// Tensor binding of the 8-bit operators: the short way from a Python call to a launch.
//
// At the sizes one state or one token has, an operator's kernel runs for 2 - 5 us and the call around it decides: checks,
// allocation and launch take the host 8 - 17 us in Python, 4 - 5.5 us here.  A function of this module takes exactly the plain case -
// dense tensors on the current device, types, shapes and strides as the kernels read them - and returns None for anything
// else: ops/int8.py then converts layouts, or says what is wrong.  It decides nothing by itself.  A launch that HIP refuses
// raises here: the work of an entry that returned a hipError_t is not tried again.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>

#include "int8_args.h"

namespace {

int (*quant_rows)(const QuantRowsArgs*, hipStream_t);
int (*dequant_rows)(DequantRowsArgs*, hipStream_t);
int (*linear_int8)(const LinearInt8Args*, hipStream_t);
int (*mlp3_int8)(Mlp3Int8Args*, hipStream_t);

using at::Tensor;

// A dense tensor of `type` on device `dev`, or null.
const Tensor* dense(PyObject* o, int dev) {
    if (!THPVariable_Check(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == dev && !t.is_neg() ? &t : nullptr;
}
// The device of the first argument, if it is the current one; -1 otherwise.
int current(PyObject* o) {
    if (!THPVariable_Check(o)) return -1;
    const Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == c10::hip::current_device() ? t.get_device() : -1;
}
int float_code(at::ScalarType t) {
    return t == at::kFloat ? F_FP32 : t == at::kBFloat16 ? F_BF16 : t == at::kHalf ? F_FP16 : F_NONE;
}
at::ScalarType float_type(long code) {
    return code == F_FP32 ? at::kFloat : code == F_BF16 ? at::kBFloat16 : at::kHalf;
}
int64_t padded(int64_t K) { return (K + 15) & ~int64_t(15); }

// [M, K] with neighbouring elements side by side.
bool rows(const Tensor* t) {
    return t && t->dim() == 2 && t->size(1) >= 1 && t->size(0) >= 1 && (t->size(1) == 1 || t->stride(1) == 1);
}
// Codes [M, K] in rows that can be read 16 bytes at a time; their row stride in `ld`.
bool code_rows(const Tensor* t, long long& ld) {
    if (!rows(t) || t->scalar_type() != at::kChar) return false;
    const int64_t M = t->size(0), K = t->size(1), kp = padded(K);
    ld = M > 1 ? t->stride(0) : kp;
    if (ld % 16 || ld < kp || reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16) return false;
    return kp == K || t->storage_offset() + (M - 1) * ld + kp <= (int64_t)t->storage().nbytes();
}
bool vector_of(const Tensor* t, int64_t n) {
    return t && t->dim() == 1 && t->size(0) == n && t->scalar_type() == at::kFloat && (n == 1 || t->stride(0) == 1);
}
Tensor new_codes(int64_t M, int64_t K, const Tensor& like) {
    Tensor q = at::empty({M, padded(K)}, like.options().dtype(at::kChar));
    return padded(K) == K ? q : q.narrow(1, 0, K);
}
hipStream_t stream(int dev) { return c10::hip::getCurrentHIPStream(dev).stream(); }
float* f32(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }
const float* f32c(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }

// 0: enqueued.  false: refused by the entry's own checks.
bool enqueued(int rc, const char* what) {
    TORCH_CHECK(rc <= 0, what, " failed with code ", rc);
    return rc == 0;
}

struct Weights {
    const signed char* w;
    const float *scale, *bias;
    long long ld;
    int64_t N;
};
// weight [N, K], weight_scale [N], bias [N] or None
bool layer(PyObject* const* o, int dev, int64_t K, Weights& l) {
    const Tensor *w = dense(o[0], dev), *s = dense(o[1], dev), *b = o[2] == Py_None ? nullptr : dense(o[2], dev);
    if (!code_rows(w, l.ld) || w->size(1) != K || K >= 131072 || w->size(0) > INT_MAX) return false;
    l.N = w->size(0);
    if (!vector_of(s, l.N) || (o[2] != Py_None && !vector_of(b, l.N))) return false;
    l.w = static_cast<const signed char*>(w->const_data_ptr()), l.scale = f32c(*s), l.bias = b ? f32c(*b) : nullptr;
    return true;
}

// linear(q, scale, weight, weight_scale, bias, activation code, type code)
PyObject* linear(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) Py_RETURN_NONE;
    const int dev = current(o[0]);
    const long act = PyLong_AsLong(o[5]), dtype = PyLong_AsLong(o[6]);
    if (dev < 0 || act < ACT_NONE || act > ACT_TANH || dtype < F_FP32 || dtype > F_FP16) Py_RETURN_NONE;
    LinearInt8Args a = {};
    const Tensor *q = dense(o[0], dev), *s = dense(o[1], dev);
    Weights l;
    if (!code_rows(q, a.ld_q) || q->size(0) > INT_MAX || !vector_of(s, q->size(0)) || !layer(o + 2, dev, q->size(1), l)) Py_RETURN_NONE;
    Tensor out = at::empty({q->size(0), l.N}, q->options().dtype(float_type(dtype)));
    a.q = static_cast<const signed char*>(q->const_data_ptr()), a.scale = f32c(*s), a.w = l.w, a.wscale = l.scale, a.bias = l.bias;
    a.out = out.data_ptr(), a.ld_w = l.ld, a.ld_out = l.N;
    a.M = (int)q->size(0), a.N = (int)l.N, a.K = (int)q->size(1), a.act = (int)act, a.dtype = (int)dtype;
    if (!enqueued(linear_int8(&a, stream(dev)), "d4pg_linear_int8")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// rows(x) -> (codes, scales);  rows(x, weight, residual, eps) -> (codes, scales, h)
PyObject* quantize(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 1 && n != 4) Py_RETURN_NONE;
    const int dev = current(o[0]);
    if (dev < 0) Py_RETURN_NONE;
    const Tensor* x = dense(o[0], dev);
    if (!rows(x) || float_code(x->scalar_type()) == F_NONE || x->size(0) > INT_MAX || x->size(1) > INT_MAX) Py_RETURN_NONE;
    QuantRowsArgs a = {};
    a.M = x->size(0), a.K = x->size(1), a.ld_x = x->stride(0), a.ld_q = padded(a.K), a.ld_h = a.K;
    a.x = x->const_data_ptr(), a.dtype = float_code(x->scalar_type()), a.wdtype = F_NONE;
    Tensor h;
    if (n == 4) {
        a.norm = 1;
        const double eps = PyFloat_Check(o[3]) ? PyFloat_AS_DOUBLE(o[3]) : -1.0;
        if (!(eps >= 0.0 && eps <= 3e38)) Py_RETURN_NONE;
        a.eps = (float)eps;
        if (o[1] != Py_None) {
            const Tensor* w = dense(o[1], dev);
            if (!w || w->dim() != 1 || w->size(0) != a.K || (a.K > 1 && w->stride(0) != 1)) Py_RETURN_NONE;
            a.weight = w->const_data_ptr(), a.wdtype = float_code(w->scalar_type());
            if (a.wdtype == F_NONE) Py_RETURN_NONE;
        }
        if (o[2] != Py_None) {
            const Tensor* r = dense(o[2], dev);
            if (!rows(r) || r->size(0) != a.M || r->size(1) != a.K || r->scalar_type() != x->scalar_type()) Py_RETURN_NONE;
            a.residual = r->const_data_ptr(), a.ld_r = r->stride(0);
            h = at::empty({a.M, a.K}, x->options());
            a.h = h.data_ptr();
        }
    }
    Tensor q = new_codes(a.M, a.K, *x), scale = at::empty({a.M}, x->options().dtype(at::kFloat));
    a.q = static_cast<signed char*>(q.data_ptr()), a.scale = f32(scale);
    if (!enqueued(quant_rows(&a, stream(dev)), "d4pg_quant_rows")) Py_RETURN_NONE;
    PyObject* t = PyTuple_New(n == 4 ? 3 : 2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(scale)));
    if (n == 4) {
        if (!h.defined()) Py_INCREF(o[0]);
        PyTuple_SET_ITEM(t, 2, h.defined() ? THPVariable_Wrap(std::move(h)) : o[0]);
    }
    return t;
    END_HANDLE_TH_ERRORS
}

// dequantize(q, scale, type code)
PyObject* dequantize(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) Py_RETURN_NONE;
    const int dev = current(o[0]);
    const long dtype = PyLong_AsLong(o[2]);
    if (dev < 0 || dtype < F_FP32 || dtype > F_FP16) Py_RETURN_NONE;
    const Tensor *q = dense(o[0], dev), *s = dense(o[1], dev);
    if (!rows(q) || q->scalar_type() != at::kChar || q->size(0) > INT_MAX || q->size(1) > INT_MAX || !vector_of(s, q->size(0))) Py_RETURN_NONE;
    Tensor out = at::empty({q->size(0), q->size(1)}, q->options().dtype(float_type(dtype)));
    DequantRowsArgs a = {};
    a.q = static_cast<const signed char*>(q->const_data_ptr()), a.scale = f32c(*s), a.out = out.data_ptr();
    a.M = q->size(0), a.K = q->size(1), a.ld_q = q->stride(0), a.dtype = (int)dtype;
    if (!enqueued(dequant_rows(&a, stream(dev)), "d4pg_dequant_rows")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// One layer on rows that are not codes yet; an undefined tensor where an entry refused.
Tensor coded_layer(const Tensor& x, const Weights& l, int act, int dtype, hipStream_t s) {
    const int64_t M = x.size(0), K = x.size(1);
    Tensor q = at::empty({M, padded(K)}, x.options().dtype(at::kChar)), scale = at::empty({M}, x.options().dtype(at::kFloat));
    QuantRowsArgs r = {};
    r.x = x.const_data_ptr(), r.q = static_cast<signed char*>(q.data_ptr()), r.scale = f32(scale);
    r.M = M, r.K = K, r.ld_x = x.stride(0), r.ld_q = padded(K), r.dtype = float_code(x.scalar_type()), r.wdtype = F_NONE;
    if (!enqueued(quant_rows(&r, s), "d4pg_quant_rows")) return Tensor();
    Tensor out = at::empty({M, l.N}, x.options().dtype(float_type(dtype)));
    LinearInt8Args a = {};
    a.q = r.q, a.scale = r.scale, a.w = l.w, a.wscale = l.scale, a.bias = l.bias, a.out = out.data_ptr();
    a.ld_q = r.ld_q, a.ld_w = l.ld, a.ld_out = l.N, a.M = (int)M, a.N = (int)l.N, a.K = (int)K, a.act = act, a.dtype = dtype;
    return enqueued(linear_int8(&a, s), "d4pg_linear_int8") ? out : Tensor();
}

// mlp3(x, weight, weight_scale, bias, ... three times, activation code, type code)
PyObject* mlp3(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12) Py_RETURN_NONE;
    const int dev = current(o[0]);
    const long act = PyLong_AsLong(o[10]), dtype = PyLong_AsLong(o[11]);
    if (dev < 0 || act < ACT_NONE || act > ACT_TANH || dtype < F_FP32 || dtype > F_FP16) Py_RETURN_NONE;
    const Tensor* x = dense(o[0], dev);
    if (!rows(x) || float_code(x->scalar_type()) == F_NONE || x->size(0) > INT_MAX) Py_RETURN_NONE;
    Mlp3Int8Args a = {};
    Weights l[3];
    int64_t K = x->size(1);
    if (K > INT_MAX) Py_RETURN_NONE;
    a.width[0] = (int)K;
    for (int i = 0; i < 3; ++i) {
        if (!layer(o + 1 + 3 * i, dev, K, l[i])) Py_RETURN_NONE;
        a.w[i] = l[i].w, a.wscale[i] = l[i].scale, a.bias[i] = l[i].bias, a.ld_w[i] = l[i].ld;
        K = l[i].N;
        a.width[i + 1] = (int)K;
    }
    Tensor out = at::empty({x->size(0), K}, x->options().dtype(float_type(dtype)));
    a.x = x->const_data_ptr(), a.ld_x = x->stride(0), a.out = out.data_ptr(), a.ld_out = K, a.M = (int)x->size(0);
    a.xdtype = float_code(x->scalar_type()), a.dtype = (int)dtype, a.act = (int)act;
    const hipStream_t s = stream(dev);
    const int rc = mlp3_int8(&a, s);
    if (rc == NOT_TAKEN) {       // wider than its LDS: a launch a step
        out = *x;
        for (int i = 0; i < 3 && out.defined(); ++i) out = coded_layer(out, l[i], i < 2 ? ACT_RELU : (int)act, i < 2 ? F_FP32 : (int)dtype, s);
        if (!out.defined()) Py_RETURN_NONE;
    } else if (!enqueued(rc, "d4pg_mlp3_int8")) {
        Py_RETURN_NONE;
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(quant_rows, dequant_rows, linear_int8, mlp3_int8): addresses of the kernel library's entries
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "four addresses are expected");
        return nullptr;
    }
    void* p[4];
    for (int i = 0; i < 4; ++i) {
        p[i] = PyLong_AsVoidPtr(o[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    quant_rows = reinterpret_cast<decltype(quant_rows)>(p[0]);
    dequant_rows = reinterpret_cast<decltype(dequant_rows)>(p[1]);
    linear_int8 = reinterpret_cast<decltype(linear_int8)>(p[2]);
    mlp3_int8 = reinterpret_cast<decltype(mlp3_int8)>(p[3]);
    Py_RETURN_NONE;
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(linear), METHOD(quantize), METHOD(dequantize), METHOD(mlp3), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_d4pg_int8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__d4pg_int8() { return PyModule_Create(&module); }
