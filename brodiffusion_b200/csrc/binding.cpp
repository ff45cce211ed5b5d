// The calls of a decoding step from Python: torch tensors to the parameter structures of include/bdattn.h.
// A step of a layer makes seven of these calls, and two of rmsnorm_rope for every four sequences, with kernels of 2 to 6 us;
// shapes, strides and pointers looked up as Python attributes took half of the host's time for one (add_rmsnorm_fwd of one row 4.2 -> 2.5 us a call,
// linear_act_fwd 4.9 -> 2.9, sdpa_window_fwd 6.2 -> 3.3; the launch itself is 2.3).  What is checked here is what the library
// cannot see: that the tensors fit one another, that rows and items are memory of their own, and that all of it lies on the
// current GPU.  Everything else it refuses itself.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <initializer_list>

#include "../../include/bdattn.h"

namespace {

PyObject* g_error = nullptr;

struct Refusal {};      // a Python error is set

[[noreturn]] void refuse(const char* message) {
    PyErr_SetString(g_error, message);
    throw Refusal();
}
[[noreturn]] void refuse(const char* what, const char* message) {
    PyErr_Format(g_error, "%s %s", what, message);
    throw Refusal();
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", what);
        throw Refusal();
    }
    return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

int integer(PyObject* o) {
    if (!PyLong_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "an integer is required");
        throw Refusal();
    }
    int overflow = 0;
    const long v = PyLong_AsLongAndOverflow(o, &overflow);
    if (overflow != 0 || v > INT32_MAX || v < INT32_MIN) {
        PyErr_SetString(PyExc_TypeError, "an integer is out of range");
        throw Refusal();
    }
    return static_cast<int>(v);
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred() != nullptr) throw Refusal();
    return static_cast<float>(v);
}
int rows_of(int64_t n, const char* what) {
    if (n > INT32_MAX) refuse(what, "has more than 2^31 - 1 rows or columns");
    return static_cast<int>(n);
}
bdattn_stream_t stream_of(PyObject* o) {
    if (o == Py_None) return reinterpret_cast<bdattn_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
    void* const p = PyLong_AsVoidPtr(o);
    if (p == nullptr && PyErr_Occurred() != nullptr) throw Refusal();
    return reinterpret_cast<bdattn_stream_t>(p);
}

int code(const at::Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return BDATTN_BF16;
        case at::kHalf: return BDATTN_F16;
        case at::kFloat: return BDATTN_F32;
        case at::kFloat8_e4m3fn: return BDATTN_E4M3;
        default: refuse(what, "has an unsupported dtype");
    }
}
// A call's tensors (their GPUs' numbers, -1: the host) lie on one GPU, and that is the current one, whose stream,
// kernels and sizes the call takes.  current: its number, -1: looked up.
void one_gpu(int current, const int* gpus, int n) {
    for (int i = 0; i < n; ++i)
        if (gpus[i] < 0) refuse("a tensor is not on the GPU");
    for (int i = 1; i < n; ++i)
        if (gpus[i] != gpus[0]) refuse("the tensors are on different GPUs");
    if (current < 0) current = c10::cuda::current_device();
    if (n > 0 && gpus[0] != current) refuse("the tensors are not on the current GPU");
}
void on_gpu(std::initializer_list<const at::Tensor*> all) {
    int gpus[16], n = 0;
    for (const at::Tensor* t : all)
        if (t != nullptr) gpus[n++] = t->is_cuda() ? static_cast<int>(t->get_device()) : -1;
    one_gpu(-1, gpus, n);
}

// A 2-D tensor with contiguous columns; the stride of a single row may be anything.
struct Matrix {
    void* data = nullptr;
    int rows = 0, cols = 0;
    long long ld = 0;
    Matrix() = default;
    Matrix(const at::Tensor& t, const char* what) {
        if (t.dim() != 2) refuse(what, "must be a 2-D tensor");
        rows = rows_of(t.size(0), what);
        cols = rows_of(t.size(1), what);
        if (cols > 1 && t.stride(1) != 1) refuse(what, "must have contiguous columns");
        ld = rows > 1 ? t.stride(0) : cols;
        // (an expanded row has a stride of 0, which the library takes for dense rows)
        if (ld < cols) refuse(what, "must have rows of its own (an expanded or strided view whose rows overlap)");
        data = t.data_ptr();
    }
    void same(const Matrix& o, const char* what) const {
        if (rows != o.rows || cols != o.cols) refuse(what, "has another shape");
    }
};
// A dense 1-D tensor of n values, or null.
void* vector(const at::Tensor* t, int64_t n, const char* what) {
    if (t == nullptr) return nullptr;
    if (t->dim() != 1 || t->size(0) != n || (n > 1 && t->stride(0) != 1)) refuse(what, "must be a dense tensor of as many values as there are rows or columns");
    return t->data_ptr();
}
void typed(const at::Tensor* t, at::ScalarType type, const char* what) {
    if (t != nullptr && t->scalar_type() != type) refuse(what, "has another dtype than the call needs");
}

PyObject* done(int rc) {
    if (rc == 0) Py_RETURN_NONE;
    refuse(bdattn_last_error());
}

// (x, out, gain, residual, residual_out, out_scale, eps, stream)
PyObject* add_rmsnorm(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0], "x"), &out = tensor(a[1], "out");
    const at::Tensor *gain = optional(a[2], "gain"), *residual = optional(a[3], "residual"),
                     *residual_out = optional(a[4], "residual_out"), *scale = optional(a[5], "out_scale");
    const float eps = real(a[6]);
    const Matrix mx(x, "x"), mo(out, "out");
    mo.same(mx, "out");
    Matrix mr, ms;
    if (residual != nullptr) (mr = Matrix(*residual, "residual")).same(mx, "residual");
    if (residual_out != nullptr) (ms = Matrix(*residual_out, "residual_out")).same(mx, "residual_out");
    typed(residual, x.scalar_type(), "residual");
    typed(residual_out, x.scalar_type(), "residual_out");
    typed(scale, at::kFloat, "out_scale");
    bdattn_add_rmsnorm_params p{};
    p.dtype = code(x, "x");
    p.rows = mx.rows;
    p.cols = mx.cols;
    p.x = mx.data;
    p.x_ld = mx.ld;
    p.residual = mr.data;
    p.residual_ld = mr.ld;
    p.residual_out = ms.data;
    p.residual_out_ld = ms.ld;
    p.gain = vector(gain, mx.cols, "gain");
    p.gain_dtype = gain != nullptr ? code(*gain, "gain") : BDATTN_F32;
    p.out = mo.data;
    p.out_ld = mo.ld;
    p.out_dtype = code(out, "out");
    p.out_scale = static_cast<float*>(vector(scale, mx.rows, "out_scale"));
    p.eps = eps;
    on_gpu({&x, &out, gain, residual, residual_out, scale});
    return done(bdattn_add_rmsnorm_fwd(&p, stream_of(a[7])));
}

// (x, w, bias, y, act, gate, residual, x_scale, w_scale, stream)
PyObject* linear_act(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w"), &y = tensor(a[3], "y");
    const at::Tensor *bias = optional(a[2], "bias"), *gate = optional(a[5], "gate"), *residual = optional(a[6], "residual"),
                     *xs = optional(a[7], "x_scale"), *ws = optional(a[8], "w_scale");
    const int act = integer(a[4]);
    const Matrix mx(x, "x"), mw(w, "w"), my(y, "y");
    if (mw.cols != mx.cols) refuse("w must have the columns of x");
    if (my.rows != mx.rows || my.cols != mw.rows) refuse("y must have the rows of x and a column for each row of w");
    Matrix mr;
    if (residual != nullptr) (mr = Matrix(*residual, "residual")).same(my, "residual");
    typed(&w, x.scalar_type(), "w");
    typed(bias, y.scalar_type(), "bias");
    typed(gate, y.scalar_type(), "gate");
    typed(residual, y.scalar_type(), "residual");
    typed(xs, at::kFloat, "x_scale");
    typed(ws, at::kFloat, "w_scale");
    bdattn_linear_act_params p{};
    p.dtype = code(y, "y");
    p.in_dtype = code(x, "x");
    p.M = mx.rows;
    p.N = mw.rows;
    p.K = mx.cols;
    p.x = mx.data;
    p.x_ld = mx.ld;
    p.w = mw.data;
    p.w_ld = mw.ld;
    p.bias = vector(bias, my.cols, "bias");
    p.gate = vector(gate, my.cols, "gate");
    p.residual = mr.data;
    p.residual_ld = mr.ld;
    p.y = my.data;
    p.y_ld = my.ld;
    p.x_scale = static_cast<const float*>(vector(xs, mx.rows, "x_scale"));
    p.w_scale = static_cast<const float*>(vector(ws, my.cols, "w_scale"));
    p.act = act;
    on_gpu({&x, &w, &y, bias, gate, residual, xs, ws});
    return done(bdattn_linear_act_fwd(&p, stream_of(a[9])));
}

// (rows, cols) or (B, rows, cols) with contiguous columns
struct Rows {
    void* data;
    int batch, rows, cols;
    long long ld, stride;
    Rows(const at::Tensor& t, const char* what) {
        const int d = static_cast<int>(t.dim());
        if (d != 2 && d != 3) refuse(what, "must be a 2-D or 3-D tensor");
        batch = d == 3 ? rows_of(t.size(0), what) : 1;
        rows = rows_of(t.size(d - 2), what);
        cols = rows_of(t.size(d - 1), what);
        if (cols > 1 && t.stride(d - 1) != 1) refuse(what, "must have contiguous columns");
        // (the strides of a single row and a single item may be anything; 0 stands for dense items)
        ld = rows > 1 ? t.stride(d - 2) : cols;
        stride = batch > 1 ? t.stride(0) : 0;
        if (batch > 1 && stride == 0) refuse(what, "has the same memory for several batch items");
        data = t.data_ptr();
    }
};

// (q, k, v, out, num_heads, window, sinks, num_kv_heads, kv_len, key_mask, softmax_scale, stream): one segment each
PyObject* sdpa_window(PyObject* const* a) {
    const int heads = integer(a[4]), window = integer(a[5]), sinks = integer(a[6]), kv_heads = integer(a[7]);
    const float scale = real(a[10]);
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &out = tensor(a[3], "out");
    const at::Tensor *kv_len = optional(a[8], "kv_len"), *mask = optional(a[9], "key_mask");
    typed(&k, q.scalar_type(), "k");
    typed(&v, q.scalar_type(), "v");
    typed(&out, q.scalar_type(), "out");
    typed(kv_len, at::kInt, "kv_len");
    typed(mask, at::kFloat, "key_mask");
    const Rows mq(q, "q"), mk(k, "k"), mv(v, "v"), mo(out, "out");
    if (mo.rows != mq.rows || mo.cols != mq.cols || mv.rows != mk.rows || mv.cols != mk.cols) refuse("out must have the shape of q and v that of k");
    if (mk.batch != mq.batch || mv.batch != mq.batch || mo.batch != mq.batch) refuse("q, k, v and out must have the same batch");
    if (heads < 1 || mq.cols % heads != 0 ||
        static_cast<int64_t>(mk.cols) * heads != static_cast<int64_t>(mq.cols) * (kv_heads != 0 ? kv_heads : heads))
        refuse("q and out must have num_heads, k and v num_kv_heads heads of the same width");
    bdattn_sdpa_params p{};
    p.dtype = code(q, "q");
    p.batch = mq.batch;
    p.num_heads = heads;
    p.head_dim = mq.cols / heads;
    p.n_q_seg = p.n_kv_seg = 1;
    p.q[0] = mq.data;
    p.q_rows[0] = mq.rows;
    p.q_ld[0] = mq.ld;
    p.q_batch_stride[0] = mq.stride;
    p.o[0] = mo.data;
    p.o_ld[0] = mo.ld;
    p.o_batch_stride[0] = mo.stride;
    p.k[0] = mk.data;
    p.kv_rows[0] = mk.rows;
    p.k_ld[0] = mk.ld;
    p.k_batch_stride[0] = mk.stride;
    p.v[0] = mv.data;
    p.v_ld[0] = mv.ld;
    p.v_batch_stride[0] = mv.stride;
    p.mask_mode = BDATTN_MASK_CAUSAL;
    p.key_mask = static_cast<const float*>(vector(mask, mk.rows, "key_mask"));
    p.softmax_scale = scale;
    p.num_kv_heads = kv_heads;
    const bdattn_window_params w{window, sinks, static_cast<const int*>(vector(kv_len, mq.batch, "kv_len"))};
    on_gpu({&q, &k, &v, &out, kv_len, mask});
    return done(bdattn_sdpa_window_fwd(&p, &w, stream_of(a[11])));
}

template <PyObject* (*kCall)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != kArgs) {
        PyErr_Format(PyExc_TypeError, "%d arguments are needed (got %zd)", kArgs, n);
        return nullptr;
    }
    try {
        return kCall(args);
    } catch (const Refusal&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// (current, gpus...): one_gpu, for the calls that Python makes
PyObject* one_gpu_entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    int gpus[16];
    if (n < 1 || n > 17) {
        PyErr_SetString(PyExc_TypeError, "1 to 17 arguments are needed");
        return nullptr;
    }
    try {
        for (Py_ssize_t i = 1; i < n; ++i) gpus[i - 1] = integer(args[i]);
        one_gpu(integer(args[0]), gpus, static_cast<int>(n - 1));
        Py_RETURN_NONE;
    } catch (const Refusal&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject* set_error(PyObject*, PyObject* type) {
    Py_INCREF(type);
    Py_XDECREF(g_error);
    g_error = type;
    Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"add_rmsnorm", fast(entry<add_rmsnorm, 8>), METH_FASTCALL, "bdattn_add_rmsnorm_fwd"},
    {"linear_act", fast(entry<linear_act, 10>), METH_FASTCALL, "bdattn_linear_act_fwd"},
    {"sdpa_window", fast(entry<sdpa_window, 12>), METH_FASTCALL, "bdattn_sdpa_window_fwd"},
    {"one_gpu", fast(one_gpu_entry), METH_FASTCALL, "refuses tensors of the host, of different GPUs, of another than the current one"},
    {"set_error", set_error, METH_O, "the exception of a refused call"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
    Py_INCREF(PyExc_RuntimeError);
    g_error = PyExc_RuntimeError;
    return PyModule_Create(&module);
}
