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

// (x, residual, residual_out, post_gain, gate, residual_scale, gain, out, out_scale, eps, stream)
PyObject* sandwich_norm(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0], "x"), &residual = tensor(a[1], "residual"), &residual_out = tensor(a[2], "residual_out");
    const at::Tensor *post = optional(a[3], "post_gain"), *gate = optional(a[4], "gate"), *gain = optional(a[6], "gain"),
                     *out = optional(a[7], "out"), *scale = optional(a[8], "out_scale");
    const float residual_scale = real(a[5]), eps = real(a[9]);
    const Matrix mx(x, "x"), mr(residual, "residual"), ms(residual_out, "residual_out");
    mr.same(mx, "residual");
    ms.same(mx, "residual_out");
    Matrix mo, mg;
    if (out != nullptr) (mo = Matrix(*out, "out")).same(mx, "out");
    typed(&residual, x.scalar_type(), "residual");
    typed(&residual_out, x.scalar_type(), "residual_out");
    typed(gate, x.scalar_type(), "gate");
    typed(scale, at::kFloat, "out_scale");
    if (gain != nullptr && post != nullptr) typed(gain, post->scalar_type(), "gain");
    if (gate != nullptr) {
        if (gate->dim() == 1) {
            mg.data = vector(gate, mx.cols, "gate");
            mg.rows = 1;
            mg.ld = mx.cols;
        } else {
            mg = Matrix(*gate, "gate");
            if (mg.cols != mx.cols || mg.rows < 1) refuse("gate must have a row at least and the columns of x");
        }
    }
    bdattn_sandwich_norm_params p{};
    p.dtype = code(x, "x");
    p.rows = mx.rows;
    p.cols = mx.cols;
    p.x = mx.data;
    p.x_ld = mx.ld;
    p.residual = mr.data;
    p.residual_ld = mr.ld;
    p.residual_out = ms.data;
    p.residual_out_ld = ms.ld;
    p.post_gain = vector(post, mx.cols, "post_gain");
    p.gain = vector(gain, mx.cols, "gain");
    p.gain_dtype = post != nullptr ? code(*post, "post_gain") : gain != nullptr ? code(*gain, "gain") : BDATTN_F32;
    p.gate = mg.data;
    p.gates = mg.rows;
    p.gate_ld = mg.ld;
    p.residual_scale = residual_scale;
    p.out = mo.data;
    p.out_ld = mo.ld;
    p.out_dtype = out != nullptr ? code(*out, "out") : p.dtype;
    p.out_scale = static_cast<float*>(vector(scale, mx.rows, "out_scale"));
    p.eps = eps;
    on_gpu({&x, &residual, &residual_out, post, gate, gain, out, scale});
    return done(bdattn_sandwich_norm_fwd(&p, stream_of(a[10])));
}

// (codes, scales, packed, group, stream)
PyObject* w4_pack(PyObject* const* a) {
    const at::Tensor &codes = tensor(a[0], "codes"), &scales = tensor(a[1], "scales"), &packed = tensor(a[2], "packed");
    const int group = integer(a[3]);
    typed(&codes, at::kByte, "codes");
    typed(&packed, at::kByte, "packed");
    if (scales.scalar_type() != at::kBFloat16 && scales.scalar_type() != at::kHalf) refuse("scales must be BF16 or F16");
    const Matrix mc(codes, "codes");
    if (group != 32 && group != 64 && group != 128) refuse("group must be 32, 64 or 128");
    if (mc.rows < 1 || mc.cols < 1 || mc.cols > INT32_MAX / 2) refuse("codes must have rows, and less than 2^31 columns of 4 bits");
    const int K = 2 * mc.cols, groups = (mc.cols - 1) / (group / 2) + 1;
    if (scales.dim() != 3 || scales.size(0) != mc.rows || scales.size(1) != groups || scales.size(2) != 2 || scales.stride(2) != 1 ||
        (groups > 1 && scales.stride(1) != 2) || (mc.rows > 1 && scales.stride(0) < 2ll * groups))
        refuse("scales must be (rows, groups, 2) with dense rows of their own");
    if (packed.dim() != 1 || static_cast<size_t>(packed.size(0)) != bdattn_w4_bytes(mc.rows, K, group) || (packed.size(0) > 1 && packed.stride(0) != 1))
        refuse("packed must be dense, of w4_bytes(rows, columns, group) bytes");
    on_gpu({&codes, &scales, &packed});
    return done(bdattn_w4_pack(mc.data, mc.ld, scales.data_ptr(), mc.rows > 1 ? scales.stride(0) : 2ll * groups, packed.data_ptr(), mc.rows, K, group,
                               stream_of(a[4])));
}

// (packed, w, group, stream)
PyObject* w4_unpack(PyObject* const* a) {
    const at::Tensor &packed = tensor(a[0], "packed"), &w = tensor(a[1], "w");
    const int group = integer(a[2]);
    typed(&packed, at::kByte, "packed");
    const Matrix mw(w, "w");
    if (packed.dim() != 1 || static_cast<size_t>(packed.size(0)) != bdattn_w4_bytes(mw.rows, mw.cols, group) || (packed.size(0) > 1 && packed.stride(0) != 1) ||
        packed.size(0) == 0)
        refuse("packed must be dense, of w4_bytes(rows of w, columns of w, group) bytes");
    const int dtype = code(w, "w");
    on_gpu({&packed, &w});
    return done(bdattn_w4_unpack(packed.data_ptr(), mw.data, mw.ld, mw.rows, mw.cols, group, dtype, stream_of(a[3])));
}

// (x, w, bias, y, group, act, gate, residual, stream)
PyObject* linear_w4(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w"), &y = tensor(a[3], "y");
    const at::Tensor *bias = optional(a[2], "bias"), *gate = optional(a[6], "gate"), *residual = optional(a[7], "residual");
    const int group = integer(a[4]), act = integer(a[5]);
    const Matrix mx(x, "x"), my(y, "y");
    if (my.rows != mx.rows) refuse("y must have the rows of x");
    Matrix mr;
    if (residual != nullptr) (mr = Matrix(*residual, "residual")).same(my, "residual");
    typed(&w, at::kByte, "w");
    typed(&x, y.scalar_type(), "x");
    typed(bias, y.scalar_type(), "bias");
    typed(gate, y.scalar_type(), "gate");
    typed(residual, y.scalar_type(), "residual");
    if (w.dim() != 1 || static_cast<size_t>(w.size(0)) != bdattn_w4_bytes(my.cols, mx.cols, group) || (w.size(0) > 1 && w.stride(0) != 1) || w.size(0) == 0)
        refuse("w must be dense, of w4_bytes(columns of y, columns of x, group) bytes");
    bdattn_linear_w4_params p{};
    p.dtype = code(y, "y");
    p.M = mx.rows;
    p.N = my.cols;
    p.K = mx.cols;
    p.group = group;
    p.x = mx.data;
    p.x_ld = mx.ld;
    p.w = w.data_ptr();
    p.bias = vector(bias, my.cols, "bias");
    p.gate = vector(gate, my.cols, "gate");
    p.residual = mr.data;
    p.residual_ld = mr.ld;
    p.y = my.data;
    p.y_ld = my.ld;
    p.act = act;
    on_gpu({&x, &w, &y, bias, gate, residual});
    return done(bdattn_linear_w4_fwd(&p, stream_of(a[8])));
}

// A cache of four tensors: (B, heads, rows, bytes) codes and (B, heads, rows, groups, 2) scales, rows of a head dense.
struct Cache4 {
    const at::Tensor *k_codes, *v_codes, *k_scales, *v_scales;
    bdattn_cache4 c{};
    explicit Cache4(PyObject* const* a) {
        k_codes = &tensor(a[0], "k_codes");
        v_codes = &tensor(a[1], "v_codes");
        k_scales = &tensor(a[2], "k_scales");
        v_scales = &tensor(a[3], "v_scales");
        typed(k_codes, at::kByte, "k_codes");
        typed(v_codes, at::kByte, "v_codes");
        typed(v_scales, k_scales->scalar_type(), "v_scales");
        if (k_codes->dim() != 4 || k_scales->dim() != 5) refuse("codes must be (batch, heads, rows, bytes), scales (batch, heads, rows, groups, 2)");
        if (k_codes->sizes() != v_codes->sizes() || k_scales->sizes() != v_scales->sizes()) refuse("K and V of the cache have other shapes");
        for (int d = 0; d < 3; ++d)
            if (k_codes->size(d) != k_scales->size(d)) refuse("codes and scales of the cache have other shapes");
        const int64_t bytes = k_codes->size(3), groups = k_scales->size(3);
        if (groups < 1 || bytes < 1 || 2 * bytes % groups != 0 || k_scales->size(4) != 2) refuse("scales must be a pair for every group of a row");
        c.dtype = code(*k_scales, "k_scales");
        c.batch = rows_of(k_codes->size(0), "the cache");
        c.num_kv_heads = rows_of(k_codes->size(1), "the cache");
        c.rows = rows_of(k_codes->size(2), "the cache");
        c.head_dim = rows_of(2 * bytes, "the cache");
        c.group = static_cast<int>(2 * bytes / groups);
        // strides of dimensions of one are anything
        auto strides = [&](const at::Tensor& k, const at::Tensor& v, int64_t row, long long* head, long long* batch) {
            for (const at::Tensor* t : {&k, &v}) {
                if (t->size(2) > 1 && t->stride(2) != row) refuse("rows of a head of the cache must be dense");
                if (t->stride(t->dim() - 1) != 1 && t->size(t->dim() - 1) > 1) refuse("rows of a head of the cache must be dense");
                if (t->dim() == 5 && t->size(3) > 1 && t->stride(3) != 2) refuse("rows of a head of the cache must be dense");
            }
            if ((c.num_kv_heads > 1 && k.stride(1) != v.stride(1)) || (c.batch > 1 && k.stride(0) != v.stride(0)))
                refuse("K and V of the cache have other strides");
            *head = c.num_kv_heads > 1 ? k.stride(1) : c.rows * row;
            *batch = c.batch > 1 ? k.stride(0) : c.num_kv_heads * *head;
            if (*head == 0 || *batch == 0) refuse("heads and batch items of the cache must be memory of their own");
        };
        strides(*k_codes, *v_codes, bytes, &c.codes_head_stride, &c.codes_batch_stride);
        strides(*k_scales, *v_scales, 2 * groups, &c.scales_head_stride, &c.scales_batch_stride);
        c.k_codes = k_codes->data_ptr();
        c.v_codes = v_codes->data_ptr();
        c.k_scales = k_scales->data_ptr();
        c.v_scales = v_scales->data_ptr();
    }
};

// (k_codes, v_codes, k_scales, v_scales, k, v, kv_len, stream)
template <bool kAppend>
PyObject* cache4_rows(PyObject* const* a) {
    const Cache4 cache(a);
    const at::Tensor &k = tensor(a[4], "k"), &v = tensor(a[5], "v");
    const at::Tensor* kv_len = optional(a[6], "kv_len");
    typed(&k, cache.k_scales->scalar_type(), "k");
    typed(&v, cache.k_scales->scalar_type(), "v");
    typed(kv_len, at::kInt, "kv_len");
    const Rows mk(k, "k"), mv(v, "v");
    if (mv.rows != mk.rows || mv.cols != mk.cols || mv.batch != mk.batch) refuse("v must have the shape of k");
    if (mk.batch != cache.c.batch || mk.cols != static_cast<int64_t>(cache.c.num_kv_heads) * cache.c.head_dim)
        refuse("k and v must have the cache's batch and heads");
    if (mk.ld < mk.cols || mv.ld < mv.cols) refuse("k and v must have rows of their own");
    bdattn_cache4_rows r{};
    r.rows = mk.rows;
    r.k = mk.data;
    r.v = mv.data;
    r.k_ld = mk.ld;
    r.v_ld = mv.ld;
    r.k_batch_stride = mk.stride;
    r.v_batch_stride = mv.stride;
    r.kv_len = static_cast<const int*>(vector(kv_len, cache.c.batch, "kv_len"));
    on_gpu({cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, &k, &v, kv_len});
    return done(kAppend ? bdattn_cache4_append(&cache.c, &r, stream_of(a[7])) : bdattn_cache4_read(&cache.c, &r, stream_of(a[7])));
}

// (k_codes, v_codes, k_scales, v_scales, q, out, num_heads, window, sinks, kv_len, key_mask, softmax_scale, stream)
PyObject* sdpa_cache4(PyObject* const* a) {
    const Cache4 cache(a);
    const at::Tensor &q = tensor(a[4], "q"), &out = tensor(a[5], "out");
    const int heads = integer(a[6]), window = integer(a[7]), sinks = integer(a[8]);
    const at::Tensor *kv_len = optional(a[9], "kv_len"), *mask = optional(a[10], "key_mask");
    const float scale = real(a[11]);
    typed(&q, cache.k_scales->scalar_type(), "q");
    typed(&out, cache.k_scales->scalar_type(), "out");
    typed(kv_len, at::kInt, "kv_len");
    typed(mask, at::kFloat, "key_mask");
    const Rows mq(q, "q"), mo(out, "out");
    if (mo.rows != mq.rows || mo.cols != mq.cols || mo.batch != mq.batch) refuse("out must have the shape of q");
    if (mq.batch != cache.c.batch || heads < 1 || mq.cols != static_cast<int64_t>(heads) * cache.c.head_dim)
        refuse("q must have the cache's batch and num_heads heads of its width");
    if (mq.ld < mq.cols || mo.ld < mo.cols) refuse("q and out must have rows of their own");
    bdattn_sdpa_cache4_params p{};
    p.num_heads = heads;
    p.q_rows = mq.rows;
    p.q = mq.data;
    p.o = mo.data;
    p.q_ld = mq.ld;
    p.o_ld = mo.ld;
    p.q_batch_stride = mq.stride;
    p.o_batch_stride = mo.stride;
    p.window = window;
    p.sinks = sinks;
    p.kv_len = static_cast<const int*>(vector(kv_len, cache.c.batch, "kv_len"));
    p.key_mask = static_cast<const float*>(vector(mask, cache.c.rows, "key_mask"));
    p.softmax_scale = scale;
    on_gpu({cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, &q, &out, kv_len, mask});
    return done(bdattn_sdpa_cache4_fwd(&cache.c, &p, stream_of(a[12])));
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
    {"sandwich_norm", fast(entry<sandwich_norm, 11>), METH_FASTCALL, "bdattn_sandwich_norm_fwd"},
    {"w4_pack", fast(entry<w4_pack, 5>), METH_FASTCALL, "bdattn_w4_pack"},
    {"w4_unpack", fast(entry<w4_unpack, 4>), METH_FASTCALL, "bdattn_w4_unpack"},
    {"linear_w4", fast(entry<linear_w4, 9>), METH_FASTCALL, "bdattn_linear_w4_fwd"},
    {"cache4_append", fast(entry<cache4_rows<true>, 8>), METH_FASTCALL, "bdattn_cache4_append"},
    {"cache4_read", fast(entry<cache4_rows<false>, 8>), METH_FASTCALL, "bdattn_cache4_read"},
    {"sdpa_cache4", fast(entry<sdpa_cache4, 13>), METH_FASTCALL, "bdattn_sdpa_cache4_fwd"},
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
