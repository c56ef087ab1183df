// torch_ops.cpp — the Python side of the norm and 4-bit operators (include/tsd_ops.h): takes torch tensors, checks
// them against each other and calls the C entry point.
//
// A CPython extension instead of ctypes because these calls are short: a call with 28 arguments and
// eight tensors spends 12-16 us in Python and ctypes, several times the kernel it launches, and 2-3
// here. tsd.py gives the functions their keyword arguments; every function here takes all of its
// arguments by position, raises ValueError for tensors that do not fit together and returns the
// entry point's status.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <exception>

#include "../../include/tsd.h"
#include "../../include/tsd_ops.h"

namespace {

struct Refused : std::exception {};   // the Python error is set

[[noreturn]] void refuse(const char * format, ...) {
    va_list a;
    va_start(a, format);
    PyErr_FormatV(PyExc_ValueError, format, a);
    va_end(a);
    throw Refused();
}

// One call's arguments, taken in order.
class Args {
public:
    Args(const char * fn, PyObject * const * v, Py_ssize_t n, Py_ssize_t want) : fn(fn), v_(v) {
        if (n != want) refuse("%s: %zd arguments, not %zd", fn, n, want);
    }
    const char * fn;
    // A tensor, or null for None.
    const at::Tensor * tensor() {
        PyObject * o = *v_++;
        ++at_;
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) refuse("%s: argument %d is not a tensor", fn, at_);
        return &THPVariable_Unpack(o);
    }
    const at::Tensor & need() {
        const at::Tensor * t = tensor();
        if (!t) refuse("%s: argument %d is missing", fn, at_);
        return *t;
    }
    int integer() {
        const long v = PyLong_AsLong(*v_++);
        ++at_;
        if (v == -1 && PyErr_Occurred()) throw Refused();
        if (v < INT32_MIN || v > INT32_MAX) refuse("%s: argument %d is out of range", fn, at_);
        return (int)v;
    }
    float real() {
        const double v = PyFloat_AsDouble(*v_++);
        ++at_;
        if (v == -1.0 && PyErr_Occurred()) throw Refused();
        return (float)v;
    }
    void * stream() {
        void * p = PyLong_AsVoidPtr(*v_++);
        ++at_;
        if (!p && PyErr_Occurred()) throw Refused();
        return p;
    }

private:
    PyObject * const * v_;
    int at_ = 0;   // arguments taken, so the number (from 1) of the last one
};

void * ptr(const at::Tensor * t) { return t ? t->data_ptr() : nullptr; }
float * ptr_f(const at::Tensor * t) { return static_cast<float *>(ptr(t)); }

// ggml type number of a tensor's dtype; -1 for one that no operator takes.
int type_of(const at::Tensor & t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TSD_TYPE_F32;
        case at::kHalf: return TSD_TYPE_F16;
        case at::kBFloat16: return TSD_TYPE_BF16;
        default: return -1;
    }
}

// Row stride of a 2-D tensor with contiguous rows, of the given shape (-1: any) and, if `f32`, float32.
int64_t rows_of(const char * fn, const char * name, const at::Tensor & t, int64_t rows, int64_t cols, bool f32) {
    if (t.dim() != 2) refuse("%s: %s must be 2-D", fn, name);
    const int64_t r = t.size(0), c = t.size(1);
    if ((rows >= 0 && r != rows) || (cols >= 0 && c != cols))
        refuse("%s: %s must be [%lld][%lld], got [%lld][%lld]", fn, name, (long long)(rows < 0 ? r : rows),
               (long long)(cols < 0 ? c : cols), (long long)r, (long long)c);
    if (r > INT32_MAX || c > INT32_MAX) refuse("%s: %s is too large", fn, name);
    if (f32 && t.scalar_type() != at::kFloat) refuse("%s: %s must be float32", fn, name);
    if (c > 1 && t.stride(1) != 1) refuse("%s: %s must have contiguous rows", fn, name);
    return r > 1 ? t.stride(0) : c;
}

void vector(const char * fn, const char * name, const at::Tensor * t, int64_t n) {
    if (t && (t->dim() != 1 || t->size(0) != n || t->scalar_type() != at::kFloat || !t->is_contiguous()))
        refuse("%s: %s must be a contiguous float32 vector of %lld", fn, name, (long long)n);
}

// Row stride of a gate or modulation: [H] for every row alike, or a row for each `div` rows.
int64_t modulation(const char * fn, const char * name, const at::Tensor & t, int64_t rows, int64_t div, int64_t H) {
    if (t.dim() == 1) {
        vector(fn, name, &t, H);
        return 0;
    }
    const int64_t ld = rows_of(fn, name, t, -1, H, true);
    if (div < 1 || t.size(0) < (rows + div - 1) / div)
        refuse("%s: %s has %lld rows, too few for %lld at %lld to each", fn, name, (long long)t.size(0), (long long)rows,
               (long long)div);
    return ld;
}

void one_float(const char * fn, const at::Tensor * t) {
    if (t && (t->numel() != 1 || t->scalar_type() != at::kFloat)) refuse("%s: an absolute maximum is one float32", fn);
}

// A 4-bit tensor: contiguous bytes [rows][K / 2] and its scale tiles.
struct Fp4 {
    int rows, K;
    Fp4(const char * fn, const char * name, const at::Tensor & codes, const at::Tensor & scales, int fmt, const at::Tensor * amax) {
        if (codes.dim() != 2 || codes.element_size() != 1 || !codes.is_contiguous())
            refuse("%s: %s must be contiguous bytes [rows][K / 2]", fn, name);
        const int64_t r = codes.size(0), k = 2 * codes.size(1), want = tsd_fp4_scale_bytes(r, k, fmt);
        if (want < 0) refuse("%s: %s: no 4-bit tensor of %lld x %lld in format %d", fn, name, (long long)r, (long long)k, fmt);
        if (scales.element_size() != 1 || !scales.is_contiguous() || scales.numel() != want)
            refuse("%s: %s needs %lld contiguous bytes of scales", fn, name, (long long)want);
        one_float(fn, amax);
        rows = (int)r;
        K = (int)k;
    }
};

// Runs a call; C++ exceptions (torch's own among them) become Python errors.
template <typename F> PyObject * call(F && f) {
    try {
        return PyLong_FromLong(f());
    } catch (const Refused &) {
    } catch (const std::exception & e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

PyObject * gate_norm(PyObject *, PyObject * const * v, Py_ssize_t n) {
    return call([&] {
        Args a("tsd_op_gate_norm", v, n, 18);
        const at::Tensor & x = a.need();
        const at::Tensor * y = a.tensor(), * x_out = a.tensor(), * h = a.tensor();
        const int post = a.integer();
        const at::Tensor * post_gain = a.tensor();
        const float post_eps = a.real();
        const at::Tensor * gate = a.tensor();
        const int gate_div = a.integer();
        const float x_scale = a.real(), y_scale = a.real();
        const int pre = a.integer();
        const at::Tensor * pre_gain = a.tensor();
        const float pre_eps = a.real();
        const at::Tensor * shift = a.tensor(), * scale = a.tensor();
        const int mod_div = a.integer();
        void * stream = a.stream();
        const int64_t ldx = rows_of(a.fn, "x", x, -1, -1, true), rows = x.size(0), H = x.size(1);
        const int64_t ldy = y ? rows_of(a.fn, "y", *y, rows, H, false) : 0;
        const int64_t ldxo = x_out ? rows_of(a.fn, "x_out", *x_out, rows, H, true) : 0;
        const int64_t ldh = h ? rows_of(a.fn, "h", *h, rows, H, false) : 0;
        vector(a.fn, "post_gain", post_gain, H);
        vector(a.fn, "pre_gain", pre_gain, H);
        const int64_t ldg = gate ? modulation(a.fn, "gate", *gate, rows, gate_div, H) : 0;
        const int64_t lds = shift ? modulation(a.fn, "shift", *shift, rows, mod_div, H) : 0;
        const int64_t ldc = scale ? modulation(a.fn, "scale", *scale, rows, mod_div, H) : 0;
        if (shift && scale && lds != ldc) refuse("%s: shift and scale must have one row stride", a.fn);
        return tsd_op_gate_norm(ptr_f(&x), ldx, ptr(y), y ? type_of(*y) : 0, ldy, (int)rows, (int)H, post, ptr_f(post_gain),
                                post_eps, ptr_f(gate), ldg, gate_div, x_scale, y_scale, ptr_f(x_out), ldxo, pre,
                                ptr_f(pre_gain), pre_eps, ptr_f(shift), ptr_f(scale), shift ? lds : ldc, mod_div, ptr(h),
                                h ? type_of(*h) : 0, ldh, stream);
    });
}

PyObject * fp4_absmax(PyObject *, PyObject * const * v, Py_ssize_t n) {
    return call([&] {
        Args a("tsd_op_fp4_absmax", v, n, 3);
        const at::Tensor & x = a.need(), & amax = a.need();
        void * stream = a.stream();
        const int64_t ldx = rows_of(a.fn, "x", x, -1, -1, false);
        one_float(a.fn, &amax);
        return tsd_op_fp4_absmax(x.data_ptr(), type_of(x), (int)x.size(0), (int)x.size(1), ldx, ptr_f(&amax), stream);
    });
}

PyObject * fp4_quantize(PyObject *, PyObject * const * v, Py_ssize_t n) {
    return call([&] {
        Args a("tsd_op_fp4_quantize", v, n, 6);
        const at::Tensor & x = a.need();
        const int fmt = a.integer();
        const at::Tensor & codes = a.need(), & scales = a.need();
        const at::Tensor * amax = a.tensor();
        void * stream = a.stream();
        const Fp4 q(a.fn, "codes", codes, scales, fmt, amax);
        const int64_t ldx = rows_of(a.fn, "x", x, q.rows, q.K, false);
        return tsd_op_fp4_quantize(x.data_ptr(), type_of(x), q.rows, q.K, ldx, fmt, ptr_f(amax), codes.data_ptr(),
                                   scales.data_ptr(), stream);
    });
}

PyObject * fp4_dequantize(PyObject *, PyObject * const * v, Py_ssize_t n) {
    return call([&] {
        Args a("tsd_op_fp4_dequantize", v, n, 6);
        const at::Tensor & codes = a.need(), & scales = a.need();
        const int fmt = a.integer();
        const at::Tensor & y = a.need();
        const at::Tensor * amax = a.tensor();
        void * stream = a.stream();
        const Fp4 q(a.fn, "codes", codes, scales, fmt, amax);
        const int64_t ldy = rows_of(a.fn, "y", y, q.rows, q.K, false);
        return tsd_op_fp4_dequantize(codes.data_ptr(), scales.data_ptr(), fmt, ptr_f(amax), q.rows, q.K, y.data_ptr(),
                                     type_of(y), ldy, stream);
    });
}

PyObject * fp4_gemm(PyObject *, PyObject * const * v, Py_ssize_t n) {
    return call([&] {
        Args a("tsd_op_fp4_gemm", v, n, 13);
        const at::Tensor & W = a.need(), & Ws = a.need(), & X = a.need(), & Xs = a.need();
        const int fmt = a.integer();
        const at::Tensor & out = a.need();
        const int mode = a.integer(), act = a.integer();
        const at::Tensor * bias = a.tensor(), * w_amax = a.tensor(), * x_amax = a.tensor(), * err = a.tensor();
        void * stream = a.stream();
        const Fp4 w(a.fn, "W", W, Ws, fmt, w_amax), x(a.fn, "X", X, Xs, fmt, x_amax);
        if (w.K != x.K) refuse("%s: W has %d columns and X %d", a.fn, w.K, x.K);
        vector(a.fn, "bias", bias, w.rows);
        if (err && (err->numel() != 1 || err->scalar_type() != at::kInt)) refuse("%s: err is one int32", a.fn);
        const int64_t ldo = rows_of(a.fn, "out", out, x.rows, mode == TSD_EPI_SWIGLU ? w.rows / 2 : w.rows, false);
        return tsd_op_fp4_gemm(W.data_ptr(), Ws.data_ptr(), ptr_f(w_amax), w.rows, X.data_ptr(), Xs.data_ptr(), ptr_f(x_amax),
                               x.rows, w.K, fmt, mode, act, ptr_f(bias), out.data_ptr(), type_of(out), ldo,
                               static_cast<int *>(ptr(err)), stream);
    });
}

PyObject * fp4_gemv(PyObject *, PyObject * const * v, Py_ssize_t n) {
    return call([&] {
        Args a("tsd_op_fp4_gemv", v, n, 9);
        const at::Tensor & W = a.need(), & Ws = a.need();
        const int fmt = a.integer();
        const at::Tensor & x = a.need(), & y = a.need();
        const at::Tensor * bias = a.tensor();
        const int act = a.integer();
        const at::Tensor * w_amax = a.tensor();
        void * stream = a.stream();
        const Fp4 w(a.fn, "W", W, Ws, fmt, w_amax);
        const int64_t ldx = rows_of(a.fn, "x", x, -1, w.K, true);
        const int64_t ldy = rows_of(a.fn, "y", y, x.size(0), w.rows, false);
        vector(a.fn, "bias", bias, w.rows);
        return tsd_op_fp4_gemv(W.data_ptr(), Ws.data_ptr(), ptr_f(w_amax), fmt, w.rows, w.K, ptr_f(&x), ldx, (int)x.size(0),
                               ptr_f(bias), act, y.data_ptr(), type_of(y), ldy, stream);
    });
}

#define TSD_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TSD_METHOD(gate_norm),      TSD_METHOD(fp4_absmax), TSD_METHOD(fp4_quantize),
                         TSD_METHOD(fp4_dequantize), TSD_METHOD(fp4_gemm),   TSD_METHOD(fp4_gemv),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "tsd_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject * PyInit_tsd_torch() { return PyModule_Create(&module); }
