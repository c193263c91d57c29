// ============================================================================
//  torchops.cpp -- the Python module `tinygnn_b200._torch_ops`: the training
//  operators' entry points on torch tensors (tinygnn_b200/training.py wraps
//  them).
//
//  Each function checks its arguments, allocates its results with torch on
//  the current stream and calls one C-ABI entry point.  Small operators are
//  bound by the host: the same checks, allocations and ctypes call written in
//  Python took 14-22 us a call, about three times the kernels.
//  A refusal raises the exception class that set_errors() was given
//  (InvalidArgument), a failed call the one for TinyGNN's other errors.
// ============================================================================
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "tinygnn_b200.h"

namespace {

PyObject* g_invalid = nullptr;  // InvalidArgument(status, message)
PyObject* g_failed = nullptr;   // TinyGNNError(status, message)

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Failed : std::runtime_error {
    tg_status status;
    Failed(tg_status s, const char* m) : std::runtime_error(m), status(s) {}
};
[[noreturn]] void refuse(const char* fn, const std::string& m) { throw Refused(std::string(fn) + ": " + m); }

void check(tg_status s) {
    if (s == TG_OK) return;
    if (s == TG_ERR_INVALID_ARGUMENT) throw Refused(tg_last_error_message());
    throw Failed(s, tg_last_error_message());
}

void raise(PyObject* cls, int status, const char* m) {
    if (!cls) {
        PyErr_SetString(PyExc_RuntimeError, m);
        return;
    }
    PyObject* e = PyObject_CallFunction(cls, "is", status, m);
    if (e) {
        PyErr_SetObject(cls, e);
        Py_DECREF(e);
    }
}

template <class F>
PyObject* guarded(F&& f) noexcept {
    try {
        return f();
    } catch (const Refused& e) {
        raise(g_invalid, TG_ERR_INVALID_ARGUMENT, e.what());
    } catch (const Failed& e) {
        raise(g_failed, e.status, e.what());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

int dtype_of(const char* fn, const char* what, at::ScalarType t) {
    if (t == at::kFloat) return TG_F32;
    if (t == at::kBFloat16) return TG_BF16;
    if (t == at::kHalf) return TG_F16;
    refuse(fn, std::string(what) + " must be float32, bfloat16 or float16");
}

std::string shape_text(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

const at::Tensor& tensor(const char* fn, const char* what, PyObject* o) {
    if (!THPVariable_Check(o)) refuse(fn, std::string(what) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}

// A matrix as the C ABI takes it.
struct Matrix {
    at::Tensor t;
    int64_t rows, cols, ld;
    int dtype;
    void* p() const { return t.data_ptr(); }
};

Matrix matrix(const char* fn, const char* what, const at::Tensor& t) {
    if (t.dim() != 2 || !t.is_cuda()) refuse(fn, std::string(what) + " must be a 2-D CUDA tensor, got shape " + shape_text(t));
    Matrix m{t, t.size(0), t.size(1), 0, dtype_of(fn, what, t.scalar_type())};
    if (m.cols < 1) refuse(fn, std::string(what) + " has no columns");
    // Rows that are strided, overlap or run backwards are laid out first.
    if ((t.stride(1) != 1 && m.cols > 1) || (t.stride(0) < m.cols && m.rows > 1)) m.t = t.contiguous();
    m.ld = std::max(m.t.stride(0), m.cols);  // (the stride of a single row is arbitrary)
    return m;
}
Matrix matrix(const char* fn, const char* what, PyObject* o) { return matrix(fn, what, tensor(fn, what, o)); }

void same_type(const char* fn, const char* what, const at::Tensor& t, const at::Tensor& like) {
    if (t.scalar_type() != like.scalar_type())
        refuse(fn, std::string(what) + " is " + c10::toString(t.scalar_type()) + ", " +
                       c10::toString(like.scalar_type()) + " is needed");
}
void same_shape(const char* fn, const char* what, const at::Tensor& t, int64_t rows, int64_t cols) {
    if (t.size(0) != rows || t.size(1) != cols)
        refuse(fn, std::string(what) + " must have shape (" + std::to_string(rows) + ", " + std::to_string(cols) +
                       "), got " + shape_text(t));
}
void same_device(const char* fn, const at::Tensor& a, const at::Tensor& b) {
    if (a.device() != b.device())
        refuse(fn, "tensors on " + a.device().str() + " and " + b.device().str());
}

// The current stream of t's device, which must be the current one.
void* stream_of(const char* fn, const at::Tensor& t) {
    const auto dev = t.device().index();
    if (dev != c10::cuda::current_device())
        refuse(fn, "the tensors are on " + t.device().str() + ", which is not the current CUDA device");
    return c10::cuda::getCurrentCUDAStream(dev).stream();
}

at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}

// A matrix in the saved form: codes (rows x cols, rows 16-byte aligned) and exponents.
struct Saved {
    at::Tensor codes, exps;
    int64_t ld, lde;
    int8_t* c() const { return static_cast<int8_t*>(codes.data_ptr()); }
    uint8_t* e() const { return static_cast<uint8_t*>(exps.data_ptr()); }
};
Saved fresh_saved(int64_t rows, int64_t cols, const at::Tensor& like) {
    const int64_t ld = (cols + 15) / 16 * 16, nb = (cols + 127) / 128;
    at::Tensor codes = fresh({rows, ld}, at::kChar, like);
    if (ld != cols) codes = codes.narrow(1, 0, cols);
    return {codes, fresh({rows, nb}, at::kByte, like), ld, nb};
}
Saved saved(const char* fn, PyObject* codes, PyObject* exps) {
    Saved s{tensor(fn, "codes", codes), tensor(fn, "exponents", exps), 0, 0};
    const at::Tensor &c = s.codes, &e = s.exps;
    if (c.dim() != 2 || e.dim() != 2 || c.scalar_type() != at::kChar || e.scalar_type() != at::kByte || !c.is_cuda() ||
        !e.is_cuda())
        refuse(fn, "a saved matrix holds a 2-D int8 and a 2-D uint8 CUDA tensor");
    if (c.size(1) < 1) refuse(fn, "the saved matrix has no columns");
    const int64_t nb = (c.size(1) + 127) / 128;
    if (e.size(0) != c.size(0) || e.size(1) != nb)
        refuse(fn, "exponents of shape " + shape_text(e) + " do not fit codes of shape " + shape_text(c));
    same_device(fn, c, e);
    s.ld = c.size(0) > 1 ? c.stride(0) : (c.size(1) + 15) / 16 * 16;
    s.lde = c.size(0) > 1 ? e.stride(0) : nb;
    if (c.size(0) > 0 && ((c.stride(1) != 1 && c.size(1) > 1) || s.ld % 16 != 0 || s.ld < c.size(1) ||
                          reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0 || (e.stride(1) != 1 && nb > 1) ||
                          s.lde < nb))
        refuse(fn, "rows of codes must be contiguous and start at multiples of 16 bytes");
    return s;
}

// A matrix given as it was (x) or saved (codes, exps): exactly one is there.
struct Either {
    bool is_saved;
    Matrix m;
    Saved s;
    const at::Tensor& t() const { return is_saved ? s.codes : m.t; }
    const void* p() const { return is_saved ? nullptr : m.p(); }
    int64_t ld() const { return is_saved ? 0 : m.ld; }
    const int8_t* c() const { return is_saved ? s.c() : nullptr; }
    const uint8_t* e() const { return is_saved ? s.e() : nullptr; }
};
Either either(const char* fn, const char* what, PyObject* x, PyObject* codes, PyObject* exps, const at::Tensor& like) {
    Either r{};
    r.is_saved = x == Py_None;
    if (r.is_saved) {
        r.s = saved(fn, codes, exps);
    } else {
        r.m = matrix(fn, what, x);
        same_type(fn, what, r.m.t, like);
    }
    same_device(fn, r.t(), like);
    return r;
}

int64_t integer(const char* fn, PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(fn, "an integer is needed");
    }
    return v;
}
float number(const char* fn, PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(fn, "a number is needed");
    }
    return static_cast<float>(v);
}

bool truth(const char* fn, PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        refuse(fn, "a truth value is needed");
    }
    return v == 1;
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
template <class... A>
PyObject* pack(A&&... a) {
    PyObject* r = PyTuple_New(sizeof...(A));
    if (!r) return nullptr;
    Py_ssize_t i = 0;
    (PyTuple_SET_ITEM(r, i++, wrap(std::forward<A>(a))), ...);
    return r;
}

void arity(const char* fn, Py_ssize_t got, Py_ssize_t want) {
    if (got != want) refuse(fn, "takes " + std::to_string(want) + " arguments, got " + std::to_string(got));
}

using Args = PyObject* const*;

// ── 8-bit saved activations ──────────────────────────────────────────────
// save8(x) -> (codes, exponents)
PyObject* py_save8(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "save8";
        arity(fn, n, 1);
        const Matrix x = matrix(fn, "x", a[0]);
        void* st = stream_of(fn, x.t);
        Saved s = fresh_saved(x.rows, x.cols, x.t);
        check(tg_save8(x.rows, x.cols, x.dtype, x.p(), x.ld, TG_ACT_NONE, 0.0f, nullptr, 0, s.c(), s.ld, s.e(), s.lde,
                       st));
        return pack(s.codes, s.exps);
    });
}

// activation_save8(x, act, alpha) -> (y, codes, exponents)
PyObject* py_activation_save8(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "activation_save8";
        arity(fn, n, 3);
        const Matrix x = matrix(fn, "x", a[0]);
        void* st = stream_of(fn, x.t);
        at::Tensor y = fresh({x.rows, x.cols}, x.t.scalar_type(), x.t);
        Saved s = fresh_saved(x.rows, x.cols, x.t);
        check(tg_save8(x.rows, x.cols, x.dtype, x.p(), x.ld, static_cast<int>(integer(fn, a[1])), number(fn, a[2]),
                       y.data_ptr(), x.cols, s.c(), s.ld, s.e(), s.lde, st));
        return pack(y, s.codes, s.exps);
    });
}

// restore8(codes, exponents, like dtype: 0 fp32, 1 bf16, 2 fp16) -> y
PyObject* py_restore8(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "restore8";
        arity(fn, n, 3);
        const Saved s = saved(fn, a[0], a[1]);
        const int64_t d = integer(fn, a[2]);
        void* st = stream_of(fn, s.codes);
        at::Tensor y = fresh(s.codes.sizes(), d == TG_F32 ? at::kFloat : (d == TG_BF16 ? at::kBFloat16 : at::kHalf),
                             s.codes);
        check(tg_restore8(y.size(0), y.size(1), s.c(), s.ld, s.e(), s.lde, static_cast<int>(d), y.data_ptr(), y.size(1),
                          st));
        return wrap(y);
    });
}

// activation_backward(dy, x, codes, exponents, act, alpha) -> dx
PyObject* py_activation_backward(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "activation_backward";
        arity(fn, n, 6);
        const Matrix dy = matrix(fn, "dy", a[0]);
        const Either x = either(fn, "x", a[1], a[2], a[3], dy.t);
        same_shape(fn, "x", x.t(), dy.rows, dy.cols);
        void* st = stream_of(fn, dy.t);
        at::Tensor dx = fresh({dy.rows, dy.cols}, dy.t.scalar_type(), dy.t);
        check(tg_activation_grad(dy.rows, dy.cols, dy.dtype, dy.p(), dy.ld, x.p(), x.ld(), x.c(), x.s.ld, x.e(), x.s.lde,
                                 static_cast<int>(integer(fn, a[4])), number(fn, a[5]), dx.data_ptr(), dy.cols, st));
        return wrap(dx);
    });
}

// ── layer norm ───────────────────────────────────────────────────────────
at::Tensor param(const char* fn, const char* what, PyObject* o, const Matrix& x) {
    const at::Tensor& t = tensor(fn, what, o);
    if (t.numel() != x.cols)
        refuse(fn, std::string(what) + " must have " + std::to_string(x.cols) + " elements, got " +
                       std::to_string(t.numel()));
    if (!t.is_cuda() || (t.scalar_type() != at::kFloat && t.scalar_type() != x.t.scalar_type()))
        refuse(fn, std::string(what) + " must be a float32 CUDA tensor or of the rows' type");
    same_device(fn, x.t, t);
    return t.is_contiguous() ? t : t.contiguous();
}

// layer_norm(x, gamma, beta, eps, save8) -> (y, stats[, codes, exponents])
PyObject* py_layer_norm(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "layer_norm";
        arity(fn, n, 5);
        const Matrix x = matrix(fn, "x", a[0]);
        const at::Tensor gamma = param(fn, "gamma", a[1], x), beta = param(fn, "beta", a[2], x);
        same_type(fn, "beta", beta, gamma);
        const bool save = truth(fn, a[4]);
        void* st = stream_of(fn, x.t);
        at::Tensor y = fresh({x.rows, x.cols}, x.t.scalar_type(), x.t), stats = fresh({x.rows, 2}, at::kFloat, x.t);
        Saved s{};
        if (save) s = fresh_saved(x.rows, x.cols, x.t);
        check(tg_layer_norm(x.rows, x.cols, x.dtype, x.p(), x.ld, dtype_of(fn, "gamma", gamma.scalar_type()),
                            gamma.data_ptr(), beta.data_ptr(), number(fn, a[3]), y.data_ptr(), x.cols,
                            static_cast<float*>(stats.data_ptr()), save ? s.c() : nullptr, s.ld,
                            save ? s.e() : nullptr, s.lde, st));
        return save ? pack(y, stats, s.codes, s.exps) : pack(y, stats);
    });
}

// layer_norm_backward(dy, x, codes, exponents, stats, gamma) -> (dx, dgamma, dbeta)
PyObject* py_layer_norm_backward(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "layer_norm_backward";
        arity(fn, n, 6);
        const Matrix dy = matrix(fn, "dy", a[0]);
        const Either x = either(fn, "saved", a[1], a[2], a[3], dy.t);
        same_shape(fn, "saved", x.t(), dy.rows, dy.cols);
        const at::Tensor& stats = tensor(fn, "stats", a[4]);
        if (stats.dim() != 2 || stats.size(0) != dy.rows || stats.size(1) != 2 || stats.scalar_type() != at::kFloat ||
            !stats.is_contiguous() || !stats.is_cuda())
            refuse(fn, "stats must be a contiguous float32 CUDA tensor of shape (" + std::to_string(dy.rows) + ", 2)");
        same_device(fn, dy.t, stats);
        const at::Tensor gamma = param(fn, "gamma", a[5], dy);
        void* st = stream_of(fn, dy.t);
        at::Tensor dx = fresh({dy.rows, dy.cols}, dy.t.scalar_type(), dy.t),
                   dg = fresh({dy.cols}, gamma.scalar_type(), dy.t), db = fresh({dy.cols}, gamma.scalar_type(), dy.t);
        check(tg_layer_norm_grad(dy.rows, dy.cols, dy.dtype, dy.p(), dy.ld, x.p(), x.ld(), x.c(), x.s.ld, x.e(),
                                 x.s.lde, static_cast<const float*>(stats.data_ptr()),
                                 dtype_of(fn, "gamma", gamma.scalar_type()), gamma.data_ptr(), dx.data_ptr(), dy.cols,
                                 dg.data_ptr(), db.data_ptr(), st));
        return pack(dx, dg, db);
    });
}

// ── typed linear maps ────────────────────────────────────────────────────
const int32_t* offsets_of(const char* fn, PyObject* o, int64_t types, const at::Tensor& like) {
    const at::Tensor& t = tensor(fn, "offsets", o);
    if (t.scalar_type() != at::kInt || !t.is_cuda() || t.dim() != 1 || !t.is_contiguous())
        refuse(fn, "offsets must be a contiguous 1-D int32 CUDA tensor");
    if (types >= 0 && t.numel() != types + 1)
        refuse(fn, std::to_string(types) + " types need " + std::to_string(types + 1) + " offsets, got " +
                       std::to_string(t.numel()));
    same_device(fn, like, t);
    return static_cast<const int32_t*>(t.data_ptr());
}

struct Weight {
    at::Tensor t;
    int64_t types, K, N, ld, stride;
};
Weight weight(const char* fn, PyObject* o, const Matrix& x, bool by_rows) {
    const at::Tensor& t = tensor(fn, "w", o);
    if (t.dim() != 3 || !t.is_cuda())
        refuse(fn, "w must be a 3-D CUDA tensor (types x inputs x outputs), got shape " + shape_text(t));
    same_type(fn, "w", t, x.t);
    Weight w{t, t.size(0), t.size(1), t.size(2), 0, 0};
    if (x.cols != (by_rows ? w.K : w.N) || w.types < 1 || w.K < 1 || w.N < 1)
        refuse(fn, "dimension mismatch — the rows are " + std::to_string(x.cols) + " wide, w has shape " + shape_text(t));
    same_device(fn, x.t, t);
    if ((t.stride(2) != 1 && w.N > 1) || (t.stride(1) < w.N && w.K > 1) ||
        (t.stride(0) < (w.K - 1) * t.stride(1) + w.N && w.types > 1))
        w.t = t.contiguous();
    w.ld = w.K > 1 ? w.t.stride(1) : std::max(w.t.stride(1), w.N);
    w.stride = w.types > 1 ? w.t.stride(0) : std::max(w.t.stride(0), (w.K - 1) * w.ld + w.N);
    return w;
}

// typed_linear(x, w, offsets, bias, act, alpha, save8) -> (y[, codes, exponents])
PyObject* py_typed_linear(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "typed_linear";
        arity(fn, n, 7);
        const Matrix x = matrix(fn, "x", a[0]);
        const Weight w = weight(fn, a[1], x, true);
        const int32_t* off = offsets_of(fn, a[2], w.types, x.t);
        at::Tensor bias;
        if (a[3] != Py_None) {
            bias = tensor(fn, "bias", a[3]);
            if (bias.dim() != 2 || bias.size(0) != w.types || bias.size(1) != w.N ||
                bias.scalar_type() != at::kFloat || !bias.is_cuda())
                refuse(fn, "bias must be a float32 CUDA tensor of shape (" + std::to_string(w.types) + ", " +
                               std::to_string(w.N) + "), got " + shape_text(bias));
            same_device(fn, x.t, bias);
            bias = bias.contiguous();
        }
        const bool save = truth(fn, a[6]);
        void* st = stream_of(fn, x.t);
        at::Tensor y = fresh({x.rows, w.N}, x.t.scalar_type(), x.t);
        Saved s{};
        if (save) s = fresh_saved(x.rows, w.N, x.t);
        check(tg_typed_linear(x.rows, w.K, w.N, w.types, x.dtype, x.p(), x.ld, w.t.data_ptr(), w.ld, w.stride, off,
                              bias.defined() ? static_cast<const float*>(bias.data_ptr()) : nullptr,
                              static_cast<int>(integer(fn, a[4])), number(fn, a[5]), y.data_ptr(), w.N,
                              save ? s.c() : nullptr, s.ld, save ? s.e() : nullptr, s.lde, st));
        return save ? pack(y, s.codes, s.exps) : pack(y);
    });
}

// typed_linear_grad_input(dy, w, offsets) -> dx
PyObject* py_typed_linear_grad_input(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&] {
        const char* fn = "typed_linear_grad_input";
        arity(fn, n, 3);
        const Matrix dy = matrix(fn, "dy", a[0]);
        const Weight w = weight(fn, a[1], dy, false);
        const int32_t* off = offsets_of(fn, a[2], w.types, dy.t);
        void* st = stream_of(fn, dy.t);
        at::Tensor dx = fresh({dy.rows, w.K}, dy.t.scalar_type(), dy.t);
        check(tg_typed_linear_grad_input(dy.rows, w.K, w.N, w.types, dy.dtype, dy.p(), dy.ld, w.t.data_ptr(), w.ld,
                                         w.stride, off, dx.data_ptr(), w.K, st));
        return wrap(dx);
    });
}

// typed_linear_grad_weight(dy, x, codes, exponents, offsets, fp32 dw, bias) -> (dw, db or None)
PyObject* py_typed_linear_grad_weight(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* fn = "typed_linear_grad_weight";
        arity(fn, n, 7);
        const Matrix dy = matrix(fn, "dy", a[0]);
        const Either x = either(fn, "x", a[1], a[2], a[3], dy.t);
        if (x.t().size(0) != dy.rows)
            refuse(fn, "x has " + std::to_string(x.t().size(0)) + " rows and dy " + std::to_string(dy.rows));
        const int64_t K = x.t().size(1), N = dy.cols;
        const int32_t* off = offsets_of(fn, a[4], -1, dy.t);
        const int64_t types = THPVariable_Unpack(a[4]).numel() - 1;
        if (types < 1) refuse(fn, "offsets need at least two elements");
        const bool wide = truth(fn, a[5]), bias = truth(fn, a[6]);
        void* st = stream_of(fn, dy.t);
        at::Tensor dw = fresh({types, K, N}, wide ? at::kFloat : dy.t.scalar_type(), dy.t), db;
        if (bias) db = fresh({types, N}, at::kFloat, dy.t);
        check(tg_typed_linear_grad_weight(dy.rows, K, N, types, dy.dtype, x.p(), x.ld(), x.c(), x.s.ld, x.e(), x.s.lde,
                                          dy.p(), dy.ld, off, wide ? static_cast<int>(TG_F32) : dy.dtype, dw.data_ptr(),
                                          N, K * N, bias ? static_cast<float*>(db.data_ptr()) : nullptr, st));
        PyObject* r = PyTuple_New(2);
        if (!r) return nullptr;
        PyTuple_SET_ITEM(r, 0, wrap(dw));
        if (bias) {
            PyTuple_SET_ITEM(r, 1, wrap(db));
        } else {
            Py_INCREF(Py_None);
            PyTuple_SET_ITEM(r, 1, Py_None);
        }
        return r;
    });
}

// check_row_offsets(offsets, rows)
PyObject* py_check_row_offsets(PyObject*, Args a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* fn = "check_row_offsets";
        arity(fn, n, 2);
        const at::Tensor& t = tensor(fn, "offsets", a[0]);
        const int32_t* off = offsets_of(fn, a[0], -1, t);
        const int64_t rows = integer(fn, a[1]);
        check(tg_typed_check_offsets(rows, t.numel() - 1, off, stream_of(fn, t)));
        Py_RETURN_NONE;
    });
}

// set_errors(InvalidArgument, TinyGNNError)
PyObject* py_set_errors(PyObject*, PyObject* args) {
    PyObject *invalid, *failed;
    if (!PyArg_ParseTuple(args, "OO", &invalid, &failed)) return nullptr;
    Py_INCREF(invalid);
    Py_INCREF(failed);
    Py_XSETREF(g_invalid, invalid);
    Py_XSETREF(g_failed, failed);
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FAST(save8),
                          FAST(activation_save8),
                          FAST(restore8),
                          FAST(activation_backward),
                          FAST(layer_norm),
                          FAST(layer_norm_backward),
                          FAST(typed_linear),
                          FAST(typed_linear_grad_input),
                          FAST(typed_linear_grad_weight),
                          FAST(check_row_offsets),
                          {"set_errors", py_set_errors, METH_VARARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", "Training operators on torch tensors.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__torch_ops() { return PyModule_Create(&kModule); }
