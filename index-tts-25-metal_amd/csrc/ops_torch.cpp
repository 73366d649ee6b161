// The operators of include/itts_ops.h on torch tensors: checks of the arguments, outputs, the current stream.
//
// Module _itts_ops, used by itts_ops.py, which documents the calls.  A call of a single-token kernel
// takes a few microseconds on the GPU; the same checks written in Python took 15 to 20 of them, so
// they stand here.  Host code only: it hands addresses to the C ABI.
#include <Python.h>

#include <initializer_list>
#include <sstream>
#include <stdexcept>
#include <string>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "itts_ops.h"

namespace {
using at::Tensor;

PyObject* g_invalid = nullptr;  // InvalidArgument, GptRuntimeError, LogicError of itts_gpt
PyObject* g_runtime = nullptr;
PyObject* g_logic = nullptr;

struct Invalid : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Failed {
    int status;
};

template <class... A>
[[noreturn]] void no(const A&... parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw Invalid(s.str());
}
const char* name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        default: return c10::toString(t);
    }
}
std::string size_of(const Tensor& t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}

int kind_of(at::ScalarType t) {
    return t == at::kFloat ? ITTS_T_F32 : t == at::kBFloat16 ? ITTS_T_BF16 : t == at::kHalf ? ITTS_T_F16 : -1;
}
at::ScalarType type_of(int kind) { return kind == ITTS_T_F32 ? at::kFloat : kind == ITTS_T_BF16 ? at::kBFloat16 : at::kHalf; }

// ------------------------------------------------------------------ arguments
const Tensor* optional(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) no(name, ": a tensor is wanted");
    return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* name) {
    const Tensor* t = optional(o, name);
    if (!t) no(name, ": a tensor is wanted");
    return *t;
}
int64_t whole(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        no(name, ": a whole number is wanted");
    }
    return v;
}
double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        no(name, ": a number is wanted");
    }
    return v;
}
int64_t group_of(PyObject* o) {
    const int64_t g = whole(o, "group");
    if (g != 32 && g != 64 && g != 128) no("group: 32, 64 or 128 is wanted, not ", g);
    return g;
}

struct Matrix {
    int kind;
    int64_t rows, cols, stride;
};
// A float matrix with unit column stride.
Matrix matrix(const Tensor& t, const char* name) {
    const int kind = kind_of(t.scalar_type());
    if (kind < 0) no(name, ": float32, bfloat16 or float16 is wanted, not ", name_of(t.scalar_type()));
    if (t.dim() != 2) no(name, ": a matrix is wanted, not ", t.dim(), " dimensions");
    const int64_t rows = t.size(0), cols = t.size(1);
    if (cols > 1 && t.stride(1) != 1) no(name, ": columns have to lie next to each other");
    return {kind, rows, cols, rows > 1 ? t.stride(0) : cols};  // (the stride of a single row says nothing)
}
// Another matrix of x's type: its row stride.
int64_t like(const Tensor& t, at::ScalarType type, int64_t rows, int64_t cols, const char* name) {
    if (t.scalar_type() != type || t.dim() != 2 || t.size(0) != rows || t.size(1) != cols)
        no(name, ": ", name_of(type), " [", rows, ", ", cols, "] is wanted, not ", name_of(t.scalar_type()), " ", size_of(t));
    return matrix(t, name).stride;
}
void vector(const Tensor& t, int64_t n, const char* name) {
    if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1)) no(name, ": ", n, " contiguous values are wanted, not ", size_of(t));
}
int norm_weight(const Tensor& w, const Tensor& x, int64_t cols, const char* name) {
    vector(w, cols, name);
    if (w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat)
        no(name, ": ", name_of(x.scalar_type()), " or float32 is wanted, not ", name_of(w.scalar_type()));
    return kind_of(w.scalar_type());
}

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct Weight {
    const Tensor *packed, *scales;
    int64_t n, k, group;
};
// A Q4Weight: (packed, scales, n, k, group).
Weight weight_of(PyObject* o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) no("weight: a Q4Weight is wanted");
    Weight w{&tensor(PyTuple_GET_ITEM(o, 0), "weight.packed"), &tensor(PyTuple_GET_ITEM(o, 1), "weight.scales"),
             whole(PyTuple_GET_ITEM(o, 2), "weight.n"), whole(PyTuple_GET_ITEM(o, 3), "weight.k"), group_of(PyTuple_GET_ITEM(o, 4))};
    if (w.n < 1 || w.k < 1 || w.n > (int64_t(1) << 40) || w.k > (int64_t(1) << 20)) no("weight: sizes out of range: ", w.n, " x ", w.k);
    const int64_t tiles = up(w.n, 16) / 16 * (up(w.k, 128) / 128);
    if (w.packed->scalar_type() != at::kByte || w.packed->numel() != tiles * 1024 || !w.packed->is_contiguous())
        no("weight: packed codes of ", w.n, " x ", w.k, " are ", tiles * 1024, " contiguous bytes");
    if (w.scales->scalar_type() != at::kBFloat16 || w.scales->numel() != tiles * (2048 / w.group) || !w.scales->is_contiguous())
        no("weight: the scales of ", w.n, " x ", w.k, " are ", tiles * (2048 / w.group), " contiguous bfloat16 values");
    return w;
}

// The device that all tensors of a call are on, made current for its scope, and its current stream.
class On {
public:
    explicit On(const Tensor& first) : first_(first) {}
    void also(const Tensor* t) const {
        if (!t) return;
        if (!t->is_cuda()) no("tensors have to be on the GPU");
        if (t->device() != first_.device()) no("tensors on ", first_.device().str(), " and ", t->device().str());
        if (t->is_neg()) no("a negated view: resolve_neg() it first");
        if (t->requires_grad() && c10::GradMode::is_enabled())
            no("these operators have no gradients: detach the tensors, or call under torch.no_grad()");
        // (a dual tensor of forward mode: its tangent would be lost)
        if (t->_fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
            no("these operators have no gradients: unpack_dual() the tensors of forward mode");
    }
    void enter() {
        also(&first_);
        const auto to = first_.device().index(), now = c10::hip::current_device();
        if (to != now) {
            c10::hip::set_device(to);
            back_ = now;
        }
        stream_ = c10::hip::getCurrentHIPStream(to).stream();
    }
    ~On() {
        if (back_ >= 0) {
            try {
                c10::hip::set_device(back_);
            } catch (...) {
            }
        }
    }
    void* stream() const { return stream_; }

private:
    const Tensor& first_;
    c10::DeviceIndex back_ = -1;
    void* stream_ = nullptr;
};
void done(int status) {
    if (status != ITTS_OK) throw Failed{status};
}
void* at_of(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

// A given output, before the call and after it: autograd has to see that its values change, by a call that is not refused.
const Tensor& writable(const Tensor& t) {
    if (t.is_inference() && !c10::InferenceMode::is_enabled()) no("an output made in inference mode, outside of it");
    return t;
}
void written(std::initializer_list<const Tensor*> given) {
    for (const Tensor* t : given)
        if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

Tensor make(at::IntArrayRef sizes, const Tensor& like_, at::ScalarType type) { return at::detail::empty_cuda(sizes, type, like_.device(), std::nullopt); }

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

// ------------------------------------------------------------------ rows to 8 bits
struct Codes {
    Tensor q, scales;
};
// q and scales as they are given, checked, or (on(): the call's tensors are on the GPU) made.
template <class F>
Codes codes(const Tensor& x, int64_t rows, int64_t cols, int64_t group, const Tensor* q, const Tensor* scales, F&& on) {
    const int64_t kp = up(cols, 128);
    if (q && (q->scalar_type() != at::kChar || q->dim() != 2 || q->size(0) != rows || q->size(1) != kp || !q->is_contiguous()))
        no("q: contiguous int8 [", rows, ", ", kp, "] is wanted");
    if (scales && (scales->scalar_type() != at::kFloat || scales->dim() != 2 || scales->size(0) != rows || scales->size(1) != kp / group ||
                   !scales->is_contiguous()))
        no("scales: contiguous float32 [", rows, ", ", kp / group, "] is wanted");
    on();
    return {q ? writable(*q) : make({rows, kp}, x, at::kChar), scales ? writable(*scales) : make({rows, kp / group}, x, at::kFloat)};
}

// (x, weight or None, eps, residual, group, h, q, scales, values) -> (h, q, scales, values)
PyObject* rows_to_codes(PyObject* const* a, bool norm) {
    const Tensor& x = tensor(a[0], "x");
    const Matrix m = matrix(x, "x");
    const int64_t group = group_of(a[4]);
    const Tensor* w = nullptr;
    int wkind = m.kind;
    double eps = 0;
    if (norm) {
        w = &tensor(a[1], "weight");
        wkind = norm_weight(*w, x, m.cols, "weight");
        eps = number(a[2], "eps");
    }
    const Tensor *residual = optional(a[3], "residual"), *h_in = optional(a[5], "h"), *v_in = nullptr;
    int64_t rs = 0, hs = m.cols, vs = m.cols;
    if (residual) rs = like(*residual, x.scalar_type(), m.rows, m.cols, "residual");
    if (h_in) hs = like(*h_in, x.scalar_type(), m.rows, m.cols, "h");
    const bool values = a[8] == Py_True;
    if (!values && a[8] != Py_False) v_in = optional(a[8], "values");
    if (v_in) vs = like(*v_in, x.scalar_type(), m.rows, m.cols, "values");
    const Tensor *q_in = optional(a[6], "q"), *s_in = optional(a[7], "scales");
    On on(x);
    const Codes c = codes(x, m.rows, m.cols, group, q_in, s_in, [&] {
        for (const Tensor* t : {w, residual, h_in, v_in, q_in, s_in}) on.also(t);
        on.enter();
    });
    Tensor h, v;
    if (h_in) h = writable(*h_in);
    else if (residual) h = make({m.rows, m.cols}, x, x.scalar_type());
    if (v_in) v = writable(*v_in);
    else if (values) v = make({m.rows, m.cols}, x, x.scalar_type());
    void* const hp = h.defined() ? h.data_ptr() : nullptr;
    void* const vp = v.defined() ? v.data_ptr() : nullptr;
    if (norm)
        done(itts_rmsnorm_q8(x.data_ptr(), m.stride, at_of(residual), rs, w->data_ptr(), wkind, m.kind, m.rows, m.cols, static_cast<float>(eps),
                             static_cast<int32_t>(group), hp, hs, vp, vs, static_cast<int8_t*>(c.q.data_ptr()), static_cast<float*>(c.scales.data_ptr()), on.stream()));
    else
        done(itts_q8_quantize(x.data_ptr(), m.stride, m.kind, m.rows, m.cols, static_cast<int32_t>(group), vp, vs, static_cast<int8_t*>(c.q.data_ptr()),
                              static_cast<float*>(c.scales.data_ptr()), on.stream()));
    written({h_in, v_in, q_in, s_in});
    PyObject* out = PyTuple_New(norm ? 4 : 3);
    if (!out) throw python_error();
    int i = 0;
    if (norm) {
        if (h.defined()) PyTuple_SET_ITEM(out, i++, wrap(h));
        else {
            Py_INCREF(a[0]);
            PyTuple_SET_ITEM(out, i++, a[0]);
        }
    }
    PyTuple_SET_ITEM(out, i++, wrap(c.q));
    PyTuple_SET_ITEM(out, i++, wrap(c.scales));
    if (v.defined()) PyTuple_SET_ITEM(out, i, wrap(v));
    else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(out, i, Py_None);
    }
    return out;
}

// ------------------------------------------------------------------ packing
// (w, group) -> (packed, scales, n, k, group)
PyObject* pack(PyObject* const* a) {
    const Tensor& w = tensor(a[0], "w");
    const Matrix m = matrix(w, "w");
    const int64_t group = group_of(a[1]);
    if (m.rows < 1 || m.cols < 1) no("w: a matrix without rows or columns");
    On on(w);
    on.enter();
    const int64_t nt = up(m.rows, 16) / 16, kb = up(m.cols, 128) / 128;
    const Tensor packed = make({nt, kb, 1024}, w, at::kByte), scales = make({nt, kb, 16, 128 / group}, w, at::kBFloat16);
    done(itts_q4_pack(w.data_ptr(), m.stride, m.kind, m.rows, m.cols, static_cast<int32_t>(group), packed.data_ptr(), scales.data_ptr(), on.stream()));
    return Py_BuildValue("(NNLLL)", wrap(packed), wrap(scales), static_cast<long long>(m.rows), static_cast<long long>(m.cols), static_cast<long long>(group));
}

int kind_arg(PyObject* o, const char* name) {
    const int64_t k = whole(o, name);
    if (k < 0 || k > 2) no(name, ": float32, bfloat16 or float16 is wanted");
    return static_cast<int>(k);
}

// (weight, kind, out) -> out
PyObject* unpack(PyObject* const* a) {
    const Weight w = weight_of(a[0]);
    const int kind = kind_arg(a[1], "dtype");
    const Tensor* given = optional(a[2], "out");
    const int64_t os = given ? like(*given, type_of(kind), w.n, w.k, "out") : w.k;
    On on(*w.packed);
    on.also(w.scales);
    on.also(given);
    on.enter();
    const Tensor out = given ? writable(*given) : make({w.n, w.k}, *w.packed, type_of(kind));
    done(itts_q4_unpack(w.packed->data_ptr(), w.scales->data_ptr(), w.n, w.k, static_cast<int32_t>(w.group), kind, out.data_ptr(), os, on.stream()));
    written({given});
    return wrap(out);
}

// ------------------------------------------------------------------ products
// What a product adds and where it goes: (bias, residual, swiglu, kind, out).
struct Product {
    const Tensor *bias, *residual, *given;
    bool swiglu;
    int kind;
    int64_t cols, rs, os;
    Product(PyObject* const* a, int64_t rows, const Weight& w) {
        kind = kind_arg(a[3], "out_dtype");
        const int truth = PyObject_IsTrue(a[2]);
        if (truth < 0) throw python_error();
        swiglu = truth;
        if (swiglu && w.n % 2) no("swiglu: pairs of columns are wanted, not ", w.n, " columns");
        cols = swiglu ? w.n / 2 : w.n;
        bias = optional(a[0], "bias");
        if (bias) {
            vector(*bias, w.n, "bias");
            if (bias->scalar_type() != at::kFloat) no("bias: float32 is wanted, not ", name_of(bias->scalar_type()));
        }
        given = optional(a[4], "out");
        os = given ? like(*given, type_of(kind), rows, cols, "out") : cols;
        residual = optional(a[1], "residual");
        rs = residual ? like(*residual, type_of(kind), rows, cols, "residual") : 0;
    }
    void on(const On& o, const Weight& w) const {
        for (const Tensor* t : {w.packed, w.scales, bias, residual, given}) o.also(t);
    }
    Tensor out(int64_t rows, const Tensor& x) const { return given ? writable(*given) : make({rows, cols}, x, type_of(kind)); }
    const float* bias_at() const { return static_cast<const float*>(at_of(bias)); }
    uint32_t flags() const { return swiglu ? ITTS_Q4_SWIGLU : 0u; }
};

// (q, scales, weight, bias, residual, swiglu, kind, out) -> out
PyObject* matmul(PyObject* const* a) {
    const Tensor &q = tensor(a[0], "q"), &s = tensor(a[1], "scales");
    const Weight w = weight_of(a[2]);
    const int64_t kp = up(w.k, 128);
    if (q.scalar_type() != at::kChar || q.dim() != 2 || q.size(1) != kp || !q.is_contiguous())
        no("q: contiguous int8 rows of ", kp, " codes are wanted, not ", c10::toString(q.scalar_type()), " ", size_of(q));
    const int64_t rows = q.size(0);
    if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != rows || s.size(1) != kp / w.group || !s.is_contiguous())
        no("scales: contiguous float32 [", rows, ", ", kp / w.group, "] is wanted, not ", c10::toString(s.scalar_type()), " ", size_of(s));
    const Product p(a + 3, rows, w);
    On on(q);
    on.also(&s);
    p.on(on, w);
    on.enter();
    const Tensor out = p.out(rows, q);
    done(itts_q4_matmul(static_cast<const int8_t*>(q.data_ptr()), static_cast<const float*>(s.data_ptr()), rows, w.packed->data_ptr(), w.scales->data_ptr(), w.n,
                        w.k, static_cast<int32_t>(w.group), p.bias_at(), at_of(p.residual), p.rs, p.flags(), p.kind, out.data_ptr(), p.os, on.stream()));
    written({p.given});
    return wrap(out);
}

// (x, weight, norm_weight, eps, bias, residual, swiglu, kind, out) -> out
PyObject* linear(PyObject* const* a) {
    const Tensor& x = tensor(a[0], "x");
    const Matrix m = matrix(x, "x");
    const Weight w = weight_of(a[1]);
    if (m.cols != w.k) no("x: rows of ", w.k, " are wanted, not ", m.cols);
    const Tensor* nw = optional(a[2], "norm_weight");
    const int wkind = nw ? norm_weight(*nw, x, m.cols, "norm_weight") : m.kind;
    const double eps = number(a[3], "eps");
    const Product p(a + 4, m.rows, w);
    On on(x);
    on.also(nw);
    p.on(on, w);
    on.enter();
    const Tensor out = p.out(m.rows, x);
    const size_t need = itts_q4_linear_workspace(m.rows, w.n, w.k, static_cast<int32_t>(w.group));
    const Tensor work = need ? make({static_cast<int64_t>(need)}, x, at::kByte) : Tensor();
    done(itts_q4_linear(x.data_ptr(), m.stride, m.kind, m.rows, at_of(nw), wkind, static_cast<float>(eps), w.packed->data_ptr(), w.scales->data_ptr(), w.n, w.k,
                        static_cast<int32_t>(w.group), p.bias_at(), at_of(p.residual), p.rs, p.flags(), p.kind, out.data_ptr(), p.os,
                        need ? work.data_ptr() : nullptr, need, on.stream()));
    written({p.given});
    return wrap(out);
}

// ------------------------------------------------------------------ module
template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t wanted, F&& f) {
    if (n != wanted) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Invalid& e) {
        PyErr_SetString(g_invalid, e.what());
    } catch (const Failed& e) {
        PyErr_SetString(e.status == ITTS_EINVAL ? g_invalid : e.status == ITTS_ERUNTIME ? g_runtime : g_logic, itts_ops_last_error());
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&] { return rows_to_codes(a, true); });
}
PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&] { return rows_to_codes(a, false); });
}
PyObject* py_pack(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 2, [&] { return pack(a); });
}
PyObject* py_unpack(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&] { return unpack(a); });
}
PyObject* py_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] { return matmul(a); });
}
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&] { return linear(a); });
}
PyObject* py_errors(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&]() -> PyObject* {
        for (int i = 0; i < 3; ++i) Py_INCREF(a[i]);
        g_invalid = a[0];
        g_runtime = a[1];
        g_logic = a[2];
        Py_RETURN_NONE;
    });
}
#define ENTRY(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY("rmsnorm_q8", py_norm), ENTRY("q8_quantize", py_quantize), ENTRY("q4_pack", py_pack), ENTRY("q4_unpack", py_unpack),
                           ENTRY("q4_matmul", py_matmul), ENTRY("q4_linear", py_linear), ENTRY("errors", py_errors), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_itts_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__itts_ops() { return PyModule_Create(&g_module); }
