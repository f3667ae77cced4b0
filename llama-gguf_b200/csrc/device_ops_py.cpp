// device_ops_py.cpp — device_ops.py's calls in C++: argument checks on torch tensors, outputs and workspaces from torch's allocator, and the C entries (include/llama_b200.h).
//
// A decoding step makes dozens of these calls, each of a few microseconds on the device; the same checks in Python and a call through ctypes took 16 us of host time for one product, in C++
// they take the time of the allocation and the launch.  The C entries are handed in as addresses (bind), so that this module works with whichever libllama_b200.so the package has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/llama_b200.h"

namespace {

using at::Tensor;

struct Entries {
    decltype(&b200_last_error) last_error = nullptr;
    decltype(&b200_dev_add_rms_norm_q8) add_rms_norm_q8 = nullptr;
    decltype(&b200_dev_read_q8) read_q8 = nullptr;
    decltype(&b200_dev_mat_mat_i8) mat_mat_i8 = nullptr;
    decltype(&b200_dev_route_experts) route_experts = nullptr;
    decltype(&b200_dev_mat_mat_i4) mat_mat_i4 = nullptr;
    decltype(&b200_dev_glu_q8) glu_q8 = nullptr;
    decltype(&b200_dev_add_gated_norm_q8) add_gated_norm_q8 = nullptr;
    decltype(&b200_dev_rope_append_q4) rope_append_q4 = nullptr;
    decltype(&b200_dev_read_q4) read_q4 = nullptr;
    decltype(&b200_dev_attention_paged_q4_workspace) attention_workspace = nullptr;
    decltype(&b200_dev_attention_paged_q4) attention = nullptr;
} E;
PyObject* errors[16];      // the package's exception classes, by -status

struct Refused {
    int status;
    std::string text;
};
struct PythonError {};      // the interpreter has it already

[[noreturn]] void refuse(int status, const char* op, const std::string& text) { throw Refused{status, std::string(op) + ": " + text}; }
void check(int rc) {
    if (rc) throw Refused{rc, E.last_error()};
}

std::string sizes(const Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

// One call: its name, its device (that of the first tensor), and the checks of its arguments.
struct Call {
    const char* op;
    PyObject* const* args;
    at::Device device{at::kCPU};

    Call(const char* name, PyObject* const* a, Py_ssize_t n, Py_ssize_t want) : op(name), args(a) {
        if (n != want) {
            PyErr_Format(PyExc_TypeError, "%s: %zd arguments expected, got %zd", name, want, n);
            throw PythonError{};
        }
    }
    // argument i, or an undefined tensor for None
    Tensor maybe(int i, const char* name) const {
        if (args[i] == Py_None) return Tensor();
        if (!THPVariable_Check(args[i])) {
            PyErr_Format(PyExc_TypeError, "%s: %s: a torch tensor expected", op, name);
            throw PythonError{};
        }
        return THPVariable_Unpack(args[i]);
    }
    Tensor tensor(int i, const char* name) const {
        Tensor t = maybe(i, name);
        if (!t.defined()) refuse(B200_ERR_INVALID_ARGUMENT, op, std::string(name) + " is None");
        return t;
    }
    int64_t integer(int i) const {
        const int64_t v = PyLong_AsLongLong(args[i]);
        if (v == -1 && PyErr_Occurred()) throw PythonError{};
        return v;
    }
    double number(int i) const {
        const double v = PyFloat_AsDouble(args[i]);
        if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
        return v;
    }
    uint32_t type(at::ScalarType t) const {
        if (t == at::kFloat) return B200_TYPE_F32;
        if (t == at::kHalf) return B200_TYPE_F16;
        if (t == at::kBFloat16) return B200_TYPE_BF16;
        refuse(B200_ERR_UNSUPPORTED_DTYPE, op, std::string(c10::toString(t)) + " (float32, float16 and bfloat16 only)");
    }
    at::ScalarType dtype(int i) const {
        if (!THPDtype_Check(args[i])) {
            PyErr_Format(PyExc_TypeError, "%s: a torch.dtype expected", op);
            throw PythonError{};
        }
        return reinterpret_cast<THPDtype*>(args[i])->scalar_type;
    }
    void typed(const char* name, const Tensor& t, at::ScalarType want) const {
        if (t.scalar_type() != want) refuse(B200_ERR_DTYPE_MISMATCH, op, std::string(name) + ": expected " + c10::toString(want) + ", got " + c10::toString(t.scalar_type()));
    }
    void vector(const char* name, const Tensor& t, int64_t n, at::ScalarType want) const {
        typed(name, t, want);
        if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1)) refuse(B200_ERR_SHAPE_MISMATCH, op, std::string(name) + ": expected [" + std::to_string(n) + "] contiguous, got " + sizes(t));
    }
    void matrix(const char* name, const Tensor& t, int64_t rows, int64_t cols, at::ScalarType want) const {
        typed(name, t, want);
        if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || (cols > 1 && t.stride(1) != 1))
            refuse(B200_ERR_SHAPE_MISMATCH, op, std::string(name) + ": expected [" + std::to_string(rows) + ", " + std::to_string(cols) + "] with contiguous rows, got " + sizes(t));
    }
    void whole(const char* name, const Tensor& t, int64_t rows, int64_t cols, at::ScalarType want) const {
        typed(name, t, want);
        if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || !t.is_contiguous())
            refuse(B200_ERR_SHAPE_MISMATCH, op, std::string(name) + ": expected [" + std::to_string(rows) + ", " + std::to_string(cols) + "] contiguous, got " + sizes(t));
    }
    void heads(const char* name, const Tensor& t, int64_t tokens, int64_t n, int64_t hd, at::ScalarType want) const {      // n < 0: any number of heads
        typed(name, t, want);
        if (t.dim() != 3 || t.size(0) != tokens || (n >= 0 && t.size(1) != n) || t.size(2) != hd || t.stride(2) != 1)
            refuse(B200_ERR_SHAPE_MISMATCH, op,
                   std::string(name) + ": expected [" + std::to_string(tokens) + ", " + (n >= 0 ? std::to_string(n) : "heads") + ", " + std::to_string(hd) + "] with contiguous channels, got " + sizes(t));
    }
    bool flag(int i) const {
        const int v = PyObject_IsTrue(args[i]);
        if (v < 0) throw PythonError{};
        return v;
    }
    // argument i, one of `names`: its place there
    template <size_t N> int choice(int i, const char* name, const char* const (&names)[N]) const {
        if (!PyUnicode_Check(args[i])) {
            PyErr_Format(PyExc_TypeError, "%s: %s: a text expected", op, name);
            throw PythonError{};
        }
        std::string all;
        for (size_t k = 0; k < N; k++) {
            if (!PyUnicode_CompareWithASCIIString(args[i], names[k])) return (int)k;
            all += std::string(k ? ", " : "") + names[k];
        }
        refuse(B200_ERR_INVALID_ARGUMENT, op, std::string(name) + ": one of " + all + " expected");
    }
    b200_q4_pages pages(const Tensor& t, int64_t hd) const {
        typed("pages", t, at::kByte);
        if (hd < 1 || t.dim() != 3 || !t.is_contiguous() || t.size(2) % (hd + 8))
            refuse(B200_ERR_SHAPE_MISMATCH, op, "pages: expected [pages, kv heads, page_size * (" + std::to_string(hd) + " + 8)] contiguous, got " + sizes(t));
        const int64_t size = t.size(2) / (hd + 8);
        if (size > 1024 || t.size(1) > 1024 || hd > 1024) refuse(B200_ERR_SHAPE_MISMATCH, op, "pages: " + sizes(t));
        return b200_q4_pages{t.data_ptr(), t.size(0), (int32_t)size, (int32_t)t.size(1), (int32_t)hd};
    }
    // all on the first one's device, a CUDA device, and none that a gradient would have to come through
    template <typename... Ts> void together(const Tensor& first, const Ts&... rest) {
        device = first.device();
        const bool grad = c10::GradMode::is_enabled(), tangent = c10::AutogradState::get_tls_state().get_fw_grad_mode();
        auto one = [&](const Tensor& t) {
            if (!t.defined()) return;
            if (grad && t.requires_grad()) refuse(B200_ERR_UNSUPPORTED, op, "an argument requires a gradient, and results carry none (detach it)");
            if (tangent && t._fw_grad(0).defined()) refuse(B200_ERR_UNSUPPORTED, op, "an argument has a forward-mode tangent, and results carry none");
            if (t.is_neg()) refuse(B200_ERR_UNSUPPORTED, op, "an argument is a view that stands for its memory's negative (resolve_neg it)");
            if (t.device() != device) refuse(B200_ERR_INVALID_ARGUMENT, op, "an argument is on " + t.device().str() + ", expected " + device.str());
        };
        one(first);
        (one(rest), ...);
        if (!device.is_cuda()) refuse(B200_ERR_INVALID_ARGUMENT, op, "tensors on a CUDA device expected, got " + device.str());
    }
    int32_t* status(int i) const {
        Tensor t = maybe(i, "status");
        if (!t.defined()) return nullptr;
        if (t.scalar_type() != at::kInt || t.numel() != 1 || t.device() != device) refuse(B200_ERR_INVALID_ARGUMENT, op, "status: one int32 on " + device.str() + " expected");
        return t.data_ptr<int32_t>();
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
    // (past the dispatcher, which takes as long as the allocation: 0.9 us of a call's 6)
    Tensor empty(at::IntArrayRef size, at::ScalarType t) const { return at::detail::empty_cuda(size, t, device, std::nullopt); }
};
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// distance of rows in elements (torch gives any number where there is one row)
int64_t ld(const Tensor& t) { return !t.defined() ? 0 : t.size(0) > 1 ? t.stride(0) : t.size(1); }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
PyObject* give(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
PyObject* give(const Tensor& a, const Tensor& b) {
    PyObject* r = PyTuple_New(2);
    if (!r) throw PythonError{};
    PyTuple_SET_ITEM(r, 0, give(a));
    PyTuple_SET_ITEM(r, 1, give(b));
    return r;
}

PyObject* add_rms_norm_q8(PyObject* const* args, Py_ssize_t n) {
    Call c("add_rms_norm_q8", args, n, 7);
    const Tensor x = c.tensor(0, "x"), w = c.tensor(1, "weight"), res = c.maybe(3, "residual");
    Tensor sum = c.maybe(4, "sum_out"), q = c.maybe(5, "out"), s = c.maybe(6, "scales");
    const double eps = c.number(2);
    if (x.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "x: expected [rows, hidden], got " + sizes(x));
    const int64_t rows = x.size(0), hidden = x.size(1);
    const uint32_t t = c.type(x.scalar_type());
    c.matrix("x", x, rows, hidden, x.scalar_type());
    c.vector("weight", w, hidden, at::kFloat);
    if (res.defined()) c.matrix("residual", res, rows, hidden, x.scalar_type());
    else if (sum.defined()) refuse(B200_ERR_INVALID_ARGUMENT, c.op, "sum_out without a residual");
    if (sum.defined()) c.matrix("sum_out", sum, rows, hidden, x.scalar_type());
    if (q.defined()) c.matrix("out", q, rows, hidden, at::kChar);
    if (s.defined()) c.vector("scales", s, rows, at::kFloat);
    c.together(x, w, res, sum, q, s);
    int64_t ldq = up16(hidden);
    if (q.defined()) ldq = ld(q);
    if (!q.defined()) {
        q = c.empty({rows, ldq}, at::kChar);
        if (ldq != hidden) q = q.narrow(1, 0, hidden);
    }
    if (!s.defined()) s = c.empty({rows}, at::kFloat);
    if (res.defined() && !sum.defined()) sum = c.empty({rows, hidden}, x.scalar_type());
    check(E.add_rms_norm_q8(c.device.index(), c.stream(), t, ptr(x), ld(x), ptr(res), ld(res), ptr(sum), ld(sum), w.data_ptr<float>(), (float)eps, (int8_t*)ptr(q), ldq, (float*)ptr(s), rows,
                            hidden));
    PyObject* r = PyTuple_New(3);
    if (!r) throw PythonError{};
    PyTuple_SET_ITEM(r, 0, give(q));
    PyTuple_SET_ITEM(r, 1, give(s));
    PyTuple_SET_ITEM(r, 2, give(sum));
    return r;
}

PyObject* read_q8(PyObject* const* args, Py_ssize_t n) {
    Call c("read_q8", args, n, 3);
    const Tensor q = c.tensor(0, "q"), s = c.tensor(1, "scales");
    const at::ScalarType dt = c.dtype(2);
    const uint32_t t = c.type(dt);
    if (q.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "q: expected [rows, n], got " + sizes(q));
    c.matrix("q", q, q.size(0), q.size(1), at::kChar);
    c.vector("scales", s, q.size(0), at::kFloat);
    c.together(q, s);
    const Tensor out = c.empty({q.size(0), q.size(1)}, dt);
    check(E.read_q8(c.device.index(), c.stream(), t, (const int8_t*)ptr(q), ld(q), (const float*)ptr(s), ptr(out), q.size(1), q.size(0), q.size(1)));
    return give(out);
}

PyObject* mat_mat_i8(PyObject* const* args, Py_ssize_t n_args) {
    Call c("mat_mat_i8", args, n_args, 7);
    const Tensor a = c.tensor(0, "a"), as = c.tensor(1, "a_scales"), w = c.tensor(2, "w"), ws = c.tensor(3, "w_scales"), bias = c.maybe(4, "bias");
    Tensor out = c.maybe(6, "out");
    if (a.dim() != 2 || w.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "expected [t, k] and [n, k], got " + sizes(a) + " and " + sizes(w));
    const int64_t rows = a.size(0), k = a.size(1), n = w.size(0);
    const at::ScalarType dt = out.defined() ? out.scalar_type() : c.dtype(5);
    const uint32_t t = c.type(dt);
    if (out.defined()) c.matrix("out", out, rows, n, dt);
    c.matrix("a", a, rows, k, at::kChar);
    c.matrix("w", w, n, k, at::kChar);
    c.vector("a_scales", as, rows, at::kFloat);
    c.vector("w_scales", ws, n, at::kFloat);
    if (bias.defined()) c.vector("bias", bias, n, at::kFloat);
    c.together(a, w, as, ws, bias, out);
    if (!out.defined()) out = c.empty({rows, n}, dt);
    auto apart = [&](const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : up16(k); };      // (one row has no distance)
    check(E.mat_mat_i8(c.device.index(), c.stream(), t, (const int8_t*)ptr(a), apart(a), (const float*)ptr(as), (const int8_t*)ptr(w), apart(w), (const float*)ptr(ws), (const float*)ptr(bias),
                       ptr(out), ld(out), rows, k, n));
    return give(out);
}

PyObject* route_experts(PyObject* const* args, Py_ssize_t n) {
    Call c("route_experts", args, n, 10);
    const Tensor z = c.tensor(0, "logits"), corr = c.maybe(3, "correction");
    Tensor experts = c.maybe(8, "experts"), weights = c.maybe(9, "weights");
    if (z.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "logits: expected [tokens, experts], got " + sizes(z));
    const int64_t tokens = z.size(0), many = z.size(1), top = c.integer(1), groups = c.integer(4), top_groups = c.integer(5);
    static const char* const scores[] = {"softmax", "sigmoid"};
    b200_route a{};
    a.type = c.type(z.scalar_type());
    a.sigmoid = c.choice(2, "score", scores);
    a.renormalise = c.flag(6);
    a.scale = (float)c.number(7);
    if (many > 1024) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "1 to 1024 experts expected");
    if (top < 1 || top > 32 || groups < 1 || groups > 32 || top_groups < 1 || top_groups > 32) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "top, groups and top_groups must be from 1 to 32");
    c.matrix("logits", z, tokens, many, z.scalar_type());
    if (corr.defined()) c.vector("correction", corr, many, at::kFloat);
    if (experts.defined()) c.whole("experts", experts, tokens, top, at::kInt);
    if (weights.defined()) c.whole("weights", weights, tokens, top, at::kFloat);
    c.together(z, corr, experts, weights);
    if (!experts.defined()) experts = c.empty({tokens, top}, at::kInt);
    if (!weights.defined()) weights = c.empty({tokens, top}, at::kFloat);
    a.device = c.device.index();
    a.stream = c.stream();
    a.logits = ptr(z);
    a.ld = ld(z);
    a.tokens = tokens;
    a.n = (int32_t)many;
    a.top = (int32_t)top;
    a.groups = (int32_t)groups;
    a.top_groups = (int32_t)top_groups;
    a.correction = (const float*)ptr(corr);
    a.experts = (int32_t*)ptr(experts);
    a.weights = (float*)ptr(weights);
    check(E.route_experts(&a));
    return give(experts, weights);
}

PyObject* mat_mat_i4(PyObject* const* args, Py_ssize_t n_args) {
    Call c("mat_mat_i4", args, n_args, 10);
    const Tensor x = c.tensor(0, "a"), xs = c.tensor(1, "a_scales"), w = c.tensor(2, "w"), ws = c.tensor(3, "w_scales"), experts = c.maybe(5, "experts"), bias = c.maybe(6, "bias");
    Tensor out = c.maybe(8, "out");
    if (x.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "a: expected [rows, k], got " + sizes(x));
    const int64_t rows = x.size(0), k = x.size(1), lead = experts.defined() ? 1 : 0;
    b200_i4_product a{};
    a.scale_type = c.type(ws.scalar_type());
    const at::ScalarType dt = out.defined() ? out.scalar_type() : c.dtype(7);
    a.out_type = c.type(dt);
    c.typed("w", w, at::kByte);
    if (w.dim() != 3 + lead || !w.is_contiguous() || w.size(lead + 2) != 512 || w.size(lead + 1) != (k + 63) / 64 || w.size(lead) < 1)
        refuse(B200_ERR_SHAPE_MISMATCH, c.op, std::string("w: expected ") + (lead ? "[experts, " : "[") + "row tiles, " + std::to_string((k + 63) / 64) + ", 512] contiguous, got " + sizes(w));
    const int64_t tiles = w.size(lead), n = args[4] == Py_None ? tiles * 16 : c.integer(4);
    if (n < 1 || (n + 15) / 16 != tiles) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "n: " + std::to_string(n) + " rows are not " + std::to_string(tiles) + " tiles of 16");
    if (ws.dim() != 4 + lead || !ws.is_contiguous() || (lead && ws.size(0) != w.size(0)) || ws.size(lead) != tiles || ws.size(lead + 1) < 1 || ws.size(lead + 2) != 8 || ws.size(lead + 3) != 2 ||
        k % ws.size(lead + 1))
        refuse(B200_ERR_SHAPE_MISMATCH, c.op, std::string("w_scales: expected ") + (lead ? "[experts, " : "[") + std::to_string(tiles) + ", groups, 8, 2] contiguous, got " + sizes(ws));
    const int64_t group = k / ws.size(lead + 1);
    if (group != 32 && group != 64 && group != 128) refuse(B200_ERR_UNSUPPORTED, c.op, "groups of " + std::to_string(group) + " channels (32, 64 and 128 only)");
    c.matrix("a", x, rows, k, at::kChar);
    c.vector("a_scales", xs, rows, at::kFloat);
    int64_t tokens = rows, many = rows;
    if (lead) {
        c.typed("experts", experts, at::kInt);
        if (experts.dim() != 2 || !experts.is_contiguous() || experts.size(1) < 1) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "experts: expected [tokens, top] contiguous, got " + sizes(experts));
        tokens = experts.size(0);
        many = experts.numel();
        if (rows != tokens && rows != many) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "a has " + std::to_string(rows) + " rows for " + std::to_string(tokens) + " tokens of " + std::to_string(experts.size(1)) + " experts");
        if (experts.size(1) > 32 || w.size(0) > 1024) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "1 to 32 places of 1 to 1024 experts expected");
    }
    if (bias.defined()) {
        if (lead) c.whole("bias", bias, w.size(0), n, at::kFloat);
        else c.vector("bias", bias, n, at::kFloat);
    }
    if (out.defined()) c.matrix("out", out, many, n, dt);
    c.together(x, xs, w, ws, experts, bias, out);
    if (!out.defined()) out = c.empty({many, n}, dt);
    a.device = c.device.index();
    a.stream = c.stream();
    a.group = (int32_t)group;
    a.a = (const int8_t*)ptr(x);
    a.lda = rows > 1 ? x.stride(0) : up16(k);      // (one row has no distance)
    a.a_scales = (const float*)ptr(xs);
    a.w = ptr(w);
    a.w_scales = ptr(ws);
    a.bias = (const float*)ptr(bias);
    a.out = ptr(out);
    a.ldo = ld(out);
    a.tokens = tokens;
    a.k = k;
    a.n = n;
    if (lead) {
        a.experts = (const int32_t*)ptr(experts);
        a.top = (int32_t)experts.size(1);
        a.n_experts = (int32_t)w.size(0);
        a.rows_per_pair = rows != tokens;
    }
    a.status = c.status(9);
    check(E.mat_mat_i4(&a));
    return give(out);
}

PyObject* glu_q8(PyObject* const* args, Py_ssize_t n) {
    Call c("glu_q8", args, n, 4);
    const Tensor x = c.tensor(0, "x");
    Tensor q = c.maybe(2, "out"), s = c.maybe(3, "scales");
    if (x.dim() != 2 || x.size(1) % 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "x: expected [rows, 2 ff], got " + sizes(x));
    const int64_t rows = x.size(0), ff = x.size(1) / 2;
    const uint32_t t = c.type(x.scalar_type());
    static const char* const acts[] = {"silu", "gelu", "relu"};
    const int act = c.choice(1, "act", acts);
    c.matrix("x", x, rows, 2 * ff, x.scalar_type());
    if (q.defined()) c.matrix("out", q, rows, ff, at::kChar);
    if (s.defined()) c.vector("scales", s, rows, at::kFloat);
    c.together(x, q, s);
    int64_t ldq = up16(ff);
    if (q.defined()) ldq = ld(q);
    if (!q.defined()) {
        q = c.empty({rows, ldq}, at::kChar);
        if (ldq != ff) q = q.narrow(1, 0, ff);
    }
    if (!s.defined()) s = c.empty({rows}, at::kFloat);
    check(E.glu_q8(c.device.index(), c.stream(), t, act, ptr(x), ld(x), (int8_t*)ptr(q), ldq, (float*)ptr(s), rows, ff));
    return give(q, s);
}

PyObject* add_gated_norm_q8(PyObject* const* args, Py_ssize_t n) {
    Call c("add_gated_norm_q8", args, n, 11);
    const Tensor y = c.tensor(0, "y"), res = c.tensor(1, "residual"), w = c.maybe(2, "weight"), mix = c.maybe(4, "mix"), post = c.maybe(5, "post_weight"), gate = c.maybe(6, "gate");
    Tensor sum = c.maybe(8, "sum_out"), q = c.maybe(9, "out"), s = c.maybe(10, "scales");
    const double eps = c.number(3), scale = c.number(7);
    if (res.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "residual: expected [rows, hidden], got " + sizes(res));
    const int64_t rows = res.size(0), hidden = res.size(1);
    const at::ScalarType dt = res.scalar_type();
    b200_gated_norm a{};
    a.type = c.type(dt);
    int64_t top = 1;
    if (mix.defined()) {
        if (mix.dim() != 2 || mix.size(1) < 1 || mix.size(1) > 32) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "mix: expected [rows, 1 to 32], got " + sizes(mix));
        top = mix.size(1);
        c.whole("mix", mix, rows, top, at::kFloat);
    }
    c.matrix("residual", res, rows, hidden, dt);
    c.matrix("y", y, rows * top, hidden, dt);
    if (post.defined()) c.vector("post_weight", post, hidden, at::kFloat);
    if (w.defined()) c.vector("weight", w, hidden, at::kFloat);
    else if (q.defined() || s.defined()) refuse(B200_ERR_INVALID_ARGUMENT, c.op, "out or scales without a weight");
    if (gate.defined()) {
        c.typed("gate", gate, dt);
        if (gate.dim() != 2 || (gate.size(0) != rows && gate.size(0) != 1) || (gate.size(1) != hidden && gate.size(1) != 1))
            refuse(B200_ERR_SHAPE_MISMATCH, c.op, "gate: expected [rows or 1, hidden or 1], got " + sizes(gate));
    }
    if (sum.defined()) c.matrix("sum_out", sum, rows, hidden, dt);
    if (q.defined()) c.matrix("out", q, rows, hidden, at::kChar);
    if (s.defined()) c.vector("scales", s, rows, at::kFloat);
    c.together(res, y, w, mix, post, gate, sum, q, s);
    int64_t ldq = up16(hidden);
    if (q.defined()) ldq = ld(q);
    if (w.defined() && !q.defined()) {
        q = c.empty({rows, ldq}, at::kChar);
        if (ldq != hidden) q = q.narrow(1, 0, hidden);
    }
    if (w.defined() && !s.defined()) s = c.empty({rows}, at::kFloat);
    if (!sum.defined()) sum = c.empty({rows, hidden}, dt);
    a.device = c.device.index();
    a.stream = c.stream();
    a.y = ptr(y);
    a.ldy = ld(y);
    a.mix = (const float*)ptr(mix);
    a.top = (int32_t)top;
    a.post_weight = (const float*)ptr(post);
    if (gate.defined()) {
        a.gate = ptr(gate);
        a.gate_row = gate.size(0) > 1 ? gate.stride(0) : 0;
        a.gate_col = gate.size(1) > 1 ? gate.stride(1) : 0;
    }
    a.residual = ptr(res);
    a.ldr = ld(res);
    a.sum = ptr(sum);
    a.lds = ld(sum);
    a.weight = (const float*)ptr(w);
    a.q = (int8_t*)ptr(q);
    a.ldq = ldq;
    a.scales = (float*)ptr(s);
    a.rows = rows;
    a.hidden = hidden;
    a.scale = (float)scale;
    a.eps = (float)eps;
    check(E.add_gated_norm_q8(&a));
    PyObject* r = PyTuple_New(3);
    if (!r) throw PythonError{};
    PyTuple_SET_ITEM(r, 0, give(q));
    PyTuple_SET_ITEM(r, 1, give(s));
    PyTuple_SET_ITEM(r, 2, give(sum));
    return r;
}

PyObject* rope_append_q4(PyObject* const* args, Py_ssize_t n) {
    Call c("rope_append_q4", args, n, 10);
    const Tensor q = c.maybe(0, "q"), k = c.tensor(1, "k"), v = c.tensor(2, "v"), table = c.tensor(3, "cos_sin"), pos = c.tensor(4, "positions"), pages = c.tensor(5, "pages"), slots = c.tensor(6, "slots");
    Tensor out = c.maybe(8, "q_out");
    if (k.dim() != 3) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "k: expected [tokens, kv heads, head_dim], got " + sizes(k));
    const int64_t tokens = k.size(0), nkv = k.size(1), hd = k.size(2);
    const at::ScalarType dt = k.scalar_type();
    b200_q4_append a{};
    a.type = c.type(dt);
    a.cache = c.pages(pages, hd);
    if (nkv != a.cache.n_kv_heads) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "k has " + std::to_string(nkv) + " heads, the cache " + std::to_string(a.cache.n_kv_heads));
    c.heads("k", k, tokens, nkv, hd, dt);
    c.heads("v", v, tokens, nkv, hd, dt);
    if (q.defined()) {
        c.heads("q", q, tokens, -1, hd, dt);
        if (q.size(1) > 65536) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "bad number of query heads");
        if (out.defined()) c.heads("q_out", out, tokens, q.size(1), hd, dt);
    } else if (out.defined()) {
        refuse(B200_ERR_INVALID_ARGUMENT, c.op, "q_out without q");
    }
    c.typed("cos_sin", table, at::kFloat);
    if (table.dim() != 2 || !table.is_contiguous() || table.size(1) > 1024) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "cos_sin: expected [positions, rot dims] contiguous, got " + sizes(table));
    c.vector("positions", pos, tokens, at::kInt);
    c.vector("slots", slots, tokens, at::kLong);
    c.together(k, q, v, table, pos, pages, slots, out);
    if (q.defined() && !out.defined()) out = c.empty({tokens, q.size(1), hd}, dt);
    a.device = c.device.index();
    a.stream = c.stream();
    a.q = ptr(q);
    a.k = ptr(k);
    a.v = ptr(v);
    a.q_out = ptr(out);
    if (q.defined()) {
        a.q_token = q.stride(0);
        a.q_head = q.stride(1);
        a.q_out_token = out.stride(0);
        a.q_out_head = out.stride(1);
        a.n_heads = (int32_t)q.size(1);
    }
    a.k_token = k.stride(0);
    a.k_head = k.stride(1);
    a.v_token = v.stride(0);
    a.v_head = v.stride(1);
    a.cos_sin = (const float*)ptr(table);
    a.table_rows = table.size(0);
    a.positions = (const int32_t*)ptr(pos);
    a.slots = (const int64_t*)ptr(slots);
    a.tokens = tokens;
    a.rot_dims = (int32_t)table.size(1);
    a.use_neox = c.flag(7);
    a.status = c.status(9);
    check(E.rope_append_q4(&a));
    return give(out);
}

PyObject* read_q4(PyObject* const* args, Py_ssize_t n) {
    Call c("read_q4", args, n, 5);
    const Tensor pages = c.tensor(0, "pages"), slots = c.tensor(1, "slots");
    const int64_t hd = c.integer(2);
    const at::ScalarType dt = c.dtype(3);
    const uint32_t t = c.type(dt);
    const b200_q4_pages p = c.pages(pages, hd);
    c.vector("slots", slots, slots.numel(), at::kLong);
    c.together(pages, slots);
    const int64_t tokens = slots.numel();
    const Tensor k = c.empty({tokens, p.n_kv_heads, hd}, dt), v = c.empty({tokens, p.n_kv_heads, hd}, dt);
    check(E.read_q4(c.device.index(), c.stream(), t, &p, (const int64_t*)ptr(slots), tokens, ptr(k), ptr(v), c.status(4)));
    return give(k, v);
}

PyObject* attention_paged_q4(PyObject* const* args, Py_ssize_t n) {
    Call c("attention_paged_q4", args, n, 10);
    const Tensor q = c.tensor(0, "q"), pages = c.tensor(1, "pages"), table = c.tensor(2, "page_table"), lens = c.tensor(3, "kv_lens"), starts = c.maybe(5, "q_starts");
    Tensor out = c.maybe(8, "out");
    if (q.dim() != 3) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "q: expected [tokens, heads, head_dim], got " + sizes(q));
    const int64_t tokens = q.size(0), nh = q.size(1), hd = q.size(2);
    const at::ScalarType dt = q.scalar_type();
    b200_q4_attention a{};
    a.type = c.type(dt);
    a.cache = c.pages(pages, hd);
    c.heads("q", q, tokens, nh, hd, dt);
    if (table.dim() != 2) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "page_table: expected [sequences, pages], got " + sizes(table));
    const int64_t seqs = table.size(0), width = table.size(1);
    c.matrix("page_table", table, seqs, width, at::kInt);
    c.vector("kv_lens", lens, seqs, at::kInt);
    if (starts.defined()) c.vector("q_starts", starts, seqs + 1, at::kInt);
    if (out.defined()) c.heads("out", out, tokens, nh, hd, dt);
    const double scale = args[4] == Py_None ? 1.0 / std::sqrt((double)hd) : c.number(4);
    if (!std::isfinite((float)scale)) refuse(B200_ERR_INVALID_ARGUMENT, c.op, "scale is not finite");
    const int64_t max_q = c.integer(6), window = c.integer(7);
    if (seqs >= INT32_MAX || width >= INT32_MAX || nh > 65536) refuse(B200_ERR_SHAPE_MISMATCH, c.op, "too many sequences, pages or heads");
    if (max_q < 0 || max_q > INT32_MAX || window < 0 || window > INT32_MAX) refuse(B200_ERR_INVALID_ARGUMENT, c.op, "max_q and window must be from 0 to 2^31 - 1");
    c.together(q, pages, table, lens, starts, out);
    if (!out.defined()) out = c.empty({tokens, nh, hd}, dt);
    a.device = c.device.index();
    a.stream = c.stream();
    a.q = ptr(q);
    a.out = ptr(out);
    a.q_token = q.stride(0);
    a.q_head = q.stride(1);
    a.out_token = out.stride(0);
    a.out_head = out.stride(1);
    a.q_starts = (const int32_t*)ptr(starts);
    a.kv_lens = (const int32_t*)ptr(lens);
    a.page_table = (const int32_t*)ptr(table);
    a.table_stride = seqs > 1 ? table.stride(0) : width;
    a.tokens = tokens;
    a.table_pages = (int32_t)width;
    a.seqs = (int32_t)seqs;
    a.max_q = (int32_t)max_q;
    a.n_heads = (int32_t)nh;
    a.window = (int32_t)window;
    a.scale = (float)scale;
    a.status = c.status(9);
    size_t need = 0;
    check(E.attention_workspace(&a, &need));
    Tensor work;      // (back to the allocator on return: it hands it out again in the order of this stream)
    if (need) {
        work = c.empty({(int64_t)need}, at::kByte);
        a.workspace = ptr(work);
        a.workspace_bytes = need;
    }
    check(E.attention(&a));
    return give(out);
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)> PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        return F(args, n);
    } catch (const Refused& r) {
        PyObject* cls = r.status < 0 && r.status > -16 && errors[-r.status] ? errors[-r.status] : PyExc_RuntimeError;
        PyErr_SetString(cls, r.text.c_str());
    } catch (const PythonError&) {
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(errors[-B200_ERR_ALLOCATION_FAILED], e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// bind({-status: exception class}, {name: address of the C entry})
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *classes, *entries;
    if (!PyArg_ParseTuple(args, "O!O!", &PyDict_Type, &classes, &PyDict_Type, &entries)) return nullptr;
    PyObject *key, *value;
    for (Py_ssize_t at = 0; PyDict_Next(classes, &at, &key, &value);) {
        const long i = -PyLong_AsLong(key);
        if (i > 0 && i < 16) {
            Py_INCREF(value);
            errors[i] = value;
        }
    }
    auto take = [&](const char* name, auto& to) {
        PyObject* v = PyDict_GetItemString(entries, name);
        if (!v) {
            PyErr_SetString(PyExc_KeyError, name);
            return false;
        }
        to = reinterpret_cast<std::decay_t<decltype(to)>>(PyLong_AsVoidPtr(v));
        return to != nullptr;
    };
    if (!take("b200_last_error", E.last_error) || !take("b200_dev_add_rms_norm_q8", E.add_rms_norm_q8) || !take("b200_dev_read_q8", E.read_q8) || !take("b200_dev_mat_mat_i8", E.mat_mat_i8) ||
        !take("b200_dev_route_experts", E.route_experts) || !take("b200_dev_mat_mat_i4", E.mat_mat_i4) || !take("b200_dev_glu_q8", E.glu_q8) ||
        !take("b200_dev_add_gated_norm_q8", E.add_gated_norm_q8) || !take("b200_dev_rope_append_q4", E.rope_append_q4) || !take("b200_dev_read_q4", E.read_q4) || !take("b200_dev_attention_paged_q4_workspace", E.attention_workspace) ||
        !take("b200_dev_attention_paged_q4", E.attention)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
        return nullptr;
    }
    Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(add_rms_norm_q8), FAST(read_q8), FAST(mat_mat_i8), FAST(route_experts), FAST(mat_mat_i4), FAST(glu_q8), FAST(add_gated_norm_q8),
                         FAST(rope_append_q4), FAST(read_q4), FAST(attention_paged_q4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_device_ops", "device_ops.py's calls", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__device_ops() { return PyModule_Create(&module); }
