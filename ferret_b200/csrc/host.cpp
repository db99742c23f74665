// host.cpp -- the host side of the operators around the expert GEMMs (the module
// ferret_b200._host that ops.py calls): checks of the tensors, allocation of the
// outputs, the C-ABI call on the tensors' device and its current stream.
//
// A single-token call of these operators runs 3-10 us on the GPU, and in Python
// the checks, the allocations and the ctypes call took 12-20 us (4-5 outputs at
// 2-3 us each, the call itself 5 us, of which the launch is 3.4): the host was what
// bounded small calls.  Here the same steps take 4.7 us (two outputs) to 6 us (four).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <initializer_list>

#include "../../include/ferret_moe.h"

namespace {

PyObject* g_check = nullptr;      // _lib.check(rc, name): raises for rc != 0
PyObject* g_no_backward = nullptr;   // ops._no_backward(name, outs, given, *inputs)

[[noreturn]] void fail(PyObject* type, const char* format, ...) {
    va_list v;
    va_start(v, format);
    PyErr_FormatV(type, format, v);
    va_end(v);
    throw python_error();
}

bool none(PyObject* o) { return o == Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, "%s must be a tensor", name);
    return THPVariable_Unpack(o);
}

const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
    const at::Tensor& t = tensor(o, name);
    if (!t.is_cuda()) fail(PyExc_ValueError, "%s must be a CUDA tensor", name);
    return t;
}

long integer(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v > INT_MAX || v < INT_MIN) fail(PyExc_ValueError, "integer argument out of range");
    return v;
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

int dtype_code(const at::Tensor& t, const char* name, bool fp32 = true) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return FERRET_BF16;
        case at::kHalf: return FERRET_FP16;
        case at::kFloat:
            if (fp32) return FERRET_FP32;
            [[fallthrough]];
        default:
            fail(PyExc_TypeError, "%s must be bf16%s, got %s", name,
                 fp32 ? ", fp16 or fp32" : " or fp16", c10::toString(t.scalar_type()));
    }
}

// Address of a contiguous tensor of that device, type and shape.
void* like(const at::Tensor& t, const char* name, const at::Tensor& ref, at::ScalarType dtype,
           std::initializer_list<int64_t> shape) {
    if (t.device() != ref.device())
        fail(PyExc_ValueError, "%s must be on the device of the first argument", name);
    if (t.scalar_type() != dtype)
        fail(PyExc_TypeError, "%s must be %s, got %s", name, c10::toString(dtype),
             c10::toString(t.scalar_type()));
    if (t.sizes() != at::IntArrayRef(shape))
        fail(PyExc_ValueError, "%s has the wrong shape: %zd dimensions, first %lld, expected %zu, %lld",
             name, (Py_ssize_t)t.dim(), t.dim() ? (long long)t.size(0) : 0LL, shape.size(),
             shape.size() ? (long long)*shape.begin() : 0LL);
    if (!t.is_contiguous()) fail(PyExc_ValueError, "%s must be contiguous", name);
    return t.data_ptr();
}

void* like(PyObject* o, const char* name, const at::Tensor& ref, at::ScalarType dtype,
           std::initializer_list<int64_t> shape) {
    return none(o) ? nullptr : like(tensor(o, name), name, ref, dtype, shape);
}

// Row stride of a matrix whose rows are contiguous and do not overlap.
long long row_stride(const at::Tensor& t, const char* name) {
    if (t.dim() != 2) fail(PyExc_ValueError, "%s must be 2-D, got %lld-D", name, (long long)t.dim());
    const int64_t T = t.size(0), K = t.size(1);
    if (T > INT_MAX || K > INT_MAX) fail(PyExc_ValueError, "%s is too large", name);
    if ((t.stride(1) != 1 && K > 1) || (t.stride(0) < K && T > 1))
        fail(PyExc_ValueError, "%s must have contiguous rows that do not overlap", name);
    return T > 1 ? t.stride(0) : K;
}

// Whether `out`, contiguous, shares bytes with the rows of `in` (1-D or 2-D, contiguous rows).
bool overlap(const at::Tensor& out, const at::Tensor& in) {
    if (out.numel() == 0 || in.numel() == 0) return false;
    auto at = [](const at::Tensor& t) { return (int64_t) reinterpret_cast<uintptr_t>(t.data_ptr()); };
    const int64_t lo = at(out), hi = lo + (int64_t)out.nbytes();
    const int64_t size = (int64_t)in.element_size(), first = at(in);
    const int64_t rows = in.dim() == 2 ? in.size(0) : 1, len = in.size(in.dim() - 1) * size;
    if (rows == 1) return first < hi && first + len > lo;
    const int64_t step = in.stride(0) * size;              // at least len
    const int64_t i = first + len > lo ? 0 : (lo - first - len) / step + 1;   // ends behind lo
    return i < rows && first + i * step < hi;
}

// A tensor that the caller passed in to be written: what an operation in place of torch's
// checks, and (written) the new version that autograd sees of it.
void writable(const at::Tensor& t, const char* name) {
    if (at::GradMode::is_enabled() && t.requires_grad() &&
        (t.is_leaf() || (t.is_view() && t._base().is_leaf())))
        fail(PyExc_RuntimeError, "%s is a leaf that requires a gradient (or a view of one) and cannot "
                                 "be written in place", name);
}
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor make(std::initializer_list<int64_t> shape, at::ScalarType dtype, const at::Tensor& ref) {
    for (int64_t n : shape)
        if (n < 0) fail(PyExc_ValueError, "negative size");
    return at::detail::empty_cuda(at::IntArrayRef(shape), dtype, ref.device(), c10::nullopt);
}

// The device of `t` for the time of a call, and its current stream.
struct On {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit On(const at::Tensor& t)
        : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

void check(int rc, const char* name) {
    if (rc == FERRET_OK) return;
    PyObject* r = PyObject_CallFunction(g_check, "is", rc, name);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", name, rc);
    throw python_error();
}

PyObject* wrap(const at::Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}

PyObject* tuple(std::initializer_list<at::Tensor> ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    if (!r) throw python_error();
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) PyTuple_SET_ITEM(r, i++, wrap(t));
    return r;
}

void expect(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) fail(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
}

// `outs` (stolen) of an operator without a backward pass, as it is returned: where
// autograd records and a tensor of `inputs` requires a gradient, tied to them, so that
// a gradient raises and is not lost.  given: the output that the caller passed in.
PyObject* no_backward(const char* name, PyObject* outs, PyObject* given,
                      std::initializer_list<PyObject*> inputs) {
    bool any = false;
    if (at::GradMode::is_enabled())
        for (PyObject* o : inputs) any = any || (!none(o) && THPVariable_Unpack(o).requires_grad());
    if (!any) return outs;
    PyObject* args = PyTuple_New((Py_ssize_t)(3 + inputs.size()));
    PyObject* label = args ? PyUnicode_FromString(name) : nullptr;
    if (!label) {
        Py_XDECREF(args);
        Py_DECREF(outs);
        throw python_error();
    }
    PyTuple_SET_ITEM(args, 0, label);
    PyTuple_SET_ITEM(args, 1, outs);
    Py_INCREF(given);
    PyTuple_SET_ITEM(args, 2, given);
    Py_ssize_t i = 3;
    for (PyObject* o : inputs) {
        Py_INCREF(o);
        PyTuple_SET_ITEM(args, i++, o);
    }
    PyObject* r = PyObject_CallObject(g_no_backward, args);
    Py_DECREF(args);
    if (!r) throw python_error();
    return r;
}

int scoring_flags(PyObject* scoring, bool renorm) {
    int flags = renorm ? FERRET_ROUTE_RENORM : 0;
    if (PyUnicode_Check(scoring)) {
        if (PyUnicode_CompareWithASCIIString(scoring, "sigmoid") == 0)
            return flags | FERRET_ROUTE_SIGMOID;
        if (PyUnicode_CompareWithASCIIString(scoring, "softmax") == 0) return flags;
    }
    fail(PyExc_ValueError, "scoring must be 'softmax' or 'sigmoid', got %R", scoring);
}

// x, weight, residual, eps, quant, use_ue8m0, normed, residual_out
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 8);
    const at::Tensor& x = cuda_tensor(a[0], "x");
    const int dt = dtype_code(x, "x");
    const long long ldx = row_stride(x, "x");
    const int64_t T = x.size(0), K = x.size(1);
    const at::Tensor& weight = tensor(a[1], "weight");
    const at::ScalarType wt = weight.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type();
    void* wp = like(weight, "weight", x, wt, {K});
    const bool quant = truth(a[4]), normed = truth(a[6]);
    long long ldr = 0;
    void* rp = nullptr;
    at::Tensor residual_out, y, q, s;
    if (!none(a[2])) {
        const at::Tensor& r = tensor(a[2], "residual");
        if (r.device() != x.device() || r.scalar_type() != x.scalar_type() || r.sizes() != x.sizes())
            fail(PyExc_ValueError, "residual must have the device, type and shape of x");
        ldr = row_stride(r, "residual");
        rp = r.data_ptr();
        residual_out = none(a[7]) ? make({T, K}, x.scalar_type(), x) : tensor(a[7], "residual_out");
        like(residual_out, "residual_out", x, x.scalar_type(), {T, K});
        if (!none(a[7])) {
            // a row is read before it is written: the same rows may be one memory, no others
            auto same = [&](const at::Tensor& t, long long ld) {
                return t.data_ptr() == residual_out.data_ptr() && ld == K;
            };
            if ((overlap(residual_out, x) && !same(x, ldx)) ||
                (overlap(residual_out, r) && !same(r, ldr)) || overlap(residual_out, weight))
                fail(PyExc_ValueError, "residual_out may be x or residual; it must not overlap an "
                                       "input in another way");
            writable(residual_out, "residual_out");
        }
    } else if (!none(a[7])) {
        fail(PyExc_ValueError, "residual_out needs a residual");
    }
    if (quant && K % 128) fail(PyExc_ValueError, "K must be a multiple of 128 for FP8 rows");
    if (!quant && !normed) fail(PyExc_ValueError, "nothing to compute: normed and quant are both off");
    if (normed) y = make({T, K}, x.scalar_type(), x);
    if (quant) {
        q = make({T, K}, at::kFloat8_e4m3fn, x);
        s = make({T, K / 128}, at::kFloat, x);
    }
    On on(x);
    check(ferret_add_rms_norm(x.data_ptr(), ldx, rp, ldr, wp, wt == at::kFloat ? FERRET_FP32 : dt, dt,
                              (int)T, (int)K, (float)number(a[3]), normed ? y.data_ptr() : nullptr,
                              rp ? residual_out.data_ptr() : nullptr, quant ? q.data_ptr() : nullptr,
                              quant ? s.data_ptr<float>() : nullptr,
                              truth(a[5]) ? FERRET_UE8M0_SCALES : 0, on.stream),
          "ferret_add_rms_norm");
    if (!none(a[7])) written(residual_out);
    return no_backward("ops.add_rms_norm", tuple({y, residual_out, q, s}), a[7],
                       {a[0], a[1], a[2], a[7]});
    END_HANDLE_TH_ERRORS
}

struct Logits {
    const at::Tensor& t;
    int dtype;
    long long ld;
    int64_t T, E;
    explicit Logits(PyObject* o) : t(cuda_tensor(o, "logits")) {
        dtype = dtype_code(t, "logits");
        ld = row_stride(t, "logits");
        T = t.size(0);
        E = t.size(1);
    }
};

// logits, topk, scoring, bias, n_group, topk_group, group_top, renormalize, scale, token_mask
PyObject* moe_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    const Logits z(a[0]);
    const int topk = (int)integer(a[1]);
    const int flags = scoring_flags(a[2], truth(a[7]));
    void* bias = like(a[3], "bias", z.t, at::kFloat, {z.E});
    void* mask = like(a[9], "token_mask", z.t, at::kBool, {z.T});
    at::Tensor w = make({z.T, topk}, at::kFloat, z.t), ids = make({z.T, topk}, at::kInt, z.t);
    On on(z.t);
    check(ferret_moe_route(z.t.data_ptr(), z.ld, z.dtype, (const float*)bias, (const uint8_t*)mask,
                           (int)z.T, (int)z.E, topk, (int)integer(a[4]), (int)integer(a[5]),
                           (int)integer(a[6]), (float)number(a[8]), flags, w.data_ptr<float>(),
                           ids.data_ptr<int32_t>(), on.stream),
          "ferret_moe_route");
    return tuple({w, ids});
    END_HANDLE_TH_ERRORS
}

// grad_weights, logits, ids, scoring, renormalize, scale
PyObject* moe_route_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6);
    const Logits z(a[1]);
    const int flags = scoring_flags(a[3], truth(a[4]));
    const at::Tensor& ids = tensor(a[2], "ids");
    if (ids.dim() != 2) fail(PyExc_ValueError, "ids must be 2-D, got %lld-D", (long long)ids.dim());
    const int64_t topk = ids.size(1);
    void* ip = like(ids, "ids", z.t, at::kInt, {z.T, topk});
    void* gp = like(tensor(a[0], "grad_weights"), "grad_weights", z.t, at::kFloat, {z.T, topk});
    at::Tensor out = make({z.T, z.E}, z.t.scalar_type(), z.t);
    On on(z.t);
    check(ferret_moe_route_backward((const float*)gp, z.t.data_ptr(), z.ld, z.dtype,
                                    (const int32_t*)ip, (int)z.T, (int)z.E, (int)topk,
                                    (float)number(a[5]), flags, out.data_ptr(), on.stream),
          "ferret_moe_route_backward");
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// logits, topk_ids, coef, scoring, token_mask
PyObject* moe_balance_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5);
    const Logits z(a[0]);
    const int flags = scoring_flags(a[3], false);
    const at::Tensor& ids = tensor(a[1], "topk_ids");
    if (ids.dim() != 2)
        fail(PyExc_ValueError, "topk_ids must be 2-D, got %lld-D", (long long)ids.dim());
    const int64_t topk = ids.size(1);
    void* ip = like(ids, "topk_ids", z.t, at::kInt, {z.T, topk});
    void* mask = like(a[4], "token_mask", z.t, at::kBool, {z.T});
    at::Tensor loss = make({}, at::kFloat, z.t), counts = make({z.E}, at::kInt, z.t),
               sums = make({z.E}, at::kFloat, z.t), live = make({1}, at::kInt, z.t);
    const size_t bytes = ferret_moe_balance_loss_workspace_size((int)z.T, (int)z.E);
    at::Tensor ws = make({(int64_t)bytes}, at::kByte, z.t);
    On on(z.t);
    check(ferret_moe_balance_loss(z.t.data_ptr(), z.ld, z.dtype, (const int32_t*)ip,
                                  (const uint8_t*)mask, (int)z.T, (int)z.E, (int)topk,
                                  (float)number(a[2]), flags, loss.data_ptr<float>(),
                                  counts.data_ptr<int32_t>(), sums.data_ptr<float>(),
                                  live.data_ptr<int32_t>(), ws.data_ptr(), bytes, on.stream),
          "ferret_moe_balance_loss");
    return tuple({loss, counts, sums, live});
    END_HANDLE_TH_ERRORS
}

// grad_loss, logits, counts, n_tokens, topk, coef, scoring, token_mask
PyObject* moe_balance_loss_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 8);
    const Logits z(a[1]);
    const int flags = scoring_flags(a[6], false);
    void* gp = like(tensor(a[0], "grad_loss"), "grad_loss", z.t, at::kFloat, {});
    void* cp = like(tensor(a[2], "counts"), "counts", z.t, at::kInt, {z.E});
    void* np = like(tensor(a[3], "n_tokens"), "n_tokens", z.t, at::kInt, {1});
    void* mask = like(a[7], "token_mask", z.t, at::kBool, {z.T});
    at::Tensor out = make({z.T, z.E}, z.t.scalar_type(), z.t);
    On on(z.t);
    check(ferret_moe_balance_loss_backward((const float*)gp, z.t.data_ptr(), z.ld, z.dtype,
                                           (const int32_t*)cp, (const int32_t*)np,
                                           (const uint8_t*)mask, (int)z.T, (int)z.E,
                                           (int)integer(a[4]), (float)number(a[5]), flags,
                                           out.data_ptr(), on.stream),
          "ferret_moe_balance_loss_backward");
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// x, w, w_scale, w_zero, bias, out
PyObject* int4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6);
    const at::Tensor& x = cuda_tensor(a[0], "x");
    const int dt = dtype_code(x, "x", false);
    const long long ldx = row_stride(x, "x");
    const int64_t T = x.size(0), K = x.size(1);
    const at::Tensor &w = tensor(a[1], "w"), &scale = tensor(a[2], "w_scale");
    if (w.dim() != 2 || scale.dim() != 2 || w.size(0) * 8 != K)
        fail(PyExc_ValueError, "w must be [K/8, N] with K = %lld, w_scale [K/g, N]", (long long)K);
    const int64_t N = w.size(1), groups = scale.size(0);
    if (groups == 0 || K % groups)
        fail(PyExc_ValueError, "w_scale's %lld rows must divide K = %lld", (long long)groups,
             (long long)K);
    if (N > INT_MAX) fail(PyExc_ValueError, "w is too large");
    void* wp = like(w, "w", x, at::kInt, {K / 8, N});
    void* sp = like(scale, "w_scale", x, x.scalar_type(), {groups, N});
    void* zp = like(a[3], "w_zero", x, at::kInt, {groups, N / 8});
    void* bp = like(a[4], "bias", x, x.scalar_type(), {N});
    at::Tensor out = none(a[5]) ? make({T, N}, x.scalar_type(), x) : tensor(a[5], "out");
    void* op = like(out, "out", x, x.scalar_type(), {T, N});
    if (!none(a[5])) {
        for (PyObject* o : {a[0], a[1], a[2], a[3], a[4]})
            if (!none(o) && overlap(out, THPVariable_Unpack(o)))
                fail(PyExc_ValueError, "out must not overlap an input");
        writable(out, "out");
    }
    On on(x);
    check(ferret_int4_linear(x.data_ptr(), ldx, (const int32_t*)wp, sp, (const int32_t*)zp, bp, dt,
                             (int)T, (int)K, (int)N, (int)(K / groups), op, on.stream),
          "ferret_int4_linear");
    if (!none(a[5])) written(out);
    return no_backward("ops.int4_linear", wrap(out), a[5], {a[0], a[2], a[4], a[5]});
    END_HANDLE_TH_ERRORS
}

PyObject* set_callbacks(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 2);
    Py_INCREF(a[0]);
    Py_XSETREF(g_check, a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(g_no_backward, a[1]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define FERRET_FN(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FERRET_FN(add_rms_norm),
                         FERRET_FN(moe_route),
                         FERRET_FN(moe_route_backward),
                         FERRET_FN(moe_balance_loss),
                         FERRET_FN(moe_balance_loss_backward),
                         FERRET_FN(int4_linear),
                         FERRET_FN(set_callbacks),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "ferret_b200._host",
                      "Host side of the operators around the expert GEMMs.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
