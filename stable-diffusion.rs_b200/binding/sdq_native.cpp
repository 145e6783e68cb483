// sdq_native.cpp -- the ordinary call of the fp8 and head-preparation entry points, in C++.
//
// A call of a few microseconds on the GPU is no faster than the interpreter that makes it: checking
// the arguments, allocating the results and converting twenty values for ctypes took 7 to 16 us.
// Each function here does that for what nearly every call is -- plain tensors of the right types on
// the current device, its current stream, no error -- and calls the same C entry point.  For anything
// else it returns None and has done nothing that lasts, and the Python function goes on to run the
// call its own way or to say what is wrong with it.  The entry points' addresses come from the library
// that the package has loaded.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "sdq.h"

namespace {

decltype(&sdq_fp8_quantize) g_quantize = nullptr;
decltype(&sdq_fp8_quantize_weight) g_quantize_weight = nullptr;
decltype(&sdq_fp8_matmul) g_matmul = nullptr;
decltype(&sdq_qk_norm_rope) g_heads = nullptr;

constexpr int64_t kBlock = 128;
constexpr auto kE4M3 = at::ScalarType::Float8_e4m3fn;
constexpr auto kE8M0 = at::ScalarType::Float8_e8m0fnu;

// A plain tensor, or nullptr.
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool here(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }
bool flat(const at::Tensor* t, int dev, at::ScalarType dt) {
    return t && here(*t, dev) && t->scalar_type() == dt && t->is_contiguous();
}
bool shaped(const at::Tensor& t, int64_t a, int64_t b) { return t.dim() == 2 && t.size(0) == a && t.size(1) == b; }

// The library's code of an unquantised type, or -1.
int code(at::ScalarType dt) { return dt == at::kBFloat16 ? SDQ_BF16 : dt == at::kFloat ? SDQ_F32 : -1; }

at::Tensor empty(at::IntArrayRef size, at::ScalarType dt, int dev) {
    return at::Tensor(at::detail::empty_cuda(size, dt, c10::Device(c10::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}
void* stream(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

PyObject* pair(at::Tensor a, at::Tensor b) {
    PyObject* t = PyTuple_New(2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
    return t;
}

// The library's call without the interpreter's lock: a launch may wait for room in the stream's queue.
template <class F, class... A>
int unlocked(F f, A... a) {
    PyThreadState* t = PyEval_SaveThread();
    const int rc = f(a...);
    PyEval_RestoreThread(t);
    return rc;
}

// quantize(x) and quantize_weight(w) -> (codes, scales)
template <bool WEIGHT>
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor* x = n == 1 && g_quantize ? tensor(args[0]) : nullptr;
    if (!x || !x->is_cuda()) Py_RETURN_NONE;
    const int dev = c10::cuda::current_device(), dt = code(x->scalar_type());
    if (!here(*x, dev) || dt < 0 || !x->is_contiguous() || (WEIGHT ? x->dim() != 2 : x->dim() < 1)) Py_RETURN_NONE;
    const int64_t k = x->size(-1);
    if (k == 0 || x->numel() == 0) Py_RETURN_NONE;
    const int64_t rows = x->numel() / k, kb = (k + kBlock - 1) / kBlock;
    at::Tensor q = empty(x->sizes(), kE4M3, dev);
    at::Tensor s = WEIGHT ? empty({(rows + kBlock - 1) / kBlock, kb}, kE8M0, dev) : empty({kb, rows}, kE8M0, dev);
    const auto f = WEIGHT ? g_quantize_weight : g_quantize;
    if (unlocked(f, x->data_ptr(), (sdq_dtype)dt, rows, k, (uint8_t*)q.data_ptr(), (uint8_t*)s.data_ptr(), stream(dev)) != SDQ_OK)
        Py_RETURN_NONE;
    return pair(std::move(q), std::move(s));
    END_HANDLE_TH_ERRORS
}

// An argument that may be None: *out is the tensor or nullptr; false when it is neither.
bool optional(PyObject* o, const at::Tensor** out) {
    *out = o == Py_None ? nullptr : tensor(o);
    return o == Py_None || *out;
}

// matmul(xq, xs, wq, ws, bias, act, gate, residual, out, out_dtype) -> y
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !g_matmul) Py_RETURN_NONE;
    const at::Tensor *xq = tensor(args[0]), *xs = tensor(args[1]), *wq = tensor(args[2]), *ws = tensor(args[3]);
    const at::Tensor *bias, *gate, *residual, *out;
    if (!xq || !xq->is_cuda() || !optional(args[4], &bias) || !optional(args[6], &gate) || !optional(args[7], &residual) ||
        !optional(args[8], &out))
        Py_RETURN_NONE;
    int act = SDQ_ACT_NONE;
    if (args[5] != Py_None) {
        if (!PyUnicode_Check(args[5])) Py_RETURN_NONE;
        if (PyUnicode_CompareWithASCIIString(args[5], "silu") == 0) act = SDQ_ACT_SILU;
        else if (PyUnicode_CompareWithASCIIString(args[5], "gelu_approx") == 0) act = SDQ_ACT_GELU_TANH;
        else Py_RETURN_NONE;
    }
    const int dev = c10::cuda::current_device();
    if (!flat(xq, dev, kE4M3) || !flat(xs, dev, kE8M0) || !flat(wq, dev, kE4M3) || !flat(ws, dev, kE8M0) || xq->dim() < 1 ||
        wq->dim() != 2 || xq->numel() == 0)
        Py_RETURN_NONE;
    const int64_t k = xq->size(-1), m = xq->numel() / k, f = wq->size(0), kb = (k + kBlock - 1) / kBlock;
    at::ScalarType dt = out ? out->scalar_type() : at::kBFloat16;
    if (args[9] != Py_None) {
        if (!THPDtype_Check(args[9])) Py_RETURN_NONE;
        const at::ScalarType asked = reinterpret_cast<THPDtype*>(args[9])->scalar_type;
        if (out && asked != dt) Py_RETURN_NONE;
        dt = asked;
    }
    if (code(dt) < 0 || wq->size(1) != k || !shaped(*xs, kb, m) || !shaped(*ws, (f + kBlock - 1) / kBlock, kb) ||
        (bias && !(flat(bias, dev, dt) && bias->numel() == f)) || (gate && !(flat(gate, dev, dt) && gate->numel() == f)) ||
        (residual && !(flat(residual, dev, dt) && residual->numel() == m * f)))
        Py_RETURN_NONE;
    c10::SmallVector<int64_t, 8> size(xq->sizes().begin(), xq->sizes().end());
    size.back() = f;
    if (out && !(flat(out, dev, dt) && out->sizes() == at::IntArrayRef(size))) Py_RETURN_NONE;
    at::Tensor y = out ? *out : empty(size, dt, dev);
    if (unlocked(g_matmul, (const uint8_t*)xq->data_ptr(), (const uint8_t*)xs->data_ptr(), m, k, (const uint8_t*)wq->data_ptr(),
                 (const uint8_t*)ws->data_ptr(), f, bias ? bias->data_ptr() : nullptr, act, gate ? gate->data_ptr() : nullptr,
                 residual ? residual->data_ptr() : nullptr, y.data_ptr(), (sdq_dtype)code(dt), stream(dev)) != SDQ_OK)
        Py_RETURN_NONE;
    if (out) return Py_NewRef(args[8]);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// heads(q, k, v, q_weight, k_weight, cos, sin, eps, positions, pairs, out) -> (q, k, v)
PyObject* heads(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11 || !g_heads) Py_RETURN_NONE;
    const at::Tensor *x[3] = {tensor(args[0]), tensor(args[1]), nullptr}, *w[2], *cos, *sin, *pos;
    if (!x[0] || !x[1] || !x[0]->is_cuda() || !optional(args[2], &x[2]) || !optional(args[3], &w[0]) ||
        !optional(args[4], &w[1]) || !optional(args[5], &cos) || !optional(args[6], &sin) || !optional(args[8], &pos) ||
        !PyFloat_Check(args[7]) || !PyUnicode_Check(args[9]))
        Py_RETURN_NONE;
    const bool inter = PyUnicode_CompareWithASCIIString(args[9], "interleaved") == 0;
    if (!inter && PyUnicode_CompareWithASCIIString(args[9], "halves") != 0) Py_RETURN_NONE;
    const int dev = c10::cuda::current_device(), dt = code(x[0]->scalar_type()), count = x[2] ? 3 : 2;
    if (dt < 0 || x[0]->dim() != 4 || x[0]->numel() == 0 || (cos == nullptr) != (sin == nullptr) || (pos && !cos)) Py_RETURN_NONE;
    const at::ScalarType type = x[0]->scalar_type();
    const int64_t b = x[0]->size(0), t = x[0]->size(1), d = x[0]->size(3);
    PyObject* const given = args[10];
    if (given != Py_None && !(PyTuple_Check(given) && PyTuple_GET_SIZE(given) == count)) Py_RETURN_NONE;
    at::Tensor made[3];
    const at::Tensor* y[3] = {};
    sdq_heads in[3] = {}, to[3] = {};
    for (int i = 0; i < count; ++i) {
        const at::Tensor& a = *x[i];
        if (!here(a, dev) || a.scalar_type() != type || a.dim() != 4 || a.size(0) != b || a.size(1) != t || a.size(3) != d ||
            a.stride(3) != 1)
            Py_RETURN_NONE;
        const int64_t h = a.size(2);
        if (given == Py_None) {
            made[i] = empty({b, h, t, d}, type, dev);
            y[i] = &made[i];
        } else {
            y[i] = tensor(PyTuple_GET_ITEM(given, i));
            if (!y[i] || !here(*y[i], dev) || y[i]->scalar_type() != type || y[i]->dim() != 4 || y[i]->size(0) != b ||
                y[i]->size(1) != h || y[i]->size(2) != t || y[i]->size(3) != d || y[i]->stride(3) != 1)
                Py_RETURN_NONE;
        }
        in[i] = {a.data_ptr(), h, a.stride(0), a.stride(1), a.stride(2)};
        to[i] = {y[i]->data_ptr(), h, y[i]->stride(0), y[i]->stride(2), y[i]->stride(1)};
    }
    for (const at::Tensor* v : w)
        if (v && !(flat(v, dev, type) && v->numel() == d)) Py_RETURN_NONE;
    int64_t rows = 0, rope = 0, stride = 0;
    int wide = 0;
    if (cos) {
        if (!flat(cos, dev, at::kFloat) || !flat(sin, dev, at::kFloat) || cos->dim() != 2 || cos->sizes() != sin->sizes()) Py_RETURN_NONE;
        rows = cos->size(0);
        rope = 2 * cos->size(1);
        if (rope > d) Py_RETURN_NONE;
    }
    if (pos) {
        wide = pos->scalar_type() == at::kLong;
        if (!here(*pos, dev) || !(wide || pos->scalar_type() == at::kInt) || !shaped(*pos, b, t) || (t > 1 && pos->stride(1) != 1))
            Py_RETURN_NONE;
        stride = pos->stride(0);
    }
    if (d > 256 || unlocked(g_heads, &in[0], &in[1], x[2] ? &in[2] : nullptr, &to[0], &to[1], x[2] ? &to[2] : nullptr, (sdq_dtype)dt, b, t,
                           (int)d, w[0] ? w[0]->data_ptr() : nullptr, w[1] ? w[1]->data_ptr() : nullptr,
                           (float)PyFloat_AS_DOUBLE(args[7]), cos ? cos->data_ptr<float>() : nullptr,
                           sin ? sin->data_ptr<float>() : nullptr, rows, (int)rope, inter, pos ? pos->data_ptr() : nullptr, wide,
                           stride, stream(dev)) != SDQ_OK)
        Py_RETURN_NONE;
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    for (int i = 0; i < 3; ++i)
        PyTuple_SET_ITEM(r, i, i >= count ? Py_NewRef(Py_None)
                                          : given == Py_None ? THPVariable_Wrap(std::move(made[i]))
                                                             : Py_NewRef(PyTuple_GET_ITEM(given, i)));
    return r;
    END_HANDLE_TH_ERRORS
}

// bind(addresses of sdq_fp8_quantize, sdq_fp8_quantize_weight, sdq_fp8_matmul, sdq_qk_norm_rope)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    void* p[4];
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
        return nullptr;
    }
    for (int i = 0; i < 4; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    g_quantize = reinterpret_cast<decltype(g_quantize)>(p[0]);
    g_quantize_weight = reinterpret_cast<decltype(g_quantize_weight)>(p[1]);
    g_matmul = reinterpret_cast<decltype(g_matmul)>(p[2]);
    g_heads = reinterpret_cast<decltype(g_heads)>(p[3]);
    Py_RETURN_NONE;
}

#define SDQ_METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    SDQ_METHOD("bind", bind),
    SDQ_METHOD("fp8_quantize", quantize<false>),
    SDQ_METHOD("fp8_quantize_weight", quantize<true>),
    SDQ_METHOD("fp8_matmul", matmul),
    SDQ_METHOD("qk_norm_rope", heads),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&g_module); }
