// Python binding of the dense operators: from tensors to the C entry points of libqkan_b200.so (include/qkan_b200.h).
//
// Small problems of these operators are bound by the host: through ctypes a layer norm of one token took 15 us around a
// kernel of 3 us, most of it descriptors, argument checks and allocations one Python call at a time. Here all of that is
// one call. Nothing is computed on this side, and there is no other path to the kernels from Python.
//
// Functions of the module (positional arguments only; functional.py has the public ones):
//   linear_forward(x, weight, bias, residual, activation, want_tape) -> (y, tape)
//   linear_backward(x, weight, gy, tape, activation, want, round_grads) -> (gx, gw, gb)
//   norm_forward(x, weight, bias, eps, want_stats) -> (y, stats)
//   norm_backward(x, weight, stats, gy, want, param_dtype) -> (gx, gw, gb)
// `want` has bit 0 for x, 1 for the weight, 2 for the bias; what is not wanted comes back as None.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <limits>
#include <string>

#include "../../include/qkan_b200.h"

namespace {

using at::Tensor;

// Numbers go into messages through std::to_string: what formats them in a stream need not be the C++ runtime that torch
// was built with.
std::string describe(const Tensor& t) {
    std::string s = c10::toString(t.scalar_type());
    s += " (";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ") on " + t.device().str();
}
std::string shape_text(at::IntArrayRef shape) {
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + ")";
}

Tensor tensor_arg(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
Tensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }

long int_arg(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

bool truth_arg(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

int io_code(at::ScalarType t, const char* what) {
    if (t == at::kFloat) return QK_F32;
    if (t == at::kBFloat16) return QK_BF16;
    TORCH_CHECK_TYPE(false, "qkan_b200 computes on float32 or bfloat16 ", what, ", got ", c10::toString(t));
}

void check_like(const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType dtype, at::Device dev) {
    TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == dtype && t.device() == dev, name, " must be ",
                      c10::toString(dtype), " of shape ", shape_text(shape), " on ", dev.str(), ", got ", describe(t));
}

// Rows and last axis of x seen as a matrix; the kernels count both in 32 bits.
void matrix_of(const Tensor& x, int64_t& rows, int64_t& width) {
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
    rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
    width = x.size(-1);
    TORCH_CHECK_VALUE(rows < (1ll << 31) && width < (1ll << 31), "x ", shape_text(x.sizes()),
                      ": rows and columns must stay below 2**31");
}

// last of the checks, so that the others can be seen without a GPU
void require_cuda(const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "qkan_b200: `x` is on ", x.device().str(),
                "; the B200 kernels are the only compute path (no CPU fallback)");
}

const void* at_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
// contiguous, and the values themselves (the imaginary part of a conjugate is a view whose sign is still to be turned)
Tensor packed(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
// and on a 16-byte boundary (a view may start anywhere in its storage)
Tensor aligned(const Tensor& t) {
    Tensor c = packed(t);
    return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone() : c;
}

// what every call works under: the tensor's device, no autograd bookkeeping, that device's current stream
struct Scope {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::OptionalCUDAGuard guard;
    void* stream;
    explicit Scope(const Tensor& x) {
        if (x.device().index() != c10::cuda::current_device()) guard.set_device(x.device());
        stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    }
};

// An error code of the library as the Python exception that _abi.check makes of it.
void check(int rc, const char* what) {
    if (rc == QK_OK) return;
    PyObject* abi = PyImport_ImportModule("qkan_b200._abi");
    if (abi) {
        Py_XDECREF(PyObject_CallMethod(abi, "check", "is", rc, what));
        Py_DECREF(abi);
    }
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
    throw python_error();
}

// An empty tensor beside x, straight from torch's allocator: through the dispatcher each took 0.25 us longer.
Tensor fresh(at::IntArrayRef shape, at::ScalarType dtype, const Tensor& x) {
    return Tensor(at::detail::empty_cuda(shape, dtype, x.device(), std::nullopt));
}

// Scratch of a call, from torch's caching allocator: kept apart per stream, and in a capture from the graph's own pool.
struct Scratch {
    size_t bytes;
    c10::DataPtr data;
    Scratch(size_t need, const char* what) : bytes(need) {
        if (need == 0) check(QK_ERR_BAD_ARGUMENT, what);
        if (need == 1) bytes = 0;  // none
        else data = c10::cuda::CUDACachingAllocator::get()->allocate(need);
    }
};

PyObject* wrap(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
PyObject* tuple_of(std::initializer_list<Tensor> ts) {
    PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
    if (!out) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor& t : ts) PyTuple_SET_ITEM(out, i++, wrap(t));
    return out;
}

void argument_count(Py_ssize_t got, Py_ssize_t want, const char* name) {
    TORCH_CHECK_TYPE(got == want, name, " takes ", std::to_string(want), " arguments, got ", std::to_string(got));
}

struct LinearCall {
    Tensor x, w;
    int64_t rows, K, N;
    c10::SmallVector<int64_t, 5> shape;  // of y
    at::ScalarType dtype;
    QkLinearDesc desc;
    LinearCall(PyObject* px, PyObject* pw, PyObject* pact) : x(tensor_arg(px, "x")), w(tensor_arg(pw, "weight")) {
        dtype = x.scalar_type();
        const int io = io_code(dtype, "activations");
        matrix_of(x, rows, K);
        TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == K && w.size(0) < (1ll << 31), "weight must be (out_features, ",
                          std::to_string(K), ") for x ", shape_text(x.sizes()), ", got ", shape_text(w.sizes()));
        N = w.size(0);
        check_like(w, "weight", w.sizes(), dtype, x.device());
        shape.assign(x.sizes().begin(), x.sizes().end());
        shape.back() = N;
        desc = {(int32_t)rows, (int32_t)K, (int32_t)N, io, (int32_t)int_arg(pact), 0};
    }
    at::ScalarType tape_type() const { return dtype == at::kFloat ? at::kFloat : at::kHalf; }
};

PyObject* linear_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    argument_count(n, 6, "linear_forward");
    LinearCall c(args[0], args[1], args[4]);
    Tensor bias = optional_arg(args[2], "bias"), residual = optional_arg(args[3], "residual");
    if (bias.defined()) check_like(bias, "bias", {c.N}, c.dtype, c.x.device());
    if (residual.defined()) check_like(residual, "residual", c.shape, c.dtype, c.x.device());
    require_cuda(c.x);
    Scope scope(c.x);
    const Tensor x = aligned(c.x), w = aligned(c.w);
    bias = packed(bias), residual = packed(residual);
    const Tensor y = fresh(c.shape, c.dtype, x);
    Tensor tape;
    if (c.desc.activation != QK_ACT_NONE && truth_arg(args[5])) tape = fresh(c.shape, c.tape_type(), x);
    const Scratch ws(qk_linear_forward_workspace_bytes(&c.desc), "qk_linear_forward_workspace_bytes");
    check(qk_linear_forward(&c.desc, x.const_data_ptr(), w.const_data_ptr(), at_or_null(bias), at_or_null(residual),
                            y.mutable_data_ptr(), const_cast<void*>(at_or_null(tape)), ws.data.get(),
                            ws.bytes, scope.stream),
          "qk_linear_forward");
    return tuple_of({y, tape});
    END_HANDLE_TH_ERRORS
}

PyObject* linear_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    argument_count(n, 7, "linear_backward");
    LinearCall c(args[0], args[1], args[4]);
    if (truth_arg(args[6])) c.desc.flags |= QK_LINEAR_ROUND_GRADS;
    Tensor gy = tensor_arg(args[2], "gy"), tape = optional_arg(args[3], "tape");
    const long want = int_arg(args[5]);
    check_like(gy, "gy", c.shape, c.dtype, c.x.device());
    if (c.desc.activation == QK_ACT_NONE) {
        tape = Tensor();
    } else {
        TORCH_CHECK_VALUE(tape.defined(), "this activation needs the tape of its forward (return_tape=True)");
        check_like(tape, "tape", c.shape, c.tape_type(), c.x.device());
    }
    require_cuda(c.x);
    Scope scope(c.x);
    const Tensor x = aligned(c.x), w = aligned(c.w);
    gy = aligned(gy), tape = packed(tape);
    Tensor gx, gw, gb;
    if (want & 1) gx = fresh(x.sizes(), x.scalar_type(), x);
    if (want & 2) gw = fresh(w.sizes(), x.scalar_type(), x);
    if (want & 4) gb = fresh({c.N}, c.dtype, x);
    const Scratch ws(qk_linear_backward_workspace_bytes(&c.desc), "qk_linear_backward_workspace_bytes");
    check(qk_linear_backward(&c.desc, x.const_data_ptr(), w.const_data_ptr(), at_or_null(tape), gy.const_data_ptr(),
                             const_cast<void*>(at_or_null(gx)), const_cast<void*>(at_or_null(gw)),
                             const_cast<void*>(at_or_null(gb)), ws.data.get(), ws.bytes, scope.stream),
          "qk_linear_backward");
    return tuple_of({gx, gw, gb});
    END_HANDLE_TH_ERRORS
}

struct NormCall {
    Tensor x, w, b;
    int64_t rows, D;
    c10::SmallVector<int64_t, 5> stats_shape;
    at::ScalarType param;
    QkNormDesc desc;
    NormCall(PyObject* px, PyObject* pw, PyObject* pb, at::ScalarType fallback, bool has_fallback)
        : x(tensor_arg(px, "x")), w(optional_arg(pw, "weight")), b(optional_arg(pb, "bias")) {
        const int io = io_code(x.scalar_type(), "activations");
        matrix_of(x, rows, D);
        TORCH_CHECK_VALUE(D >= 1, "layer_norm needs at least one element per row");
        param = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : has_fallback ? fallback : x.scalar_type();
        const int code = io_code(param, "layer norm parameters");
        if (w.defined()) check_like(w, "weight", {D}, param, x.device());
        if (b.defined()) check_like(b, "bias", {D}, param, x.device());
        stats_shape.assign(x.sizes().begin(), x.sizes().end());
        stats_shape.back() = 2;
        desc = {(int32_t)rows, (int32_t)D, io, code, 0.f, 0};
    }
};

PyObject* norm_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    argument_count(n, 5, "norm_forward");
    NormCall c(args[0], args[1], args[2], at::kFloat, false);
    const double eps = PyFloat_AsDouble(args[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(eps >= 0.0 && eps <= std::numeric_limits<float>::max(),
                      "eps must be >= 0 and finite in float32, got ", std::to_string(eps));
    c.desc.eps = (float)eps;
    require_cuda(c.x);
    Scope scope(c.x);
    const Tensor x = packed(c.x), w = packed(c.w), b = packed(c.b);
    const Tensor y = fresh(x.sizes(), x.scalar_type(), x);
    Tensor stats;
    if (truth_arg(args[4])) stats = fresh(c.stats_shape, at::kFloat, x);
    check(qk_layer_norm_forward(&c.desc, x.const_data_ptr(), at_or_null(w), at_or_null(b), y.mutable_data_ptr(),
                                static_cast<float*>(const_cast<void*>(at_or_null(stats))), scope.stream),
          "qk_layer_norm_forward");
    return tuple_of({y, stats});
    END_HANDLE_TH_ERRORS
}

PyObject* norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    argument_count(n, 6, "norm_backward");
    at::ScalarType fallback = at::kFloat;
    if (args[5] != Py_None) {
        TORCH_CHECK_TYPE(THPDtype_Check(args[5]), "param_dtype must be a torch.dtype");
        fallback = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    }
    NormCall c(args[0], args[1], Py_None, fallback, args[5] != Py_None);
    Tensor stats = tensor_arg(args[2], "stats"), gy = tensor_arg(args[3], "gy");
    const long want = int_arg(args[4]);
    check_like(gy, "gy", c.x.sizes(), c.x.scalar_type(), c.x.device());
    check_like(stats, "stats", c.stats_shape, at::kFloat, c.x.device());
    require_cuda(c.x);
    Scope scope(c.x);
    const Tensor x = packed(c.x), w = packed(c.w);
    gy = packed(gy), stats = aligned(stats);  // the kernels read a row's two numbers at once
    Tensor gx, gw, gb;
    if (want & 1) gx = fresh(x.sizes(), x.scalar_type(), x);
    if (want & 2) gw = fresh({c.D}, c.param, x);
    if (want & 4) gb = fresh({c.D}, c.param, x);
    const Scratch ws(qk_layer_norm_backward_workspace_bytes(&c.desc), "qk_layer_norm_backward_workspace_bytes");
    check(qk_layer_norm_backward(&c.desc, x.const_data_ptr(), at_or_null(w),
                                 static_cast<const float*>(stats.const_data_ptr()), gy.const_data_ptr(),
                                 const_cast<void*>(at_or_null(gx)), const_cast<void*>(at_or_null(gw)),
                                 const_cast<void*>(at_or_null(gb)), ws.data.get(), ws.bytes,
                                 scope.stream),
          "qk_layer_norm_backward");
    return tuple_of({gx, gw, gb});
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction method() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyObject* abi_version(PyObject*, PyObject*) { return PyLong_FromLong(QK_ABI_VERSION); }

PyMethodDef kMethods[] = {{"linear_forward", method<linear_forward>(), METH_FASTCALL, nullptr},
                          {"linear_backward", method<linear_backward>(), METH_FASTCALL, nullptr},
                          {"norm_forward", method<norm_forward>(), METH_FASTCALL, nullptr},
                          {"norm_backward", method<norm_backward>(), METH_FASTCALL, nullptr},
                          {"abi_version", abi_version, METH_NOARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_dense", "Dense operators of libqkan_b200.so on torch tensors.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dense() { return PyModule_Create(&kModule); }
