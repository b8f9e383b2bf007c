// The common calls of libmvquant.so's operators as Python functions, for their host time: a
// ctypes call and the argument checks in Python cost several times what the small
// kernels take. Each function here takes the usual case -- exact CUDA tensors on the
// current device, contiguous or with strided rows, no gradients, outputs allocated
// here -- and returns None for any other, which the Python wrappers then check, run or
// refuse as they would have without it. No state but the entry points' addresses.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <optional>

#include "mvquant.h"

namespace {

decltype(&mvq_w4_linear) g_linear;
decltype(&mvq_w4_dequantize) g_dequantize;
decltype(&mvq_add_rms_norm) g_norm;
decltype(&mvq_silu_mul_quant) g_silu;

// MVQ_DTYPE_* of a type, or -1.
int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MVQ_DTYPE_F32;
        case at::kHalf: return MVQ_DTYPE_F16;
        case at::kBFloat16: return MVQ_DTYPE_BF16;
        case at::kChar: return MVQ_DTYPE_I8;
        case at::kFloat8_e4m3fn: return MVQ_DTYPE_E4M3;
        default: return -1;
    }
}

// Inside a function transform, or with a tangent of forward-mode differentiation.
bool transformed(const at::Tensor& t) {
    return t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched,
                                                    c10::DispatchKey::FuncTorchGradWrapper,
                                                    c10::DispatchKey::Functionalize})) ||
           (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined());
}

// A plain tensor of the device, or null.
const at::Tensor* tensor_of(PyObject* o, int device) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || (t.requires_grad() && at::GradMode::is_enabled()) ||
        transformed(t))
        return nullptr;
    return device < 0 || t.get_device() == device ? &t : nullptr;
}

// Row stride of t [..., width] as [rows, width], or -1 where it cannot be seen so.
int64_t row_stride(const at::Tensor& t, int64_t width) {
    if (t.is_contiguous()) return width;
    if (t.dim() != 2 || (t.stride(1) != 1 && width != 1)) return -1;
    return t.stride(0);
}

// Device `device` is current, and no mode is on that means to see torch's calls.
bool current(int device) {
    return c10::cuda::current_device() == device && !c10::impl::TorchDispatchModeTLS::any_modes_set();
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Device& device) {
    return at::detail::empty_cuda(shape, type, device, std::nullopt);
}

// A status that is not MVQ_OK: back to Python, which repeats the call and raises its message.
PyObject* none() { Py_RETURN_NONE; }

// linear(x, weight's fixed fields, weight's device, bias, residual, x_scale, out_dtype)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 7 || !PyBytes_CheckExact(a[1])) return none();
    const at::Tensor* x = tensor_of(a[0], -1);
    if (!x) return none();
    const int device = static_cast<int>(x->get_device());
    if (PyLong_AsLong(a[2]) != device || !current(device)) return none();
    MvqLinearArgs args = {};
    static_assert(offsetof(MvqLinearArgs, bias) - offsetof(MvqLinearArgs, records) == 48, "fixed fields");
    if (PyBytes_GET_SIZE(a[1]) != 48) return none();
    std::memcpy(&args.records, PyBytes_AS_STRING(a[1]), 48);
    args.x_dtype = code_of(x->scalar_type());
    const int64_t k = args.k, n = args.n;
    if (args.x_dtype < 0 || x->dim() < 1 || x->size(-1) != k) return none();
    args.x = x->data_ptr();
    args.x_stride_row = row_stride(*x, k);
    if (args.x_stride_row < 0) return none();
    args.m = x->numel() / k;
    if (args.m == 0) return none();
    const at::Tensor *bias = nullptr, *residual = nullptr;
    if (a[3] != Py_None && !(bias = tensor_of(a[3], device))) return none();
    if (a[4] != Py_None && !(residual = tensor_of(a[4], device))) return none();
    at::ScalarType type = x->scalar_type();
    if (THPDtype_Check(a[6])) type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
    else if (a[6] != Py_None) return none();
    else if (residual) type = residual->scalar_type();
    else if (bias) type = bias->scalar_type();
    args.out_dtype = code_of(type);
    if (args.out_dtype < 0 || args.out_dtype > MVQ_DTYPE_BF16) return none();
    if (a[5] != Py_None) {
        const at::Tensor* scale = tensor_of(a[5], device);
        if (!scale || scale->scalar_type() != at::kFloat || scale->numel() != args.m || !scale->is_contiguous()) return none();
        args.x_scale = scale->data_ptr();
    } else if (args.x_dtype > MVQ_DTYPE_BF16) {
        return none();
    }
    if (bias) {
        if (bias->scalar_type() != type || bias->dim() != 1 || bias->size(0) != n || !bias->is_contiguous()) return none();
        args.bias = bias->data_ptr();
    }
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = n;
    if (residual) {
        if (residual->scalar_type() != type || residual->sizes() != at::IntArrayRef(shape)) return none();
        args.residual = residual->data_ptr();
        args.residual_stride_row = row_stride(*residual, n);
        if (args.residual_stride_row < 0) return none();
    }
    at::Tensor out = fresh(shape, type, x->device());
    args.out = out.data_ptr();
    args.out_stride_row = n;
    if (g_linear(&args, stream_of(device)) != MVQ_OK) return none();
    return THPVariable_Wrap(std::move(out));
}

// dequantize(weight's fixed fields, weight's records, dtype)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 3 || !PyBytes_CheckExact(a[0]) || PyBytes_GET_SIZE(a[0]) != 48 || !THPDtype_Check(a[2])) return none();
    const at::Tensor* records = tensor_of(a[1], -1);
    if (!records) return none();
    const int device = static_cast<int>(records->get_device());
    if (!current(device)) return none();
    MvqDequantizeArgs args = {};
    static_assert(offsetof(MvqDequantizeArgs, out) == 48, "fixed fields");
    std::memcpy(&args.records, PyBytes_AS_STRING(a[0]), 48);
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    args.out_dtype = code_of(type);
    if (args.out_dtype < 0 || args.out_dtype > MVQ_DTYPE_BF16) return none();
    at::Tensor out = fresh({args.n, args.k}, type, records->device());
    args.out = out.data_ptr();
    args.out_stride_row = args.k;
    if (g_dequantize(&args, stream_of(device)) != MVQ_OK) return none();
    return THPVariable_Wrap(std::move(out));
}

// Rows [..., width] whose rows do not overlap: their stride, or -1.
int64_t input_rows(const at::Tensor& t, int64_t width) {
    const int64_t stride = row_stride(t, width);
    return stride < 0 || (t.numel() > width && stride < width) ? -1 : stride;
}

PyObject* tuple_of(at::Tensor&& a, at::Tensor&& b) {
    PyObject* tuple = PyTuple_New(2);
    if (!tuple) return nullptr;
    PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(tuple, 1, THPVariable_Wrap(std::move(b)));
    return tuple;
}

// norm(x, residual or None, weight, eps, out's dtype): (out, scales or None, residual_out)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 5 || !PyFloat_CheckExact(a[3]) || !THPDtype_Check(a[4])) return none();
    const at::Tensor* x = tensor_of(a[0], -1);
    if (!x || x->dim() < 1 || x->numel() == 0) return none();
    const int device = static_cast<int>(x->get_device());
    const at::Tensor *residual = nullptr, *weight = tensor_of(a[2], device);
    if (a[1] != Py_None && !(residual = tensor_of(a[1], device))) return none();
    const at::ScalarType type = x->scalar_type(), out_type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    const int64_t hidden = x->size(-1);
    MvqNormArgs args = {};
    args.dtype = code_of(type);
    args.out_dtype = code_of(out_type);
    const bool eight = args.out_dtype > MVQ_DTYPE_BF16;
    if (!weight || !current(device) || args.dtype < 0 || args.dtype > MVQ_DTYPE_BF16 || (!eight && out_type != type) ||
        weight->scalar_type() != type || weight->dim() != 1 || weight->size(0) != hidden || !weight->is_contiguous() ||
        (residual && (residual->scalar_type() != type || residual->sizes() != x->sizes())))
        return none();
    args.x = x->data_ptr();
    args.x_stride_row = input_rows(*x, hidden);
    args.residual_stride_row = residual ? input_rows(*residual, hidden) : 0;
    if (args.x_stride_row < 0 || args.residual_stride_row < 0) return none();
    args.weight = weight->data_ptr();
    args.rows = x->numel() / hidden;
    args.hidden = hidden;
    args.eps = PyFloat_AS_DOUBLE(a[3]);
    at::Tensor out = fresh(x->sizes(), out_type, x->device()), total, scales;
    args.out = out.data_ptr();
    args.out_stride_row = hidden;
    if (residual) {
        total = fresh(x->sizes(), type, x->device());
        args.residual = residual->data_ptr();
        args.residual_out = total.data_ptr();
        args.residual_out_stride_row = hidden;
    }
    if (eight) {
        scales = fresh(x->sizes().slice(0, x->dim() - 1), at::kFloat, x->device());
        args.scales = scales.data_ptr();
    }
    if (g_norm(&args, stream_of(device)) != MVQ_OK) return none();
    PyObject* tuple = PyTuple_New(3);
    if (!tuple) return nullptr;
    PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(out)));
    if (!eight) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(tuple, 1, eight ? THPVariable_Wrap(std::move(scales)) : Py_None);
    if (!residual) Py_INCREF(a[0]);
    PyTuple_SET_ITEM(tuple, 2, residual ? THPVariable_Wrap(std::move(total)) : a[0]);
    return tuple;
}

// silu(gate_up, out's dtype): (out, scales)
PyObject* silu(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 2 || !THPDtype_Check(a[1])) return none();
    const at::Tensor* x = tensor_of(a[0], -1);
    if (!x || x->dim() < 1 || x->numel() == 0 || x->size(-1) % 2) return none();
    const int device = static_cast<int>(x->get_device());
    const int64_t both = x->size(-1);
    MvqSiluArgs args = {};
    args.dtype = code_of(x->scalar_type());
    const at::ScalarType out_type = reinterpret_cast<THPDtype*>(a[1])->scalar_type;
    args.out_dtype = code_of(out_type);
    args.stride_row = input_rows(*x, both);
    if (!current(device) || args.dtype < 0 || args.dtype > MVQ_DTYPE_BF16 || args.out_dtype <= MVQ_DTYPE_BF16 ||
        args.stride_row < 0)
        return none();
    args.gate_up = x->data_ptr();
    args.width = both / 2;
    args.rows = x->numel() / both;
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = args.width;
    at::Tensor out = fresh(shape, out_type, x->device());
    at::Tensor scales = fresh(x->sizes().slice(0, x->dim() - 1), at::kFloat, x->device());
    args.out = out.data_ptr();
    args.out_stride_row = args.width;
    args.scales = scales.data_ptr();
    if (g_silu(&args, stream_of(device)) != MVQ_OK) return none();
    return tuple_of(std::move(out), std::move(scales));
}

// A C++ exception (an allocation that fails) becomes Python's.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    return F(self, a, count);
    END_HANDLE_TH_ERRORS
}

// any_transformed(tensors or None...): whether one is transformed, or a mode is on.
PyObject* any_transformed(PyObject*, PyObject* const* a, Py_ssize_t count) {
    bool found = c10::impl::TorchDispatchModeTLS::any_modes_set();
    for (Py_ssize_t i = 0; i < count && !found; ++i)
        found = THPVariable_Check(a[i]) && transformed(THPVariable_Unpack(a[i]));
    return PyBool_FromLong(found);
}

// bind(linear, dequantize, norm, silu): the loaded library's entry points, as addresses.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 4) {
        PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
        return nullptr;
    }
    void* at[4];
    for (int i = 0; i < 4; ++i) {
        at[i] = PyLong_AsVoidPtr(a[i]);
        if (!at[i] && PyErr_Occurred()) return nullptr;
    }
    g_linear = reinterpret_cast<decltype(g_linear)>(at[0]);
    g_dequantize = reinterpret_cast<decltype(g_dequantize)>(at[1]);
    g_norm = reinterpret_cast<decltype(g_norm)>(at[2]);
    g_silu = reinterpret_cast<decltype(g_silu)>(at[3]);
    Py_RETURN_NONE;
}

#define MVQ_METHOD(name, function) \
    {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)), METH_FASTCALL, nullptr}

PyMethodDef g_methods[] = {MVQ_METHOD("linear", guarded<linear>), MVQ_METHOD("dequantize", guarded<dequantize>),
                           MVQ_METHOD("norm", guarded<norm>), MVQ_METHOD("silu", guarded<silu>),
                           MVQ_METHOD("any_transformed", guarded<any_transformed>),
                           MVQ_METHOD("bind", bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_mvq_binding", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__mvq_binding() { return PyModule_Create(&g_module); }
