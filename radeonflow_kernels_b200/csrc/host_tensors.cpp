// CPython extension `_tensors`: checks, results and call of the FP8 quantisations, on torch's C++ interface.
//
// The kernels take 2 to 3 us for a decode batch, and what stands around them in Python took 12.3 us of host time (24 x 7168 fp16):
// two results made at 2.4 us each, the attributes of the operand, the conversion of ten arguments, and the launch, 2.1 us.  Native
// code that makes its results through their Python constructors still takes 7.9; with torch's own allocation 4 to 5.
// Where anything is not as the hot path wants it, every function answers None and the Python code that it stands in front of
// runs, with its errors; so it does where this file could not be built or loaded.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace {

using RowsFn = int (*)(const void*, int, long long, const int*, int, int, int, void*, float*, void*);
using SwigluFn = int (*)(const void*, int, long long, int, int, void*, float*, void*);
using BlocksFn = int (*)(const void*, int, int, int, int, long long, long long, long long, void*, float*, void*);

RowsFn g_rows = nullptr;
SwigluFn g_swiglu = nullptr;
BlocksFn g_blocks = nullptr;

// setup(addresses of rf_fp8_quantize, rf_fp8_swiglu_quantize, rf_fp8_quantize_blocks)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "setup: three arguments");
        return nullptr;
    }
    uintptr_t fn[3];
    for (int i = 0; i < 3; ++i) fn[i] = static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(args[i]));
    if (PyErr_Occurred()) return nullptr;
    g_rows = reinterpret_cast<RowsFn>(fn[0]);
    g_swiglu = reinterpret_cast<SwigluFn>(fn[1]);
    g_blocks = reinterpret_cast<BlocksFn>(fn[2]);
    Py_RETURN_NONE;
}

// The tensor's type as the library numbers it, -1 for another one.
int type_of(const at::Tensor& x) {
    switch (x.scalar_type()) {
        case at::kHalf: return 0;
        case at::kBFloat16: return 1;
        case at::kFloat: return 2;
        default: return -1;
    }
}

// The tensor behind `o` if it is a plain one, on the current device, of a type that is quantised; else null.
const at::Tensor* operand(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& x = THPVariable_Unpack(o);
    if (!x.is_cuda() || x.layout() != at::kStrided || type_of(x) < 0 || x.device().index() != c10::cuda::current_device()) return nullptr;
    return &x;
}

// Makes both results, calls launch(q, scale, stream), returns them; None where the library refused.
template <class Launch>
PyObject* results(const at::Tensor& x, at::IntArrayRef q_shape, at::IntArrayRef s_shape, Launch launch) {
    const at::Tensor q(at::detail::empty_cuda(q_shape, at::kFloat8_e4m3fn, x.device(), std::nullopt));
    const at::Tensor s(at::detail::empty_cuda(s_shape, at::kFloat, x.device(), std::nullopt));
    void* stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = launch(q.data_ptr(), static_cast<float*>(s.data_ptr()), stream);
    Py_END_ALLOW_THREADS
    if (status != 0) Py_RETURN_NONE;
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(q));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(s));
    if (!PyTuple_GET_ITEM(pair, 0) || !PyTuple_GET_ITEM(pair, 1)) Py_CLEAR(pair);
    return pair;
}

// quantize(x, rows or None) -> (q, scale) or None
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor* x = n == 2 && g_rows ? operand(args[0]) : nullptr;
    if (!x || x->dim() != 2 || x->size(1) % 128 != 0 || x->size(1) == 0 || x->stride(1) != 1 || x->size(0) > INT32_MAX ||
        x->size(1) > INT32_MAX)
        Py_RETURN_NONE;
    int64_t m = x->size(0);
    const int k = (int)x->size(1), n_src = (int)m;
    const int* rows = nullptr;
    if (args[1] != Py_None) {
        if (!THPVariable_CheckExact(args[1])) Py_RETURN_NONE;
        const at::Tensor& r = THPVariable_Unpack(args[1]);
        if (r.scalar_type() != at::kInt || r.dim() != 1 || !r.is_contiguous() || r.device() != x->device() || m == 0 ||
            r.size(0) > INT32_MAX)
            Py_RETURN_NONE;
        m = r.size(0);
        rows = static_cast<const int*>(r.data_ptr());
    }
    const int64_t q[2] = {m, k}, s[2] = {m, k / 128};
    return results(*x, at::IntArrayRef(q, 2), at::IntArrayRef(s, 2), [&](void* tq, float* ts, void* stream) {
        return g_rows(x->data_ptr(), type_of(*x), x->stride(0), rows, n_src, (int)m, k, tq, ts, stream);
    });
    END_HANDLE_TH_ERRORS
}

// swiglu_quantize(gate_up) -> (q, scale) or None
PyObject* swiglu_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor* x = n == 1 && g_swiglu ? operand(args[0]) : nullptr;
    if (!x || x->dim() != 2 || x->size(1) % 256 != 0 || x->size(1) == 0 || x->stride(1) != 1 || x->size(0) > INT32_MAX ||
        x->size(1) > INT32_MAX)
        Py_RETURN_NONE;
    const int64_t m = x->size(0), f = x->size(1) / 2, q[2] = {m, f}, s[2] = {m, f / 128};
    return results(*x, at::IntArrayRef(q, 2), at::IntArrayRef(s, 2), [&](void* tq, float* ts, void* stream) {
        return g_swiglu(x->data_ptr(), type_of(*x), x->stride(0), (int)m, (int)f, tq, ts, stream);
    });
    END_HANDLE_TH_ERRORS
}

// quantize_blocks(w) -> (q, scale) or None
PyObject* quantize_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor* w = n == 1 && g_blocks ? operand(args[0]) : nullptr;
    if (!w || (w->dim() != 2 && w->dim() != 3)) Py_RETURN_NONE;
    const int64_t d = w->dim(), rows = w->size(d - 2), k = w->size(d - 1), e = d == 3 ? w->size(0) : 1;
    if (k % 128 != 0 || k == 0 || (w->stride(d - 1) != 1 && w->stride(d - 2) != 1) || rows > INT32_MAX || k > INT32_MAX || e > INT32_MAX)
        Py_RETURN_NONE;
    int64_t s[3] = {e, 0, 0};
    s[d - 2] = (rows + 127) / 128;
    s[d - 1] = k / 128;
    return results(*w, w->sizes(), at::IntArrayRef(s, (size_t)d), [&](void* tq, float* ts, void* stream) {
        return g_blocks(w->data_ptr(), type_of(*w), (int)e, (int)rows, (int)k, d == 3 ? w->stride(0) : 0, w->stride(d - 2),
                        w->stride(d - 1), tq, ts, stream);
    });
    END_HANDLE_TH_ERRORS
}

template <class F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {{"setup", fast(setup), METH_FASTCALL, nullptr},
                         {"quantize", fast(quantize), METH_FASTCALL, nullptr},
                         {"swiglu_quantize", fast(swiglu_quantize), METH_FASTCALL, nullptr},
                         {"quantize_blocks", fast(quantize_blocks), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
