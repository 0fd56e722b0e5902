// CPython extension `_host`: the checks and the call of the two hot Python entry points, in native code.
//
// A small GEMM runs in 3.5 to 6.5 us, and the Python boundary around it took 6.5 to 7.3 us of host time, which bounded such
// calls when they follow one another: 1.7 us of attribute reads and comparisons, 1.8 us to convert ten arguments through
// ctypes, the rest interpreter.  This module reads the same attributes of the same objects, and where everything is as the
// hot path wants it, calls the library: 4.2 to 5.4 us, of which the launch is 2.  Where anything is not, it answers "not
// here", and the Python code that it stands in front of runs as ever, with its errors.  (It includes no torch header: it
// reads tensors through their Python attributes.)  The addresses of a MoE layer's expert weights are gathered the same way:
// 64 experts, 96 us of host time for a layer, now 70.  So are the FP8 quantisations, whose kernels take 2 to 3 us for a decode
// batch, their two results included (24 x 7168: 12.3 us of host time in Python), and the grouped product.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <vector>

namespace {

using RunFn = void (*)(void*, void*, void*, void*, void*, int, int, int, void*, void*);

using RowsFn = int (*)(const void*, int, long long, const int*, int, int, int, void*, float*, void*);
using SwigluFn = int (*)(const void*, int, long long, int, int, void*, float*, void*);
using BlocksFn = int (*)(const void*, int, int, int, int, long long, long long, long long, void*, float*, void*);
using GroupedFn = int (*)(const void*, const void*, const float*, const float*, const int*, void*, int, int, int, int, int, void*);

RunFn g_run = nullptr;
RowsFn g_rows = nullptr;
SwigluFn g_swiglu = nullptr;
BlocksFn g_blocks = nullptr;
GroupedFn g_grouped = nullptr;
PyObject *g_get_device = nullptr, *g_get_stream = nullptr;
PyObject *g_fp8 = nullptr, *g_f32 = nullptr, *g_bf16 = nullptr, *g_f16 = nullptr;
PyObject* g_i32 = nullptr;
PyObject *s_is_cuda, *s_is_contiguous, *s_dtype, *s_shape, *s_data_ptr, *s_stride, *s_get_device, *s_new_empty, *s_kw_dtype;

// 1 / 0 = the attribute is (is not) `want`; -1 = an exception is set
int attr_is(PyObject* o, PyObject* name, PyObject* want) {
    PyObject* v = PyObject_GetAttr(o, name);
    if (!v) return -1;
    const int r = v == want;
    Py_DECREF(v);
    return r;
}

int contiguous(PyObject* o) {
    PyObject* v = PyObject_CallMethodNoArgs(o, s_is_contiguous);
    if (!v) return -1;
    const int r = v == Py_True;
    Py_DECREF(v);
    return r;
}

// a contiguous CUDA tensor of this type
int hot_tensor(PyObject* o, PyObject* dtype) {
    int r = attr_is(o, s_is_cuda, Py_True);
    if (r == 1) r = attr_is(o, s_dtype, dtype);
    if (r == 1) r = contiguous(o);
    return r;
}

int shape2(PyObject* o, long long* rows, long long* cols) {
    PyObject* v = PyObject_GetAttr(o, s_shape);
    if (!v) return -1;
    int r = 0;
    if (PyTuple_Check(v) && PyTuple_GET_SIZE(v) == 2) {
        *rows = PyLong_AsLongLong(PyTuple_GET_ITEM(v, 0));
        *cols = PyLong_AsLongLong(PyTuple_GET_ITEM(v, 1));
        r = PyErr_Occurred() ? -1 : 1;
    }
    Py_DECREF(v);
    return r;
}

bool data_ptr(PyObject* o, uint64_t* p) {
    PyObject* v = PyObject_CallMethodNoArgs(o, s_data_ptr);
    if (!v) return false;
    *p = PyLong_AsUnsignedLongLong(v);
    Py_DECREF(v);
    return !PyErr_Occurred();
}

// setup(address of `run`, get_device, get_raw_stream, float8_e4m3fn, float32, bfloat16, float16)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "setup: seven arguments");
        return nullptr;
    }
    const unsigned long long run = PyLong_AsUnsignedLongLong(args[0]);
    if (PyErr_Occurred()) return nullptr;
    PyObject** slots[6] = {&g_get_device, &g_get_stream, &g_fp8, &g_f32, &g_bf16, &g_f16};
    for (int i = 0; i < 6; ++i) {
        Py_INCREF(args[1 + i]);
        Py_XSETREF(*slots[i], args[1 + i]);
    }
    g_run = reinterpret_cast<RunFn>(static_cast<uintptr_t>(run));
    Py_RETURN_NONE;
}

// gemm(a, b, a_scale, b_scale, c) -> True: launched; False: not the hot form, nothing done
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 5 || !g_run) Py_RETURN_FALSE;
    PyObject* const dtypes[5] = {g_fp8, g_fp8, g_f32, g_f32, g_bf16};
    long long rows[5], cols[5];
    for (int i = 0; i < 5; ++i) {
        int r = hot_tensor(args[i], dtypes[i]);
        if (r == 1) r = shape2(args[i], &rows[i], &cols[i]);
        if (r < 0) return nullptr;
        if (r == 0) Py_RETURN_FALSE;
    }
    const long long m = rows[0], k = cols[0], nn = rows[1], kb = k / 128;
    if (cols[1] != k || rows[4] != m || cols[4] != nn || rows[2] != m || cols[2] != kb || rows[3] != (nn + 127) / 128 ||
        cols[3] != kb || m > INT32_MAX || nn > INT32_MAX || k > INT32_MAX)
        Py_RETURN_FALSE;
    uint64_t p[5];
    for (int i = 0; i < 5; ++i)
        if (!data_ptr(args[i], &p[i])) return nullptr;
    PyObject* device = PyObject_CallNoArgs(g_get_device);
    if (!device) return nullptr;
    PyObject* stream = PyObject_CallOneArg(g_get_stream, device);
    Py_DECREF(device);
    if (!stream) return nullptr;
    const unsigned long long s = PyLong_AsUnsignedLongLong(stream);
    Py_DECREF(stream);
    if (PyErr_Occurred()) return nullptr;
    auto ptr = [](unsigned long long v) { return reinterpret_cast<void*>(static_cast<uintptr_t>(v)); };
    Py_BEGIN_ALLOW_THREADS
    g_run(ptr(p[0]), ptr(p[1]), ptr(p[2]), ptr(p[3]), ptr(p[4]), (int)m, (int)nn, (int)k, nullptr, ptr(s));
    Py_END_ALLOW_THREADS
    Py_RETURN_TRUE;
}

// fp16_addresses(weights, names) -> bytes: the 64-bit addresses of weights[name], all of them contiguous CUDA fp16
// tensors; None: not all are
PyObject* fp16_addresses(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !g_run || !PyDict_CheckExact(args[0]) || !PyTuple_CheckExact(args[1])) Py_RETURN_NONE;
    const Py_ssize_t count = PyTuple_GET_SIZE(args[1]);
    std::vector<uint64_t> out((size_t)count);
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject* t = PyDict_GetItemWithError(args[0], PyTuple_GET_ITEM(args[1], i));
        if (!t) {
            if (PyErr_Occurred()) return nullptr;
            Py_RETURN_NONE;
        }
        Py_INCREF(t);       // (attribute reads run Python code, which could take it out of the dict)
        const int r = hot_tensor(t, g_f16);
        const bool ok = r == 1 && data_ptr(t, &out[(size_t)i]);
        Py_DECREF(t);
        if (!ok) {
            if (PyErr_Occurred()) return nullptr;
            Py_RETURN_NONE;
        }
    }
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(out.data()), count * (Py_ssize_t)sizeof(uint64_t));
}

// setup_fp8(addresses of rf_fp8_quantize, rf_fp8_swiglu_quantize, rf_fp8_quantize_blocks, rf_fp8_grouped_gemm; int32)
PyObject* setup_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "setup_fp8: five arguments");
        return nullptr;
    }
    uintptr_t fn[4];
    for (int i = 0; i < 4; ++i) fn[i] = static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(args[i]));
    if (PyErr_Occurred()) return nullptr;
    g_rows = reinterpret_cast<RowsFn>(fn[0]);
    g_swiglu = reinterpret_cast<SwigluFn>(fn[1]);
    g_blocks = reinterpret_cast<BlocksFn>(fn[2]);
    g_grouped = reinterpret_cast<GroupedFn>(fn[3]);
    Py_INCREF(args[4]);
    Py_XSETREF(g_i32, args[4]);
    Py_RETURN_NONE;
}

// The numbers of a tuple of at most `most`; their count, or -1 (an exception is set) or 0
int numbers(PyObject* v, long long* out, int most) {
    if (!v) return -1;
    int n = 0;
    if (PyTuple_Check(v) && PyTuple_GET_SIZE(v) <= most) {
        n = (int)PyTuple_GET_SIZE(v);
        for (int i = 0; i < n; ++i) out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(v, i));
    }
    Py_DECREF(v);
    return PyErr_Occurred() ? -1 : n;
}

// The current device and its current stream; false: an exception is set
bool device_and_stream(long long* device, void** stream) {
    PyObject* d = PyObject_CallNoArgs(g_get_device);
    if (!d) return false;
    *device = PyLong_AsLongLong(d);
    PyObject* s = PyObject_CallOneArg(g_get_stream, d);
    Py_DECREF(d);
    if (!s) return false;
    *stream = reinterpret_cast<void*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(s)));
    Py_DECREF(s);
    return !PyErr_Occurred();
}

// 1: on that device; 0: not; -1: an exception is set
int on_device(PyObject* o, long long device) {
    PyObject* v = PyObject_CallMethodNoArgs(o, s_get_device);
    if (!v) return -1;
    const long long d = PyLong_AsLongLong(v);
    Py_DECREF(v);
    return PyErr_Occurred() ? -1 : d == device;
}

// A matrix to quantise: a CUDA tensor in one of the three types (source), on the current device (here).
struct Source {
    int dtype;          // as the library numbers them
    int dims;
    long long shape[3], stride[3];
    long long device;
    void* stream;
    uint64_t ptr;
};
int source(PyObject* o, Source* s) {
    int r = attr_is(o, s_is_cuda, Py_True);
    if (r != 1) return r;
    PyObject* t = PyObject_GetAttr(o, s_dtype);
    if (!t) return -1;
    s->dtype = t == g_f16 ? 0 : t == g_bf16 ? 1 : t == g_f32 ? 2 : -1;
    Py_DECREF(t);
    if (s->dtype < 0) return 0;
    s->dims = numbers(PyObject_GetAttr(o, s_shape), s->shape, 3);
    if (s->dims <= 0) return s->dims;
    const int n = numbers(PyObject_CallMethodNoArgs(o, s_stride), s->stride, 3);
    if (n != s->dims) return n < 0 ? -1 : 0;
    for (int i = 0; i < n; ++i)
        if (s->shape[i] > INT32_MAX) return 0;
    return data_ptr(o, &s->ptr) ? 1 : -1;
}
int here(PyObject* o, Source* s) { return device_and_stream(&s->device, &s->stream) ? on_device(o, s->device) : -1; }

// A new tensor on o's device and its address; null: an exception is set
PyObject* new_tensor(PyObject* o, const long long* shape, int dims, PyObject* dtype, uint64_t* ptr) {
    PyObject* sizes = PyTuple_New(dims);
    if (!sizes) return nullptr;
    for (int i = 0; i < dims; ++i) {
        PyObject* v = PyLong_FromLongLong(shape[i]);
        if (!v) {
            Py_DECREF(sizes);
            return nullptr;
        }
        PyTuple_SET_ITEM(sizes, i, v);
    }
    PyObject* call[3] = {o, sizes, dtype};
    PyObject* t = PyObject_VectorcallMethod(s_new_empty, call, 2, s_kw_dtype);
    Py_DECREF(sizes);
    if (t && !data_ptr(t, ptr)) Py_CLEAR(t);
    return t;
}

inline void* at(uint64_t v) { return reinterpret_cast<void*>(static_cast<uintptr_t>(v)); }

// Both results of a quantisation, `launch(q, scale)` between their making and their return; None: the library refused.
template <class Launch>
PyObject* results(PyObject* o, const long long* q_shape, const long long* s_shape, int dims, Launch launch) {
    uint64_t q, s;
    PyObject* tq = new_tensor(o, q_shape, dims, g_fp8, &q);
    PyObject* ts = tq ? new_tensor(o, s_shape, dims, g_f32, &s) : nullptr;
    PyObject* out = nullptr;
    if (ts) {
        int st;
        Py_BEGIN_ALLOW_THREADS
        st = launch(at(q), static_cast<float*>(at(s)));
        Py_END_ALLOW_THREADS
        out = st == 0 ? PyTuple_Pack(2, tq, ts) : Py_NewRef(Py_None);
    }
    Py_XDECREF(tq);
    Py_XDECREF(ts);
    return out;
}

// quantize(x, rows or None) -> (q, scale); None: not the hot form, nothing done
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !g_rows) Py_RETURN_NONE;
    Source x;
    int r = source(args[0], &x);
    if (r < 0) return nullptr;
    if (r == 0 || x.dims != 2 || x.shape[1] % 128 != 0 || x.shape[1] == 0 || x.stride[1] != 1) Py_RETURN_NONE;
    if ((r = here(args[0], &x)) < 0) return nullptr;
    if (r == 0) Py_RETURN_NONE;
    long long m = x.shape[0];
    uint64_t rows = 0;
    if (args[1] != Py_None) {
        long long len[3];
        r = hot_tensor(args[1], g_i32);
        if (r == 1) r = numbers(PyObject_GetAttr(args[1], s_shape), len, 3) == 1 ? 1 : PyErr_Occurred() ? -1 : 0;
        if (r == 1) r = on_device(args[1], x.device);
        if (r == 1 && !data_ptr(args[1], &rows)) r = -1;
        if (r < 0) return nullptr;
        m = len[0];
        if (r == 0 || x.shape[0] == 0 || m > INT32_MAX) Py_RETURN_NONE;
    }
    const long long q[2] = {m, x.shape[1]}, s[2] = {m, x.shape[1] / 128};
    return results(args[0], q, s, 2, [&](void* tq, float* ts) {
        return g_rows(at(x.ptr), x.dtype, x.stride[0], static_cast<const int*>(at(rows)), (int)x.shape[0], (int)m, (int)x.shape[1], tq, ts,
                      x.stream);
    });
}

// swiglu_quantize(gate_up) -> (q, scale) or None
PyObject* swiglu_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 1 || !g_swiglu) Py_RETURN_NONE;
    Source x;
    int r = source(args[0], &x);
    if (r < 0) return nullptr;
    if (r == 0 || x.dims != 2 || x.shape[1] % 256 != 0 || x.shape[1] == 0 || x.stride[1] != 1) Py_RETURN_NONE;
    if ((r = here(args[0], &x)) < 0) return nullptr;
    if (r == 0) Py_RETURN_NONE;
    const long long f = x.shape[1] / 2, q[2] = {x.shape[0], f}, s[2] = {x.shape[0], f / 128};
    return results(args[0], q, s, 2, [&](void* tq, float* ts) {
        return g_swiglu(at(x.ptr), x.dtype, x.stride[0], (int)x.shape[0], (int)f, tq, ts, x.stream);
    });
}

// quantize_blocks(w) -> (q, scale) or None
PyObject* quantize_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 1 || !g_blocks) Py_RETURN_NONE;
    Source w;
    int r = source(args[0], &w);
    if (r < 0) return nullptr;
    if (r == 0 || w.dims < 2) Py_RETURN_NONE;
    const int d = w.dims;
    const long long rows = w.shape[d - 2], k = w.shape[d - 1];
    if (k % 128 != 0 || k == 0 || (w.stride[d - 1] != 1 && w.stride[d - 2] != 1)) Py_RETURN_NONE;
    if ((r = here(args[0], &w)) < 0) return nullptr;
    if (r == 0) Py_RETURN_NONE;
    long long s[3] = {w.shape[0], 0, 0};
    s[d - 2] = (rows + 127) / 128;
    s[d - 1] = k / 128;
    return results(args[0], w.shape, s, d, [&](void* tq, float* ts) {
        return g_blocks(at(w.ptr), w.dtype, d == 3 ? (int)w.shape[0] : 1, (int)rows, (int)k, d == 3 ? w.stride[0] : 0, w.stride[d - 2],
                        w.stride[d - 1], tq, ts, w.stream);
    });
}

// grouped(a, b, a_scale, b_scale, offsets, c) -> True: launched; False: not the hot form, or refused
PyObject* grouped(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 6 || !g_grouped) Py_RETURN_FALSE;
    PyObject* const dtypes[6] = {g_fp8, g_fp8, g_f32, g_f32, g_i32, nullptr};
    const int dims[6] = {2, 3, 2, 3, 1, 2};
    long long shape[6][3];
    uint64_t p[6];
    int f16 = 0;
    for (int i = 0; i < 6; ++i) {
        int r;
        if (i < 5) {
            r = hot_tensor(args[i], dtypes[i]);
        } else {
            f16 = attr_is(args[i], s_dtype, g_f16);
            r = f16 < 0 ? -1 : hot_tensor(args[i], f16 ? g_f16 : g_bf16);
        }
        if (r == 1) r = numbers(PyObject_GetAttr(args[i], s_shape), shape[i], 3) == dims[i] ? 1 : PyErr_Occurred() ? -1 : 0;
        if (r == 1 && !data_ptr(args[i], &p[i])) r = -1;
        if (r < 0) return nullptr;
        if (r == 0) Py_RETURN_FALSE;
    }
    const long long m = shape[0][0], k = shape[0][1], e = shape[1][0], nn = shape[1][1], kb = k / 128, nb = (nn + 127) / 128;
    if (shape[1][2] != k || shape[2][0] != m || shape[2][1] != kb || shape[3][0] != e || shape[3][1] != nb || shape[3][2] != kb ||
        shape[4][0] != e + 1 || shape[5][0] != m || shape[5][1] != nn || m > INT32_MAX || k > INT32_MAX || nn > INT32_MAX || e > INT32_MAX)
        Py_RETURN_FALSE;
    long long device;
    void* stream;
    if (!device_and_stream(&device, &stream)) return nullptr;
    for (int i = 0; i < 6; ++i) {
        const int r = on_device(args[i], device);
        if (r < 0) return nullptr;
        if (r == 0) Py_RETURN_FALSE;
    }
    int st;
    Py_BEGIN_ALLOW_THREADS
    st = g_grouped(at(p[0]), at(p[1]), static_cast<float*>(at(p[2])), static_cast<float*>(at(p[3])), static_cast<int*>(at(p[4])), at(p[5]),
                   f16 ? 0 : 1, (int)m, (int)e, (int)nn, (int)k, stream);
    Py_END_ALLOW_THREADS
    return PyBool_FromLong(st == 0);
}

template <class F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {{"setup", fast(setup), METH_FASTCALL, nullptr},
                         {"gemm", fast(gemm), METH_FASTCALL, nullptr},
                         {"fp16_addresses", fast(fp16_addresses), METH_FASTCALL, nullptr},
                         {"setup_fp8", fast(setup_fp8), METH_FASTCALL, nullptr},
                         {"quantize", fast(quantize), METH_FASTCALL, nullptr},
                         {"swiglu_quantize", fast(swiglu_quantize), METH_FASTCALL, nullptr},
                         {"quantize_blocks", fast(quantize_blocks), METH_FASTCALL, nullptr},
                         {"grouped", fast(grouped), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_shape = PyUnicode_InternFromString("shape");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_stride = PyUnicode_InternFromString("stride");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_new_empty = PyUnicode_InternFromString("new_empty");
    s_kw_dtype = s_dtype ? PyTuple_Pack(1, s_dtype) : nullptr;
    if (!s_is_cuda || !s_is_contiguous || !s_dtype || !s_shape || !s_data_ptr || !s_stride || !s_get_device || !s_new_empty || !s_kw_dtype)
        return nullptr;
    return PyModule_Create(&module);
}
