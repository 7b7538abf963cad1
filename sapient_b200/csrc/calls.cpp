// Python's way to the calls on fp8 rows and logits in device memory, without the one to two microseconds that ctypes takes to convert
// 9 to 16 arguments: from Python a call of few rows is bound by the host (1 row of 4096 columns, norm: 4.5 us through ctypes, of which
// the launch is 1.9; GPU time 2 to 3). bind() takes the library's functions by address, so that this module links with nothing;
// each call gives back their status.
#define Py_LIMITED_API 0x030A0000
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <tuple>
#include <utility>

#include "../../include/sapient_cuda.h"

namespace {

bool get(PyObject* o, int64_t& v) {
    v = PyLong_AsLongLong(o);
    return v != -1 || !PyErr_Occurred();
}
bool get(PyObject* o, int32_t& v) {
    int64_t w;
    if (!get(o, w)) return false;
    v = (int32_t)w;
    if (v == w) return true;
    PyErr_SetString(PyExc_OverflowError, "argument does not fit 32 bits");
    return false;
}
bool get(PyObject* o, float& v) {
    const double d = PyFloat_AsDouble(o);
    v = (float)d;
    return d != -1.0 || !PyErr_Occurred();
}
template <typename T>
bool get(PyObject* o, T*& p) {  // an address; None: null
    p = nullptr;
    if (o == Py_None) return true;
    PyObject* const i = PyNumber_Index(o);
    if (!i) return false;
    p = static_cast<T*>(PyLong_AsVoidPtr(i));
    Py_DECREF(i);
    return p || !PyErr_Occurred();
}

template <typename... A, size_t... I>
PyObject* call_with(int32_t (*f)(A...), PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<A...> a;
    if (!(get(args[I], std::get<I>(a)) && ...)) return nullptr;
    int32_t status;
    Py_BEGIN_ALLOW_THREADS
    status = f(std::get<I>(a)...);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}
template <typename... A>
PyObject* call(int32_t (*f)(A...), PyObject* const* args, Py_ssize_t n) {
    if (!f) {
        PyErr_SetString(PyExc_RuntimeError, "bind() has not been called");
        return nullptr;
    }
    if (n != (Py_ssize_t)sizeof...(A)) {
        PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd expected", n, (Py_ssize_t)sizeof...(A));
        return nullptr;
    }
    return call_with(f, args, std::index_sequence_for<A...>());
}

#define CALLS(X) X(rms_norm_fp8) X(swiglu_fp8) X(quant_fp8) X(matmul_fp8) X(logprobs) X(cache_fp8_append) X(cache_fp8_read) X(attention_fp8)
#define DEFINE(name)                                        \
    decltype(&sp_cuda_##name##_dev) f_##name = nullptr;     \
    PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n) { return call(f_##name, args, n); }
CALLS(DEFINE)

PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 8) {
        PyErr_SetString(PyExc_TypeError, "eight addresses expected");
        return nullptr;
    }
    Py_ssize_t i = 0;
#define BIND(name)                                                          \
    {                                                                       \
        void* p = nullptr;                                                  \
        if (!get(args[i++], p)) return nullptr;                             \
        f_##name = reinterpret_cast<decltype(f_##name)>(p);                 \
    }
    CALLS(BIND)
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr},
PyMethodDef methods[] = {CALLS(METHOD){"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
