// What the modules of calls have in common: arguments as Python gives them, the checks of tensors, launches without the interpreter's lock, exceptions.
#pragma once
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <limits>
#include <stdexcept>
#include <string>

namespace {

PyObject* kernel_error;          // exception of a launch that fails, set by bind()

struct Refused : std::invalid_argument {
    using std::invalid_argument::invalid_argument;
};
struct Raised {};                // a Python exception is set

// ---- arguments ------------------------------------------------------------------------------------------------------------------
constexpr int MOST = 32;
struct Signature {
    const char* name;
    int positional, n;           // the first `positional` may be given by position; all by name
    const char* names[MOST];
    PyObject* interned[MOST] = {};
    void intern() {
        for (int i = 0; i < n; i++) interned[i] = PyUnicode_InternFromString(names[i]);
    }
};

void parse(const Signature& s, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames, PyObject** out) {
    std::fill(out, out + s.n, nullptr);
    if (nargs > s.positional) {
        PyErr_Format(PyExc_TypeError, "%s() takes %d positional arguments but %zd were given", s.name, s.positional, nargs);
        throw Raised();
    }
    std::copy(args, args + nargs, out);
    const Py_ssize_t more = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    int hint = (int)nargs;
    for (Py_ssize_t k = 0; k < more; k++) {
        PyObject* name = PyTuple_GET_ITEM(kwnames, k);
        int at = -1;
        for (int i = 0; i < s.n && at < 0; i++) {      // names come in about the signature's order
            const int j = (hint + i) % s.n;
            if (s.interned[j] == name) at = j;
        }
        for (int i = 0; i < s.n && at < 0; i++)
            if (PyUnicode_Compare(name, s.interned[i]) == 0) at = i;
        if (at < 0 || out[at]) {
            PyErr_Format(PyExc_TypeError, at < 0 ? "%s() got an unexpected keyword argument '%U'" : "%s() got multiple values for argument '%U'", s.name, name);
            throw Raised();
        }
        out[at] = args[nargs + k];
        hint = at + 1;
    }
}

PyObject* required(const Signature& s, PyObject** a, int i) {
    if (!a[i]) {
        PyErr_Format(PyExc_TypeError, "%s() missing required argument: '%s'", s.name, s.names[i]);
        throw Raised();
    }
    return a[i];
}
bool given(PyObject* o) { return o && o != Py_None; }
long as_long(PyObject* o, long other) {
    if (!o) return other;
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return std::min(std::max(v, -(1l << 31)), (1l << 31) - 1);
}
double as_double(PyObject* o, double other) {
    if (!o) return other;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}
bool as_bool(PyObject* o, bool other) {
    if (!o) return other;
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v;
}
struct Ref {                     // an attribute, held
    PyObject* o;
    Ref(PyObject* of, PyObject* name) : o(PyObject_GetAttr(of, name)) {
        if (!o) throw Raised();
    }
    ~Ref() { Py_DECREF(o); }
};
template <typename T>
T as_struct(PyObject* o) {       // a ctypes structure's bytes
    Py_buffer b;
    if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE)) throw Raised();
    const bool fits = b.len == (Py_ssize_t)sizeof(T);
    T v;
    if (fits) std::memcpy(&v, b.buf, sizeof(T));
    PyBuffer_Release(&b);
    if (!fits) {
        PyErr_SetString(PyExc_TypeError, "a structure of another size");
        throw Raised();
    }
    return v;
}

// ---- tensors --------------------------------------------------------------------------------------------------------------------
std::string told(const at::Tensor& t) {
    std::string s = "(";
    for (auto n : t.sizes()) s += std::to_string(n) + ",";
    return s + ") " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}
[[noreturn]] void refuse(const Signature& s, const std::string& what) { throw Refused(std::string(s.name) + ": " + what); }

const at::Tensor& tensor(const Signature& s, PyObject* o, const char* name) {
    if (!given(o)) refuse(s, std::string(name) + " is missing");
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s(): %s must be a tensor, not %s", s.name, name, Py_TYPE(o)->tp_name);
        throw Raised();
    }
    return THPVariable_Unpack(o);
}
// A tensor of the type, on the device, in one piece.
const at::Tensor& piece(const Signature& s, PyObject* o, const char* name, at::ScalarType type, c10::Device dev) {
    const at::Tensor& t = tensor(s, o, name);
    if (t.scalar_type() != type || t.device() != dev || !t.is_contiguous()) refuse(s, std::string(name) + " " + told(t));
    return t;
}
template <typename... N>
const at::Tensor& shaped(const Signature& s, PyObject* o, const char* name, at::ScalarType type, c10::Device dev, N... sizes) {
    const at::Tensor& t = piece(s, o, name, type, dev);
    const int64_t want[] = {(int64_t)sizes...};
    if (!t.sizes().equals(want)) refuse(s, std::string(name) + " " + told(t));
    return t;
}
const at::Tensor& vector(const Signature& s, PyObject* o, const char* name, at::ScalarType type, c10::Device dev, int64_t least) {
    const at::Tensor& t = piece(s, o, name, type, dev);
    if (t.dim() != 1 || t.numel() < least) refuse(s, std::string(name) + " " + told(t));
    return t;
}
// Rows are a dimension of the merge's grid.
void few_rows(const Signature& s, long n) {
    if (n > 65535) refuse(s, std::to_string(n) + " rows");
}
// From a row to the next of rows that stand beside one another.
long row_step(const Signature& s, const at::Tensor& t, const char* name) {
    const long step = t.size(0) > 1 ? t.stride(0) : t.size(1);
    if (step < t.size(1) || step > (1l << 31) - 1) refuse(s, std::string(name) + " " + told(t) + " with rows " + std::to_string(step) + " apart");
    return step;
}
// read or written 16 bytes at a time
const at::Tensor& wide(const Signature& s, const at::Tensor& t, const char* name) {
    if ((uintptr_t)t.data_ptr() & 15) refuse(s, std::string(name) + " is not on a 16-byte boundary");
    return t;
}
constexpr at::ScalarType F32 = at::kFloat, F64 = at::kDouble, I32 = at::kInt, F16 = at::kHalf, B16 = at::kBFloat16;

c10::Device on_gpu(const Signature& s, const at::Tensor& t) {
    if (!t.is_cuda()) refuse(s, "tensors on " + t.device().str());
    return t.device();
}
void launched(const Signature& s, int rc) {
    if (rc == 0) return;
    PyErr_Format(kernel_error, "%s failed with CUDA error %d", s.name, rc);
    throw Raised();
}
// Other threads run while memory is found and kernels are launched: either may have to wait, for blocks that are given back or for room in the launch queue.  What the call holds
// (its arguments, which the caller holds) stays.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
int unlocked(c10::Device dev, F launch) {
    const Unlocked lock;
    const c10::cuda::CUDAGuard guard(dev);
    return launch(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}
at::Tensor floats(c10::Device dev, long n) { return at::empty({n}, at::TensorOptions().dtype(F32).device(dev)); }
int sms_of(c10::Device dev) {
    static int sms[64] = {};
    int& n = sms[dev.index() & 63];
    if (!n && (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev.index()) != cudaSuccess || n < 1)) n = 148;
    return n;
}

// ---- a call ---------------------------------------------------------------------------------------------------------------------
template <const Signature& S, bool (*bound)(), typename F>
PyObject* called(F f, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    try {
        PyObject* a[MOST];
        parse(S, args, nargs, kwnames, a);
        if (!bound()) {
            PyErr_SetString(PyExc_RuntimeError, "the kernel library has not been bound");
            throw Raised();
        }
        return f(a);
    } catch (const Raised&) {
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_SetString(type ? type : PyExc_MemoryError, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
PyObject* none() { Py_RETURN_NONE; }

}  // namespace
