// What the host paths of the convolutions (dcn_torch.cpp) and of the sequence operators (seq_torch.cpp) share.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <nvtx3/nvToolsExt.h>

#include <cstdlib>
#include <cstring>
#include <string>

#include "../../include/dcn.h"

namespace dcn_host {

using at::Tensor;

extern PyObject* g_error;               // the package's DcnError
extern PyMethodDef sequence_methods[];

struct DcnFailure {
    std::string text;
};
[[noreturn]] inline void fail(const std::string& text) { throw DcnFailure{text}; }

inline void check(int status, const char* what) {
    if (status != DCN_OK)
        fail(std::string(what) + " failed: " + dcn_status_string(status) + " (status " + std::to_string(status) + ")");
}

inline bool env_set(const char* name) {
    const char* e = getenv(name);
    return e != nullptr && e[0] != '\0' && strcmp(e, "0") != 0;
}

struct Range {
    bool on;
    explicit Range(const char* name) : on(env_set("DCN_NVTX")) {
        if (on) nvtxRangePushA(name);
    }
    ~Range() {
        if (on) nvtxRangePop();
    }
};

inline std::string dtype_name(const Tensor& t) { return std::string("torch.") + torch::getTHPDtype(t.scalar_type())->name; }

inline Tensor tensor_arg(PyObject* o, const char* name, bool optional = false) {
    if (optional && o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a Tensor, not %s", name, Py_TYPE(o)->tp_name);
        throw python_error();
    }
    return THPVariable_Unpack(o);
}

inline int64_t int_arg(PyObject* o) {
    PyObject* i = PyNumber_Index(o);
    if (i == nullptr) throw python_error();
    const int64_t v = PyLong_AsLongLong(i);
    Py_DECREF(i);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

inline void count_arg(Py_ssize_t n, Py_ssize_t lo, Py_ssize_t hi) {
    if (n >= lo && n <= hi) return;
    PyErr_Format(PyExc_TypeError, "expected %zd to %zd arguments, got %zd", lo, hi, n);
    throw python_error();
}

#define DCN_FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL

}  // namespace dcn_host
