// Reads lists of torch tensors for kernels.adamw_step: the addresses and sizes
// that the C entry point takes, and the checks of types, layout and device. In
// Python each question to each tensor costs about 0.07 us: for 12 layers of a
// model (146 tensors, six lists with 8-bit states) 200 us of calls, as long as
// the update itself takes on the GPU; here 5 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <vector>

namespace {

// The tensors of a list or tuple, or null with an error set.
PyObject** items(PyObject* list, Py_ssize_t* n) {
    if (!PyList_Check(list) && !PyTuple_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "lists or tuples of tensors are wanted");
        return nullptr;
    }
    *n = PySequence_Fast_GET_SIZE(list);
    return PySequence_Fast_ITEMS(list);
}

// read(lists, dtypes, block) -> (addresses, sizes): of k lists of n tensors, as
// k * n unsigned and n signed 64-bit numbers. List i has tensors of dtypes[i],
// all contiguous and on one GPU. Lists 0 to 3 agree in their sizes, the others
// have one value for each `block` of those. No address of lists 0, 2, 3 ...
// (what is written) appears twice.
PyObject* read(PyObject*, PyObject* args) {
    PyObject *lists, *dtypes;
    long long block;
    if (!PyArg_ParseTuple(args, "O!O!L", &PyTuple_Type, &lists, &PyTuple_Type, &dtypes, &block))
        return nullptr;
    const Py_ssize_t k = PyTuple_GET_SIZE(lists);
    if (k < 1 || PyTuple_GET_SIZE(dtypes) != k || block < 1) {
        PyErr_SetString(PyExc_ValueError, "one dtype for each list is wanted");
        return nullptr;
    }
    try {
        Py_ssize_t n = 0;
        if (!items(PyTuple_GET_ITEM(lists, 0), &n)) return nullptr;
        std::vector<uint64_t> at(k * n), written;
        std::vector<int64_t> sizes(n);
        c10::Device device(c10::kCPU);
        for (Py_ssize_t i = 0; i < k; ++i) {
            Py_ssize_t m = 0;
            PyObject** const of = items(PyTuple_GET_ITEM(lists, i), &m);
            if (!of) return nullptr;
            if (m != n) {
                PyErr_SetString(PyExc_ValueError, "the lists differ in length");
                return nullptr;
            }
            PyObject* const kind = PyTuple_GET_ITEM(dtypes, i);
            if (!THPDtype_Check(kind)) {
                PyErr_SetString(PyExc_TypeError, "a dtype is wanted for each list");
                return nullptr;
            }
            const at::ScalarType type = reinterpret_cast<THPDtype*>(kind)->scalar_type;
            for (Py_ssize_t j = 0; j < n; ++j) {
                if (!THPVariable_Check(of[j])) {
                    PyErr_SetString(PyExc_TypeError, "tensors are wanted");
                    return nullptr;
                }
                const at::Tensor& t = THPVariable_Unpack(of[j]);
                if (t.scalar_type() != type) {
                    PyErr_Format(PyExc_TypeError, "list %zd has tensors of %R", i, kind);
                    return nullptr;
                }
                if (i == 0 && j == 0) device = t.device();
                if (!t.device().is_cuda() || t.device() != device) {
                    PyErr_SetString(PyExc_ValueError, "every tensor must be on one GPU");
                    return nullptr;
                }
                if (!t.is_contiguous()) {
                    PyErr_SetString(PyExc_ValueError, "every tensor must be contiguous");
                    return nullptr;
                }
                const int64_t size = t.numel();
                if (i == 0) {
                    sizes[j] = size;
                } else if (size != (i < 4 ? sizes[j] : (sizes[j] + block - 1) / block)) {
                    PyErr_SetString(PyExc_ValueError,
                                    i < 4 ? "a gradient or state differs in size from its parameter"
                                          : "there is one scale for each block of values");
                    return nullptr;
                }
                at[i * n + j] = reinterpret_cast<uint64_t>(size ? t.data_ptr() : nullptr);
                if (size && i != 1) written.push_back(at[i * n + j]);
            }
        }
        std::sort(written.begin(), written.end());
        if (std::adjacent_find(written.begin(), written.end()) != written.end()) {
            PyErr_SetString(PyExc_ValueError, "a parameter or state appears twice");
            return nullptr;
        }
        return Py_BuildValue("(y#y#)", reinterpret_cast<const char*>(at.data()),
                             static_cast<Py_ssize_t>(at.size() * 8),
                             reinterpret_cast<const char*>(sizes.data()),
                             static_cast<Py_ssize_t>(sizes.size() * 8));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"read", read, METH_VARARGS, "read(lists, dtypes, block) -> (addresses, sizes)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists() { return PyModule_Create(&module); }
