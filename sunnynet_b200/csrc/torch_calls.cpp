// The parts of kernels.py that cost more in Python than their kernels take.
//
// read: the lists of torch tensors of an AdamW step, as the addresses and sizes
// that the C entry point takes, and the checks of types, layout and device. In
// Python each question to each tensor costs about 0.07 us: for 12 layers of a
// model (146 tensors, six lists with 8-bit states) 200 us of calls, as long as
// the update itself takes on the GPU; here 25 us.
//
// layer_norm: the call and its node in the autograd graph. A call and its
// gradients take 75 us of the host's time (torch's own layer norm 70), as a
// Function in Python 110; a call without a graph 8 us instead of 11.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "sn_abi.h"

namespace {

// The library's entry points (it is loaded by ctypes).
struct {
    decltype(&sn_abi_layer_norm) norm = nullptr;
    decltype(&sn_abi_layer_norm_bwd) norm_bwd = nullptr;
    decltype(&sn_abi_layer_norm_bwd_ws) norm_bwd_ws = nullptr;
    decltype(&sn_abi_last_error) last_error = nullptr;
} lib;

std::string last_error() {
    char text[512] = "";
    lib.last_error(text, sizeof text);
    return text;
}

int32_t code(at::ScalarType t) {
    return t == at::kFloat ? SN_F32 : t == at::kBFloat16 ? SN_BF16 : SN_F16;
}

// t as rows of D values at one stride; ld: that stride in elements.
at::Tensor rows_of(const at::Tensor& t, int64_t D, int64_t* ld) {
    *ld = D;
    if (t.is_contiguous()) return t;
    at::Tensor r = t.reshape({-1, D});  // a view wherever the rows lie at one stride
    if (r.stride(1) != 1 || (r.size(0) > 1 && r.stride(0) < D))
        return r.contiguous();  // among these what a sum's gradient broadcasts
    *ld = std::max(r.stride(0), D);
    return r;
}

void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* stream_of(const at::Tensor& t) {
    return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

int32_t weight_code(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b) {
    return code(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
}

// y; x, w, b: what was given, made rows and contiguous. stats: (2, rows), or none.
at::Tensor norm_forward(at::Tensor& x, at::Tensor& w, at::Tensor& b, double eps,
                        at::Tensor* stats) {
    const int64_t D = x.size(-1), rows = x.numel() / D;
    at::Tensor y = x.is_contiguous() ? at::empty_like(x) : at::empty(x.sizes(), x.options());
    int64_t ld;
    x = rows_of(x, D, &ld);
    if (w.defined()) w = w.contiguous();
    if (b.defined()) b = b.contiguous();
    float* mean = nullptr;
    if (stats) {
        *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
        mean = stats->data_ptr<float>();
    }
    const int rc = lib.norm(address(x), ld, address(w), address(b), address(y), mean,
                            stats ? mean + rows : nullptr, code(x.scalar_type()),
                            weight_code(x, w, b), rows, (int32_t)D, (float)eps, stream_of(x));
    TORCH_CHECK(rc == SN_OK, "layer_norm: ", last_error());
    return y;
}

struct Norm : torch::autograd::Function<Norm> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x_,
                              const std::optional<at::Tensor>& w_,
                              const std::optional<at::Tensor>& b_, double eps) {
        at::Tensor x = x_, w = w_.value_or(at::Tensor()), b = b_.value_or(at::Tensor()), stats;
        const int32_t wcode = weight_code(x, w, b);
        const bool has_w = w.defined(), has_b = b.defined();
        at::Tensor y = norm_forward(x, w, b, eps, &stats);
        ctx->save_for_backward({x, w, stats});
        ctx->saved_data["call"] = (int64_t)(wcode | has_w << 4 | has_b << 5);
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        // with create_graph: its own gradient is not there
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm can be differentiated once");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &stats = saved[2], &dy = grads[0];
        const int64_t call = ctx->saved_data["call"].toInt();
        const int32_t wcode = (int32_t)(call & 15);
        const bool has_w = call >> 4 & 1, has_b = call >> 5 & 1;
        const bool want_x = ctx->needs_input_grad(0), want_w = has_w && ctx->needs_input_grad(1),
                   want_b = has_b && ctx->needs_input_grad(1 + has_w);
        const int64_t D = dy.size(-1), rows = dy.numel() / D;
        int64_t ldx, ldg;
        const at::Tensor xr = rows_of(x, D, &ldx), g = rows_of(dy, D, &ldg);
        const int32_t c = code(x.scalar_type());
        at::Tensor dx, dw, db, ws;
        if (want_x) dx = at::empty(dy.sizes(), dy.options());
        const auto wide = dy.options().dtype(wcode == SN_F32 ? at::kFloat : dy.scalar_type());
        if (want_w) dw = at::empty({D}, wide);
        if (want_b) db = at::empty({D}, wide);
        int64_t need = 0;
        if (want_w || want_b) {
            need = lib.norm_bwd_ws(rows, (int32_t)D, c);
            ws = at::empty({need}, dy.options().dtype(at::kByte));
        }
        const float* mean = stats.data_ptr<float>();
        const int rc = lib.norm_bwd(address(g), ldg, address(xr), ldx, address(w), mean,
                                    mean + rows, address(dx), address(dw), address(db),
                                    address(ws), need, c, wcode, rows, (int32_t)D, stream_of(x));
        TORCH_CHECK(rc == SN_OK, "layer_norm_bwd: ", last_error());
        return {dx, dw, db, at::Tensor()};
    }
};

// A tensor or None (an undefined one); false with an error set for others.
bool tensor_of(PyObject* o, at::Tensor* t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "layer_norm: tensors are wanted");
        return false;
    }
    *t = THPVariable_Unpack(o);
    return true;
}

// layer_norm(x, weight, bias, eps), the arguments as kernels.layer_norm checked them.
PyObject* layer_norm(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *xo, *wo, *bo;
    double eps;
    if (!PyArg_ParseTuple(args, "OOOd", &xo, &wo, &bo, &eps)) return nullptr;
    at::Tensor x, w, b;
    if (!tensor_of(xo, &x) || !tensor_of(wo, &w) || !tensor_of(bo, &b)) return nullptr;
    // (neither path carries a tangent on)
    const auto moves = [](const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); };
    TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
                  (moves(x) || moves(w) || moves(b))),
                "layer_norm has no forward-mode derivative");
    const auto grows = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
    if (at::GradMode::is_enabled() && (grows(x) || grows(w) || grows(b)))
        return THPVariable_Wrap(
            Norm::apply(x, w.defined() ? std::optional<at::Tensor>(w) : std::nullopt,
                        b.defined() ? std::optional<at::Tensor>(b) : std::nullopt, eps));
    return THPVariable_Wrap(norm_forward(x, w, b, eps, nullptr));
    END_HANDLE_TH_ERRORS
}

// use(layer_norm, layer_norm_bwd, layer_norm_bwd_ws, last_error): their addresses.
PyObject* use(PyObject*, PyObject* args) {
    unsigned long long p[4];
    if (!PyArg_ParseTuple(args, "KKKK", p, p + 1, p + 2, p + 3)) return nullptr;
    lib.norm = reinterpret_cast<decltype(lib.norm)>(p[0]);
    lib.norm_bwd = reinterpret_cast<decltype(lib.norm_bwd)>(p[1]);
    lib.norm_bwd_ws = reinterpret_cast<decltype(lib.norm_bwd_ws)>(p[2]);
    lib.last_error = reinterpret_cast<decltype(lib.last_error)>(p[3]);
    Py_RETURN_NONE;
}

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
// have one value for each `block` of those. No memory of lists 0, 2, 3 ...
// (what is written) belongs to two of their tensors.
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
        std::vector<uint64_t> at(k * n);
        std::vector<std::pair<uint64_t, uint64_t>> written;  // begin and end
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
                if (size && i != 1)
                    written.emplace_back(at[i * n + j], at[i * n + j] + size * t.element_size());
            }
        }
        std::sort(written.begin(), written.end());
        if (std::adjacent_find(written.begin(), written.end(), [](const auto& a, const auto& b) {
                return b.first < a.second;
            }) != written.end()) {
            PyErr_SetString(PyExc_ValueError, "a parameter or state appears twice, or overlaps another");
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

// read_grads(list, apart) -> (addresses, sizes, types, index of the GPU): tensors
// of float types on one GPU, whose values fill one run of memory in any order;
// with `apart`, no memory belongs to two of them.
PyObject* read_grads(PyObject*, PyObject* args) {
    PyObject* list;
    int apart;
    if (!PyArg_ParseTuple(args, "Op", &list, &apart)) return nullptr;
    try {
        Py_ssize_t n = 0;
        PyObject** const of = items(list, &n);
        if (!of) return nullptr;
        std::vector<uint64_t> at(n);
        std::vector<int64_t> sizes(n);
        std::vector<int32_t> types(n);
        std::vector<std::pair<uint64_t, uint64_t>> written;
        c10::Device device(c10::kCPU);
        for (Py_ssize_t j = 0; j < n; ++j) {
            if (!THPVariable_Check(of[j])) {
                PyErr_SetString(PyExc_TypeError, "tensors are wanted");
                return nullptr;
            }
            const at::Tensor& t = THPVariable_Unpack(of[j]);
            if (t.layout() != at::kStrided) {
                PyErr_SetString(PyExc_ValueError, "sparse gradients are not supported");
                return nullptr;
            }
            const at::ScalarType type = t.scalar_type();
            if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) {
                PyErr_SetString(PyExc_TypeError, "gradients are of float32, bfloat16 or float16");
                return nullptr;
            }
            if (j == 0) device = t.device();
            if (!t.device().is_cuda() || t.device() != device) {
                PyErr_SetString(PyExc_ValueError, "every gradient must be on one GPU");
                return nullptr;
            }
            if (!t.is_non_overlapping_and_dense()) {
                PyErr_SetString(PyExc_ValueError, "a gradient's values must fill one run of memory");
                return nullptr;
            }
            sizes[j] = t.numel();
            types[j] = code(type);
            at[j] = reinterpret_cast<uint64_t>(sizes[j] ? t.data_ptr() : nullptr);
            if (apart && sizes[j]) written.emplace_back(at[j], at[j] + sizes[j] * t.element_size());
        }
        std::sort(written.begin(), written.end());
        if (std::adjacent_find(written.begin(), written.end(), [](const auto& a, const auto& b) {
                return b.first < a.second;
            }) != written.end()) {
            PyErr_SetString(PyExc_ValueError, "a gradient appears twice, or overlaps another");
            return nullptr;
        }
        return Py_BuildValue("(y#y#y#i)", reinterpret_cast<const char*>(at.data()),
                             static_cast<Py_ssize_t>(n * 8), reinterpret_cast<const char*>(sizes.data()),
                             static_cast<Py_ssize_t>(n * 8), reinterpret_cast<const char*>(types.data()),
                             static_cast<Py_ssize_t>(n * 4), n ? (int)device.index() : -1);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"read", read, METH_VARARGS, "read(lists, dtypes, block) -> (addresses, sizes)"},
    {"read_grads", read_grads, METH_VARARGS,
     "read_grads(list, apart) -> (addresses, sizes, types, index of the GPU)"},
    {"layer_norm", layer_norm, METH_VARARGS, "layer_norm(x, weight, bias, eps) -> y"},
    {"use", use, METH_VARARGS, "use(addresses of the library's entry points)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls() { return PyModule_Create(&module); }
