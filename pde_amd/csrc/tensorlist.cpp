// Host side of the operators over many tensors: reads addresses, lengths and types of a list of torch tensors into the host arrays
// that include/pinnjet.h's entry points take, and checks them on the way.  From Python the same takes 0.6 us a tensor, which for the
// 240 tensors of 24 nets is five times the step itself; here it is 0.02.
//
// A Python extension module without GPU code; it knows nothing of a device beyond comparing tensors' devices.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <stdint.h>

namespace {

int code_of(const at::Tensor &t)                // PINN_F32, PINN_BF16, PINN_F16; -1: none of them
{
    switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
    }
}

bool tensor_at(PyObject *list, Py_ssize_t i, const char *what)
{
    if (THPVariable_Check(PyList_GET_ITEM(list, i))) return true;
    PyErr_Format(PyExc_TypeError, "%s %zd is a %s, a tensor is needed", what, i, Py_TYPE(PyList_GET_ITEM(list, i))->tp_name);
    return false;
}

bool plain(const at::Tensor &t) { return t.layout() == at::kStrided && !t.is_neg() && !t.is_conj(); }

// same order in memory: strides may differ where a dimension has one element
bool same_order(const at::Tensor &a, const at::Tensor &b)
{
    if (a.is_contiguous() && b.is_contiguous()) return true;
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

// no gaps and no overlaps
bool dense(const at::Tensor &t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

template <class F>
PyObject *guarded(F f)
{
    try {
        return f();
    } catch (const std::exception &e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// gather(params, numel, dtype, p, g, count) -> (gradients found, [indices whose gradient lies in another order than its parameter], whether
// a parameter lies elsewhere than p said before)
// numel, dtype: int64 and int32 arrays, what the plan was made for; p, g: uint64 arrays that take the addresses (g: 0 without a gradient);
// count: int64 array, the gradient's length or 0.  Arrays are given by their address.  The parameters that have a gradient count as written to.
PyObject *gather(PyObject *, PyObject *args)
{
    PyObject *params;
    unsigned long long a_numel, a_dtype, a_p, a_g, a_count;
    if (!PyArg_ParseTuple(args, "O!KKKKK", &PyList_Type, &params, &a_numel, &a_dtype, &a_p, &a_g, &a_count)) return nullptr;
    const auto found = guarded([&]() -> PyObject * {
        const int64_t *numel = (const int64_t *)(uintptr_t)a_numel;
        const int32_t *dtype = (const int32_t *)(uintptr_t)a_dtype;
        uint64_t *p_out = (uint64_t *)(uintptr_t)a_p, *g_out = (uint64_t *)(uintptr_t)a_g;
        int64_t *count = (int64_t *)(uintptr_t)a_count;
        const Py_ssize_t n = PyList_GET_SIZE(params);
        PyObject *other = PyList_New(0);
        if (!other) return nullptr;
        Py_ssize_t given = 0;
        bool moved = false;
        c10::Device device(c10::DeviceType::CPU);
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (!tensor_at(params, i, "parameter")) { Py_DECREF(other); return nullptr; }
            const at::Tensor &p = THPVariable_Unpack(PyList_GET_ITEM(params, i));
            if (i == 0) device = p.device();
            if (!plain(p) || code_of(p) != dtype[i] || p.numel() != numel[i] || p.device() != device || !dense(p)) {
                PyErr_Format(PyExc_ValueError, "parameter %zd is not what it was when the optimizer was made (type, size, device or layout)", i);
                Py_DECREF(other);
                return nullptr;
            }
            const uint64_t at = (uint64_t)(uintptr_t)p.data_ptr();
            moved |= p_out[i] != at;
            p_out[i] = at;
            g_out[i] = 0;
            count[i] = 0;
            const at::Tensor &g = p.grad();
            if (!g.defined()) continue;
            if (!plain(g) || g.scalar_type() != p.scalar_type() || g.device() != device || !g.sizes().equals(p.sizes())) {
                PyErr_Format(PyExc_ValueError, "the gradient of parameter %zd is not a dense tensor of its parameter's type, shape and device", i);
                Py_DECREF(other);
                return nullptr;
            }
            if (numel[i] == 0) continue;
            ++given;
            count[i] = numel[i];
            if (same_order(p, g)) {
                g_out[i] = (uint64_t)(uintptr_t)g.data_ptr();
            } else {
                PyObject *k = PyLong_FromSsize_t(i);
                const bool bad = !k || PyList_Append(other, k) != 0;
                Py_XDECREF(k);
                if (bad) { Py_DECREF(other); return nullptr; }
            }
        }
        for (Py_ssize_t i = 0; i < n; ++i)
            if (count[i]) {
                const at::Tensor &p = THPVariable_Unpack(PyList_GET_ITEM(params, i));
                if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
            }
        return Py_BuildValue("(nNO)", given, other, moved ? Py_True : Py_False);
    });
    if (!found && a_p && PyList_GET_SIZE(params) > 0) *(uint64_t *)(uintptr_t)a_p = 0;   // the next call says "moved" again
    return found;
}

// describe(tensors, of_grads, x, numel, dtype) -> (how many, [(place in the arrays, index) of those that are neither contiguous nor another
// order of the same memory], index of their GPU, elements in all); of_grads: the gradients of those tensors that have one, 2: and they
// count as written to
PyObject *describe(PyObject *, PyObject *args)
{
    PyObject *list;
    int of_grads;
    unsigned long long a_x, a_numel, a_dtype;
    if (!PyArg_ParseTuple(args, "O!iKKK", &PyList_Type, &list, &of_grads, &a_x, &a_numel, &a_dtype)) return nullptr;
    return guarded([&]() -> PyObject * {
        uint64_t *x = (uint64_t *)(uintptr_t)a_x;
        int64_t *numel = (int64_t *)(uintptr_t)a_numel;
        int32_t *dtype = (int32_t *)(uintptr_t)a_dtype;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        PyObject *other = PyList_New(0);
        if (!other) return nullptr;
        c10::Device device(c10::DeviceType::CPU);
        Py_ssize_t k = 0;
        int64_t total = 0;
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (!tensor_at(list, i, "tensor")) { Py_DECREF(other); return nullptr; }
            const at::Tensor &given = THPVariable_Unpack(PyList_GET_ITEM(list, i));
            const at::Tensor &t = of_grads ? given.grad() : given;
            if (!t.defined()) continue;
            if (k == 0) device = t.device();
            if (!t.is_cuda() && !t.is_meta() && t.device() == device) {
                static PyObject *native_error = nullptr;
                if (!native_error) {
                    PyObject *m = PyImport_ImportModule("pde_amd._native");
                    native_error = m ? PyObject_GetAttrString(m, "NativeError") : nullptr;
                    Py_XDECREF(m);
                }
                if (native_error)
                    PyErr_Format(native_error, "tensor %zd is on %s: pde_amd needs an AMD GPU; there is no CPU fallback", i, t.device().str().c_str());
                Py_DECREF(other);
                return nullptr;
            }
            if (!plain(t) || code_of(t) < 0 || t.device() != device) {
                PyErr_Format(PyExc_ValueError, "tensor %zd: dense float32, bfloat16 or float16 tensors on one device are needed, got %s on %s (the first is on %s)", i,
                             !plain(t) ? "another layout" : c10::toString(t.scalar_type()), t.device().str().c_str(), device.str().c_str());
                Py_DECREF(other);
                return nullptr;
            }
            x[k] = t.numel() ? (uint64_t)(uintptr_t)t.data_ptr() : 0;
            numel[k] = t.numel();
            total += t.numel();
            dtype[k] = code_of(t);
            if (!dense(t)) {
                PyObject *pair = Py_BuildValue("(nn)", k, i);
                const bool bad = !pair || PyList_Append(other, pair) != 0;
                Py_XDECREF(pair);
                if (bad) { Py_DECREF(other); return nullptr; }
            }
            ++k;
        }
        if (of_grads == 2)
            for (Py_ssize_t i = 0; i < n; ++i) {
                const at::Tensor &g = THPVariable_Unpack(PyList_GET_ITEM(list, i)).grad();
                if (g.defined() && !g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
            }
        if (k == 0) return Py_BuildValue("(nNOi)", k, other, Py_None, 0);
        return Py_BuildValue("(nNnL)", k, other, (Py_ssize_t)device.index(), (long long)total);
    });
}

PyMethodDef methods[] = {{"gather", gather, METH_VARARGS, nullptr},
                         {"describe", describe, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensorlist", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensorlist()
{
    PyObject *m = PyModule_Create(&module);
    // which torch's tensors this was compiled for: they are read by its headers
    if (m && PyModule_AddStringConstant(m, "torch_version", PINN_TORCH) != 0) Py_CLEAR(m);
    return m;
}
