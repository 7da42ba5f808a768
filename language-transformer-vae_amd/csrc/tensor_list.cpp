// Host helper of grad_ops: walks Python lists of tensors and writes the table that lvae_clip_grads takes.
//
// A model has hundreds of gradients, and asking each for its address, size, type, device and layout from Python costs
// about 0.15 us a question: 400 us for 264 tensors and their destinations, several times what the GPU needs for them.
// Here it is a few microseconds.  No tensor arithmetic, no state.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>

#include "../../include/lvae.h"
#include "tensor_checks.h"

namespace {

int code(at::ScalarType t) {
    return t == at::kFloat ? LVAE_F32 : t == at::kBFloat16 ? LVAE_BF16 : t == at::kHalf ? LVAE_F16 : -1;
}

// the tensor at list[i], checked; NULL with a Python error set otherwise
const at::Tensor* tensor_at(PyObject* list, Py_ssize_t i, const char* name, const at::Device* device) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s[%zd] must be a torch.Tensor", name, i);
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (const char* why = t.defined() ? more_than_memory(t) : nullptr) {
        PyErr_Format(PyExc_RuntimeError, "%s[%zd] %s", name, i, why);
        return nullptr;
    }
    if (!t.defined() || !t.is_cuda()) {
        PyErr_Format(PyExc_RuntimeError, "%s[%zd] is not on a GPU: the HIP path needs GPU tensors (no CPU fallback)", name, i);
        return nullptr;
    }
    if (t.layout() != at::kStrided || code(t.scalar_type()) < 0) {
        PyErr_Format(PyExc_TypeError, "%s[%zd] must be a dense float32, bfloat16 or float16 tensor", name, i);
        return nullptr;
    }
    if (device && t.device() != *device) {
        PyErr_Format(PyExc_ValueError, "%s[%zd] is on another device than the first tensor: one device a call", name, i);
        return nullptr;
    }
    return &t;
}

// whether elements of the tensor share memory, as those of a broadcast one do
bool repeats(const at::Tensor& t) {
    for (int64_t k = 0; k < t.dim(); ++k)
        if (t.size(k) > 1 && t.stride(k) == 0) return t.numel() > 0;
    return false;
}

// table(src, dst or None, whether they will be written) -> (table as bytes, device index, whether one requires grad, [places that need a dense copy])
PyObject* table(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *src, *dst;
    int writes = 0;
    if (!PyArg_ParseTuple(args, "O!Op", &PyList_Type, &src, &dst, &writes)) return nullptr;
    if (being_traced()) {
        PyErr_SetString(PyExc_RuntimeError, "the norm of gradients and their clipping cannot be traced: a trace would not hold their kernels");
        return nullptr;
    }
    const bool out = dst != Py_None;
    const Py_ssize_t n = PyList_GET_SIZE(src);
    if (out && (!PyList_Check(dst) || PyList_GET_SIZE(dst) != n)) {
        PyErr_SetString(PyExc_ValueError, "as many tensors in out as gradients are wanted");
        return nullptr;
    }
    PyObject* bytes = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(lvae_grad_entry));
    if (!bytes) return nullptr;
    PyObject* odd = PyList_New(0);
    if (!odd) {
        Py_DECREF(bytes);
        return nullptr;
    }
    lvae_grad_entry* e = (lvae_grad_entry*)PyBytes_AS_STRING(bytes);
    bool wants_grad = false, ok = true;
    at::Device device(at::kCPU);
    try {
        for (Py_ssize_t i = 0; ok && i < n; ++i) {
            const at::Tensor* s = tensor_at(src, i, "grads", i ? &device : nullptr);
            ok = s != nullptr;
            if (!ok) break;
            if (i == 0) device = s->device();
            wants_grad = wants_grad || s->requires_grad();
            // a negated view (the imaginary part of a conjugate) holds the other sign in memory
            bool plain = (s->is_contiguous() || s->is_non_overlapping_and_dense()) && !s->is_neg();
            const at::Tensor* d = nullptr;
            if (out) {
                d = tensor_at(dst, i, "out", &device);
                ok = d != nullptr;
                if (!ok) break;
                wants_grad = wants_grad || d->requires_grad();
                if (s->sizes() != d->sizes()) {
                    PyErr_Format(PyExc_ValueError, "out[%zd] has another shape than grads[%zd]", i, i);
                    ok = false;
                    break;
                }
                plain = plain && !d->is_neg() && (s->strides() == d->strides() || (s->is_contiguous() && d->is_contiguous()));
            }
            if (writes && !plain && repeats(d ? *d : *s)) {
                PyErr_Format(PyExc_RuntimeError, "%s[%zd] is broadcast: several of its elements are one place in memory", d ? "out" : "grads", i);
                ok = false;
                break;
            }
            e[i].src = s->const_data_ptr();
            e[i].dst = d ? d->mutable_data_ptr() : nullptr;
            e[i].n = s->numel();
            e[i].dtype = code(s->scalar_type());
            e[i].out_dtype = d ? code(d->scalar_type()) : e[i].dtype;
            if (!plain && e[i].n) {
                PyObject* k = PyLong_FromSsize_t(i);
                ok = k && PyList_Append(odd, k) == 0;
                Py_XDECREF(k);
            }
        }
    } catch (...) {
        Py_DECREF(bytes);
        Py_DECREF(odd);
        throw;
    }
    if (!ok) {
        Py_DECREF(bytes);
        Py_DECREF(odd);
        return nullptr;
    }
    return Py_BuildValue("NiNN", bytes, n ? (int)device.index() : -1, PyBool_FromLong(wants_grad), odd);
    END_HANDLE_TH_ERRORS
}

// written(tensors): a graph that has saved one of them sees that it has changed
PyObject* written(PyObject*, PyObject* list) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
        const at::Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(list, i));
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"table", table, METH_VARARGS, "table(src, dst or None, writes) -> (bytes, device, requires_grad, odd)"},
                         {"written", written, METH_O, "written(tensors of a list that table() has taken)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_list", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddIntConstant(m, "VERSION", LVAE_VERSION) != 0) Py_CLEAR(m);
    return m;
}
