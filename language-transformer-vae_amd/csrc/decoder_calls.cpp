// Host helper of decoder_ops: checks the tensors of a call, lays them out as lvae_vocab_problem, allocates what it
// writes and calls liblvae.
//
// A training step of a few hundred tokens is 80 us of GPU work; the same in Python, through ctypes, took 45 us of host time
// in a warm loop and twice that between the threads of autograd, more than the rest of the step.  The entry points are
// those of the library that Python has loaded (bind), so there is one library and one place that finds it.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>

#include "../../include/lvae.h"

namespace {

struct Library {
    decltype(&lvae_vocab_ll_workspace_bytes) ll_bytes;
    decltype(&lvae_vocab_ll_kept_bytes) kept_bytes;
    decltype(&lvae_vocab_ll) ll;
    decltype(&lvae_vocab_ll_bwd_workspace_bytes) bwd_bytes;
    decltype(&lvae_vocab_ll_bwd) bwd;
    decltype(&lvae_segment_sum_f32) segment_sum;
    decltype(&lvae_last_error) last_error;
    PyObject *error, *raw_stream;           // the exception class; device index -> handle of its current stream
} lib;

// How the log-likelihoods of the tokens are put together: as they are, summed over the last axis, or one loss
enum { TOKENS = 0, SEQUENCES = 1, MEAN = 2, SUM = 3 };

int code(at::ScalarType t) {
    return t == at::kFloat ? LVAE_F32 : t == at::kBFloat16 ? LVAE_BF16 : t == at::kHalf ? LVAE_F16 : -1;
}

[[noreturn]] void fail(PyObject* type, const std::string& what) {
    PyErr_SetString(type, what.c_str());
    throw python_error();
}
void check(int rc) {
    if (rc != LVAE_OK) fail(lib.error, "liblvae status " + std::to_string(rc) + ": " + lib.last_error());
}
std::string text(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + (v.size() == 1 ? ",)" : ")");
}

// The token dimensions as three axes on which every tensor (n of them, at most 8) steps evenly; false where there are more
bool common_axes(at::IntArrayRef shape, const at::IntArrayRef* strides, int n, int64_t size[3], int64_t (*step)[3]) {
    int64_t s[3], st[8][3];
    int axes = 0;
    for (size_t i = 0; i < shape.size(); ++i) {
        if (shape[i] == 1) continue;
        bool joins = axes > 0;
        for (int k = 0; k < n; ++k) joins = joins && st[k][axes - 1] == shape[i] * strides[k][i];
        if (!joins && axes == 3) return false;
        if (!joins) s[axes++] = 1;
        s[axes - 1] *= shape[i];
        for (int k = 0; k < n; ++k) st[k][axes - 1] = strides[k][i];
    }
    for (int a = 0; a < 3; ++a) {
        const int from = a - (3 - axes);
        size[a] = from < 0 ? 1 : s[from];
        for (int k = 0; k < n; ++k) step[k][a] = from < 0 ? 0 : st[k][from];
    }
    return true;
}

// Checked arguments of one call: the C structure and the tensors that its pointers belong to
struct Problem {
    at::Tensor hidden, weight, targets, bias;           // bias undefined where there is none
    lvae_vocab_problem c;
    at::DimVector shape;                                // of the tokens
    int64_t tokens;
    at::Device device = at::Device(at::kCPU);
    void* stream;

    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType t) const { return at::empty(sizes, at::TensorOptions(device).dtype(t)); }
};

at::Tensor tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string(name) + " must be a torch.Tensor");
    at::Tensor t = THPVariable_Unpack(o);
    if (!t.is_cuda()) fail(lib.error, std::string(name) + " is on " + t.device().str() + ": the HIP path needs a GPU tensor (no CPU fallback)");
    return t;
}

void prepare(Problem& q, PyObject* hidden, PyObject* weight, PyObject* targets, PyObject* bias, int64_t ignore_index) {
    q.hidden = tensor(hidden, "hidden");
    q.weight = tensor(weight, "weight");
    q.targets = tensor(targets, "targets");
    if (bias != Py_None) q.bias = tensor(bias, "bias");
    q.device = q.hidden.device();
    if (q.weight.device() != q.device || q.targets.device() != q.device || (q.bias.defined() && q.bias.device() != q.device))
        fail(PyExc_ValueError, "hidden, weight, targets and bias must be on one device");
    const int dtype = code(q.hidden.scalar_type());
    if (dtype < 0 || q.weight.scalar_type() != q.hidden.scalar_type())
        fail(PyExc_TypeError, std::string("hidden and weight must be of one type, float32, bfloat16 or float16: ") +
                                  toString(q.hidden.scalar_type()) + ", " + toString(q.weight.scalar_type()));
    const int bias_dtype = q.bias.defined() ? code(q.bias.scalar_type()) : 0;
    if (bias_dtype < 0) fail(PyExc_TypeError, std::string("bias must be float32, bfloat16 or float16: ") + toString(q.bias.scalar_type()));
    if (q.targets.scalar_type() != at::kLong) fail(PyExc_TypeError, std::string("targets must be int64: ") + toString(q.targets.scalar_type()));
    if (q.hidden.layout() != at::kStrided || q.weight.layout() != at::kStrided || q.targets.layout() != at::kStrided ||
        (q.bias.defined() && q.bias.layout() != at::kStrided))
        fail(PyExc_TypeError, "hidden, weight, targets and bias must be dense tensors");
    if (q.hidden.dim() < 1 || q.weight.dim() != 2 || q.weight.size(1) != q.hidden.size(-1))
        fail(PyExc_ValueError, "shape mismatch: hidden " + text(q.hidden.sizes()) + ", weight " + text(q.weight.sizes()));
    const int64_t V = q.weight.size(0), H = q.weight.size(1);
    if (V < 1 || H < 1) fail(PyExc_ValueError, "weight " + text(q.weight.sizes()) + " is empty");
    if (q.bias.defined() && (q.bias.dim() != 1 || q.bias.size(0) != V))
        fail(PyExc_ValueError, "bias " + text(q.bias.sizes()) + " must be (" + std::to_string(V) + ",)");
    const at::IntArrayRef all = q.hidden.sizes(), shape = all.slice(0, all.size() - 1);
    q.shape.assign(shape.begin(), shape.end());
    if (q.targets.sizes() != shape) {
        const at::IntArrayRef t = q.targets.sizes();
        bool fits = t.size() <= shape.size();
        for (size_t i = 0; fits && i < t.size(); ++i) fits = t[i] == 1 || t[i] == shape[shape.size() - t.size() + i];
        if (!fits) fail(PyExc_ValueError, "targets " + text(t) + " do not expand to " + text(shape));
        q.targets = q.targets.expand(q.shape);
    }
    if (q.hidden.stride(-1) != 1 && H > 1) q.hidden = q.hidden.contiguous();
    if ((q.weight.stride(1) != 1 && H > 1) || (q.weight.stride(0) < H && V > 1)) q.weight = q.weight.contiguous();
    if (q.bias.defined() && !q.bias.is_contiguous()) q.bias = q.bias.contiguous();
    int64_t step[2][3];
    for (int again = 0;; ++again) {
        const at::IntArrayRef hs = q.hidden.strides();
        const at::IntArrayRef strides[2] = {hs.slice(0, hs.size() - 1), q.targets.strides()};
        if (common_axes(q.shape, strides, 2, q.c.size, step) || again) break;
        q.hidden = q.hidden.contiguous();
        q.targets = q.targets.contiguous();
    }
    for (int a = 0; a < 3; ++a) {
        q.c.hidden_stride[a] = step[0][a];
        q.c.target_stride[a] = step[1][a];
    }
    q.tokens = q.targets.numel();
    q.c.hidden = q.hidden.const_data_ptr();
    q.c.weight = q.weight.const_data_ptr();
    q.c.bias = q.bias.defined() ? q.bias.const_data_ptr() : nullptr;
    q.c.targets = (const int64_t*)q.targets.const_data_ptr();
    q.c.V = V;
    q.c.weight_stride = V > 1 ? q.weight.stride(0) : H;
    q.c.ignore_index = ignore_index;
    q.c.H = (int32_t)std::min<int64_t>(H, 1 << 30);      // refused there
    q.c.dtype = dtype;
    q.c.bias_dtype = bias_dtype;
    q.c.reserved = 0;
    THPObjectPtr stream(PyObject_CallFunction(lib.raw_stream, "i", (int)q.device.index()));
    if (!stream) throw python_error();
    q.stream = PyLong_AsVoidPtr(stream);
    if (!q.stream && PyErr_Occurred()) throw python_error();
}

template <class F> int without_gil(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

void* data(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
PyObject* wrap(const at::Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
at::Tensor unwrap(PyObject* o) { return o == Py_None ? at::Tensor() : THPVariable_Unpack(o); }

// forward(hidden, weight, targets, bias, ignore_index, how, for_backward) -> result, or with for_backward
// (result, hidden, weight, targets, bias as they are read, LSE of every token, factor of every token in a loss, what is kept of
// the weights)
PyObject* forward(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *hidden, *weight, *targets, *bias;
    long long ignore_index;
    int how, for_backward;
    if (!PyArg_ParseTuple(args, "OOOOLip", &hidden, &weight, &targets, &bias, &ignore_index, &how, &for_backward)) return nullptr;
    Problem q;
    prepare(q, hidden, weight, targets, bias, ignore_index);
    const c10::DeviceGuard guard(q.device);
    const at::Tensor ll = q.empty(q.shape, at::kFloat);
    at::Tensor lse, kept, loss, each, out = ll;
    int64_t kept_bytes = 0;
    if (for_backward) {
        lse = q.empty(q.shape, at::kFloat);
        if (q.tokens) check(lib.kept_bytes(&q.c, &kept_bytes));
        if (kept_bytes) kept = q.empty({kept_bytes}, at::kByte);
    }
    if (how >= MEAN) {
        const at::TensorOptions o = at::TensorOptions(q.device).dtype(at::kFloat);
        loss = q.tokens ? at::empty({}, o) : at::zeros({}, o);
        each = q.tokens ? at::empty({}, o) : at::zeros({}, o);
        out = loss;
    }
    if (how == SEQUENCES) out = q.empty(at::IntArrayRef(q.shape).slice(0, q.shape.size() - 1), at::kFloat);
    if (q.tokens) {
        int64_t bytes = 0;
        check(lib.ll_bytes(&q.c, &bytes));
        if (kept_bytes) bytes -= kept_bytes - 256;
        const at::Tensor ws = q.empty({bytes}, at::kByte);
        check(without_gil([&] {
            return lib.ll(&q.c, (float*)data(ll), (float*)data(lse), data(kept), (float*)data(loss), (float*)data(each),
                          how == MEAN, data(ws), bytes, q.stream);
        }));
    }
    if (how == SEQUENCES && out.numel())
        check(without_gil([&] { return lib.segment_sum((const float*)data(ll), out.numel(), q.shape.back(), (float*)data(out), q.stream); }));
    if (!for_backward) return wrap(out);
    return Py_BuildValue("NNNNNNNN", wrap(out), wrap(q.hidden), wrap(q.weight), wrap(q.targets), wrap(q.bias), wrap(lse), wrap(each),
                         wrap(kept));
    END_HANDLE_TH_ERRORS
}

// backward(hidden, weight, targets, bias, ignore_index, how, lse, each, kept, g, three truth values) -> gradients of
// hidden, weight and bias, None where not wanted
PyObject* backward(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *hidden, *weight, *targets, *bias, *lse_, *each_, *kept_, *g_;
    long long ignore_index;
    int how, want_h, want_w, want_b;
    if (!PyArg_ParseTuple(args, "OOOOLiOOOOppp", &hidden, &weight, &targets, &bias, &ignore_index, &how, &lse_, &each_, &kept_, &g_,
                          &want_h, &want_w, &want_b))
        return nullptr;
    // planned anew: a hook of the saved tensors may have moved them or laid them out in another way
    Problem q;
    prepare(q, hidden, weight, targets, bias, ignore_index);
    const c10::DeviceGuard guard(q.device);
    at::Tensor lse = unwrap(lse_).contiguous(), each = unwrap(each_), kept = unwrap(kept_), g = unwrap(g_);
    if (g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
    int64_t g_stride[3] = {0, 0, 0};
    if (how < MEAN) {
        // sequences: one value for all positions of a sentence; the problem's axes join dimensions, so spread it out
        g = (how == TOKENS ? g : g.unsqueeze(-1).expand(q.shape)).contiguous();
        g_stride[0] = q.c.size[1] * q.c.size[2];
        g_stride[1] = q.c.size[2];
        g_stride[2] = 1;
    }
    at::Tensor d_h, d_w, d_b;
    if (want_h) d_h = q.empty(q.hidden.sizes(), q.hidden.scalar_type());
    if (want_w) d_w = q.empty(q.weight.sizes(), q.weight.scalar_type());
    if (want_b) d_b = q.empty(q.bias.sizes(), q.bias.scalar_type());
    if (q.tokens) {
        int64_t bytes = 0;
        check(lib.bwd_bytes(&q.c, want_h, want_w, want_b, &bytes));
        if (kept.defined()) bytes -= kept.numel() - 256;
        const at::Tensor ws = q.empty({bytes}, at::kByte);
        check(without_gil([&] {
            return lib.bwd(&q.c, (const float*)data(lse), (const float*)data(g), g_stride, (const float*)data(each),
                           data(kept), data(d_h), data(d_w), data(d_b), data(ws), bytes, q.stream);
        }));
    } else {
        if (want_w) d_w.zero_();
        if (want_b) d_b.zero_();
    }
    return Py_BuildValue("NNN", wrap(d_h), wrap(d_w), wrap(d_b));
    END_HANDLE_TH_ERRORS
}

// common_axes(shape, [strides of each tensor]) -> (sizes, [strides of each]) of three axes, or None
PyObject* py_common_axes(PyObject*, PyObject* args) {
    PyObject *shape_, *strides_;
    if (!PyArg_ParseTuple(args, "OO!", &shape_, &PyList_Type, &strides_)) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(strides_);
    std::vector<int64_t> v[9];
    for (Py_ssize_t k = -1; k < n && k < 8; ++k) {
        THPObjectPtr s(PySequence_Fast(k < 0 ? shape_ : PyList_GET_ITEM(strides_, k), "a sequence of integers"));
        if (!s) return nullptr;
        for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(s.get()); ++i) v[k + 1].push_back(PyLong_AsLongLong(PySequence_Fast_GET_ITEM(s.get(), i)));
        if (PyErr_Occurred()) return nullptr;
        if (n > 8 || v[k + 1].size() != v[0].size()) {
            PyErr_SetString(PyExc_ValueError, "strides of up to 8 tensors, one for each dimension");
            return nullptr;
        }
    }
    at::IntArrayRef strides[8];
    for (Py_ssize_t k = 0; k < n; ++k) strides[k] = v[k + 1];
    int64_t size[3], step[8][3];
    if (!common_axes(v[0], strides, (int)n, size, step)) Py_RETURN_NONE;
    PyObject* list = PyList_New(n);
    for (Py_ssize_t k = 0; list && k < n; ++k) PyList_SET_ITEM(list, k, Py_BuildValue("[LLL]", step[k][0], step[k][1], step[k][2]));
    return Py_BuildValue("[LLL]N", size[0], size[1], size[2], list);
}

// bind([addresses of the entry points, in the order of Library], exception class, device index -> stream handle)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[7];
    PyObject *error, *raw_stream;
    if (!PyArg_ParseTuple(args, "(KKKKKKK)OO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &error, &raw_stream)) return nullptr;
    Py_INCREF(error);
    Py_INCREF(raw_stream);
    lib.ll_bytes = (decltype(lib.ll_bytes))a[0];
    lib.kept_bytes = (decltype(lib.kept_bytes))a[1];
    lib.ll = (decltype(lib.ll))a[2];
    lib.bwd_bytes = (decltype(lib.bwd_bytes))a[3];
    lib.bwd = (decltype(lib.bwd))a[4];
    lib.segment_sum = (decltype(lib.segment_sum))a[5];
    lib.last_error = (decltype(lib.last_error))a[6];
    Py_XDECREF(lib.error);
    Py_XDECREF(lib.raw_stream);
    lib.error = error;
    lib.raw_stream = raw_stream;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "bind(entry points, exception class, stream of a device)"},
                         {"forward", forward, METH_VARARGS, "forward(hidden, weight, targets, bias, ignore_index, how, for_backward)"},
                         {"backward", backward, METH_VARARGS, "backward(hidden, weight, targets, bias, ignore_index, how, lse, each, kept, g, wanted...)"},
                         {"common_axes", py_common_axes, METH_VARARGS, "common_axes(shape, [strides of each tensor])"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decoder_calls() { return PyModule_Create(&module); }
