// Host side of decoder_ops: checks the tensors of a call, lays them out as lvae_vocab_problem, allocates what it writes,
// calls liblvae, and stands in autograd's graph.
//
// A training step of a few hundred tokens is 50-80 us of GPU work; with all this in Python, through ctypes, it took 45 us of
// host time in a warm loop and twice that between the threads of autograd, more than the rest of the step (340 float16
// tokens, 9,999 words: 160 us so, 102 us with calls and layout here, 82 us with the node of the graph here too).  The
// entry points are those of the library that Python has loaded (bind), so there is one library and one place that finds it.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/object_ptr.h>
#include <pybind11/pybind11.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>

#include "../../include/lvae.h"
#include "tensor_checks.h"

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

// what Python has set, as an exception that may cross threads: a backward runs on one of autograd's own
[[noreturn]] void throw_python() {
    python_error e;
    e.persist();
    throw e;
}
[[noreturn]] void fail(PyObject* type, const std::string& what) {
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(type, what.c_str());
    throw_python();
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

void* current_stream(at::Device device) {
    pybind11::gil_scoped_acquire gil;
    THPObjectPtr h(PyObject_CallFunction(lib.raw_stream, "i", (int)device.index()));
    void* stream = h ? PyLong_AsVoidPtr(h) : nullptr;
    if (!stream && PyErr_Occurred()) throw_python();
    return stream;
}

void on_gpu(const at::Tensor& t, const char* name) {
    if (!t.is_cuda()) fail(lib.error, std::string(name) + " is on " + t.device().str() + ": the HIP path needs a GPU tensor (no CPU fallback)");
}

// refused wherever it lives: its result would be wrong without a word
void check_plain(const at::Tensor& t, const char* name) {
    if (!t.defined()) return;
    if (const char* why = more_than_memory(t)) fail(lib.error, std::string(name) + " " + why);
}
void check_not_traced() {
    if (being_traced()) fail(lib.error, "the log-likelihoods cannot be traced: a trace would not hold their kernels");
}

void prepare(Problem& q, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets, const at::Tensor& bias, int64_t ignore_index) {
    on_gpu(hidden, "hidden");
    on_gpu(weight, "weight");
    on_gpu(targets, "targets");
    if (bias.defined()) on_gpu(bias, "bias");
    // a negated view (the imaginary part of a conjugate) holds the other sign in memory
    q.hidden = hidden.resolve_neg();
    q.weight = weight.resolve_neg();
    q.targets = targets.resolve_neg();
    q.bias = bias.defined() ? bias.resolve_neg() : bias;
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
    q.stream = current_stream(q.device);
}

// f() while other Python threads may run
template <class F> int without_gil(F f) {
    if (!PyGILState_Check()) return f();
    pybind11::gil_scoped_release released;
    return f();
}

void* data(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// What a forward leaves for its backward: the LSE of every token, the factor of every token in a loss, limbs of the weights
struct Saved {
    at::Tensor lse, each, kept;
};

at::Tensor run_forward(const Problem& q, int how, Saved* saved) {
    const c10::DeviceGuard guard(q.device);
    const at::Tensor ll = q.empty(q.shape, at::kFloat);
    at::Tensor lse, kept, loss, each, out = ll;
    int64_t kept_bytes = 0;
    if (saved) {
        lse = q.empty(q.shape, at::kFloat);
        if (q.tokens) check(lib.kept_bytes(&q.c, &kept_bytes));
        if (kept_bytes) kept = q.empty({kept_bytes}, at::kByte);
    }
    if (how >= MEAN) {
        loss = q.empty({}, at::kFloat);
        each = q.empty({}, at::kFloat);
        if (!q.tokens) {
            loss.zero_();
            each.zero_();
        }
        out = loss;
    }
    if (how == SEQUENCES) out = q.empty(at::IntArrayRef(q.shape).slice(0, q.shape.size() - 1), at::kFloat);
    if (q.tokens) {
        int64_t bytes = 0;
        check(lib.ll_bytes(&q.c, &bytes));
        if (kept_bytes) bytes -= kept_bytes - 256;
        const at::Tensor ws = q.empty({bytes}, at::kByte);
        check(without_gil([&] {
            return lib.ll(&q.c, (float*)data(ll), (float*)data(lse), data(kept), (float*)data(loss), (float*)data(each), how == MEAN,
                          data(ws), bytes, q.stream);
        }));
    }
    if (how == SEQUENCES && out.numel())
        check(without_gil([&] { return lib.segment_sum((const float*)data(ll), out.numel(), q.shape.back(), (float*)data(out), q.stream); }));
    if (saved) *saved = Saved{lse, each, kept};
    return out;
}

struct Gradients {
    at::Tensor hidden, weight, bias;
};

Gradients run_backward(const Problem& q, int how, const Saved& saved, at::Tensor g, bool want_h, bool want_w, bool want_b) {
    const c10::DeviceGuard guard(q.device);
    const at::Tensor lse = saved.lse.contiguous();
    g = g.resolve_neg();
    if (g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
    int64_t g_stride[3] = {0, 0, 0};
    if (how < MEAN) {
        // sequences: one value for all positions of a sentence; the problem's axes join dimensions, so spread it out
        g = (how == TOKENS ? g : g.unsqueeze(-1).expand(q.shape)).contiguous();
        g_stride[0] = q.c.size[1] * q.c.size[2];
        g_stride[1] = q.c.size[2];
        g_stride[2] = 1;
    }
    Gradients d;
    if (want_h) d.hidden = q.empty(q.hidden.sizes(), q.hidden.scalar_type());
    if (want_w) d.weight = q.empty(q.weight.sizes(), q.weight.scalar_type());
    if (want_b) d.bias = q.empty(q.bias.sizes(), q.bias.scalar_type());
    if (q.tokens) {
        int64_t bytes = 0;
        check(lib.bwd_bytes(&q.c, want_h, want_w, want_b, &bytes));
        if (saved.kept.defined()) bytes -= saved.kept.numel() - 256;
        const at::Tensor ws = q.empty({bytes}, at::kByte);
        check(without_gil([&] {
            return lib.bwd(&q.c, (const float*)data(lse), (const float*)data(g), g_stride, (const float*)data(saved.each), data(saved.kept),
                           data(d.hidden), data(d.weight), data(d.bias), data(ws), bytes, q.stream);
        }));
    } else {
        if (want_w) d.weight.zero_();
        if (want_b) d.bias.zero_();
    }
    return d;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A gradient that refuses to be differentiated again, rather than to count as a constant
struct Once : torch::autograd::Function<Once> {
    static at::Tensor forward(AutogradContext*, const at::Tensor& t, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&,
                              const at::Tensor&) {
        return t.view_as(t);
    }
    static variable_list backward(AutogradContext*, const variable_list&) {
        fail(lib.error, "the log-likelihoods have no second derivatives");
    }
};

// Token log-likelihoods, put together, with a HIP backward: the softmax is computed again from the saved LSE, a piece of
// the vocabulary at a time
struct LogLikelihood : torch::autograd::Function<LogLikelihood> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                              const std::optional<at::Tensor>& bias, int64_t ignore_index, int64_t how) {
        Problem q;
        prepare(q, hidden, weight, targets, bias.value_or(at::Tensor()), ignore_index);
        Saved saved;
        const at::Tensor out = run_forward(q, (int)how, &saved);
        ctx->save_for_backward({q.hidden, q.weight, q.targets, q.bias, saved.lse, saved.each, saved.kept});
        ctx->saved_data["ignore_index"] = ignore_index;
        ctx->saved_data["how"] = how;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& g) {
        const variable_list s = ctx->get_saved_variables();
        const at::Tensor &hidden = s[0], &weight = s[1], &bias = s[3];
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = bias.defined() && ctx->needs_input_grad(3);
        variable_list d(6);
        if (!want_h && !want_w && !want_b) return d;
        check_not_traced();
        check_plain(g[0], "the upstream gradient");
        Gradients got;
        {
            const at::NoGradGuard no_grad;
            // planned anew: a hook of the saved tensors may have moved them or laid them out in another way
            Problem q;
            prepare(q, hidden, weight, s[2], bias, ctx->saved_data["ignore_index"].toInt());
            got = run_backward(q, (int)ctx->saved_data["how"].toInt(), Saved{s[4], s[5], s[6]}, g[0], want_h, want_w, want_b);
        }
        const std::optional<at::Tensor> b = bias.defined() ? std::optional<at::Tensor>(bias) : std::nullopt;
        auto once = [&](const at::Tensor& t) {
            return t.defined() && at::GradMode::is_enabled() ? Once::apply(t, hidden, weight, b, g[0]) : t;      // create_graph
        };
        d[0] = once(got.hidden);
        d[1] = once(got.weight);
        d[3] = once(got.bias);
        return d;
    }
};

at::Tensor tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string(name) + " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}

// log_likelihood(hidden, weight, targets, bias, ignore_index, how)
PyObject* log_likelihood(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *hidden_, *weight_, *targets_, *bias_;
    long long ignore_index;
    int how;
    if (!PyArg_ParseTuple(args, "OOOOLi", &hidden_, &weight_, &targets_, &bias_, &ignore_index, &how)) return nullptr;
    const at::Tensor hidden = tensor(hidden_, "hidden"), weight = tensor(weight_, "weight"), targets = tensor(targets_, "targets");
    const at::Tensor bias = bias_ == Py_None ? at::Tensor() : tensor(bias_, "bias");
    check_not_traced();
    check_plain(hidden, "hidden");
    check_plain(weight, "weight");
    check_plain(bias, "bias");
    check_plain(targets, "targets");
    if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad())))
        return THPVariable_Wrap(LogLikelihood::apply(hidden, weight, targets, bias.defined() ? std::optional<at::Tensor>(bias) : std::nullopt,
                                                     (int64_t)ignore_index, (int64_t)how));
    Problem q;
    prepare(q, hidden, weight, targets, bias, ignore_index);
    return THPVariable_Wrap(run_forward(q, how, nullptr));
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
                         {"log_likelihood", log_likelihood, METH_VARARGS, "log_likelihood(hidden, weight, targets, bias, ignore_index, how)"},
                         {"common_axes", py_common_axes, METH_VARARGS, "common_axes(shape, [strides of each tensor])"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decoder_calls() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddIntConstant(m, "VERSION", LVAE_VERSION) != 0) Py_CLEAR(m);
    return m;
}
