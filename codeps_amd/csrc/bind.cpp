// codeps_amd/_bind.so: the Python side of the channel norms, AdamW's step and the gradient norm, in C++ on torch's own API (tensors, autograd nodes).
// The arithmetic is in libcodeps_hip.so behind its C ABI (include/codeps_hip.h), whose entry points this module is handed as addresses, so that both follow
// the one library that the package has loaded.
//
// Why not ctypes and torch.autograd.Function as elsewhere: these calls are short.  A backward pass written in Python runs on autograd's worker thread and
// has to wait for the interpreter lock there; a list of 160 gradients costs 0.2 us per tensor in Python.  Per call, Python / this module: one-row norm
// 9.4 / 6.1 us, small norm with its gradients 103 / 69 us, gradient norm of 160 small tensors 37 / 12 us, AdamW's step over them 54 / 13 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/codeps_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct {
    decltype(&codeps_last_error) last_error;
    decltype(&codeps_channel_norm_fwd) norm_fwd;
    decltype(&codeps_channel_norm_bwd_workspace_bytes) norm_bwd_bytes;
    decltype(&codeps_channel_norm_bwd) norm_bwd;
    decltype(&codeps_grad_norm_workspace_bytes) grad_norm_bytes;
    decltype(&codeps_grad_norm) grad_norm;
    decltype(&codeps_adamw_step) adamw_step;
} api;
PyObject *error_class = nullptr, *memory_error = nullptr;              // CodepsHipError, torch.OutOfMemoryError

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };
template <typename... A> [[noreturn]] void refuse(const A&... parts) { throw Refused(c10::str(parts...)); }
void check(int rc, const char* what) {
    if (rc != 0) refuse(what, " failed (", rc, "): ", api.last_error());
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return CODEPS_F32;
        case at::kBFloat16: return CODEPS_BF16;
        case at::kHalf: return CODEPS_F16;
        default: return -1;
    }
}
void* at_(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
codeps_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
std::string described(const Tensor& t) { return c10::str(t.sizes(), " ", t.scalar_type(), " on ", t.device()); }

// ------------------------------------------------------------------------------------------------------------------------ channel norms
constexpr int64_t MAX_CHANNELS = 8192, MAX_PITCH = 1 << 24;

// t itself when its channels are dense and its rows lie at one distance (elements, in `pitch`), else a contiguous copy.  (A view that negates on reading --
// the imaginary part of a conjugate -- holds the other sign in memory.)
Tensor pitched(const Tensor& given, int64_t& pitch) {
    const Tensor t = given.is_neg() ? given.resolve_neg() : given;
    const int64_t c = t.size(-1);
    pitch = c;
    if (t.is_contiguous()) return t;
    if (t.stride(-1) == 1 || c == 1) {
        int64_t step = -1, span = 1;
        bool even = true;
        for (int64_t i = t.dim() - 2; i >= 0 && even; --i) {
            if (t.size(i) == 1) continue;
            if (step < 0) step = t.stride(i);
            else even = t.stride(i) == step * span;
            span *= t.size(i);
        }
        if (step < 0) return t;
        if (even && step >= c && step < MAX_PITCH) { pitch = step; return t; }
    }
    return t.contiguous();
}

struct Norm {
    codeps_channel_norm_desc d{};
    Tensor x, residual, gate, weight, bias, next_weight, next_bias;   // as given (vectors contiguous)
    Tensor xr, rr, gr;                                                // rows that the kernels read: the tensors themselves, or copies
    Tensor y, h, stats;
};

void forward(Norm& n, bool want_stats) {
    auto& d = n.d;
    const int64_t c = n.x.size(-1);
    d.channels = (int32_t)c;
    d.rows = n.x.numel() / c;
    if (d.rows >= (int64_t)1 << 31) refuse("channel norm: ", d.rows, " rows, at most 2^31 - 1");
    n.xr = pitched(n.x, d.x_pitch);
    d.res_pitch = d.gate_pitch = d.dy_pitch = d.dh_pitch = c;
    d.x_type = d.res_type = type_of(n.x);
    if (n.residual.defined()) {
        n.rr = pitched(n.residual, d.res_pitch);
        d.res_type = type_of(n.residual);
    }
    if (n.gate.defined()) {
        n.gr = pitched(n.gate, d.gate_pitch);
        d.gate_type = type_of(n.gate);
    }
    const Tensor &v = n.weight.defined() ? n.weight : n.bias, &nv = n.next_weight.defined() ? n.next_weight : n.next_bias;
    d.weight_type = v.defined() ? type_of(v) : 0;
    d.next_weight_type = nv.defined() ? type_of(nv) : 0;
    if (d.full) n.y = at::empty(n.x.sizes(), n.residual.defined() ? n.residual.options() : n.x.options());
    if (d.next_kind || !d.full) n.h = at::empty(n.x.sizes(), n.x.options());
    if (want_stats) n.stats = at::empty({d.rows, d.full ? 4 : 2}, n.x.options().dtype(at::kFloat));
    c10::DeviceGuard guard(n.x.device());
    check(api.norm_fwd(&d, at_(n.xr), at_(n.rr), at_(n.gr), at_(n.weight), at_(n.bias), at_(n.next_weight), at_(n.next_bias), at_(n.y), at_(n.h),
                       (float*)at_(n.stats), stream_of(n.x)), "codeps_channel_norm_fwd");
}

// Inputs in edge order: x, residual, gate, weight, bias, next_weight, next_bias.  Outputs: (h) or (y[, h]).
struct ChannelNormBackward : public torch::autograd::Node {
    codeps_channel_norm_desc desc;
    SavedVariable x, residual, gate, weight, bias, next_weight, stats;
    std::vector<int64_t> x_sizes, gate_sizes;
    at::TensorOptions options, res_options, gate_options, vec_options[4];
    Tensor sinks[4];                                                  // flat-gradient views that take a vector's gradient in place

    std::string name() const override { return "ChannelNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* s : {&x, &residual, &gate, &weight, &bias, &next_weight, &stats}) s->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        if (!at::GradMode::is_enabled()) return run(grads);
        variable_list out;
        {
            at::NoGradGuard off;                                      // (create_graph: a second derivative raises instead of being silently zero)
            out = run(grads);
        }
        auto error = std::make_shared<torch::autograd::DelayedError>("the channel norms have no second derivative", (int)out.size());
        return (*error)(std::move(out));
    }
    variable_list run(const variable_list& grads) {
        std::lock_guard<std::mutex> lock(mutex_);
        codeps_channel_norm_desc d = desc;
        Tensor dy, dh;
        if (d.full) {
            dy = grads[0];
            if (d.next_kind) dh = grads[1];
        } else {
            dh = grads[0];
        }
        variable_list out(7);
        if (!dy.defined() && !dh.defined()) return out;
        const Tensor given = dy, xs = x.unpack(), gs = gate.unpack(), ws = weight.unpack(), bs = bias.unpack(), nws = next_weight.unpack(), st = stats.unpack();
        Tensor rs = residual.unpack();
        if (dy.defined()) dy = pitched(dy, d.dy_pitch);
        if (dh.defined()) dh = pitched(dh, d.dh_pitch);
        else if (d.next_kind) { d.next_kind = 0; rs = Tensor(); }     // h is not part of the loss: the block's end alone
        if (task_should_compute_output(0)) out[0] = at::empty(x_sizes, options);
        // without a next norm y's gradient is the residual's: handed on, not copied
        const bool res = task_should_compute_output(1);
        if (res) out[1] = d.next_kind ? at::empty(x_sizes, res_options) : given;
        if (task_should_compute_output(2)) out[2] = d.rows ? at::empty(gate_sizes, gate_options) : at::zeros(gate_sizes, gate_options);
        void* vec[4] = {};
        Tensor twice[4];                                              // one parameter as two of the vectors: the second gradient is added behind the pass
        int acc = 0;
        for (int i = 0; i < (d.next_kind ? 4 : 2); ++i) {
            if (!task_should_compute_output(3 + i)) continue;
            if (sinks[i].defined()) {
                vec[i] = sinks[i].data_ptr();
                for (int j = 0; j < i; ++j)
                    if (vec[j] == vec[i]) twice[i] = at::empty({d.channels}, sinks[i].options());
                if (twice[i].defined()) vec[i] = twice[i].data_ptr();
                else acc |= 1 << i;
            } else {
                out[3 + i] = at::empty({d.channels}, vec_options[i]);
                vec[i] = out[3 + i].data_ptr();
            }
        }
        const size_t bytes = api.norm_bwd_bytes(&d);
        if (bytes == 0) check(CODEPS_ERR_ARG, "codeps_channel_norm_bwd_workspace_bytes");
        const Tensor work = at::empty({(int64_t)bytes}, options.dtype(at::kByte));            // not a cached one: captured graphs must not share it
        c10::DeviceGuard guard(options.device());
        check(api.norm_bwd(&d, at_(xs), at_(rs), at_(gs), at_(ws), at_(bs), at_(nws), (const float*)at_(st), at_(dy), at_(dh), at_(out[0]),
                           res && d.next_kind ? at_(out[1]) : nullptr, at_(out[2]), vec[0], vec[1], vec[2], vec[3], acc, work.data_ptr(), bytes, stream_of(xs)),
              "codeps_channel_norm_bwd");
        for (int i = 0; i < 4; ++i)
            if (twice[i].defined()) sinks[i].add_(twice[i].view(sinks[i].sizes()));
        return out;
    }
};

// A leaf's accumulation node runs on the stream that was current when its oldest living graph was built.  Where that is the default stream and the current
// one is captured, the backward pass would put work on a stream that cannot be captured, in the middle of a capture: refused while nothing has happened yet.
void check_capture(const Tensor* const (&in)[7]) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor* t : in) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto stream = node->stream();
        if (stream && stream->id() == c10::hip::getDefaultHIPStream(t->device().index()).id())
            refuse("channel norm under graph capture: a graph that was built eagerly on the default stream still refers to a leaf of shape ", t->sizes(),
                   "; drop it before the capture, or build it on another stream");
    }
}

// y[, h] or h, with a node behind them where a gradient is wanted; sinks: 4 tensors, undefined where there is none
void apply(Norm& n, const Tensor (&sinks)[4]) {
    const Tensor* in[7] = {&n.x, &n.residual, &n.gate, &n.weight, &n.bias, &n.next_weight, &n.next_bias};
    bool grad = false;
    if (at::GradMode::is_enabled())
        for (const Tensor* t : in) grad = grad || (t->defined() && t->requires_grad());
    if (grad) check_capture(in);
    {
        at::NoGradGuard off;
        forward(n, grad);
    }
    if (!grad) return;
    auto node = std::shared_ptr<ChannelNormBackward>(new ChannelNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(n.x, n.residual, n.gate, n.weight, n.bias, n.next_weight, n.next_bias));
    node->desc = n.d;
    node->x = SavedVariable(n.xr, false);
    if (n.d.next_kind) node->residual = SavedVariable(n.rr, false);
    node->gate = SavedVariable(n.gr, false);
    node->weight = SavedVariable(n.weight, false);
    node->bias = SavedVariable(n.bias, false);
    node->next_weight = SavedVariable(n.next_weight, false);
    node->stats = SavedVariable(n.stats, false);
    node->x_sizes = n.x.sizes().vec();
    node->options = n.x.options();
    if (n.residual.defined()) node->res_options = n.residual.options();
    if (n.gate.defined()) { node->gate_sizes = n.gate.sizes().vec(); node->gate_options = n.gate.options(); }
    for (int i = 0; i < 4; ++i) {
        if (in[3 + i]->defined()) node->vec_options[i] = in[3 + i]->options();
        node->sinks[i] = sinks[i];
    }
    if (n.y.defined()) torch::autograd::set_history(n.y, node);
    if (n.h.defined()) torch::autograd::set_history(n.h, node);
}

void check_rows(const Tensor& x, const char* what) {
    if (!x.is_cuda()) refuse("codeps_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback");
    if (type_of(x) < 0) refuse(what, ": fp32, bf16 or fp16, got ", x.scalar_type());
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > MAX_CHANNELS) refuse(what, ": [..., channels] with 1 .. ", MAX_CHANNELS, " channels, got ", x.sizes());
}
void check_vectors(Tensor& weight, Tensor& bias, double eps, const Tensor& x, const char* what) {
    if (!(eps >= 0.0)) refuse(what, ": eps = ", eps);
    for (Tensor* v : {&weight, &bias}) {
        if (!v->defined()) continue;
        if (v->dim() != 1 || v->size(0) != x.size(-1) || type_of(*v) < 0 || v->device() != x.device())
            refuse(what, ": weight and bias have one value per channel (", x.size(-1), ") in fp32, bf16 or fp16 on ", x.device(), ", got ", described(*v));
        if (v->is_neg()) *v = v->resolve_neg();
        if (!v->is_contiguous()) *v = v->contiguous();
    }
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
        refuse(what, ": weight (", weight.scalar_type(), ") and bias (", bias.scalar_type(), ") have one type");
}

// ------------------------------------------------------------------------------------------------------------------------ Python calls
// The kernels read addresses, and autograd's forward mode does not see that: the derivative would be dropped without a word.
void check_forward_mode(const Tensor& t, const char* what) {
    if (t._fw_grad(0).defined()) refuse(what, ": no forward-mode derivative (an input is a dual tensor)");
}
// torch.jit.trace does not see them either, and would keep the outputs of the example as constants.
void check_trace(const char* what) {
    if (at::tracer::impl::is_dispatch_enabled()) refuse(what, ": torch.jit.trace cannot record it");
}
Tensor tensor_of(PyObject* o, const char* what) {
    if (o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) refuse(what, ": a tensor or None, got ", Py_TYPE(o)->tp_name);
    const Tensor& t = THPVariable_Unpack(o);
    check_forward_mode(t, what);
    return t;
}
void sinks_of(PyObject* o, Tensor (&sinks)[4]) {                      // None, or 4 tensors / Nones
    if (o == Py_None) return;
    for (int i = 0; i < 4; ++i) sinks[i] = tensor_of(PyTuple_GetItem(o, i), "sink");
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); refuse("a number is wanted, got ", Py_TYPE(o)->tp_name); }
    return v;
}
// no C++ exception leaves a call
template <typename F> PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    } catch (python_error& e) {                                       // from a hook on saved tensors (re-computation ends its pass with one)
        e.restore();
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(memory_error ? memory_error : PyExc_MemoryError, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "codeps_amd._bind: unknown error");
    }
    return nullptr;
}
bool count(Py_ssize_t got, Py_ssize_t want) {
    if (got == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are wanted", got, want);
    return false;
}

// channel_norm(x, weight, bias, kind, eps, sinks)
PyObject* py_channel_norm(PyObject*, PyObject* const* a, Py_ssize_t na) {
    if (!count(na, 6)) return nullptr;
    return guarded([&]() -> PyObject* {
        const char* what = "channel_norm";
        check_trace(what);
        Norm n;
        n.x = tensor_of(a[0], what);
        if (!n.x.defined()) refuse(what, ": x is None");
        n.weight = tensor_of(a[1], what);
        n.bias = tensor_of(a[2], what);
        n.d.kind = (int)PyLong_AsLong(a[3]);
        const double eps = number(a[4]);
        check_rows(n.x, what);
        check_vectors(n.weight, n.bias, eps, n.x, what);
        n.d.eps = (float)eps;
        n.d.scale = 1.f;
        n.d.rows_per_item = 1;
        Tensor sinks[4];
        sinks_of(a[5], sinks);
        apply(n, sinks);
        return THPVariable_Wrap(n.h);
    });
}

// channel_norm_residual(x, residual, weight, bias, kind, eps, gate, act, scale, next_kind, next_weight, next_bias, next_eps, sinks)
PyObject* py_channel_norm_residual(PyObject*, PyObject* const* a, Py_ssize_t na) {
    if (!count(na, 14)) return nullptr;
    return guarded([&]() -> PyObject* {
        const char* what = "channel_norm_residual";
        check_trace(what);
        Norm n;
        auto& d = n.d;
        n.x = tensor_of(a[0], what);
        if (!n.x.defined()) refuse(what, ": x is None");
        n.residual = tensor_of(a[1], what);
        n.weight = tensor_of(a[2], what);
        n.bias = tensor_of(a[3], what);
        d.full = 1;
        d.kind = (int)PyLong_AsLong(a[4]);
        const double eps = number(a[5]), next_eps = number(a[12]);
        n.gate = tensor_of(a[6], what);
        d.gate_act = (int)PyLong_AsLong(a[7]);
        d.scale = (float)number(a[8]);
        d.next_kind = (int)PyLong_AsLong(a[9]);
        n.next_weight = tensor_of(a[10], what);
        n.next_bias = tensor_of(a[11], what);
        d.eps = (float)eps;
        d.next_eps = (float)next_eps;
        const Tensor& x = n.x;
        check_rows(x, what);
        check_vectors(n.weight, n.bias, eps, x, what);
        check_vectors(n.next_weight, n.next_bias, next_eps, x, what);
        if (!d.next_kind && (n.next_weight.defined() || n.next_bias.defined())) refuse(what, ": next_weight / next_bias without next_kind");
        const Tensor& r = n.residual;
        if (r.defined() && (r.sizes() != x.sizes() || r.device() != x.device() || (r.scalar_type() != x.scalar_type() && r.scalar_type() != at::kFloat)))
            refuse(what, ": residual has x's shape and device, and x's type or fp32: got ", described(r), " for ", described(x));
        const int64_t c = x.size(-1);
        const Tensor& g = n.gate;
        d.rows_per_item = 1;
        if (!g.defined()) {
            if (d.gate_act) refuse(what, ": gate_act goes with a gate");
        } else {
            if (type_of(g) < 0 || g.device() != x.device() || g.dim() < 1 || g.size(-1) != c)
                refuse(what, ": gate [..., ", c, "] in fp32, bf16 or fp16 on ", x.device(), ", got ", described(g));
            const bool item = x.dim() > 2 && (g.dim() == 2 || g.dim() == x.dim()) && g.size(0) == x.size(0) && g.numel() == g.size(0) * c;
            if (g.dim() == 1) {
                d.gate_mode = CODEPS_GATE_CHANNEL;
            } else if (g.sizes() == x.sizes() && (g.scalar_type() == x.scalar_type() || !item)) {
                d.gate_mode = CODEPS_GATE_ELEMENT;
                if (g.scalar_type() != x.scalar_type()) refuse(what, ": a gate of x's shape has x's type, got ", g.scalar_type(), " for ", x.scalar_type());
            } else if (item) {                                        // (items of one row each: x's shape as well, but of any type)
                d.gate_mode = CODEPS_GATE_ITEM;
                const int64_t rows = x.numel() / c;
                d.rows_per_item = (int32_t)std::max<int64_t>(1, std::min<int64_t>(rows / std::max<int64_t>(1, x.size(0)), INT32_MAX));
            } else {
                refuse(what, ": gate is [", c, "], one row per item of x's first dimension, or x's shape: got ", g.sizes(), " for ", x.sizes());
            }
        }
        Tensor sinks[4];
        sinks_of(a[13], sinks);
        apply(n, sinks);
        if (!d.next_kind) return THPVariable_Wrap(n.y);
        PyObject *y = THPVariable_Wrap(n.y), *h = THPVariable_Wrap(n.h);
        PyObject* both = y && h ? PyTuple_Pack(2, y, h) : nullptr;
        Py_XDECREF(y);
        Py_XDECREF(h);
        return both;
    });
}

// ---- lists of gradients
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

struct Sequence {                                                     // a list or tuple, or anything that becomes one
    PyObject* seq;
    explicit Sequence(PyObject* o) : seq(PySequence_Fast(o, "")) {
        if (!seq) { PyErr_Clear(); refuse("a list of tensors is wanted, got ", Py_TYPE(o)->tp_name); }
    }
    ~Sequence() { Py_DECREF(seq); }
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq); }
    PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq, i); }
};
void check_gradient(const Tensor& g, c10::Device device, const char* what) {
    if (!g.is_cuda()) refuse("codeps_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback");
    if (type_of(g) < 0 || g.device() != device || g.layout() != at::kStrided)
        refuse(what, ": gradients are fp32, bf16 or fp16 tensors on ", device, ", got ", described(g));
}

// grad_norm(grads, scale) -> tensor
PyObject* py_grad_norm(PyObject*, PyObject* const* a, Py_ssize_t na) {
    if (!count(na, 2)) return nullptr;
    return guarded([&]() -> PyObject* {
        check_trace("grad_norm");
        const Sequence list(a[0]);
        const double scale = number(a[1]);
        std::vector<const void*> ptrs;
        std::vector<unsigned char> types;
        std::vector<long long> numels;
        std::vector<Tensor> copies;
        ptrs.reserve(list.size()); types.reserve(list.size()); numels.reserve(list.size());
        Tensor first;
        const bool recording = at::GradMode::is_enabled();
        at::NoGradGuard off;
        for (Py_ssize_t i = 0; i < list.size(); ++i) {
            if (list[i] == Py_None) continue;
            if (!THPVariable_Check(list[i])) refuse("grad_norm: tensors, got ", Py_TYPE(list[i])->tp_name);
            const Tensor& g = THPVariable_Unpack(list[i]);
            if (!first.defined()) first = g;
            check_forward_mode(g, "grad_norm");
            if (recording && g.requires_grad())
                refuse("grad_norm: the norm has no derivative and tensor ", i, " requires one: call it under torch.no_grad(), or detach them");
            check_gradient(g, first.device(), "grad_norm");
            if (dense(g)) {
                ptrs.push_back(g.data_ptr());
            } else {
                copies.push_back(g.contiguous());
                ptrs.push_back(copies.back().data_ptr());
            }
            types.push_back((unsigned char)type_of(g));
            numels.push_back(g.numel());
        }
        if (!first.defined()) refuse("grad_norm: no gradients");
        const int n = (int)ptrs.size();
        const Tensor out = at::empty({}, first.options().dtype(at::kFloat).requires_grad(false));
        const size_t bytes = api.grad_norm_bytes(n);
        const Tensor work = at::empty({(int64_t)bytes}, first.options().dtype(at::kByte).requires_grad(false));
        c10::DeviceGuard guard(first.device());
        check(api.grad_norm(ptrs.data(), types.data(), numels.data(), n, scale, (float*)out.data_ptr(), work.data_ptr(), bytes, stream_of(first)), "codeps_grad_norm");
        return THPVariable_Wrap(out);
    });
}

// What stays the same from step to step (codeps_amd.optim.AdamW fills it once, as a ctypes structure with these fields)
struct StepBlock {
    const void* items;
    long long n_items;
    const int* chunk_items;
    const long long *chunk0, *numels;
    const codeps_adamw_group* groups;
    long long n_groups;
    long long* steps;
    float *exp_avg, *exp_avg_sq;
    unsigned char *exp_avg_codes, *exp_avg_exponents, *root_codes, *root_exponents;
    float* norm;
    void* workspace;
    unsigned long long workspace_bytes, seed;
    const unsigned long long* addresses;                              // where the parameters and the tensors beside them were when the items were filled
};

// adamw_step(params, beside, grads, address of the StepBlock, grad_scale, max_norm, skip_nonfinite, ema_alpha) -> 0 when the step is launched; without a
// launch 1: a parameter or a tensor beside it (EMA, copy) has moved, 2: a gradient lies in another order than its parameter, 3: both
PyObject* py_adamw_step(PyObject*, PyObject* const* a, Py_ssize_t na) {
    if (!count(na, 8)) return nullptr;
    return guarded([&]() -> PyObject* {
        const char* what = "AdamW.step";
        check_trace(what);
        const Sequence params(a[0]), beside(a[1]), grads(a[2]);
        const StepBlock* block = PyLong_Check(a[3]) ? (const StepBlock*)PyLong_AsVoidPtr(a[3]) : nullptr;
        const Py_ssize_t n = params.size();
        if (!block) refuse(what, ": no step block");
        if (block->n_items != n) refuse(what, ": ", n, " parameters, ", block->n_items, " were listed");
        if (grads.size() != n) refuse(what, ": one gradient (or None) per parameter (", n, "), got ", grads.size());
        const double grad_scale = number(a[4]), max_norm = number(a[5]), ema_alpha = number(a[7]);
        const int skip = a[6] == Py_True;
        std::vector<const void*> ptrs(n);
        std::vector<unsigned char> types(n);
        bool moved = false, mixed = false;
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (!THPVariable_Check(params[i])) refuse(what, ": parameters are tensors, got ", Py_TYPE(params[i])->tp_name);
            const Tensor& p = THPVariable_Unpack(params[i]);
            moved = moved || (unsigned long long)(uintptr_t)p.data_ptr() != block->addresses[i] || p.numel() != block->numels[i];
            if (grads[i] == Py_None) continue;
            if (!THPVariable_Check(grads[i])) refuse(what, ": gradients are tensors or None, got ", Py_TYPE(grads[i])->tp_name);
            const Tensor& g = THPVariable_Unpack(grads[i]);
            check_gradient(g, p.device(), what);
            if (g.sizes() != p.sizes()) refuse(what, ": gradient ", i, " is ", g.sizes(), ", its parameter ", p.sizes());
            mixed = mixed || g.is_neg() || !dense(p) || !(g.strides() == p.strides() || (g.is_contiguous() && p.is_contiguous()));
            ptrs[i] = g.numel() ? g.data_ptr() : (const void*)16;                      // (an empty tensor has no address, but a gradient)
            types[i] = (unsigned char)type_of(g);
        }
        for (Py_ssize_t i = 0; i < beside.size() && !moved; ++i)
            moved = !THPVariable_Check(beside[i]) || (unsigned long long)(uintptr_t)THPVariable_Unpack(beside[i]).data_ptr() != block->addresses[n + i];
        if (moved || mixed) return PyLong_FromLong((moved ? 1 : 0) | (mixed ? 2 : 0));
        const Tensor& first = THPVariable_Unpack(params[0]);
        c10::DeviceGuard guard(first.device());
        check(api.adamw_step(block->items, (int)n, block->chunk_items, block->chunk0, ptrs.data(), types.data(), block->numels, block->groups, (int)block->n_groups,
                             block->steps, block->exp_avg, block->exp_avg_sq, block->exp_avg_codes, block->exp_avg_exponents, block->root_codes,
                             block->root_exponents, grad_scale, max_norm, skip, block->norm, block->seed, ema_alpha, block->workspace,
                             (size_t)block->workspace_bytes, stream_of(first)), "codeps_adamw_step");
        // what the kernel has rewritten: saved tensors of a graph that is still to run backward must notice, and packs of frozen weights are kept by version
        const auto rewritten = [](const Tensor& t) {
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        };
        for (Py_ssize_t i = 0; i < n; ++i) rewritten(THPVariable_Unpack(params[i]));
        for (Py_ssize_t i = 0; i < beside.size(); ++i) {              // averages (fp32; left alone with ema_alpha < 0), 16-bit copies
            const Tensor& t = THPVariable_Unpack(beside[i]);
            if (ema_alpha >= 0.0 || t.scalar_type() != at::kFloat) rewritten(t);
        }
        return PyLong_FromLong(0);
    });
}

// init(CodepsHipError, torch.OutOfMemoryError, addresses of the C entries in the order of `api`)
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t na) {
    if (!count(na, 9)) return nullptr;
    void* p[7];
    for (int i = 0; i < 7; ++i) {
        p[i] = PyLong_AsVoidPtr(a[2 + i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
            return nullptr;
        }
    }
    Py_INCREF(a[0]);
    Py_XSETREF(error_class, a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(memory_error, a[1]);
    api.last_error = (decltype(api.last_error))p[0];
    api.norm_fwd = (decltype(api.norm_fwd))p[1];
    api.norm_bwd_bytes = (decltype(api.norm_bwd_bytes))p[2];
    api.norm_bwd = (decltype(api.norm_bwd))p[3];
    api.grad_norm_bytes = (decltype(api.grad_norm_bytes))p[4];
    api.grad_norm = (decltype(api.grad_norm))p[5];
    api.adamw_step = (decltype(api.adamw_step))p[6];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"init", (PyCFunction)(void*)py_init, METH_FASTCALL, nullptr},
                         {"channel_norm", (PyCFunction)(void*)py_channel_norm, METH_FASTCALL, nullptr},
                         {"channel_norm_residual", (PyCFunction)(void*)py_channel_norm_residual, METH_FASTCALL, nullptr},
                         {"grad_norm", (PyCFunction)(void*)py_grad_norm, METH_FASTCALL, nullptr},
                         {"adamw_step", (PyCFunction)(void*)py_adamw_step, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Python side of the training-step operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) { return PyModule_Create(&module); }
