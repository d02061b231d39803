// Python entry points of the short launches (a layer at a few images), where
// the host's time per call is what a caller waits for: the checks, the output
// tensor, the stream and the C ABI call in one native function.  Every
// function returns None for a call it does not take (other layouts, dtypes,
// tensor types, large launches, any error): the caller then runs its Python
// path, which takes or refuses the call.  One layer at one row, host time per
// call: 10.4 us through ctypes, 4.5 us here.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <unordered_set>
#include <vector>

#include "../../include/rpfq.h"

namespace {

// Launches of at least this many operations are left to the Python path,
// which chooses between more kernels; the host is not what bounds them.
constexpr double kMostOps = 1.5e9;

// The C ABI as the library that _native.load() opened exports it: this module
// links none, so that another build of the library (RPFQ_LIBRARY) serves these
// calls too.  Null until bind().
#define RPFQ_HOST_CALLS(X)                                                                              \
    X(rpfq_wide_linear_kernel) X(rpfq_row_scales) X(rpfq_wide_linear_scaled)                            \
    X(rpfq_layer_norm_wide_linear_fusable) X(rpfq_layer_norm_wide_linear) X(rpfq_act_quant_wide_linear) \
    X(rpfq_attention) X(rpfq_last_error) X(rpfq_linear_int8_workspace_bytes) X(rpfq_linear_int8)        \
    X(rpfq_linear_cross_entropy_workspace_bytes) X(rpfq_linear_cross_entropy)                           \
    X(rpfq_linear_cross_entropy_grad) X(rpfq_adamw)
struct Api {
#define X(f) decltype(&::f) f;
    RPFQ_HOST_CALLS(X)
#undef X
} api = {};
constexpr const char* kCalls[] = {
#define X(f) #f,
    RPFQ_HOST_CALLS(X)
#undef X
};
constexpr Py_ssize_t kNumCalls = sizeof(kCalls) / sizeof(kCalls[0]);
static_assert(sizeof(Api) == kNumCalls * sizeof(void*), "one pointer per call");

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return RPFQ_F32;
        case at::kHalf: return RPFQ_F16;
        case at::kBFloat16: return RPFQ_BF16;
        default: return -1;
    }
}

// A plain strided device tensor (no subclass), or NULL.
const at::Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj() ? &t : nullptr;
}

bool rows16(const at::Tensor& t) {
    return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// None or a contiguous float32 device vector of n values.
bool vec(PyObject* o, int64_t n, const float** p) {
    *p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = plain(o);
    if (!t || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() != n) return false;
    *p = t->const_data_ptr<float>();
    return true;
}

// The numbers of a call: false where o is not one (the Python error goes).
bool number(PyObject* o, int64_t* v) {
    *v = PyLong_AsLongLong(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
}
bool number(PyObject* o, float* v) {
    *v = (float)PyFloat_AsDouble(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
}

struct Call {
    const rpfq_wide_desc* d;
    const at::Tensor *blob, *x;
    const void* res = nullptr;
    int64_t m = 0;
    int xdt = 0, ydt = 0;
    at::ScalarType yt{};
    c10::SmallVector<int64_t, 6> shape;
    at::Tensor y;
    void* stream = nullptr;
    // the output and the stream, once it is known that the call is taken here
    void take() {
        y = at::empty(shape, x->options().dtype(yt));
        stream = c10::hip::getCurrentHIPStream(x->device().index()).stream();
    }
};

// The operands the layer calls share: desc address, blob, x, residual, the
// output's dtype (None: x's).
bool layer(PyObject* desc, PyObject* blob, PyObject* x, PyObject* residual, PyObject* out_dtype, Call& c) {
    int64_t at;
    if (!api.rpfq_attention || !number(desc, &at)) return false;
    c.d = reinterpret_cast<const rpfq_wide_desc*>(at);
    c.blob = plain(blob);
    c.x = plain(x);
    if (!c.d || !c.blob || !c.x || c.x->dim() < 1) return false;
    const int64_t in = 2 * c.d->k_complex, out = 2 * c.d->n_complex;
    if (c.x->size(-1) != in || !rows16(*c.x)) return false;
    c.m = c.x->numel() / in;
    c.yt = c.x->scalar_type();
    if (out_dtype != Py_None) {
        if (!THPDtype_Check(out_dtype)) return false;
        c.yt = reinterpret_cast<THPDtype*>(out_dtype)->scalar_type;
    }
    c.xdt = dtype_code(c.x->scalar_type());
    c.ydt = dtype_code(c.yt);
    if (c.m < 1 || c.xdt < 0 || c.ydt < 0 || 2.0 * (double)c.m * (double)in * (double)out >= kMostOps) return false;
    c.shape.assign(c.x->sizes().begin(), c.x->sizes().end());
    c.shape.back() = out;
    if (residual != Py_None) {
        const at::Tensor* r = plain(residual);
        if (!r || r->scalar_type() != c.yt || r->sizes() != at::IntArrayRef(c.shape) || !rows16(*r)) return false;
        c.res = r->data_ptr();
    }
    return true;
}

// Allocations and launches run without the interpreter lock, as through torch
// and ctypes: one that waits for memory or for room in the queue must not hold
// up the other threads, or a host function in that queue that needs the lock.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* done(int rc, const at::Tensor& y) {
    if (rc != RPFQ_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
}

// linear(desc, blob, x, bias, residual, out_dtype, flags, guard): guard bit 0:
// float32 / bf16 rows get their prescales, bit 1: rows that go to the DMA
// kernel as prescaled fp16 (many rows) are left to the Python path.
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Call c;
    const float* bias;
    int64_t flags, guard;
    if (n != 8 || !number(a[6], &flags) || !number(a[7], &guard) || !layer(a[0], a[1], a[2], a[4], a[5], c) ||
        !vec(a[3], 2 * c.d->n_complex, &bias))
        Py_RETURN_NONE;
    const int64_t in = 2 * c.d->k_complex;
    const bool scaled = c.xdt != RPFQ_F16 && (guard & 1);
    int kernel = -1;
    if (scaled && (guard & 2) && in <= 4096 &&
        api.rpfq_wide_linear_kernel(c.d, c.m, RPFQ_F16, c.ydt, (int)flags, &kernel) == RPFQ_OK && kernel == RPFQ_KERNEL_DMA)
        Py_RETURN_NONE;
    int rc = RPFQ_OK;
    {
        Unlocked u;
        c.take();
        at::Tensor s;
        if (scaled) {
            s = at::empty({c.m}, c.x->options().dtype(at::kFloat));
            rc = api.rpfq_row_scales(c.x->data_ptr(), c.xdt, c.m, in, s.data_ptr<float>(), c.stream);
        }
        if (rc == RPFQ_OK)
            rc = api.rpfq_wide_linear_scaled(c.d, c.blob->data_ptr(), c.blob->nbytes(), c.x->data_ptr(), c.xdt, c.m,
                                             scaled ? s.const_data_ptr<float>() : nullptr, bias, c.res, c.y.data_ptr(),
                                             c.ydt, (int)flags, c.stream);
    }
    return done(rc, c.y);
    END_HANDLE_TH_ERRORS
}

// layer_norm_linear(desc, blob, x, ln_weight, ln_bias, eps, bias, out_dtype, flags)
// where the launch takes the LayerNorm in its prologue.
PyObject* layer_norm_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Call c;
    const float *w, *b, *bias;
    float eps;
    int64_t flags;
    int fusable = 0;
    if (n != 9 || !number(a[5], &eps) || !number(a[8], &flags) || !layer(a[0], a[1], a[2], Py_None, a[7], c)) Py_RETURN_NONE;
    const int64_t in = 2 * c.d->k_complex;
    if (!vec(a[3], in, &w) || !vec(a[4], in, &b) || !vec(a[6], 2 * c.d->n_complex, &bias) ||
        api.rpfq_layer_norm_wide_linear_fusable(c.d, c.m, c.xdt, c.ydt, &fusable) != RPFQ_OK || !fusable)
        Py_RETURN_NONE;
    int rc;
    {
        Unlocked u;
        c.take();
        rc = api.rpfq_layer_norm_wide_linear(c.d, c.blob->data_ptr(), c.blob->nbytes(), c.x->data_ptr(), c.xdt, c.m, w, b,
                                             eps, bias, c.y.data_ptr(), c.ydt, (int)flags, c.stream);
    }
    return done(rc, c.y);
    END_HANDLE_TH_ERRORS
}

// act_quant_linear(desc, blob, x, bits, bias, residual, out_dtype, flags) where
// the launch takes the act quant in its prologue.
PyObject* act_quant_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Call c;
    const float* bias;
    int64_t bits, flags;
    int fusable = 0;
    if (n != 8 || !number(a[3], &bits) || !number(a[7], &flags) || !layer(a[0], a[1], a[2], a[5], a[6], c) || !vec(a[4], 2 * c.d->n_complex, &bias) ||
        api.rpfq_layer_norm_wide_linear_fusable(c.d, c.m, c.xdt, c.ydt, &fusable) != RPFQ_OK || !fusable)
        Py_RETURN_NONE;
    int rc;
    {
        Unlocked u;
        c.take();
        rc = api.rpfq_act_quant_wide_linear(c.d, c.blob->data_ptr(), c.blob->nbytes(), c.x->data_ptr(), c.xdt, c.m,
                                            (int)bits, 0, nullptr, nullptr, 0.0f, bias, c.res, c.y.data_ptr(), c.ydt,
                                            (int)flags, c.stream);
    }
    return done(rc, c.y);
    END_HANDLE_TH_ERRORS
}

// attention(qkv, heads, scale)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t h;
    float scale;
    if (n != 3 || !number(a[1], &h) || !number(a[2], &scale)) Py_RETURN_NONE;
    const at::Tensor* q = api.rpfq_attention ? plain(a[0]) : nullptr;
    if (!q || q->dim() != 3 || h < 1 || q->size(2) != 192 * h ||
        q->numel() == 0 || !rows16(*q))
        Py_RETURN_NONE;
    at::Tensor y;
    int rc;
    {
        Unlocked u;
        y = at::empty({q->size(0), q->size(1), 64 * h}, q->options());
        rc = api.rpfq_attention(q->data_ptr(), dtype_code(q->scalar_type()), q->size(0), q->size(1), h, 64, scale,
                                y.data_ptr(), c10::hip::getCurrentHIPStream(q->device().index()).stream());
    }
    return done(rc, y);
    END_HANDLE_TH_ERRORS
}

bool needs_grad(const at::Tensor* t) { return t && t->defined() && at::GradMode::is_enabled() && t->requires_grad(); }

// Tensors that stand for others (vmap, dual numbers) are left to torch's own rules.
bool transformed(const at::Tensor& t) {
    constexpr c10::DispatchKeySet keys{c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                       c10::DispatchKey::Batched, c10::DispatchKey::Functionalize};
    return t.key_set().has_any(keys) || t._fw_grad(0).defined();
}

at::ScalarType dtype_or(PyObject* o, at::ScalarType t) {
    if (o == Py_None) return t;
    return THPDtype_Check(o) ? reinterpret_cast<THPDtype*>(o)->scalar_type : at::ScalarType::Undefined;
}

void* stream_on(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// linear_int8(x, weight, weight_scale, bias, out_dtype)
PyObject* linear_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const float *scale, *bias;
    const at::Tensor* x = n == 5 && api.rpfq_linear_int8 ? plain(a[0]) : nullptr;
    const at::Tensor* w = x ? plain(a[1]) : nullptr;
    if (!w || x->dim() < 1 || w->dim() != 2 || w->scalar_type() != at::kChar || x->size(-1) != w->size(1) || !rows16(*x) ||
        x->numel() == 0 || (w->size(1) > 1 && w->stride(1) != 1) || w->size(0) < 1 || transformed(*x))
        Py_RETURN_NONE;
    const int64_t out = w->size(0), k = w->size(1), m = x->numel() / k;
    const int64_t ld = out > 1 ? w->stride(0) : std::max(k, w->stride(0));
    if (ld > 1 << 20) Py_RETURN_NONE;  // rows further apart than the library takes are copied
    // rows are read in whole 16 bytes: the last one's too have to be there (rows
    // of exactly K that do not fill them are copied by the library)
    if (ld >= (k + 15) / 16 * 16 &&
        (size_t)(w->storage_offset() + (out - 1) * ld + (k + 15) / 16 * 16) > w->storage().nbytes())
        Py_RETURN_NONE;
    const at::ScalarType yt = dtype_or(a[4], x->scalar_type());
    const int xdt = dtype_code(x->scalar_type()), ydt = dtype_code(yt);
    const at::Tensor* b = a[3] == Py_None ? nullptr : plain(a[3]);
    if (xdt < 0 || ydt < 0 || ld < k || !vec(a[2], out, &scale) || !scale || !vec(a[3], out, &bias) || needs_grad(x) ||
        needs_grad(b) || w->device() != x->device() || plain(a[2])->device() != x->device() ||
        (b && b->device() != x->device()) || plain(a[2])->dim() != 1 || (b && b->dim() != 1))
        Py_RETURN_NONE;
    at::Tensor y;
    int rc;
    {
        Unlocked u;
        const c10::DeviceGuard guard(x->device());
        c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
        shape.back() = out;
        y = at::empty(shape, x->options().dtype(yt));
        const int8_t* wp = reinterpret_cast<const int8_t*>(w->data_ptr());
        const size_t bytes = api.rpfq_linear_int8_workspace_bytes(x->data_ptr(), xdt, m, out, k, wp, ld);
        at::Tensor work;
        if (bytes) work = at::empty({(int64_t)bytes}, x->options().dtype(at::kByte));
        rc = api.rpfq_linear_int8(x->data_ptr(), xdt, nullptr, wp, ld, scale, bias, m, out, k, y.data_ptr(), ydt,
                                  bytes ? work.data_ptr() : nullptr, bytes, stream_on(*x));
    }
    return done(rc, y);
    END_HANDLE_TH_ERRORS
}

// The cross entropy of a classifier under autograd, as ops._LinearCrossEntropy.
struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
    static rpfq_ce_desc describe(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, int64_t ignore,
                                 double smoothing, int64_t reduction) {
        return {x.size(0), w.size(0), x.size(1), ignore, dtype_code(x.scalar_type()),
                bias.defined() ? dtype_code(bias.scalar_type()) : RPFQ_F32, (int32_t)reduction, (float)smoothing};
    }
    static void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

    // (loss, stat)
    static std::pair<at::Tensor, at::Tensor> loss(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target,
                                                  const at::Tensor& bias, const rpfq_ce_desc& d) {
        const c10::DeviceGuard guard(x.device());
        const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
        at::Tensor stat = at::empty({3 * d.M + 1}, f32);
        at::Tensor out = d.reduction == RPFQ_REDUCE_NONE ? at::empty({d.M}, f32) : at::empty({}, f32);
        const size_t bytes = api.rpfq_linear_cross_entropy_workspace_bytes(&d, 0);
        at::Tensor work = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
        float* s = stat.data_ptr<float>();
        const int rc = api.rpfq_linear_cross_entropy(&d, x.data_ptr(), w.data_ptr(), ptr(bias), target.data_ptr<int64_t>(),
                                                     out.data_ptr<float>(), s, s + 3 * d.M, work.data_ptr(), bytes,
                                                     stream_on(x));
        TORCH_CHECK(rc == RPFQ_OK, "rpfq_linear_cross_entropy: ", api.rpfq_last_error());
        return {out, stat};
    }

    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                              const at::Tensor& target, const std::optional<at::Tensor>& given, int64_t ignore,
                              double smoothing, int64_t reduction) {
        const at::Tensor bias = given ? *given : at::Tensor();
        auto [out, stat] = loss(x, w, target, bias, describe(x, w, bias, ignore, smoothing, reduction));
        ctx->save_for_backward({x, w, target, bias, stat});
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["smoothing"] = smoothing;
        ctx->saved_data["reduction"] = reduction;
        return out;
    }

    // Under capture: whether the engine, here or further on, would hand a gradient
    // to a leaf on the default stream, where an eager graph that is still alive has
    // bound it; joining that stream to the capture ends the process, not the call.
    // grad() hands it over too, before it takes it out.
    static bool leaves_capture() {
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return false;
        const auto* only = torch::autograd::get_current_graph_task_exec_info();  // not empty: of grad() and backward(inputs=)
        const auto here = torch::autograd::get_current_node();
        if (!here) return false;
        std::vector<torch::autograd::Node*> todo{here.get()};
        std::unordered_set<torch::autograd::Node*> seen;
        while (!todo.empty()) {
            const auto* node = todo.back();
            todo.pop_back();
            for (const auto& edge : node->next_edges()) {
                auto* next = edge.function.get();
                if (!next || !seen.insert(next).second) continue;
                if (!dynamic_cast<torch::autograd::AccumulateGrad*>(next)) {
                    todo.push_back(next);
                    continue;
                }
                if (only && !only->empty()) {
                    const auto found = only->find(next);
                    if (found == only->end() || !found->second.should_execute()) continue;
                }
                const auto s = next->stream();
                if (s && s->id() == 0) return true;  // the default stream
            }
        }
        return false;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!leaves_capture(), "linear_cross_entropy: backward under capture while an eager graph of the same leaves is "
                    "alive: let go of its outputs first");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &target = saved[2], &bias = saved[3], &stat = saved[4];
        const c10::DeviceGuard guard(x.device());
        const rpfq_ce_desc d = describe(x, w, bias, ctx->saved_data["ignore"].toInt(), ctx->saved_data["smoothing"].toDouble(),
                                        ctx->saved_data["reduction"].toInt());
        torch::autograd::variable_list out(7);
        at::Tensor gx, gw, gb;
        {
            const at::NoGradGuard plain_results;
            const at::Tensor g = grads[0].to(at::kFloat).contiguous();
            if (ctx->needs_input_grad(0)) gx = at::empty(x.sizes(), x.options());
            if (ctx->needs_input_grad(1)) gw = at::empty(w.sizes(), w.options());
            if (bias.defined() && ctx->needs_input_grad(3)) gb = at::empty(bias.sizes(), bias.options());
            if (!gx.defined() && !gw.defined() && !gb.defined()) return out;
            const size_t bytes = api.rpfq_linear_cross_entropy_workspace_bytes(&d, 1);
            at::Tensor work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
            const float* s = stat.const_data_ptr<float>();
            const int rc = api.rpfq_linear_cross_entropy_grad(&d, x.data_ptr(), w.data_ptr(), ptr(bias),
                                                              target.data_ptr<int64_t>(), s, s + 3 * d.M,
                                                              g.const_data_ptr<float>(), ptr(gx), ptr(gw), ptr(gb),
                                                              work.data_ptr(), bytes, stream_on(x));
            TORCH_CHECK(rc == RPFQ_OK, "rpfq_linear_cross_entropy_grad: ", api.rpfq_last_error());
        }
        out[0] = gx;
        out[1] = gw;
        out[3] = gb;
        if (at::GradMode::is_enabled()) {  // create_graph: these gradients cannot be differentiated again
            auto error = std::make_shared<torch::autograd::DelayedError>(
                "linear_cross_entropy is differentiable once", (int)out.size());
            torch::autograd::variable_list wrapped(out.size());
            for (size_t i = 0; i < out.size(); ++i)
                if (out[i].defined()) {
                    at::Tensor t = out[i].detach();
                    t.requires_grad_(true);
                    wrapped[i] = t;
                }
            return (*error)(std::move(wrapped));
        }
        return out;
    }
};

// linear_cross_entropy(x, weight, target, bias, ignore_index, smoothing, reduction)
PyObject* linear_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t ignore, reduction;
    const at::Tensor* x = n == 7 && api.rpfq_linear_cross_entropy ? plain(a[0]) : nullptr;
    const at::Tensor* w = x ? plain(a[1]) : nullptr;
    const at::Tensor* t = w ? plain(a[2]) : nullptr;
    const at::Tensor* b = a[3] == Py_None ? nullptr : plain(a[3]);
    if (!t || (a[3] != Py_None && !b) || !number(a[4], &ignore) || !number(a[6], &reduction)) Py_RETURN_NONE;
    const double smoothing = PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const at::Tensor none;
    const at::Tensor& bias = b ? *b : none;
    if (x->dim() != 2 || w->dim() != 2 || x->size(1) != w->size(1) || x->numel() == 0 || w->numel() == 0 || t->dim() != 1 ||
        t->scalar_type() != at::kLong || t->size(0) != x->size(0) || !t->is_contiguous() ||
        x->scalar_type() != w->scalar_type() || dtype_code(x->scalar_type()) < 0 || !rows16(*x) || !rows16(*w) ||
        w->device() != x->device() || t->device() != x->device() || !(smoothing >= 0.0 && smoothing <= 1.0) || reduction < 0 ||
        reduction > 2 || at::autocast::is_autocast_enabled(at::kCUDA) || transformed(*x) || transformed(*w) ||
        (b && (b->dim() != 1 || b->size(0) != w->size(0) || !b->is_contiguous() || dtype_code(b->scalar_type()) < 0 ||
               b->device() != x->device() || transformed(*b))))
        Py_RETURN_NONE;
    const rpfq_ce_desc d = CrossEntropy::describe(*x, *w, bias, ignore, smoothing, reduction);
    if (!api.rpfq_linear_cross_entropy_workspace_bytes(&d, 0)) Py_RETURN_NONE;
    at::Tensor y;
    {
        Unlocked u;
        if (needs_grad(x) || needs_grad(w) || needs_grad(b))
            y = CrossEntropy::apply(*x, *w, *t, b ? std::optional<at::Tensor>(*b) : std::nullopt, ignore, smoothing, reduction);
        else
            y = CrossEntropy::loss(*x, *w, *t, bias, d).first;
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// The tensors of a list, or false where it is not a list of plain ones.
bool tensors(PyObject* list, std::vector<const at::Tensor*>& out) {
    if (!PyList_CheckExact(list)) return false;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    out.resize(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* o = PyList_GET_ITEM(list, i);
        if (!THPVariable_Check(o)) return false;  // parameters among them
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous() || t.is_inference() || t.is_neg() || t.is_conj() ||
            t.key_set().has(c10::DispatchKey::Python))
            return false;
        out[i] = &t;
    }
    return true;
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, step,
//       (lr, beta1, beta2, eps, weight_decay), lr, grad_scale, found_inf): True where
// the step was taken; lists of scales are empty with 32-bit states.
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    std::vector<const at::Tensor*> p, g, m, v, sm, sv;
    if (n != 11 || !api.rpfq_adamw || !tensors(a[0], p) || !tensors(a[1], g) || !tensors(a[2], m) || !tensors(a[3], v) ||
        !tensors(a[4], sm) || !tensors(a[5], sv) || p.empty() || !PyTuple_CheckExact(a[7]) || PyTuple_GET_SIZE(a[7]) != 5)
        Py_RETURN_NONE;
    const size_t count = p.size();
    const bool small = !sm.empty();
    if (g.size() != count || m.size() != count || v.size() != count || sm.size() != (small ? count : 0) || sv.size() != sm.size())
        Py_RETURN_NONE;
    rpfq_adamw_hyper h;
    double* field = &h.lr;
    for (int i = 0; i < 5; ++i) field[i] = PyFloat_AsDouble(PyTuple_GET_ITEM(a[7], i));
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const at::Tensor* scalar[4];  // step, lr, grad_scale, found_inf
    for (int i = 0; i < 4; ++i) {
        PyObject* o = a[i == 0 ? 6 : 7 + i];
        scalar[i] = o == Py_None ? nullptr : plain(o);
        if (o == Py_None ? i == 0 : !scalar[i] || scalar[i]->scalar_type() != at::kFloat || scalar[i]->numel() != 1) Py_RETURN_NONE;
    }
    const at::Device device = scalar[0]->device();
    for (int i = 1; i < 4; ++i)
        if (scalar[i] && scalar[i]->device() != device) Py_RETURN_NONE;
    const at::ScalarType type = p[0]->scalar_type();
    const int code = dtype_code(type);
    if (code < 0 || scalar[0]->is_inference()) Py_RETURN_NONE;
    std::vector<rpfq_adamw_tensor> table(count);
    std::vector<std::pair<const char*, const char*>> seen;  // what the step writes
    seen.reserve(5 * count + 1);
    auto writes = [&](const void* at, int64_t bytes) {
        const char* c = reinterpret_cast<const char*>(at);
        if (bytes) seen.emplace_back(c, c + bytes);
    };
    writes(scalar[0]->data_ptr(), 4);
    const int64_t es = p[0]->element_size(), ss = small ? 1 : 4;
    for (size_t i = 0; i < count; ++i) {
        const int64_t size = p[i]->numel();
        if (p[i]->scalar_type() != type || g[i]->scalar_type() != type || g[i]->sizes() != p[i]->sizes() ||
            m[i]->scalar_type() != (small ? at::kChar : at::kFloat) || v[i]->scalar_type() != (small ? at::kByte : at::kFloat) ||
            m[i]->numel() != size || v[i]->numel() != size || p[i]->device() != device || g[i]->device() != device ||
            m[i]->device() != device || v[i]->device() != device)
            Py_RETURN_NONE;
        rpfq_adamw_tensor& t = table[i];
        t = {p[i]->data_ptr(), g[i]->data_ptr(), m[i]->data_ptr(), v[i]->data_ptr(), nullptr, nullptr, size};
        if (small) {
            for (const at::Tensor* s : {sm[i], sv[i]})
                if (s->scalar_type() != at::kFloat || s->numel() != (size + 255) / 256 || s->device() != device) Py_RETURN_NONE;
            t.exp_avg_scale = sm[i]->data_ptr<float>();
            t.exp_avg_sq_scale = sv[i]->data_ptr<float>();
            writes(t.exp_avg_scale, (size + 255) / 256 * 4);
            writes(t.exp_avg_sq_scale, (size + 255) / 256 * 4);
        }
        writes(t.param, size * es);
        writes(t.exp_avg, size * ss);
        writes(t.exp_avg_sq, size * ss);
    }
    std::sort(seen.begin(), seen.end());
    for (size_t i = 1; i < seen.size(); ++i)
        if (seen[i].first < seen[i - 1].second) Py_RETURN_NONE;
    for (const rpfq_adamw_tensor& t : table) {  // gradients may share memory with each other only
        const char *first = reinterpret_cast<const char*>(t.grad), *last = first + t.numel * es;
        const auto next = std::lower_bound(seen.begin(), seen.end(), std::make_pair(last, last));
        if (first < last && next != seen.begin() && std::prev(next)->second > first) Py_RETURN_NONE;
    }
    int rc;
    {
        Unlocked u;
        const c10::DeviceGuard guard(device);
        at::Tensor work = at::empty({8}, scalar[0]->options().requires_grad(false));
        auto at_ = [&](int i) { return scalar[i] ? scalar[i]->data_ptr<float>() : nullptr; };
        rc = api.rpfq_adamw(table.data(), (int64_t)count, code, small ? 8 : 32, &h, at_(0), at_(1), at_(2), at_(3),
                            work.data_ptr<float>(), stream_on(*scalar[0]));
    }
    if (rc != RPFQ_OK) Py_RETURN_NONE;
    for (const auto* list : {&p, &m, &v, &sm, &sv})
        for (const at::Tensor* t : *list) t->unsafeGetTensorImpl()->bump_version();
    scalar[0]->unsafeGetTensorImpl()->bump_version();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// bind(addresses): the functions named by CALLS, in that order.
PyObject* bind(PyObject*, PyObject* addresses) {
    Api next;
    if (!PyTuple_Check(addresses) || PyTuple_GET_SIZE(addresses) != kNumCalls) {
        PyErr_SetString(PyExc_ValueError, "bind takes a tuple of one address per name in CALLS");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < kNumCalls; ++i) {
        void* f = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i));
        if (!f) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address");
            return nullptr;
        }
        std::memcpy(reinterpret_cast<char*>(&next) + i * sizeof(void*), &f, sizeof(f));
    }
    api = next;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {"layer_norm_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_linear)), METH_FASTCALL, nullptr},
    {"act_quant_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(act_quant_linear)), METH_FASTCALL, nullptr},
    {"linear_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_int8)), METH_FASTCALL, nullptr},
    {"linear_cross_entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_cross_entropy)), METH_FASTCALL, nullptr},
    {"adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    PyObject* m = PyModule_Create(&module);
    PyObject* names = m ? PyTuple_New(kNumCalls) : nullptr;
    for (Py_ssize_t i = 0; names && i < kNumCalls; ++i) {
        PyObject* name = PyUnicode_FromString(kCalls[i]);
        if (!name) Py_CLEAR(names);
        else PyTuple_SET_ITEM(names, i, name);
    }
    if (!names || PyModule_AddObject(m, "CALLS", names) < 0) {
        Py_XDECREF(names);
        Py_XDECREF(m);
        return nullptr;
    }
    return m;
}
