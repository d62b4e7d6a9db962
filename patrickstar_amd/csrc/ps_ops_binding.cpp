// rotate_qk, norm_rotate_qk, top_logits and distill_loss from Python arguments to the library, and their gradients from the autograd
// engine, without Python in between.
//
// A call on few tokens takes the GPU 3 to 10 us and took the host 16 (forward alone) to 160 (with its gradient) through Python: checks,
// descriptors filled field by field, functions of Python's under the autograd engine.
//
// The functions here take calls of the ordinary form only: plain tensors of the right types and shapes, on the current device, the
// elements of a row next to one another.  Whatever else they are given they leave alone and return None; the caller then goes through
// its general path (rotary.py, distill.py), which accepts or refuses it as always.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <array>
#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ps_ops.h"
#include "ps_ops_binding.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
    decltype(&ps_rotate_heads) rotate;
    decltype(&ps_norm_rotate_heads_workspace_bytes) workspace_bytes;
    decltype(&ps_norm_rotate_heads_backward) norm_backward;
    decltype(&ps_top_logits) top;
    decltype(&ps_distill_loss) distill;
    decltype(&ps_distill_loss_backward) distill_backward;
    decltype(&ps_last_error) last_error;
} library;

void check(int rc, const char* what)
{
    if (rc != 0) throw std::runtime_error(std::string(what) + " failed (code " + std::to_string(rc) + "): " + library.last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)t.get_device()).stream(); }

// ------------------------------------------------------------------------------------------------------ arguments

// A plain tensor of the GPU `device` (-1: the current one; then it is set).
bool plain(PyObject* o, int& device, Tensor& out)
{
    if (!THPVariable_CheckExact(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || !t.has_storage() || t.is_conj() || t.is_neg()) return false;
    if (device < 0) device = c10::hip::current_device();
    if (t.get_device() != device) return false;
    out = t;
    return true;
}

// The same, or None: then it stays undefined.
bool plain_or_none(PyObject* o, int& device, Tensor& out) { return o == Py_None || plain(o, device, out); }

bool element_type(const Tensor& t, int& type)
{
    switch (t.scalar_type()) {
        case at::kHalf: type = PS_F16; return true;
        case at::kBFloat16: type = PS_BF16; return true;
        case at::kFloat: type = PS_F32; return true;
        default: return false;
    }
}

bool whole(const Tensor& t, int& bytes)
{
    bytes = t.scalar_type() == at::kLong ? 8 : 4;
    return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt;
}

bool number(PyObject* o, double& out)
{
    if (PyFloat_Check(o)) {
        out = PyFloat_AS_DOUBLE(o);
        return true;
    }
    if (!PyLong_CheckExact(o)) return false;
    out = PyLong_AsDouble(o);
    if (out == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

bool integer(PyObject* o, int64_t lo, int64_t hi, int64_t& out)
{
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    out = PyLong_AsLongLongAndOverflow(o, &overflow);
    return !overflow && out >= lo && out <= hi;
}

bool differentiable(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Outputs of a gradient that is itself differentiated: an error, when that happens.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    std::shared_ptr<torch::autograd::DelayedError> error(
        new torch::autograd::DelayedError("trying to differentiate twice a function that can be differentiated once", (int64_t)grads.size()),
        torch::autograd::deleteNode);
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    return (*error)(std::move(grads));
}

// Calls f, which gives a new reference, with C++ exceptions as Python ones.
template <typename F>
PyObject* guarded(F f)
{
    try {
        return f();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown exception");
    }
    return nullptr;
}

// What f gives, made without the GIL: a launch waits where the queue is full.
template <typename F>
auto without_gil(F f)
{
    struct Back {
        PyThreadState* state = PyEval_SaveThread();
        ~Back() { PyEval_RestoreThread(state); }
    } back;
    return f();
}

std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// A tuple of the tensors; None for one that is undefined.
PyObject* tuple_of(const variable_list& tensors)
{
    PyObject* tuple = PyTuple_New((Py_ssize_t)tensors.size());
    if (!tuple) return nullptr;
    for (size_t i = 0; i < tensors.size(); ++i) {
        PyObject* t;
        if (tensors[i].defined()) {
            t = THPVariable_Wrap(tensors[i]);
        } else {
            t = Py_None;
            Py_INCREF(t);
        }
        if (!t) {
            Py_DECREF(tuple);
            return nullptr;
        }
        PyTuple_SET_ITEM(tuple, (Py_ssize_t)i, t);
    }
    return tuple;
}

// ------------------------------------------------------------------------------------------------------ rotations

struct HeadsPlan {
    int64_t axes, rotary;
    bool interleaved, norm;
    double eps;
};

Tensor rows_of(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

void strides_of(const Tensor& t, int64_t (&out)[3])
{
    const bool three = t.dim() == 3;
    out[0] = three ? 0 : t.stride(0);
    out[1] = t.stride(three ? 0 : 1);
    out[2] = t.stride(three ? 1 : 2);
}

// x: queries and keys, either may be undefined, but not both.
ps_heads_call heads_call(const Tensor (&x)[2], const Tensor (&weight)[2], const Tensor& positions, const Tensor& table, const HeadsPlan& plan)
{
    ps_heads_call c = {};
    const Tensor& some = x[x[0].defined() ? 0 : 1];
    element_type(some, c.dtype);
    c.weight_dtype = c.dtype;
    for (int w = 0; w < 2; ++w) {
        if (!x[w].defined()) continue;
        c.x[w] = x[w].data_ptr();
        c.heads[w] = (int32_t)x[w].size(-2);
        strides_of(x[w], c.x_stride[w]);
        if (weight[w].defined()) {
            c.weight[w] = weight[w].data_ptr();
            element_type(weight[w], c.weight_dtype);
        }
    }
    const bool three = some.dim() == 3, several = plan.axes > 1;
    c.positions = positions.data_ptr();
    c.plan = static_cast<const int64_t*>(table.data_ptr());
    c.position_stride[0] = several ? positions.stride(0) : 0;
    c.position_stride[1] = three ? 0 : positions.stride(several);
    c.position_stride[2] = positions.stride(several + (three ? 0 : 1));
    c.batch = three ? 1 : some.size(0);
    c.tokens = some.size(three ? 0 : 1);
    c.dim = (int32_t)some.size(-1);
    c.rotary = (int32_t)plan.rotary;
    c.axes = (int32_t)plan.axes;
    c.position_bytes = (int32_t)positions.element_size();
    c.interleaved = plan.interleaved;
    c.norm = plan.norm;
    c.eps = (float)plan.eps;
    return c;
}

void make_outputs(ps_heads_call& c, const Tensor (&like)[2], Tensor (&out)[2])
{
    for (int w = 0; w < 2; ++w) {
        if (!like[w].defined()) continue;
        out[w] = at::empty(like[w].sizes(), like[w].options());
        c.out[w] = out[w].data_ptr();
    }
}

variable_list rotate(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight, const Tensor& positions, const Tensor& table,
                     const HeadsPlan& plan, bool inverse = false)
{
    const Tensor x[2] = {q, k}, weight[2] = {q_weight, k_weight};
    Tensor out[2];
    ps_heads_call c = heads_call(x, weight, positions, table, plan);
    c.inverse = inverse;
    make_outputs(c, x, out);
    check(library.rotate(&c, stream_of(positions)), "ps_rotate_heads");
    return {out[0], out[1]};
}

int64_t packed(const HeadsPlan& p) { return p.axes << 16 | p.rotary << 2 | (int64_t)p.interleaved << 1 | (int64_t)p.norm; }
HeadsPlan unpacked(int64_t v, double eps) { return {v >> 16, v >> 2 & 0x3FFF, (v & 2) != 0, (v & 1) != 0, eps}; }

// A rotation's gradient is the gradient, turned back; with the norm the roots are made again from the inputs.
struct HeadsFunction : torch::autograd::Function<HeadsFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k, const std::optional<Tensor>& q_weight,
                                 const std::optional<Tensor>& k_weight, const Tensor& positions, const Tensor& table, const HeadsPlan& plan)
    {
        const Tensor none;
        const Tensor &kk = k ? *k : none, &wq = q_weight ? *q_weight : none, &wk = k_weight ? *k_weight : none;
        ctx->set_materialize_grads(false);
        if (plan.norm)
            ctx->save_for_backward({positions, table, q, kk, wq, wk});
        else
            ctx->save_for_backward({positions, table});
        ctx->saved_data["plan"] = packed(plan);
        ctx->saved_data["eps"] = plan.eps;
        variable_list out = rotate(q, kk, wq, wk, positions, table, plan);
        if (!kk.defined()) out.pop_back();
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(7);
        Tensor grad[2] = {grads[0], grads.size() > 1 ? grads[1] : Tensor()};
        if (!grad[0].defined() && !grad[1].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const HeadsPlan plan = unpacked(ctx->saved_data["plan"].toInt(), ctx->saved_data["eps"].toDouble());
        const c10::DeviceGuard guard(saved[0].device());
        for (Tensor& g : grad)
            if (g.defined()) g = rows_of(g);
        if (!plan.norm) {
            const variable_list turned = rotate(grad[0], grad[1], Tensor(), Tensor(), saved[0], saved[1], plan, true);
            out[0] = turned[0], out[1] = turned[1];
            return once(std::move(out));
        }
        // (an output that went nowhere has no part in it)
        Tensor x[2], weight[2], made[2];
        for (int w = 0; w < 2; ++w)
            if (grad[w].defined()) x[w] = saved[2 + w], weight[w] = saved[4 + w];
        ps_heads_call c = heads_call(x, weight, saved[0], saved[1], plan);
        make_outputs(c, x, made);
        for (int w = 0; w < 2; ++w) {
            if (!grad[w].defined()) continue;
            c.grad[w] = grad[w].data_ptr();
            strides_of(grad[w], c.grad_stride[w]);
            if (differentiable(weight[w])) {
                out[2 + w] = at::empty(weight[w].sizes(), weight[w].options());
                c.weight_grad[w] = out[2 + w].data_ptr();
            }
            out[w] = made[w];
        }
        const size_t size = library.workspace_bytes(&c);
        Tensor workspace;
        if (size) workspace = at::empty({(int64_t)size}, saved[0].options().dtype(at::kByte));
        check(library.norm_backward(&c, size ? workspace.data_ptr() : nullptr, size, stream_of(saved[0])), "ps_norm_rotate_heads_backward");
        return once(std::move(out));
    }
};

bool weight_fits(const Tensor& w, const Tensor& q)
{
    return !w.defined() || (w.dim() == 1 && w.is_contiguous() && w.size(0) == q.size(-1) && (w.scalar_type() == q.scalar_type() || w.scalar_type() == at::kFloat));
}

}  // namespace

// (q, k or None, q_weight or None, k_weight or None, positions, plan's table, axes, rotary, interleaved, norm, eps) -> (q, k or None)
PyObject* ps_ops_heads(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    int device = -1, type, bytes;
    Tensor q, k, wq, wk, positions, table;
    HeadsPlan plan;
    if (n != 11 || c10::impl::dispatch_mode_enabled() || !plain(args[0], device, q) || !plain_or_none(args[1], device, k) ||
        !plain_or_none(args[2], device, wq) || !plain_or_none(args[3], device, wk) || !plain(args[4], device, positions) ||
        !plain(args[5], device, table) || !integer(args[6], 1, 1 << 20, plan.axes) || !integer(args[7], 2, PS_MAX_HEAD_DIM, plan.rotary) ||
        !number(args[10], plan.eps))
        Py_RETURN_NONE;
    plan.interleaved = args[8] == Py_True;
    plan.norm = args[9] == Py_True;
    const int64_t dims = q.dim(), lead = dims - 2;
    if ((dims != 3 && dims != 4) || !element_type(q, type) || (q.stride(-1) != 1 && q.size(-1) != 1) || q.size(-1) > PS_MAX_HEAD_DIM ||
        q.size(-1) < plan.rotary || !whole(positions, bytes) || !(plan.eps >= 0.0))
        Py_RETURN_NONE;
    if (k.defined() && (k.scalar_type() != q.scalar_type() || k.dim() != dims || (k.stride(-1) != 1 && k.size(-1) != 1) || k.size(-1) != q.size(-1) ||
                        k.sizes().slice(0, lead) != q.sizes().slice(0, lead)))
        Py_RETURN_NONE;
    if (!k.defined() && wk.defined()) Py_RETURN_NONE;
    const int64_t several = plan.axes > 1;
    if (positions.dim() != lead + several || (several && positions.size(0) != plan.axes) || positions.sizes().slice(several) != q.sizes().slice(0, lead))
        Py_RETURN_NONE;
    if (!weight_fits(wq, q) || !weight_fits(wk, q) || (wq.defined() && wk.defined() && wq.scalar_type() != wk.scalar_type())) Py_RETURN_NONE;
    return guarded([&] {
        const variable_list out = without_gil([&]() -> variable_list {
            if (!at::GradMode::is_enabled() || !(differentiable(q) || differentiable(k) || differentiable(wq) || differentiable(wk)))
                return rotate(q, k, wq, wk, positions, table, plan);
            return HeadsFunction::apply(q, maybe(k), maybe(wq), maybe(wk), positions, table, plan);
        });
        return tuple_of({out[0], k.defined() ? out[1] : Tensor()});
    });
}

// ------------------------------------------------------------------------------------------------------ logits

namespace {

// [..., n] as [rows, n].
Tensor flat(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

// The dimensions in front of the last one.
at::IntArrayRef lead_of(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

// [rows] or [rows, n] as they are in front of the last dimension of `like`, with n behind.
Tensor spread(const Tensor& t, const Tensor& like)
{
    if (like.dim() == 2) return t;
    std::vector<int64_t> sizes = lead_of(like).vec();
    if (t.dim() == 2) sizes.push_back(t.size(1));
    return t.view(sizes);
}

}  // namespace

// (logits, k, temperature) -> (values, ids, log-sum-exp)
PyObject* ps_ops_top(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    int device = -1;
    Tensor logits;
    int64_t k;
    double temperature;
    ps_top_call c = {};
    if (n != 3 || c10::impl::dispatch_mode_enabled() || !plain(args[0], device, logits) || !integer(args[1], 1, PS_MAX_TOP, k) ||
        !number(args[2], temperature) || !element_type(logits, c.dtype) || logits.dim() < 1 || logits.numel() == 0 || logits.stride(-1) != 1 || logits.size(-1) < k ||
        logits.size(-1) > 1 << 30 || !((float)temperature > 0.0f && std::isfinite((float)temperature)))
        Py_RETURN_NONE;
    return guarded([&] {
        const variable_list out = without_gil([&]() -> variable_list {
            const Tensor rows = flat(logits.detach());
            const Tensor values = at::empty({rows.size(0), k}, rows.options());
            const Tensor ids = at::empty({rows.size(0), k}, values.options().dtype(at::kInt));
            const Tensor lse = at::empty({rows.size(0)}, values.options().dtype(at::kFloat));
            c.logits = rows.data_ptr();
            c.values = values.data_ptr();
            c.ids = static_cast<int32_t*>(ids.data_ptr());
            c.lse = static_cast<float*>(lse.data_ptr());
            c.rows = rows.size(0);
            c.vocab = rows.size(1);
            c.row_stride = rows.stride(0);
            c.k = (int32_t)k;
            c.temperature = temperature;
            check(library.top(&c, stream_of(rows)), "ps_top_logits");
            return {spread(values, logits), spread(ids, logits), spread(lse, logits)};
        });
        return tuple_of(out);
    });
}

namespace {

enum { kMean, kSum, kNone };  // distill.REDUCTIONS

struct DistillOptions {
    double label_weight, temperature;
    int64_t ignore_index;
    int reduction;
};

ps_distill_call distill_call(const Tensor& logits, const Tensor& ids, const Tensor& values, const Tensor& lse, const Tensor& labels, const DistillOptions& o)
{
    ps_distill_call c = {};
    c.logits = logits.data_ptr();
    c.ids = ids.data_ptr();
    c.values = values.data_ptr();
    if (lse.defined()) c.teacher_lse = static_cast<const float*>(lse.data_ptr());
    if (labels.defined()) {
        c.labels = labels.data_ptr();
        whole(labels, c.labels_bytes);
    }
    c.rows = logits.size(0);
    c.vocab = logits.size(1);
    c.row_stride = logits.stride(0);
    c.ids_stride = ids.stride(0);
    c.values_stride = values.stride(0);
    c.ignore_index = o.ignore_index;
    c.k = (int32_t)ids.size(1);
    element_type(logits, c.dtype);
    element_type(values, c.values_dtype);
    whole(ids, c.ids_bytes);
    c.mean = o.reduction == kMean;
    c.temperature = o.temperature;
    c.label_weight = (float)o.label_weight;
    return c;
}

struct Ahead {  // the factor that backward is going to arrive with
    bool there = false;
    Tensor tensor;
    double value = 0.0;
};

// Loss; what backward needs (stats of every row, factor of the gradient made here, denominator); that gradient.
std::array<Tensor, 3> distill(const Tensor& logits, const Tensor& ids, const Tensor& values, const Tensor& lse, const Tensor& labels,
                              const DistillOptions& o, bool backward, const Ahead& ahead)
{
    ps_distill_call c = distill_call(logits, ids, values, lse, labels, o);
    const auto options = logits.options().dtype(at::kFloat).requires_grad(false);
    const int64_t n = c.rows;
    Tensor row_loss = at::empty({n}, options), loss = row_loss, grad;
    c.row_loss = static_cast<float*>(row_loss.data_ptr());
    if (o.reduction != kNone) {
        loss = at::empty({}, options);
        c.loss = static_cast<float*>(loss.data_ptr());
    }
    const int64_t size = backward ? 4 * n + 2 : 1;
    const Tensor kept = at::empty({size}, options);
    float* at = static_cast<float*>(kept.data_ptr());
    c.denominator = at + size - 1;
    if (backward) {
        c.stats = at;
        if (ahead.there) {
            grad = at::empty({n, c.vocab}, logits.options().requires_grad(false));
            c.grad = grad.data_ptr();
            c.upstream_used = at + size - 2;
            if (ahead.tensor.defined())
                c.upstream = static_cast<const float*>(ahead.tensor.data_ptr());
            else
                c.upstream_value = (float)ahead.value;
        }
    }
    check(library.distill(&c, stream_of(logits)), "ps_distill_loss");
    return {loss, kept, grad};
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& values, const std::optional<Tensor>& lse,
                          const std::optional<Tensor>& labels, const DistillOptions& o, const Ahead& ahead)
    {
        const Tensor none;
        const Tensor &l = lse ? *lse : none, &y = labels ? *labels : none;
        const auto made = distill(logits, ids, values, l, y, o, true, ahead);
        ctx->save_for_backward({logits, ids, values, l, y, made[1]});
        if (made[2].defined()) ctx->saved_data["grad"] = made[2];
        ctx->saved_data["label_weight"] = o.label_weight;
        ctx->saved_data["temperature"] = o.temperature;
        ctx->saved_data["ignore_index"] = o.ignore_index;
        ctx->saved_data["reduction"] = (int64_t)o.reduction;
        return made[0];
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream)
    {
        const variable_list saved = ctx->get_saved_variables();
        const DistillOptions o = {ctx->saved_data["label_weight"].toDouble(), ctx->saved_data["temperature"].toDouble(),
                                  ctx->saved_data["ignore_index"].toInt(), (int)ctx->saved_data["reduction"].toInt()};
        const c10::DeviceGuard guard(saved[0].device());
        ps_distill_call c = distill_call(saved[0], saved[1], saved[2], saved[3], saved[4], o);
        float* kept = static_cast<float*>(saved[5].data_ptr());
        c.stats = kept;
        c.denominator = kept + saved[5].size(0) - 1;
        c.upstream = static_cast<const float*>(upstream[0].data_ptr());
        c.upstream_stride = upstream[0].dim() ? upstream[0].stride(0) : 0;
        // the gradient that forward made is handed out once: whoever gets it may write to it
        Tensor grad;
        const auto made = ctx->saved_data.find("grad");
        if (made != ctx->saved_data.end()) {
            grad = made->second.toTensor();
            ctx->saved_data.erase(made);
            c.upstream_used = kept + saved[5].size(0) - 2;
        } else {
            grad = at::empty({c.rows, c.vocab}, saved[0].options().requires_grad(false));
        }
        c.grad = grad.data_ptr();
        check(library.distill_backward(&c, stream_of(saved[0])), "ps_distill_loss_backward");
        variable_list out(7);
        out[0] = grad;
        return once(std::move(out));
    }
};

}  // namespace

// (logits, ids, values, log-sum-exp or None, labels or None, label_weight, temperature, ignore_index, reduction's number, grad_scale or
// None) -> loss
PyObject* ps_ops_distill(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    int device = -1, type, bytes;
    Tensor logits, ids, values, lse, labels;
    DistillOptions o;
    Ahead ahead;
    int64_t reduction;
    if (n != 10 || c10::impl::dispatch_mode_enabled() || !plain(args[0], device, logits) || !plain(args[1], device, ids) ||
        !plain(args[2], device, values) || !plain_or_none(args[3], device, lse) || !plain_or_none(args[4], device, labels) ||
        !number(args[5], o.label_weight) || !number(args[6], o.temperature) || !integer(args[7], INT64_MIN, INT64_MAX, o.ignore_index) ||
        !integer(args[8], kMean, kNone, reduction))
        Py_RETURN_NONE;
    o.reduction = (int)reduction;
    if (logits.dim() < 1 || logits.numel() == 0 || logits.stride(-1) != 1 || !element_type(logits, type) || ids.dim() != logits.dim() ||
        lead_of(ids) != lead_of(logits) || ids.size(-1) < 1 || ids.size(-1) > PS_MAX_TOP || ids.stride(-1) != 1 || !whole(ids, bytes) ||
        values.sizes() != ids.sizes() || values.stride(-1) != 1 || !element_type(values, type))
        Py_RETURN_NONE;
    if (lse.defined() && (lse.scalar_type() != at::kFloat || lse.sizes() != lead_of(logits) || !lse.is_contiguous())) Py_RETURN_NONE;
    if (labels.defined() && (!whole(labels, bytes) || labels.sizes() != lead_of(logits) || !labels.is_contiguous())) Py_RETURN_NONE;
    if (!(o.label_weight >= 0.0 && o.label_weight <= 1.0) || (o.label_weight > 0.0 && !labels.defined()) ||
        !((float)o.temperature > 0.0f && std::isfinite((float)o.temperature)))
        Py_RETURN_NONE;
    if (args[9] != Py_None) {
        if (reduction == kNone) Py_RETURN_NONE;
        ahead.there = true;
        if (!number(args[9], ahead.value) && (!plain(args[9], device, ahead.tensor) || ahead.tensor.numel() != 1)) Py_RETURN_NONE;
    }
    return guarded([&] {
        const variable_list out = without_gil([&]() -> variable_list {
            Tensor loss;
            const Tensor rows = flat(logits), listed = flat(ids), given = flat(values.detach());
            if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
                loss = distill(rows, listed, given, lse, labels, o, false, Ahead())[0];
            } else {
                if (ahead.tensor.defined()) ahead.tensor = ahead.tensor.detach().to(at::kFloat);
                loss = DistillFunction::apply(rows, listed, given, maybe(lse.defined() ? lse.detach() : lse), maybe(labels), o, ahead);
            }
            return {o.reduction == kNone ? spread(loss, logits) : loss};
        });
        return THPVariable_Wrap(out[0]);
    });
}

// (addresses of the entry points, in the order of Library's members)
PyObject* ps_ops_use(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    int64_t at[7];
    bool good = n == 7;
    for (int i = 0; i < 7 && good; ++i) good = integer(args[i], 1, INT64_MAX, at[i]);
    if (!good) {
        PyErr_SetString(PyExc_TypeError, "ops_use takes the addresses of seven entry points");
        return nullptr;
    }
    library.rotate = reinterpret_cast<decltype(library.rotate)>(at[0]);
    library.workspace_bytes = reinterpret_cast<decltype(library.workspace_bytes)>(at[1]);
    library.norm_backward = reinterpret_cast<decltype(library.norm_backward)>(at[2]);
    library.top = reinterpret_cast<decltype(library.top)>(at[3]);
    library.distill = reinterpret_cast<decltype(library.distill)>(at[4]);
    library.distill_backward = reinterpret_cast<decltype(library.distill_backward)>(at[5]);
    library.last_error = reinterpret_cast<decltype(library.last_error)>(at[6]);
    Py_RETURN_NONE;
}
