// pxg_torch.cpp -- the operators of include/pxg.h on torch tensors (_pxgtorch, used by torch_ops.py, which checks the arguments).
//
// What a training step pays for a small call is the host: an autograd node in Python costs more than its kernels.  Here a call fills
// the C structs, allocates its results and workspaces from torch's allocator (so streams and graphs own them as they own any
// tensor), launches on the current stream of the tensors' device, and the autograd nodes run without the interpreter.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <unordered_set>
#include "../../include/pxg.h"

namespace py = pybind11;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// the entry points of libpxg.so, as the ctypes binding has them loaded
struct Library {
    decltype(&pxg_decay_workspace_bytes) decay_workspace_bytes;
    decltype(&pxg_decay_forward) decay_forward;
    decltype(&pxg_decay_backward) decay_backward;
    decltype(&pxg_decay_step) decay_step;
    decltype(&pxg_top_logits) top_logits;
    decltype(&pxg_distill_forward) distill_forward;
    decltype(&pxg_distill_backward) distill_backward;
} lib;

void use_library(const std::vector<uintptr_t>& at)
{
    TORCH_CHECK(at.size() == sizeof lib / sizeof(void*), "another number of entry points");
    std::memcpy(&lib, at.data(), sizeof lib);
}

[[noreturn]] void fail(const char* what, int rc)
{
    py::gil_scoped_acquire gil;                  // an autograd thread may not hold it
    PyErr_Format(py::module_::import("poreplex_amd.native").attr("PxgError").ptr(), "%s failed (%d)", what, rc);
    throw py::error_already_set();
}

void check(const char* what, int rc)
{
    if (rc) fail(what, rc);
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int32_t dtype_of(const Tensor& t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return PXG_DT_F32;
    case at::kBFloat16: return PXG_DT_BF16;
    case at::kHalf: return PXG_DT_F16;
    default: return -1;
    }
}

// the kernels take any strides but that of the width
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

Tensor contiguous(const MaybeTensor& t) { return t && t->defined() ? t->contiguous() : Tensor(); }

template <typename V> V* data(const Tensor& t) { return t.defined() ? (V*)t.data_ptr() : nullptr; }

Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }

// A leaf's gradient is accumulated on the stream where its oldest living graph was built.  Captured on another stream, the backward
// pass would have to wait for that stream from inside the capture, which ends the process: refused here instead, for every leaf
// that the arguments come from.
void refuse_captured_leaves(std::initializer_list<const Tensor*> tensors, const Tensor& any)
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto now = c10::hip::getCurrentHIPStream(any.device().index());
    std::vector<torch::autograd::Node*> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    const auto visit = [&](torch::autograd::Node* node) {
        if (node && seen.insert(node).second) todo.push_back(node);
    };
    std::vector<std::shared_ptr<torch::autograd::Node>> held;
    for (const Tensor* t : tensors) {
        if (!t->defined() || !t->requires_grad()) continue;
        held.push_back(t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t));
        visit(held.back().get());
    }
    while (!todo.empty()) {
        torch::autograd::Node* const node = todo.back();
        todo.pop_back();
        const bool leaf = node->num_outputs() == 0;           // it passes nothing on: it accumulates
        if (leaf && node->stream() && node->stream()->id() != now.id())
            TORCH_CHECK(false, "capturing a differentiable call while a graph of the same leaf, built on another stream outside the "
                        "capture, is alive: free that graph first, or capture decay_attention_backward / "
                        "distillation_loss_and_gradient, which need no autograd graph");
        for (const auto& edge : node->next_edges()) visit(edge.function.get());
    }
}

// The autograd nodes here have no forward mode, and where no gradient is wanted there is no node at all to say so: a dual tensor's
// tangent would be dropped without a word.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors)
{
    for (const Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

// A recording of torch's own calls holds nothing of what the kernels write: its result would be an empty tensor.
void refuse_recording(const char* what)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                                what, " cannot be traced (torch.jit.trace, make_fx): a recording does not see its kernels");
}

bool wants_graph(std::initializer_list<const Tensor*> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

void refuse_second_derivative(const char* what)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), what, " has no second derivative (create_graph)");
}

// ---- decay attention --------------------------------------------------------------------------------------------------------
struct DecayCall {
    pxg_decay s = {};
    Tensor q, k, v, log_decay, lengths, initial;      // what the pointers point at

    static pxg_sequence sequence(const Tensor& t)
    {
        pxg_sequence r = {t.data_ptr(), t.stride(0), t.dim() == 4 ? t.stride(1) : 0, t.stride(t.dim() - 2)};
        return r;
    }
    // [batch, steps, heads, width], or one step without the second axis
    DecayCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay_, const MaybeTensor& lengths_,
              const MaybeTensor& initial_)
        : q(rows(q_)), k(rows(k_)), v(rows(v_)), log_decay(log_decay_.contiguous()), lengths(contiguous(lengths_)),
          initial(contiguous(initial_))
    {
        s.struct_bytes = sizeof s, s.dtype = dtype_of(q);
        s.batch = q.size(0), s.steps = q.dim() == 4 ? q.size(1) : 1, s.heads = (int32_t)q.size(q.dim() - 2);
        s.dk = (int32_t)q.size(-1), s.dv = (int32_t)v.size(-1);
        s.q = sequence(q), s.k = sequence(k), s.v = sequence(v);
        s.log_decay = data<float>(log_decay), s.initial_state = data<float>(initial);
        s.lengths = data<void>(lengths), s.lengths_are_64 = lengths.defined() && lengths.scalar_type() == at::kLong;
    }
    Tensor workspace(int backward)
    {
        const int64_t n = lib.decay_workspace_bytes(&s, backward);
        if (n < 0) fail("pxg_decay_workspace_bytes", (int)n);
        if (n == 0) return {};
        Tensor t = empty({n}, q, at::kByte);
        s.workspace = t.data_ptr(), s.workspace_bytes = n;
        return t;
    }
    Tensor new_state() const { return empty({s.batch, s.heads, s.dk, s.dv}, q, at::kFloat); }
};

std::pair<Tensor, Tensor> decay_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                        const MaybeTensor& lengths, const MaybeTensor& initial, bool want_state)
{
    const c10::DeviceGuard device(q.device());
    DecayCall c(q, k, v, log_decay, lengths, initial);
    Tensor out = empty(v.sizes(), v, v.scalar_type()), state;
    c.s.out = out.data_ptr();
    if (want_state) state = c.new_state(), c.s.final_state = data<float>(state);
    const Tensor work = c.workspace(0);
    check("pxg_decay_forward", lib.decay_forward(&c.s, stream_of(q)));
    return {out, state};
}

struct DecayGradients {
    Tensor q, k, v, log_decay, initial;
};

DecayGradients decay_backward(const Tensor& grad_out_, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                              const MaybeTensor& lengths, const MaybeTensor& initial, const MaybeTensor& grad_state_, bool want_decay,
                              bool want_initial)
{
    const c10::DeviceGuard device(q.device());
    DecayCall c(q, k, v, log_decay, lengths, initial);
    const Tensor grad_out = rows(grad_out_), grad_state = contiguous(grad_state_);
    c.s.grad_out = DecayCall::sequence(grad_out), c.s.grad_final_state = data<float>(grad_state);
    DecayGradients g;
    g.q = empty(q.sizes(), q, q.scalar_type()), g.k = empty(k.sizes(), k, k.scalar_type()), g.v = empty(v.sizes(), v, v.scalar_type());
    c.s.grad_q = g.q.data_ptr(), c.s.grad_k = g.k.data_ptr(), c.s.grad_v = g.v.data_ptr();
    if (want_decay) g.log_decay = empty(log_decay.sizes(), log_decay, at::kFloat), c.s.grad_log_decay = data<float>(g.log_decay);
    if (want_initial) g.initial = c.new_state(), c.s.grad_initial_state = data<float>(g.initial);
    const Tensor work = c.workspace(1);
    check("pxg_decay_backward", lib.decay_backward(&c.s, stream_of(q)));
    return g;
}

struct DecayAttention : torch::autograd::Function<DecayAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                 const MaybeTensor& initial, const MaybeTensor& lengths, bool want_state)
    {
        auto [out, state] = decay_forward(q, k, v, log_decay, lengths, initial, want_state);
        ctx->save_for_backward({q, k, v, log_decay, initial.value_or(Tensor()), lengths.value_or(Tensor())});
        ctx->set_materialize_grads(false);
        return want_state ? variable_list{out, state} : variable_list{out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        refuse_second_derivative("decay_attention");
        const auto t = ctx->get_saved_variables();
        Tensor grad_out = grads[0], grad_state = grads.size() > 1 ? grads[1] : Tensor();
        variable_list r(7);
        if (!grad_out.defined() && !grad_state.defined()) return r;
        if (!grad_out.defined()) grad_out = at::zeros_like(t[2], at::MemoryFormat::Contiguous);
        const auto g = decay_backward(grad_out, t[0], t[1], t[2], t[3], t[5], t[4], grad_state, ctx->needs_input_grad(3),
                                      t[4].defined() && ctx->needs_input_grad(4));
        if (ctx->needs_input_grad(0)) r[0] = g.q;
        if (ctx->needs_input_grad(1)) r[1] = g.k;
        if (ctx->needs_input_grad(2)) r[2] = g.v;
        r[3] = g.log_decay, r[4] = g.initial;
        return r;
    }
};

std::pair<Tensor, MaybeTensor> decay_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                               const MaybeTensor& lengths, const MaybeTensor& initial, bool want_state)
{
    const Tensor start = initial.value_or(Tensor());
    refuse_recording("decay_attention");
    refuse_tangents("decay_attention", {&q, &k, &v, &log_decay, &start});
    Tensor out, state;
    if (wants_graph({&q, &k, &v, &log_decay, &start})) {
        refuse_captured_leaves({&q, &k, &v, &log_decay, &start}, q);
        const variable_list r = DecayAttention::apply(q, k, v, log_decay, initial, lengths, want_state);
        out = r[0];
        if (want_state) state = r[1];
    } else {
        std::tie(out, state) = decay_forward(q, k, v, log_decay, lengths, initial, want_state);
    }
    return {out, want_state ? MaybeTensor(state) : std::nullopt};
}

py::tuple decay_attention_backward(const Tensor& grad_out, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                   const MaybeTensor& lengths, const MaybeTensor& initial, const MaybeTensor& grad_state)
{
    at::NoGradGuard no_grad;
    const Tensor start = initial.value_or(Tensor()), end = grad_state.value_or(Tensor());
    refuse_recording("decay_attention_backward");
    refuse_tangents("decay_attention_backward", {&grad_out, &q, &k, &v, &log_decay, &start, &end});
    const auto g = decay_backward(grad_out, q, k, v, log_decay, lengths, initial, grad_state, true, initial.has_value());
    return py::make_tuple(g.q, g.k, g.v, g.log_decay, initial ? py::cast(g.initial) : py::object(py::none()));
}

Tensor decay_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const MaybeTensor& active_)
{
    at::NoGradGuard no_grad;
    refuse_recording("decay_attention_step");
    refuse_tangents("decay_attention_step", {&q, &k, &v, &log_decay, &state});
    const c10::DeviceGuard device(q.device());
    DecayCall c(q, k, v, log_decay, std::nullopt, std::nullopt);
    const Tensor active = contiguous(active_), out = empty(v.sizes(), v, v.scalar_type());
    c.s.lengths = data<void>(active), c.s.out = out.data_ptr(), c.s.final_state = data<float>(state);
    state.unsafeGetTensorImpl()->bump_version();      // written in place; first, for this is what refuses a state of inference mode
    check("pxg_decay_step", lib.decay_step(&c.s, stream_of(q)));
    return out;
}

// ---- learning from a teacher ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& logits_, int64_t k, double temperature)
{
    at::NoGradGuard no_grad;
    refuse_recording("top_logits");
    const c10::DeviceGuard device(logits_.device());
    const Tensor logits = rows(logits_);
    const int64_t n = logits.size(0);
    Tensor values = empty({n, k}, logits, logits.scalar_type()), indices = empty({n, k}, logits, at::kInt), rest = empty({n}, logits, at::kFloat);
    check("pxg_top_logits", lib.top_logits(dtype_of(logits), n, logits.size(1), logits.data_ptr(), logits.stride(0), (int32_t)k,
                                           (float)temperature, values.data_ptr(), data<int32_t>(indices), data<float>(rest),
                                           stream_of(logits)));
    return {values, indices, rest};
}

enum Reduction { MEAN, SUM, NONE };

struct DistillCall {
    pxg_distill s = {};
    Tensor logits, values, indices, rest, weight;

    DistillCall(const Tensor& logits_, const Tensor& values_, const Tensor& indices_, const MaybeTensor& rest_, const MaybeTensor& weight_,
                double temperature, int reduction)
        : logits(rows(logits_)), values(values_.contiguous()), indices(indices_.contiguous()), rest(contiguous(rest_)),
          weight(contiguous(weight_))
    {
        s.struct_bytes = sizeof s, s.dtype = dtype_of(logits);
        s.rows = logits.size(0), s.classes = logits.size(1), s.row_stride = logits.stride(0);
        s.logits = logits.data_ptr(), s.k = (int32_t)values.size(1), s.value_dtype = dtype_of(values);
        s.values = values.data_ptr(), s.indices = indices.data_ptr(), s.indices_are_64 = indices.scalar_type() == at::kLong;
        s.rest = data<float>(rest), s.weight = data<float>(weight);
        s.temperature = (float)temperature, s.mean = reduction == MEAN;
    }
};

// (loss, what the backward pass needs)
std::pair<Tensor, Tensor> distill_forward(const Tensor& logits, const Tensor& values, const Tensor& indices, const MaybeTensor& rest,
                                          const MaybeTensor& weight, double temperature, int reduction)
{
    const c10::DeviceGuard device(logits.device());
    DistillCall c(logits, values, indices, rest, weight, temperature, reduction);
    const int64_t n = c.s.rows, stats = n * (4 + c.s.k);
    Tensor held = empty({stats + (reduction == NONE ? 0 : n)}, logits, at::kFloat);
    Tensor loss = reduction == NONE ? empty({n}, logits, at::kFloat) : empty({}, logits, at::kFloat);
    c.s.stats = data<float>(held);
    c.s.row_loss = reduction == NONE ? data<float>(loss) : c.s.stats + stats;
    c.s.loss = reduction == NONE ? nullptr : data<float>(loss);
    check("pxg_distill_forward", lib.distill_forward(&c.s, stream_of(logits)));
    return {loss, held};
}

Tensor distill_backward(const Tensor& grad_loss_, const Tensor& logits, const Tensor& values, const Tensor& indices,
                        const MaybeTensor& weight, const Tensor& held, double temperature, int reduction)
{
    const c10::DeviceGuard device(logits.device());
    DistillCall c(logits, values, indices, std::nullopt, weight, temperature, reduction);
    const Tensor grad_loss = grad_loss_.to(at::kFloat).contiguous(), grad = empty(logits.sizes(), logits, logits.scalar_type());
    c.s.stats = data<float>(held), c.s.grad_loss = data<float>(grad_loss), c.s.grad_per_row = reduction == NONE;
    c.s.grad_logits = grad.data_ptr();
    check("pxg_distill_backward", lib.distill_backward(&c.s, stream_of(logits)));
    return grad;
}

struct Distillation : torch::autograd::Function<Distillation> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& values, const Tensor& indices, const MaybeTensor& rest,
                          const MaybeTensor& weight, double temperature, int64_t reduction)
    {
        auto [loss, held] = distill_forward(logits, values, indices, rest, weight, temperature, (int)reduction);
        ctx->save_for_backward({logits, values, indices, weight.value_or(Tensor()), held});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        refuse_second_derivative("distillation_loss");
        const auto t = ctx->get_saved_variables();
        variable_list r(7);
        r[0] = distill_backward(grads[0], t[0], t[1], t[2], t[3], t[4], ctx->saved_data["temperature"].toDouble(),
                                (int)ctx->saved_data["reduction"].toInt());
        return r;
    }
};

Tensor distillation_loss(const Tensor& logits, const Tensor& values, const Tensor& indices, const MaybeTensor& rest,
                         const MaybeTensor& weight, double temperature, int reduction)
{
    const Tensor r = rest.value_or(Tensor()), w = weight.value_or(Tensor());
    refuse_recording("distillation_loss");
    refuse_tangents("distillation_loss", {&logits, &values, &r, &w});
    if (!wants_graph({&logits})) return distill_forward(logits, values, indices, rest, weight, temperature, reduction).first;
    refuse_captured_leaves({&logits}, logits);
    return Distillation::apply(logits, values, indices, rest, weight, temperature, (int64_t)reduction);
}

std::pair<Tensor, Tensor> distillation_loss_and_gradient(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                                         const MaybeTensor& rest, const MaybeTensor& weight, double temperature,
                                                         int reduction, const MaybeTensor& grad_loss)
{
    at::NoGradGuard no_grad;
    const Tensor r = rest.value_or(Tensor()), w = weight.value_or(Tensor()), from = grad_loss.value_or(Tensor());
    refuse_recording("distillation_loss_and_gradient");
    refuse_tangents("distillation_loss_and_gradient", {&logits, &values, &r, &w, &from});
    auto [loss, held] = distill_forward(logits, values, indices, rest, weight, temperature, reduction);
    const Tensor scale = grad_loss ? *grad_loss : at::ones(loss.sizes(), loss.options());
    return {loss, distill_backward(scale, logits, values, indices, weight, held, temperature, reduction)};
}

}  // namespace

PYBIND11_MODULE(_pxgtorch, m)
{
    m.def("use_library", &use_library);
    m.def("decay_attention", &decay_attention);
    m.def("decay_attention_backward", &decay_attention_backward);
    m.def("decay_step", &decay_step);
    m.def("top_logits", &top_logits);
    m.def("distillation_loss", &distillation_loss);
    m.def("distillation_loss_and_gradient", &distillation_loss_and_gradient);
}
