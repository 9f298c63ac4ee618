// The tensor operators as torch sees them: outputs allocated, layouts lined up, gradients recorded as native autograd nodes, so
// that a call costs little more than its launch.  Host code only: the C entries' addresses (include/muzero_amd.h) and the raw
// stream come from Python, which has checked types, shapes and devices; a backward pass runs on its forward pass's stream.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <initializer_list>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/muzero_amd.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

static struct Entries {
    decltype(&mz_linear_recurrence) recurrence, recurrence_backward;
    decltype(&mz_linear_recurrence_workspace) recurrence_workspace;
    decltype(&mz_distill_loss) distill_loss, distill_grad, distill_loss_grad;
    decltype(&mz_verify_drafts) verify;
    decltype(&mz_last_error) last_error;
} entry;

static void bind(const std::vector<int64_t> &at)
{
    TORCH_CHECK(at.size() * sizeof(void *) == sizeof(entry), "bind: one address for every entry");
    std::copy(at.begin(), at.end(), reinterpret_cast<int64_t *>(&entry));
}

static void check(int rc)
{
    TORCH_CHECK_VALUE(rc != MZ_ERR_ARG, entry.last_error());
    TORCH_CHECK(rc == MZ_OK, entry.last_error());
}

static int type_of(const Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return MZ_F32;
    case at::kBFloat16: return MZ_BF16;
    case at::kHalf: return MZ_F16;
    default: return MZ_F64;
    }
}

static void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// What the kernels compute is no torch operation, so a tangent would be dropped and a trace would hold outputs that nothing
// fills: both are errors.
static void refuse(const char *fn, std::initializer_list<Tensor> inputs)
{
    for (const Tensor &t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), fn, ": no forward-mode derivatives");
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), fn,
                                " cannot be traced");
}
static Tensor given(const std::optional<Tensor> &t) { return t.value_or(Tensor()); }

// A gradient taken with create_graph: the operators are differentiable once, and a second time is an error, not a zero.
static variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    for (auto &g : grads) if (g.defined()) g = g.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once", (int)grads.size());
    return (*error)(std::move(grads));
}

// ------------------------------------------------------------------------------------------------ recurrence

// `t` itself where the kernels read its layout well: channels contiguous, or (one channel, or time contiguous) any.
static Tensor lined_up(const Tensor &t, bool channels) { return channels && t.stride(2) != 1 ? t.contiguous() : t; }

static Tensor like(const Tensor &x, bool channels)
{
    Tensor y = at::empty_like(x);
    return channels && y.stride(2) != 1 ? at::empty(x.sizes(), x.options()) : y;
}

static bool by_channels(const Tensor &x) { return x.size(2) > 1 && (x.stride(2) == 1 || x.stride(1) != 1); }

static at::TensorOptions wide(const Tensor &x) { return x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat); }

// fine: [B, positions / 4, D, 4] bytes, undefined where nothing is kept
static void run_recurrence(bool backward, Tensor gate, Tensor x, const Tensor &state, bool reverse, Tensor out, Tensor y, Tensor out_gate,
                           const Tensor &last, const Tensor &grad_last, const Tensor &out_state, Tensor fine, int64_t stream)
{
    mz_recurrence a{};
    int64_t B = x.size(0), T = x.size(1), D = x.size(2);
    Tensor *views[] = {&gate, &x, &out, &y, &out_gate};
    if (D == 1 && B > 1 && x.stride(0) == 1 && (T == 1 || x.stride(1) != 1)) {
        // one channel, time-major (or a single position): the sequences are the channels of one
        bool all = true;
        for (Tensor *v : views) all &= !v->defined() || v->stride(0) == 1;
        if (all) {
            for (Tensor *v : views) if (v->defined()) *v = v->transpose(0, 2);
            if (fine.defined()) fine = fine.transpose(0, 2);
            D = B, B = 1;
        }
    }
    mz_strided *to[] = {&a.gate, &a.x, &a.out, &a.y, &a.out_gate};
    for (int i = 0; i < 5; i++)
        if (views[i]->defined()) *to[i] = {views[i]->data_ptr(), views[i]->stride(0), views[i]->stride(1), views[i]->stride(2)};
    TORCH_CHECK_VALUE(B <= INT32_MAX && D <= INT32_MAX, "linear_recurrence: sizes must be positive, and B * D at most 2^30");
    a.type = type_of(x), a.B = (int32_t)B, a.D = (int32_t)D, a.T = T, a.reverse = reverse;
    a.state = ptr(state), a.last = ptr(last), a.grad_last = ptr(grad_last), a.out_state = ptr(out_state);
    if (fine.defined()) a.fine = {fine.data_ptr(), fine.stride(0), fine.stride(1), fine.stride(2)};
    Tensor space;
    if (T > 256) {   // shorter records need none
        check(entry.recurrence_workspace(&a, backward, &a.workspace_bytes));
        if (a.workspace_bytes) {
            space = at::empty({a.workspace_bytes}, x.options().dtype(at::kByte));
            a.workspace = space.data_ptr();
        }
    }
    c10::DeviceGuard guard(x.device());
    check((backward ? entry.recurrence_backward : entry.recurrence)(&a, reinterpret_cast<void *>(stream)));
}

// y, the last state, and with keep what the rounding of a 16-bit y lost
static std::tuple<Tensor, Tensor, Tensor> recurrence_forward(const Tensor &gate, const Tensor &x, const Tensor &state, bool reverse, bool keep, int64_t stream)
{
    if (x.numel() == 0) return {at::empty_like(x), state.defined() ? state.clone() : at::zeros({x.size(0), x.size(2)}, wide(x)), {}};
    const bool channels = by_channels(x);
    const Tensor xl = lined_up(x, channels);
    Tensor y = like(xl, channels), last = at::empty({x.size(0), x.size(2)}, wide(x));
    Tensor fine;
    if (keep && x.element_size() == 2) {   // as close together as y's elements
        const int64_t B = x.size(0), words = (x.size(1) + 3) / 4, D = x.size(2);
        const auto bytes = x.options().dtype(at::kChar);
        fine = channels ? at::empty({B, words, D, 4}, bytes)
             : D == 1 && y.stride(0) == 1 ? at::empty({words, B, D, 4}, bytes).transpose(0, 1) : at::empty({B, D, words, 4}, bytes).transpose(1, 2);
    }
    run_recurrence(false, lined_up(gate, channels), xl, state, reverse, y, {}, {}, last, {}, {}, fine, stream);
    return {y, last, fine};
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext *ctx, const Tensor &gate, const Tensor &x, const std::optional<Tensor> &first, bool reverse,
                                 int64_t stream)
    {
        const Tensor state = given(first);
        auto [y, last, fine] = recurrence_forward(gate, x, state, reverse, gate.requires_grad(), stream);
        ctx->set_materialize_grads(false);
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["stream"] = stream;
        ctx->save_for_backward({gate, gate.requires_grad() ? y : Tensor(), state, fine});
        return {y, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        Tensor dy = grads[0], dlast = grads[1];
        if (!dy.defined() && !dlast.defined()) return {{}, {}, {}, {}, {}};
        const auto saved = ctx->get_saved_variables();
        Tensor gate = saved[0].detach(), y = saved[1], state = saved[2], fine = saved[3];
        const bool want_gate = ctx->needs_input_grad(0), want_x = ctx->needs_input_grad(1), want_state = state.defined() && ctx->needs_input_grad(2);
        variable_list out(5);
        {
            at::AutoGradMode off(false);
            if (!dy.defined()) dy = at::zeros_like(gate);
            if (dlast.defined()) dlast = dlast.contiguous();
            Tensor dstate = want_state ? at::empty({dy.size(0), dy.size(2)}, wide(dy)) : Tensor();
            if (dy.numel() == 0) {
                if (want_gate) out[0] = at::empty_like(dy);
                if (want_x) out[1] = at::empty_like(dy);
                if (want_state) out[2] = dlast.defined() ? dlast.clone() : dstate.zero_();
            } else {
                const bool channels = by_channels(dy);
                dy = lined_up(dy, channels);
                Tensor dx = like(dy, channels), dgate = want_gate ? like(dy, channels) : Tensor();
                run_recurrence(true, lined_up(gate, channels), dy, state, ctx->saved_data["reverse"].toBool(), dx,
                               want_gate ? lined_up(y, channels) : Tensor(), dgate, {}, dlast, dstate, fine, ctx->saved_data["stream"].toInt());
                out[0] = dgate, out[1] = want_x ? dx : Tensor(), out[2] = dstate;
            }
        }
        return once(std::move(out));
    }
};

static std::tuple<Tensor, Tensor> linear_recurrence(const Tensor &gate, const Tensor &x, const std::optional<Tensor> &state, bool reverse, int64_t stream)
{
    refuse("linear_recurrence", {gate, x, given(state)});
    const Tensor s = state ? state->contiguous() : Tensor();
    if (at::GradMode::is_enabled() && (gate.requires_grad() || x.requires_grad() || (s.defined() && s.requires_grad()))) {
        auto out = Recurrence::apply(gate, x, s.defined() ? std::optional<Tensor>(s) : std::nullopt, reverse, stream);
        return {out[0], out[1]};
    }
    auto [y, last, fine] = recurrence_forward(gate, x, s, reverse, false, stream);
    return {y, last};
}

// ------------------------------------------------------------------------------------------------ distillation

// logits, index, teacher, lse, weight as a call points to them
static mz_distill distill_args(variable_list &t, double temperature)
{
    if (t[0].stride(1) != 1) t[0] = t[0].contiguous();
    for (int i = 1; i < 5; i++) if (t[i].defined()) t[i] = t[i].contiguous();
    mz_distill a{};
    TORCH_CHECK_VALUE(t[0].size(0) <= INT32_MAX && t[0].size(1) <= INT32_MAX && t[1].size(1) <= INT32_MAX, "distillation: sizes outside the limits");
    a.type = type_of(t[0]), a.teacher_type = type_of(t[2]), a.index64 = t[1].scalar_type() == at::kLong;
    a.R = (int32_t)t[0].size(0), a.V = (int32_t)t[0].size(1), a.K = (int32_t)t[1].size(1), a.temperature = (float)temperature;
    a.logits = t[0].data_ptr(), a.logits_stride = t[0].stride(0), a.index = t[1].data_ptr(), a.teacher = t[2].data_ptr();
    a.lse = (const float *)ptr(t[3]), a.weight = (const float *)ptr(t[4]);
    return a;
}

struct Distillation : torch::autograd::Function<Distillation> {
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &index, const Tensor &teacher,
                          const std::optional<Tensor> &lse, const std::optional<Tensor> &weight, double temperature, int64_t stream)
    {
        variable_list t{logits.detach(), index, teacher.detach(), given(lse), given(weight)};
        mz_distill a = distill_args(t, temperature);
        const auto f32 = logits.options().dtype(at::kFloat);
        Tensor loss = at::empty({logits.size(0)}, f32), stats = at::empty({logits.size(0), 4}, f32);
        a.loss = loss.data_ptr<float>(), a.stats = stats.data_ptr<float>();
        c10::DeviceGuard guard(logits.device());
        if (a.R) check(entry.distill_loss(&a, reinterpret_cast<void *>(stream)));
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["stream"] = stream;
        ctx->save_for_backward({t[0], t[1], t[2], t[3], t[4], stats});
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        auto t = ctx->get_saved_variables();
        Tensor grad;
        {
            at::AutoGradMode off(false);
            const Tensor stats = t[5], up = grads[0].contiguous();
            for (auto &v : t) if (v.defined()) v = v.detach();
            mz_distill a = distill_args(t, ctx->saved_data["temperature"].toDouble());
            grad = at::empty(t[0].sizes(), t[0].options());
            a.grad_loss = up.data_ptr<float>(), a.grad = grad.data_ptr(), a.stats = stats.data_ptr<float>();
            c10::DeviceGuard guard(grad.device());
            if (a.R) check(entry.distill_grad(&a, reinterpret_cast<void *>(ctx->saved_data["stream"].toInt())));
        }
        return once({grad, {}, {}, {}, {}, {}, {}});
    }
};

static Tensor distillation_loss(const Tensor &logits, const Tensor &index, const Tensor &teacher, const std::optional<Tensor> &lse,
                                const std::optional<Tensor> &weight, double temperature, int64_t stream)
{
    refuse("distillation_loss", {logits, index, teacher, given(lse), given(weight)});
    auto plain = [](const std::optional<Tensor> &t) { return t ? std::optional<Tensor>(t->detach()) : std::nullopt; };
    return Distillation::apply(logits, index, teacher.detach(), plain(lse), plain(weight), temperature, stream);
}

static std::tuple<Tensor, Tensor> distillation_loss_grad(const Tensor &logits, const Tensor &index, const Tensor &teacher,
                                                         const std::optional<Tensor> &lse, const std::optional<Tensor> &weight,
                                                         double temperature, int64_t stream)
{
    refuse("distillation_loss_grad", {logits, index, teacher, given(lse), given(weight)});
    at::AutoGradMode off(false);
    variable_list t{logits, index, teacher, given(lse), given(weight)};
    mz_distill a = distill_args(t, temperature);
    Tensor loss = at::empty({logits.size(0)}, logits.options().dtype(at::kFloat)), grad = at::empty(logits.sizes(), logits.options());
    a.loss = loss.data_ptr<float>(), a.grad = grad.data_ptr();
    c10::DeviceGuard guard(logits.device());
    if (a.R) check(entry.distill_loss_grad(&a, reinterpret_cast<void *>(stream)));
    return {loss, grad};
}

// ------------------------------------------------------------------------------------------------ verification

static std::tuple<Tensor, Tensor> verify_drafts(Tensor tokens, std::optional<Tensor> draft, Tensor target, Tensor u_accept, Tensor u_sample,
                                                std::optional<Tensor> lengths, int64_t stream)
{
    refuse("verify_drafts", {tokens, given(draft), target, u_accept, u_sample, given(lengths)});
    at::AutoGradMode off(false);
    const int64_t B = tokens.size(0), K = tokens.size(1), V = target.size(2);
    Tensor accepted = at::empty({B}, target.options().dtype(at::kInt)), out = at::empty({B, K + 1}, tokens.options());
    if (B == 0) return {accepted, out};
    TORCH_CHECK_VALUE(B <= INT32_MAX && K < INT32_MAX && V <= INT32_MAX, "verify_drafts: sizes outside the limits");
    if (target.stride(2) != 1 && V > 1) target = target.contiguous();
    if (draft && draft->stride(2) != 1 && V > 1) draft = draft->contiguous();
    tokens = tokens.contiguous(), u_accept = u_accept.contiguous(), u_sample = u_sample.contiguous();
    if (lengths) lengths = lengths->contiguous();
    mz_verify a{};
    a.type = type_of(target), a.token64 = tokens.scalar_type() == at::kLong, a.B = (int32_t)B, a.K = (int32_t)K, a.V = (int32_t)V;
    a.tokens = tokens.data_ptr(), a.target = target.data_ptr(), a.target_stride_b = target.stride(0), a.target_stride_k = target.stride(1);
    if (draft) a.draft = draft->data_ptr(), a.draft_stride_b = draft->stride(0), a.draft_stride_k = draft->stride(1);
    a.u_accept = u_accept.data_ptr<double>(), a.u_sample = u_sample.data_ptr<double>();
    if (lengths) a.lengths = lengths->data_ptr<int32_t>();
    a.accepted = accepted.data_ptr<int32_t>(), a.out = out.data_ptr();
    c10::DeviceGuard guard(target.device());
    check(entry.verify(&a, reinterpret_cast<void *>(stream)));
    return {accepted, out};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.attr("built_for") = BUILT_FOR_TORCH;
    m.def("bind", &bind);
    m.def("linear_recurrence", &linear_recurrence);
    m.def("distillation_loss", &distillation_loss);
    m.def("distillation_loss_grad", &distillation_loss_grad);
    m.def("verify_drafts", &verify_drafts);
}
