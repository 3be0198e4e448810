// PyTorch binding of the routing, sequence log-probability and preference
// entry points of the C ABI (torch.ops.dot_amd.*) for HIP tensors, and their
// autograd functions for HIP and CPU tensors (the CPU implementations are in
// cpu_training.cpp).  The Python functions check arguments; the operators
// check again what a kernel's indexing relies on.
//
// The autograd functions are C++: a training step over a small batch is bound
// by the host's work, and a node that runs without the interpreter takes less
// of it.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/dot_amd.h"

namespace {

using at::Tensor;
using c10::optional;

void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == DOT_OK, what, " failed (code ", rc, "): ", dot_last_error());
}

dot_stream_t stream_of(const Tensor& t) {
    return reinterpret_cast<dot_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// Scratch of a call, none where it needs none (an allocation takes the host
// over a microsecond).
Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}
void* ptr_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int dtype_tag(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return DOT_F32;
        case at::kHalf: return DOT_F16;
        case at::kBFloat16: return DOT_BF16;
        default: TORCH_CHECK(false, name, " must be float32, float16 or bfloat16");
    }
}

int to_int(int64_t v, const char* name) {
    TORCH_CHECK(v >= 0 && v <= INT32_MAX, name, " out of range");
    return int(v);
}

void check_on(const Tensor& t, const Tensor& with, const char* name) {
    TORCH_CHECK(t.device() == with.device(), name, " must be on ", with.device(), ", got ", t.device());
}

// Rows of unit stride, in place where they are so already.
Tensor unit_rows(const Tensor& t) { return t.stride(2) == 1 || t.size(2) <= 1 ? t : t.contiguous(); }

const float* floats(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
Tensor f32c(const optional<Tensor>& t, const Tensor& like, const char* name) {
    if (!t.has_value()) return Tensor();
    check_on(*t, like, name);
    return t->to(at::kFloat).contiguous();
}

// An upstream gradient and whether it is one value for all (an expanded
// scalar, as the gradient of a sum is).
Tensor upstream(const Tensor& g, const Tensor& like, int& scalar) {
    check_on(g, like, "grad");
    bool one = g.numel() > 1;
    for (int64_t d = 0; d < g.dim(); ++d) one = one && (g.stride(d) == 0 || g.size(d) == 1);
    scalar = one;
    if (one) return g.as_strided({1}, {1}).to(at::kFloat);
    return g.to(at::kFloat).contiguous();
}

Tensor mask_of(const optional<Tensor>& mask, const Tensor& x) {
    if (!mask.has_value()) return Tensor();
    check_on(*mask, x, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kBool && mask->dim() == 2 && mask->size(0) == x.size(0) &&
                    mask->size(1) == x.size(1),
                "mask must be bool of the leading two sizes");
    return mask->contiguous();
}
const uint8_t* mask_ptr(const Tensor& m) {
    return m.defined() ? reinterpret_cast<const uint8_t*>(m.const_data_ptr()) : nullptr;
}

Tensor ints_of(const Tensor& t, const Tensor& like, const char* name) {
    check_on(t, like, name);
    TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
    return t.contiguous();
}

void check_rows(const Tensor& x, const char* name) {
    TORCH_CHECK(x.device().is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(x.dim() == 3, name, " must be 3D");
}

// -> [counts, loss], then [weights, experts] where the call selects, then [tokens]
// where there is a mask (all N without one)
std::vector<Tensor> routing_forward_op(Tensor scores_, int64_t k, int64_t scoring, bool normalize,
                                       optional<Tensor> bias_, optional<Tensor> mask_, optional<Tensor> given_) {
    check_rows(scores_, "scores");
    c10::OptionalDeviceGuard guard(scores_.device());
    const Tensor scores = unit_rows(scores_);
    const int64_t B = scores.size(0), N = scores.size(1), E = scores.size(2);
    const Tensor mask = mask_of(mask_, scores);
    const Tensor bias = f32c(bias_, scores, "bias");
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == E), "bias must have shape [E]");
    Tensor given;
    if (given_.has_value()) {
        given = ints_of(*given_, scores, "experts");
        TORCH_CHECK(given.dim() == 3 && given.size(0) == B && given.size(1) == N && given.size(2) == k,
                    "experts must have shape [B, N, k]");
    }
    const auto f32 = scores.options().dtype(at::kFloat), i32 = scores.options().dtype(at::kInt);
    const bool select = !given.defined();
    std::vector<Tensor> out{at::empty({B, E}, i32), at::empty({B}, f32)};
    if (select) {
        out.push_back(at::empty({B, N, k}, f32));
        out.push_back(at::empty({B, N, k}, i32));
    }
    if (mask.defined()) out.push_back(at::empty({B}, i32));
    dot_routing_fwd_args a{};
    a.dtype = dtype_tag(scores, "scores");
    a.B = to_int(B, "B");
    a.N = to_int(N, "N");
    a.E = to_int(E, "E");
    a.k = to_int(k, "k");
    a.scores = scores.const_data_ptr();
    a.stride_b = scores.stride(0);
    a.stride_n = scores.stride(1);
    a.scoring = int(scoring);
    a.normalize = normalize;
    a.bias = floats(bias);
    a.mask = mask_ptr(mask);
    // an empty batch has no entries to point at: any address says "given"
    a.given = select ? nullptr : given.numel() ? given.const_data_ptr() : out[0].const_data_ptr();
    a.given_is_int64 = !select && given.scalar_type() == at::kLong;
    a.counts = out[0].data_ptr<int32_t>();
    a.loss = out[1].data_ptr<float>();
    a.weights = select ? out[2].data_ptr<float>() : nullptr;
    a.experts = select ? out[3].data_ptr<int32_t>() : nullptr;
    a.tokens = mask.defined() ? out.back().data_ptr<int32_t>() : nullptr;
    a.workspace_bytes = dot_routing_forward_workspace_bytes(a.B, a.N, a.E);
    const Tensor ws = workspace(a.workspace_bytes, scores);
    a.workspace = ptr_of(ws);
    check_rc(dot_routing_forward(&a, stream_of(scores)), "dot_routing_forward");
    return out;
}

Tensor routing_backward_op(Tensor scores_, int64_t k, int64_t scoring, bool normalize, optional<Tensor> mask_,
                           Tensor counts, optional<Tensor> tokens, optional<Tensor> grad_loss_,
                           optional<Tensor> weights, optional<Tensor> experts, optional<Tensor> grad_weights_) {
    check_rows(scores_, "scores");
    c10::OptionalDeviceGuard guard(scores_.device());
    const Tensor scores = unit_rows(scores_);
    const int64_t B = scores.size(0), N = scores.size(1), E = scores.size(2);
    const Tensor mask = mask_of(mask_, scores);
    check_on(counts, scores, "counts");
    TORCH_CHECK(counts.scalar_type() == at::kInt && counts.is_contiguous() && counts.numel() == B * E,
                "counts must be as the forward returned them");
    TORCH_CHECK(tokens.has_value() == mask.defined(), "tokens come with a mask");
    if (tokens.has_value()) {
        check_on(*tokens, scores, "tokens");
        TORCH_CHECK(tokens->scalar_type() == at::kInt && tokens->is_contiguous() && tokens->numel() == B,
                    "tokens must be as the forward returned them");
    }
    Tensor grad = at::empty({B, N, E}, scores.options().memory_format(at::MemoryFormat::Contiguous));
    dot_routing_bwd_args a{};
    Tensor gl, gw, w, e;
    if (grad_loss_.has_value()) {
        gl = upstream(*grad_loss_, scores, a.grad_loss_scalar);
        TORCH_CHECK(grad_loss_->numel() == B, "grad_loss must have shape [B]");
    }
    if (grad_weights_.has_value()) {
        TORCH_CHECK(weights.has_value() && experts.has_value(), "grad_weights needs weights and experts");
        gw = f32c(grad_weights_, scores, "grad_weights");
        w = f32c(weights, scores, "weights");
        e = ints_of(*experts, scores, "experts");
        TORCH_CHECK(gw.numel() == B * N * k && w.numel() == B * N * k && e.numel() == B * N * k &&
                        e.scalar_type() == at::kInt,
                    "weights, experts and grad_weights must have shape [B, N, k]");
    }
    a.scores = scores.const_data_ptr();
    a.dtype = dtype_tag(scores, "scores");
    a.stride_b = scores.stride(0);
    a.stride_n = scores.stride(1);
    a.B = to_int(B, "B");
    a.N = to_int(N, "N");
    a.E = to_int(E, "E");
    a.k = to_int(k, "k");
    a.scoring = int(scoring);
    a.normalize = normalize;
    a.mask = mask_ptr(mask);
    a.counts = counts.const_data_ptr<int32_t>();
    a.tokens = tokens.has_value() ? tokens->const_data_ptr<int32_t>() : nullptr;
    a.grad_loss = floats(gl);
    a.weights = floats(w);
    a.experts = e.defined() ? e.const_data_ptr<int32_t>() : nullptr;
    a.grad_weights = floats(gw);
    a.grad_scores = grad.data_ptr();
    check_rc(dot_routing_backward(&a, stream_of(scores)), "dot_routing_backward");
    return grad;
}

template <class A>
void fill_rows(A& a, const Tensor& logits, const Tensor& tokens, const Tensor& mask, double tau, int64_t reduction) {
    a.logits = logits.const_data_ptr();
    a.dtype = dtype_tag(logits, "logits");
    a.stride_b = logits.stride(0);
    a.stride_s = logits.stride(1);
    a.B = to_int(logits.size(0), "B");
    a.S = to_int(logits.size(1), "S");
    a.V = to_int(logits.size(2), "V");
    a.tokens = tokens.const_data_ptr();
    a.tokens_are_int64 = tokens.scalar_type() == at::kLong;
    a.mask = mask_ptr(mask);
    a.tau = tau;
    a.reduction = int(reduction);
}

Tensor tokens_of(const Tensor& tokens, const Tensor& logits) {
    Tensor t = ints_of(tokens, logits, "tokens");
    TORCH_CHECK(t.dim() == 2 && t.size(0) == logits.size(0) && t.size(1) == logits.size(1),
                "tokens must have shape [B, S]");
    return t;
}

// -> [out], with keep [out, saved]: the row statistics [B, S, 2] and the sequences'
// weights [B] that the backward takes, one after the other
std::vector<Tensor> sequence_logp_forward_op(Tensor logits_, Tensor tokens_, optional<Tensor> ref_,
                                             optional<Tensor> mask_, double tau, int64_t reduction, bool keep) {
    check_rows(logits_, "logits");
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = unit_rows(logits_);
    const int64_t B = logits.size(0), S = logits.size(1);
    const Tensor tokens = tokens_of(tokens_, logits), mask = mask_of(mask_, logits);
    Tensor ref;
    if (ref_.has_value()) {
        check_on(*ref_, logits, "ref_logp");
        ref = ref_->scalar_type() == at::kDouble ? ref_->contiguous() : ref_->to(at::kFloat).contiguous();
        TORCH_CHECK((ref.dim() == 1 && ref.size(0) == B) || (ref.dim() == 2 && ref.size(0) == B && ref.size(1) == S),
                    "ref_logp must have shape [B] or [B, S]");
    }
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor out = at::empty(reduction == DOT_REDUCE_NONE ? at::IntArrayRef({B, S}) : at::IntArrayRef({B}), f32);
    const Tensor saved = keep ? at::empty({(2 * S + 1) * B}, f32) : Tensor();
    dot_seqlogp_fwd_args a{};
    fill_rows(a, logits, tokens, mask, tau, reduction);
    a.ref = ref.defined() ? ref.const_data_ptr() : nullptr;
    a.ref_is_f64 = ref.defined() && ref.scalar_type() == at::kDouble;
    a.ref_per_token = ref.defined() && ref.dim() == 2;
    a.out = out.data_ptr<float>();
    a.row_stats = keep ? saved.data_ptr<float>() : nullptr;
    a.weight = keep ? saved.data_ptr<float>() + 2 * B * S : nullptr;
    a.workspace_bytes = dot_seqlogp_forward_workspace_bytes(a.B, a.S, a.V, a.dtype);
    const Tensor ws = workspace(a.workspace_bytes, logits);
    a.workspace = ptr_of(ws);
    check_rc(dot_seqlogp_forward(&a, stream_of(logits)), "dot_seqlogp_forward");
    if (!keep) return {out};
    return {out, saved};
}

Tensor sequence_logp_backward_op(Tensor logits_, Tensor tokens_, optional<Tensor> mask_, double tau,
                                 int64_t reduction, Tensor saved, Tensor grad_out_) {
    check_rows(logits_, "logits");
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = unit_rows(logits_);
    const int64_t B = logits.size(0), S = logits.size(1), V = logits.size(2);
    const Tensor tokens = tokens_of(tokens_, logits), mask = mask_of(mask_, logits);
    check_on(saved, logits, "saved");
    TORCH_CHECK(saved.scalar_type() == at::kFloat && saved.is_contiguous() && saved.numel() == (2 * S + 1) * B,
                "saved must be as the forward returned it");
    TORCH_CHECK(grad_out_.numel() == (reduction == DOT_REDUCE_NONE ? B * S : B), "grad_out has the wrong size");
    Tensor grad = at::empty({B, S, V}, logits.options().memory_format(at::MemoryFormat::Contiguous));
    dot_seqlogp_bwd_args a{};
    fill_rows(a, logits, tokens, mask, tau, reduction);
    const Tensor go = upstream(grad_out_, logits, a.grad_out_scalar);
    a.row_stats = saved.const_data_ptr<float>();
    a.weight = a.row_stats + 2 * B * S;
    a.grad_out = floats(go);
    a.grad_logits = grad.data_ptr();
    check_rc(dot_seqlogp_backward(&a, stream_of(logits)), "dot_seqlogp_backward");
    return grad;
}

// Sizes of the two sets from [P + Q] ratios and a [P, Q] plan (or pairs).
template <class A>
void fill_preference(A& a, const Tensor& ratio, const Tensor& plan, int64_t type, double beta, double smoothing) {
    TORCH_CHECK(ratio.dim() == 1, "log_ratio must be 1D");
    const int64_t n = ratio.size(0);
    const int64_t P = plan.defined() ? plan.size(0) : n / 2, Q = plan.defined() ? plan.size(1) : n / 2;
    TORCH_CHECK(P + Q == n, "log_ratio must hold the P + Q answers of a [P, Q] plan, or pairs");
    a.ratio = floats(ratio);
    a.plan = plan.defined() && plan.numel() ? floats(plan) : nullptr;
    a.P = to_int(P, "P");
    a.Q = to_int(Q, "Q");
    a.loss_type = int(type);
    a.beta = float(beta);
    // what is left is a whole number of at most 2^29 units
    if (std::isnormal(a.beta))
        a.beta_tail = int(std::ldexp(beta - double(a.beta), 53 - std::ilogb(a.beta)));
    a.smoothing = float(smoothing);
}

Tensor plan_of(const optional<Tensor>& plan, const Tensor& ratio) {
    TORCH_CHECK(!plan.has_value() || plan->dim() == 2, "plan must be 2D [P, Q]");
    return f32c(plan, ratio, "plan");
}

Tensor preference_forward_op(Tensor ratio_, optional<Tensor> plan_, int64_t type, double beta, double smoothing) {
    TORCH_CHECK(ratio_.device().is_cuda(), "log_ratio must be a CUDA tensor");
    c10::OptionalDeviceGuard guard(ratio_.device());
    const Tensor ratio = f32c(ratio_, ratio_, "log_ratio"), plan = plan_of(plan_, ratio_);
    dot_preference_fwd_args a{};
    fill_preference(a, ratio, plan, type, beta, smoothing);
    Tensor loss = at::empty({a.P}, ratio.options());
    a.loss = loss.data_ptr<float>();
    check_rc(dot_preference_forward(&a, stream_of(ratio)), "dot_preference_forward");
    return loss;
}

// -> [grad_ratio, grad_plan (empty without want_plan)]
std::vector<Tensor> preference_backward_op(Tensor ratio_, optional<Tensor> plan_, int64_t type, double beta,
                                           double smoothing, Tensor grad_loss_, bool want_plan) {
    TORCH_CHECK(ratio_.device().is_cuda(), "log_ratio must be a CUDA tensor");
    c10::OptionalDeviceGuard guard(ratio_.device());
    const Tensor ratio = f32c(ratio_, ratio_, "log_ratio"), plan = plan_of(plan_, ratio_);
    dot_preference_bwd_args a{};
    fill_preference(a, ratio, plan, type, beta, smoothing);
    TORCH_CHECK(grad_loss_.numel() == a.P, "grad_loss must have shape [P]");
    const Tensor gl = upstream(grad_loss_, ratio, a.grad_loss_scalar);
    Tensor grad_ratio = at::empty_like(ratio);
    Tensor grad_plan = want_plan && plan.defined() ? at::empty_like(plan) : at::empty({0}, ratio.options());
    a.grad_loss = floats(gl);
    a.grad_ratio = grad_ratio.data_ptr<float>();
    a.grad_plan = grad_plan.numel() ? grad_plan.data_ptr<float>() : nullptr;
    a.workspace_bytes = dot_preference_backward_workspace_bytes(a.P, a.Q, plan.defined());
    const Tensor ws = workspace(a.workspace_bytes, ratio);
    a.workspace = ptr_of(ws);
    check_rc(dot_preference_backward(&a, stream_of(ratio)), "dot_preference_backward");
    return {grad_ratio, grad_plan};
}

// ---------------------------------------------------------------------------
// Autograd
// ---------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Whether a call has to be recorded.
bool records(const Tensor& x) { return at::GradMode::is_enabled() && x.requires_grad(); }
bool records(const optional<Tensor>& x) { return x.has_value() && records(*x); }

// A tangent of forward-mode differentiation would be dropped below autograd, so
// that the derivative came out as zero: an error instead.
void check_no_tangent(const Tensor& x) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !x._fw_grad(0).defined(),
                                "dot_amd operators have no forward-mode derivative");
}

// The gradient of an operator that has no second derivative: a backward
// through it is an error, not a wrong result.  The error's node leads on to all
// that the gradient is a function of (the inputs and the upstream gradients):
// the engine runs only nodes on a way to what it is asked for.
Tensor once(const Tensor& grad, const variable_list& of) {
    if (!at::GradMode::is_enabled() || !grad.defined()) return grad;
    auto refuse = std::make_shared<torch::autograd::Error>(
        "dot_amd operators are differentiable once: no gradient flows through their backward",
        torch::autograd::collect_next_edges(of));
    Tensor out = grad.detach();
    torch::autograd::set_history(out, refuse);
    return out;
}

template <class F>
auto op_handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

std::vector<Tensor> call_routing(const Tensor& scores, int64_t k, int64_t scoring, bool normalize,
                                 const optional<Tensor>& bias, const optional<Tensor>& mask,
                                 const optional<Tensor>& given) {
    static const auto op = op_handle<decltype(routing_forward_op)>("dot_amd::routing_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(scores, k, scoring, normalize, bias, mask, given);
}

optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

struct RoutingFunction : torch::autograd::Function<RoutingFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& scores, int64_t k, int64_t scoring,
                                 bool normalize, const optional<Tensor>& bias, const optional<Tensor>& mask,
                                 const optional<Tensor>& given) {
        std::vector<Tensor> o = call_routing(scores, k, scoring, normalize, bias, mask, given);
        const bool select = !given.has_value(), masked = mask.has_value();
        ctx->save_for_backward({scores, mask.value_or(Tensor()), o[0], masked ? o.back() : Tensor(),
                                select ? o[2] : Tensor(), select ? o[3] : Tensor()});
        ctx->saved_data["args"] = k * 8 + scoring * 2 + normalize;
        variable_list counts{o[0]};
        if (select) counts.push_back(o[3]);
        if (masked) counts.push_back(o.back());
        ctx->mark_non_differentiable(counts);
        ctx->set_materialize_grads(false);
        return o;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        const bool select = s[4].defined();
        const Tensor gw = select ? grads[2] : Tensor(), gl = grads[1];
        const int64_t args = ctx->saved_data["args"].toInt();
        Tensor g;
        if (gw.defined() || gl.defined()) {
            static const auto op = op_handle<decltype(routing_backward_op)>("dot_amd::routing_backward");
            at::AutoDispatchBelowADInplaceOrView below;
            g = op.call(s[0], args / 8, args / 2 % 4, args % 2, maybe(s[1]), s[2], maybe(s[3]), maybe(gl),
                        gw.defined() ? maybe(s[4]) : c10::nullopt, gw.defined() ? maybe(s[5]) : c10::nullopt,
                        maybe(gw));
        }
        return {once(g, {s[0], gl, gw}), {}, {}, {}, {}, {}, {}};
    }
};

std::vector<Tensor> routing_forward_autograd(Tensor scores, int64_t k, int64_t scoring, bool normalize,
                                             optional<Tensor> bias, optional<Tensor> mask, optional<Tensor> given) {
    check_no_tangent(scores);
    if (!records(scores)) return call_routing(scores, k, scoring, normalize, bias, mask, given);
    return RoutingFunction::apply(scores, k, scoring, normalize, bias, mask, given);
}

std::vector<Tensor> call_sequence_logp(const Tensor& logits, const Tensor& tokens, const optional<Tensor>& ref,
                                       const optional<Tensor>& mask, double tau, int64_t reduction, bool keep) {
    static const auto op = op_handle<decltype(sequence_logp_forward_op)>("dot_amd::sequence_logp_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, tokens, ref, mask, tau, reduction, keep);
}

struct SequenceLogpFunction : torch::autograd::Function<SequenceLogpFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                                 const optional<Tensor>& ref, const optional<Tensor>& mask, double tau,
                                 int64_t reduction) {
        std::vector<Tensor> o = call_sequence_logp(logits, tokens, ref, mask, tau, reduction, true);
        ctx->save_for_backward({logits, tokens, mask.value_or(Tensor()), o[1]});
        ctx->saved_data["tau"] = tau;
        ctx->saved_data["reduction"] = reduction;
        ctx->mark_non_differentiable({o[1]});
        ctx->set_materialize_grads(false);
        return o;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        Tensor g;
        if (grads[0].defined()) {
            static const auto op = op_handle<decltype(sequence_logp_backward_op)>("dot_amd::sequence_logp_backward");
            at::AutoDispatchBelowADInplaceOrView below;
            g = op.call(s[0], s[1], maybe(s[2]), ctx->saved_data["tau"].toDouble(),
                        ctx->saved_data["reduction"].toInt(), s[3], grads[0]);
        }
        return {once(g, {s[0], grads[0]}), {}, {}, {}, {}, {}};
    }
};

std::vector<Tensor> sequence_logp_forward_autograd(Tensor logits, Tensor tokens, optional<Tensor> ref,
                                                   optional<Tensor> mask, double tau, int64_t reduction, bool keep) {
    check_no_tangent(logits);
    if (!records(logits)) return call_sequence_logp(logits, tokens, ref, mask, tau, reduction, keep);
    return SequenceLogpFunction::apply(logits, tokens, ref, mask, tau, reduction);
}

Tensor call_preference(const Tensor& ratio, const optional<Tensor>& plan, int64_t type, double beta,
                       double smoothing) {
    static const auto op = op_handle<decltype(preference_forward_op)>("dot_amd::preference_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(ratio, plan, type, beta, smoothing);
}

struct PreferenceFunction : torch::autograd::Function<PreferenceFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ratio, const optional<Tensor>& plan, int64_t type,
                          double beta, double smoothing) {
        ctx->save_for_backward({ratio, plan.value_or(Tensor())});
        ctx->saved_data["type"] = type;
        ctx->saved_data["beta"] = beta;
        ctx->saved_data["smoothing"] = smoothing;
        ctx->set_materialize_grads(false);
        return call_preference(ratio, plan, type, beta, smoothing);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        Tensor gr, gp;
        if (grads[0].defined()) {
            const bool want_plan = s[1].defined() && ctx->needs_input_grad(1);
            static const auto op = op_handle<decltype(preference_backward_op)>("dot_amd::preference_backward");
            at::AutoDispatchBelowADInplaceOrView below;
            const std::vector<Tensor> g =
                op.call(s[0], maybe(s[1]), ctx->saved_data["type"].toInt(), ctx->saved_data["beta"].toDouble(),
                        ctx->saved_data["smoothing"].toDouble(), grads[0], want_plan);
            gr = g[0].to(s[0].scalar_type());
            if (want_plan) gp = g[1].to(s[1].scalar_type());
        }
        const variable_list of{s[0], s[1], grads[0]};
        return {once(gr, of), once(gp, of), {}, {}, {}};
    }
};

Tensor preference_forward_autograd(Tensor ratio, optional<Tensor> plan, int64_t type, double beta, double smoothing) {
    check_no_tangent(ratio);
    if (plan.has_value()) check_no_tangent(*plan);
    if (!records(ratio) && !records(plan)) return call_preference(ratio, plan, type, beta, smoothing);
    return PreferenceFunction::apply(ratio, plan, type, beta, smoothing);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(dot_amd, m) {
    m.def("routing_forward(Tensor scores, int k, int scoring, bool normalize, Tensor? bias, Tensor? mask, Tensor? given) -> Tensor[]");
    m.def("routing_backward(Tensor scores, int k, int scoring, bool normalize, Tensor? mask, Tensor counts, Tensor? tokens, Tensor? grad_loss, Tensor? weights, Tensor? experts, Tensor? grad_weights) -> Tensor");
    m.def("sequence_logp_forward(Tensor logits, Tensor tokens, Tensor? ref, Tensor? mask, float tau, int reduction, bool keep) -> Tensor[]");
    m.def("sequence_logp_backward(Tensor logits, Tensor tokens, Tensor? mask, float tau, int reduction, Tensor saved, Tensor grad_out) -> Tensor");
    m.def("preference_forward(Tensor log_ratio, Tensor? plan, int loss_type, float beta, float smoothing) -> Tensor");
    m.def("preference_backward(Tensor log_ratio, Tensor? plan, int loss_type, float beta, float smoothing, Tensor grad_loss, bool want_plan) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(dot_amd, CUDA, m) {
    m.impl("routing_forward", routing_forward_op);
    m.impl("routing_backward", routing_backward_op);
    m.impl("sequence_logp_forward", sequence_logp_forward_op);
    m.impl("sequence_logp_backward", sequence_logp_backward_op);
    m.impl("preference_forward", preference_forward_op);
    m.impl("preference_backward", preference_backward_op);
}

TORCH_LIBRARY_IMPL(dot_amd, Autograd, m) {
    m.impl("routing_forward", routing_forward_autograd);
    m.impl("sequence_logp_forward", sequence_logp_forward_autograd);
    m.impl("preference_forward", preference_forward_autograd);
}
