// PyTorch binding of the top log-probability, distillation and beam search entry
// points of the C ABI (torch.ops.dot_amd.*) for HIP tensors, and the autograd
// function of the distillation loss for HIP and CPU tensors (the CPU
// implementations are in cpu_generation.cpp).  The Python functions check
// arguments; the operators check again what a kernel's indexing relies on.
#include "beam_states.hpp"
#include "torch_common.hpp"

namespace {

template <class A>
void fill_logits(A& a, const Tensor& logits, double tau) {
    a.logits = logits.const_data_ptr();
    a.dtype = dtype_tag(logits, "logits");
    a.stride_b = logits.stride(0);
    a.B = to_int(logits.size(0), "B");
    a.V = to_int(logits.size(2), "V");
    a.tau = tau;
}

// -> [logp, tokens]
std::vector<Tensor> top_logp_op(Tensor logits_, int64_t k, double tau, optional<Tensor> mask_) {
    check_rows(logits_, "logits");
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = unit_rows(logits_);
    const int64_t B = logits.size(0), S = logits.size(1);
    const Tensor mask = mask_of(mask_, logits);
    dot_top_logp_args a{};
    fill_logits(a, logits, tau);
    a.stride_s = logits.stride(1);
    a.S = to_int(S, "S");
    a.k = to_int(k, "k");
    a.mask = mask_ptr(mask);
    std::vector<Tensor> out{at::empty({B, S, k}, logits.options().dtype(at::kFloat)),
                            at::empty({B, S, k}, logits.options().dtype(at::kInt))};
    a.logp = out[0].data_ptr<float>();
    a.tokens = out[1].data_ptr<int32_t>();
    a.workspace_bytes = dot_top_logp_workspace_bytes(a.B, a.S, a.V, a.dtype, a.k);
    const Tensor ws = workspace(a.workspace_bytes, logits);
    a.workspace = ptr_of(ws);
    check_rc(dot_top_logp(&a, stream_of(logits)), "dot_top_logp");
    return out;
}

// Where the backward finds what the forward kept, in floats: row statistics [B, S, 2], the
// named tokens' gradients [B, S, K], these tokens (int32) and the sequences' weights [B].
struct Kept {
    int64_t own, tokens, weight, size;
    Kept(int64_t B, int64_t S, int64_t K)
        : own(2 * B * S), tokens(own + B * S * K), weight(tokens + B * S * K), size(weight + B) {}
};

// -> [out], with keep [out, saved]
std::vector<Tensor> distill_forward_op(Tensor logits_, Tensor logp_, Tensor tokens_, optional<Tensor> mask_,
                                       double tau, int64_t direction, int64_t rest, int64_t reduction, bool keep) {
    check_rows(logits_, "logits");
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = unit_rows(logits_);
    const int64_t B = logits.size(0), S = logits.size(1);
    const Tensor tokens = ints_of(tokens_, logits, "teacher_tokens"), mask = mask_of(mask_, logits);
    TORCH_CHECK(tokens.dim() == 3 && tokens.size(0) == B && tokens.size(1) == S,
                "teacher_tokens must have shape [B, S, K]");
    const int64_t K = tokens.size(2);
    const Tensor logp = f32c(logp_, logits, "teacher_logp");
    TORCH_CHECK(logp.sizes() == tokens.sizes(), "teacher_logp must be shaped as teacher_tokens");
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor out = at::empty(reduction == DOT_REDUCE_NONE ? at::IntArrayRef({B, S}) : at::IntArrayRef({B}), f32);
    const Kept kept(B, S, K);
    const Tensor saved = keep ? at::empty({kept.size}, f32) : Tensor();
    dot_distill_fwd_args a{};
    fill_logits(a, logits, tau);
    a.stride_s = logits.stride(1);
    a.S = to_int(S, "S");
    a.K = to_int(K, "K");
    a.tokens = tokens.const_data_ptr();
    a.tokens_are_int64 = tokens.scalar_type() == at::kLong;
    a.logp = floats(logp);
    a.mask = mask_ptr(mask);
    a.direction = int(direction);
    a.rest = int(rest);
    a.reduction = int(reduction);
    a.out = out.data_ptr<float>();
    if (keep) {
        float* p = saved.data_ptr<float>();
        a.row_stats = p;
        a.own_grad = p + kept.own;
        a.own_tokens = reinterpret_cast<int32_t*>(p + kept.tokens);
        a.weight = p + kept.weight;
    }
    a.workspace_bytes = dot_distill_forward_workspace_bytes(a.B, a.S, a.V, a.dtype, a.reduction);
    const Tensor ws = workspace(a.workspace_bytes, logits);
    a.workspace = ptr_of(ws);
    check_rc(dot_distill_forward(&a, stream_of(logits)), "dot_distill_forward");
    if (!keep) return {out};
    return {out, saved};
}

Tensor distill_backward_op(Tensor logits_, int64_t K, double tau, int64_t reduction, Tensor saved, Tensor grad_out_) {
    check_rows(logits_, "logits");
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = unit_rows(logits_);
    const int64_t B = logits.size(0), S = logits.size(1), V = logits.size(2);
    const Kept kept(B, S, K);
    check_on(saved, logits, "saved");
    TORCH_CHECK(K >= 1 && saved.scalar_type() == at::kFloat && saved.is_contiguous() && saved.numel() == kept.size,
                "saved must be as the forward returned it");
    TORCH_CHECK(grad_out_.numel() == (reduction == DOT_REDUCE_NONE ? B * S : B), "grad_out has the wrong size");
    Tensor grad = at::empty({B, S, V}, logits.options().memory_format(at::MemoryFormat::Contiguous));
    dot_distill_bwd_args a{};
    fill_logits(a, logits, tau);
    a.stride_s = logits.stride(1);
    a.S = to_int(S, "S");
    a.K = to_int(K, "K");
    a.reduction = int(reduction);
    const Tensor go = upstream(grad_out_, logits, a.grad_out_scalar);
    a.row_stats = saved.const_data_ptr<float>();
    a.own_grad = a.row_stats + kept.own;
    a.own_tokens = reinterpret_cast<const int32_t*>(a.row_stats + kept.tokens);
    a.weight = a.row_stats + kept.weight;
    a.grad_out = floats(go);
    a.grad_logits = grad.data_ptr();
    check_rc(dot_distill_backward(&a, stream_of(logits)), "dot_distill_backward");
    return grad;
}

// -> [scores, beams, tokens], with eos >= 0 [..., finished]
std::vector<Tensor> beam_step_op(Tensor logits_, Tensor scores_, int64_t n, double tau, optional<Tensor> finished_,
                                 int64_t eos) {
    check_rows(logits_, "logits");
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = unit_rows(logits_);
    const int64_t B = logits.size(0), W = logits.size(1);
    const Tensor scores = f32c(scores_, logits, "scores");
    TORCH_CHECK(scores.dim() == 2 && scores.size(0) == B && scores.size(1) == W, "scores must have shape [B, W]");
    Tensor finished;
    if (finished_.has_value()) {
        check_on(*finished_, logits, "finished");
        TORCH_CHECK(finished_->scalar_type() == at::kBool && finished_->sizes() == scores.sizes(),
                    "finished must be bool of shape [B, W]");
        finished = finished_->contiguous();
    }
    dot_beam_step_args a{};
    fill_logits(a, logits, tau);
    a.stride_w = logits.stride(1);
    a.W = to_int(W, "W");
    a.n = to_int(n, "n");
    a.scores = floats(scores);
    a.finished = mask_ptr(finished);
    TORCH_CHECK(eos < INT32_MAX, "eos out of range");
    a.eos = eos < 0 ? -1 : int(eos);
    const auto i32 = logits.options().dtype(at::kInt);
    std::vector<Tensor> out{at::empty({B, n}, scores.options()), at::empty({B, n}, i32), at::empty({B, n}, i32)};
    if (eos >= 0) out.push_back(at::empty({B, n}, logits.options().dtype(at::kBool)));
    a.out_scores = out[0].data_ptr<float>();
    a.out_beams = out[1].data_ptr<int32_t>();
    a.out_tokens = out[2].data_ptr<int32_t>();
    a.out_finished = eos >= 0 ? reinterpret_cast<uint8_t*>(out[3].data_ptr<bool>()) : nullptr;
    a.workspace_bytes = dot_beam_step_workspace_bytes(a.B, a.W, a.V, a.dtype, a.n);
    const Tensor ws = workspace(a.workspace_bytes, logits);
    a.workspace = ptr_of(ws);
    check_rc(dot_beam_step(&a, stream_of(logits)), "dot_beam_step");
    return out;
}

void beam_reorder_op(at::TensorList states, const Tensor& beams_, const optional<Tensor>& lengths_,
                     optional<int64_t> dim) {
    TORCH_CHECK_VALUE(beams_.device().is_cuda(), "states must be on ", beams_.device(), ", as beams are");
    c10::OptionalDeviceGuard guard(beams_.device());
    const std::vector<dot_beam_state> s = beam_states(states, beams_, lengths_, dim);
    const Tensor beams = beams_.contiguous(), lengths = lengths_.has_value() ? lengths_->contiguous() : Tensor();
    dot_beam_reorder_args a{};
    a.states = s.data();
    a.count = int(s.size());
    a.B = to_int(beams.size(0), "B");
    a.W = to_int(beams.size(1), "W");
    a.beams = beams.const_data_ptr();
    a.beams_are_int64 = beams.scalar_type() == at::kLong;
    a.lengths = lengths.defined() ? lengths.const_data_ptr() : nullptr;
    a.lengths_are_int64 = lengths.defined() && lengths.scalar_type() == at::kLong;
    const int rc = dot_beam_reorder(&a, stream_of(beams));
    TORCH_CHECK_VALUE(rc != DOT_ERR_INVALID_ARG, dot_last_error());
    check_rc(rc, "dot_beam_reorder");
    states_changed(states);
}

// ---------------------------------------------------------------------------
// Autograd
// ---------------------------------------------------------------------------
std::vector<Tensor> call_distill(const Tensor& logits, const Tensor& logp, const Tensor& tokens,
                                 const optional<Tensor>& mask, double tau, int64_t direction, int64_t rest,
                                 int64_t reduction, bool keep) {
    static const auto op = op_handle<decltype(distill_forward_op)>("dot_amd::distill_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, logp, tokens, mask, tau, direction, rest, reduction, keep);
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& logp, const Tensor& tokens,
                                 const optional<Tensor>& mask, double tau, int64_t direction, int64_t rest,
                                 int64_t reduction) {
        std::vector<Tensor> o = call_distill(logits, logp, tokens, mask, tau, direction, rest, reduction, true);
        ctx->save_for_backward({logits, o[1]});
        ctx->saved_data["tau"] = tau;
        ctx->saved_data["args"] = tokens.size(2) * 4 + reduction;
        ctx->mark_non_differentiable({o[1]});
        ctx->set_materialize_grads(false);
        return o;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        Tensor g;
        if (grads[0].defined()) {
            static const auto op = op_handle<decltype(distill_backward_op)>("dot_amd::distill_backward");
            at::AutoDispatchBelowADInplaceOrView below;
            const int64_t args = ctx->saved_data["args"].toInt();
            g = op.call(s[0], args / 4, ctx->saved_data["tau"].toDouble(), args % 4, s[1], grads[0]);
        }
        return {once(g, {s[0], grads[0]}), {}, {}, {}, {}, {}, {}, {}};
    }
};

std::vector<Tensor> distill_forward_autograd(Tensor logits, Tensor logp, Tensor tokens, optional<Tensor> mask,
                                             double tau, int64_t direction, int64_t rest, int64_t reduction,
                                             bool keep) {
    check_no_tangent(logits);
    if (!records(logits)) return call_distill(logits, logp, tokens, mask, tau, direction, rest, reduction, keep);
    return DistillFunction::apply(logits, logp, tokens, mask, tau, direction, rest, reduction);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(dot_amd, m) {
    m.def("top_logp(Tensor logits, int k, float tau, Tensor? mask) -> Tensor[]");
    m.def("distill_forward(Tensor logits, Tensor logp, Tensor tokens, Tensor? mask, float tau, int direction, int rest, int reduction, bool keep) -> Tensor[]");
    m.def("distill_backward(Tensor logits, int K, float tau, int reduction, Tensor saved, Tensor grad_out) -> Tensor");
    m.def("beam_step(Tensor logits, Tensor scores, int n, float tau, Tensor? finished, int eos) -> Tensor[]");
    m.def("beam_reorder(Tensor(a!)[] states, Tensor beams, Tensor? lengths, int? dim) -> ()");
}

TORCH_LIBRARY_IMPL(dot_amd, CUDA, m) {
    m.impl("top_logp", top_logp_op);
    m.impl("distill_forward", distill_forward_op);
    m.impl("distill_backward", distill_backward_op);
    m.impl("beam_step", beam_step_op);
    m.impl("beam_reorder", beam_reorder_op);
}

TORCH_LIBRARY_IMPL(dot_amd, Autograd, m) { m.impl("distill_forward", distill_forward_autograd); }
