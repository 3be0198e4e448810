// CPU implementations of the top log-probability, distillation and beam search
// operators (torch.ops.dot_amd.* under the CPU dispatch key): the definitions of
// include/dot_amd.h, row by row, in 64 bits.  Rows run in parallel; sums over rows
// are formed in row order, so results do not depend on the thread count.
#include <ATen/ATen.h>
#include <ATen/Parallel.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <limits>
#include <unordered_map>
#include <vector>

#include "beam_states.hpp"

namespace {

using at::Tensor;
using c10::optional;

constexpr double kInf = std::numeric_limits<double>::infinity();

Tensor rows_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.device().is_cpu() && t.dim() == 3 && t.size(2) >= 1, name, " must be a 3D CPU tensor with V >= 1");
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16,
                name, " must be float32, float16 or bfloat16");
    return t.to(at::kFloat).contiguous();
}

Tensor flags_of(const optional<Tensor>& m, const Tensor& x, const char* name) {
    if (!m.has_value()) return Tensor();
    TORCH_CHECK(m->device().is_cpu() && m->scalar_type() == at::kBool && m->dim() == 2 && m->size(0) == x.size(0) &&
                    m->size(1) == x.size(1),
                name, " must be a CPU bool tensor of the leading two sizes");
    return m->contiguous();
}
bool flag(const Tensor& m, int64_t r) { return m.defined() && m.const_data_ptr<bool>()[r]; }

// The largest logit and log sum exp((x - largest) / tau) of a row.
struct Lse {
    double top = -kInf, log_sum = -kInf;
    Lse(const float* x, int64_t V, double tau) {
        float most = -std::numeric_limits<float>::infinity();
        for (int64_t v = 0; v < V; ++v) most = std::max(most, x[v]);
        top = std::isinf(most) && most < 0 ? 0.0 : double(most);
        double sum = 0.0;
        for (int64_t v = 0; v < V; ++v) sum += std::exp((double(x[v]) - top) / tau);
        log_sum = std::log(sum);
    }
    // The logits are scaled and their difference taken in fp32, in 64 bits where that ends.
    double operator()(float x, double tau) const {
        const float inv = 1.0f / float(tau), zx = x * inv, zm = float(top) * inv, d = zx - zm;
        return (std::isnormal(inv) && std::isfinite(d) ? double(d) : (double(x) - top) / tau) - log_sum;
    }
};

// The k first tokens of a row by descending logit, equal ones by the lowest token.
std::vector<int64_t> best_of(const float* x, int64_t V, int64_t k) {
    std::vector<int64_t> at;
    for (int64_t v = 0; v < V; ++v)
        if (x[v] > -std::numeric_limits<float>::infinity()) at.push_back(v);  // not NaN either
    const auto end = at.begin() + std::min<int64_t>(k, int64_t(at.size()));
    std::partial_sort(at.begin(), end, at.end(),
                      [x](int64_t a, int64_t b) { return x[a] > x[b] || (x[a] == x[b] && a < b); });
    at.erase(end, at.end());
    return at;
}

std::vector<Tensor> top_logp_cpu(Tensor logits_, int64_t k, double tau, optional<Tensor> mask_) {
    const Tensor logits = rows_of(logits_, "logits"), mask = flags_of(mask_, logits, "mask");
    const int64_t B = logits.size(0), S = logits.size(1), V = logits.size(2);
    TORCH_CHECK(k >= 1 && k <= std::min<int64_t>(V, DOT_TOP_MAX) && tau > 0.0, "k or tau out of range");
    Tensor logp = at::full({B, S, k}, -kInf, logits.options());
    Tensor tokens = at::full({B, S, k}, -1, logits.options().dtype(at::kInt));
    const float* x = logits.const_data_ptr<float>();
    float* lp = logp.data_ptr<float>();
    int32_t* tp = tokens.data_ptr<int32_t>();
    at::parallel_for(0, B * S, 1, [&](int64_t r0, int64_t r1) {
        for (int64_t r = r0; r < r1; ++r) {
            if (mask.defined() && !flag(mask, r)) continue;
            const Lse lse(x + r * V, V, tau);
            const std::vector<int64_t> at = best_of(x + r * V, V, k);
            for (size_t e = 0; e < at.size(); ++e) {
                lp[r * k + int64_t(e)] = float(lse(x[r * V + at[e]], tau));
                tp[r * k + int64_t(e)] = int32_t(at[e]);
            }
        }
    });
    return {logp, tokens};
}

std::vector<Tensor> beam_step_cpu(Tensor logits_, Tensor scores_, int64_t n, double tau, optional<Tensor> finished_,
                                  int64_t eos) {
    const Tensor logits = rows_of(logits_, "logits"), finished = flags_of(finished_, logits, "finished");
    const int64_t B = logits.size(0), W = logits.size(1), V = logits.size(2);
    TORCH_CHECK(scores_.device().is_cpu() && scores_.dim() == 2 && scores_.size(0) == B && scores_.size(1) == W,
                "scores must be a CPU tensor of shape [B, W]");
    TORCH_CHECK(n >= 1 && n <= std::min<int64_t>(W * V, DOT_TOP_MAX) && tau > 0.0, "n or tau out of range");
    TORCH_CHECK(!finished.defined() || (eos >= 0 && eos < V), "finished beams need an eos in [0, V)");
    const Tensor scores = scores_.to(at::kFloat).contiguous();
    const auto i32 = logits.options().dtype(at::kInt);
    Tensor out = at::full({B, n}, -kInf, scores.options()), beams = at::full({B, n}, -1, i32);
    Tensor tokens = at::full({B, n}, -1, i32), done = at::zeros({B, n}, logits.options().dtype(at::kBool));
    const float *x = logits.const_data_ptr<float>(), *sp = scores.const_data_ptr<float>();
    struct Candidate {
        double total;
        int64_t beam, token;
    };
    at::parallel_for(0, B, 1, [&](int64_t b0, int64_t b1) {
        for (int64_t b = b0; b < b1; ++b) {
            std::vector<Candidate> all;
            for (int64_t w = 0; w < W; ++w) {
                const int64_t r = b * W + w;
                if (!(sp[r] > -std::numeric_limits<float>::infinity())) continue;
                if (flag(finished, r)) {
                    all.push_back({double(sp[r]), w, eos});
                    continue;
                }
                const Lse lse(x + r * V, V, tau);
                for (int64_t v : best_of(x + r * V, V, n)) {
                    const double total = double(sp[r]) + lse(x[r * V + v], tau);
                    if (total > -kInf) all.push_back({total, w, v});  // not NaN either
                }
            }
            std::stable_sort(all.begin(), all.end(),
                             [](const Candidate& p, const Candidate& q) { return p.total > q.total; });
            for (int64_t e = 0; e < std::min<int64_t>(n, int64_t(all.size())); ++e) {
                const Candidate& c = all[size_t(e)];
                out.data_ptr<float>()[b * n + e] = float(c.total);
                beams.data_ptr<int32_t>()[b * n + e] = int32_t(c.beam);
                tokens.data_ptr<int32_t>()[b * n + e] = int32_t(c.token);
                done.data_ptr<bool>()[b * n + e] = c.token == eos || flag(finished, b * W + c.beam);
            }
        }
    });
    if (eos < 0) return {out, beams, tokens};
    return {out, beams, tokens, done};
}

// ---------------------------------------------------------------------------
// Distillation
// ---------------------------------------------------------------------------
std::vector<Tensor> distill_forward_cpu(Tensor logits_, Tensor logp_, Tensor tokens_, optional<Tensor> mask_,
                                        double tau, int64_t direction, int64_t rest, int64_t reduction, bool keep) {
    const Tensor logits = rows_of(logits_, "logits"), mask = flags_of(mask_, logits, "mask");
    const int64_t B = logits.size(0), S = logits.size(1), V = logits.size(2);
    TORCH_CHECK(tokens_.device().is_cpu() && tokens_.dim() == 3 && tokens_.size(0) == B && tokens_.size(1) == S &&
                    (tokens_.scalar_type() == at::kInt || tokens_.scalar_type() == at::kLong),
                "teacher_tokens must be int32 or int64 of shape [B, S, K] on the CPU");
    TORCH_CHECK(logp_.device().is_cpu() && logp_.sizes() == tokens_.sizes(),
                "teacher_logp must be shaped as teacher_tokens");
    const int64_t K = tokens_.size(2);
    TORCH_CHECK(K >= 1 && K <= DOT_TOP_MAX && tau > 0.0, "K or tau out of range");
    const bool reverse = direction == DOT_DISTILL_REVERSE, bucket = rest == DOT_REST_BUCKET;
    TORCH_CHECK(bucket || !reverse, "the reverse direction needs the rest as a bucket");
    const Tensor tokens = tokens_.to(at::kLong).contiguous(), logp = logp_.to(at::kFloat).contiguous();
    const auto f32 = logits.options();
    Tensor value = at::zeros({B, S}, f32.dtype(at::kDouble)), live = at::zeros({B, S}, f32.dtype(at::kBool));
    // as for HIP tensors: row statistics, the named tokens' gradients, these tokens, weights
    const int64_t rows = B * S;
    Tensor saved = at::ones({keep ? 2 * rows + 2 * rows * K + B : 0}, f32);
    float* kept = saved.data_ptr<float>();
    float *own = kept + 2 * rows, *weight = own + 2 * rows * K;
    int32_t* own_tokens = reinterpret_cast<int32_t*>(own + rows * K);
    const float* xp = logits.const_data_ptr<float>();
    at::parallel_for(0, rows, 1, [&](int64_t r0, int64_t r1) {
        std::vector<int64_t> tok(static_cast<size_t>(K));
        for (int64_t r = r0; r < r1; ++r) {
            const float *x = xp + r * V, *t = logp.const_data_ptr<float>() + r * K;
            if (keep) kept[2 * r] = std::numeric_limits<float>::quiet_NaN();
            if (mask.defined() && !flag(mask, r)) continue;
            std::unordered_map<int64_t, int64_t> named;
            for (int64_t e = 0; e < K; ++e) {
                int64_t v = tokens.const_data_ptr<int64_t>()[r * K + e];
                if (v < 0 || v >= V || t[e] == -std::numeric_limits<float>::infinity()) v = -1;
                if (v >= 0 && !named.emplace(v, e).second) v = -1;
                tok[size_t(e)] = v;
            }
            if (named.empty()) continue;
            live.data_ptr<bool>()[r] = true;
            double top = -kInf, others_top = -kInf, s = 0.0, z = 0.0, most = -kInf, mass = 0.0;
            for (int64_t v = 0; v < V; ++v) {
                top = std::max(top, double(x[v]));
                if (!named.count(v)) others_top = std::max(others_top, double(x[v]));
            }
            if (top == -kInf) top = 0.0;
            const double base = others_top == -kInf ? 0.0 : others_top;
            for (int64_t v = 0; v < V; ++v)
                if (!named.count(v)) s += std::exp((double(x[v]) - base) / tau);
            for (int64_t e = 0; e < K; ++e)
                if (tok[size_t(e)] >= 0) {
                    z += std::exp((double(x[tok[size_t(e)]]) - top) / tau);
                    most = std::max(most, double(t[e]));
                }
            const bool none = s == 0.0;
            const double lr = none ? -kInf : (base - top) / tau + std::log(s);
            const double lz = std::log(z + std::exp(lr)), log_qr = lr - lz, qr = std::exp(log_qr);
            const double less = bucket ? 0.0 : most;
            for (int64_t e = 0; e < K; ++e)
                if (tok[size_t(e)] >= 0) mass += std::exp(double(t[e]) - less);
            const double scale = bucket ? 0.0 : std::log(mass) + less;  // of log P
            double pr = 0.0;
            if (bucket) {
                pr = 1.0 - mass;
                if (pr < 0.0) pr = 0.0;
            }
            double total = 0.0;
            for (int64_t e = 0; e < K; ++e) {
                if (tok[size_t(e)] < 0) continue;
                const double lp = double(t[e]) - scale, lq = (double(x[tok[size_t(e)]]) - top) / tau - lz;
                const double p = std::exp(lp);
                if (!reverse) total += p == 0.0 ? 0.0 : p * (lp - lq);
                else total += lq == -kInf ? 0.0 : std::exp(lq) * (lq - lp);
            }
            double other, all = 1.0;  // all: the sum of the P that the forward loss has
            if (!reverse) {
                const bool left = bucket && !(pr == 0.0 || (none && pr <= DOT_REST_ROUNDING));
                if (left) total += pr * (std::log(pr) - log_qr);
                else if (bucket) all = mass;
                other = all * qr - (left ? pr : 0.0);
            } else {
                const double log_pr = std::log(std::isnan(pr) ? pr : std::max(pr, std::ldexp(1.0, -24)));
                if (!none) total += qr * (log_qr - log_pr);
                other = none ? 0.0 : qr * (log_qr - log_pr - total);
            }
            value.data_ptr<double>()[r] = total;
            if (!keep) continue;
            kept[2 * r] = float(base);
            kept[2 * r + 1] = none ? 0.0f : float(other / s);
            for (int64_t e = 0; e < K; ++e) {
                own_tokens[r * K + e] = int32_t(tok[size_t(e)]);
                if (tok[size_t(e)] < 0) continue;
                const double lp = double(t[e]) - scale, lq = (double(x[tok[size_t(e)]]) - top) / tau - lz;
                const double q = std::exp(lq);
                own[r * K + e] = float(!reverse ? all * q - std::exp(lp) : lq == -kInf ? 0.0 : q * (lq - lp - total));
            }
        }
    });
    if (reduction == DOT_REDUCE_NONE) return {value.to(at::kFloat), saved};
    Tensor out = at::empty({B}, f32);
    for (int64_t b = 0; b < B; ++b) {
        double sum = 0.0;
        int64_t n = 0;
        for (int64_t r = b * S; r < (b + 1) * S; ++r) {
            sum += value.data_ptr<double>()[r];
            n += live.data_ptr<bool>()[r];
        }
        const double w = reduction == DOT_REDUCE_MEAN ? 1.0 / double(std::max<int64_t>(n, 1)) : 1.0;
        out.data_ptr<float>()[b] = float(sum * w);
        if (keep) weight[b] = float(w);
    }
    return {out, saved};
}

Tensor distill_backward_cpu(Tensor logits_, int64_t K, double tau, int64_t reduction, Tensor saved, Tensor grad_out_) {
    const Tensor logits = rows_of(logits_, "logits");
    const int64_t B = logits.size(0), S = logits.size(1), V = logits.size(2), rows = B * S;
    const bool per_token = reduction == DOT_REDUCE_NONE;
    TORCH_CHECK(grad_out_.device().is_cpu() && grad_out_.numel() == (per_token ? rows : B) &&
                    saved.scalar_type() == at::kFloat && saved.is_contiguous() &&
                    saved.numel() == 2 * rows + 2 * rows * K + B,
                "grad_out or saved has the wrong size");
    const Tensor go = grad_out_.to(at::kFloat).contiguous();
    const float *kept = saved.const_data_ptr<float>(), *own = kept + 2 * rows, *weight = own + 2 * rows * K;
    const int32_t* own_tokens = reinterpret_cast<const int32_t*>(own + rows * K);
    Tensor grad = at::zeros({B, S, V}, logits.options());
    float* out = grad.data_ptr<float>();
    at::parallel_for(0, rows, 1, [&](int64_t r0, int64_t r1) {
        for (int64_t r = r0; r < r1; ++r) {
            if (std::isnan(kept[2 * r])) continue;
            const double up = go.const_data_ptr<float>()[per_token ? r : r / S];
            const double c = (reduction == DOT_REDUCE_MEAN ? up * weight[r / S] : up) / tau;
            const float* x = logits.const_data_ptr<float>() + r * V;
            for (int64_t v = 0; v < V; ++v)
                out[r * V + v] = float(c * kept[2 * r + 1] * std::exp((double(x[v]) - kept[2 * r]) / tau));
            for (int64_t e = 0; e < K; ++e)
                if (own_tokens[r * K + e] >= 0) out[r * V + own_tokens[r * K + e]] = float(c * own[r * K + e]);
        }
    });
    return grad.to(logits_.scalar_type());
}

// ---------------------------------------------------------------------------
// Beams
// ---------------------------------------------------------------------------
void beam_reorder_cpu(at::TensorList states, const Tensor& beams_, const optional<Tensor>& lengths_,
                     optional<int64_t> dim) {
    const std::vector<dot_beam_state> all = beam_states(states, beams_, lengths_, dim);
    const Tensor chosen = beams_.contiguous(), used_of = lengths_.has_value() ? lengths_->contiguous() : Tensor();
    dot_beam_reorder_args a{};
    a.states = all.data();
    a.count = int(all.size());
    a.B = int(beams_.size(0));
    a.W = int(beams_.size(1));
    a.beams = chosen.const_data_ptr();
    a.beams_are_int64 = chosen.scalar_type() == at::kLong;
    a.lengths = used_of.defined() ? used_of.const_data_ptr() : nullptr;
    a.lengths_are_int64 = used_of.defined() && used_of.scalar_type() == at::kLong;
    const int rc = dot_beam_reorder_check(&a);
    TORCH_CHECK_VALUE(rc != DOT_ERR_INVALID_ARG, dot_last_error());
    TORCH_CHECK(rc == DOT_OK, "dot_beam_reorder_check failed (code ", rc, "): ", dot_last_error());
    const Tensor beams = chosen.to(at::kLong), lengths = used_of.defined() ? used_of.to(at::kLong) : Tensor();
    const int64_t* parents = beams.const_data_ptr<int64_t>();
    for (const dot_beam_state& s : all) {
        std::vector<char> was;
        for (int64_t b = 0; b < a.B; ++b) {
            int64_t used = s.positions;
            if (lengths.defined())
                used = std::min(std::max<int64_t>(lengths.const_data_ptr<int64_t>()[b], 0), s.positions);
            const size_t one = size_t(s.outer * used * s.inner);
            was.resize(one * size_t(a.W));
            auto copy = [&](int64_t w, char* dense, bool in) {
                for (int64_t o = 0; o < s.outer; ++o)
                    for (int64_t p = 0; p < used; ++p, dense += s.inner) {
                        char* at = static_cast<char*>(s.data) + b * s.stride_b + w * s.stride_w +
                                   o * s.stride_outer + p * s.stride_p;
                        if (in) std::memcpy(dense, at, size_t(s.inner));
                        else std::memcpy(at, dense, size_t(s.inner));
                    }
            };
            for (int64_t w = 0; w < a.W; ++w) copy(w, was.data() + size_t(w) * one, true);
            for (int64_t w = 0; w < a.W; ++w) {
                const int64_t p = parents[b * a.W + w];
                if (p >= 0 && p < a.W && p != w) copy(w, was.data() + size_t(p) * one, false);
            }
        }
    }
    states_changed(states);
}

}  // namespace

TORCH_LIBRARY_IMPL(dot_amd, CPU, m) {
    m.impl("top_logp", top_logp_cpu);
    m.impl("distill_forward", distill_forward_cpu);
    m.impl("distill_backward", distill_backward_cpu);
    m.impl("beam_step", beam_step_cpu);
    m.impl("beam_reorder", beam_reorder_cpu);
}
