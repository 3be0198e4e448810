// CPU implementations of the routing, sequence log-probability and preference
// operators (torch.ops.dot_amd.* under the CPU dispatch key): the definitions
// of include/dot_amd.h, row by row, with sums and statistics in 64 bits.  Rows
// run in parallel; sums over rows are formed in row order, so results do not
// depend on the thread count.
#include <ATen/ATen.h>
#include <ATen/Parallel.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <vector>

#include "../../include/dot_amd.h"

namespace {

using at::Tensor;
using c10::optional;

constexpr double kInf = std::numeric_limits<double>::infinity();

void check_cpu(const Tensor& t, const char* name) {
    TORCH_CHECK(t.device().is_cpu(), name, " must be a CPU tensor");
}

void check_floats(const Tensor& t, const char* name) {
    check_cpu(t, name);
    TORCH_CHECK(t.dim() == 3, name, " must be 3D");
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16,
                name, " must be float32, float16 or bfloat16");
}

Tensor f32c(const optional<Tensor>& t, const char* name) {
    if (!t.has_value()) return Tensor();
    check_cpu(*t, name);
    return t->to(at::kFloat).contiguous();
}

Tensor longs(const Tensor& t, const char* name) {
    check_cpu(t, name);
    TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
    return t.to(at::kLong).contiguous();
}

Tensor mask_of(const optional<Tensor>& mask, const Tensor& x) {
    if (!mask.has_value()) return Tensor();
    check_cpu(*mask, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kBool && mask->dim() == 2 && mask->size(0) == x.size(0) &&
                    mask->size(1) == x.size(1),
                "mask must be bool of the leading two sizes");
    return mask->contiguous();
}
const bool* mask_ptr(const Tensor& m) { return m.defined() ? m.const_data_ptr<bool>() : nullptr; }

double logistic(double x) { return x >= 0 ? 1.0 / (1.0 + std::exp(-x)) : std::exp(x) / (1.0 + std::exp(x)); }

// Masses whose sum is below the smallest normal fp32 count as none (the device
// forms the reciprocal in fp32), and so does the logistic mass of a single score
// (the device's exponential ends there); NaN stays NaN.
bool none(double mass) { return std::fabs(mass) < double(std::numeric_limits<float>::min()); }

double logistic_mass(double x) {
    const double q = logistic(x);
    return none(q) ? 0.0 : q;
}

// Masses of a row of E scores; returns their sum (softmax: q sums to 1, or to 0
// where every score is -inf).
double row_masses(const float* s, int64_t E, int64_t scoring, double* q) {
    double sum = 0.0;
    if (scoring == DOT_SCORING_SOFTMAX) {
        float top = -std::numeric_limits<float>::infinity();
        for (int64_t e = 0; e < E; ++e) top = std::max(top, s[e]);
        const double base = std::isinf(top) && top < 0 ? 0.0 : double(top);
        for (int64_t e = 0; e < E; ++e) sum += q[e] = std::exp(double(s[e]) - base);
        for (int64_t e = 0; e < E; ++e) q[e] = sum == 0.0 ? 0.0 : q[e] / sum;
        return sum == 0.0 ? 0.0 : sum / sum;
    }
    for (int64_t e = 0; e < E; ++e) {
        q[e] = scoring == DOT_SCORING_SIGMOID ? logistic_mass(s[e]) : double(s[e]) == -kInf ? 0.0 : double(s[e]);
        sum += q[e];
    }
    return sum;
}

void check_routing(int64_t E, int64_t k, int64_t scoring, bool select) {
    TORCH_CHECK(E >= 1 && E <= DOT_ROUTING_MAX_EXPERTS, "E out of range");
    TORCH_CHECK(k >= 1 && k <= DOT_ROUTING_MAX_K && (!select || k <= E), "k out of range");
    TORCH_CHECK(scoring >= DOT_SCORING_SOFTMAX && scoring <= DOT_SCORING_PLAN, "unknown scoring");
}

std::vector<Tensor> routing_forward_cpu(Tensor scores_, int64_t k, int64_t scoring, bool normalize,
                                        optional<Tensor> bias_, optional<Tensor> mask_, optional<Tensor> given_) {
    check_floats(scores_, "scores");
    const Tensor scores = scores_.to(at::kFloat).contiguous();
    const int64_t B = scores.size(0), N = scores.size(1), E = scores.size(2);
    const bool select = !given_.has_value();
    check_routing(E, k, scoring, select);
    const Tensor mask = mask_of(mask_, scores), bias = f32c(bias_, "bias");
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == E), "bias must have shape [E]");
    Tensor given;
    if (!select) {
        given = longs(*given_, "experts");
        TORCH_CHECK(given.dim() == 3 && given.size(0) == B && given.size(1) == N && given.size(2) == k,
                    "experts must have shape [B, N, k]");
    }
    const auto f32 = scores.options(), i32 = scores.options().dtype(at::kInt);
    Tensor weights = select ? at::zeros({B, N, k}, f32) : at::empty({0}, f32);
    Tensor experts = select ? at::full({B, N, k}, -1, i32) : at::empty({0}, i32);
    Tensor counts = at::zeros({B, E}, i32), tokens = at::zeros({B}, i32), loss = at::zeros({B}, f32);
    const float* sp = scores.const_data_ptr<float>();
    const float* bp = bias.defined() ? bias.const_data_ptr<float>() : nullptr;
    const bool* mp = mask_ptr(mask);
    const float neg = -std::numeric_limits<float>::infinity();
    if (select) {
        float* wp = weights.data_ptr<float>();
        int32_t* ep = experts.data_ptr<int32_t>();
        at::parallel_for(0, B * N, 64, [&](int64_t r0, int64_t r1) {
            std::vector<std::pair<float, int32_t>> keys;
            std::vector<double> q(static_cast<size_t>(E));
            for (int64_t r = r0; r < r1; ++r) {
                if (mp && !mp[r]) continue;
                const float* s = sp + r * E;
                const double sum = row_masses(s, E, scoring, q.data());
                keys.clear();
                for (int64_t e = 0; e < E; ++e) {
                    const float key = s[e] + (bp ? bp[e] : 0.0f);
                    if (key > neg && (scoring != DOT_SCORING_PLAN || s[e] > 0.0f)) keys.emplace_back(key, int32_t(e));
                }
                const int64_t have = std::min<int64_t>(k, int64_t(keys.size()));
                std::partial_sort(keys.begin(), keys.begin() + have, keys.end(), [](const auto& a, const auto& b) {
                    return a.first > b.first || (a.first == b.first && a.second < b.second);
                });
                float most = neg;
                for (int64_t i = 0; i < have; ++i) most = std::max(most, s[keys[size_t(i)].second]);
                double w[DOT_ROUTING_MAX_K], z = 0.0;
                for (int64_t i = 0; i < have; ++i) {
                    const int32_t e = keys[size_t(i)].second;
                    w[i] = normalize && scoring == DOT_SCORING_SOFTMAX ? std::exp(double(s[e]) - most) + (sum - sum)
                                                                       : q[size_t(e)];
                    z += w[i];
                }
                for (int64_t i = 0; i < have; ++i) {
                    ep[r * k + i] = keys[size_t(i)].second;
                    wp[r * k + i] = float(!normalize ? w[i] : none(z) ? 0.0 : w[i] / z);
                }
            }
        });
    }
    const int32_t* ep = select ? experts.const_data_ptr<int32_t>() : nullptr;
    const int64_t* gp = select ? nullptr : given.const_data_ptr<int64_t>();
    int32_t *cp = counts.data_ptr<int32_t>(), *tp = tokens.data_ptr<int32_t>();
    float* lp = loss.data_ptr<float>();
    at::parallel_for(0, B, 1, [&](int64_t b0, int64_t b1) {
        std::vector<double> q(static_cast<size_t>(E)), share(static_cast<size_t>(E));
        for (int64_t b = b0; b < b1; ++b) {
            std::fill(share.begin(), share.end(), 0.0);
            for (int64_t r = b * N; r < (b + 1) * N; ++r) {
                if (mp && !mp[r]) continue;
                ++tp[b];
                for (int64_t i = 0; i < k; ++i) {
                    const int64_t e = select ? ep[r * k + i] : gp[r * k + i];
                    if (e >= 0 && e < E) ++cp[b * E + e];
                }
                const double sum = row_masses(sp + r * E, E, scoring, q.data());
                if (none(sum)) continue;
                for (int64_t e = 0; e < E; ++e) share[size_t(e)] += q[size_t(e)] / sum;
            }
            double dot = 0.0;
            for (int64_t e = 0; e < E; ++e) dot += share[size_t(e)] * cp[b * E + e];
            const double n = tp[b];
            lp[b] = n > 0 ? float(dot * E / (k * n * n)) : 0.0f;
        }
    });
    std::vector<Tensor> out{counts, loss};
    if (select) out.insert(out.end(), {weights, experts});
    if (mask.defined()) out.push_back(tokens);
    return out;
}

Tensor routing_backward_cpu(Tensor scores_, int64_t k, int64_t scoring, bool normalize, optional<Tensor> mask_,
                            Tensor counts_, optional<Tensor> tokens_, optional<Tensor> grad_loss_,
                            optional<Tensor> weights_, optional<Tensor> experts_, optional<Tensor> grad_weights_) {
    check_floats(scores_, "scores");
    const Tensor scores = scores_.to(at::kFloat).contiguous();
    const int64_t B = scores.size(0), N = scores.size(1), E = scores.size(2);
    check_routing(E, k, scoring, false);
    const Tensor mask = mask_of(mask_, scores);
    const Tensor counts = longs(counts_, "counts");
    TORCH_CHECK(tokens_.has_value() == mask.defined(), "tokens come with a mask");
    const Tensor tokens = tokens_.has_value() ? longs(*tokens_, "tokens") : at::full({B}, N, counts.options());
    const Tensor gl = f32c(grad_loss_, "grad_loss"), gw = f32c(grad_weights_, "grad_weights");
    TORCH_CHECK(counts.numel() == B * E && tokens.numel() == B && (!gl.defined() || gl.numel() == B),
                "counts, tokens and grad_loss must have shapes [B, E], [B] and [B]");
    Tensor w, ex;
    if (gw.defined()) {
        TORCH_CHECK(weights_.has_value() && experts_.has_value(), "grad_weights needs weights and experts");
        w = f32c(weights_, "weights");
        ex = longs(*experts_, "experts");
        TORCH_CHECK(gw.numel() == B * N * k && w.numel() == B * N * k && ex.numel() == B * N * k,
                    "weights, experts and grad_weights must have shape [B, N, k]");
    }
    Tensor grad = at::zeros({B, N, E}, scores.options());
    const float* sp = scores.const_data_ptr<float>();
    float* out = grad.data_ptr<float>();
    const bool* mp = mask_ptr(mask);
    at::parallel_for(0, B * N, 64, [&](int64_t r0, int64_t r1) {
        std::vector<double> q(static_cast<size_t>(E)), h(static_cast<size_t>(E)), add(static_cast<size_t>(E));
        for (int64_t r = r0; r < r1; ++r) {
            if (mp && !mp[r]) continue;
            const int64_t b = r / N;
            const float* s = sp + r * E;
            const double sum = row_masses(s, E, scoring, q.data());
            const double n = double(tokens.const_data_ptr<int64_t>()[b]);
            const double coef = gl.defined() && n > 0 ? gl.const_data_ptr<float>()[b] * double(E) / (k * n * n) : 0.0;
            for (int64_t e = 0; e < E; ++e) {
                h[size_t(e)] = coef * double(counts.const_data_ptr<int64_t>()[b * E + e]);
                add[size_t(e)] = 0.0;
            }
            const bool soft = scoring == DOT_SCORING_SOFTMAX;
            if (gw.defined()) {
                const float *wp = w.const_data_ptr<float>() + r * k, *dp = gw.const_data_ptr<float>() + r * k;
                const int64_t* ep = ex.const_data_ptr<int64_t>() + r * k;
                double dot = 0.0, mass = 0.0;
                for (int64_t i = 0; i < k; ++i)
                    if (ep[i] >= 0 && ep[i] < E) {
                        dot += double(wp[i]) * dp[i];
                        mass += q[size_t(ep[i])];
                    }
                for (int64_t i = 0; i < k; ++i) {
                    if (ep[i] < 0 || ep[i] >= E) continue;
                    double v = dp[i];
                    if (normalize) v = soft ? wp[i] * (v - dot) : none(mass) ? 0.0 : (v - dot) / mass;
                    if (soft && !normalize) h[size_t(ep[i])] += v;
                    else add[size_t(ep[i])] = v;
                }
            }
            const double inv = none(sum) ? 0.0 : 1.0 / sum;
            double ph = 0.0;
            for (int64_t e = 0; e < E; ++e) ph += q[size_t(e)] * inv * h[size_t(e)];
            for (int64_t e = 0; e < E; ++e) {
                double g = (h[size_t(e)] - ph) * (soft ? q[size_t(e)] : inv) + add[size_t(e)];
                if (scoring == DOT_SCORING_SIGMOID) {
                    const double t = std::exp(-std::fabs(double(s[e])));
                    g *= none(t) ? 0.0 : t / ((1.0 + t) * (1.0 + t));
                }
                out[r * E + e] = float(g);
            }
        }
    });
    return grad.to(scores_.scalar_type());
}

// Log-sum-exp of x / tau over a row: (max, sum of exp((x - max) / tau)).
std::pair<double, double> row_lse(const float* x, int64_t V, double tau) {
    float top = -std::numeric_limits<float>::infinity();
    for (int64_t v = 0; v < V; ++v) top = std::max(top, x[v]);
    const double base = std::isinf(top) && top < 0 ? 0.0 : double(top);
    double sum = 0.0;
    for (int64_t v = 0; v < V; ++v) sum += std::exp((double(x[v]) - base) / tau);
    return {base, sum};
}

struct Positions {
    Tensor logits, tokens, mask;
    int64_t B, S, V;
    Positions(const Tensor& logits_, const Tensor& tokens_, const optional<Tensor>& mask_) {
        check_floats(logits_, "logits");
        logits = logits_.to(at::kFloat).contiguous();
        tokens = longs(tokens_, "tokens");
        B = logits.size(0), S = logits.size(1), V = logits.size(2);
        TORCH_CHECK(V >= 1, "V must be >= 1");
        TORCH_CHECK(tokens.dim() == 2 && tokens.size(0) == B && tokens.size(1) == S, "tokens must have shape [B, S]");
        mask = mask_of(mask_, logits);
    }
    int64_t token(int64_t r) const {
        if (mask.defined() && !mask.const_data_ptr<bool>()[r]) return -1;
        const int64_t t = tokens.const_data_ptr<int64_t>()[r];
        return t >= 0 && t < V ? t : -1;
    }
    const float* row(int64_t r) const { return logits.const_data_ptr<float>() + r * V; }
};

std::vector<Tensor> sequence_logp_forward_cpu(Tensor logits, Tensor tokens, optional<Tensor> ref_,
                                              optional<Tensor> mask, double tau, int64_t reduction, bool keep) {
    TORCH_CHECK(tau > 0.0, "tau must be > 0");
    const Positions p(logits, tokens, mask);
    const auto f32 = p.logits.options();
    Tensor ref;
    if (ref_.has_value()) {
        check_cpu(*ref_, "ref_logp");
        ref = ref_->to(at::kDouble).contiguous();
        TORCH_CHECK((ref.dim() == 1 && ref.size(0) == p.B && reduction != DOT_REDUCE_NONE) ||
                        (ref.dim() == 2 && ref.size(0) == p.B && ref.size(1) == p.S),
                    "ref_logp must have shape [B] or [B, S]");
    }
    Tensor value = at::zeros({p.B, p.S}, f32.dtype(at::kDouble));
    // as for HIP tensors: row statistics (which the backward here forms again), then weights
    Tensor saved = at::ones({keep ? (2 * p.S + 1) * p.B : 0}, f32);
    double* vp = value.data_ptr<double>();
    at::parallel_for(0, p.B * p.S, 1, [&](int64_t r0, int64_t r1) {
        for (int64_t r = r0; r < r1; ++r) {
            const int64_t t = p.token(r);
            if (t < 0) continue;
            const auto [top, sum] = row_lse(p.row(r), p.V, tau);
            vp[r] = (double(p.row(r)[t]) - top) / tau - std::log(sum);
            if (ref.defined() && ref.dim() == 2) vp[r] -= ref.const_data_ptr<double>()[r];
        }
    });
    if (reduction == DOT_REDUCE_NONE) return {value.to(at::kFloat), saved};
    Tensor out = at::empty({p.B}, f32);
    for (int64_t b = 0; b < p.B; ++b) {
        double sum = 0.0;
        int64_t n = 0;
        for (int64_t r = b * p.S; r < (b + 1) * p.S; ++r) {
            if (p.token(r) < 0) continue;
            sum += vp[r];
            ++n;
        }
        const double w = reduction == DOT_REDUCE_MEAN ? 1.0 / double(std::max<int64_t>(n, 1)) : 1.0;
        sum *= w;
        if (ref.defined() && ref.dim() == 1) sum -= ref.const_data_ptr<double>()[b];
        out.data_ptr<float>()[b] = float(sum);
        if (keep) saved.data_ptr<float>()[2 * p.B * p.S + b] = float(w);
    }
    return {out, saved};
}

Tensor sequence_logp_backward_cpu(Tensor logits, Tensor tokens, optional<Tensor> mask, double tau, int64_t reduction,
                                  Tensor saved_, Tensor grad_out_) {
    const Positions p(logits, tokens, mask);
    const Tensor go = f32c(grad_out_, "grad_out"), saved = f32c(saved_, "saved");
    const bool per_token = reduction == DOT_REDUCE_NONE;
    TORCH_CHECK(go.numel() == (per_token ? p.B * p.S : p.B) && saved.numel() == (2 * p.S + 1) * p.B, "grad_out has the wrong size");
    const float* weight = saved.const_data_ptr<float>() + 2 * p.B * p.S;
    Tensor grad = at::zeros({p.B, p.S, p.V}, p.logits.options());
    float* out = grad.data_ptr<float>();
    at::parallel_for(0, p.B * p.S, 1, [&](int64_t r0, int64_t r1) {
        for (int64_t r = r0; r < r1; ++r) {
            const int64_t t = p.token(r);
            if (t < 0) continue;
            const int64_t b = r / p.S;
            const double c = double(go.const_data_ptr<float>()[per_token ? r : b]) * weight[b] / tau;
            const float* x = p.row(r);
            const auto [top, sum] = row_lse(x, p.V, tau);
            for (int64_t v = 0; v < p.V; ++v)
                out[r * p.V + v] = float(c * ((v == t ? 1.0 : 0.0) - std::exp((double(x[v]) - top) / tau) / sum));
        }
    });
    return grad.to(logits.scalar_type());
}

struct PairLoss {
    int64_t type;
    double beta, smoothing;
    // f(d) and its slope
    std::pair<double, double> operator()(double gap) const {
        if (type == DOT_PREFER_SIGMOID) {
            const double d = beta * gap, tail = std::log1p(std::exp(-std::fabs(d)));
            double f = tail + (1.0 - smoothing) * std::max(-d, 0.0);
            if (smoothing > 0.0) f += smoothing * std::max(d, 0.0);
            return {f, beta * (smoothing * logistic(d) - (1.0 - smoothing) * logistic(-d))};
        }
        if (type == DOT_PREFER_HINGE) {
            const double room = 1.0 - beta * gap;
            if (room <= 0.0) return {0.0, 0.0};
            return {room, std::isnan(room) ? room : -beta};
        }
        const double miss = gap - 0.5 / beta;
        return {miss * miss, 2.0 * miss};
    }
};

struct Sides {
    Tensor ratio, plan;
    int64_t P, Q;
    Sides(const Tensor& ratio_, const optional<Tensor>& plan_) {
        ratio = f32c(ratio_, "log_ratio");
        plan = f32c(plan_, "plan");
        TORCH_CHECK(ratio.dim() == 1 && (!plan.defined() || plan.dim() == 2), "log_ratio must be 1D, plan 2D");
        P = plan.defined() ? plan.size(0) : ratio.size(0) / 2;
        Q = plan.defined() ? plan.size(1) : ratio.size(0) / 2;
        TORCH_CHECK(P + Q == ratio.size(0), "log_ratio must hold the P + Q answers of a [P, Q] plan, or pairs");
    }
};

Tensor preference_forward_cpu(Tensor ratio_, optional<Tensor> plan_, int64_t type, double beta, double smoothing) {
    const Sides s(ratio_, plan_);
    const PairLoss f{type, beta, smoothing};
    Tensor loss = at::empty({s.P}, s.ratio.options());
    const float* r = s.ratio.const_data_ptr<float>();
    for (int64_t i = 0; i < s.P; ++i) {
        double sum = 0.0;
        if (!s.plan.defined()) sum = f(double(r[i]) - r[s.P + i]).first;
        else
            for (int64_t j = 0; j < s.Q; ++j) {
                const double x = s.plan.const_data_ptr<float>()[i * s.Q + j];
                if (x != 0.0) sum += x * f(double(r[i]) - r[s.P + j]).first;  // 0 leaves the pair out
            }
        loss.data_ptr<float>()[i] = float(sum);
    }
    return loss;
}

std::vector<Tensor> preference_backward_cpu(Tensor ratio_, optional<Tensor> plan_, int64_t type, double beta,
                                            double smoothing, Tensor grad_loss_, bool want_plan) {
    const Sides s(ratio_, plan_);
    const PairLoss f{type, beta, smoothing};
    const Tensor gl = f32c(grad_loss_, "grad_loss");
    TORCH_CHECK(gl.numel() == s.P, "grad_loss must have shape [P]");
    std::vector<double> acc(size_t(s.P + s.Q), 0.0);
    Tensor grad_plan = want_plan && s.plan.defined() ? at::empty_like(s.plan) : at::empty({0}, s.ratio.options());
    const float* r = s.ratio.const_data_ptr<float>();
    for (int64_t i = 0; i < s.P; ++i) {
        const double g = gl.const_data_ptr<float>()[i];
        for (int64_t j = s.plan.defined() ? 0 : i; j < (s.plan.defined() ? s.Q : i + 1); ++j) {
            const auto [v, slope] = f(double(r[i]) - r[s.P + j]);
            const double x = s.plan.defined() ? double(s.plan.const_data_ptr<float>()[i * s.Q + j]) : 1.0;
            const double pull = x == 0.0 ? 0.0 : g * slope * x;
            acc[size_t(i)] += pull;
            acc[size_t(s.P + j)] -= pull;
            if (grad_plan.numel()) grad_plan.data_ptr<float>()[i * s.Q + j] = x == 0.0 && !(v < kInf) ? 0.0f : float(g * v);
        }
    }
    Tensor grad_ratio = at::empty_like(s.ratio);
    for (size_t i = 0; i < acc.size(); ++i) grad_ratio.data_ptr<float>()[i] = float(acc[i]);
    return {grad_ratio, grad_plan};
}

}  // namespace

TORCH_LIBRARY_IMPL(dot_amd, CPU, m) {
    m.impl("routing_forward", routing_forward_cpu);
    m.impl("routing_backward", routing_backward_cpu);
    m.impl("sequence_logp_forward", sequence_logp_forward_cpu);
    m.impl("sequence_logp_backward", sequence_logp_backward_cpu);
    m.impl("preference_forward", preference_forward_cpu);
    m.impl("preference_backward", preference_backward_cpu);
}
