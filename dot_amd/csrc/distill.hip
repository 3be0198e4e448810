// C ABI of the distillation loss: argument checks and launches.
#include <algorithm>
#include <cmath>

#include "distill.cuh"
#include "host.hpp"

namespace dot_amd {
namespace {

// Workgroups per row: rows alone fill the chip, fewer are split, into spans of at least two
// packs per thread, and into as many as keep the bits of a span in LDS.  The forward is
// split for fewer workgroups, since its parts are joined by a launch more (774 rows of
// 50021 fp32 whole 23.2 us, in 3 parts 20.3 + 7.7).
int splits_of(int B, int S, int V, int dtype, bool backward) {
    const int64_t rows = int64_t(B) * S, fill = backward ? 2048 : 512;
    const int packs = V / (16 / dtype_bytes(dtype));
    const int64_t want = rows > 0 ? (fill + rows - 1) / rows : 1;
    const int64_t most = std::max(1, packs / (2 * kBlock));
    const int64_t least = (int64_t(V) + distill::kMaxSpan - 1) / distill::kMaxSpan;
    return int(std::max(std::min(want, most), least));
}

// Bytes of LDS for the bits of a span: its whole packs, a head and a tail.
size_t words_bytes(int V, int dtype, int splits) {
    const int pn = 16 / dtype_bytes(dtype);
    const int packs = V / pn, per = (packs + splits - 1) / splits;
    return size_t(32 + per * pn + 2 * pn + 31) / 32 * 4;
}

template <class A>
int check(const A* a) {
    if (!known_dtype(a->dtype)) return fail(DOT_ERR_INVALID_ARG, "dtype must be DOT_F32, DOT_F16 or DOT_BF16");
    if (a->B < 0 || a->S < 0) return fail(DOT_ERR_INVALID_ARG, "B and S must be >= 0");
    if (a->V < 1) return fail(DOT_ERR_INVALID_ARG, "V must be >= 1");
    if (a->K < 1) return fail(DOT_ERR_INVALID_ARG, "K must be >= 1");
    if (a->K > DOT_TOP_MAX) return fail(DOT_ERR_UNSUPPORTED, "at most DOT_TOP_MAX tokens of a position are supported");
    // a grid dimension holds less than 2^32 threads
    if (a->V > (1 << 24) || int64_t(a->B) * a->S > (1 << 23) ||
        int64_t(a->B) * a->S * splits_of(a->B, a->S, a->V, a->dtype, true) > (1 << 23))
        return fail(DOT_ERR_UNSUPPORTED, "V must be at most 2^24 and B * S (times V / 2^18) at most 2^23");
    if (!(a->tau > 0.0) || !std::isfinite(a->tau)) return fail(DOT_ERR_INVALID_ARG, "tau must be > 0");
    if (a->tau < 1e-20 || a->tau > 1e20) return fail(DOT_ERR_UNSUPPORTED, "tau must be in [1e-20, 1e20]");
    if (a->reduction != DOT_REDUCE_NONE && a->reduction != DOT_REDUCE_SUM && a->reduction != DOT_REDUCE_MEAN)
        return fail(DOT_ERR_INVALID_ARG, "reduction must be a DOT_REDUCE_* value");
    return DOT_OK;
}

template <class A>
seqlogp::Rows rows_of(const A* a, bool training, bool backward) {
    seqlogp::Rows r{};
    r.logits = a->logits;
    r.sb = a->stride_b;
    r.ss = a->stride_s;
    r.B = a->B;
    r.S = a->S;
    r.V = a->V;
    r.mask = a->mask;
    const double k = 1.4426950408889634074 / a->tau;
    r.k = float(k);
    r.klo = 0.0f;
    if (a->dtype == DOT_F32) {  // klo > 0, as in the sequence log-probabilities
        if (double(r.k) >= k) r.k = std::nextafter(r.k, 0.0f);
        r.klo = float(k - double(r.k));
    }
    r.splits = splits_of(a->B, a->S, a->V, a->dtype, backward);
    // past the caches but for the rows that the backward begins with, as for the
    // sequence log-probabilities
    const int64_t rows = int64_t(a->B) * a->S, row_bytes = int64_t(a->V) * dtype_bytes(a->dtype);
    r.cached = 0;
    if (rows * row_bytes > (int64_t(256) << 20))
        r.cached = training ? std::max<int64_t>(0, rows - (int64_t(224) << 20) / row_bytes) : rows;
    return r;
}

}  // namespace
}  // namespace dot_amd

using namespace dot_amd;

namespace {
struct Workspace {
    distill::Value* values;
    distill::Part* parts;
    size_t bytes;
};
Workspace carve(void* ws, int B, int S, int V, int dtype, int reduction) {
    Carver c(ws);
    Workspace w{};
    const size_t rows = size_t(B) * S;
    if (reduction != DOT_REDUCE_NONE) w.values = c.take<distill::Value>(rows);
    const int splits = splits_of(B, S, V, dtype, false);
    if (splits > 1) w.parts = c.take<distill::Part>(rows * splits);
    w.bytes = c.used();
    return w;
}
}  // namespace

extern "C" size_t dot_distill_forward_workspace_bytes(int B, int S, int V, int dtype, int reduction) {
    if (B < 0 || S < 0 || V < 1 || !known_dtype(dtype)) return 0;
    return carve(nullptr, B, S, V, dtype, reduction).bytes;
}

extern "C" int dot_distill_forward(const dot_distill_fwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (int rc = check(a)) return rc;
    if (a->direction != DOT_DISTILL_FORWARD && a->direction != DOT_DISTILL_REVERSE)
        return fail(DOT_ERR_INVALID_ARG, "direction must be a DOT_DISTILL_* value");
    if (a->rest != DOT_REST_BUCKET && a->rest != DOT_REST_NONE)
        return fail(DOT_ERR_INVALID_ARG, "rest must be a DOT_REST_* value");
    if (a->direction == DOT_DISTILL_REVERSE && a->rest == DOT_REST_NONE)
        return fail(DOT_ERR_INVALID_ARG, "the reverse direction needs DOT_REST_BUCKET");
    const int64_t rows = int64_t(a->B) * a->S;
    if (a->B == 0 || (rows == 0 && a->reduction == DOT_REDUCE_NONE)) return ok();
    if (!a->out) return fail(DOT_ERR_INVALID_ARG, "out must be non-NULL");
    if (rows > 0 && (!a->logits || !a->tokens || !a->logp))
        return fail(DOT_ERR_INVALID_ARG, "logits, tokens and logp must be non-NULL");
    if (a->row_stats && (!a->own_tokens || !a->own_grad))
        return fail(DOT_ERR_INVALID_ARG, "row_stats comes with own_tokens and own_grad");
    const Workspace w = carve(a->workspace, a->B, a->S, a->V, a->dtype, a->reduction);
    if (w.bytes > 0 && (!a->workspace || a->workspace_bytes < w.bytes))
        return fail(DOT_ERR_WORKSPACE, "workspace smaller than dot_distill_forward_workspace_bytes()");
    const seqlogp::Rows r = rows_of(a, a->row_stats != nullptr, false);
    const distill::Teacher t{a->tokens, a->tokens_are_int64, a->logp, a->K};
    distill::Out o{};
    o.direction = a->direction;
    o.rest = a->rest;
    o.reduction = a->reduction;
    o.out = a->out;
    o.values = w.values;
    o.stats = reinterpret_cast<float2*>(a->row_stats);
    o.at = a->own_tokens;
    o.own = a->own_grad;
    if (rows > 0)
        dispatch_dtype(a->dtype, [&](auto tag) {
            using T = decltype(tag);
            {
                ProfScope prof("distill_row_stats", stream);
                hipLaunchKernelGGL((distill::row_stats<T>), dim3(unsigned(rows * r.splits)), dim3(kBlock),
                                   words_bytes(a->V, a->dtype, r.splits), stream, r, t, o, w.parts);
            }
            if (r.splits > 1) {
                ProfScope prof("distill_finish", stream);
                const unsigned blocks = unsigned((rows + kWavesPerBlock - 1) / kWavesPerBlock);
                hipLaunchKernelGGL((distill::finish_rows<T>), dim3(blocks), dim3(kBlock), 0, stream, r, t, o,
                                   static_cast<const distill::Part*>(w.parts));
            }
        });
    if (a->reduction != DOT_REDUCE_NONE) {
        ProfScope prof("distill_sum", stream);
        hipLaunchKernelGGL(distill::sum, batch_grid(1, a->B), dim3(seqlogp::kJoinBlock), 0, stream, a->B, a->S,
                           a->reduction, static_cast<const distill::Value*>(w.values), a->out, a->weight);
    }
    return check_launch("dot_distill_forward");
}

extern "C" int dot_distill_backward(const dot_distill_bwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (int rc = check(a)) return rc;
    const int64_t rows = int64_t(a->B) * a->S;
    if (rows == 0) return ok();
    if (!a->logits || !a->row_stats || !a->own_tokens || !a->own_grad || !a->grad_out || !a->grad_logits)
        return fail(DOT_ERR_INVALID_ARG,
                    "logits, row_stats, own_tokens, own_grad, grad_out and grad_logits must be non-NULL");
    if (a->reduction == DOT_REDUCE_MEAN && !a->weight)
        return fail(DOT_ERR_INVALID_ARG, "the gradient of a mean needs weight");
    const seqlogp::Rows r = rows_of(a, true, true);
    distill::GradArgs g{};
    g.K = a->K;
    g.inv_tau = float(1.0 / a->tau);
    g.reduction = a->reduction;
    g.stats = reinterpret_cast<const float2*>(a->row_stats);
    g.at = a->own_tokens;
    g.own = a->own_grad;
    g.weight = a->weight;
    g.grad_out = a->grad_out;
    g.grad_out_scalar = a->grad_out_scalar;
    g.grad = a->grad_logits;
    dispatch_dtype(a->dtype, [&](auto t) {
        ProfScope prof("distill_backward", stream);
        hipLaunchKernelGGL((distill::backward<decltype(t)>), dim3(unsigned(rows * r.splits)), dim3(kBlock), 0, stream,
                           r, g);
    });
    return check_launch("dot_distill_backward");
}
