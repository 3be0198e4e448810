// C ABI of the sequence log-probabilities: argument checks and launches.
#include <algorithm>
#include <cmath>

#include "host.hpp"
#include "seqlogp.cuh"

namespace dot_amd {
namespace {

// Workgroups per row: rows alone fill the chip (2048 workgroups, eight per
// CU); fewer rows are split, into spans of at least two packs per thread.  Split
// and whole, bf16: 1 x 131072 3.9 and 14.3 us, 7 x 32768 4.1 and 6.8, 64 x 131072
// 7.8 and 15.5, 512 x 32768 10.5 and 10.2 (4 parts).
int splits_of(int B, int S, int V, int dtype) {
    const int64_t rows = int64_t(B) * S;
    const int packs = V / (16 / dtype_bytes(dtype));
    const int64_t want = rows > 0 ? (2048 + rows - 1) / rows : 1;
    const int64_t most = std::max(1, packs / (2 * kBlock));
    return int(std::min(want, most));
}

int check_shape(int dtype, int B, int S, int V, double tau, int reduction) {
    if (!known_dtype(dtype)) return fail(DOT_ERR_INVALID_ARG, "dtype must be DOT_F32, DOT_F16 or DOT_BF16");
    if (B < 0 || S < 0) return fail(DOT_ERR_INVALID_ARG, "B and S must be >= 0");
    if (V < 1) return fail(DOT_ERR_INVALID_ARG, "V must be >= 1");
    // a grid dimension holds less than 2^32 threads
    if (V > (1 << 30) || int64_t(B) * S > (1 << 23))
        return fail(DOT_ERR_UNSUPPORTED, "V must be at most 2^30 and B * S at most 2^23");
    if (!(tau > 0.0) || !std::isfinite(tau)) return fail(DOT_ERR_INVALID_ARG, "tau must be > 0");
    // log2(e) / tau and its rest are normal floats
    if (tau < 1e-20 || tau > 1e20) return fail(DOT_ERR_UNSUPPORTED, "tau must be in [1e-20, 1e20]");
    if (reduction != DOT_REDUCE_NONE && reduction != DOT_REDUCE_SUM && reduction != DOT_REDUCE_MEAN)
        return fail(DOT_ERR_INVALID_ARG, "reduction must be a DOT_REDUCE_* value");
    return DOT_OK;
}

// First row that is read through the caches: all rows of logits that fit the
// 256 MB last-level cache; of larger ones the last 224 MB where a backward is to
// follow, none otherwise.  Forward + backward in us with all rows through the
// caches, all past them, and this: 2.1 GB bf16 370 + 817, 325 + 808, 314 + 787;
// 0.5 GB bf16 100 + 195, 85 + 189, 89 + 178; 1.1 GB fp32 181 + 399, 156 + 399,
// 154 + 373; the backward of a 155 MB tensor 49.4, 51.6, 49.4.
int64_t cached_from(int B, int S, int V, int dtype, bool training) {
    const int64_t rows = int64_t(B) * S, row_bytes = int64_t(V) * dtype_bytes(dtype);
    if (rows * row_bytes <= (int64_t(256) << 20)) return 0;
    return training ? std::max<int64_t>(0, rows - (int64_t(224) << 20) / row_bytes) : rows;
}

template <class A>
seqlogp::Rows rows_of(const A* a, bool training) {
    seqlogp::Rows r{};
    r.logits = a->logits;
    r.sb = a->stride_b;
    r.ss = a->stride_s;
    r.B = a->B;
    r.S = a->S;
    r.V = a->V;
    r.tokens = a->tokens;
    r.tokens64 = a->tokens_are_int64;
    r.mask = a->mask;
    const double k = 1.4426950408889634074 / a->tau;
    r.k = float(k);
    if (double(r.k) >= k) r.k = std::nextafter(r.k, 0.0f);
    r.klo = float(k - double(r.k));
    r.splits = splits_of(a->B, a->S, a->V, a->dtype);
    r.cached = cached_from(a->B, a->S, a->V, a->dtype, training);
    return r;
}

}  // namespace
}  // namespace dot_amd

using namespace dot_amd;

extern "C" size_t dot_seqlogp_forward_workspace_bytes(int B, int S, int V, int dtype) {
    if (B < 0 || S < 0 || V < 1 || !known_dtype(dtype)) return 0;
    return size_t(B) * S * splits_of(B, S, V, dtype) * sizeof(seqlogp::Part);
}

extern "C" int dot_seqlogp_forward(const dot_seqlogp_fwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (int rc = check_shape(a->dtype, a->B, a->S, a->V, a->tau, a->reduction)) return rc;
    if (a->reduction == DOT_REDUCE_NONE && a->ref && !a->ref_per_token)
        return fail(DOT_ERR_INVALID_ARG, "a reference per sequence needs a reduction");
    const int64_t rows = int64_t(a->B) * a->S;
    if (a->B == 0 || (rows == 0 && a->reduction == DOT_REDUCE_NONE)) return ok();
    if (!a->out) return fail(DOT_ERR_INVALID_ARG, "out must be non-NULL");
    if (rows > 0 && (!a->logits || !a->tokens))
        return fail(DOT_ERR_INVALID_ARG, "logits and tokens must be non-NULL");
    if (rows > 0 && (!a->workspace ||
                     a->workspace_bytes < dot_seqlogp_forward_workspace_bytes(a->B, a->S, a->V, a->dtype)))
        return fail(DOT_ERR_WORKSPACE, "workspace smaller than dot_seqlogp_forward_workspace_bytes()");
    const seqlogp::Rows r = rows_of(a, a->row_stats != nullptr);
    auto* parts = static_cast<seqlogp::Part*>(a->workspace);
    seqlogp::JoinArgs j{};
    j.ref = a->ref;
    j.ref64 = a->ref_is_f64;
    j.ref_per_token = a->ref_per_token;
    j.reduction = a->reduction;
    j.out = a->out;
    j.stats = reinterpret_cast<float2*>(a->row_stats);
    j.weight = a->weight;
    dispatch_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        if (rows > 0) {
            ProfScope prof("seqlogp_row_stats", stream);
            hipLaunchKernelGGL((seqlogp::row_stats<T>), dim3(unsigned(rows * r.splits)), dim3(kBlock), 0, stream, r, j,
                               parts);
        }
        // unsplit rows write their positions' values themselves
        if (a->reduction == DOT_REDUCE_NONE && r.splits == 1) return;
        ProfScope prof("seqlogp_join", stream);
        hipLaunchKernelGGL((seqlogp::join<T>), batch_grid(1, a->B), dim3(seqlogp::kJoinBlock), 0, stream, r, parts, j);
    });
    return check_launch("dot_seqlogp_forward");
}

extern "C" int dot_seqlogp_backward(const dot_seqlogp_bwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (int rc = check_shape(a->dtype, a->B, a->S, a->V, a->tau, a->reduction)) return rc;
    const int64_t rows = int64_t(a->B) * a->S;
    if (rows == 0) return ok();
    if (!a->logits || !a->tokens || !a->row_stats || !a->grad_out || !a->grad_logits)
        return fail(DOT_ERR_INVALID_ARG, "logits, tokens, row_stats, grad_out and grad_logits must be non-NULL");
    if (a->reduction == DOT_REDUCE_MEAN && !a->weight)
        return fail(DOT_ERR_INVALID_ARG, "the gradient of a mean needs weight");
    const seqlogp::Rows r = rows_of(a, true);
    seqlogp::GradArgs g{};
    g.inv_tau = float(1.0 / a->tau);
    g.reduction = a->reduction;
    g.stats = reinterpret_cast<const float2*>(a->row_stats);
    g.weight = a->weight;
    g.grad_out = a->grad_out;
    g.grad_out_scalar = a->grad_out_scalar;
    g.grad = a->grad_logits;
    dispatch_dtype(a->dtype, [&](auto t) {
        ProfScope prof("seqlogp_backward", stream);
        hipLaunchKernelGGL((seqlogp::backward<decltype(t)>), dim3(unsigned(rows * r.splits)), dim3(kBlock), 0, stream,
                           r, g);
    });
    return check_launch("dot_seqlogp_backward");
}
