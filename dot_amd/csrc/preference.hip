// C ABI of the preference loss: argument checks and launches.
#include <algorithm>
#include <cmath>

#include "host.hpp"
#include "preference.cuh"

namespace dot_amd {
namespace {

constexpr int kMaxSide = 1 << 22;  // answers of a set

int check_common(int P, int Q, bool has_plan, int type, float beta, float smoothing) {
    if (P < 0 || Q < 0) return fail(DOT_ERR_INVALID_ARG, "P and Q must be >= 0");
    if (P > kMaxSide || Q > kMaxSide) return fail(DOT_ERR_UNSUPPORTED, "P and Q must be at most 2^22");
    if (!has_plan && P != Q) return fail(DOT_ERR_INVALID_ARG, "pairs need P = Q");
    if (type != DOT_PREFER_SIGMOID && type != DOT_PREFER_HINGE && type != DOT_PREFER_SQUARE)
        return fail(DOT_ERR_INVALID_ARG, "loss_type must be a DOT_PREFER_* value");
    if (!(beta > 0.0f) || !std::isfinite(beta)) return fail(DOT_ERR_INVALID_ARG, "beta must be > 0");
    if (!(smoothing >= 0.0f && smoothing < 1.0f)) return fail(DOT_ERR_INVALID_ARG, "smoothing must be in [0, 1)");
    if (smoothing != 0.0f && type != DOT_PREFER_SIGMOID)
        return fail(DOT_ERR_INVALID_ARG, "smoothing needs DOT_PREFER_SIGMOID");
    return DOT_OK;
}

preference::Loss loss_of_args(float beta, int beta_tail, float smoothing) {
    return {beta, smoothing, double(beta) + std::ldexp(double(beta_tail), std::ilogb(beta) - 53)};
}

struct BwdLayout {
    int strip, nstrips, ncols;
    float* colpart;
    float* rowpart;
    size_t bytes;
};

// Strips of up to kMaxStrip rows, shorter while the tiles are fewer than 1024
// (four workgroups per CU; 4096 x 4096: 24.4 us, with 512 of twice the rows 28.1).
BwdLayout bwd_layout(void* ws, int P, int Q) {
    BwdLayout L{};
    L.ncols = std::max(1, (Q + preference::kCols - 1) / preference::kCols);
    L.strip = preference::kMaxStrip;
    while (L.strip > 4 && int64_t((P + L.strip - 1) / L.strip) * L.ncols < 1024) L.strip /= 2;
    L.nstrips = std::max(1, (P + L.strip - 1) / L.strip);
    Carver c(ws);
    L.colpart = c.take<float>(size_t(L.nstrips) * Q);
    L.rowpart = c.take<float>(size_t(L.ncols) * P);
    L.bytes = c.used();
    return L;
}

unsigned blocks_of(int n) { return unsigned((n + kBlock - 1) / kBlock); }

}  // namespace
}  // namespace dot_amd

using namespace dot_amd;

extern "C" int dot_preference_forward(const dot_preference_fwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    // an empty plan has no entries to point at
    const bool has_plan = a->plan || a->P == 0 || a->Q == 0;
    if (int rc = check_common(a->P, a->Q, has_plan, a->loss_type, a->beta, a->smoothing)) return rc;
    if (a->P == 0) return ok();
    if (!a->ratio || !a->loss) return fail(DOT_ERR_INVALID_ARG, "ratio and loss must be non-NULL");
    const preference::Loss l = loss_of_args(a->beta, a->beta_tail, a->smoothing);
    preference::dispatch_type(a->loss_type, a->smoothing, [&](auto type) {
        constexpr int T = decltype(type)::value;
        ProfScope prof(has_plan ? "preference_plan_forward" : "preference_pairs_forward", stream);
        if (!has_plan)
            hipLaunchKernelGGL((preference::pairs_forward<T>), dim3(blocks_of(a->P)), dim3(kBlock), 0, stream,
                               a->ratio, a->P, l, a->loss);
        else if (a->Q % preference::kVec == 0 && aligned16(a->plan))
            hipLaunchKernelGGL((preference::plan_forward<T, true>), dim3(unsigned(a->P)), dim3(kBlock), 0, stream,
                               a->ratio, a->plan, a->P, a->Q, l, a->loss);
        else
            hipLaunchKernelGGL((preference::plan_forward<T, false>), dim3(unsigned(a->P)), dim3(kBlock), 0, stream,
                               a->ratio, a->plan, a->P, a->Q, l, a->loss);
    });
    return check_launch("dot_preference_forward");
}

extern "C" size_t dot_preference_backward_workspace_bytes(int P, int Q, int has_plan) {
    if (P < 0 || Q < 0 || P > kMaxSide || Q > kMaxSide) return 0;
    return has_plan ? bwd_layout(nullptr, P, Q).bytes : 0;
}

extern "C" int dot_preference_backward(const dot_preference_bwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    const bool has_plan = a->plan || a->P == 0 || a->Q == 0;
    if (int rc = check_common(a->P, a->Q, has_plan, a->loss_type, a->beta, a->smoothing)) return rc;
    if (a->P == 0 && a->Q == 0) return ok();
    if (!a->ratio || (a->P > 0 && !a->grad_loss) || !a->grad_ratio)
        return fail(DOT_ERR_INVALID_ARG, "ratio, grad_loss and grad_ratio must be non-NULL");
    const preference::Loss l = loss_of_args(a->beta, a->beta_tail, a->smoothing);
    if (!has_plan) {
        preference::dispatch_type(a->loss_type, a->smoothing, [&](auto type) {
            ProfScope prof("preference_pairs_backward", stream);
            hipLaunchKernelGGL((preference::pairs_backward<decltype(type)::value>), dim3(blocks_of(a->P)),
                               dim3(kBlock), 0, stream, a->ratio, a->P, l, a->grad_loss, a->grad_loss_scalar,
                               a->grad_ratio);
        });
        return check_launch("dot_preference_backward");
    }
    if (a->P == 0 || a->Q == 0) {  // an empty plan: no gradient reaches the ratios
        fill_zero_words(a->grad_ratio, size_t(a->P) + size_t(a->Q), stream);
        return check_launch("dot_preference_backward");
    }
    const BwdLayout L = bwd_layout(a->workspace, a->P, a->Q);
    if (!a->workspace || a->workspace_bytes < L.bytes)
        return fail(DOT_ERR_WORKSPACE, "workspace smaller than dot_preference_backward_workspace_bytes()");
    preference::PlanBwd x{};
    x.ratio = a->ratio;
    x.plan = a->plan;
    x.P = a->P;
    x.Q = a->Q;
    x.l = l;
    x.grad = a->grad_loss;
    x.grad_scalar = a->grad_loss_scalar;
    x.grad_plan = a->grad_plan;
    x.strip = L.strip;
    x.nstrips = L.nstrips;
    x.ncols = L.ncols;
    x.colpart = L.colpart;
    x.rowpart = L.rowpart;
    const dim3 grid(unsigned(L.nstrips) * unsigned(L.ncols));
    preference::dispatch_type(a->loss_type, a->smoothing, [&](auto type) {
        constexpr int T = decltype(type)::value;
        ProfScope prof("preference_plan_backward", stream);
        if (a->Q % preference::kVec == 0 && aligned16(a->plan) && (!a->grad_plan || aligned16(a->grad_plan)))
            hipLaunchKernelGGL((preference::plan_backward<T, true>), grid, dim3(kBlock), 0, stream, x);
        else
            hipLaunchKernelGGL((preference::plan_backward<T, false>), grid, dim3(kBlock), 0, stream, x);
    });
    {
        ProfScope prof("preference_plan_fold", stream);
        const int row_blocks = (a->P + preference::kFoldCols - 1) / preference::kFoldCols;
        const int col_blocks = (a->Q + preference::kFoldCols - 1) / preference::kFoldCols;
        hipLaunchKernelGGL(preference::plan_fold, dim3(unsigned(row_blocks + col_blocks)),
                           dim3(preference::kFoldBlock), 0, stream, x, row_blocks, a->grad_ratio);
    }
    return check_launch("dot_preference_backward");
}
