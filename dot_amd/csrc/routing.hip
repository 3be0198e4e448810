// C ABI of the routing operators: argument checks and launches.
#include <algorithm>

#include "host.hpp"
#include "routing.cuh"

namespace dot_amd {
namespace {

// Lanes of a row and vectors of a lane for E experts.
struct Lanes {
    int g, r;
};
template <bool PAIRS>
Lanes lanes_of(int E) {
    Lanes l{};
    routing::dispatch_shape<true, PAIRS>(E, [&](auto s) { l = {decltype(s)::G, decltype(s)::R}; });
    return l;
}

struct FwdLayout {
    float* psum;
    int32_t* pcount;
    int32_t* ptokens;
    double* dots;
    uint32_t* done;
    Lanes lanes;
    int threads, rows, nchunks, colblocks;
    size_t bytes;
};

// About 512 workgroups, two per CU.
FwdLayout fwd_layout(void* ws, int B, int N, int E, bool select) {
    Carver c(ws);
    FwdLayout L{};
    const Lanes lanes = select ? lanes_of<true>(E) : lanes_of<false>(E);
    L.lanes = lanes;
    L.threads = routing::fwd_block(lanes.r);
    L.rows = L.threads / lanes.g;
    L.nchunks = routing::chunks_of(B, N, L.rows, 512);
    L.colblocks = (E + routing::kFinishCols - 1) / routing::kFinishCols;
    if (L.nchunks == 1) return L;
    const size_t parts = size_t(B) * L.nchunks;
    L.psum = c.take<float>(parts * E);
    L.pcount = c.take<int32_t>(parts * E);
    L.ptokens = c.take<int32_t>(parts);
    L.dots = c.take<double>(size_t(B) * L.colblocks);
    L.done = c.take<uint32_t>(B);
    L.bytes = c.used();
    return L;
}

int check_shape(int dtype, int B, int N, int E, int k, int scoring) {
    if (!known_dtype(dtype)) return fail(DOT_ERR_INVALID_ARG, "dtype must be DOT_F32, DOT_F16 or DOT_BF16");
    if (B < 0 || N < 0) return fail(DOT_ERR_INVALID_ARG, "B and N must be >= 0");
    if (N > (1 << 30)) return fail(DOT_ERR_UNSUPPORTED, "N exceeds 2^30");
    if (E < 1) return fail(DOT_ERR_INVALID_ARG, "E must be >= 1");
    if (E > DOT_ROUTING_MAX_EXPERTS) return fail(DOT_ERR_UNSUPPORTED, "E exceeds DOT_ROUTING_MAX_EXPERTS");
    if (k < 1) return fail(DOT_ERR_INVALID_ARG, "k must be >= 1");
    if (k > DOT_ROUTING_MAX_K) return fail(DOT_ERR_UNSUPPORTED, "k exceeds DOT_ROUTING_MAX_K");
    if (scoring != DOT_SCORING_SOFTMAX && scoring != DOT_SCORING_SIGMOID && scoring != DOT_SCORING_PLAN)
        return fail(DOT_ERR_INVALID_ARG, "scoring must be a DOT_SCORING_* value");
    return DOT_OK;
}

// Whether rows can be read 16 bytes at a time.
bool rows_aligned(const void* p, int64_t sb, int64_t sn, int E, int dtype) {
    const int64_t bytes = dtype_bytes(dtype);
    return E % routing::kV == 0 && aligned16(p) && (sb * bytes) % 16 == 0 && (sn * bytes) % 16 == 0;
}

template <bool PAIRS, class F>
void dispatch(int dtype, int E, bool vec, F&& f) {
    dispatch_dtype(dtype, [&](auto t) {
        if (vec) routing::dispatch_shape<true, PAIRS>(E, [&](auto s) { f(t, s); });
        else routing::dispatch_shape<false, PAIRS>(E, [&](auto s) { f(t, s); });
    });
}

}  // namespace
}  // namespace dot_amd

using namespace dot_amd;

extern "C" size_t dot_routing_forward_workspace_bytes(int B, int N, int E) {
    if (B < 0 || N < 0 || E < 1) return 0;
    return std::max(fwd_layout(nullptr, B, N, E, true).bytes, fwd_layout(nullptr, B, N, E, false).bytes);
}

extern "C" int dot_routing_forward(const dot_routing_fwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (int rc = check_shape(a->dtype, a->B, a->N, a->E, a->k, a->scoring)) return rc;
    const bool select = a->given == nullptr;
    if (select && a->k > a->E) return fail(DOT_ERR_INVALID_ARG, "k must be at most E");
    if (a->B == 0) return ok();
    if (!a->counts || !a->loss) return fail(DOT_ERR_INVALID_ARG, "counts and loss must be non-NULL");
    if (a->N > 0 && (!a->scores || (select && (!a->weights || !a->experts))))
        return fail(DOT_ERR_INVALID_ARG, "scores, weights and experts must be non-NULL");
    const FwdLayout L = fwd_layout(a->workspace, a->B, a->N, a->E, select);
    if (L.bytes > 0 && (!a->workspace || a->workspace_bytes < L.bytes))
        return fail(DOT_ERR_WORKSPACE, "workspace smaller than dot_routing_forward_workspace_bytes()");
    routing::FwdArgs x{};
    x.scores = a->scores;
    x.sb = a->stride_b;
    x.sn = a->stride_n;
    x.B = a->B;
    x.N = a->N;
    x.E = a->E;
    x.k = a->k;
    x.scoring = a->scoring;
    x.normalize = a->normalize;
    x.bias = a->bias;
    x.mask = a->mask;
    x.given = a->given;
    x.given64 = a->given_is_int64;
    x.weights = a->weights;
    x.experts = a->experts;
    x.nchunks = L.nchunks;
    x.chunk_rows = (a->N + L.nchunks - 1) / L.nchunks;
    x.psum = L.psum;
    x.pcount = L.pcount;
    x.ptokens = L.ptokens;
    x.done = L.done;
    x.counts = a->counts;
    x.tokens = a->tokens;
    x.loss = a->loss;
    const dim3 grid = batch_grid(unsigned(L.nchunks), a->B);
    const size_t lds = routing::fwd_lds_bytes(a->E, a->k, L.lanes.g, L.lanes.r, L.rows, select);
    const bool vec = rows_aligned(a->scores, a->stride_b, a->stride_n, a->E, a->dtype);
    {
        ProfScope prof("routing_forward", stream);
        if (select)
            dispatch<true>(a->dtype, a->E, vec, [&](auto t, auto s) {
                hipLaunchKernelGGL((routing::forward<decltype(t), decltype(s), true>), grid, dim3(L.threads), lds,
                                   stream, x);
            });
        else
            dispatch<false>(a->dtype, a->E, vec, [&](auto t, auto s) {
                hipLaunchKernelGGL((routing::forward<decltype(t), decltype(s), false>), grid, dim3(L.threads), lds,
                                   stream, x);
            });
    }
    if (L.nchunks > 1) {
        ProfScope prof("routing_finish", stream);
        const routing::FinishArgs f{a->B, a->E, a->k, L.nchunks, L.psum, L.pcount, L.ptokens, L.dots, L.done,
                                    a->counts, a->tokens, a->loss};
        hipLaunchKernelGGL(routing::finish, batch_grid(unsigned(L.colblocks), a->B), dim3(routing::kFinishBlock), 0,
                           stream, f);
    }
    return check_launch("dot_routing_forward");
}

extern "C" int dot_routing_backward(const dot_routing_bwd_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (int rc = check_shape(a->dtype, a->B, a->N, a->E, a->k, a->scoring)) return rc;
    if (a->B == 0 || a->N == 0) return ok();
    if (!a->scores || !a->grad_scores) return fail(DOT_ERR_INVALID_ARG, "scores and grad_scores must be non-NULL");
    if (a->grad_loss && (!a->counts || (a->mask && !a->tokens)))
        return fail(DOT_ERR_INVALID_ARG, "grad_loss needs counts, and tokens where there is a mask");
    if (a->grad_weights && (!a->weights || !a->experts))
        return fail(DOT_ERR_INVALID_ARG, "grad_weights needs weights and experts");
    routing::BwdArgs x{};
    x.scores = a->scores;
    x.sb = a->stride_b;
    x.sn = a->stride_n;
    x.B = a->B;
    x.N = a->N;
    x.E = a->E;
    x.k = a->k;
    x.scoring = a->scoring;
    x.normalize = a->normalize;
    x.mask = a->mask;
    x.counts = a->counts;
    x.tokens = a->tokens;
    x.grad_loss = a->grad_loss;
    x.grad_loss_scalar = a->grad_loss_scalar;
    x.weights = a->weights;
    x.experts = a->experts;
    x.grad_weights = a->grad_weights;
    x.grad_scores = a->grad_scores;
    // about 1024 workgroups: 131072 x 128 bf16 in 17.2 us, 18.2 with 512, a third more with 4096
    x.nchunks = routing::chunks_of(a->B, a->N, kBlock / lanes_of<false>(a->E).g, 1024);
    x.chunk_rows = (a->N + x.nchunks - 1) / x.nchunks;
    const dim3 grid = batch_grid(unsigned(x.nchunks), a->B);
    const bool vec = rows_aligned(a->scores, a->stride_b, a->stride_n, a->E, a->dtype) && aligned16(a->grad_scores);
    dispatch<false>(a->dtype, a->E, vec, [&](auto t, auto s) {
        using S = decltype(s);
        ProfScope prof("routing_backward", stream);
        const size_t lds = routing::bwd_lds_bytes(kWave * S::EL, a->grad_weights != nullptr);
        if (a->grad_weights)
            hipLaunchKernelGGL((routing::backward<decltype(t), S, true>), grid, dim3(kBlock), lds, stream, x);
        else
            hipLaunchKernelGGL((routing::backward<decltype(t), S, false>), grid, dim3(kBlock), lds, stream, x);
    });
    return check_launch("dot_routing_backward");
}
