// C ABI of the top log-probabilities and of beam steps: argument checks and launches.
#include <algorithm>
#include <cmath>

#include "host.hpp"
#include "toplist.cuh"

namespace dot_amd {
namespace {

constexpr int kMaxVocabulary = 1 << 24;  // places of all lists of a batch element fit an int

struct Split {
    int parts, per;
};

// Spans of a row: at most 16 packs a thread.  A row that is its own list (`alone`) and
// fits a span stays whole: 8 x 32768 bf16 in one launch 8.8 us, in 64 spans and a join
// 6.8 + 6.4.  Others are split towards 64 workgroups, down to one pack a thread; further
// splitting makes the joins longer (256 x 131072 bf16 in 4 and 8 spans: 17.5 + 7.0 and
// 18.2 + 8.6 us).
Split split_of(int64_t rows, int V, int dtype, bool alone) {
    const int pn = 16 / dtype_bytes(dtype);
    const int packs = (V + pn - 1) / pn;
    const int least = (packs + kBlock * toplist::kMaxPacks - 1) / (kBlock * toplist::kMaxPacks);
    if (alone && least == 1) return {1, packs};
    const int most = (packs + kBlock - 1) / kBlock;
    const int64_t want = rows > 0 ? (64 + rows - 1) / rows : 1;
    const int parts = int(std::min<int64_t>(std::max<int64_t>(want, least), most));
    const int per = (packs + parts - 1) / parts;
    return {(packs + per - 1) / per, per};
}

int check_rows(int dtype, int64_t rows, int V, int n, double tau) {
    if (!known_dtype(dtype)) return fail(DOT_ERR_INVALID_ARG, "dtype must be DOT_F32, DOT_F16 or DOT_BF16");
    if (V < 1) return fail(DOT_ERR_INVALID_ARG, "V must be >= 1");
    if (V > kMaxVocabulary || rows > (1 << 23))
        return fail(DOT_ERR_UNSUPPORTED, "V must be at most 2^24 and the rows at most 2^23");
    if (n < 1) return fail(DOT_ERR_INVALID_ARG, "at least one entry must be asked for");
    if (n > DOT_TOP_MAX) return fail(DOT_ERR_UNSUPPORTED, "at most DOT_TOP_MAX entries are supported");
    if (!(tau > 0.0) || !std::isfinite(tau)) return fail(DOT_ERR_INVALID_ARG, "tau must be > 0");
    if (tau < 1e-20 || tau > 1e20) return fail(DOT_ERR_UNSUPPORTED, "tau must be in [1e-20, 1e20]");
    return DOT_OK;
}

toplist::Lists carve(void* workspace, size_t& bytes, int64_t rows, const Split& sp, int n) {
    Carver c(workspace);
    toplist::Lists l{};
    l.parts = c.take<toplist::Part>(size_t(rows) * sp.parts);
    l.items = c.take<toplist::Item>(size_t(rows) * sp.parts * n);
    bytes = c.used();
    return l;
}

template <int P, bool DIRECT>
void launch_scan(int dtype, const toplist::Rows& r, const toplist::Lists& l, const toplist::TopOut& o,
                 hipStream_t stream) {
    dispatch_dtype(dtype, [&](auto t) {
        hipLaunchKernelGGL((toplist::scan<decltype(t), P, DIRECT>), batch_grid(unsigned(r.parts), r.rows), dim3(kBlock),
                           0, stream, r, l, o);
    });
}
template <bool DIRECT>
void scan(int dtype, const toplist::Rows& r, const toplist::Lists& l, const toplist::TopOut& o, hipStream_t stream) {
    ProfScope prof("toplist_scan", stream);
    const int packs = (r.per + kBlock - 1) / kBlock;
    if (packs <= 1) launch_scan<1, DIRECT>(dtype, r, l, o, stream);
    else if (packs <= 2) launch_scan<2, DIRECT>(dtype, r, l, o, stream);
    else if (packs <= 4) launch_scan<4, DIRECT>(dtype, r, l, o, stream);
    else if (packs <= 8) launch_scan<8, DIRECT>(dtype, r, l, o, stream);
    else launch_scan<16, DIRECT>(dtype, r, l, o, stream);
}

// Four waves for up to 1024 entries of a join, so that four of a thread stay in its
// registers, sixteen for more.  Eight for 257 to 512 entries: 999 rows of 4 lists of 128
// 13.8 us instead of 12.5, 32 times 8 beams of 4 lists of 16 7.5 instead of 7.
template <bool BEAM>
void join(const toplist::Rows& r, const toplist::Lists& l, const toplist::JoinArgs& a, hipStream_t stream) {
    ProfScope prof("toplist_join", stream);
    const int beams = BEAM ? r.inner : 1, entries = beams * r.parts * r.n;
    const int waves = entries <= 1024 ? 4 : 16;
    auto go = [&](auto lists, auto each) {
        constexpr int R = decltype(lists)::value, EACH = decltype(each)::value;
        hipLaunchKernelGGL((toplist::join<R, BEAM, EACH>), batch_grid(1, r.rows / beams),
                           dim3(unsigned(waves) * kWave), toplist::join_shared(R, waves, beams, entries), stream, r, l, a);
    };
    using std::integral_constant;
    auto with = [&](auto lists) {
        if (entries <= 4 * waves * kWave) go(lists, integral_constant<int, 4>{});
        else go(lists, integral_constant<int, 0>{});
    };
    if (r.n <= 64) with(integral_constant<int, 1>{});
    else if (r.n <= 128) with(integral_constant<int, 2>{});
    else with(integral_constant<int, 4>{});
}

void set_tau(toplist::Rows& r, double tau) {
    r.inv_tau = 1.0f / float(tau);
    r.k = float(1.4426950408889634074 * double(r.inv_tau));
}

}  // namespace
}  // namespace dot_amd

using namespace dot_amd;

extern "C" size_t dot_top_logp_workspace_bytes(int B, int S, int V, int dtype, int k) {
    if (B < 0 || S < 0 || V < 1 || V > kMaxVocabulary || k < 1 || k > DOT_TOP_MAX || !known_dtype(dtype)) return 0;
    const int64_t rows = int64_t(B) * S;
    const Split sp = split_of(rows, V, dtype, true);
    if (sp.parts == 1) return 0;
    size_t bytes = 0;
    carve(nullptr, bytes, rows, sp, k);
    return bytes;
}

extern "C" int dot_top_logp(const dot_top_logp_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (a->B < 0 || a->S < 0) return fail(DOT_ERR_INVALID_ARG, "B and S must be >= 0");
    const int64_t rows = int64_t(a->B) * a->S;
    if (int rc = check_rows(a->dtype, rows, a->V, a->k, a->tau)) return rc;
    if (a->k > a->V) return fail(DOT_ERR_INVALID_ARG, "k must be at most V");
    if (rows == 0) return ok();
    if (!a->logits || !a->logp || !a->tokens)
        return fail(DOT_ERR_INVALID_ARG, "logits, logp and tokens must be non-NULL");
    const Split sp = split_of(rows, a->V, a->dtype, true);
    toplist::Rows r{};
    r.logits = a->logits;
    r.so = a->stride_b;
    r.si = a->stride_s;
    r.inner = a->S;
    r.rows = int(rows);
    r.V = a->V;
    r.mask = a->mask;
    set_tau(r, a->tau);
    r.n = a->k;
    r.parts = sp.parts;
    r.per = sp.per;
    if (sp.parts == 1) {
        scan<true>(a->dtype, r, toplist::Lists{}, toplist::TopOut{a->logp, a->tokens}, stream);
        return check_launch("dot_top_logp");
    }
    size_t need = 0;
    const toplist::Lists l = carve(a->workspace, need, rows, sp, a->k);
    if (!a->workspace || a->workspace_bytes < need)
        return fail(DOT_ERR_WORKSPACE, "workspace smaller than dot_top_logp_workspace_bytes()");
    scan<false>(a->dtype, r, l, toplist::TopOut{}, stream);
    toplist::JoinArgs j{};
    j.scores = a->logp;
    j.tokens = a->tokens;
    join<false>(r, l, j, stream);
    return check_launch("dot_top_logp");
}

extern "C" size_t dot_beam_step_workspace_bytes(int B, int W, int V, int dtype, int n) {
    if (B < 0 || W < 1 || W > DOT_BEAM_MAX || V < 1 || V > kMaxVocabulary || n < 1 || n > DOT_TOP_MAX ||
        !known_dtype(dtype))
        return 0;
    const int64_t rows = int64_t(B) * W;
    size_t bytes = 0;
    carve(nullptr, bytes, rows, split_of(rows, V, dtype, false), n);
    return bytes;
}

extern "C" int dot_beam_step(const dot_beam_step_args* a, dot_stream_t stream_) {
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (a->B < 0 || a->W < 1) return fail(DOT_ERR_INVALID_ARG, "B must be >= 0 and W >= 1");
    if (a->W > DOT_BEAM_MAX) return fail(DOT_ERR_UNSUPPORTED, "at most DOT_BEAM_MAX beams are supported");
    const int64_t rows = int64_t(a->B) * a->W;
    if (int rc = check_rows(a->dtype, rows, a->V, a->n, a->tau)) return rc;
    if (int64_t(a->n) > int64_t(a->W) * a->V) return fail(DOT_ERR_INVALID_ARG, "n must be at most W * V");
    if (a->finished && (a->eos < 0 || a->eos >= a->V))
        return fail(DOT_ERR_INVALID_ARG, "finished beams need an eos in [0, V)");
    if (rows == 0) return ok();
    if (!a->logits || !a->scores || !a->out_scores || !a->out_beams || !a->out_tokens)
        return fail(DOT_ERR_INVALID_ARG, "logits, scores, out_scores, out_beams and out_tokens must be non-NULL");
    const Split sp = split_of(rows, a->V, a->dtype, false);
    toplist::Rows r{};
    r.logits = a->logits;
    r.so = a->stride_b;
    r.si = a->stride_w;
    r.inner = a->W;
    r.rows = int(rows);
    r.V = a->V;
    r.scores = a->scores;
    r.finished = a->finished;
    set_tau(r, a->tau);
    r.n = a->n;
    r.parts = sp.parts;
    r.per = sp.per;
    size_t need = 0;
    const toplist::Lists l = carve(a->workspace, need, rows, sp, a->n);
    if (!a->workspace || a->workspace_bytes < need)
        return fail(DOT_ERR_WORKSPACE, "workspace smaller than dot_beam_step_workspace_bytes()");
    scan<false>(a->dtype, r, l, toplist::TopOut{}, stream);
    toplist::JoinArgs j{};
    j.eos = a->eos;
    j.scores = a->out_scores;
    j.beams = a->out_beams;
    j.tokens = a->out_tokens;
    j.finished = a->out_finished;
    join<true>(r, l, j, stream);
    return check_launch("dot_beam_step");
}
