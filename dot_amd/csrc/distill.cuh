// Divergence of rows of logits from a teacher's few log-probabilities, and the
// gradient of the logits.
//
// With a position's K tokens i_k of log-probability t_k, P_k = exp t_k, z = x / tau,
// Q = softmax(z) and Q_r the sum of Q over the other tokens:
//   forward  L = sum_k P_k (t_k - log Q_k) + P_r (log P_r - log Q_r)
//   reverse  L = sum_k Q_k (log Q_k - t_k) + Q_r (log Q_r - log P_r)
// P_r = 1 - sum_k P_k, 0 where that is negative; with DOT_REST_NONE P is made to sum to
// 1 and P_r = 0.  The gradient of a named token is a value of its own, that of any other
// token its share w_j = Q_j / Q_r of one value for the row; with M = sum_k P_k + P_r, which
// is 1 but where P_r is 0 (log-probabilities kept in few bits):
//   tau dL/dx_j = M Q_j - P_j,                   w_j (M Q_r - P_r)
//   tau dL/dx_j = Q_j (log Q_j - t_j - L),       w_j Q_r (log Q_r - log P_r - L)
// So the row is read once for s = sum 2^((x - m) k) of the others alone, m the largest
// of the first of them, or of all where a term next to that one would be too large.
// The named tokens are left out of it by a bit for each token of the span in LDS
// (a byte for a pack: one read of LDS per 16 bytes of logits) and added in 64 bits:
// next to a likely named token the others keep their digits, and differences of
// probabilities near 1 theirs.  An m of the others' own keeps their shares from
// vanishing where a named token is far likelier.  The backward writes
// w_j = 2^((x_j - m) k) / s times the row's value, then the named tokens'.
#pragma once

#include "seqlogp.cuh"

namespace dot_amd {
namespace distill {

using seqlogp::Rows;
using seqlogp::Span;

constexpr int kMaxSpan = 1 << 18;  // tokens whose bits a workgroup holds (32 KB)
constexpr int kPerLane = DOT_TOP_MAX / kWave;

struct Teacher {
    const void* tokens;  // [B,S,K]
    int tokens64;
    const float* logp;   // [B,S,K]
    int K;
};

struct Value {
    double v;
    int live, pad;
};

// What a split leaves of a row: a sum, and whether two entries name the same of its tokens.
struct Part {
    double s;
    float m;
    int twice;
};

struct Out {
    int direction, rest, reduction;
    float* out;       // [B,S] with DOT_REDUCE_NONE
    Value* values;    // [B,S] otherwise
    float2* stats;    // [B,S]: the others' m (NaN: left out) and the row's value / s
    int32_t* at;      // [B,S,K]: the tokens that have a gradient of their own, or -1
    float* own;       // [B,S,K]: that gradient
};

// The row of a position, which Rows has no token for.
__device__ __forceinline__ bool masked(const Rows& r, int64_t at) { return r.mask && !r.mask[at]; }

// The token of an entry, or -1 where it names none.
__device__ __forceinline__ int named(const Rows& r, const Teacher& t, int64_t entry) {
    const int64_t v = int_at(t.tokens, t.tokens64, entry);
    return v >= 0 && v < r.V && !(t.logp[entry] == -__builtin_inff()) ? int(v) : -1;
}

// s = sum 2^((x - m) k) of some logits, m one of them near the largest (-inf: of none but
// -inf).  k + klo of fp32 logits, for all other types (klo = 0) the same one float here
// and everywhere else: a temperature that is off by up to 6e-8 of itself moves a loss by
// that share of sum (Q - P) x / tau, and a gradient by less than it is rounded to.
struct Sum {
    float m = -__builtin_inff();
    double s = 0.0;
    __device__ __forceinline__ void join(const Sum& b, double kn) {
        if (b.m == -__builtin_inff() && b.s == 0.0) return;
        const float to = fmaxf(m, b.m);
        const double mine = s == 0.0 ? 0.0 : s * short_exp((double(m) - double(to)) * kn);
        s = mine + b.s * short_exp((double(b.m) - double(to)) * kn);
        m = to;
    }
};
// 1 / tau
__device__ __forceinline__ double inverse_tau(const Rows& r) {
    return (double(r.k) + double(r.klo)) * 0.693147180559945309417;
}
// d log2(e) / tau of a difference
template <class T>
__device__ __forceinline__ float scaled(const Rows& r, float d) {
    if constexpr (std::is_same_v<T, float>) return seqlogp::scaled(r, d);
    else return d * r.k;
}

__device__ __forceinline__ void leave_out(const Out& o, int64_t at) {
    if (o.reduction == DOT_REDUCE_NONE) o.out[at] = 0.0f;
    else o.values[at] = Value{0.0, 0, 0};
    if (o.stats) o.stats[at] = make_float2(__builtin_nanf(""), 0.0f);
}

// A position's entries as one wave holds them, entry i * 64 + lane in [i]: the token, -1
// where the entry names none or one that an earlier entry names, its logit and its t.
struct Entries {
    int tok[kPerLane];
    float x[kPerLane], t[kPerLane];
};

// The value of a position and what its gradient is made of, by one wave, from its
// entries and the statistics of its other tokens.
__device__ __forceinline__ void finish(const Rows& r, int K, const Out& o, int64_t at, const Entries& in,
                                       const Sum& others) {
    const int lane = int(threadIdx.x) % kWave;
    const double kn = inverse_tau(r);
    const int (&tok)[kPerLane] = in.tok;
    const float (&x)[kPerLane] = in.x;
    float top = others.m, most = -__builtin_inff();
    double tl[kPerLane], p[kPerLane];
    double mass = 0.0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        tl[i] = p[i] = 0.0;
        if (tok[i] < 0) continue;
        tl[i] = double(in.t[i]);
        most = fmaxf(most, in.t[i]);
        top = fmaxf(top, x[i]);
    }
    const bool bucket = o.rest == DOT_REST_BUCKET, reverse = o.direction == DOT_DISTILL_REVERSE;
    top = wave_max(top);
    if (top == -__builtin_inff()) top = 0.0f;
    // P made to sum to 1 keeps its digits however small it is
    const double less = bucket ? 0.0 : double(wave_max(most));
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
        if (tok[i] >= 0) mass += p[i] = short_exp(tl[i] - less);
    mass = wave_sum64(mass);
    double z = 0.0, q[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        q[i] = tok[i] >= 0 ? short_exp((double(x[i]) - double(top)) * kn) : 0.0;
        z += q[i];
    }
    const bool none = others.s == 0.0;  // no other token is possible
    const double lr = none ? -__builtin_inf() : (double(others.m) - double(top)) * kn + short_log(others.s);
    const double er = short_exp(lr);
    z = wave_sum64(z) + er;
    const double lz = short_log(z), log_qr = lr - lz, iz = 1.0 / z, qr = er * iz;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) q[i] *= iz;
    double pr = 0.0;
    if (bucket) {
        pr = 1.0 - mass;
        if (pr < 0.0) pr = 0.0;
    }
    if (!bucket) {
        const double lm = short_log(mass) + less;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            p[i] /= mass;
            tl[i] -= lm;
        }
    }
    double value = 0.0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        if (tok[i] < 0) continue;
        const double lq = (double(x[i]) - double(top)) * kn - lz;
        if (!reverse) value += p[i] == 0.0 ? 0.0 : p[i] * (tl[i] - lq);
        else value += lq == -__builtin_inf() ? 0.0 : q[i] * (lq - tl[i]);
    }
    value = wave_sum64(value);
    const double log_pr = short_log(reverse ? fmax(pr, 0x1p-24) : pr);
    double other;        // gradient of the others together
    double total = 1.0;  // sum of the P that the forward loss has: the entries' alone where they leave no rest
    if (!reverse) {
        // where no other token is possible, what rounding leaves of P_r is nothing
        const bool left = bucket && !(pr == 0.0 || (none && pr <= DOT_REST_ROUNDING));
        if (left) value += pr * (log_pr - log_qr);
        else if (bucket) total = mass;
        other = total * qr - (left ? pr : 0.0);
    } else {
        if (!none) value += qr * (log_qr - log_pr);
        other = none ? 0.0 : qr * (log_qr - log_pr - value);
    }
    if (lane == 0) {
        if (o.reduction == DOT_REDUCE_NONE) o.out[at] = float(value);
        else o.values[at] = Value{value, 1, 0};
        if (o.stats) o.stats[at] = make_float2(none ? 0.0f : others.m, none ? 0.0f : float(other / others.s));
    }
    if (!o.stats) return;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int e = i * kWave + lane;
        if (e >= K) break;
        float g = 0.0f;
        if (tok[i] >= 0) {
            const double lq = (double(x[i]) - double(top)) * kn - lz;
            if (!reverse) g = float(total * q[i] - p[i]);
            else g = lq == -__builtin_inf() ? 0.0f : float(q[i] * (lq - tl[i] - value));
        }
        o.at[at * K + e] = tok[i];
        o.own[at * K + e] = g;
    }
}

// Leaves a token that several entries name to the first of them.  `list` holds the
// entries' tokens, DOT_TOP_MAX of them.
__device__ __forceinline__ void only_first(int K, const int* list, Entries& in) {
    const int lane = int(threadIdx.x) % kWave;
    for (int j = 0; j < K; j += 4) {
        const int4 v = *reinterpret_cast<const int4*>(list + j);
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            if (i * kWave >= K) break;
            const int e = i * kWave + lane;
            if ((in.tok[i] == v.x && j < e) || (in.tok[i] == v.y && j + 1 < e) || (in.tok[i] == v.z && j + 2 < e) ||
                (in.tok[i] == v.w && j + 3 < e))
                in.tok[i] = -1;
        }
    }
}

// The other tokens' statistics of every row, one for each split; an unsplit row is
// finished at once.  The entries, a thread each, and the row's first packs are on their
// way while the bits are made.
//
// Bound by HBM in long rows (about 4500 of 131072 bf16: 218 us, 5.4 TB/s), in shorter ones by
// what a workgroup does before and behind its logits as well (as
// many of 32768, 64 entries: 67 us, 4.4 TB/s; half of 774 of 50021 fp32, 100 entries:
// 22 us), and by latency in few (74 of 1000 fp32: 6.2 us).  seqlogp::kUnroll
// packs at once: 2 and 8 of them, or a bound on registers for more workgroups, were slower.
template <class T>
__global__ __launch_bounds__(kBlock) void row_stats(Rows r, Teacher t, Out o, Part* parts) {
    extern __shared__ __attribute__((aligned(16))) uint32_t words[];
    __shared__ float sm[kWavesPerBlock];
    __shared__ double ss[kWavesPerBlock];
    __shared__ int list[DOT_TOP_MAX] __attribute__((aligned(16)));
    __shared__ float list_x[DOT_TOP_MAX], list_t[DOT_TOP_MAX];
    __shared__ int twice;
    static_assert(DOT_TOP_MAX == kBlock, "a thread an entry");
    constexpr int PN = Pack<T>::N, U = seqlogp::kUnroll;
    const int64_t at = blockIdx.x / unsigned(r.splits);
    const int part = int(blockIdx.x % unsigned(r.splits));
    const bool whole = r.splits == 1;
    if (masked(r, at)) {
        if (whole && threadIdx.x == 0) leave_out(o, at);
        return;
    }
    const int e = int(threadIdx.x);
    const int64_t entry = at * t.K + min(e, t.K - 1);
    const int64_t named = int_at(t.tokens, t.tokens64, entry);
    const float tl = t.logp[entry];
    const T* row = seqlogp::row_of<T>(r, at);
    const Span sp = seqlogp::span_of(row, r.V, part, r.splits);
    const T* body = row + sp.head;
    const bool stream = at < r.cached;
    Pack<T> next[U];
    if (sp.p0 + U * kBlock <= sp.p1) {
        const T* from = body + int64_t(sp.p0 + e) * PN;
#pragma unroll
        for (int u = 0; u < U; ++u)
            next[u] = stream ? load_pack_stream(from + u * kBlock * PN) : load_pack(from + u * kBlock * PN);
    }
    const int v0 = part == 0 ? 0 : sp.head + sp.p0 * PN;
    const int v1 = part == r.splits - 1 ? r.V : sp.head + sp.p1 * PN;
    const int first = sp.head + sp.p0 * PN - 32;  // token of bit 0
    const int nwords = (v1 - first + 31) / 32;
    for (int i = threadIdx.x; i < nwords; i += kBlock) words[i] = 0;
    if (threadIdx.x == 0) twice = 0;
    const int tok = e < t.K && named >= 0 && named < r.V && !(tl == -__builtin_inff()) ? int(named) : -1;
    list[e] = tok;
    // left out without an entry; the barrier is that of the zeros as well
    if (!__syncthreads_or(tok >= 0)) {
        if (whole && threadIdx.x == 0) leave_out(o, at);
        return;
    }
    float x = -__builtin_inff();
    if (tok >= 0) {
        if (whole) x = to_float(row[tok]);
        if (tok >= v0 && tok < v1) {
            const uint32_t bit = 1u << ((tok - first) % 32);
            if (atomicOr(&words[(tok - first) / 32], bit) & bit) twice = 1;
        }
    }
    __syncthreads();  // the bits are whole
    auto bit = [&](int v) { return words[(v - first) / 32] >> ((v - first) % 32) & 1u; };
    // A pack's logits, those of named tokens as -inf.
    auto values = [&](const Pack<T>& x, int p, float* f) {
#pragma unroll
        for (int i = 0; i < PN; ++i) f[i] = to_float(x.v[i]);
        uint32_t b = reinterpret_cast<const uint8_t*>(words)[(32 + (p - sp.p0) * PN) / 8];
        if (PN == 4) b = (p - sp.p0) % 2 ? b >> 4 : b & 15u;
        if (b) {
#pragma unroll
            for (int i = 0; i < PN; ++i)
                if (b >> i & 1u) f[i] = -__builtin_inff();
        }
    };
    // The unaligned logits before and behind, one a thread; then all a thread's logits,
    // PN at a time, the first group from `next`.
    const float none = -__builtin_inff();
    const int tail = sp.tail + e;
    const float before = part == 0 && e < sp.head && !bit(e) ? to_float(row[e]) : none;
    const float behind = part == r.splits - 1 && tail < r.V && !bit(tail) ? to_float(row[tail]) : none;
    const bool groups = sp.p0 + U * kBlock <= sp.p1;
    auto each = [&](auto use, auto past) {
        constexpr bool PAST = decltype(past)::value;
        int q = sp.p0;
        for (; q + U * kBlock <= sp.p1; q += U * kBlock) {
            const bool more = q + 2 * U * kBlock <= sp.p1;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[PN];
                values(next[u], q + u * kBlock + e, f);
                if (more) next[u] = seqlogp::row_pack<PAST>(body + int64_t(q + (U + u) * kBlock + e) * PN);
                use(f);
            }
        }
        for (int p = q + e; p < sp.p1; p += kBlock) {
            float f[PN];
            values(seqlogp::row_pack<PAST>(body + int64_t(p) * PN), p, f);
            use(f);
        }
    };
    // The terms are relative to the largest logit of the wave's first packs: none of them
    // is larger than 1 by much, or the sum is formed again.
    float m = fmaxf(before, behind);
    if (groups) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[PN];
            values(next[u], sp.p0 + u * kBlock + e, f);
#pragma unroll
            for (int i = 0; i < PN; ++i) m = fmaxf(m, f[i]);
        }
    } else if (sp.p0 + e < sp.p1) {
        float f[PN];
        values(load_pack(body + int64_t(sp.p0 + e) * PN), sp.p0 + e, f);
#pragma unroll
        for (int i = 0; i < PN; ++i) m = fmaxf(m, f[i]);
    }
    m = wave_max(m);
    const float mk = m * r.k;
    Sum a;
    a.m = m;
    // x k - m k in one rounding where m k has digits behind the point
    const bool near = fabsf(mk) < 65536.0f;
    if (near) {
        auto term = [&](float x) {
            float y = fmaf(x, r.k, -mk);
            if constexpr (std::is_same_v<T, float>) y = fmaf(x, r.klo, y);
            return __builtin_amdgcn_exp2f(y);
        };
        a.s = double(term(before)) + double(term(behind));
        auto sum = [&](const float* f) {
            float y[PN];
#pragma unroll
            for (int i = 0; i < PN; ++i) y[i] = term(f[i]);
            a.s += double(pairwise<PN>(y));
        };
        if (stream) each(sum, std::true_type{});
        else each(sum, std::false_type{});
        a.s = wave_sum64(a.s);
        // what rounding m k left
        a.s *= short_exp((double(mk) - double(m) * (double(r.k) + double(r.klo))) * 0.693147180559945309417);
    }
    if (!near || a.s > 0x1p60) {
        // the largest logit of all, then the terms; from the caches
        if (groups) {
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load_pack(body + int64_t(sp.p0 + u * kBlock + e) * PN);
        }
        m = fmaxf(before, behind);
        each([&](const float* f) {
            for (int i = 0; i < PN; ++i) m = fmaxf(m, f[i]);
        }, std::false_type{});
        m = a.m = wave_max(m);
        const float base = m == none ? 0.0f : m;
        auto term = [&](float x) { return double(__builtin_amdgcn_exp2f(scaled<T>(r, x - base))); };
        a.s = term(before) + term(behind);
        if (groups) {
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load_pack(body + int64_t(sp.p0 + u * kBlock + e) * PN);
        }
        each([&](const float* f) {
            for (int i = 0; i < PN; ++i) a.s += term(f[i]);
        }, std::false_type{});
        a.s = wave_sum64(a.s);
    }
    list_x[e] = x;
    list_t[e] = tl;
    if (threadIdx.x % kWave == 0) {
        sm[threadIdx.x / kWave] = a.m;
        ss[threadIdx.x / kWave] = a.s;
    }
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    // the waves' sums, a lane of a quad each
    Sum all{fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ss[e % 4]};
    if (all.s != 0.0) all.s *= short_exp((double(sm[e % 4]) - double(all.m)) * inverse_tau(r));
    all.s += dpp_move<kDppQuadXor1>(all.s);
    all.s += dpp_move<kDppQuadXor2>(all.s);
    if (!whole) {
        if (threadIdx.x == 0) parts[blockIdx.x] = Part{all.s, all.m, twice};
        return;
    }
    Entries in;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        in.tok[i] = list[i * kWave + e];
        in.x[i] = list_x[i * kWave + e];
        in.t[i] = list_t[i * kWave + e];
    }
    if (twice) only_first(t.K, list, in);
    finish(r, t.K, o, at, in, all);
}

// Joins the parts of split rows, one wave a row.  Bound by latency: 4 rows of 131072 bf16
// in 32 parts, 64 entries 4.3 us, 256 entries 8.
template <class T>
__global__ __launch_bounds__(kBlock) void finish_rows(Rows r, Teacher t, Out o, const Part* parts) {
    __shared__ int lists[kWavesPerBlock][DOT_TOP_MAX] __attribute__((aligned(16)));
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    const int64_t at = int64_t(blockIdx.x) * kWavesPerBlock + wave;
    if (at >= int64_t(r.B) * r.S) return;
    Entries in;
    bool any = false;
    if (!masked(r, at)) {
        const T* row = seqlogp::row_of<T>(r, at);
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int e = i * kWave + lane;
            in.tok[i] = e < t.K ? named(r, t, at * t.K + e) : -1;
            in.x[i] = in.tok[i] >= 0 ? to_float(row[in.tok[i]]) : 0.0f;
            in.t[i] = in.tok[i] >= 0 ? t.logp[at * t.K + e] : 0.0f;
            lists[wave][e] = in.tok[i];
            any |= in.tok[i] >= 0;
        }
    }
    if (__ballot(any) == 0) {
        if (lane == 0) leave_out(o, at);
        return;
    }
    Sum mine;
    bool twice = false;
    for (int i = lane; i < r.splits; i += kWave) {
        const Part p = parts[at * r.splits + i];
        mine.join(Sum{p.m, p.s}, inverse_tau(r));
        twice |= p.twice != 0;
    }
    Sum all{wave_max(mine.m), 0.0};
    if (mine.s != 0.0) mine.s *= short_exp((double(mine.m) - double(all.m)) * inverse_tau(r));
    all.s = wave_sum64(mine.s);
    wave_lds_fence();
    if (__ballot(twice)) only_first(t.K, lists[wave], in);
    finish(r, t.K, o, at, in, all);
}

// The positions' values of each sequence, added up.
__global__ __launch_bounds__(seqlogp::kJoinBlock) void sum(int B, int S, int reduction, const Value* values,
                                                          float* out, float* weight) {
    constexpr int waves = seqlogp::kJoinBlock / kWave;
    __shared__ double wsum[waves];
    __shared__ int wcount[waves];
    const int b = batch_of_block();
    if (b >= B) return;
    double total = 0.0;
    int count = 0;
    for (int s = threadIdx.x; s < S; s += seqlogp::kJoinBlock) {
        const Value v = values[int64_t(b) * S + s];
        total += v.v;
        count += v.live;
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        total += __shfl_xor(total, d);
        count += __shfl_xor(count, d);
    }
    if (threadIdx.x % kWave == 0) {
        wsum[threadIdx.x / kWave] = total;
        wcount[threadIdx.x / kWave] = count;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    total = 0.0;
    count = 0;
    for (int w = 0; w < waves; ++w) {
        total += wsum[w];
        count += wcount[w];
    }
    const double of = reduction == DOT_REDUCE_MEAN ? 1.0 / (count > 0 ? count : 1) : 1.0;
    out[b] = float(total * of);
    if (weight) weight[b] = float(of);
}

struct GradArgs {
    int K;
    float inv_tau;
    int reduction;
    const float2* stats;
    const int32_t* at;
    const float* own;
    const float* weight;
    const float* grad_out;
    int grad_out_scalar;
    void* grad;
};

// dx of one span of a row.  Bound by HBM: 8192 rows of 131072 bf16, 55 % of them read,
// 3.3 GB in 666 us, 5.0 TB/s; 8184 of 32768, 0.83 GB in 148 us, 5.6 TB/s.
template <class T>
__global__ __launch_bounds__(kBlock) void backward(Rows r, GradArgs g) {
    // last rows first: the forward has just read them
    const int64_t at = int64_t(r.B) * r.S - 1 - blockIdx.x / unsigned(r.splits);
    const int part = int(blockIdx.x % unsigned(r.splits));
    constexpr int PN = Pack<T>::N;
    T* out = static_cast<T*>(g.grad) + at * r.V;
    const Span sp = seqlogp::span_of(out, r.V, part, r.splits);
    const float2 st = g.stats[at];
    if (st.x != st.x) {
        const Pack<T> zero{};
        for (int p = sp.p0 + int(threadIdx.x); p < sp.p1; p += kBlock)
            store_pack_stream(out + sp.head + int64_t(p) * PN, zero);
        if (part == 0 && int(threadIdx.x) < sp.head) out[threadIdx.x] = T{};
        if (part == r.splits - 1 && sp.tail + int(threadIdx.x) < r.V) out[sp.tail + threadIdx.x] = T{};
        return;
    }
    const T* row = seqlogp::row_of<T>(r, at);
    const int64_t b = at / r.S;
    const float up = g.grad_out[g.grad_out_scalar ? 0 : g.reduction == DOT_REDUCE_NONE ? at : b];
    const float c = (g.reduction == DOT_REDUCE_MEAN ? up * g.weight[b] : up) * g.inv_tau;
    const float scale = c * st.y;
    auto value = [&](float x) { return __builtin_amdgcn_exp2f(scaled<T>(r, x - st.x)) * scale; };
    const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    auto pack_in = [&](int p, auto stream) {
        const T* at_p = row + sp.head + int64_t(p) * PN;
        if (together) return seqlogp::row_pack<decltype(stream)::value>(at_p);
        Pack<T> x;
#pragma unroll
        for (int i = 0; i < PN; ++i) x.v[i] = at_p[i];
        return x;
    };
    auto pack_out = [&](int p, const Pack<T>& x) {
        Pack<T> y;
#pragma unroll
        for (int i = 0; i < PN; ++i) y.v[i] = from_float<T>(value(to_float(x.v[i])));
        store_pack_stream(out + sp.head + int64_t(p) * PN, y);
    };
    // A named token's gradient is written over what the packs put there, soon enough to
    // meet them in L2: behind all of the row 64 such stores cost 12 % of a row of 32768 bf16.
    const int mine = int(threadIdx.x) < g.K ? g.at[at * g.K + threadIdx.x] : -1;
    const T own = from_float<T>(mine >= 0 ? c * g.own[at * g.K + threadIdx.x] : 0.0f);
    auto name = [&](int from, int to) {
        __syncthreads();
        if (mine >= from && mine < to) out[mine] = own;
    };
    auto packs = [&](auto stream) {
        constexpr int U = seqlogp::kUnroll;
        int q = sp.p0;
        for (; q + U * kBlock <= sp.p1; q += U * kBlock) {
            const int p = q + int(threadIdx.x);
            Pack<T> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = pack_in(p + u * kBlock, stream);
#pragma unroll
            for (int u = 0; u < U; ++u) pack_out(p + u * kBlock, x[u]);
            name(sp.head + q * PN, sp.head + (q + U * kBlock) * PN);
        }
        for (int p = q + int(threadIdx.x); p < sp.p1; p += kBlock) pack_out(p, pack_in(p, stream));
        return sp.head + q * PN;
    };
    const int behind = at < r.cached ? packs(std::true_type{}) : packs(std::false_type{});
    if (part == 0 && int(threadIdx.x) < sp.head) out[threadIdx.x] = from_float<T>(value(to_float(row[threadIdx.x])));
    const int v = sp.tail + int(threadIdx.x);
    if (part == r.splits - 1 && v < r.V) out[v] = from_float<T>(value(to_float(row[v])));
    name(behind, part == r.splits - 1 ? r.V : sp.head + sp.p1 * PN);
    if (part == 0) name(0, sp.head);
}

}  // namespace distill
}  // namespace dot_amd
