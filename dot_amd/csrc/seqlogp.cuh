// Log-probabilities of tokens from rows of logits, summed over sequences, and
// the gradient of the logits.
//
// The forward reads each row once with a running maximum m and sum
// s = sum_v 2^((x_v - m) k), k = log2(e) / tau, over the vocabulary without the
// position's own token, which is added in 64 bits: next to a likely token's 1
// the others' terms of 1e-7 each would lose their digits.  The 4 or 8 terms of a
// pack are added pairwise in 32 bits, at most 3 roundings (2e-7 of their sum, of
// either sign from pack to pack), and the packs' sums in 64 bits.  A row may be
// split over several workgroups, whose (m, s) the second kernel joins.  That
// kernel also forms the position's value and the sequence's sum in 64 bits: the
// log ratio of two models is a small difference of large sums.  x - m is formed
// before the scale, so rows at the type's lowest value give finite statistics.  The
// backward reads the row again and writes dx_v = c (delta_va - p_v) with
// p_v = 2^((x_v - m) k) / s.  Where the token a is likelier than not, 1 - p_a
// is kept as the others' share of the sum, formed in 64 bits: as a difference it
// would lose the digits that the forward keeps.  Rows that are left out are not
// read.
#pragma once

#include "elem.cuh"
#include "row.cuh"
#include "wave.cuh"

namespace dot_amd {
namespace seqlogp {

constexpr int kUnroll = 4;       // packs of a thread in flight (8: 2 % slower)
constexpr int kJoinBlock = 1024; // threads of the per-sequence kernel

struct Rows {
    const void* logits;
    int64_t sb, ss;
    int B, S, V;
    const void* tokens;
    int tokens64;
    const uint8_t* mask;
    // log2(e) / tau = k + klo, both > 0.  One float is off by up to 6e-8 of
    // itself, which shifts every position's value the same way: 1e-7 each on
    // typical rows, 1e-4 over a thousand positions.
    float k, klo;
    int splits;  // workgroups per row
    // Rows from here on are read through the caches and may stay in the last
    // level for the backward, which takes the rows in the other order; those
    // before are read past the caches.
    int64_t cached;
};

// d log2(e) / tau of a difference d <= 0 (-inf stays -inf: klo is not 0).
__device__ __forceinline__ float scaled(const Rows& r, float d) { return fmaf(d, r.k, d * r.klo); }

// The token of a position, or -1 where it is left out.
__device__ __forceinline__ int token_of(const Rows& r, int64_t at) {
    if (r.mask && !r.mask[at]) return -1;
    const int64_t t = int_at(r.tokens, r.tokens64, at);
    return t >= 0 && t < r.V ? int(t) : -1;
}

template <class T>
__device__ __forceinline__ const T* row_of(const Rows& r, int64_t at) {
    const int64_t b = at / r.S, s = at - b * r.S;
    return static_cast<const T*>(r.logits) + b * r.sb + s * r.ss;
}

// Split `part` of `parts` of a row of V elements: whole packs [p0, p1) after
// `head` unaligned elements; the first split takes the head, the last the tail
// from `tail` on.
struct Span {
    int head, tail;
    int p0, p1;
};
template <class T>
__device__ __forceinline__ Span span_of(const T* row, int V, int part, int parts) {
    constexpr int PN = Pack<T>::N;
    Span s;
    const int off = int((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    s.head = min((PN - off) % PN, V);
    const int packs = (V - s.head) / PN;
    s.tail = s.head + packs * PN;
    const int per = (packs + parts - 1) / parts;
    s.p0 = min(part * per, packs);
    s.p1 = min(s.p0 + per, packs);
    return s;
}

// A pack of logits, through the caches or (STREAM) past them.
template <bool STREAM, class T>
__device__ __forceinline__ Pack<T> row_pack(const T* p) {
    if constexpr (STREAM) return load_pack_stream(p);
    else return load_pack(p);
}

// 16 bytes of -inf of each type.
__device__ const uint32_t kNothing[3][4] __attribute__((aligned(16))) = {
    {0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u},
    {0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u},
    {0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u}};
__device__ __forceinline__ const void* nothing_of(float) { return kNothing[DOT_F32]; }
__device__ __forceinline__ const void* nothing_of(F16) { return kNothing[DOT_F16]; }
__device__ __forceinline__ const void* nothing_of(BF16) { return kNothing[DOT_BF16]; }

// Sum of N values, pairwise.
template <int N>
__device__ __forceinline__ float pairwise(const float* x) {
    if constexpr (N == 1) return x[0];
    else return pairwise<N / 2>(x) + pairwise<N - N / 2>(x + N / 2);
}

// Largest value and sum of 2^((x - m) k) so far; m = -inf: nothing but -inf.
struct MaxSum {
    float m = -__builtin_inff();
    double s = 0.0;
    __device__ __forceinline__ float base() const { return m == -__builtin_inff() ? 0.0f : m; }
    __device__ __forceinline__ void raise(float to, const Rows& r) {
        const float old = m;
        m = fmaxf(m, to);
        s *= double(__builtin_amdgcn_exp2f(scaled(r, old - base())));
    }
    // N values at once, in 32 bits over M of them
    template <int M, int N>
    __device__ __forceinline__ void add(const float (&x)[N], const Rows& r) {
        float most = x[0], e[N];
#pragma unroll
        for (int i = 1; i < N; ++i) most = fmaxf(most, x[i]);
        raise(most, r);
        const float c = base();
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = __builtin_amdgcn_exp2f(scaled(r, x[i] - c));
#pragma unroll
        for (int i = 0; i < N; i += M) s += double(pairwise<M>(e + i));
    }
    __device__ __forceinline__ void join(float om, double os, const Rows& r) {
        raise(om, r);
        s += os * double(__builtin_amdgcn_exp2f(scaled(r, om - base())));
    }
};

struct Part {
    double s;
    float m;
};

struct JoinArgs {
    const void* ref;
    int ref64, ref_per_token;
    int reduction;
    float* out;
    float2* stats;
    float* weight;
};

__device__ __forceinline__ double float_at(const void* p, int is64, int64_t i) {
    return is64 ? static_cast<const double*>(p)[i] : double(static_cast<const float*>(p)[i]);
}

// What a position needs besides its row's statistics.
struct Own {
    float x;     // its token's logit
    double ref;  // the reference's log-probability
};
template <class T>
__device__ __forceinline__ Own own_of(const Rows& r, const JoinArgs& j, int64_t at, int tok) {
    return Own{to_float(row_of<T>(r, at)[tok]), j.ref && j.ref_per_token ? float_at(j.ref, j.ref64, at) : 0.0};
}

// The value of a position from the statistics of its row's other logits.  Those
// of the whole row are kept for the backward: the largest logit m, and 1 / s; or,
// where the token's share is above 1/2 (it is the largest then, its term is 1),
// -(1 - p_a) = -(s - 1) / s, from which 1 / s = p_a follows.
__device__ __forceinline__ double position(const Rows& r, const JoinArgs& j, int64_t at, const Own& own, MaxSum t) {
    const double kn = (double(r.k) + double(r.klo)) * 0.693147180559945309417;  // 1 / tau
    const MaxSum others = t;
    t.join(own.x, 1.0, r);
    const float base = t.base();
    if (j.stats) {
        const double rest = others.s * double(__builtin_amdgcn_exp2f(scaled(r, others.m - base)));
        const bool likely = own.x == base && t.s < 2.0;  // not NaN
        j.stats[at] = make_float2(base, likely ? -float(rest / t.s) : float(1.0 / t.s));
    }
    return (double(own.x) - double(base)) * kn - log(t.s) - own.ref;
}

// Partial statistics of every row, one for each split; a row that is not split
// gets its position's value at once (in the place of s, or in the output).
template <class T>
__global__ __launch_bounds__(kBlock) void row_stats(Rows r, JoinArgs j, Part* parts) {
    __shared__ float sm[kWavesPerBlock];
    __shared__ double ss[kWavesPerBlock];
    const int64_t at = blockIdx.x / unsigned(r.splits);
    const int part = int(blockIdx.x % unsigned(r.splits));
    const int tok = token_of(r, at);
    auto put = [&](double v) {
        if (j.reduction == DOT_REDUCE_NONE) j.out[at] = float(v);
        else parts[at].s = v;
    };
    if (tok < 0) {
        if (r.splits == 1 && threadIdx.x == 0) put(0.0);
        return;
    }
    Own own{};
    if (r.splits == 1) own = own_of<T>(r, j, at, tok);  // on its way while the row is read
    const T* row = row_of<T>(r, at);
    const Span sp = span_of(row, r.V, part, r.splits);
    const T* body = row + sp.head;
    constexpr int PN = Pack<T>::N;
    // The token's pack is read as logits of -inf; its other logits are added one
    // by one at the end.  They are on their way while the row is read.
    const int tok_pack = tok < sp.head || tok >= sp.tail ? -1 : (tok - sp.head) / PN;
    float beside = -__builtin_inff();
    if (tok_pack >= sp.p0 && tok_pack < sp.p1 && int(threadIdx.x) < PN) {
        const int v = sp.head + tok_pack * PN + int(threadIdx.x);
        if (v != tok) beside = to_float(row[v]);
    }
    const T* nothing = reinterpret_cast<const T*>(nothing_of(T{}));
    MaxSum a;
    auto packs = [&](auto stream) {
        auto pack = [&](int p) {
            return row_pack<decltype(stream)::value>(p == tok_pack ? nothing : body + int64_t(p) * PN);
        };
        int p = sp.p0 + int(threadIdx.x);
        for (; p + (kUnroll - 1) * kBlock < sp.p1; p += kUnroll * kBlock) {
            Pack<T> x[kUnroll];
            float f[kUnroll * PN];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) x[u] = pack(p + u * kBlock);
#pragma unroll
            for (int i = 0; i < kUnroll * PN; ++i) f[i] = to_float(x[i / PN].v[i % PN]);
            a.add<PN>(f, r);
        }
        for (; p < sp.p1; p += kBlock) {
            const Pack<T> x = pack(p);
            float f[PN];
#pragma unroll
            for (int i = 0; i < PN; ++i) f[i] = to_float(x.v[i]);
            a.add<PN>(f, r);
        }
    };
    if (at < r.cached) packs(std::true_type{});
    else packs(std::false_type{});
    {
        const float f[1] = {beside};
        a.add<1>(f, r);
    }
    if (part == 0 && int(threadIdx.x) < sp.head && int(threadIdx.x) != tok) {
        const float f[1] = {to_float(row[threadIdx.x])};
        a.add<1>(f, r);
    }
    if (part == r.splits - 1 && sp.tail + int(threadIdx.x) < r.V && sp.tail + int(threadIdx.x) != tok) {
        const float f[1] = {to_float(row[sp.tail + threadIdx.x])};
        a.add<1>(f, r);
    }
    const float m = wave_max(a.m);
    a.raise(m, r);
    double s = a.s;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) s += __shfl_xor(s, d);
    if (threadIdx.x % kWave == 0) {
        sm[threadIdx.x / kWave] = m;
        ss[threadIdx.x / kWave] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        MaxSum t;
        for (int w = 0; w < kWavesPerBlock; ++w) t.join(sm[w], ss[w], r);
        if (r.splits == 1) put(position(r, j, at, own, t));
        else parts[blockIdx.x] = Part{t.s, t.m};
    }
}

// One workgroup per sequence: joins the parts of its split rows, and adds up the
// values of its positions.
template <class T>
__global__ __launch_bounds__(kJoinBlock) void join(Rows r, const Part* parts, JoinArgs j) {
    __shared__ double wsum[kJoinBlock / kWave];
    __shared__ int wcount[kJoinBlock / kWave];
    const int b = batch_of_block();
    if (b >= r.B) return;
    double sum = 0.0;
    int count = 0;
    for (int s = threadIdx.x; s < r.S; s += kJoinBlock) {
        const int64_t at = int64_t(b) * r.S + s;
        const bool whole = r.splits == 1;
        // positions are counted for the mean; an unsplit row has its value already
        const int tok = !whole || j.reduction == DOT_REDUCE_MEAN ? token_of(r, at) : -1;
        double v = 0.0;
        if (whole) {
            v = parts[at].s;
        } else if (tok >= 0) {
            MaxSum t;
            for (int i = 0; i < r.splits; ++i) {
                const Part p = parts[at * r.splits + i];
                t.join(p.m, p.s, r);
            }
            v = position(r, j, at, own_of<T>(r, j, at, tok), t);
        }
        sum += v;
        count += tok >= 0;
        if (j.reduction == DOT_REDUCE_NONE) j.out[at] = float(v);
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        sum += __shfl_xor(sum, d);
        count += __shfl_xor(count, d);
    }
    if (threadIdx.x % kWave == 0) {
        wsum[threadIdx.x / kWave] = sum;
        wcount[threadIdx.x / kWave] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        int n = 0;
        for (int w = 0; w < kJoinBlock / kWave; ++w) {
            t += wsum[w];
            n += wcount[w];
        }
        const double weight = j.reduction == DOT_REDUCE_MEAN ? 1.0 / (n > 0 ? n : 1) : 1.0;
        if (j.reduction == DOT_REDUCE_MEAN && j.weight) j.weight[b] = float(weight);
        if (j.reduction != DOT_REDUCE_NONE) {
            t *= weight;
            if (j.ref && !j.ref_per_token) t -= float_at(j.ref, j.ref64, b);
            j.out[b] = float(t);
        }
    }
}

struct GradArgs {
    float inv_tau;
    int reduction;
    const float2* stats;
    const float* weight;
    const float* grad_out;
    int grad_out_scalar;
    void* grad;
};

// dx of one span of a row.
template <class T>
__global__ __launch_bounds__(kBlock) void backward(Rows r, GradArgs g) {
    // last rows first: the forward has just read them
    const int64_t at = int64_t(r.B) * r.S - 1 - blockIdx.x / unsigned(r.splits);
    const int part = int(blockIdx.x % unsigned(r.splits));
    constexpr int PN = Pack<T>::N;
    const int tok = token_of(r, at);
    T* out = static_cast<T*>(g.grad) + at * r.V;
    if (tok < 0) {
        const Span sp = span_of(out, r.V, part, r.splits);
        const Pack<T> zero{};
        for (int p = sp.p0 + int(threadIdx.x); p < sp.p1; p += kBlock)
            store_pack_stream(out + sp.head + int64_t(p) * PN, zero);
        if (part == 0 && int(threadIdx.x) < sp.head) out[threadIdx.x] = T{};
        if (part == r.splits - 1 && sp.tail + int(threadIdx.x) < r.V) out[sp.tail + threadIdx.x] = T{};
        return;
    }
    const T* row = row_of<T>(r, at);
    const int64_t b = at / r.S;
    const float2 st = g.stats[at];
    const float up = g.grad_out[g.grad_out_scalar ? 0 : g.reduction == DOT_REDUCE_NONE ? at : b];
    const float c = (g.reduction == DOT_REDUCE_MEAN ? up * g.weight[b] : up) * g.inv_tau;
    const bool likely = __builtin_bit_cast(int, st.y) < 0;  // -(1 - p_a), -0 among them
    const float scale = -c * (likely ? 1.0f + st.y : st.y);
    const float taken = likely ? c * -st.y : c, with = likely ? 0.0f : 1.0f;
    auto value = [&](float x, int v) {
        const float y = __builtin_amdgcn_exp2f(scaled(r, x - st.x)) * scale;
        return v == tok ? fmaf(with, y, taken) : y;
    };
    const bool together = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    const Span sp = span_of(out, r.V, part, r.splits);
    auto pack_in = [&](int p, auto stream) {
        const T* at_p = row + sp.head + int64_t(p) * PN;
        if (together) return row_pack<decltype(stream)::value>(at_p);
        // A strided view whose rows are not aligned as the gradient's.  The bytes bound it
        // all the same: logits[:, :-1] of 4 x 1025 x 50257 bf16 148.8 us, in one piece 148.0.
        Pack<T> x;
#pragma unroll
        for (int i = 0; i < PN; ++i) x.v[i] = at_p[i];
        return x;
    };
    auto pack_out = [&](int p, const Pack<T>& x) {
        const int v0 = sp.head + p * PN;
        Pack<T> y;
#pragma unroll
        for (int i = 0; i < PN; ++i) y.v[i] = from_float<T>(value(to_float(x.v[i]), v0 + i));
        store_pack_stream(out + v0, y);
    };
    auto packs = [&](auto stream) {
        int p = sp.p0 + int(threadIdx.x);
        for (; p + (kUnroll - 1) * kBlock < sp.p1; p += kUnroll * kBlock) {
            Pack<T> x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) x[u] = pack_in(p + u * kBlock, stream);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) pack_out(p + u * kBlock, x[u]);
        }
        for (; p < sp.p1; p += kBlock) pack_out(p, pack_in(p, stream));
    };
    if (at < r.cached) packs(std::true_type{});
    else packs(std::false_type{});
    if (part == 0 && int(threadIdx.x) < sp.head)
        out[threadIdx.x] = from_float<T>(value(to_float(row[threadIdx.x]), int(threadIdx.x)));
    const int v = sp.tail + int(threadIdx.x);
    if (part == r.splits - 1 && v < r.V) out[v] = from_float<T>(value(to_float(row[v]), v));
}

}  // namespace seqlogp
}  // namespace dot_amd
