// Routing of tokens to experts: the k largest keys of each row of scores, the
// masses behind them, per-expert counts and column sums, and the gradient.
//
// A row of E scores lies in a group of G lanes of one wave (64 / G rows per
// wave at once), 8 R elements per lane in registers, so softmax, selection and
// gradient are register work plus log2(G) lane exchanges, and a row is read
// once.  Column sums of the shares p are kept in registers over the rows that
// a wave visits; counts go to a histogram in LDS (integers: any order gives
// the same sum).  Each workgroup writes one partial row of both; `finish`
// adds them in chunk order, so results do not depend on scheduling.
#pragma once

#include "elem.cuh"
#include "row.cuh"
#include "wave.cuh"

namespace dot_amd {
namespace routing {

constexpr int kV = 8;  // elements of a lane's vector

// G lanes per row, R vectors per lane.  VEC: the vectors are contiguous
// (16-byte loads; E a multiple of 8, rows 16-byte aligned); otherwise the
// lanes of a group take consecutive elements.
template <int G_, int R_, bool VEC_>
struct Shape {
    static constexpr int G = G_, R = R_, EL = kV * R_, RPW = kWave / G_;
    static constexpr bool VEC = VEC_;
    // The expert of a lane's element j; grows with j.
    __device__ static __forceinline__ int expert(int gl, int j) {
        if constexpr (VEC) return ((j / kV) * G + gl) * kV + j % kV;
        else return j * G + gl;
    }
};

// f(Shape) of the smallest group that holds E <= DOT_ROUTING_MAX_EXPERTS elements.
template <bool VEC, class F>
void dispatch_shape(int E, F&& f) {
    if (E <= 8) f(Shape<1, 1, VEC>{});
    else if (E <= 16) f(Shape<2, 1, VEC>{});
    else if (E <= 32) f(Shape<4, 1, VEC>{});
    else if (E <= 64) f(Shape<8, 1, VEC>{});
    else if (E <= 128) f(Shape<16, 1, VEC>{});
    else if (E <= 256) f(Shape<32, 1, VEC>{});
    else if (E <= 512) f(Shape<64, 1, VEC>{});
    else if (E <= 1024) f(Shape<64, 2, VEC>{});
    else if (E <= 2048) f(Shape<64, 4, VEC>{});
    else f(Shape<64, 8, VEC>{});
}

// Rows that a workgroup visits at once.
inline int rows_per_pass(int E) {
    int g = 1;
    while (g < kWave && g * kV < E) g *= 2;
    return kWavesPerBlock * (kWave / g);
}

// Workgroups per batch element: four per CU over the whole grid, none without
// a full pass of rows.
inline int chunks_of(int B, int N, int E) {
    const int rpp = rows_per_pass(E);
    const int most = (N + rpp - 1) / rpp;
    const int want = (1024 + B - 1) / (B > 0 ? B : 1);
    return most < want ? (most > 0 ? most : 1) : want;
}

// All-reduce over the groups of G lanes of a wave; every lane is active.
template <int G, class X, class Op>
__device__ __forceinline__ X group_reduce(X x, Op op) {
    auto as_f = [](X v) { return __builtin_bit_cast(float, v); };
    auto as_x = [](float v) { return __builtin_bit_cast(X, v); };
    if constexpr (G >= 2) x = op(x, as_x(dpp_move<kDppQuadXor1>(as_f(x))));
    if constexpr (G >= 4) x = op(x, as_x(dpp_move<kDppQuadXor2>(as_f(x))));
    if constexpr (G >= 8) x = op(x, as_x(dpp_move<kDppRowHalfMirror>(as_f(x))));
    if constexpr (G >= 16) x = op(x, as_x(dpp_move<kDppRowMirror>(as_f(x))));
    if constexpr (G >= 32) x = op(x, as_x(swizzle_xor16(as_f(x))));
    if constexpr (G >= 64) x = op(as_x(read_lane(as_f(x), 0)), as_x(read_lane(as_f(x), 32)));
    return x;
}

struct OpMinInt {
    __device__ __forceinline__ int operator()(int a, int b) const { return a < b ? a : b; }
};

// Orders this wave's LDS writes before its later LDS reads.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr float kNegInf = -__builtin_inff();

// A row in registers; elements beyond E, and rows that are not live, are -inf.
template <class T, class S>
__device__ __forceinline__ void load_row(const T* row, int gl, int E, bool live, float (&x)[S::EL]) {
#pragma unroll
    for (int r = 0; r < S::R; ++r) {
        if constexpr (S::VEC) {
            const int c = (r * S::G + gl) * kV;
            if (live && c < E) {
                constexpr int PN = Pack<T>::N;
#pragma unroll
                for (int h = 0; h < kV / PN; ++h) {
                    const Pack<T> p = load_pack(row + c + h * PN);
#pragma unroll
                    for (int i = 0; i < PN; ++i) x[r * kV + h * PN + i] = to_float(p.v[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kV; ++i) x[r * kV + i] = kNegInf;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const int c = S::expert(gl, r * kV + i);
                x[r * kV + i] = (live && c < E) ? to_float(row[c]) : kNegInf;
            }
        }
    }
}

template <class T, class S>
__device__ __forceinline__ void store_row(T* row, int gl, int E, const float (&x)[S::EL]) {
#pragma unroll
    for (int r = 0; r < S::R; ++r) {
        if constexpr (S::VEC) {
            const int c = (r * S::G + gl) * kV;
            if (c < E) {
                constexpr int PN = Pack<T>::N;
#pragma unroll
                for (int h = 0; h < kV / PN; ++h) {
                    Pack<T> p;
#pragma unroll
                    for (int i = 0; i < PN; ++i) p.v[i] = from_float<T>(x[r * kV + h * PN + i]);
                    store_pack_stream(row + c + h * PN, p);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                const int c = S::expert(gl, r * kV + i);
                if (c < E) row[c] = from_float<T>(x[r * kV + i]);
            }
        }
    }
}

// exp(-|x|) and 1 / (1 + exp(-|x|)), from which the logistic function and its
// slope follow without cancellation; NaN stays NaN.
__device__ __forceinline__ void logistic_parts(float x, float& t, float& u) {
    const float d = -fabsf(x);
    t = d < -88.0f ? 0.0f : exp_compensated(d);
    u = __builtin_amdgcn_rcpf(1.0f + t);
}

// The mass of one score where it needs no row statistics.
__device__ __forceinline__ float mass_of(float x, int scoring) {
    if (scoring == DOT_SCORING_SIGMOID) {
        float t, u;
        logistic_parts(x, t, u);
        return x < 0.0f ? t * u : u;
    }
    return x == kNegInf ? 0.0f : x;
}

// Masses q of a row (softmax: exp(x - top), not yet divided), and 1 / sum q
// (0 where the row has no mass; NaN stays NaN).
template <class S>
__device__ __forceinline__ void row_masses(const float (&x)[S::EL], int scoring, float (&q)[S::EL], float& top,
                                           float& inv) {
    float sum = 0.0f;
    top = 0.0f;
    if (scoring == DOT_SCORING_SOFTMAX) {
        float m = kNegInf;
#pragma unroll
        for (int j = 0; j < S::EL; ++j) m = fmaxf(m, x[j]);
        m = group_reduce<S::G>(m, OpMax{});
        top = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < S::EL; ++j) q[j] = fast_exp(x[j] - top);
    } else {
#pragma unroll
        for (int j = 0; j < S::EL; ++j) q[j] = mass_of(x[j], scoring);
    }
#pragma unroll
    for (int j = 0; j < S::EL; ++j) sum += q[j];
    sum = group_reduce<S::G>(sum, OpSum{});
    inv = sum == 0.0f ? 0.0f : 1.0f / sum;
}

struct FwdArgs {
    const void* scores;
    int64_t sb, sn;
    int B, N, E, k;
    int scoring, normalize;
    const float* bias;
    const uint8_t* mask;
    const void* given;
    int given64;
    float* weights;
    int32_t* experts;
    int nchunks, chunk_rows;
    float* psum;       // [B, nchunks, E]
    int32_t* pcount;   // [B, nchunks, E]
    int32_t* ptokens;  // [B, nchunks]
};

// LDS words of forward: column sums and counts, and per wave the (expert,
// score) of the selected slots of its rows.
inline size_t fwd_lds_bytes(int E, int k, int rows, bool select) {
    return (2 * size_t(E) + (select ? 2 * size_t(rows) * size_t(k) : 0)) * 4;
}

template <class T, class S, bool SELECT>
__global__ __launch_bounds__(kBlock) void forward(FwdArgs a) {
    extern __shared__ float lds[];
    __shared__ int ntokens;
    const int b = batch_of_block();
    if (b >= a.B) return;
    const int E = a.E, k = a.k;
    float* col = lds;
    int* hist = reinterpret_cast<int*>(lds + E);
    for (int e = threadIdx.x; e < E; e += kBlock) {
        col[e] = 0.0f;
        hist[e] = 0;
    }
    if (threadIdx.x == 0) ntokens = 0;
    __syncthreads();

    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int gl = lane % S::G, sub = lane / S::G;
    struct Slot {
        int e;
        float s;
    };
    Slot* stage = reinterpret_cast<Slot*>(lds + 2 * E) + size_t(wave) * S::RPW * k + size_t(sub) * k;
    float bias[S::EL];
#pragma unroll
    for (int j = 0; j < S::EL; ++j) {
        const int e = S::expert(gl, j);
        bias[j] = (SELECT && a.bias && e < E) ? a.bias[e] : 0.0f;
    }
    float acc[S::EL];
#pragma unroll
    for (int j = 0; j < S::EL; ++j) acc[j] = 0.0f;
    int live_rows = 0;

    const int begin = int(blockIdx.x) * a.chunk_rows;
    const int end = min(begin + a.chunk_rows, a.N);
    for (int base = begin + wave * S::RPW; base < end; base += kWavesPerBlock * S::RPW) {
        const int n = base + sub;
        const bool in = n < end;
        const int64_t at = int64_t(b) * a.N + n;
        const bool live = in && (!a.mask || a.mask[at]);
        live_rows += live && gl == 0;
        float x[S::EL], q[S::EL], top, inv;
        load_row<T, S>(static_cast<const T*>(a.scores) + int64_t(b) * a.sb + int64_t(n) * a.sn, gl, E, live, x);
        row_masses<S>(x, a.scoring, q, top, inv);
#pragma unroll
        for (int j = 0; j < S::EL; ++j) acc[j] = fmaf(q[j], inv, acc[j]);

        if constexpr (!SELECT) {
            for (int r = gl; r < k; r += S::G) {
                const int64_t e = live ? int_at(a.given, a.given64, at * k + r) : -1;
                if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
            }
        } else {
            // Keys; what is not available, or already taken, is -inf.
            float key[S::EL];
#pragma unroll
            for (int j = 0; j < S::EL; ++j) {
                const float t = x[j] + bias[j];
                const bool open = t > kNegInf && (a.scoring != DOT_SCORING_PLAN || x[j] > 0.0f);
                key[j] = open ? t : kNegInf;
            }
            float most = kNegInf;  // largest selected score of this lane
            for (int r = 0; r < k; ++r) {
                float m = key[0];
#pragma unroll
                for (int j = 1; j < S::EL; ++j) m = fmaxf(m, key[j]);
                m = group_reduce<S::G>(m, OpMax{});
                const bool any = m > kNegInf;
                int e = INT32_MAX;
#pragma unroll
                for (int j = S::EL - 1; j >= 0; --j) e = key[j] == m ? S::expert(gl, j) : e;
                e = group_reduce<S::G>(e, OpMinInt{});
                float s = 0.0f;
                bool owner = false;
#pragma unroll
                for (int j = 0; j < S::EL; ++j) {
                    const bool hit = any && S::expert(gl, j) == e;
                    owner |= hit;
                    s = hit ? x[j] : s;
                    key[j] = hit ? kNegInf : key[j];
                }
                if (owner) {
                    stage[r] = Slot{e, s};
                    most = fmaxf(most, s);
                    atomicAdd(&hist[e], 1);
                } else if (!any && gl == 0) {
                    stage[r] = Slot{-1, 0.0f};
                }
            }
            wave_lds_fence();
            // Weights: exp(s - top) or q(s), over the row's or the selected ones' sum.
            const bool soft = a.scoring == DOT_SCORING_SOFTMAX;
            float scale = soft ? inv : 1.0f;
            if (a.normalize) {
                if (soft) {
                    const float m = group_reduce<S::G>(most, OpMax{});
                    top = m == kNegInf ? 0.0f : m;
                }
                float z = 0.0f;
                for (int r = gl; r < k; r += S::G) {
                    const Slot t = stage[r];
                    if (t.e >= 0) z += soft ? fast_exp(t.s - top) : mass_of(t.s, a.scoring);
                }
                z = group_reduce<S::G>(z, OpSum{});
                scale = z == 0.0f ? 0.0f : 1.0f / z;
                if (soft) scale += inv - inv;  // a row with NaN has no weights
            }
            for (int r = gl; r < k; r += S::G) {
                const Slot t = stage[r];
                const float w = soft ? fast_exp(t.s - top) : mass_of(t.s, a.scoring);
                if (in) {
                    a.weights[at * k + r] = t.e >= 0 ? w * scale : 0.0f;
                    a.experts[at * k + r] = t.e;
                }
            }
            wave_lds_fence();  // the next rows write the slots again
        }
    }

    // Column sums of this workgroup: over the rows of a wave, then wave by wave.
#pragma unroll
    for (int j = 0; j < S::EL; ++j) {
#pragma unroll
        for (int d = S::G; d < kWave; d *= 2) acc[j] += __shfl_xor(acc[j], d);
    }
    if (live_rows) atomicAdd(&ntokens, live_rows);
    for (int w = 0; w < kWavesPerBlock; ++w) {
        if (wave == w && sub == 0) {
#pragma unroll
            for (int j = 0; j < S::EL; ++j) {
                const int e = S::expert(gl, j);
                if (e < E) col[e] += acc[j];
            }
        }
        __syncthreads();
    }
    const int64_t part = int64_t(b) * a.nchunks + blockIdx.x;
    for (int e = threadIdx.x; e < E; e += kBlock) {
        a.psum[part * E + e] = col[e];
        a.pcount[part * E + e] = hist[e];
    }
    if (threadIdx.x == 0) a.ptokens[part] = ntokens;
}

// Counts, tokens and the loss of a batch element from its chunks' partials.
__global__ __launch_bounds__(kBlock) void finish(int B, int E, int k, int nchunks, const float* psum,
                                                 const int32_t* pcount, const int32_t* ptokens, int32_t* counts,
                                                 int32_t* tokens, float* loss) {
    __shared__ double wsum[kWavesPerBlock];
    const int b = batch_of_block();
    if (b >= B) return;
    const int64_t first = int64_t(b) * nchunks;
    int n = 0;
    for (int c = 0; c < nchunks; ++c) n += ptokens[first + c];
    double dot = 0.0;
    for (int e = threadIdx.x; e < E; e += kBlock) {
        double s = 0.0;
        int cnt = 0;
        for (int c = 0; c < nchunks; ++c) {
            s += psum[(first + c) * E + e];
            cnt += pcount[(first + c) * E + e];
        }
        counts[int64_t(b) * E + e] = cnt;
        dot += s * cnt;
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) dot += __shfl_xor(dot, d);
    if (threadIdx.x % kWave == 0) wsum[threadIdx.x / kWave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < kWavesPerBlock; ++w) t += wsum[w];
        tokens[b] = n;
        loss[b] = n > 0 ? float(t * E / (double(k) * n * n)) : 0.0f;
    }
}

struct BwdArgs {
    const void* scores;
    int64_t sb, sn;
    int B, N, E, k;
    int scoring, normalize;
    const uint8_t* mask;
    const int32_t* counts;
    const int32_t* tokens;
    const float* grad_loss;
    int grad_loss_scalar;
    const float* weights;
    const int32_t* experts;
    const float* grad_weights;
    void* grad_scores;
    int nchunks, chunk_rows;
};

// With h_e = dL/dp_e = g E counts_e / (k n^2) (and, for softmax weights that are
// not normalised, the weights' gradient at the selected experts):
//   softmax  ds = p (h - sum p h)  [+ w (dw - sum w dw) at the selected]
//   others   ds = q' ((h - sum p h) / sum q + (dw or (dw - sum w dw) / Q at the selected))
// The k values of a row go to their lanes through a zeroed row in LDS.
template <class T, class S, bool WEIGHTS>
__global__ __launch_bounds__(kBlock) void backward(BwdArgs a) {
    extern __shared__ float lds[];
    const int b = batch_of_block();
    if (b >= a.B) return;
    const int E = a.E, k = a.k;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int gl = lane % S::G, sub = lane / S::G;
    float* spread = lds + (wave * S::RPW + sub) * (S::G * S::EL);
    const bool soft = a.scoring == DOT_SCORING_SOFTMAX;

    // h less its mean over the experts: h - sum p h is the same, as the shares
    // sum to 1, and does not lose the digits that balanced counts share.
    float slope[S::EL];
    double coef = 0.0, mean = 0.0;
    if (a.grad_loss && a.tokens[b] > 0) {
        const double n = a.tokens[b];
        coef = double(a.grad_loss[a.grad_loss_scalar ? 0 : b]) * E / (double(k) * n * n);
        mean = double(k) * n / E;
    }
#pragma unroll
    for (int j = 0; j < S::EL; ++j) {
        const int e = S::expert(gl, j);
        slope[j] = (a.grad_loss && e < E) ? float(coef * (double(a.counts[int64_t(b) * E + e]) - mean)) : 0.0f;
    }

    const int begin = int(blockIdx.x) * a.chunk_rows;
    const int end = min(begin + a.chunk_rows, a.N);
    for (int base = begin + wave * S::RPW; base < end; base += kWavesPerBlock * S::RPW) {
        const int n = base + sub;
        const bool in = n < end;
        const int64_t at = int64_t(b) * a.N + n;
        const bool live = in && (!a.mask || a.mask[at]);
        const T* row = static_cast<const T*>(a.scores) + int64_t(b) * a.sb + int64_t(n) * a.sn;
        float x[S::EL], q[S::EL], top, inv;
        load_row<T, S>(row, gl, E, live, x);
        row_masses<S>(x, a.scoring, q, top, inv);
        float add[S::EL];
#pragma unroll
        for (int j = 0; j < S::EL; ++j) add[j] = 0.0f;
        if constexpr (WEIGHTS) {
#pragma unroll
            for (int j = 0; j < S::EL; ++j) spread[S::expert(gl, j)] = 0.0f;
            float dot = 0.0f, scale = 1.0f;
            if (a.normalize) {
                float mass = 0.0f;
                for (int r = gl; r < k; r += S::G) {
                    const int e = live ? a.experts[at * k + r] : -1;
                    if (e >= 0 && e < E) {
                        dot = fmaf(a.weights[at * k + r], a.grad_weights[at * k + r], dot);
                        if (!soft) mass += mass_of(to_float(row[e]), a.scoring);
                    }
                }
                dot = group_reduce<S::G>(dot, OpSum{});
                if (!soft) {
                    mass = group_reduce<S::G>(mass, OpSum{});
                    scale = mass == 0.0f ? 0.0f : 1.0f / mass;
                }
            }
            wave_lds_fence();
            for (int r = gl; r < k; r += S::G) {
                const int e = live ? a.experts[at * k + r] : -1;
                if (e >= 0 && e < E) {
                    float v = (a.grad_weights[at * k + r] - dot) * scale;
                    if (soft && a.normalize) v *= a.weights[at * k + r];
                    spread[e] = v;
                }
            }
            wave_lds_fence();
#pragma unroll
            for (int j = 0; j < S::EL; ++j) add[j] = spread[S::expert(gl, j)];
            wave_lds_fence();
        }
        float ph = 0.0f;
        const bool in_h = soft && !a.normalize;  // the weights are p itself
#pragma unroll
        for (int j = 0; j < S::EL; ++j) {
            const float h = slope[j] + (in_h ? add[j] : 0.0f);
            ph = fmaf(q[j] * inv, h, ph);
        }
        ph = group_reduce<S::G>(ph, OpSum{});
        float g[S::EL];
#pragma unroll
        for (int j = 0; j < S::EL; ++j) {
            if (soft) {
                const float h = slope[j] + (in_h ? add[j] : 0.0f);
                g[j] = fmaf(q[j] * inv, h - ph, in_h ? 0.0f : add[j]);
            } else {
                g[j] = fmaf(slope[j] - ph, inv, add[j]);
                if (a.scoring == DOT_SCORING_SIGMOID) {
                    // q (1 - q) = t u^2: exact where q is near 1
                    float t, u;
                    logistic_parts(x[j], t, u);
                    g[j] *= t * u * u;
                }
            }
            g[j] = live ? g[j] : 0.0f;
        }
        if (in) store_row<T, S>(static_cast<T*>(a.grad_scores) + at * E, gl, E, g);
    }
}

inline size_t bwd_lds_bytes(int lanes_elems, bool weights) {
    return weights ? size_t(kWavesPerBlock) * size_t(lanes_elems) * sizeof(float) : 0;
}

}  // namespace routing
}  // namespace dot_amd
