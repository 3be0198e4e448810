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

// f(Shape) of a group that holds E <= DOT_ROUTING_MAX_EXPERTS elements.  A round
// of the selection costs a wave about 8 + 1.5 EL + log2(G) instructions for its
// 64 / G rows, so a forward that selects (PAIRS) takes two vectors per lane from
// 128 experts on: 65536 x 256 fp32, k = 8, 32.0 us, with twice the lanes 36.8.
// Without a selection, and in the backward, twice the lanes are faster: 13.7 us
// against 15.4, and 35.0 against 39.1.
template <bool VEC, bool PAIRS, class F>
void dispatch_shape(int E, F&& f) {
    if (E <= 8) f(Shape<1, 1, VEC>{});
    else if (E <= 16) f(Shape<2, 1, VEC>{});
    else if (E <= 32) f(Shape<4, 1, VEC>{});
    else if (E <= 64) f(Shape<8, 1, VEC>{});
    else if (E <= 128) f(Shape<16, 1, VEC>{});
    else if (E <= 256) f(Shape<PAIRS ? 16 : 32, PAIRS ? 2 : 1, VEC>{});
    else if (E <= 512) f(Shape<PAIRS ? 32 : 64, PAIRS ? 2 : 1, VEC>{});
    else if (E <= 1024) f(Shape<64, 2, VEC>{});
    else if (E <= 2048) f(Shape<64, 4, VEC>{});
    else f(Shape<64, 8, VEC>{});
}

// Threads of a forward workgroup.  Few partial rows make `finish` short, so
// workgroups are large where a lane's registers allow it (up to two vectors; the
// forward above takes 38.3 us with 512 workgroups of 256 threads).
constexpr int fwd_block(int R) { return R <= 2 ? 512 : 256; }
// Waves per SIMD that the registers have to leave room for: two workgroups per CU.
constexpr int fwd_waves(int R) { return R <= 2 ? 4 : 1; }
// Rows of column sums in LDS: one per wave, or, for the longest rows, one that
// the waves add to in turn.
constexpr int fwd_col_rows(int R) { return R <= 2 ? fwd_block(R) / kWave : 1; }

// Workgroups per batch element: `total` over the whole grid, none without a
// full pass of rows.
inline int chunks_of(int B, int N, int rows_per_pass, int total) {
    const int most = (N + rows_per_pass - 1) / rows_per_pass;
    const int want = (total + B - 1) / (B > 0 ? B : 1);
    return most < want ? (most > 0 ? most : 1) : want;
}

// x of a lane combined with that of the lane in the other row of its pair of
// rows of 16 (or in the other half of the wave): the swap instructions exchange
// the odd rows of one operand with the even rows of the other, so with x in
// both, one result holds the even row's value and the other the odd row's in
// every lane.
template <int D, class X, class Op>
__device__ __forceinline__ X swapped(X x, Op op) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    unsigned even, odd;
    if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        even = r[0], odd = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        even = r[0], odd = r[1];
    }
    return op(__builtin_bit_cast(X, even), __builtin_bit_cast(X, odd));
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
    if constexpr (G >= 32) x = swapped<16>(x, op);
    if constexpr (G >= 64) x = swapped<32>(x, op);
    return x;
}

// Floats as integers of the same order (-0 below 0), and back.  Integer
// maxima fuse with the lane exchanges, those of floats do not.
constexpr int kTaken = INT32_MIN;  // below every float
__device__ __forceinline__ int ordered(float x) {
    const int i = __builtin_bit_cast(int, x);
    return i ^ ((i >> 31) & INT32_MAX);
}
__device__ __forceinline__ float unordered(int i) {
    return __builtin_bit_cast(float, i ^ ((i >> 31) & INT32_MAX));
}

struct OpMaxInt {
    __device__ __forceinline__ int operator()(int a, int b) const { return a > b ? a : b; }
};
struct OpMaxUint {
    __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a > b ? a : b; }
};
struct OpMinInt {
    __device__ __forceinline__ int operator()(int a, int b) const { return a < b ? a : b; }
};

// All-reduce by sums over the lanes with the same place in their groups of G.
template <int G>
__device__ __forceinline__ float across_groups(float x) {
    constexpr int kRowRor = 0x120;  // rotation inside a row of 16 lanes
    if constexpr (G <= 8) x += dpp_move<kRowRor + 8>(x);
    if constexpr (G <= 4) x += dpp_move<kRowRor + 4>(x);
    if constexpr (G <= 2) x += dpp_move<kRowRor + 2>(x);
    if constexpr (G <= 1) x += dpp_move<kRowRor + 1>(x);
    if constexpr (G <= 16) x = swapped<16>(x, OpSum{});
    if constexpr (G <= 32) x = swapped<32>(x, OpSum{});
    return x;
}

// Orders this wave's LDS writes before its later LDS reads.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr float kNegInf = -__builtin_inff();

// A row as it lies in memory, in registers.
template <class T, class S>
struct RawRow {
    static constexpr int PN = Pack<T>::N, PACKS = S::EL / PN;
    union {
        Pack<T> pack[PACKS];
        T one[S::EL];
    };
    bool live;

    __device__ __forceinline__ void load(const T* row, int gl, int E, bool live_) {
        live = live_;
        if (!live) return;
        if constexpr (S::VEC) {
#pragma unroll
            for (int r = 0; r < S::R; ++r) {
                const int c = (r * S::G + gl) * kV;
                if (c < E) {
#pragma unroll
                    for (int h = 0; h < kV / PN; ++h) pack[r * (kV / PN) + h] = load_pack(row + c + h * PN);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < S::EL; ++j) {
                const int c = S::expert(gl, j);
                if (c < E) one[j] = row[c];
            }
        }
    }
    // As floats; elements beyond E, and rows that are not live, are -inf.
    __device__ __forceinline__ void get(int gl, int E, float (&x)[S::EL]) const {
        if constexpr (S::VEC) {
#pragma unroll
            for (int r = 0; r < S::R; ++r) {
                const bool in = live && (r * S::G + gl) * kV < E;
#pragma unroll
                for (int j = r * kV; j < (r + 1) * kV; ++j) x[j] = in ? to_float(one[j]) : kNegInf;
            }
        } else {
#pragma unroll
            for (int j = 0; j < S::EL; ++j) x[j] = live && S::expert(gl, j) < E ? to_float(one[j]) : kNegInf;
        }
    }
};

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

// e^x of x <= 0.  FULL: to 1.25 ulp; otherwise the argument's product is rounded
// once, (|x| + 2) 2^-23 of the result.  Weights and fp32 gradients are results of
// single tokens and take the former (backward of 65536 x 256 fp32: 34.5 us with
// the short one, 35.0; the forward's weights no difference).
template <bool FULL>
__device__ __forceinline__ float exp_of(float x) {
    if constexpr (FULL) return exp_compensated_below(x);
    else return fast_exp(x);
}

// t = exp(-|x|) and u = 1 / (1 + t), from which the logistic function and its
// slope t u^2 follow without cancellation; NaN stays NaN.
template <bool FULL>
__device__ __forceinline__ void logistic_parts(float x, float& t, float& u) {
    t = exp_of<FULL>(-fabsf(x));
    u = __builtin_amdgcn_rcpf(1.0f + t);
}

// The mass of one score where it needs no row statistics.
__device__ __forceinline__ float mass_of(float x, int scoring) {
    if (scoring != DOT_SCORING_SIGMOID) return x == kNegInf ? 0.0f : x;
    float t, u;
    logistic_parts<true>(x, t, u);
    return x < 0.0f ? t * u : u;
}

// Masses q of a row (softmax: exp(x - top), not yet divided), and 1 / sum q
// (0 where the row has no mass: below the smallest normal float; NaN stays NaN).  SLOPE: x becomes dq/dx of the
// masses that need no row statistics.
template <class S, bool FULL, bool SLOPE>
__device__ __forceinline__ void row_masses(float (&x)[S::EL], int scoring, float (&q)[S::EL], float& top,
                                           float& inv) {
    float sum = 0.0f;
    top = 0.0f;
    if (scoring == DOT_SCORING_SOFTMAX) {
        float m = kNegInf;
#pragma unroll
        for (int j = 0; j < S::EL; ++j) m = fmaxf(m, x[j]);
        m = unordered(group_reduce<S::G>(ordered(m), OpMaxInt{}));
        top = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < S::EL; ++j) q[j] = exp_of<FULL>(x[j] - top);
    } else if (scoring == DOT_SCORING_SIGMOID) {
#pragma unroll
        for (int j = 0; j < S::EL; ++j) {
            float t, u;
            logistic_parts<FULL>(x[j], t, u);
            q[j] = x[j] < 0.0f ? t * u : u;
            if (SLOPE) x[j] = t * u * u;  // q (1 - q), exact where q is near 1
        }
    } else {
#pragma unroll
        for (int j = 0; j < S::EL; ++j) {
            q[j] = x[j] == kNegInf ? 0.0f : x[j];
            if (SLOPE) x[j] = 1.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < S::EL; ++j) sum += q[j];
    sum = group_reduce<S::G>(sum, OpSum{});
    inv = fabsf(sum) < FLT_MIN ? 0.0f : 1.0f / sum;
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
    // one row of partials per workgroup: column sums, counts, tokens
    float* psum;       // [B, nchunks, E]
    int32_t* pcount;   // [B, nchunks, E]
    int32_t* ptokens;  // [B, nchunks]
    uint32_t* done;    // [B] column blocks that `finish` is through with; cleared here
    int32_t* counts;   // the results, written here where there is one chunk
    int32_t* tokens;
    float* loss;
};

struct Slot {
    int e;
    float s;
};

// LDS of forward: column sums and counts, from word bias_at() on (16-byte
// aligned) the bias, with a place for every element of a group, and the selected
// slots of each row.
__host__ __device__ constexpr int bias_at(int col_rows, int E) { return ((col_rows + 1) * E + 3) & ~3; }
inline size_t fwd_lds_bytes(int E, int k, int G, int R, int rows, bool select) {
    const size_t words = size_t(bias_at(fwd_col_rows(R), E)) + size_t(G) * R * kV;
    return words * 4 + (select ? size_t(rows) * size_t(k) * sizeof(Slot) : 0);
}

__device__ __forceinline__ float loss_value(double dot, int E, int k, int n) {
    return n > 0 ? float(dot * E / (double(k) * n * n)) : 0.0f;
}

__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d);
    return x;
}

// The experts of the k largest keys score + bias of a row to stage[0..k), equal
// keys by the lowest expert, -1 where none is left.
//
// Keys are 31-bit integers, the ordered key above and the inverted expert below,
// so that no two are the same.  A round then needs no search and no marking of
// what was taken: with m the last winner, u - m as an unsigned number is large
// only for the u below m, and largest for the one next to it.  16-bit scores
// without a bias fit whole.  A 32-bit key loses its low bits; where two winners
// in a row agree in what is left (the one behind the last among them), their
// wave selects again by whole keys.  65536 rows of 256 fp32 scores, k = 8:
// 36 us for the forward, 52 with the whole keys alone.
template <class T, class S>
__device__ __forceinline__ void select(const T* row, const RawRow<T, S>& raw, const float* bias, bool biased, bool plan,
                                       int gl, int E, int k, Slot* stage) {
    constexpr unsigned kMask = S::G * S::EL - 1;  // a power of two less one
    constexpr int kBits = __builtin_popcount(kMask);
    // A row's scores with the bias (0 where there is none; -0 becomes 0), and
    // whether an expert is available.
    float x[S::EL];
    bool open[S::EL];
    auto load = [&](const RawRow<T, S>& from) {
        from.get(gl, E, x);
#pragma unroll
        for (int j = 0; j < S::EL; ++j) open[j] = x[j] > (plan ? 0.0f : kNegInf);
#pragma unroll
        for (int j = 0; j < S::EL; ++j) {
            x[j] += bias[S::expert(gl, j)];
            open[j] = open[j] & (x[j] > kNegInf);
        }
    };
    load(raw);
    unsigned u[S::EL];
#pragma unroll
    for (int j = 0; j < S::EL; ++j) {
        // the key's low bits give way to the expert (those of a 16-bit score are all alike)
        const unsigned i = __builtin_bit_cast(unsigned, x[j]);
        const unsigned upper = (i ^ (unsigned(int(i) >> 31) | 0x80000000u)) >> 1;
        const unsigned both = (upper & ~kMask) | (kMask - unsigned(S::expert(gl, j)));
        u[j] = open[j] ? both : 0u;
    }
    unsigned m = 0x80000000u;
    bool close = false;  // winners that agree in the key's upper bits
    for (int r0 = 0; r0 <= k; r0 += S::G) {
        const unsigned last = m;
        unsigned mine = 0;  // the winner of round r0 + gl
        const int rounds = min(k + 1 - r0, S::G);
        for (int r = 0; r < rounds; ++r) {
            unsigned d = u[0] - m;
#pragma unroll
            for (int j = 1; j < S::EL; ++j) d = max(d, u[j] - m);
            d = group_reduce<S::G>(d, OpMaxUint{});
            m = m == 0u ? 0u : m + d;
            mine = r == gl ? m : mine;
        }
        if (r0 + gl < k) stage[r0 + gl].e = mine ? int(kMask - (mine & kMask)) : -1;
        const unsigned beside = __shfl_up(mine, 1);
        const unsigned before = gl == 0 ? last : beside;
        close |= mine != 0u && ((mine ^ before) >> kBits) == 0u;
    }
    wave_lds_fence();
    const bool whole = sizeof(T) == 2 && !biased;
    if (whole || !__any(close)) return;

    // Whole keys; the row is read again rather than kept over the rounds above.
    RawRow<T, S> again;
    again.load(row, gl, E, raw.live);
    load(again);
    int key[S::EL];
#pragma unroll
    for (int j = 0; j < S::EL; ++j) key[j] = open[j] ? ordered(x[j]) : kTaken;
    for (int r = 0; r < k; ++r) {
        int top = key[0];
#pragma unroll
        for (int j = 1; j < S::EL; ++j) top = max(top, key[j]);
        top = group_reduce<S::G>(top, OpMaxInt{});
        int first = INT32_MAX;  // this lane's first element with that key
#pragma unroll
        for (int j = S::EL - 1; j >= 0; --j) first = key[j] == top ? j : first;
        const int mine = first == INT32_MAX ? INT32_MAX : S::expert(gl, first);
        const int e = group_reduce<S::G>(mine, OpMinInt{});
        const int take = e == mine ? first : -1;
#pragma unroll
        for (int j = 0; j < S::EL; ++j) key[j] = j == take ? kTaken : key[j];
        if (gl == (r & (S::G - 1))) stage[r].e = top == kTaken ? -1 : e;
    }
    wave_lds_fence();
}

template <class T, class S, bool SELECT>
__global__ __launch_bounds__(fwd_block(S::R), fwd_waves(S::R)) void forward(FwdArgs a) {
    constexpr int kThreads = fwd_block(S::R), kWaves = kThreads / kWave;
    extern __shared__ float lds[];
    __shared__ int ntokens;
    __shared__ double wdot[kWaves];
    const int b = batch_of_block();
    if (b >= a.B) return;
    const int E = a.E, k = a.k;
    constexpr int kColRows = fwd_col_rows(S::R);
    float* col = lds;
    int* hist = reinterpret_cast<int*>(lds + kColRows * E);
    float* bias = lds + bias_at(kColRows, E);
    for (int e = threadIdx.x; e < E; e += kThreads) hist[e] = 0;
    if (SELECT)
        for (int e = threadIdx.x; e < S::G * S::EL; e += kThreads) bias[e] = a.bias && e < E ? a.bias[e] + 0.0f : 0.0f;
    if (threadIdx.x == 0) ntokens = 0;
    __syncthreads();

    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int gl = lane % S::G, sub = lane / S::G;
    Slot* stage = reinterpret_cast<Slot*>(lds + bias_at(kColRows, E) + S::G * S::EL) + size_t(wave * S::RPW + sub) * k;
    float acc[S::EL];
#pragma unroll
    for (int j = 0; j < S::EL; ++j) acc[j] = 0.0f;
    int live_rows = 0;

    const int begin = int(blockIdx.x) * a.chunk_rows;
    const int end = min(begin + a.chunk_rows, a.N);
    const T* scores = static_cast<const T*>(a.scores) + int64_t(b) * a.sb;
    const int64_t row0 = int64_t(b) * a.N;

    RawRow<T, S> next;
    auto fetch = [&](int base) {
        const int n = base + sub;
        const bool live = n < end && (!a.mask || a.mask[row0 + n]);
        next.load(scores + int64_t(n) * a.sn, gl, E, live);
    };
    fetch(begin + wave * S::RPW);
    if constexpr (!SELECT) {
        const int64_t first = (row0 + begin) * k, count = int64_t(max(end - begin, 0)) * k;
        for (int64_t i = threadIdx.x; i < count; i += kThreads) {
            const int64_t e = int_at(a.given, a.given64, first + i);
            if (e >= 0 && e < E && (!a.mask || a.mask[(first + i) / k])) atomicAdd(&hist[e], 1);
        }
    }
    for (int base = begin + wave * S::RPW; base < end; base += kWaves * S::RPW) {
        const RawRow<T, S> raw = next;
        fetch(base + kWaves * S::RPW);
        const int n = base + sub;
        const bool in = n < end;
        live_rows += raw.live && gl == 0;
        float x[S::EL], q[S::EL], top, inv;
        raw.get(gl, E, x);
        // The shares are summed over many tokens into one fp32: the short exponential
        // (65536 x 256 fp32 without a selection 13.5 us, with the other 14.9).
        row_masses<S, false, false>(x, a.scoring, q, top, inv);
#pragma unroll
        for (int j = 0; j < S::EL; ++j) acc[j] = fmaf(q[j], inv, acc[j]);

        if constexpr (SELECT) {
            const T* row = scores + int64_t(n) * a.sn;
            select<T, S>(row, raw, bias, a.bias != nullptr, a.scoring == DOT_SCORING_PLAN, gl, E, k, stage);
            const bool soft = a.scoring == DOT_SCORING_SOFTMAX;
            const int64_t at = (row0 + n) * k;
            // The score of a slot's expert, which is counted.
            auto score = [&](int e) {
                if (e < 0) return kNegInf;
                atomicAdd(&hist[e], 1);
                return to_float(row[e]);
            };
            // A slot's mass: exp(s - top) or q(s); 0 for an empty one.
            auto mass = [&](int e, float s) {
                return e < 0 ? 0.0f : soft ? exp_of<true>(s - top) : mass_of(s, a.scoring);
            };
            // The largest selected score, from the lanes' largest.
            auto largest = [&](float s) {
                s = group_reduce<S::G>(s, OpMax{});
                top = s == kNegInf ? 0.0f : s;
            };
            // Weights: masses over the row's sum, or over that of the selected ones (a
            // division, so that a single expert's weight is 1 and its gradient 0; a
            // row with NaN has no softmax weights).
            float scale = soft ? inv : 1.0f, over = 1.0f;
            auto normalizer = [&](float z) {
                z = group_reduce<S::G>(z, OpSum{});
                over = fabsf(z) < FLT_MIN ? __builtin_inff() : z;
                scale = soft ? 1.0f + (inv - inv) : 1.0f;
            };
            if (k <= S::G) {  // a slot per lane
                const int e = gl < k ? stage[gl].e : -1;
                const float s = score(e);
                if (a.normalize && soft) largest(s);
                const float w = mass(e, s);
                if (a.normalize) normalizer(w);
                if (in && gl < k) {
                    a.weights[at + gl] = e < 0 ? 0.0f : w * scale / over;
                    a.experts[at + gl] = e;
                }
            } else {
                float most = kNegInf, z = 0.0f;
                for (int r = gl; r < k; r += S::G) {
                    const float s = score(stage[r].e);
                    stage[r].s = s;
                    most = fmaxf(most, s);
                }
                if (a.normalize && soft) largest(most);
                for (int r = gl; r < k; r += S::G) z += mass(stage[r].e, stage[r].s);
                if (a.normalize) normalizer(z);
                for (int r = gl; r < k; r += S::G) {
                    const Slot t = stage[r];
                    if (in) {
                        a.weights[at + r] = t.e < 0 ? 0.0f : mass(t.e, t.s) * scale / over;
                        a.experts[at + r] = t.e;
                    }
                }
            }
            wave_lds_fence();  // the next rows write the slots again
        }
    }

    // Column sums of this workgroup: over the rows of a wave, then over the waves in order.
#pragma unroll
    for (int j = 0; j < S::EL; ++j) acc[j] = across_groups<S::G>(acc[j]);
    if (live_rows) atomicAdd(&ntokens, live_rows);
    for (int w = 0; w < kWaves; w += kColRows) {
        if (wave >= w && wave < w + kColRows && sub == 0) {
#pragma unroll
            for (int j = 0; j < S::EL; ++j) {
                const int e = S::expert(gl, j);
                if (e < E) col[(wave - w) * E + e] = acc[j] + (w ? col[(wave - w) * E + e] : 0.0f);
            }
        }
        __syncthreads();
    }
    if constexpr (kColRows > 1) {
        for (int e = threadIdx.x; e < E; e += kThreads) {
            float s = col[e];
            for (int w = 1; w < kColRows; ++w) s += col[w * E + e];
            col[e] = s;
        }
        // the thread that adds up a column is the one that reads it below
    }
    if (a.nchunks == 1) {  // nothing to join
        double dot = 0.0;
        for (int e = threadIdx.x; e < E; e += kThreads) {
            a.counts[int64_t(b) * E + e] = hist[e];
            dot += double(col[e]) * hist[e];
        }
        dot = wave_sum_f64(dot);
        if (lane == 0) wdot[wave] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kWaves; ++w) dot += wdot[w];
            if (a.tokens) a.tokens[b] = ntokens;
            a.loss[b] = loss_value(dot, E, k, ntokens);
        }
        return;
    }
    const int64_t part = int64_t(b) * a.nchunks + blockIdx.x;
    for (int e = threadIdx.x; e < E; e += kThreads) {
        a.psum[part * E + e] = col[e];
        a.pcount[part * E + e] = hist[e];
    }
    if (threadIdx.x == 0) {
        a.ptokens[part] = ntokens;
        if (blockIdx.x == 0) a.done[b] = 0;
    }
}

constexpr int kFinishBlock = 1024, kFinishCols = 64, kSlices = kFinishBlock / kFinishCols;

struct FinishArgs {
    int B, E, k, nchunks;
    const float* psum;
    const int32_t* pcount;
    const int32_t* ptokens;
    double* dots;    // [B, gridDim.x]
    uint32_t* done;  // [B], 0
    int32_t* counts;
    int32_t* tokens;
    float* loss;
};

// Counts and loss of a batch element from its chunks' partials: kFinishCols
// experts per workgroup, whose shares of the loss the last workgroup of the
// element to arrive adds up in order.
__global__ __launch_bounds__(kFinishBlock) void finish(FinishArgs a) {
    __shared__ double sums[kSlices][kFinishCols];
    __shared__ int cnts[kSlices][kFinishCols];
    __shared__ int ntok[kFinishBlock / kWave];
    const int b = batch_of_block();
    if (b >= a.B) return;
    const int lane = threadIdx.x % kFinishCols, slice = threadIdx.x / kFinishCols;
    const int e = int(blockIdx.x) * kFinishCols + lane;
    const int64_t first = int64_t(b) * a.nchunks;
    double s = 0.0;
    int cnt = 0, n = 0;
    if (e < a.E) {
#pragma unroll 8
        for (int c = slice; c < a.nchunks; c += kSlices) {
            s += a.psum[(first + c) * a.E + e];
            cnt += a.pcount[(first + c) * a.E + e];
        }
    }
    for (int c = threadIdx.x; c < a.nchunks; c += kFinishBlock) n += a.ptokens[first + c];
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) n += __shfl_xor(n, d);
    sums[slice][lane] = s;
    cnts[slice][lane] = cnt;
    if (lane == 0) ntok[slice] = n;
    __syncthreads();
    if (slice != 0) return;
    for (int t = 1; t < kSlices; ++t) {
        s += sums[t][lane];
        cnt += cnts[t][lane];
        n += ntok[t];
    }
    if (e < a.E) a.counts[int64_t(b) * a.E + e] = cnt;
    double dot = wave_sum_f64(s * cnt);
    if (lane != 0) return;
    if (gridDim.x > 1) {
        double* dots = a.dots + int64_t(b) * gridDim.x;
        __hip_atomic_store(dots + blockIdx.x, dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const uint32_t before = __hip_atomic_fetch_add(a.done + b, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        if (before + 1 < gridDim.x) return;
        dot = 0.0;
        for (unsigned i = 0; i < gridDim.x; ++i)
            dot += __hip_atomic_load(dots + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (a.tokens) a.tokens[b] = n;
    a.loss[b] = loss_value(dot, a.E, a.k, n);
}
static_assert(kFinishCols == kWave, "a slice is one wave");

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
// The k values of a row go to their lanes through a zeroed row in LDS.  A lane of
// the widest shape (more than 2048 experts) holds 64 scores, shares, slopes and
// additions: with WEIGHTS and rows of any alignment that takes all 256 registers,
// and 57 (fp32) or 27 (16 bits) are spilled; no other instance spills.
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
    const double n_b = a.tokens ? a.tokens[b] : a.N;
    if (a.grad_loss && n_b > 0) {
        coef = double(a.grad_loss[a.grad_loss_scalar ? 0 : b]) * E / (double(k) * n_b * n_b);
        mean = double(k) * n_b / E;
    }
#pragma unroll
    for (int j = 0; j < S::EL; ++j) {
        const int e = S::expert(gl, j);
        slope[j] = (a.grad_loss && e < E) ? float(coef * (double(a.counts[int64_t(b) * E + e]) - mean)) : 0.0f;
    }

    const int begin = int(blockIdx.x) * a.chunk_rows;
    const int end = min(begin + a.chunk_rows, a.N);
    const T* scores = static_cast<const T*>(a.scores) + int64_t(b) * a.sb;
    // The next row: its scores, and the first of this lane's slots.
    struct Slot {
        int e;
        float w, dw;
    };
    auto slot = [&](int64_t at, int r, bool live) {
        Slot s{-1, 0.0f, 0.0f};
        if (live && r < k) {
            s.e = a.experts[at * k + r];
            s.dw = a.grad_weights[at * k + r];
            if (a.normalize) s.w = a.weights[at * k + r];
            if (unsigned(s.e) >= unsigned(E)) s = Slot{-1, 0.0f, 0.0f};
        }
        return s;
    };
    RawRow<T, S> next;
    Slot next_slot{};
    auto fetch = [&](int base) {
        const int n = base + sub;
        const int64_t at = int64_t(b) * a.N + n;
        const bool live = n < end && (!a.mask || a.mask[at]);
        next.load(scores + int64_t(n) * a.sn, gl, E, live);
        if constexpr (WEIGHTS) next_slot = slot(at, gl, live);
    };
    fetch(begin + wave * S::RPW);
    for (int base = begin + wave * S::RPW; base < end; base += kWavesPerBlock * S::RPW) {
        const RawRow<T, S> raw = next;
        const Slot first = next_slot;
        fetch(base + kWavesPerBlock * S::RPW);
        const int n = base + sub;
        const bool in = n < end, live = raw.live;
        const int64_t at = int64_t(b) * a.N + n;
        float x[S::EL], q[S::EL], top, inv;
        raw.get(gl, E, x);
        row_masses<S, sizeof(T) == 4, true>(x, a.scoring, q, top, inv);  // 16 bits hold less than either
        float add[S::EL];
#pragma unroll
        for (int j = 0; j < S::EL; ++j) add[j] = 0.0f;
        if constexpr (WEIGHTS) {
            float dot = 0.0f, over = 1.0f;
            if (a.normalize) {
                float mass = 0.0f;
                if (!soft) {  // the selected masses, from their lanes
#pragma unroll
                    for (int j = 0; j < S::EL; ++j) spread[S::expert(gl, j)] = q[j];
                    wave_lds_fence();
                }
                for (int r = gl; r < k; r += S::G) {
                    const Slot s = r == gl ? first : slot(at, r, live);
                    if (s.e < 0) continue;
                    dot = fmaf(s.w, s.dw, dot);
                    if (!soft) mass += spread[s.e];
                }
                dot = group_reduce<S::G>(dot, OpSum{});
                if (!soft) {
                    mass = group_reduce<S::G>(mass, OpSum{});
                    over = fabsf(mass) < FLT_MIN ? __builtin_inff() : mass;
                    wave_lds_fence();
                }
            }
#pragma unroll
            for (int j = 0; j < S::EL; ++j) spread[S::expert(gl, j)] = 0.0f;
            wave_lds_fence();
            for (int r = gl; r < k; r += S::G) {
                const Slot s = r == gl ? first : slot(at, r, live);
                if (s.e < 0) continue;
                const float v = s.dw - dot;
                spread[s.e] = !a.normalize ? s.dw : soft ? s.w * v : v / over;
            }
            wave_lds_fence();
#pragma unroll
            for (int j = 0; j < S::EL; ++j) add[j] = spread[S::expert(gl, j)];
            wave_lds_fence();
        }
        // The gradient takes the place of the shares.
        float ph = 0.0f;
#pragma unroll
        for (int j = 0; j < S::EL; ++j) q[j] *= inv;
        if (WEIGHTS && soft && !a.normalize) {  // the weights are p itself: add belongs to h
#pragma unroll
            for (int j = 0; j < S::EL; ++j) {
                add[j] += slope[j];
                ph = fmaf(q[j], add[j], ph);
            }
            ph = group_reduce<S::G>(ph, OpSum{});
#pragma unroll
            for (int j = 0; j < S::EL; ++j) q[j] *= add[j] - ph;
        } else {
#pragma unroll
            for (int j = 0; j < S::EL; ++j) ph = fmaf(q[j], slope[j], ph);
            ph = group_reduce<S::G>(ph, OpSum{});
            if (soft) {
#pragma unroll
                for (int j = 0; j < S::EL; ++j) q[j] = fmaf(q[j], slope[j] - ph, add[j]);
            } else {
#pragma unroll
                for (int j = 0; j < S::EL; ++j) q[j] = fmaf(slope[j] - ph, inv, add[j]) * x[j];
            }
        }
#pragma unroll
        for (int j = 0; j < S::EL; ++j) q[j] = live ? q[j] : 0.0f;
        if (in) store_row<T, S>(static_cast<T*>(a.grad_scores) + at * E, gl, E, q);
    }
}

inline size_t bwd_lds_bytes(int lanes_elems, bool weights) {
    return weights ? size_t(kWavesPerBlock) * size_t(lanes_elems) * sizeof(float) : 0;
}

}  // namespace routing
}  // namespace dot_amd
