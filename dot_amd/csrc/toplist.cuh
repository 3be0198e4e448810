// The largest logits of rows over a vocabulary, and what is built on them: the
// top log-probabilities of positions and the step of a beam search.
//
// scan: a workgroup holds a span of a row in registers (64 KB at most, 16 packs a
// thread), so that maximum, sum of exponentials and selection take one read.  It
// writes the span's n largest logits in order (a list), its maximum m and
// s = sum_v 2^((x_v - m) k), k = log2(e) / tau.  Packs are dealt to threads by their
// place in the row, not by their address: equal rows have equal sums, bit for bit,
// wherever they lie, and beams that tie stay tied.
//
// join: the lists of a row's spans, or of all beams of a batch element, in one list.
// Keys are 64-bit: the logit itself, or the hypothesis's total score.
//
// An entry is ordered by its value (descending), equal ones by their index
// (ascending).  -inf and NaN are never selected.
#pragma once

#include "elem.cuh"
#include "row.cuh"
#include "wave.cuh"

namespace dot_amd {
namespace toplist {

constexpr int kMaxPacks = 16;  // packs of a thread

struct Rows {
    const void* logits;  // row (o, i) at o * so + i * si elements
    int64_t so, si;
    int inner;           // rows per o
    int rows, V;
    // Rows that are not read: those with 0 in `mask`, with a score of -inf, or finished.
    const uint8_t* mask;
    const float* scores;
    const uint8_t* finished;
    float inv_tau;
    float k;             // log2(e) times it
    int n;               // entries of a list
    int parts, per;      // spans of a row, packs of a span
};

struct Part {
    double s;
    float m;
};

// What the scan leaves for the join: [rows, parts] statistics, [rows, parts, n] entries.
struct Lists {
    Part* parts;
    float* value;
    int32_t* token;
};

__device__ __forceinline__ bool read_row(const Rows& r, int row) {
    return !(r.mask && !r.mask[row]) && !(r.scores && !(r.scores[row] > -__builtin_inff())) &&
           !(r.finished && r.finished[row]);
}

template <class T>
__device__ __forceinline__ const T* row_of(const Rows& r, int row) {
    const int o = row / r.inner, i = row - o * r.inner;
    return static_cast<const T*>(r.logits) + int64_t(o) * r.so + int64_t(i) * r.si;
}

// 16 bytes from an address that is aligned to an element only.
template <class T>
__device__ __forceinline__ Pack<T> load_pack_any(const T* p) {
    Pack<T> x;
    __builtin_memcpy(&x, p, sizeof(x));
    return x;
}

__device__ __forceinline__ float minus_inf(float) { return -__builtin_inff(); }
__device__ __forceinline__ F16 minus_inf(F16) { return F16{0xFC00}; }
__device__ __forceinline__ BF16 minus_inf(BF16) { return BF16{0xFF80}; }

// Floats in an order of unsigned integers (of -0 and 0, which are equal, callers add 0 first).
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __builtin_bit_cast(float, o ^ (o & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu));
}

// An entry as one key: larger is better.
__device__ __forceinline__ uint64_t entry_of(float x, int index) {
    return uint64_t(order_of(x + 0.0f)) << 32 | uint32_t(~index);
}

// Sum of N values, pairwise.
template <int N>
__device__ __forceinline__ float pairwise(const float* x) {
    if constexpr (N == 1) return x[0];
    else return pairwise<N / 2>(x) + pairwise<N - N / 2>(x + N / 2);
}

// Sum over the workgroup of a count that is uniform in each wave; `sh` alternates
// between two sets so that one barrier is enough.
__device__ __forceinline__ int block_count(int c, int (&sh)[2][kWavesPerBlock], int& turn) {
    int (&s)[kWavesPerBlock] = sh[turn];
    turn ^= 1;
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = c;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kWavesPerBlock; ++w) sum += s[w];
    return sum;
}

// x / tau - m / tau as a program has it that scales its logits in fp32 and then takes
// its differences (rounded twice, 2^-24 of the logits each), so that what is next to
// a border here is so there; in 64 bits where fp32 ends.
__device__ __forceinline__ double share_of(const Rows& r, float x, float m) {
    const float d = __fsub_rn(__fmul_rn(x, r.inv_tau), __fmul_rn(m, r.inv_tau));
    return fabsf(d) < __builtin_inff() ? double(d) : (double(x) - double(m)) * double(r.inv_tau);
}

struct TopOut {
    float* logp;      // [rows, n]
    int32_t* token;   // [rows, n]
};

// One span of a row.  DIRECT: the row is one span, and its list the output.
template <class T, int P, bool DIRECT>
__global__ __launch_bounds__(kBlock) void scan(Rows r, Lists lists, TopOut out) {
    constexpr int PN = Pack<T>::N, NE = P * PN;
    __shared__ uint64_t found[DOT_TOP_MAX];
    __shared__ int counts[2][kWavesPerBlock];
    __shared__ float wm[kWavesPerBlock];
    __shared__ double ws[kWavesPerBlock];
    __shared__ int places;
    int turn = 0;
    const int row = batch_of_block(), part = int(blockIdx.x);
    if (row >= r.rows) return;
    if (!read_row(r, row)) {
        if (DIRECT)
            for (int e = threadIdx.x; e < r.n; e += kBlock) {
                out.logp[int64_t(row) * r.n + e] = -__builtin_inff();
                out.token[int64_t(row) * r.n + e] = -1;
            }
        return;
    }
    const T* x0 = row_of<T>(r, row);
    const int p0 = part * r.per, whole = r.V / PN;
    const int p1 = min(p0 + r.per, (r.V + PN - 1) / PN);
    Pack<T> x[P];
#pragma unroll
    for (int u = 0; u < P; ++u) {
        const int p = p0 + u * kBlock + int(threadIdx.x);
        if (p < min(p1, whole)) {
            x[u] = load_pack_any(x0 + int64_t(p) * PN);
        } else {
#pragma unroll
            for (int i = 0; i < PN; ++i) {
                const int v = p * PN + i;
                x[u].v[i] = minus_inf(T{});
                if (p < p1 && v < r.V) x[u].v[i] = x0[v];
            }
        }
    }
    if (threadIdx.x == 0) places = 0;
    float m = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < NE; ++e) m = fmaxf(m, to_float(x[e / PN].v[e % PN]));
    m = wave_max(m);
    if (threadIdx.x % kWave == 0) wm[threadIdx.x / kWave] = m;
    __syncthreads();
    m = wm[0];
    for (int w = 1; w < kWavesPerBlock; ++w) m = fmaxf(m, wm[w]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    double s = 0.0;
#pragma unroll
    for (int u = 0; u < P; ++u) {
        float e[PN];
#pragma unroll
        for (int i = 0; i < PN; ++i) e[i] = __builtin_amdgcn_exp2f((to_float(x[u].v[i]) - base) * r.k);
        s += double(pairwise<PN>(e));
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) s += __shfl_xor(s, d);
    if (threadIdx.x % kWave == 0) ws[threadIdx.x / kWave] = s;

    // Entries of the span that `is` holds for.
    auto count = [&](auto is) {
        int c = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int v = (p0 + (e / PN) * kBlock + int(threadIdx.x)) * PN + e % PN;
            c += __builtin_popcountll(__ballot(is(to_float(x[e / PN].v[e % PN]), v)));
        }
        return block_count(c, counts, turn);
    };
    const float lowest = -__FLT_MAX__;
    const int want = min(r.n, count([&](float f, int) { return f >= lowest; }));
    float least = __builtin_inff();
    int last = -1;
    if (want > 0) {
        // the want-th largest value
        uint32_t lo = order_of(lowest), hi = order_of(m + 0.0f) + 1;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const float t = value_of(mid);
            if (count([&](float f, int) { return f >= t; }) >= want) lo = mid;
            else hi = mid;
        }
        least = value_of(lo);
        // and the last index of those equal to it
        const int equal = want - count([&](float f, int) { return f > least; });
        int below = p0 * PN - 1;
        last = min(p1 * PN, r.V) - 1;
        while (last - below > 1) {
            const int mid = below + (last - below) / 2;
            if (count([&](float f, int v) { return f == least && v <= mid; }) >= equal) last = mid;
            else below = mid;
        }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const float f = to_float(x[e / PN].v[e % PN]);
        const int v = (p0 + (e / PN) * kBlock + int(threadIdx.x)) * PN + e % PN;
        if (f > least || (f == least && v <= last)) found[atomicAdd(&places, 1)] = entry_of(f, v);
    }
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kWavesPerBlock; ++w) total += ws[w];
    const int64_t list = DIRECT ? int64_t(row) : int64_t(row) * r.parts + part;
    if (!DIRECT && threadIdx.x == 0) lists.parts[list] = Part{total, base};
    const double shift = DIRECT ? log(total) : 0.0;
    for (int c = threadIdx.x; c < r.n; c += kBlock) {
        if (c < want) {
            const uint64_t mine = found[c];
            int rank = 0;
            for (int j = 0; j < want; ++j) rank += found[j] > mine;
            const float f = value_of(uint32_t(mine >> 32));
            const int v = int(~uint32_t(mine));
            if (DIRECT) {
                out.logp[list * r.n + rank] = float(share_of(r, f, base) - shift);
                out.token[list * r.n + rank] = v;
            } else {
                lists.value[list * r.n + rank] = f;
                lists.token[list * r.n + rank] = v;
            }
        } else if (DIRECT) {
            out.logp[list * r.n + c] = -__builtin_inff();
            out.token[list * r.n + c] = -1;
        } else {
            lists.value[list * r.n + c] = -__builtin_inff();
            lists.token[list * r.n + c] = -1;
        }
    }
}

// ---------------------------------------------------------------------------
// Lists in one
// ---------------------------------------------------------------------------
// An entry of a list under its 64-bit key; `id` is its place among the lists.
// Larger keys first, equal ones by their place.
struct Entry {
    double key;
    int id;
};
__device__ __forceinline__ Entry nothing() { return Entry{-__builtin_inf(), 0x7FFFFFFF}; }
__device__ __forceinline__ bool before(const Entry& a, const Entry& b) {
    return a.key > b.key || (a.key == b.key && a.id < b.id);
}
__device__ __forceinline__ Entry shuffle(const Entry& a, int mask) {
    return Entry{__shfl_xor(a.key, mask), __shfl_xor(a.id, mask)};
}

// A wave's 64 R best entries in order: entry r * 64 + lane in e[r].
template <int R>
struct Best {
    static constexpr int N = R * kWave;
    Entry e[R];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r) e[r] = nothing();
    }
    // The best N of these and of an ordered list whose entries lie reversed: other[r] is
    // entry N - 1 - (r * 64 + lane).  The better ones of each pair are a bitonic sequence.
    __device__ __forceinline__ void merge(const Entry (&other)[R]) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (before(other[r], e[r])) e[r] = other[r];
#pragma unroll
        for (int d = R / 2; d >= 1; d /= 2)
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (!(r & d) && before(e[r | d], e[r])) {
                    const Entry t = e[r];
                    e[r] = e[r | d];
                    e[r | d] = t;
                }
        const int lane = int(threadIdx.x) % kWave;
#pragma unroll
        for (int d = kWave / 2; d >= 1; d /= 2)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const Entry o = shuffle(e[r], d);
                if (before(o, e[r]) == !(lane & d)) e[r] = o;
            }
    }
};

struct JoinArgs {
    int eos;               // token of a finished hypothesis, or -1
    float* scores;         // [B, n] of a beam step
    int32_t* beams;
    int32_t* tokens;       // [B, n], or [rows, n] of top log-probabilities (their values in `scores`)
    uint8_t* finished;     // or NULL
};

// The lists of `lists_of` spans (BEAM: of all spans of a batch element's beams) in one.
template <int R, bool BEAM>
__global__ void join(Rows r, Lists lists, JoinArgs a) {
    extern __shared__ char shared[];
    constexpr int N = R * kWave;
    const int b = batch_of_block();
    const int beams = BEAM ? r.inner : 1;
    if (b >= r.rows / beams) return;
    const int waves = int(blockDim.x) / kWave, wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    Entry* held = reinterpret_cast<Entry*>(shared);                           // [waves / 2][N]
    double* shift = reinterpret_cast<double*>(held + max(waves / 2, 1) * N);  // [beams]: what a logit's share lacks
    float* top = reinterpret_cast<float*>(shift + beams);                     // [beams]: the largest logit
    int* kind = reinterpret_cast<int*>(top + beams);                          // [beams]: 0 no entries, 1 lists, 2 itself
    const double kn = double(r.k) * 0.693147180559945309417;
    for (int w = threadIdx.x; w < beams; w += blockDim.x) {
        const int row = b * beams + w;
        const bool read = read_row(r, row);
        float m = -__builtin_inff();
        double s = 0.0;
        if (read) {
            bool any = false;
            for (int p = 0; p < r.parts; ++p) {
                const Part q = lists.parts[int64_t(row) * r.parts + p];
                // a span of nothing but -inf has a sum of 0
                if (q.s == 0.0) continue;
                m = any ? fmaxf(m, q.m) : q.m;
                any = true;
            }
            for (int p = 0; p < r.parts; ++p) {
                const Part q = lists.parts[int64_t(row) * r.parts + p];
                if (q.s != 0.0) s += q.s * exp((double(q.m) - double(m)) * kn);
            }
        }
        const float score = BEAM ? r.scores[row] : 0.0f;
        top[w] = m;
        shift[w] = (BEAM ? double(score) : 0.0) - log(s);
        kind[w] = read ? 1 : BEAM && r.finished && r.finished[row] && score > -__builtin_inff() ? 2 : 0;
    }
    __syncthreads();
    Best<R> best;
    best.clear();
    const int count = beams * r.parts;
    for (int l = wave; l < count; l += waves) {
        const int w = BEAM ? l / r.parts : 0;
        if (kind[w] == 0 || (kind[w] == 2 && l != w * r.parts)) continue;
        const int64_t list = int64_t(b) * count + l;
        Entry other[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int at = N - 1 - (i * kWave + lane);
            other[i] = nothing();
            if (kind[w] == 2) {
                if (at == 0) other[i] = Entry{double(r.scores[b * beams + w]), l * r.n};
            } else if (at < r.n) {
                const float f = lists.value[list * r.n + at];
                const double key = BEAM ? shift[w] + share_of(r, f, top[w]) : double(f);
                if (key > -__builtin_inf()) other[i] = Entry{key, l * r.n + at};
            }
        }
        best.merge(other);
    }
    for (int half = waves / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int i = 0; i < R; ++i) held[(wave - half) * N + i * kWave + lane] = best.e[i];
        __syncthreads();
        if (wave < half) {
            Entry other[R];
#pragma unroll
            for (int i = 0; i < R; ++i) other[i] = held[wave * N + N - 1 - (i * kWave + lane)];
            best.merge(other);
        }
    }
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int e = i * kWave + lane;
        if (e >= r.n) continue;
        const int64_t to = int64_t(b) * r.n + e;
        const Entry x = best.e[i];
        if (x.id == 0x7FFFFFFF) {
            a.scores[to] = -__builtin_inff();
            a.tokens[to] = -1;
            if (BEAM) a.beams[to] = -1;
            if (BEAM && a.finished) a.finished[to] = 0;
            continue;
        }
        const int l = x.id / r.n, w = BEAM ? l / r.parts : 0;
        const bool itself = BEAM && kind[w] == 2;
        const int token = itself ? a.eos : lists.token[int64_t(b) * count * r.n + x.id];
        a.tokens[to] = token;
        if (BEAM) {
            a.scores[to] = float(x.key);
            a.beams[to] = w;
            if (a.finished) a.finished[to] = itself || token == a.eos;
        } else {
            a.scores[to] = float(share_of(r, float(x.key), top[0]) + shift[0]);
        }
    }
}

}  // namespace toplist
}  // namespace dot_amd
