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
//
// The logits are read once; everything else is small next to them (4096 x 131072 bf16
// and 64 entries: 1.07 GB of logits, 4 MB of entries).  4096 x 131072 bf16 takes 191 us in
// the scan, 5.6 TB/s, and 20 us in the join.
#pragma once

#include <type_traits>

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
    // log2(e) times it, in one float: off by 6e-8 of itself at most, and a sum by that share of
    // E[(m - x) / tau], less than its shares of a logit scaled in fp32 are.  A second float for the
    // rest brought the log-probabilities no nearer (999 x 50021 fp32, 128 entries: 5.0e-7 off in the
    // mean square, with one float 4.7e-7; the exponential's own error is left) and cost 4 %
    // (4096 x 131072 bf16 222 us, with one 213).
    float k;
    int n;               // entries of a list
    int parts, per;      // spans of a row, packs of a span
};

struct Part {
    double s;
    float m;
};

// What the scan leaves for the join: [rows, parts] statistics, [rows, parts, n] entries.
struct Item {
    float x;    // -inf: none
    int token;
};
struct Lists {
    Part* parts;
    Item* items;
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

// A pack of -inf.
template <class T>
__device__ __forceinline__ Pack<T> nothing_pack() {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const uint32_t w = std::is_same_v<T, float> ? 0xFF800000u : std::is_same_v<T, F16> ? 0xFC00FC00u : 0xFF80FF80u;
    return __builtin_bit_cast(Pack<T>, u4{w, w, w, w});
}

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
#pragma clang fp contract(off)
    const float zx = x * r.inv_tau, zm = m * r.inv_tau;
    const float d = zx - zm;
    return fabsf(d) < __builtin_inff() ? double(d) : (double(x) - double(m)) * double(r.inv_tau);
}

struct TopOut {
    float* logp;      // [rows, n]
    int32_t* token;   // [rows, n]
};

// A value that at least `r` of the wave's G * 64 values reach, and few more: the r-th
// largest to within an eighth of r, by bisection with ballots.  Where fewer than r are
// above -inf: the lowest finite value.
template <int G>
__device__ __forceinline__ float reached_by(const float (&v)[G], int r) {
    const float lowest = -__FLT_MAX__;
    auto count = [&](float t) {
        int c = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) c += __builtin_popcountll(__ballot(v[g] >= t));
        return c;
    };
    float most = v[0], least = __builtin_inff();
#pragma unroll
    for (int g = 0; g < G; ++g) {
        most = fmaxf(most, v[g]);
        if (v[g] >= lowest) least = fminf(least, v[g]);
    }
    most = wave_max(most);
    least = wave_reduce(least, [](float a, float b) { return fminf(a, b); });
    if (count(lowest) < r) return lowest;
    uint32_t lo = order_of(least + 0.0f), hi = order_of(most + 0.0f) + 1;
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const int c = count(value_of(mid));
        if (c >= r) lo = mid;
        else hi = mid;
        if (c >= r && c <= r + r / 8) break;
    }
    return value_of(lo);
}

// One span of a row.  DIRECT: the row is one span, and its list the output.
//
// Each wave finds a value that its share of the n entries reaches, from the maxima of
// its lanes (of parts of them where its share is above a quarter of its lanes); the
// lowest of the four values is reached by n entries of the span at least, and by few more
// on logits in no particular order.
// Those are collected, each wave in a place of its own, and ranked by counting.  Where
// they are too many (ties, orders in which the largest lie in few lanes), the n-th
// largest entry is found by bisection over all of them instead.
//
// Bound by HBM where there are many spans; where they are few, by one workgroup's way
// through its phases: 8 rows of 32768 bf16, 20 entries, 8.6 us, of which the loads are
// half; 240 rows of 50021 fp32 in 4 spans, 96 entries, 17.4 us for 48 MB.  16 packs a
// thread, not 8: half the lists for the join, and 4096 x 131072 bf16 took 297 us with 8
// where 16 took 219.
template <class T, int P, bool DIRECT>
__global__ __launch_bounds__(kBlock, 4) void scan(Rows r, Lists lists, TopOut out) {
    constexpr int PN = Pack<T>::N;
    constexpr int LONG = 64;   // entries of a list above which the waves' are put in order first
    constexpr int G = 4;       // values of a lane to find what is reached, where one is too few
    constexpr int ROOM = 512;  // entries that a wave collects
    constexpr int STEP = 8;
    constexpr int HELD = 204;  // packs that a wave looks into: for 256 entries 128 are too few now and then
    __shared__ uint64_t found[kWavesPerBlock][ROOM + STEP];
    // a wave's packs, and when it is through with them its entries in order
    __shared__ union {
        struct {
            Pack<T> packs[HELD];
            int places[HELD];
        };
        uint64_t sorted[ROOM];
    } own[kWavesPerBlock] __attribute__((aligned(16)));
    __shared__ int counts[2][kWavesPerBlock];
    __shared__ float wm[kWavesPerBlock], wt[kWavesPerBlock];
    __shared__ double ws[kWavesPerBlock], wo[kWavesPerBlock];
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
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    const T* x0 = row_of<T>(r, row);
    const int p0 = part * r.per, whole = r.V / PN;
    const int p1 = min(p0 + r.per, (r.V + PN - 1) / PN);
    Pack<T> x[P];
    const int end = min(p1, whole);
    if (end - p0 >= P * kBlock) {
        const T* from = x0 + int64_t(p0) * PN;  // uniform: one 32-bit offset a load
#pragma unroll
        for (int u = 0; u < P; ++u) x[u] = load_pack_any(from + (unsigned(u) * kBlock + threadIdx.x) * unsigned(PN));
    } else if (end > p0) {
        // packs past the span are the last whole one (a cache hit), then nothing
#pragma unroll
        for (int u = 0; u < P; ++u)
            x[u] = load_pack_any(x0 + int64_t(min(p0 + u * kBlock + int(threadIdx.x), end - 1)) * PN);
    }
    if (end - p0 < P * kBlock) {
#pragma unroll
        for (int u = 0; u < P; ++u)
            if (p0 + u * kBlock + int(threadIdx.x) >= end) x[u] = nothing_pack<T>();
        if (p1 > whole) {  // the row's last elements
            Pack<T> last = nothing_pack<T>();
#pragma unroll
            for (int i = 0; i < PN; ++i)
                if (whole * PN + i < r.V) last.v[i] = x0[whole * PN + i];
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (p0 + u * kBlock + int(threadIdx.x) == whole) x[u] = last;
        }
    }
    // Maxima and terms in one pass.  The terms are relative to the largest logit of the
    // wave's first packs: it is near the largest of all, or the sum is formed again below.
    // x k - m k takes one rounding where m k has digits behind the point.  Behind packs of
    // nothing but -inf the terms are relative to 1: as long as the largest is within 2^32
    // of that, rounding x k costs 2^-24 of 22 at most, and no term that counts is below the
    // smallest float (a row's largest logit at -69 and many 20 below it: 2e-5 of the sum were).
    // Past that the sum is formed again too: 1024 x 131072 bf16 62 us, then 104.
    float pm[P];  // the largest logit of each pack
    float m = -__builtin_inff(), mk = 0.0f;
    float reach = 100.0f;
    bool near = true;
    double s = 0.0;
#pragma unroll
    for (int u = 0; u < P; ++u) {
        if (u > P / 2 && u * kBlock >= p1 - p0) {  // nothing but -inf
            pm[u] = -__builtin_inff();
            continue;
        }
        float f[PN];
#pragma unroll
        for (int i = 0; i < PN; ++i) f[i] = to_float(x[u].v[i]);
        pm[u] = f[0];
#pragma unroll
        for (int i = 1; i < PN; ++i) pm[u] = fmaxf(pm[u], f[i]);
        m = fmaxf(m, pm[u]);
        if (u == 0) {
            const float first = wave_max(m);
            mk = first == -__builtin_inff() ? 0.0f : first * r.k;
            if (first == -__builtin_inff()) reach = 32.0f;
            near = fabsf(mk) < 65536.0f;
            if (!near) mk = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < PN; ++i) f[i] = __builtin_amdgcn_exp2f(fmaf(f[i], r.k, -mk));
        s += double(pairwise<PN>(f));
    }
    // The wave's share of the n entries, by what it has of the span's elements (16 rows of
    // 2050 bf16 in 2 spans, 16 entries: 5.6 us, by equal shares 93, nearly all being ranked).
    // A wave of a few packs beside full ones has none: the largest of so few is often small.
    int np = p1 - p0, elements = min(p1 * PN, r.V) - p0 * PN;
    if (np > kWave && np < kBlock && np % kWave > 0 && np % kWave < kWave / 4) {
        np -= np % kWave;
        elements = np * PN;
    }
    const int at_wave = __builtin_amdgcn_readfirstlane(wave);
    const int has = np / kBlock * kWave + min(max(np % kBlock - at_wave * kWave, 0), kWave);
    const int missing = (np - 1) % kBlock / kWave == at_wave ? np * PN - elements : 0;  // of the last pack
    const int share = (r.n * (has * PN - missing) + elements - 1) / elements;
    float least;
    if (has == 0) {
        least = __builtin_inff();
    } else if (share * 4 <= min(has, kWave)) {
        const float v[1] = {m};
        least = reached_by(v, share);
    } else {
        float v[G];
        if constexpr (P <= 2) {
#pragma unroll
            for (int g = 0; g < G; ++g) v[g] = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < P; ++u)
#pragma unroll
                for (int i = 0; i < PN; ++i) {
                    const int g = i % (G / P) * P + u;
                    v[g] = fmaxf(v[g], to_float(x[u].v[i]));
                }
        } else {
#pragma unroll
            for (int u = 0; u < P; ++u) v[u % G] = u < G ? pm[u] : fmaxf(v[u % G], pm[u]);
        }
        least = reached_by(v, share);
    }
    // The span again from the caches, for what is rare.  All lanes of a wave go round
    // together: `use` may hold ballots.
    auto each = [&](auto use) {
        for (int p = p0; p < p1; p += kBlock) {
            const int mine = p + int(threadIdx.x);
            Pack<T> y;
            if (mine < end) y = load_pack_any(x0 + int64_t(mine) * PN);
            for (int i = 0; i < PN; ++i) {
                const int v = mine * PN + i;
                float f = -__builtin_inff();
                if (mine < end) f = to_float(y.v[i]);
                else if (mine < p1 && v < r.V) f = to_float(x0[v]);
                use(f, v);
            }
        }
    };
    m = wave_max(m);
    // what the wave's terms are relative to, as a binary logarithm
    double of = double(mk);
    if (m > -__builtin_inff() && !(near && fabsf(m * r.k - mk) < reach)) {
        s = 0.0;
        of = double(m) * double(r.k);
        each([&](float f, int) { s += double(__builtin_amdgcn_exp2f((f - m) * r.k)); });
    }
    s = wave_sum64(s);
    if (lane == 0) {
        wm[wave] = m;
        wt[wave] = least;
        ws[wave] = s;
        wo[wave] = of;
    }
    __syncthreads();
    m = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    least = fminf(fminf(wt[0], wt[1]), fminf(wt[2], wt[3]));
    const float base = m == -__builtin_inff() ? 0.0f : m;

    // Entries of -inf and NaN are below `least`.  Each wave's go to a place of its own:
    // first the packs that hold any, then, a lane an element, what is in them.
    int found_here = 0;
    auto put = [&](float f, int v, bool in) {
        const uint64_t all = __ballot(in);
        if (all == 0) return;
        const int at = found_here + __builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0));
        if (in && at < ROOM) found[wave][at] = entry_of(f, v);
        found_here += __builtin_popcountll(all);
    };
    int held = 0;
#pragma unroll
    for (int u = 0; u < P; ++u) {
        const bool in = pm[u] >= least;
        const uint64_t all = __ballot(in);
        if (all == 0) continue;
        const int at = held + __builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0));
        if (in && at < HELD) {
            own[wave].packs[at] = x[u];
            own[wave].places[at] = p0 + u * kBlock + int(threadIdx.x);
        }
        held += __builtin_popcountll(all);
    }
    wave_lds_fence();
    for (int j = lane; j - lane < min(held, HELD) * PN; j += kWave) {
        const bool in = j < held * PN;
        const int c = min(j / PN, min(held, HELD) - 1);
        const float f = to_float(own[wave].packs[c].v[j % PN]);
        put(f, own[wave].places[c] * PN + j % PN, in && f >= least);
    }
    if (held > HELD) found_here = ROOM + 1;
    auto ready = [&] {
        if (lane == 0) counts[0][wave] = found_here;
        if (lane < STEP) found[wave][min(found_here, ROOM) + lane] = 0;
    };
    ready();
    __syncthreads();
    int most = counts[0][0];
    for (int w = 1; w < kWavesPerBlock; ++w) most = max(most, counts[0][w]);
    if (most > ROOM) {
        int turn = 1;
        auto count = [&](auto is) {
            int c = 0;
            each([&](float f, int v) { c += __builtin_popcountll(__ballot(is(f, v))); });
            return block_count(c, counts, turn);
        };
        // the want-th largest value, of those that `least` let through
        const int want = min(r.n, count([&](float f, int) { return f >= least; }));
        uint32_t lo = order_of(least + 0.0f), hi = order_of(m + 0.0f) + 1;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const float t = value_of(mid);
            if (count([&](float f, int) { return f >= t; }) >= want) lo = mid;
            else hi = mid;
        }
        const float value = value_of(lo);
        // and the last index of those equal to it
        const int equal = want - count([&](float f, int) { return f > value; });
        int below = p0 * PN - 1, last = min(p1 * PN, r.V) - 1;
        while (last - below > 1) {
            const int mid = below + (last - below) / 2;
            if (count([&](float f, int v) { return f == value && v <= mid; }) >= equal) last = mid;
            else below = mid;
        }
        found_here = 0;
        each([&](float f, int v) { put(f, v, f > value || (f == value && v <= last)); });
        __syncthreads();
        ready();
        __syncthreads();
    }
    const int64_t list = DIRECT ? int64_t(row) : int64_t(row) * r.parts + part;
    // the waves' sums relative to the largest logit, a lane of a quad a wave's
    double z = ws[lane % 4];
    if (z != 0.0) z *= short_exp((wo[lane % 4] - double(base) * double(r.k)) * 0.693147180559945309417);
    z += dpp_move<kDppQuadXor1>(z);
    z += dpp_move<kDppQuadXor2>(z);
    if (!DIRECT && threadIdx.x == 0) lists.parts[list] = Part{z, base};
    const double shift = DIRECT ? short_log(z) : 0.0;
    auto write = [&](int rank, uint64_t entry) {
        const float f = value_of(uint32_t(entry >> 32));
        const int v = int(~uint32_t(entry));
        if (DIRECT) {
            out.logp[list * r.n + rank] = float(share_of(r, f, base) - shift);
            out.token[list * r.n + rank] = v;
        } else {
            lists.items[list * r.n + rank] = Item{f, v};
        }
    };
    int total = 0, longest = 0;
    for (int w = 0; w < kWavesPerBlock; ++w) {
        total += counts[0][w];
        longest = max(longest, counts[0][w]);
    }
    // How many of found[w] are better than an entry (they end in zeros, below any entry, up
    // to a whole step).
    auto better = [&](int w, uint64_t mine) {
        int n = 0;
        for (int j = 0; j < counts[0][w]; j += STEP) {
            uint64_t other[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) other[i] = found[w][j + i];
#pragma unroll
            for (int i = 0; i < STEP; ++i) n += other[i] > mine;
        }
        return n;
    };
    // Short lists: a quad counts for an entry, each lane among one wave's.  Long ones: each
    // wave orders its own by counting, then finds each one's place among the others' by
    // halving.  550 x 50021 fp32, n 20: 26.9 and 28.5 us, n 128: 49.9 and 38.8;
    // 2200 x 65536, n 64: 108 and 111.
    if (r.n <= LONG) {
        for (int c = int(threadIdx.x) / 4; c < total; c += kBlock / 4) {
            int w = 0, at = c;
#pragma unroll
            for (int i = 0; i < kWavesPerBlock - 1; ++i)
                if (w == i && at >= counts[0][i]) {
                    at -= counts[0][i];
                    ++w;
                }
            const uint64_t mine = found[w][at];
            int rank = better(int(threadIdx.x) % 4, mine);
            rank += __builtin_amdgcn_update_dpp(0, rank, kDppQuadXor1, 0xF, 0xF, false);
            rank += __builtin_amdgcn_update_dpp(0, rank, kDppQuadXor2, 0xF, 0xF, false);
            if (threadIdx.x % 4 == 0 && rank < r.n) write(rank, mine);
        }
    } else {
        for (int c = lane; c < found_here; c += kWave) {
            const uint64_t mine = found[wave][c];
            own[wave].sorted[better(wave, mine)] = mine;
        }
        __syncthreads();
        const int half = longest > 0 ? 1 << (31 - __builtin_clz(longest)) : 0;
        for (int c = lane; c < min(found_here, r.n); c += kWave) {
            const uint64_t mine = own[wave].sorted[c];
            int before[kWavesPerBlock - 1] = {};
            for (int step = half; step > 0; step /= 2)
#pragma unroll
                for (int i = 0; i < kWavesPerBlock - 1; ++i) {
                    const int w = (wave + 1 + i) % kWavesPerBlock, to = before[i] + step;
                    if (to <= counts[0][w] && own[w].sorted[to - 1] > mine) before[i] = to;
                }
            const int rank = c + before[0] + before[1] + before[2];
            if (rank < r.n) write(rank, mine);
        }
    }
    for (int c = total + int(threadIdx.x); c < r.n; c += kBlock) {
        if (DIRECT) {
            out.logp[list * r.n + c] = -__builtin_inff();
            out.token[list * r.n + c] = -1;
        } else {
            lists.items[list * r.n + c] = Item{-__builtin_inff(), -1};
        }
    }
}

// ---------------------------------------------------------------------------
// Lists in one
// ---------------------------------------------------------------------------
// An entry of a list: its key, and what orders equal ones: the beam, then the logit,
// then the place among the lists (which ascends with the token among equal logits).
// Larger is better in both; no entry has a key of 0.
struct Entry {
    uint64_t key, tie;
};
constexpr int kPlaceBits = 25;  // beams * spans * entries: 2^7 * 2^10 * 2^8
__device__ __forceinline__ uint64_t tie_of(int beam, float x, int place) {
    return uint64_t(DOT_BEAM_MAX - 1 - beam) << (32 + kPlaceBits) | uint64_t(order_of(x)) << kPlaceBits |
           uint64_t((1 << kPlaceBits) - 1 - place);
}
__device__ __forceinline__ int place_of(uint64_t tie) {
    return (1 << kPlaceBits) - 1 - int(tie & ((1u << kPlaceBits) - 1));
}
__device__ __forceinline__ Entry nothing() { return Entry{0, 0}; }
__device__ __forceinline__ bool before(const Entry& a, const Entry& b) {
    return a.key > b.key || (a.key == b.key && a.tie > b.tie);
}
__device__ __forceinline__ uint64_t shuffle(uint64_t x, int mask) {
    const uint32_t lo = __shfl_xor(uint32_t(x), mask), hi = __shfl_xor(uint32_t(x >> 32), mask);
    return uint64_t(hi) << 32 | lo;
}
__device__ __forceinline__ Entry shuffle(const Entry& a, int mask) {
    return Entry{shuffle(a.key, mask), shuffle(a.tie, mask)};
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

// A 64-bit key in an order of unsigned integers, of which 0 is below any.
__device__ __forceinline__ uint64_t order_of64(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return b ^ (uint64_t(int64_t(b) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of64(uint64_t o) {
    return __builtin_bit_cast(double, o ^ (o >> 63 ? 0x8000000000000000ull : ~0ull));
}

// A float that a larger key never has a smaller one of.
__device__ __forceinline__ float float_of(double key) { return float(key); }

constexpr int kJoinRoom = 1024;  // entries that are ranked
constexpr int kJoinPad = 64;     // behind them, of nothing: a whole step of 16 lanes

// The maximum over the 16 lanes of a row of the wave.
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp_move<kDppQuadXor1>(x));
    x = fmaxf(x, dpp_move<kDppQuadXor2>(x));
    x = fmaxf(x, dpp_move<kDppRowHalfMirror>(x));
    return fmaxf(x, dpp_move<kDppRowMirror>(x));
}

// LDS of a join of `waves` waves over `beams` beams with lists of n <= 64 R entries:
// what is ranked, or in its place what is merged; then the beams.
__host__ __device__ inline size_t join_shared_entries(int R, int waves, int entries) {
    const int room = (entries < kJoinRoom ? entries : kJoinRoom) + kJoinPad;
    const size_t ranked = size_t(room) * sizeof(Entry) + size_t(room + room % 2) * sizeof(int);
    const size_t merged = entries > kJoinRoom ? size_t(waves / 2) * R * kWave * sizeof(Entry) : 0;
    return ranked > merged ? ranked : merged;
}
inline size_t join_shared(int R, int waves, int beams, int entries) {
    return join_shared_entries(R, waves, entries) + size_t(beams) * (sizeof(double) + sizeof(float) + sizeof(int));
}

// The lists of a row's spans (BEAM: of all spans of a batch element's beams) in one.
//
// As in the scan: each wave finds a value that its share of the n entries reaches, those
// above the lowest of these values are collected and ranked by counting, 4 or 16 lanes an
// entry.  The values are keys rounded to floats, which keeps their order: at least n
// entries reach the lowest value, so the n best do.  Where too many do (ties), each wave
// keeps its best entries while it merges list after list, and the waves' are merged.
// EACH entries of a thread stay in registers; with 0 they are read again.
//
// One workgroup a list, so bound by its latency: the sums of the spans, a bound, what
// reaches it, the ranks.  4 beams, 4 entries and 16 spans each 5.1 us; 8 beams, 16
// entries and 4 spans 6.6; 48 beams, 96 entries and 4 spans 18.2; 4096 rows of 4 spans
// and 64 entries 20, 999 of 128 entries 12.
template <int R, bool BEAM, int EACH>
__global__ __launch_bounds__(1024) void join(Rows r, Lists lists, JoinArgs a) {
    extern __shared__ __attribute__((aligned(16))) char shared[];
    __shared__ float wt[16];
    __shared__ int places;
    constexpr int N = R * kWave;
    const int b = batch_of_block();
    const int beams = BEAM ? r.inner : 1;
    if (b >= r.rows / beams) return;
    const int threads = int(blockDim.x), waves = threads / kWave;
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    const int count = beams * r.parts, entries = count * r.n;
    const int room = min(entries, kJoinRoom);
    Entry* ranked = reinterpret_cast<Entry*>(shared);              // [room + kJoinPad]
    int* tokens = reinterpret_cast<int*>(ranked + room + kJoinPad);
    Entry* held = ranked;                                          // [waves / 2][N], in their place
    double* shift = reinterpret_cast<double*>(shared + join_shared_entries(R, waves, entries));
    float* top = reinterpret_cast<float*>(shift + beams);    // [beams]: the largest logit
    int* kind = reinterpret_cast<int*>(top + beams);         // [beams]: 0 no entries, 1 lists, 2 itself
    const Item* items = lists.items + int64_t(b) * entries;
    const double kn = double(r.k) * 0.693147180559945309417;
    // The lists are in order: neighbouring entries go to different waves and lanes, so
    // that the lanes' maxima are as if there were no order.  97 is odd: `threads` places.
    auto entry_at = [&](int i) { return i * threads + ((int(threadIdx.x) * 97 + i * 61) & (threads - 1)); };
    // loads that depend on nothing are on their way first
    constexpr int U = 4;
    Item x[EACH > 0 ? EACH : U];
    const int first = __builtin_amdgcn_readfirstlane(wave);
    auto first_of = [&](int l) { return items[int64_t(min(l, count - 1)) * r.n + min(lane, r.n - 1)]; };
    if constexpr (EACH > 0) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) x[i] = items[min(entry_at(i), entries - 1)];
    } else {
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = first_of(first + i * waves);
    }
    if (threadIdx.x == 0) places = 0;
    for (int i = threadIdx.x; i < room + kJoinPad; i += threads) ranked[i] = nothing();
    // the sums of the beams' rows, 16 lanes a beam
    for (int w = int(threadIdx.x) / 16; w < beams; w += threads / 16) {
        const int row = b * beams + w;
        const bool read = read_row(r, row);
        float m = -__builtin_inff();
        double s = 0.0;
        for (int p = int(threadIdx.x) % 16; read && p < r.parts; p += 16) {
            const Part q = lists.parts[int64_t(row) * r.parts + p];
            if (q.s == 0.0) continue;  // nothing but -inf
            const float to = fmaxf(m, q.m);
            if (m > -__builtin_inff()) s *= short_exp((double(m) - double(to)) * kn);
            s += q.m == to ? q.s : q.s * short_exp((double(q.m) - double(to)) * kn);
            m = to;
        }
        const float most = row_max(m);
        if (m != most) s = m > -__builtin_inff() ? s * short_exp((double(m) - double(most)) * kn) : s;
        s = row_sum64(s);
        if (threadIdx.x % 16 == 0) {
            const float score = BEAM ? r.scores[row] : 0.0f;
            top[w] = most;
            shift[w] = (BEAM ? double(score) : 0.0) - short_log(s);  // what a logit's share lacks
            kind[w] = read ? 1 : BEAM && r.finished && r.finished[row] && score > -__builtin_inff() ? 2 : 0;
        }
    }
    __syncthreads();
    // The key of entry `at` of list l, of beam w: -inf where there is none.
    auto key_of = [&](int l, int w, int at, float f) {
        if (!BEAM) return kind[0] == 1 && f > -__builtin_inff() ? double(f) : -__builtin_inf();
        double key = -__builtin_inf();
        if (kind[w] == 1 && f > -__builtin_inff()) {
            const double total = shift[w] + share_of(r, f, top[w]);
            if (total > key) key = total;  // not NaN
        } else if (kind[w] == 2 && l == w * r.parts && at == 0) {
            key = double(r.scores[b * beams + w]);
        }
        return key;
    };
    auto beam_of = [&](int l) { return BEAM ? l / r.parts : 0; };
    auto tie_at = [&](int e, int w, float f) { return tie_of(w, kind[w] == 1 ? f : 0.0f, e); };
    // Of K entries of each lane those that reach `least` go to the ranked ones, one atomic a
    // wave; which of the K the last lane has among them, by bits.
    float least = 0.0f;
    auto collect = [&](auto many, const int* e, const int* w, const double* key, const Item* y) {
        constexpr int K = decltype(many)::value;
        uint64_t all[K];
        int total = 0, last = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            // totals below the lowest float are entries too
            all[i] = __ballot(least == -__FLT_MAX__ ? key[i] > -__builtin_inf() : float_of(key[i]) >= least);
            total += __builtin_popcountll(all[i]);
            last |= int(all[i] >> (kWave - 1)) << i;
        }
        if (total == 0) return last;
        int from = 0;
        if (lane == 0) from = atomicAdd(&places, total);
        from = __builtin_amdgcn_readfirstlane(from);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (all[i] == 0) continue;
            const int at = from + __builtin_amdgcn_mbcnt_hi(uint32_t(all[i] >> 32),
                                                            __builtin_amdgcn_mbcnt_lo(uint32_t(all[i]), 0));
            if ((all[i] >> lane & 1u) && at < kJoinRoom) {
                ranked[at] = Entry{order_of64(key[i]), tie_at(e[i], w[i], y[i].x)};
                tokens[at] = y[i].token;
            }
            from += __builtin_popcountll(all[i]);
        }
        return last;
    };
    // Keys that at least n entries reach the lowest of: each thread's largest, of all
    // entries or (EACH = 0) of the first few of each list, one a thread and 2 n at least.
    constexpr int K = EACH > 0 ? EACH : U;
    int e[K], w[K];
    double key[K];
    float most[1] = {-__builtin_inff()};
    if constexpr (EACH > 0) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            e[i] = w[i] = 0;
            key[i] = -__builtin_inf();
            if (i * threads >= entries) continue;
            e[i] = min(entry_at(i), entries - 1);
            const int l = e[i] / r.n;
            w[i] = beam_of(l);
            if (entry_at(i) < entries) key[i] = key_of(l, w[i], e[i] - l * r.n, x[i].x);
            most[0] = fmaxf(most[0], float_of(key[i]));
        }
    } else {
        const int heads = min(r.n, (max(2 * r.n, threads) + count - 1) / count);
        for (int i = lane * waves + wave; i < count * heads; i += threads) {
            const int l = i / heads, at = i - l * heads;
            most[0] = fmaxf(most[0], float_of(key_of(l, beam_of(l), at, items[int64_t(l) * r.n + at].x)));
        }
    }
    // one value of a lane where that is half of them at most, or there are no others (256
    // rows of 2 lists of 256: 19.5 us, of one value 41; 999 of 4 lists of 128: 13.1 and 12.0)
    const int share = (r.n + waves - 1) / waves;
    float reached;
    if (EACH == 0 || share * 2 <= kWave) {
        reached = reached_by(most, share);
    } else {
        float v[K];
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] = float_of(key[i]);
        reached = reached_by(v, share);
    }
    if (lane == 0) wt[wave] = reached;
    __syncthreads();
    least = wt[0];
    for (int i = 1; i < waves; ++i) least = fminf(least, wt[i]);
    int found;
    for (int again = 0;; ++again) {
        if constexpr (EACH > 0) {
            collect(std::integral_constant<int, K>{}, e, w, key, x);
        } else {
            // A list at a time and wave, as far as its entries reach `least`.  The code runs
            // once and comes from memory, so it is short: U lists at a time, the next ones on
            // their way, and one copy for what lies behind the first 64 entries (5 batch
            // elements, 48 beams of 4 lists of 96: 18.3 us; twelve lists at once 1 us more).
#pragma unroll 1
            for (int l0 = first; l0 < count; l0 += U * waves) {
                Item next[U];
#pragma unroll
                for (int i = 0; i < U; ++i) next[i] = first_of(l0 + (U + i) * waves);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int l = l0 + i * waves;
                    w[i] = beam_of(min(l, count - 1));
                    e[i] = l * r.n + lane;
                    key[i] = l < count && lane < r.n ? key_of(l, w[i], lane, x[i].x) : -__builtin_inf();
                }
                int more = collect(std::integral_constant<int, U>{}, e, w, key, x);
#pragma unroll 1
                for (; more && r.n > kWave; more &= more - 1) {
                    const int l = l0 + __builtin_ctz(more) * waves, wl = beam_of(l);
#pragma unroll 1
                    for (int at = kWave + lane; at - lane < r.n; at += kWave) {
                        const Item z = items[int64_t(l) * r.n + min(at, r.n - 1)];
                        const double one = at < r.n ? key_of(l, wl, at, z.x) : -__builtin_inf();
                        const int place = l * r.n + at;
                        if (!collect(std::integral_constant<int, 1>{}, &place, &wl, &one, &z)) break;
                    }
                }
#pragma unroll
                for (int i = 0; i < U; ++i) x[i] = next[i];
            }
        }
        __syncthreads();
        found = places;
        if (found <= kJoinRoom || again == 4) break;
        // Too many: some beams are far better than others, and their lists go deeper than
        // what the bound was taken from.  n of the entries that were collected, one of each
        // of 1024 threads, give a better one (16 batch elements, 64 beams of 256 entries, 8 of
        // them far ahead: 31 us, by the merging below 43).
        const float one[1] = {float_of(value_of64(ranked[lane * waves + wave].key))};
        const float better = reached_by(one, share);
        __syncthreads();
        for (int i = threadIdx.x; i < room; i += threads) ranked[i] = nothing();
        if (lane == 0) wt[wave] = better;
        if (threadIdx.x == 0) places = 0;
        __syncthreads();
        float bound = wt[0];
        for (int i = 1; i < waves; ++i) bound = fminf(bound, wt[i]);
        if (!(bound > least)) break;
        least = bound;
        if constexpr (EACH == 0) {
#pragma unroll
            for (int i = 0; i < U; ++i) x[i] = first_of(first + i * waves);
        }
    }
    // Ranking costs found^2: where there are many more than n, a bound of theirs, one of each
    // thread, leaves fewer (16 batch elements, 64 beams of 2 lists of 128 entries, 585 found:
    // 23.5 us, without this 64).
    if (threads == kJoinRoom && found > 2 * r.n + kWave && found <= kJoinRoom) {
        const int mine = lane * waves + wave;
        const Entry y = ranked[mine];
        const int token = tokens[mine];
        const float one[1] = {mine < found ? float_of(value_of64(y.key)) : -__builtin_inff()};
        const float better = reached_by(one, share);
        __syncthreads();
        ranked[mine] = nothing();
        if (lane == 0) wt[wave] = better;
        if (threadIdx.x == 0) places = 0;
        __syncthreads();
        float bound = wt[0];
        for (int i = 1; i < waves; ++i) bound = fminf(bound, wt[i]);
        const bool in = mine < found && (bound == -__FLT_MAX__ || one[0] >= bound);
        const uint64_t all = __ballot(in);
        int from = 0;
        if (lane == 0 && all) from = atomicAdd(&places, int(__builtin_popcountll(all)));
        from = __builtin_amdgcn_readfirstlane(from) +
               __builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0));
        if (in) {
            ranked[from] = y;
            tokens[from] = token;
        }
        __syncthreads();
        found = places;
    }
    auto write = [&](int to_entry, double key, int id, int token) {
        const int64_t to = int64_t(b) * r.n + to_entry;
        if (id < 0) {
            a.scores[to] = -__builtin_inff();
            a.tokens[to] = -1;
            if (BEAM) a.beams[to] = -1;
            if (BEAM && a.finished) a.finished[to] = 0;
            return;
        }
        const int w = BEAM ? id / r.n / r.parts : 0;
        const bool itself = BEAM && kind[w] == 2;
        if (itself) token = a.eos;
        a.tokens[to] = token;
        if (BEAM) {
            a.scores[to] = float(key);
            a.beams[to] = w;
            if (a.finished) a.finished[to] = itself || token == a.eos;
        } else {
            a.scores[to] = float(share_of(r, float(key), top[0]) + shift[0]);
        }
    };
    if (found <= kJoinRoom) {
        const int lanes = found * 16 <= threads ? 16 : 4;
        const int sub = int(threadIdx.x) % lanes;
        for (int c = int(threadIdx.x) / lanes; c < found; c += threads / lanes) {
            const Entry mine = ranked[c];
            int rank = 0;
            for (int j = sub; j < found; j += 4 * lanes) {
                Entry other[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) other[i] = ranked[j + i * lanes];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    rank += int(other[i].key > mine.key) | (int(other[i].key == mine.key) & int(other[i].tie > mine.tie));
            }
            rank += __builtin_amdgcn_update_dpp(0, rank, kDppQuadXor1, 0xF, 0xF, false);
            rank += __builtin_amdgcn_update_dpp(0, rank, kDppQuadXor2, 0xF, 0xF, false);
            if (lanes == 16) {
                rank += __builtin_amdgcn_update_dpp(0, rank, kDppRowHalfMirror, 0xF, 0xF, false);
                rank += __builtin_amdgcn_update_dpp(0, rank, kDppRowMirror, 0xF, 0xF, false);
            }
            if (sub == 0 && rank < r.n) write(rank, value_of64(mine.key), place_of(mine.tie), tokens[c]);
        }
        for (int e = found + int(threadIdx.x); e < r.n; e += threads) write(e, 0.0, -1, -1);
        return;
    }
    __syncthreads();  // `held` takes the place of the keys
    Best<R> best;
    best.clear();
    for (int l = wave; l < count; l += waves) {
        Entry other[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int at = N - 1 - (i * kWave + lane);
            other[i] = nothing();
            if (at >= r.n) continue;
            const float f = items[l * r.n + at].x;
            const double key = key_of(l, beam_of(l), at, f);
            if (key > -__builtin_inf()) other[i] = Entry{order_of64(key), tie_at(l * r.n + at, beam_of(l), f)};
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
        const int id = best.e[i].key == 0 ? -1 : place_of(best.e[i].tie);
        write(e, value_of64(best.e[i].key), id, id < 0 ? -1 : items[id].token);
    }
}

}  // namespace toplist
}  // namespace dot_amd
