// Preference loss over pairs of log ratios or over a transport plan between
// two sets of them, and its gradients.
//
// Over a plan the loss of answer i is sum_j plan_ij f(ratio_i - ratio_{P+j}):
// one read of the plan, with f from registers.  The backward reads the plan
// once more, writes f as its gradient and adds up plan f' along rows and
// columns: a workgroup takes a strip of rows of kCols columns, keeps the
// column sums of its strip in registers and writes one partial row of them;
// `fold` adds the partials in strip order.  An entry of 0 leaves its pair out,
// whatever their ratios.
#pragma once

#include <type_traits>

#include "row.cuh"
#include "wave.cuh"

#include "../../include/dot_amd.h"

namespace dot_amd {
namespace preference {

constexpr int kVec = 4;                  // columns of a thread
constexpr int kCols = kBlock * kVec;     // columns of a workgroup's tile
constexpr int kMaxStrip = 32;            // rows of a strip at most
constexpr int kFoldBlock = 1024;         // threads of a fold workgroup,
constexpr int kFoldCols = 64;            // of as many columns (or rows)

struct Loss {
    float beta, smoothing;
    double whole;  // beta with all its digits
};

// The loss types of the kernels: those of the C ABI, and the sigmoid loss
// without smoothing.
constexpr int kPlain = 3;

// f(integral_constant) of a loss type.
template <class F>
void dispatch_type(int loss_type, float smoothing, F&& f) {
    if (loss_type == DOT_PREFER_HINGE) f(std::integral_constant<int, DOT_PREFER_HINGE>{});
    else if (loss_type == DOT_PREFER_SQUARE) f(std::integral_constant<int, DOT_PREFER_SQUARE>{});
    else if (smoothing > 0.0f) f(std::integral_constant<int, DOT_PREFER_SIGMOID>{});
    else f(std::integral_constant<int, kPlain>{});
}

// log(1 + e) for e in [0, 1]: 2 atanh(z) with z = e / (2 + e) <= 1/3, as
// 2 z (1 + w p(w)), w = z^2.  p has the cubic's coefficients that fit
// (atanh(z) / z - 1) / w on [0, 1/9] best in the maximum norm of the result
// (iterated least squares): 5e-9 relative, so a few ulp down to the smallest e,
// where 1 + e would round it away.
__device__ __forceinline__ float log1p_unit(float e) {
    const float z = e * __builtin_amdgcn_rcpf(2.0f + e);
    const float w = z * z;
    float s = 0.1401222944f;
    s = fmaf(s, w, 0.1399957091f);
    s = fmaf(s, w, 0.2001084983f);
    s = fmaf(s, w, 0.3333320618f);
    const float z2 = z + z;
    return fmaf(z2 * w, s, z2);
}

// 1 - beta d in 64 bits, each operation rounded as the definition has it.
__device__ __forceinline__ double room_of(double beta, double gap) {
#pragma clang fp contract(off)
    return 1.0 - beta * gap;
}

// f(x - y) and, with SLOPE, its derivative.
template <int TYPE, bool SLOPE>
__device__ __forceinline__ float loss_of(const Loss& l, float x, float y, float& slope) {
    const float gap = x - y;
    if constexpr (TYPE == DOT_PREFER_HINGE) {
        // The slope jumps where the room is 0: a difference or a beta rounded to
        // 32 bits would take a pair within 1e-7 of it to the other side.
        const double room = room_of(l.whole, double(x) - double(y));
        const bool shut = room <= 0.0;  // not NaN
        if (SLOPE) slope = shut ? 0.0f : room == room ? -l.beta : float(room);
        return shut ? 0.0f : float(room);
    } else if constexpr (TYPE == DOT_PREFER_SQUARE) {
        const float miss = gap - 0.5f / l.beta;
        if (SLOPE) slope = 2.0f * miss;
        return miss * miss;
    } else {
        const float keep = TYPE == kPlain ? 1.0f : 1.0f - l.smoothing;
        const float d = l.beta * gap;
        // d is rounded twice, to |d| 2^-23 of e: an exponential without the rounding of
        // its own product (|d| 2^-23.5) would hardly be nearer.
        const float e = fast_exp(-fabsf(d));
        if (SLOPE) {
            const float u = __builtin_amdgcn_rcpf(1.0f + e), eu = e * u;
            const float down = d < 0.0f ? u : eu;  // 1 / (1 + exp(d)); the other one without a difference
            slope = -l.beta * keep * down;
            if constexpr (TYPE != kPlain) slope = fmaf(l.beta * l.smoothing, d < 0.0f ? eu : u, slope);
        }
        // log(1 + exp(-d)) and log(1 + exp(d)) share their tail
        float f = fmaf(keep, fmaxf(-d, 0.0f), log1p_unit(e));
        if constexpr (TYPE != kPlain) f = fmaf(l.smoothing, fmaxf(d, 0.0f), f);
        return f;
    }
}

template <int TYPE>
__global__ __launch_bounds__(kBlock) void pairs_forward(const float* ratio, int P, Loss l, float* loss) {
    const int i = int(blockIdx.x) * kBlock + int(threadIdx.x);
    float slope;
    if (i < P) loss[i] = loss_of<TYPE, false>(l, ratio[i], ratio[P + i], slope);
}

template <int TYPE>
__global__ __launch_bounds__(kBlock) void pairs_backward(const float* ratio, int P, Loss l, const float* grad,
                                                         int grad_scalar, float* grad_ratio) {
    const int i = int(blockIdx.x) * kBlock + int(threadIdx.x);
    if (i >= P) return;
    float slope;
    loss_of<TYPE, true>(l, ratio[i], ratio[P + i], slope);
    const float g = grad[grad_scalar ? 0 : i] * slope;
    grad_ratio[i] = g;
    grad_ratio[P + i] = -g;
}

// A thread's kVec columns of the tile from c0 on: four in a row (VEC, Q a
// multiple of four: all in the plan or none), or every kBlock-th.
template <bool VEC>
__device__ __forceinline__ int column(int c0, int v) {
    return VEC ? c0 + int(threadIdx.x) * kVec + v : c0 + int(threadIdx.x) + v * kBlock;
}
template <bool VEC>
__device__ __forceinline__ void load4(const float* p, int c0, int Q, float (&x)[kVec]) {
    if constexpr (VEC) {
        const float4 t = *reinterpret_cast<const float4*>(p + column<VEC>(c0, 0));
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
    } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const int c = column<VEC>(c0, v);
            x[v] = c < Q ? p[c] : 0.0f;
        }
    }
}

// One workgroup per row.
template <int TYPE, bool VEC>
__global__ __launch_bounds__(kBlock) void plan_forward(const float* ratio, const float* plan, int P, int Q, Loss l,
                                                       float* loss) {
    __shared__ float sm[kWavesPerBlock];
    const int i = blockIdx.x;
    const float ri = ratio[i];
    const float* row = plan + int64_t(i) * Q;
    float sum = 0.0f;
#pragma unroll 2
    for (int c0 = 0; c0 < Q; c0 += kCols) {
        if (column<VEC>(c0, 0) >= Q) break;
        float x[kVec], slope;
        load4<VEC>(row, c0, Q, x);
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const int c = column<VEC>(c0, v);
            if (!VEC && c >= Q) continue;
            const float f = loss_of<TYPE, false>(l, ri, ratio[P + c], slope);
            sum = x[v] != 0.0f ? fmaf(x[v], f, sum) : sum;
        }
    }
    sum = block_reduce<kWavesPerBlock>(wave_sum(sum), sm, OpSum{});
    if (threadIdx.x == 0) loss[i] = sum;
}

struct PlanBwd {
    const float* ratio;
    const float* plan;
    int P, Q;
    Loss l;
    const float* grad;
    int grad_scalar;
    float* grad_plan;
    int strip, nstrips, ncols;  // rows of a strip, strips, column tiles
    float* colpart;             // [nstrips, Q]
    float* rowpart;             // [ncols, P]
};

// One tile: a strip of rows by kCols columns.
template <int TYPE, bool VEC>
__global__ __launch_bounds__(kBlock) void plan_backward(PlanBwd a) {
    __shared__ float sm[kMaxStrip][kWavesPerBlock];
    const int tile = blockIdx.x % unsigned(a.ncols), strip = blockIdx.x / unsigned(a.ncols);
    const int i0 = strip * a.strip, rows = min(a.strip, a.P - i0), c0 = tile * kCols;
    const bool some = column<VEC>(c0, 0) < a.Q;
    float rj[kVec], col[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        const int c = column<VEC>(c0, v);
        rj[v] = c < a.Q ? a.ratio[a.P + c] : 0.0f;
        col[v] = 0.0f;
    }
    for (int r = 0; r < rows; ++r) {
        const int i = i0 + r;
        const float ri = a.ratio[i], g = a.grad[a.grad_scalar ? 0 : i];
        float sum = 0.0f;
        if (some) {
            float x[kVec], f[kVec], slope[kVec], all = 1.0f;
            load4<VEC>(a.plan + int64_t(i) * a.Q, c0, a.Q, x);
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                f[v] = loss_of<TYPE, true>(a.l, ri, rj[v], slope[v]);
                all *= x[v];
            }
            if (!(all > 0.0f)) {  // perhaps pairs that are left out
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    if (x[v] != 0.0f) continue;
                    f[v] = f[v] < __builtin_inff() ? f[v] : 0.0f;
                    slope[v] = 0.0f;
                }
            }
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                f[v] *= g;
                const float pull = g * x[v] * slope[v];
                sum += pull;
                col[v] += pull;
            }
            if (a.grad_plan) {
                float* out = a.grad_plan + int64_t(i) * a.Q;
                if constexpr (VEC) {
                    *reinterpret_cast<float4*>(out + column<VEC>(c0, 0)) = make_float4(f[0], f[1], f[2], f[3]);
                } else {
#pragma unroll
                    for (int v = 0; v < kVec; ++v)
                        if (column<VEC>(c0, v) < a.Q) out[column<VEC>(c0, v)] = f[v];
                }
            }
        }
        sum = wave_sum(sum);
        if (threadIdx.x % kWave == 0) sm[r][threadIdx.x / kWave] = sum;
    }
    __syncthreads();
    if (int(threadIdx.x) < rows) {
        float s = 0.0f;
        for (int w = 0; w < kWavesPerBlock; ++w) s += sm[threadIdx.x][w];
        a.rowpart[int64_t(tile) * a.P + i0 + threadIdx.x] = s;
    }
    float* cp = a.colpart + int64_t(strip) * a.Q;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        const int c = column<VEC>(c0, v);
        if (c < a.Q) cp[c] = col[v];
    }
}

// grad_ratio from the partials: workgroups before `row_blocks` add up rows'
// column tiles, the others columns' strips (with the other sign).
__global__ __launch_bounds__(kFoldBlock) void plan_fold(PlanBwd a, int row_blocks, float* grad_ratio) {
    constexpr int kSlices = kFoldBlock / kFoldCols;
    __shared__ float sm[kSlices][kFoldCols];
    const bool rows = int(blockIdx.x) < row_blocks;
    const int lane = threadIdx.x % kFoldCols, slice = threadIdx.x / kFoldCols;
    const int at = (rows ? int(blockIdx.x) : int(blockIdx.x) - row_blocks) * kFoldCols + lane;
    const int len = rows ? a.P : a.Q, parts = rows ? a.ncols : a.nstrips;
    const float* src = rows ? a.rowpart : a.colpart;
    float s = 0.0f;
    if (at < len) {
#pragma unroll 8
        for (int p = slice; p < parts; p += kSlices) s += src[int64_t(p) * len + at];
    }
    sm[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && at < len) {
        for (int t = 1; t < kSlices; ++t) s += sm[t][lane];
        if (rows) grad_ratio[at] = s;
        else grad_ratio[a.P + at] = -s;
    }
}

}  // namespace preference
}  // namespace dot_amd
