// Preference loss over pairs of log ratios or over a transport plan between
// two sets of them, and its gradients.
//
// Over a plan the loss of answer i is sum_j plan_ij f(ratio_i - ratio_{P+j}):
// one read of the plan, with f from registers.  The backward reads the plan
// once more, writes f as its gradient and adds up plan f' along rows and
// columns: a workgroup takes a strip of rows of kCols columns, keeps the
// column sums of its strip in registers and writes one partial row of them;
// `fold` adds the partials in strip order.
#pragma once

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
    int type;
    float beta, smoothing;
};

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

// f(gap) and, with SLOPE, df / dgap.
template <bool SLOPE>
__device__ __forceinline__ float loss_of(const Loss& l, float gap, float& slope) {
    if (l.type == DOT_PREFER_SIGMOID) {
        const float d = l.beta * gap;
        const float e = fast_exp(-fabsf(d));
        if (SLOPE) {
            const float u = __builtin_amdgcn_rcpf(1.0f + e);
            const float up = d < 0.0f ? e * u : u;    // 1 / (1 + exp(-d))
            const float down = d < 0.0f ? u : e * u;  // 1 - up, without the difference
            slope = l.beta * (l.smoothing * up - (1.0f - l.smoothing) * down);
        }
        // log(1 + exp(-d)) and log(1 + exp(d)) share their tail
        float f = fmaf(1.0f - l.smoothing, fmaxf(-d, 0.0f), log1p_unit(e));
        if (l.smoothing > 0.0f) f = fmaf(l.smoothing, fmaxf(d, 0.0f), f);
        return f;
    }
    if (l.type == DOT_PREFER_HINGE) {
        const float room = fmaf(-l.beta, gap, 1.0f);
        if (SLOPE) slope = room > 0.0f ? -l.beta : (room == room ? 0.0f : room);
        return room > 0.0f ? room : (room == room ? 0.0f : room);
    }
    const float miss = gap - 0.5f / l.beta;
    if (SLOPE) slope = 2.0f * miss;
    return miss * miss;
}

__global__ __launch_bounds__(kBlock) void pairs_forward(const float* ratio, int P, Loss l, float* loss) {
    const int i = int(blockIdx.x) * kBlock + int(threadIdx.x);
    float slope;
    if (i < P) loss[i] = loss_of<false>(l, ratio[i] - ratio[P + i], slope);
}

__global__ __launch_bounds__(kBlock) void pairs_backward(const float* ratio, int P, Loss l, const float* grad,
                                                         int grad_scalar, float* grad_ratio) {
    const int i = int(blockIdx.x) * kBlock + int(threadIdx.x);
    if (i >= P) return;
    float slope;
    loss_of<true>(l, ratio[i] - ratio[P + i], slope);
    const float g = grad[grad_scalar ? 0 : i] * slope;
    grad_ratio[i] = g;
    grad_ratio[P + i] = -g;
}

// kVec columns from j on; a column beyond Q is `fill`.
template <bool VEC>
__device__ __forceinline__ void load4(const float* p, int j, int Q, float (&x)[kVec], float fill) {
    if constexpr (VEC) {
        if (j < Q) {
            const float4 t = *reinterpret_cast<const float4*>(p + j);
            x[0] = t.x;
            x[1] = t.y;
            x[2] = t.z;
            x[3] = t.w;
        } else {
            x[0] = x[1] = x[2] = x[3] = fill;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = j + i * kBlock < Q ? p[j + i * kBlock] : fill;
    }
}

// First of a thread's columns in the tile from c0 on: four in a row, or every
// kBlock-th.
template <bool VEC>
__device__ __forceinline__ int first_col(int c0) {
    return c0 + (VEC ? int(threadIdx.x) * kVec : int(threadIdx.x));
}

// One workgroup per row.
template <bool VEC>
__global__ __launch_bounds__(kBlock) void plan_forward(const float* ratio, const float* plan, int P, int Q, Loss l,
                                                       float* loss) {
    __shared__ float sm[kWavesPerBlock];
    const int i = blockIdx.x;
    const float ri = ratio[i];
    const float* row = plan + int64_t(i) * Q;
    float sum = 0.0f;
    for (int c0 = 0; c0 < Q; c0 += kCols) {
        const int j = first_col<VEC>(c0);
        float x[kVec], rj[kVec], slope;
        load4<VEC>(row, j, Q, x, 0.0f);
        if (VEC && P % kVec == 0) {
            load4<true>(ratio + P, j, Q, rj, 0.0f);
        } else {
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                const int c = VEC ? j + v : j + v * kBlock;
                rj[v] = c < Q ? ratio[P + c] : 0.0f;
            }
        }
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const int c = VEC ? j + v : j + v * kBlock;
            if (c < Q) sum = fmaf(x[v], loss_of<false>(l, ri - rj[v], slope), sum);
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
template <bool VEC>
__global__ __launch_bounds__(kBlock) void plan_backward(PlanBwd a) {
    __shared__ float sm[kMaxStrip][kWavesPerBlock];
    const int tile = blockIdx.x % unsigned(a.ncols), strip = blockIdx.x / unsigned(a.ncols);
    const int i0 = strip * a.strip, rows = min(a.strip, a.P - i0);
    const int j = first_col<VEC>(tile * kCols);
    float rj[kVec], col[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        const int c = VEC ? j + v : j + v * kBlock;
        rj[v] = c < a.Q ? a.ratio[a.P + c] : 0.0f;
        col[v] = 0.0f;
    }
    for (int r = 0; r < rows; ++r) {
        const int i = i0 + r;
        const float ri = a.ratio[i], g = a.grad[a.grad_scalar ? 0 : i];
        float x[kVec], f[kVec], slope, sum = 0.0f;
        load4<VEC>(a.plan + int64_t(i) * a.Q, j, a.Q, x, 0.0f);
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const int c = VEC ? j + v : j + v * kBlock;
            if (c < a.Q) {
                f[v] = g * loss_of<true>(a.l, ri - rj[v], slope);
                const float pull = g * x[v] * slope;
                sum += pull;
                col[v] += pull;
            }
        }
        if (a.grad_plan) {
            float* out = a.grad_plan + int64_t(i) * a.Q;
            if constexpr (VEC) {
                if (j < a.Q) *reinterpret_cast<float4*>(out + j) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int v = 0; v < kVec; ++v)
                    if (j + v * kBlock < a.Q) out[j + v * kBlock] = f[v];
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
        const int c = VEC ? j + v : j + v * kBlock;
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
