// wave64 reduction primitives for gfx950 (CDNA4).
//
// Replaces the reference's warp-32 shuffle reductions (src/sinkhorn/kernels.cu:27-69,
// src/bidirectional_softmax/kernels.cu:41-83).  A wave is 64 lanes; a reduction
// is four DPP steps inside each 16-lane row, one ds_swizzle step across the two
// rows of each 32-lane half, and a scalar combine of the two halves through
// v_readlane.  The combine order is fixed, so results are bitwise reproducible.
// Every lane of the wave must be active when these are called.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace dot_amd {

constexpr int kWave = 64;

// DPP control words (GFX9 encoding).
constexpr int kDppQuadXor1 = 0xB1;       // quad_perm [1,0,3,2]
constexpr int kDppQuadXor2 = 0x4E;       // quad_perm [2,3,0,1]
constexpr int kDppRowHalfMirror = 0x141; // lane i <- 7-i inside each 8-lane half-row
constexpr int kDppRowMirror = 0x140;     // lane i <- 15-i inside each 16-lane row
// ds_swizzle bit-mask mode: and=0x1F, or=0, xor=0x10 -> lane ^ 16 inside 32 lanes.
constexpr int kSwizzleXor16 = (0x10 << 10) | 0x1F;

template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}

__device__ __forceinline__ float swizzle_xor16(float x) {
    return __builtin_bit_cast(float,
                              __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), kSwizzleXor16));
}

__device__ __forceinline__ float read_lane(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

struct OpSum {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct OpMax {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// All-reduce over the 64 lanes; the result is wave-uniform.
template <class Op>
__device__ __forceinline__ float wave_reduce(float x, Op op) {
    x = op(x, dpp_move<kDppQuadXor1>(x));
    x = op(x, dpp_move<kDppQuadXor2>(x));
    x = op(x, dpp_move<kDppRowHalfMirror>(x));
    x = op(x, dpp_move<kDppRowMirror>(x));
    x = op(x, swizzle_xor16(x));
    return op(read_lane(x, 0), read_lane(x, 32));
}

__device__ __forceinline__ float wave_sum(float x) { return wave_reduce(x, OpSum{}); }
__device__ __forceinline__ float wave_max(float x) { return wave_reduce(x, OpMax{}); }

template <int CTRL>
__device__ __forceinline__ double dpp_move(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double read_lane(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane(int(uint32_t(b)), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(int(uint32_t(b >> 32)), lane);
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
// Sums in 64 bits over the 16 lanes of a row, and over the wave (wave-uniform).
__device__ __forceinline__ double row_sum64(double x) {
    x += dpp_move<kDppQuadXor1>(x);
    x += dpp_move<kDppQuadXor2>(x);
    x += dpp_move<kDppRowHalfMirror>(x);
    return x + dpp_move<kDppRowMirror>(x);
}
__device__ __forceinline__ double wave_sum64(double x) {
    x = row_sum64(x);
    return (read_lane(x, 0) + read_lane(x, 16)) + (read_lane(x, 32) + read_lane(x, 48));
}

// Sum of N values of a lane, pairwise: of the 4 or 8 terms of a pack, before they enter a
// 64-bit sum, at most 3 roundings (2e-7 of their sum, of either sign).
template <int N>
__device__ __forceinline__ float pairwise(const float* x) {
    if constexpr (N == 1) return x[0];
    else return pairwise<N / 2>(x) + pairwise<N - N / 2>(x + N / 2);
}

// Orders this wave's LDS writes before its later LDS reads.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Workgroup all-reduce of one value per wave through LDS, combined in wave order.
// `scratch` needs kMaxWaves floats; contains a barrier on entry and exit.
template <int NWAVES, class Op>
__device__ __forceinline__ float block_reduce(float wave_value, float* scratch, Op op) {
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if ((threadIdx.x % kWave) == 0) scratch[wave] = wave_value;
    __syncthreads();
    float r = scratch[0];
#pragma unroll
    for (int w = 1; w < NWAVES; ++w) r = op(r, scratch[w]);
    return r;
}

// Exponentials.  The reference's safe_exp (src/sinkhorn/kernels.cu:21-25):
// 0 below -88, exp(88) above 88.  fast_exp2 is the hardware v_exp_f32 (2^x).
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

// e^x = 2^(x log2 e) with the base change made exact to first order: t =
// fl(x * kLog2E) and its rounding error e = fma(x, kLog2E, -t) + x * (log2 e - kLog2E)
// (the FMA two-product, an error-free transformation), then 2^t (1 + e ln 2)
// with the hardware exp2.  Six instructions; measured on gfx950 over 4M points
// of [-88, 88]: at most 1.25 ulp from e^x (expf: 0.85 ulp in ~17
// instructions; exp2(x * L2E) alone: 64 ulp).  Results below FLT_MIN may
// flush to 0.
__device__ __forceinline__ float exp_compensated(float x) {
    constexpr float kLog2ELo = 1.92596303e-8f;  // log2 e - kLog2E
    const float t = x * kLog2E;
    const float e = fmaf(x, kLog2ELo, fmaf(x, kLog2E, -t));
    const float r = __builtin_amdgcn_exp2f(t);
    return fmaf(r, e * kLn2, r);
}

// exp_compensated of x <= 0, -inf (0) and NaN (NaN) among them.
__device__ __forceinline__ float exp_compensated_below(float x) {
    return exp_compensated(x < -100.0f ? -100.0f : x);
}

// e^x of x <= 709 in 64 bits to 1e-11 of itself: 2^n e^f with f = x - n ln 2, |f| <= 0.347,
// by the exponential series up to f^10 / 10! (the next term is below 3e-13).  14
// instructions of 8 cycles a wave; the library's, to 1e-16, takes three times as many.
__device__ __forceinline__ double short_exp(double x) {
    if (x < -745.0) return 0.0;
    const double n = __builtin_rint(x * 1.4426950408889634074);
    constexpr double kHi = double(0.693147180559945309f), kLo = 0.693147180559945309417 - kHi;  // n kHi is exact
    const double f = fma(-n, kLo, fma(-n, kHi, x));
    double y = 1.0 / 3628800;
    y = fma(y, f, 1.0 / 362880);
    y = fma(y, f, 1.0 / 40320);
    y = fma(y, f, 1.0 / 5040);
    y = fma(y, f, 1.0 / 720);
    y = fma(y, f, 1.0 / 120);
    y = fma(y, f, 1.0 / 24);
    y = fma(y, f, 1.0 / 6);
    y = fma(y, f, 0.5);
    y = fma(y, f, 1.0);
    y = fma(y, f, 1.0);
    return ldexp(y, int(n));
}
// log x of a normal float's range in 64 bits, off by 1e-11: l = logf(x) and what x e^-l is
// beside 1, a 1e-6 at most, whose logarithm is d - d^2 / 2.
__device__ __forceinline__ double short_log(double x) {
    const double l = double(__logf(float(x)));
    const double d = fma(x, short_exp(-l), -1.0);
    return l + fma(-0.5 * d, d, d);
}

__device__ __forceinline__ float safe_exp(float x) {
    if (x < -88.0f) return 0.0f;
    return exp_compensated(fminf(x, 88.0f));
}

// safe_exp's clamps on the hardware exponential (relative error ~1e-6 for
// |x| <= 88, against ~1e-7 for expf); used where the result feeds a gradient.
__device__ __forceinline__ float safe_fast_exp(float x) {
    return x < -88.0f ? 0.0f : fast_exp(fminf(x, 88.0f));
}

}  // namespace dot_amd
