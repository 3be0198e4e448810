// States of the chosen beams, in place.
//
// A thread holds one unit (16 bytes at most) of the same place in every beam: it
// loads what the moving beams' parents have there, then stores it.  No place is read
// by another thread than the one that writes it, so neither a second copy of the
// states nor an order among the threads is needed, whatever the parents are.  Beams
// that stay are not written, parents that no moving beam has are not read; a parent
// of several is read from memory once.
//
// Bound by HBM.  16 caches of 8 x 4 x 8 x 1024 x 128 bf16, three quarters of the
// positions in use, 0.98 GB: 201 us; on inputs that take 205, loads and stores that stay in
// the caches 213, and each workgroup striding through one state of its own 215 (226):
// neighbouring workgroups at neighbouring places meet open pages of the memory.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "elem.cuh"
#include "row.cuh"

namespace dot_amd {
namespace reorder {

constexpr int kMaxStates = 32;  // of a launch: their descriptions travel with its arguments

struct State {
    char* data;
    int64_t sb, sw, so, sp;
    int64_t outer, positions;
    uint32_t inner;  // units of a position
};
struct States {
    State s[kMaxStates];
    int count;
    const void* beams;
    int beams64;
    const void* lengths;
    int lengths64;
    int B, W;
};

template <int BYTES>
struct UnitOf;
template <>
struct UnitOf<1> {
    using type = uint8_t;
};
template <>
struct UnitOf<2> {
    using type = uint16_t;
};
template <>
struct UnitOf<4> {
    using type = uint32_t;
};
template <>
struct UnitOf<8> {
    using type = uint64_t;
};
template <>
struct UnitOf<16> {
    typedef uint32_t type __attribute__((ext_vector_type(4)));
};

// u / by, both at most `total`.
__device__ __forceinline__ uint64_t quotient(uint64_t u, uint64_t by, uint64_t total) {
    return total >> 32 ? u / by : uint64_t(uint32_t(u) / uint32_t(by));
}

// MAX: the most beams that a thread has registers for; units of 8 bytes above 16 beams and
// of 4 above 64 (2 x 64 caches of 8 x 512 x 128 bf16, 8 of them: 370 us, 4.8 TB/s; in units
// of 4 and registers for 128 beams 600 us).
template <int BYTES, int MAX>
__global__ __launch_bounds__(kBlock) void move(States a) {
    using U = typename UnitOf<BYTES>::type;
    __shared__ int parent[MAX];
    const int b = batch_of_block();
    if (b >= a.B) return;
    bool moves = false;
    for (int w = threadIdx.x; w < MAX; w += kBlock) {
        const int64_t p = w < a.W ? int_at(a.beams, a.beams64, int64_t(b) * a.W + w) : -1;
        parent[w] = p >= 0 && p < a.W && p != w ? int(p) : -1;
        moves |= parent[w] >= 0;
    }
    if (!__syncthreads_or(moves)) return;
    int64_t used = INT64_MAX;
    if (a.lengths) used = max(int_at(a.lengths, a.lengths64, b), int64_t(0));
    // The workgroups of a batch element go through its states side by side.
    uint64_t chunk = blockIdx.x;
    for (int i = 0; i < a.count; ++i) {
        const State& s = a.s[i];
        const uint64_t run = uint64_t(min(used, s.positions)) * s.inner, total = uint64_t(s.outer) * run;
        const uint64_t chunks = (total + kBlock - 1) / kBlock;
        char* base = s.data + int64_t(b) * s.sb;
        const bool dense = s.sp == int64_t(s.inner) * BYTES;
        for (; chunk < chunks; chunk += gridDim.x) {
            const uint64_t u = chunk * kBlock + threadIdx.x;
            if (u >= total) continue;
            const uint64_t o = quotient(u, run, total), at = u - o * run;
            int64_t off = int64_t(o) * s.so;
            if (dense) {
                off += int64_t(at) * BYTES;
            } else {
                const uint64_t p = quotient(at, s.inner, total);
                off += int64_t(p) * s.sp + int64_t(at - p * s.inner) * BYTES;
            }
            U x[MAX];
#pragma unroll
            for (int w = 0; w < MAX; ++w)
                if (parent[w] >= 0)
                    x[w] = __builtin_nontemporal_load(reinterpret_cast<const U*>(base + off + int64_t(parent[w]) * s.sw));
#pragma unroll
            for (int w = 0; w < MAX; ++w)
                if (parent[w] >= 0)
                    __builtin_nontemporal_store(x[w], reinterpret_cast<U*>(base + off + int64_t(w) * s.sw));
        }
        chunk -= chunks;
    }
}

}  // namespace reorder
}  // namespace dot_amd
