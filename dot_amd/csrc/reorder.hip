// C ABI of the reordering of beams: argument checks and launches.
#include <algorithm>
#include <array>
#include <functional>
#include <new>
#include <vector>

#include "host.hpp"
#include "reorder.cuh"

namespace dot_amd {
namespace {

struct Dim {
    int64_t stride, size;
};

// Whether places that differ in some dimension are all apart: each stride passes
// what the smaller ones reach.
template <size_t N>
bool apart(std::array<Dim, N> d, int64_t inner) {
    std::sort(d.begin(), d.end(), [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    __int128 reach = inner;
    for (const Dim& x : d) {
        if (x.size <= 1) continue;
        if (x.stride < reach) return false;
        reach += __int128(x.stride) * (x.size - 1);
    }
    return reach <= (__int128(1) << 62);
}

std::array<Dim, 4> dims_of(const dot_beam_state& s, int B, int W) {
    return {Dim{s.stride_b, B}, Dim{s.stride_w, W}, Dim{s.stride_outer, s.outer}, Dim{s.stride_p, s.positions}};
}

int64_t reach_of(const dot_beam_state& s, int B, int W) {
    return s.stride_b * (B - 1) + s.stride_w * (W - 1) + s.stride_outer * (s.outer - 1) +
           s.stride_p * (s.positions - 1) + s.inner;
}

bool empty(const dot_beam_state& s) { return s.outer == 0 || s.positions == 0 || s.inner == 0; }

// Whether sum_d k_d stride_d falls into [lo, hi] for some k_d of [least_d, most_d], the
// strides descending; also where that is not settled in `steps` trials.
struct Term {
    int64_t stride, least, most;
};
using Wide = __int128;  // sums over two states, each up to 2^62
bool meets(const Term* t, int n, Wide lo, Wide hi, int& steps) {
    if (--steps < 0) return true;
    Wide below = 0, above = 0;  // what the later terms can add
    for (int i = 1; i < n; ++i) {
        below += Wide(t[i].stride) * t[i].least;
        above += Wide(t[i].stride) * t[i].most;
    }
    if (n == 0) return lo <= 0 && hi >= 0;
    auto floor_of = [&](Wide x) { return x / t[0].stride - (x % t[0].stride < 0); };
    const Wide first = std::max<Wide>(t[0].least, -floor_of(above - lo)), last = std::min<Wide>(t[0].most, floor_of(hi - below));
    for (Wide k = first; k <= last; ++k)
        if (meets(t + 1, n - 1, lo - k * t[0].stride, hi - k * t[0].stride, steps)) return true;
    return false;
}

// Whether two states have no byte in common: they lie apart, or within each other's
// gaps, as keys and values of one tensor do.
bool disjoint(const dot_beam_state& x, const dot_beam_state& y, int B, int W) {
    const char *px = static_cast<const char*>(x.data), *py = static_cast<const char*>(y.data);
    if (px + reach_of(x, B, W) <= py || py + reach_of(y, B, W) <= px) return true;
    const std::array<Dim, 4> dx = dims_of(x, B, W), dy = dims_of(y, B, W);
    if (x.stride_b == y.stride_b && x.stride_w == y.stride_w && x.stride_outer == y.stride_outer &&
        x.stride_p == y.stride_p && x.outer == y.outer && x.positions == y.positions && x.inner == y.inner &&
        apart(std::array<Dim, 5>{dx[0], dx[1], dx[2], dx[3], Dim{px < py ? py - px : px - py, 2}}, x.inner))
        return true;
    // px + sum i_d sx_d + a = py + sum j_d sy_d + b, equal strides in one term: at most three
    // values of each k_d = i_d - j_d come into question, since what is left of either state
    // is shorter than the stride
    std::array<Term, 8> t;
    int n = 0;
    auto add = [&](const Dim& d, int64_t least, int64_t most) {
        if (d.size <= 1 || d.stride == 0) return;
        Term* same = std::find_if(t.data(), t.data() + n, [&](const Term& u) { return u.stride == d.stride; });
        if (same == t.data() + n) t[size_t(n++)] = Term{d.stride, 0, 0};
        same->least += least;
        same->most += most;
    };
    for (const Dim& d : dx) add(d, 0, d.size - 1);
    for (const Dim& d : dy) add(d, 1 - d.size, 0);
    std::sort(t.data(), t.data() + n, [](const Term& u, const Term& v) { return u.stride > v.stride; });
    int steps = 4096;
    const Wide apart_by = py - px;
    return !meets(t.data(), n, apart_by - (x.inner - 1), apart_by + (y.inner - 1), steps);
}

// Bytes of a unit: the largest power of two that divides every address.
int unit_of(const dot_beam_state& s, int B, int W) {
    uint64_t all = uint64_t(reinterpret_cast<uintptr_t>(s.data)) | uint64_t(s.inner) | 16u;
    if (B > 1) all |= uint64_t(s.stride_b);
    if (W > 1) all |= uint64_t(s.stride_w);
    if (s.outer > 1) all |= uint64_t(s.stride_outer);
    if (s.positions > 1) all |= uint64_t(s.stride_p);
    return int(all & (~all + 1));
}

template <int BYTES>
void launch(const reorder::States& a, unsigned blocks, hipStream_t stream) {
    const dim3 grid = batch_grid(blocks, a.B), block(kBlock);
    if (a.W <= 4) hipLaunchKernelGGL((reorder::move<BYTES, 4>), grid, block, 0, stream, a);
    else if (a.W <= 8) hipLaunchKernelGGL((reorder::move<BYTES, 8>), grid, block, 0, stream, a);
    else if (a.W <= 16) hipLaunchKernelGGL((reorder::move<BYTES, 16>), grid, block, 0, stream, a);
    else if constexpr (BYTES <= 8) {
        if (a.W <= 32) hipLaunchKernelGGL((reorder::move<BYTES, 32>), grid, block, 0, stream, a);
        else if (a.W <= 64) hipLaunchKernelGGL((reorder::move<BYTES, 64>), grid, block, 0, stream, a);
        else if constexpr (BYTES <= 4) hipLaunchKernelGGL((reorder::move<BYTES, 128>), grid, block, 0, stream, a);
    }
}

}  // namespace
}  // namespace dot_amd

using namespace dot_amd;

// The states that have something to move, by their address; DOT_OK or why there are none.
static int checked(const dot_beam_reorder_args* a, std::vector<const dot_beam_state*>& moved) {
    if (!a) return fail(DOT_ERR_INVALID_ARG, "args is NULL");
    if (a->B < 0 || a->W < 1 || a->count < 0)
        return fail(DOT_ERR_INVALID_ARG, "B and count must be >= 0 and W >= 1");
    if (a->W > DOT_BEAM_MAX) return fail(DOT_ERR_UNSUPPORTED, "at most DOT_BEAM_MAX beams are supported");
    if (a->B == 0 || a->count == 0) return ok();
    if (!a->states || !a->beams) return fail(DOT_ERR_INVALID_ARG, "states and beams must be non-NULL");
    for (int i = 0; i < a->count; ++i) {
        const dot_beam_state& s = a->states[i];
        if (s.outer < 0 || s.positions < 0 || s.inner < 0 || s.stride_b < 0 || s.stride_w < 0 || s.stride_outer < 0 ||
            s.stride_p < 0)
            return fail(DOT_ERR_INVALID_ARG, "sizes and strides of a state must be >= 0");
        if (empty(s)) continue;
        if (!s.data) return fail(DOT_ERR_INVALID_ARG, "data of a state must be non-NULL");
        if (s.inner > (int64_t(1) << 31)) return fail(DOT_ERR_UNSUPPORTED, "inner must be at most 2^31");
        if (!apart(dims_of(s, a->B, a->W), s.inner))
            return fail(DOT_ERR_INVALID_ARG, "places of a state overlap");
        moved.push_back(&s);
    }
    std::sort(moved.begin(), moved.end(),
              [](const dot_beam_state* x, const dot_beam_state* y) { return std::less<void*>()(x->data, y->data); });
    for (size_t i = 0; i < moved.size(); ++i)
        for (size_t j = i + 1; j < moved.size(); ++j) {
            const char* end = static_cast<const char*>(moved[i]->data) + reach_of(*moved[i], a->B, a->W);
            if (static_cast<const char*>(moved[j]->data) >= end) break;  // and so are those behind it
            if (!disjoint(*moved[i], *moved[j], a->B, a->W))
                return fail(DOT_ERR_INVALID_ARG,
                            "states share memory, or interleave with too many strides to tell that they do not");
        }
    // the call reads these while it writes the states
    auto inside = [&](const void* p, int64_t bytes) {
        const dot_beam_state one{const_cast<void*>(p), 0, 0, 0, 0, 1, 1, bytes};
        for (const dot_beam_state* s : moved)
            if (!disjoint(*s, one, a->B, a->W)) return true;
        return false;
    };
    if (inside(a->beams, int64_t(a->B) * a->W * (a->beams_are_int64 ? 8 : 4)) ||
        (a->lengths && inside(a->lengths, int64_t(a->B) * (a->lengths_are_int64 ? 8 : 4))))
        return fail(DOT_ERR_INVALID_ARG, "beams and lengths must not share memory with a state");
    return ok();
}

static int reorder_states(const dot_beam_reorder_args* a, hipStream_t stream) {
    std::vector<const dot_beam_state*> moved;
    if (int rc = checked(a, moved)) return rc;
    if (moved.empty()) return ok();
    if (a->W == 1) return ok();
    // Launches of states of one unit.
    for (int unit = 16; unit >= 1; unit /= 2) {
        const int most = a->W <= 16 ? 16 : a->W <= 64 ? 8 : 4;  // units of all beams in 64 or 128 registers
        if (unit > most) continue;
        size_t i = 0;
        while (i < moved.size()) {
            reorder::States g{};
            int64_t chunks = 0;
            for (; i < moved.size() && g.count < reorder::kMaxStates; ++i) {
                const dot_beam_state& s = *moved[i];
                if (std::min(unit_of(s, a->B, a->W), most) != unit) continue;
                chunks += (s.outer * s.positions * (s.inner / unit) + kBlock - 1) / kBlock;
                g.s[g.count++] = reorder::State{static_cast<char*>(s.data), s.stride_b,    s.stride_w,
                                                s.stride_outer,             s.stride_p,    s.outer,
                                                s.positions,                uint32_t(s.inner / unit)};
            }
            if (g.count == 0) break;
            g.beams = a->beams;
            g.beams64 = a->beams_are_int64;
            g.lengths = a->lengths;
            g.lengths64 = a->lengths_are_int64;
            g.B = a->B;
            g.W = a->W;
            // about 4096 workgroups: 2048, 4096 and 8192 take 211, 205 and 199 us for 16 caches of
            // 8 x 4 x 8 x 1024 x 128 bf16 in use to three quarters, and 17, 19 and 32 with 8 positions in use
            const int64_t blocks = std::min(std::max<int64_t>(1, 4096 / a->B), chunks);
            ProfScope prof("beam_reorder", stream);
            if (unit == 16) launch<16>(g, unsigned(blocks), stream);
            else if (unit == 8) launch<8>(g, unsigned(blocks), stream);
            else if (unit == 4) launch<4>(g, unsigned(blocks), stream);
            else if (unit == 2) launch<2>(g, unsigned(blocks), stream);
            else launch<1>(g, unsigned(blocks), stream);
        }
    }
    return check_launch("dot_beam_reorder");
}

template <class F>
static int guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return fail(DOT_ERR_WORKSPACE, "out of host memory");
    }
}

extern "C" int dot_beam_reorder_check(const dot_beam_reorder_args* args) {
    return guarded([&] {
        std::vector<const dot_beam_state*> moved;
        return checked(args, moved);
    });
}

extern "C" int dot_beam_reorder(const dot_beam_reorder_args* args, dot_stream_t stream) {
    return guarded([&] { return reorder_states(args, reinterpret_cast<hipStream_t>(stream)); });
}
