// The states of a beam search as the C ABI describes them: from a tensor of shape
// [B, W, ...] with a dimension of positions among the others, or none.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/InferenceMode.h>

#include <algorithm>
#include <vector>

#include "../../include/dot_amd.h"

namespace {

// Dimensions 2.. but `dim` (-1: none) are joined where one continues the other, in
// the order of their strides: what is left is a run of neighbouring elements and at
// most one further dimension (two without `dim`, the second in the positions' place).
inline dot_beam_state beam_state(const at::Tensor& t, int64_t dim) {
    struct Dim {
        int64_t size, stride;
    };
    const int64_t bytes = int64_t(t.element_size());
    std::vector<Dim> dims;
    bool empty = false;
    for (int64_t d = 2; d < t.dim(); ++d) {
        empty |= t.size(d) == 0;
        if (d != dim && t.size(d) > 1) dims.push_back({t.size(d), t.stride(d) * bytes});
    }
    dot_beam_state s{};
    s.data = t.data_ptr();
    s.stride_b = t.stride(0) * bytes;
    s.stride_w = t.stride(1) * bytes;
    s.outer = s.positions = empty ? 0 : 1;
    s.inner = bytes;
    if (empty) return s;
    if (dim >= 0) {
        s.positions = t.size(dim);
        s.stride_p = t.stride(dim) * bytes;
    }
    std::sort(dims.begin(), dims.end(), [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    std::vector<Dim> joined;
    for (const Dim& d : dims) {
        if (joined.empty() && d.stride == s.inner) s.inner *= d.size;
        else if (!joined.empty() && d.stride == joined.back().stride * joined.back().size) joined.back().size *= d.size;
        else joined.push_back(d);
    }
    TORCH_CHECK_VALUE(joined.size() <= (dim >= 0 ? 1u : 2u), "a state of shape ", t.sizes(), " and strides ", t.strides(),
                      " has too many separate dimensions; make it contiguous");
    if (!joined.empty()) {
        s.outer = joined.back().size;
        s.stride_outer = joined.back().stride;
    }
    if (joined.size() == 2) {
        s.positions = joined[0].size;
        s.stride_p = joined[0].stride;
    }
    return s;
}

// Arguments that fit together, as both devices' implementations need them: looked over
// here, not in Python, for a step reorders the caches of all layers.
inline std::vector<dot_beam_state> beam_states(at::TensorList states, const at::Tensor& beams,
                                               const c10::optional<at::Tensor>& lengths, c10::optional<int64_t> dim) {
    TORCH_CHECK(beams.dim() == 2 && (beams.scalar_type() == at::kInt || beams.scalar_type() == at::kLong),
                "beams must be int32 or int64 of shape [B, W]");
    if (lengths.has_value())
        TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == beams.size(0) &&
                        (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong) &&
                        lengths->device() == beams.device() && dim.has_value(),
                    "lengths must be int32 or int64 of shape [B], and come with dim");
    std::vector<dot_beam_state> out;
    out.reserve(states.size());
    const bool records = at::GradMode::is_enabled();
    for (const at::Tensor& t : states) {
        TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.dim() >= 2 && t.size(0) == beams.size(0) &&
                              t.size(1) == beams.size(1),
                          "states must be dense and have shape (", beams.size(0), ", ", beams.size(1), ", ...), got ",
                          t.sizes());
        TORCH_CHECK_VALUE(t.device() == beams.device(), "states must be on ", beams.device(), ", got ", t.device());
        const int64_t named = !dim.has_value() ? 2 : *dim < 0 ? *dim + t.dim() : *dim;
        TORCH_CHECK_VALUE(!dim.has_value() || (named >= 2 && named < t.dim()),
                          "dim must name a dimension behind the beams of every state, got ", *dim, " for ", t.sizes());
        TORCH_CHECK_VALUE(!records || !t.requires_grad(), "states that require a gradient cannot be reordered in place");
        TORCH_CHECK_VALUE(!t.is_inference() || c10::InferenceMode::is_enabled(),
                          "states of inference mode cannot be reordered outside of it");
        const int64_t d = lengths.has_value() ? named : -1;  // the positions matter with lengths alone
        out.push_back(beam_state(t, d));
    }
    return out;
}

// The states are other than what autograd may have kept of them.
inline void states_changed(at::TensorList states) {
    for (const at::Tensor& t : states) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace
