// What the PyTorch bindings of the language model operators share: checks of
// tensors, streams and workspaces, and the parts of their autograd functions.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <memory>
#include <string>
#include <vector>

#include "../../include/dot_amd.h"

namespace {

using at::Tensor;
using c10::optional;

inline void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == DOT_OK, what, " failed (code ", rc, "): ", dot_last_error());
}

inline dot_stream_t stream_of(const Tensor& t) {
    return reinterpret_cast<dot_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// Scratch of a call, none where it needs none (an allocation takes the host
// over a microsecond).
inline Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}
inline void* ptr_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline int dtype_tag(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return DOT_F32;
        case at::kHalf: return DOT_F16;
        case at::kBFloat16: return DOT_BF16;
        default: TORCH_CHECK(false, name, " must be float32, float16 or bfloat16");
    }
}

inline int to_int(int64_t v, const char* name) {
    TORCH_CHECK(v >= 0 && v <= INT32_MAX, name, " out of range");
    return int(v);
}

inline void check_on(const Tensor& t, const Tensor& with, const char* name) {
    TORCH_CHECK(t.device() == with.device(), name, " must be on ", with.device(), ", got ", t.device());
}

// Rows of unit stride, in place where they are so already.
inline Tensor unit_rows(const Tensor& t) { return t.stride(2) == 1 || t.size(2) <= 1 ? t : t.contiguous(); }

inline const float* floats(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
inline Tensor f32c(const optional<Tensor>& t, const Tensor& like, const char* name) {
    if (!t.has_value()) return Tensor();
    check_on(*t, like, name);
    return t->to(at::kFloat).contiguous();
}

// An upstream gradient and whether it is one value for all (an expanded
// scalar, as the gradient of a sum is).
inline Tensor upstream(const Tensor& g, const Tensor& like, int& scalar) {
    check_on(g, like, "grad");
    bool one = g.numel() > 1;
    for (int64_t d = 0; d < g.dim(); ++d) one = one && (g.stride(d) == 0 || g.size(d) == 1);
    scalar = one;
    if (one) return g.as_strided({1}, {1}).to(at::kFloat);
    return g.to(at::kFloat).contiguous();
}

inline Tensor mask_of(const optional<Tensor>& mask, const Tensor& x) {
    if (!mask.has_value()) return Tensor();
    check_on(*mask, x, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kBool && mask->dim() == 2 && mask->size(0) == x.size(0) &&
                    mask->size(1) == x.size(1),
                "mask must be bool of the leading two sizes");
    return mask->contiguous();
}
inline const uint8_t* mask_ptr(const Tensor& m) {
    return m.defined() ? reinterpret_cast<const uint8_t*>(m.const_data_ptr()) : nullptr;
}

inline Tensor ints_of(const Tensor& t, const Tensor& like, const char* name) {
    check_on(t, like, name);
    TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
    return t.contiguous();
}

inline void check_rows(const Tensor& x, const char* name) {
    TORCH_CHECK(x.device().is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(x.dim() == 3, name, " must be 3D");
}

// ---------------------------------------------------------------------------
// Autograd
// ---------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Whether a call has to be recorded.
inline bool records(const Tensor& x) { return at::GradMode::is_enabled() && x.requires_grad(); }
inline bool records(const optional<Tensor>& x) { return x.has_value() && records(*x); }

// A tangent of forward-mode differentiation would be dropped below autograd, so
// that the derivative came out as zero: an error instead.
inline void check_no_tangent(const Tensor& x) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !x._fw_grad(0).defined(),
                                "dot_amd operators have no forward-mode derivative");
}

// The gradient of an operator that has no second derivative: a backward
// through it is an error, not a wrong result.  The error's node leads on to all
// that the gradient is a function of (the inputs and the upstream gradients):
// the engine runs only nodes on a way to what it is asked for.
inline Tensor once(const Tensor& grad, const variable_list& of) {
    if (!at::GradMode::is_enabled() || !grad.defined()) return grad;
    auto refuse = std::make_shared<torch::autograd::Error>(
        "dot_amd operators are differentiable once: no gradient flows through their backward",
        torch::autograd::collect_next_edges(of));
    Tensor out = grad.detach();
    torch::autograd::set_history(out, refuse);
    return out;
}

template <class F>
auto op_handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

inline optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

}  // namespace
