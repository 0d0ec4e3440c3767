// What the bindings of the operators on [N,H,L,D] rows of fp32, fp16 or bf16 share: checks, views, and what a call may keep for its backward pass.
#pragma once
#include "fwp_torch.hpp"

#include <torch/csrc/autograd/variable.h>

#include <limits>
#include <optional>

namespace fwp_host {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Optional = std::optional<at::Tensor>;

inline at::Tensor given(const Optional &t) { return t.has_value() ? *t : at::Tensor(); }

inline int type_of(const at::Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return FWP_F32;
        case at::kHalf: return FWP_F16;
        case at::kBFloat16: return FWP_BF16;
        default: fail(std::string(name) + " must be fp32, fp16 or bf16");
    }
}

[[noreturn]] inline void misfit(const char *name, const at::Tensor &t, const char *wanted) {
    fail(std::string("shape mismatch: ") + name + shape_of(t) + ", expected " + wanted);
}

inline void same_type(const at::Tensor &t, const at::Tensor &like, const char *name) {
    if (t.defined() && t.scalar_type() != like.scalar_type()) fail(std::string(name) + " must have the type of the other rows");
}

// Contiguous, and with the values that its memory holds: a view with its sign still to be changed (the imaginary part of a conjugate) is a copy too
inline at::Tensor plain(const at::Tensor &t) { return !t.defined() ? t : t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }

// A parameter: fp32, of this shape, contiguous (a copy if it is not)
inline at::Tensor parameter(const at::Tensor &t, at::IntArrayRef shape, const char *name, const char *wanted) {
    if (!t.defined()) return t;
    if (t.scalar_type() != at::kFloat) fail(std::string(name) + " must be fp32");
    if (t.sizes() != shape) misfit(name, t, wanted);
    return plain(t);
}

// lengths [N]: int64
inline at::Tensor lengths_of(const at::Tensor &t, int64_t N) {
    if (!t.defined()) return t;
    if (t.scalar_type() != at::kLong || !same_shape(t, {N})) fail("lengths must be an int64 tensor [N]");
    return t.contiguous();
}

constexpr int64_t kMaxStep = FWP_SCAN_MAX_STEP;

// [N,H,L,D] rows whose last axis is contiguous; a copy where it is not, and of rows too far apart
inline at::Tensor rows_of(const at::Tensor &t, int64_t most = std::numeric_limits<int64_t>::max()) {
    if (!t.defined() || (!t.is_neg() && (t.size(3) == 1 || t.stride(3) == 1) && (t.size(2) == 1 || t.stride(2) <= most))) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

inline fwp_rows view(const at::Tensor &t) {
    return t.defined() ? fwp_rows{t.const_data_ptr(), t.stride(0), t.stride(1), t.size(2) > 1 ? t.stride(2) : 0} : fwp_rows{};
}
inline fwp_out_rows out_view(const at::Tensor &t) {
    return t.defined() ? fwp_out_rows{t.data_ptr(), t.stride(0), t.stride(1), t.size(2) > 1 ? t.stride(2) : 0} : fwp_out_rows{};
}

// Do these rows lie with the steps outermost, as a layer's permuted views do?  Results take the order of the rows they belong to.
inline bool steps_lead(const at::Tensor &t, int64_t heads, int64_t most) {
    const int64_t N = t.size(0), H = t.size(1), L = t.size(2);
    return L > 1 && (N > 1 || H > 1) && N * heads * t.size(3) <= most && (N == 1 || t.stride(2) > t.stride(0)) && (H == 1 || t.stride(2) > t.stride(1));
}
inline at::Tensor empty_rows(const at::Tensor &like, int64_t heads = 0, int64_t most = kMaxStep) {
    const int64_t N = like.size(0), H = heads ? heads : like.size(1), L = like.size(2), D = like.size(3);
    return steps_lead(like, H, most) ? at::empty({L, N, H, D}, like.options()).permute({1, 2, 0, 3}) : at::empty({N, H, L, D}, like.options());
}

inline const float *floats(const at::Tensor &t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
inline float *floats_out(const at::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
inline const int64_t *whole_numbers(const at::Tensor &t) { return t.defined() ? t.const_data_ptr<int64_t>() : nullptr; }

inline at::TensorOptions fp32(const at::Tensor &t) { return t.options().dtype(at::kFloat); }
inline at::Tensor scratch(int64_t n, const at::Tensor &t) {
    if (n < 0) fail("dimensions beyond what the kernels take");
    return at::empty({std::max<int64_t>(n, 1)}, fp32(t));
}

// Room for a tensor of its own like this one, where there is one
inline at::Tensor room_like(const at::Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options()) : t; }

inline void require_sizes(std::initializer_list<int64_t> sizes) {
    for (const int64_t n : sizes)
        if (n < 1 || n > std::numeric_limits<int>::max()) fail("every dimension must be at least 1 and fit 32 bits");
}

// What autograd may have kept of a state's values is of an earlier version from here on.
inline void overwritten(const at::Tensor &t) {
    if (t.defined() && !t.is_inference()) torch::autograd::impl::bump_version(t);
}

inline void once_only() {
    if (at::GradMode::is_enabled()) fail("the gradients of this operator cannot be differentiated again (create_graph)");
}

inline bool records(std::initializer_list<const at::Tensor *> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Autograd refuses to keep an inference tensor, but only once the call is done and a state has gone on: refused before that.
inline void may_be_kept(std::initializer_list<at::Tensor> ts) {
    for (const at::Tensor &t : ts)
        if (t.defined() && t.is_inference()) fail("an inference tensor cannot be kept for a backward pass: clone it outside inference mode");
}

// A tangent of forward-mode differentiation would be lost without a word: its tensor need not require a gradient.
inline void no_tangents(std::initializer_list<const at::Tensor *> ts) {
    for (const at::Tensor *t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) fail("this operator has no forward-mode derivative: a tensor of the call has a tangent");
}

}  // namespace fwp_host
