// torch_common.h -- what the modules over torch share (train_autograd.cpp, lm_autograd.cpp):
// checks of arguments, allocations on the current stream, gradients of gradients refused.
#pragma once

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "need_scan.h"

namespace need_torch {

using at::Tensor;
using torch::autograd::variable_list;

template <class... Args>
void check_value(bool ok, const Args&... args) {
    if (!ok) throw py::value_error(c10::str(args...));
}
inline void check(const char* fn, int rc) {
    if (rc != NEED_OK)
        throw std::runtime_error(c10::str(fn, " failed (status ", rc, "): ", need_last_error()));
}

inline int32_t dtype_of(at::ScalarType t) {
    return t == at::kFloat ? NEED_F32 : t == at::kBFloat16 ? NEED_BF16 : NEED_F16;
}
inline int32_t dtype_of(const Tensor& t) { return dtype_of(t.scalar_type()); }

using OptTensor = std::optional<Tensor>;
inline Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
inline OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// CUDA tensors of one device, x of a dtype the kernels take.
inline void check_tensors(const char* name, const Tensor& x, std::initializer_list<const Tensor*> others) {
    if (!x.is_cuda())
        throw std::runtime_error(c10::str(name, " takes CUDA tensors only (no CPU fallback); got ", x.sizes(), " on ", x.device()));
    for (const Tensor* t : others)
        if (t->defined() && t->device() != x.device())
            throw std::runtime_error("all tensors must be on the same CUDA device (no CPU fallback)");
    const auto ty = x.scalar_type();
    if (ty != at::kFloat && ty != at::kBFloat16 && ty != at::kHalf)
        throw py::type_error(c10::str(name, " takes fp32, bf16 or f16 data; got ", c10::toString(ty)));
}
// The reset mask as the kernels read it.
inline Tensor mask_of(const Tensor& seg, int64_t B, int64_t T) {
    if (!seg.defined()) return seg;
    check_value(seg.dim() == 2 && seg.size(0) == B && seg.size(1) == T, "seg_start must be [B, T] = [", B, ", ", T,
                "]; got ", seg.sizes());
    return seg.scalar_type() == at::kByte ? seg : seg.ne(0).to(at::kByte);
}

inline Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

inline Tensor scratch(const Tensor& like, size_t bytes) { return empty(like, {static_cast<int64_t>(bytes)}, at::kByte); }
inline Tensor floats(const Tensor& like, at::IntArrayRef shape) { return empty(like, shape, at::kFloat); }
template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
// The current stream of t's device, which is made current for the guard's life.
struct On {
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index())) {}
    c10::cuda::CUDAGuard guard;
    c10::cuda::CUDAStream stream;
};

inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Whether one of them carries a forward-mode tangent.  A node refuses it; a plain launch
// would drop it.
inline bool has_tangent(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) return true;
    return false;
}

// Under create_graph: gradients of these gradients raise instead of being left out.
inline variable_list once(variable_list g) {
    if (!at::GradMode::is_enabled()) return g;
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "need_b200: the training operators have no second derivative", static_cast<int>(g.size()));
    variable_list in;
    for (Tensor& t : g) in.push_back(t.defined() ? t.detach().requires_grad_() : t);
    return (*node)(std::move(in));
}

// The distance of t's rows (all dims but the last, as one) where they are evenly
// apart with channel stride 1; else 0.
inline int64_t row_stride(const Tensor& t) {
    if (t.stride(-1) != 1 && t.size(-1) > 1) return 0;
    int64_t step = 0, next = 0;  // of the innermost dim of more than one, and what the next must be
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (step == 0) step = t.stride(d);
        else if (t.stride(d) != next) return 0;
        if (step <= 0) return 0;
        next = t.stride(d) * t.size(d);
    }
    return step == 0 ? t.size(-1) : step;
}
inline Tensor even_rows(const Tensor& t) { return row_stride(t) != 0 ? t : t.clone(at::MemoryFormat::Contiguous); }

}  // namespace need_torch
