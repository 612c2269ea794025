// What the host operators of all files share: errors of the C ABI as exceptions, pointers and streams, allocations, checks.
#pragma once
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <optional>
#include <vector>

#include "../../include/dsa_attn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void check(int rc, const char *what) {
    if (rc == 0) return;
    const std::string msg = std::string(what) + " failed (" + std::to_string(rc) + "): " + dsa_last_error();
    if (rc == DSA_ERR_ARG) TORCH_CHECK_VALUE(false, msg);
    TORCH_CHECK(false, msg);
}

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const int32_t *iptr(const Tensor &t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }
float *fptr(const Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

void need_gpu(const Tensor &t) {
    if (t.defined() && !t.is_cuda())
        TORCH_CHECK(false, "dsa attention runs on the GPU only (tensor on ", t.device().str(), "); there is no CPU path");
}

// The operators have no forward-mode derivative.  Asked of every differentiable input before anything else: a dual tensor need not
// require a gradient, so a call that builds no graph would drop its tangent without a word.
bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
void no_forward_mode(std::initializer_list<const Tensor *> inputs, const char *what) {
    for (const Tensor *t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*t), what, ": forward-mode differentiation is not implemented");
}

Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const Tensor &like) {
    return Tensor(at::detail::empty_cuda(size, dtype, like.device(), std::nullopt));
}
Tensor empty_bytes(size_t bytes, const Tensor &like) { return empty({(int64_t)std::max<size_t>(bytes, 4)}, at::kByte, like); }

bool aligned16(const Tensor &t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
// contiguous bf16 on a 16-byte boundary: keys, values and index queries go into LDS 16 bytes at a time (a view can start anywhere)
Tensor as_bf16(const Tensor &t) {
    const Tensor c = (t.scalar_type() == at::kBFloat16 ? t : t.to(at::kBFloat16)).contiguous();
    return aligned16(c) ? c : c.clone();
}

Tensor checked_cu(const Tensor &cu) {
    TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 2, "cu_seqlens must be 1-D with at least two entries");
    return (cu.scalar_type() == at::kInt ? cu : cu.to(at::kInt)).contiguous();
}

}  // namespace
