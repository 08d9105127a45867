// What the sources of liboeq_torch share.
#pragma once
#include <ATen/ATen.h>

#include "../../include/oeq_b200.h"

namespace oeq_torch {

using at::Tensor;
typedef at::ArrayRef<Tensor> Args;

inline void check(int rc) { TORCH_CHECK(rc == OEQ_OK, "oeq_b200: ", oeq_last_error()); }

inline const int64_t* index_ptr(const Tensor& t) { return static_cast<const int64_t*>(t.const_data_ptr()); }

// The gradients that an autograd node computes.  Plain CUDA tensors that nothing differentiates go straight to the
// kernels; anything else (tracing modes, tensor subclasses, batched tensors, negated or zero tensors whose memory does not
// hold their values, derivatives of the derivative) through the dispatcher.
inline bool direct(Args in) {
    using c10::DispatchKey;
    const auto tls = c10::impl::tls_local_dispatch_key_set().included_;
    if (at::GradMode::is_enabled() || tls.has(DispatchKey::Python) || tls.has(DispatchKey::PythonTLSSnapshot) ||
        tls.has(DispatchKey::FuncTorchDynamicLayerFrontMode) || tls.has(DispatchKey::Functionalize))
        return false;
    // keys of a dense CUDA tensor; a tensor with any other one is not plain
    static const uint64_t plain = c10::DispatchKeySet({DispatchKey::CUDA, DispatchKey::ADInplaceOrView, DispatchKey::AutogradCUDA, DispatchKey::AutocastCUDA}).raw_repr();
    for (const Tensor& t : in)
        if (!t.defined() || !t.is_cuda() || (t.key_set().raw_repr() & ~plain) != 0) return false;
    return true;
}

}  // namespace oeq_torch
