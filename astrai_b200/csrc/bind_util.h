// What the bindings of short calls share.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <torch/extension.h>

namespace astrai_bind {

using OptTensor = c10::optional<at::Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Uninitialised memory straight from the caching allocator: a call of a few microseconds feels the dispatcher's share
// of at::empty.
inline at::Tensor new_like(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, t.device(), c10::nullopt));
}

// starts on a 16-byte boundary, as the kernels' widest loads and bulk copies want it
inline bool on_grid(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

inline cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

}  // namespace astrai_bind
