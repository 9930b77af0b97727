// What the torch dispatcher operators over the C ABI share: checks of tensors, the current stream
// and a workspace of a call's own.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <tuple>

#include "mtl_gptq.h"
#include "mtl_paged.h"

namespace mtl_ops {

using OptTensor = c10::optional<at::Tensor>;

inline void check_status(int status, const char* what) {
  TORCH_CHECK(status == 0, what, ": ", mtl_status_string(status), " (status ", status, ")");
}

inline int32_t row_type(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "expected ", name,
              " to be bfloat16 or float16, got ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? MTL_T_BF16 : MTL_T_F16;
}

inline void check_same_device(const at::Tensor& a, std::initializer_list<const at::Tensor*> others,
                              const char* what = "the paged cache") {
  TORCH_CHECK(a.is_cuda() || a.is_meta(), what, " runs on a HIP device");
  for (const at::Tensor* t : others)
    TORCH_CHECK(t->device() == a.device(), "all tensors must be on one HIP device, got ",
                a.device(), " and ", t->device());
}

// A dimension's stride, 0 where the dimension has one element and torch's number means nothing.
inline int64_t step(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// The tensors' memory: null for meta tensors, which make the checks only.
template <class T>
T* ptr(const at::Tensor& t) {
  return t.is_meta() ? nullptr : static_cast<T*>(t.data_ptr());
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A tensor that is written (at most 5 dimensions): no two of its elements may be the same memory.
// Each stride has to pass over all that the smaller ones reach.
inline void check_apart(const at::Tensor& t, const char* name) {
  if (t.numel() == 0) return;
  std::array<std::pair<int64_t, int64_t>, 5> dims;
  int64_t n = 0;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims[n++] = {t.stride(d), t.size(d)};
  std::sort(dims.begin(), dims.begin() + n);
  int64_t reach = 1;
  for (int64_t i = 0; i < n; ++i) {
    const auto& [stride, size] = dims[i];
    TORCH_CHECK(stride >= reach, name, "'s elements overlap, several of them are a single memory "
                "location: ", t.sizes(), " with strides ", t.strides());
    reach += (size - 1) * stride;
  }
}

inline hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// Memory of a call's own from torch's caching allocator, without a tensor around it.
struct Workspace {
  c10::DataPtr data;
  int64_t bytes;
  Workspace(const at::Tensor& like, int64_t n)
      : data(n > 0 ? c10::GetAllocator(like.device().type())->allocate(n) : c10::DataPtr()),
        bytes(n) {}
  void* get() const { return data.get(); }
};

}  // namespace mtl_ops
