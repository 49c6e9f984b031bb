// What the PyTorch dispatcher kernels of the sequence operators share: types, checks and row layouts.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "convnd_hip.h"

namespace torch_convnd_hip {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<at::Tensor>;

inline bool native_type(at::ScalarType type) {
  return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

inline convnd_hip_dtype sequence_dtype(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return CONVND_HIP_FLOAT32;
    case at::kHalf:
      return CONVND_HIP_FLOAT16;
    default:
      return CONVND_HIP_BFLOAT16;
  }
}

inline void check_status(int status) {
  TORCH_CHECK(status == CONVND_HIP_SUCCESS, convnd_hip_last_error());
}

inline void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline const void* data_or_null(const OptionalTensor& t) {
  return t.has_value() ? t->const_data_ptr() : nullptr;
}

inline bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
inline bool wants_grad(const OptionalTensor& t) { return t.has_value() && wants_grad(*t); }

inline void check_once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name,
              " is differentiable once on the gfx950 kernels; use backend='torch' for "
              "create_graph=True");
}

// Rows of contiguous channels a fixed stride apart: the tensor itself where its layout allows,
// else a contiguous copy.
struct Rows {
  at::Tensor tensor;
  int64_t stride;
};
inline Rows as_rows(const at::Tensor& t) {
  const int64_t last = t.dim() - 1, channels = t.size(last);
  if (t.is_contiguous()) return {t, channels};
  bool regular = t.stride(last) == 1 || channels == 1;
  int64_t stride = -1, span = 1;
  for (int64_t a = last - 1; a >= 0 && regular; --a) {
    if (t.size(a) == 1) continue;
    if (stride < 0) stride = t.stride(a);
    regular = t.stride(a) == stride * span;
    span *= t.size(a);
  }
  if (!regular || t.numel() == 0) return {t.contiguous(), channels};
  return {t, stride < 0 ? channels : stride};
}

inline OptionalTensor contiguous(const OptionalTensor& t) {
  if (!t.has_value()) return std::nullopt;
  return t->contiguous();
}

// Rows no closer than their length, as the kernels take them.
inline Rows as_apart_rows(const at::Tensor& t) {
  auto r = as_rows(t);
  if (r.stride >= t.size(-1) && r.stride < (int64_t{1} << 21)) return r;
  return {t.contiguous(), t.size(-1)};
}

}  // namespace torch_convnd_hip
