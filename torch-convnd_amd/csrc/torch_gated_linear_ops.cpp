// PyTorch dispatcher kernels of torch_convnd::gated_linear and its backward operator, a thin layer over the
// C ABI. The schemas are defined from Python (torch_convnd/_operators.py); no counterpart in the reference.

#include "torch_sequence.h"

namespace torch_convnd_hip {
namespace {

int gated_activation(c10::string_view activation) {
  if (activation == "silu") return CONVND_HIP_ACT_SILU;
  if (activation == "relu") return CONVND_HIP_ACT_RELU;
  if (activation == "gelu") return CONVND_HIP_ACT_GELU;
  if (activation == "gelu_tanh") return CONVND_HIP_ACT_GELU_TANH;
  TORCH_CHECK(false, "gated_linear activation must be 'silu', 'relu', 'gelu' or 'gelu_tanh'");
}

std::vector<int64_t> gated_shape(const at::Tensor& input, const at::Tensor& weight) {
  auto shape = input.sizes().vec();
  shape.back() = weight.size(0) / 2;
  return shape;
}

void check_gated_input(const at::Tensor& input, const at::Tensor& weight) {
  TORCH_CHECK(native_type(input.scalar_type()),
              "native gated_linear supports float16, bfloat16 and float32");
  TORCH_CHECK(weight.dim() == 2 && input.dim() >= 1 && weight.size(0) > 0 && weight.size(0) % 2 == 0 &&
                  weight.size(1) > 0 && input.size(-1) == weight.size(1),
              "gated_linear expects an input of [..., inputs] and a weight of [2 * outputs, inputs]");
  TORCH_CHECK(weight.device() == input.device() && weight.scalar_type() == input.scalar_type(),
              "input and weight must have the same device and dtype");
}

convnd_hip_linear_problem gated_problem(const at::Tensor& input, const at::Tensor& weight, const Rows& x,
                                        int activation) {
  convnd_hip_linear_problem p{};
  p.rows = input.numel() / weight.size(1);
  p.inputs = weight.size(1);
  p.outputs = weight.size(0) / 2;
  p.input_stride = x.stride;
  p.grad_stride = p.outputs;
  p.activation = activation;
  return p;
}

std::tuple<at::Tensor, at::Tensor> gated_linear_device(const at::Tensor& input, const at::Tensor& weight,
                                                       const OptionalTensor& bias,
                                                       c10::string_view activation, bool keep) {
  const int act = gated_activation(activation);
  check_gated_input(input, weight);
  if (bias.has_value())
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0) &&
                    bias->device() == input.device() && bias->scalar_type() == input.scalar_type(),
                "bias must match the weight's rows, device and dtype");
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = as_apart_rows(input);
  const auto w = weight.contiguous();
  const auto b = contiguous(bias);
  const auto p = gated_problem(input, weight, x, act);
  const auto dtype = sequence_dtype(input);
  const auto bytes_of = input.options().dtype(at::kByte);
  auto output = at::empty(gated_shape(input, weight), input.options());
  auto kept = at::empty({keep ? static_cast<int64_t>(convnd_hip_gated_linear_kept_size(dtype, &p)) : 0}, bytes_of);
  const size_t bytes =
      convnd_hip_gated_linear_workspace_size(dtype, &p, x.tensor.const_data_ptr(), w.const_data_ptr());
  at::Tensor workspace;
  if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, bytes_of);
  check_status(convnd_hip_gated_linear(
      dtype, &p, x.tensor.const_data_ptr(), w.const_data_ptr(), data_or_null(b), output.mutable_data_ptr(),
      kept.numel() > 0 ? kept.mutable_data_ptr() : nullptr, bytes > 0 ? workspace.mutable_data_ptr() : nullptr,
      bytes, stream_of(input)));
  return {output, kept};
}

std::tuple<OptionalTensor, OptionalTensor, OptionalTensor> gated_linear_backward_device(
    const at::Tensor& grad_output, const at::Tensor& input, const at::Tensor& weight, const at::Tensor& kept,
    c10::string_view activation, std::array<bool, 3> output_mask) {
  const int act = gated_activation(activation);
  check_gated_input(input, weight);
  const auto shape = gated_shape(input, weight);
  TORCH_CHECK(grad_output.sizes() == at::IntArrayRef(shape) && grad_output.device() == input.device() &&
                  grad_output.scalar_type() == input.scalar_type(),
              "gated_linear grad_output must match the output's shape, device and dtype");
  OptionalTensor dx, dw, db;
  if (!output_mask[0] && !output_mask[1] && !output_mask[2]) return {dx, dw, db};
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = as_apart_rows(input), dy = as_apart_rows(grad_output);
  const auto w = weight.contiguous();
  auto p = gated_problem(input, weight, x, act);
  p.grad_stride = dy.stride;
  const auto dtype = sequence_dtype(input);
  TORCH_CHECK(kept.scalar_type() == at::kByte && kept.is_contiguous() && kept.device() == input.device() &&
                  kept.numel() == static_cast<int64_t>(convnd_hip_gated_linear_kept_size(dtype, &p)),
              "gated_linear kept must be what its forward kept");
  if (output_mask[0]) dx = at::empty(input.sizes(), input.options());
  if (output_mask[1]) dw = at::empty(weight.sizes(), weight.options());
  if (output_mask[2]) db = at::empty({weight.size(0)}, weight.options());
  const size_t bytes = convnd_hip_gated_linear_backward_workspace_size(
      dtype, &p, x.tensor.const_data_ptr(), w.const_data_ptr(), output_mask[0], output_mask[1], output_mask[2]);
  at::Tensor workspace;
  if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte));
  check_status(convnd_hip_gated_linear_backward(
      dtype, &p, dy.tensor.const_data_ptr(), x.tensor.const_data_ptr(), w.const_data_ptr(), kept.const_data_ptr(),
      dx.has_value() ? dx->mutable_data_ptr() : nullptr, dw.has_value() ? dw->mutable_data_ptr() : nullptr,
      db.has_value() ? db->mutable_data_ptr() : nullptr, bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes,
      stream_of(input)));
  return {dx, dw, db};
}

const auto& gated_linear_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::gated_linear", "")
                             .typed<decltype(gated_linear_device)>();
  return op;
}
const auto& gated_linear_backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::gated_linear_backward", "")
                             .typed<decltype(gated_linear_backward_device)>();
  return op;
}

class GatedLinearFunction : public torch::autograd::Function<GatedLinearFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& input, const at::Tensor& weight,
                               const OptionalTensor& bias, const std::string& activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [output, kept] = gated_linear_op().call(input, weight, bias, activation, true);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["bias"] = bias.has_value() && bias->defined();
    ctx->save_for_backward({input, weight, kept});
    ctx->mark_non_differentiable({kept});
    ctx->set_materialize_grads(false);
    return {output, kept};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_linear");
    if (!grads[0].defined()) return variable_list(4);
    at::AutoDispatchBelowADInplaceOrView below;
    const auto saved = ctx->get_saved_variables();
    const std::array<bool, 3> mask = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                      ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2)};
    auto [dx, dw, db] = gated_linear_backward_op().call(grads[0], saved[0], saved[1], saved[2],
                                                        ctx->saved_data["activation"].toStringRef(), mask);
    return {dx.value_or(at::Tensor()), dw.value_or(at::Tensor()), db.value_or(at::Tensor()), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> gated_linear_autograd(const at::Tensor& input, const at::Tensor& weight,
                                                         const OptionalTensor& bias,
                                                         c10::string_view activation, bool keep) {
  if (!at::GradMode::is_enabled() || !(wants_grad(input) || wants_grad(weight) || wants_grad(bias))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return gated_linear_op().call(input, weight, bias, activation, keep);
  }
  auto out = GatedLinearFunction::apply(input, weight, bias, std::string(activation));
  return {out[0], out[1]};
}

}  // namespace
}  // namespace torch_convnd_hip

TORCH_LIBRARY_IMPL(torch_convnd, Autograd, library) {
  library.impl("gated_linear", &torch_convnd_hip::gated_linear_autograd);
}

TORCH_LIBRARY_IMPL(torch_convnd, CUDA, library) {
  library.impl("gated_linear", &torch_convnd_hip::gated_linear_device);
  library.impl("gated_linear_backward", &torch_convnd_hip::gated_linear_backward_device);
}
