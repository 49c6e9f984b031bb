// PyTorch dispatcher kernels of the sequence operators: torch_convnd::layer_norm, linear_act and
// gated_recurrence with their backward operators, a thin layer over the C ABI. The
// schemas are defined from Python (torch_convnd/_operators.py); no counterpart in the reference.

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
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<at::Tensor>;

bool native_type(at::ScalarType type) {
  return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

convnd_hip_dtype sequence_dtype(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return CONVND_HIP_FLOAT32;
    case at::kHalf:
      return CONVND_HIP_FLOAT16;
    default:
      return CONVND_HIP_BFLOAT16;
  }
}

void check_status(int status) {
  TORCH_CHECK(status == CONVND_HIP_SUCCESS, convnd_hip_last_error());
}

void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

const void* data_or_null(const OptionalTensor& t) {
  return t.has_value() ? t->const_data_ptr() : nullptr;
}

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptionalTensor& t) { return t.has_value() && wants_grad(*t); }

void check_once(const char* name) {
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
Rows as_rows(const at::Tensor& t) {
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

// ---- layer norm ----------------------------------------------------------------------------

void check_norm_parameter(const OptionalTensor& p, const at::Tensor& input, const char* name) {
  if (!p.has_value()) return;
  TORCH_CHECK(p->dim() == 1 && p->size(0) == input.size(-1) && p->device() == input.device() &&
                  (p->scalar_type() == input.scalar_type() || p->scalar_type() == at::kFloat),
              "layer_norm ", name,
              " must match the input's channels and device, in its dtype or float32");
}

void check_norm_input(const at::Tensor& input, const OptionalTensor& weight,
                      const OptionalTensor& bias) {
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) > 0,
              "layer_norm expects an input with channels in its last dimension");
  TORCH_CHECK(native_type(input.scalar_type()),
              "native layer_norm supports float16, bfloat16 and float32");
  check_norm_parameter(weight, input, "weight");
  check_norm_parameter(bias, input, "bias");
  TORCH_CHECK(!weight.has_value() || !bias.has_value() ||
                  weight->scalar_type() == bias->scalar_type(),
              "layer_norm weight and bias must have the same dtype");
}

convnd_hip_dtype parameter_dtype(const at::Tensor& input, const OptionalTensor& weight,
                                 const OptionalTensor& bias) {
  if (weight.has_value()) return sequence_dtype(*weight);
  return bias.has_value() ? sequence_dtype(*bias) : sequence_dtype(input);
}

OptionalTensor contiguous(const OptionalTensor& t) {
  if (!t.has_value()) return std::nullopt;
  return t->contiguous();
}

std::tuple<at::Tensor, at::Tensor> layer_norm_device(const at::Tensor& input,
                                                     const OptionalTensor& weight,
                                                     const OptionalTensor& bias, double eps,
                                                     bool keep_statistics) {
  check_norm_input(input, weight, bias);
  const c10::OptionalDeviceGuard guard(input.device());
  const int64_t channels = input.size(-1), rows = input.numel() / channels;
  const auto x = as_rows(input);
  const auto w = contiguous(weight), b = contiguous(bias);
  auto output = at::empty(input.sizes(), input.options());
  auto statistics = at::empty({2, keep_statistics ? rows : 0}, input.options().dtype(at::kFloat));
  float* mean = keep_statistics && rows > 0 ? statistics.mutable_data_ptr<float>() : nullptr;
  check_status(convnd_hip_layer_norm(
      sequence_dtype(input), parameter_dtype(input, weight, bias), x.tensor.const_data_ptr(),
      x.stride, data_or_null(w), data_or_null(b), output.mutable_data_ptr(), mean,
      mean == nullptr ? nullptr : mean + rows, rows, channels, eps, stream_of(input)));
  return {output, statistics};
}

std::tuple<OptionalTensor, OptionalTensor, OptionalTensor> layer_norm_backward_device(
    const at::Tensor& grad_output, const at::Tensor& input, const OptionalTensor& weight,
    const OptionalTensor& bias, const at::Tensor& statistics, std::array<bool, 3> output_mask) {
  check_norm_input(input, weight, bias);
  const int64_t channels = input.size(-1), rows = input.numel() / channels;
  TORCH_CHECK(grad_output.sizes() == input.sizes() && grad_output.device() == input.device() &&
                  grad_output.scalar_type() == input.scalar_type(),
              "layer_norm grad_output must match the input's shape, device and dtype");
  TORCH_CHECK(statistics.scalar_type() == at::kFloat && statistics.numel() == 2 * rows &&
                  statistics.is_contiguous() && statistics.device() == input.device(),
              "layer_norm statistics must be those its forward kept");
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = as_rows(input), dy = as_rows(grad_output);
  const auto w = contiguous(weight);
  OptionalTensor dx, dw, db;
  if (output_mask[0]) dx = at::empty(input.sizes(), input.options());
  if (output_mask[1] && weight.has_value()) dw = at::empty({channels}, weight->options());
  if (output_mask[2] && bias.has_value()) db = at::empty({channels}, bias->options());
  const auto dtype = sequence_dtype(input);
  const size_t bytes = dw.has_value() || db.has_value()
                           ? convnd_hip_layer_norm_backward_workspace_size(dtype, rows, channels)
                           : 0;
  auto workspace = at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte));
  const float* mean = rows > 0 ? statistics.const_data_ptr<float>() : nullptr;
  check_status(convnd_hip_layer_norm_backward(
      dtype, parameter_dtype(input, weight, bias), dy.tensor.const_data_ptr(), dy.stride,
      x.tensor.const_data_ptr(), x.stride, data_or_null(w), mean,
      rows > 0 ? mean + rows : nullptr, dx.has_value() ? dx->mutable_data_ptr() : nullptr,
      dw.has_value() ? dw->mutable_data_ptr() : nullptr,
      db.has_value() ? db->mutable_data_ptr() : nullptr, rows, channels,
      bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, stream_of(input)));
  return {dx, dw, db};
}

const auto& layer_norm_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::layer_norm", "")
                             .typed<decltype(layer_norm_device)>();
  return op;
}
const auto& layer_norm_backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::layer_norm_backward", "")
                             .typed<decltype(layer_norm_backward_device)>();
  return op;
}

class LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& input,
                               const OptionalTensor& weight, const OptionalTensor& bias,
                               double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [output, statistics] = layer_norm_op().call(input, weight, bias, eps, true);
    ctx->save_for_backward({input, weight.value_or(at::Tensor()), bias.value_or(at::Tensor()),
                            statistics});
    ctx->mark_non_differentiable({statistics});
    ctx->set_materialize_grads(false);
    return {output, statistics};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const auto optional = [](const at::Tensor& t) {
      return t.defined() ? OptionalTensor(t) : std::nullopt;
    };
    if (!grads[0].defined()) return variable_list(4);
    // Refused above where it would be differentiated, so no autograd kernel is needed below.
    at::AutoDispatchBelowADInplaceOrView below;
    // Needed edges are counted over the tensors that were given.
    int edge = 0;
    std::array<bool, 3> mask{};
    for (int i = 0; i < 3; ++i)
      if (saved[i].defined()) mask[i] = ctx->needs_input_grad(edge++);
    auto [dx, dw, db] = layer_norm_backward_op().call(
        grads[0], saved[0], optional(saved[1]), optional(saved[2]), saved[3], mask);
    return {dx.value_or(at::Tensor()), dw.value_or(at::Tensor()), db.value_or(at::Tensor()),
            at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> layer_norm_autograd(const at::Tensor& input,
                                                       const OptionalTensor& weight,
                                                       const OptionalTensor& bias, double eps,
                                                       bool keep_statistics) {
  if (!at::GradMode::is_enabled() ||
      !(wants_grad(input) || wants_grad(weight) || wants_grad(bias))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_op().call(input, weight, bias, eps, keep_statistics);
  }
  auto out = LayerNormFunction::apply(input, weight, bias, eps);
  return {out[0], out[1]};
}

// ---- linear --------------------------------------------------------------------------------

int linear_activation(c10::string_view activation) {
  if (activation == "none") return CONVND_HIP_ACT_NONE;
  if (activation == "relu") return CONVND_HIP_ACT_RELU;
  if (activation == "gelu") return CONVND_HIP_ACT_GELU;
  if (activation == "gelu_tanh") return CONVND_HIP_ACT_GELU_TANH;
  TORCH_CHECK(false, "activation must be 'none', 'relu', 'gelu' or 'gelu_tanh'");
}

std::vector<int64_t> linear_shape(const at::Tensor& input, const at::Tensor& weight) {
  auto shape = input.sizes().vec();
  shape.back() = weight.size(0);
  return shape;
}

void check_linear_input(const at::Tensor& input, const at::Tensor& weight) {
  TORCH_CHECK(native_type(input.scalar_type()),
              "native linear_act supports float16, bfloat16 and float32");
  TORCH_CHECK(weight.dim() == 2 && input.dim() >= 1 && weight.size(0) > 0 && weight.size(1) > 0 &&
                  input.size(-1) == weight.size(1),
              "linear_act expects an input of [..., inputs] and a weight of [outputs, inputs]");
  TORCH_CHECK(weight.device() == input.device() && weight.scalar_type() == input.scalar_type(),
              "input and weight must have the same device and dtype");
}

// Rows no closer than their length, as the kernels take them.
Rows as_apart_rows(const at::Tensor& t) {
  auto r = as_rows(t);
  if (r.stride >= t.size(-1) && r.stride < (int64_t{1} << 21)) return r;
  return {t.contiguous(), t.size(-1)};
}

convnd_hip_linear_problem linear_problem(const at::Tensor& input, const at::Tensor& weight,
                                         const Rows& x, int activation) {
  convnd_hip_linear_problem p{};
  p.rows = input.numel() / weight.size(1);
  p.inputs = weight.size(1);
  p.outputs = weight.size(0);
  p.input_stride = x.stride;
  p.residual_stride = p.grad_stride = p.outputs;
  p.activation = activation;
  return p;
}

// The element type of the kept slopes.
at::ScalarType slope_type(const at::Tensor& input) {
  return input.scalar_type() == at::kFloat ? at::kFloat : at::kShort;
}

std::tuple<at::Tensor, at::Tensor> linear_act_device(const at::Tensor& input,
                                                     const at::Tensor& weight,
                                                     const OptionalTensor& bias,
                                                     const OptionalTensor& residual,
                                                     c10::string_view activation, bool keep_slope) {
  const int act = linear_activation(activation);
  check_linear_input(input, weight);
  if (bias.has_value())
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0) &&
                    bias->device() == input.device() && bias->scalar_type() == input.scalar_type(),
                "bias must match the outputs, device and dtype");
  const auto shape = linear_shape(input, weight);
  if (residual.has_value())
    TORCH_CHECK(residual->sizes() == at::IntArrayRef(shape) &&
                    residual->device() == input.device() &&
                    residual->scalar_type() == input.scalar_type(),
                "residual must match the output's shape, device and dtype");
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = as_apart_rows(input);
  const auto w = weight.contiguous();
  const auto b = contiguous(bias);
  auto p = linear_problem(input, weight, x, act);
  Rows r;
  if (residual.has_value()) {
    r = as_apart_rows(*residual);
    p.residual_stride = r.stride;
  }
  const auto dtype = sequence_dtype(input);
  auto output = at::empty(shape, input.options());
  const bool keep = keep_slope && act != CONVND_HIP_ACT_NONE;
  const auto kept = input.options().dtype(slope_type(input));
  auto slope = keep ? at::empty(shape, kept) : at::empty({0}, kept);
  const size_t bytes =
      convnd_hip_linear_workspace_size(dtype, &p, x.tensor.const_data_ptr(), w.const_data_ptr());
  at::Tensor workspace;
  if (bytes > 0)
    workspace = at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte));
  check_status(convnd_hip_linear(
      dtype, &p, x.tensor.const_data_ptr(), w.const_data_ptr(), data_or_null(b),
      residual.has_value() ? r.tensor.const_data_ptr() : nullptr, output.mutable_data_ptr(),
      keep ? slope.mutable_data_ptr() : nullptr, bytes > 0 ? workspace.mutable_data_ptr() : nullptr,
      bytes, stream_of(input)));
  return {output, slope};
}

std::tuple<OptionalTensor, OptionalTensor, OptionalTensor> linear_act_backward_device(
    const at::Tensor& grad_output, const at::Tensor& input, const at::Tensor& weight,
    const at::Tensor& slope, c10::string_view activation, std::array<bool, 3> output_mask) {
  const int act = linear_activation(activation);
  check_linear_input(input, weight);
  const auto shape = linear_shape(input, weight);
  TORCH_CHECK(grad_output.sizes() == at::IntArrayRef(shape) &&
                  grad_output.device() == input.device() &&
                  grad_output.scalar_type() == input.scalar_type(),
              "linear_act grad_output must match the output's shape, device and dtype");
  TORCH_CHECK(act == CONVND_HIP_ACT_NONE ||
                  (slope.sizes() == at::IntArrayRef(shape) && slope.is_contiguous() &&
                   slope.device() == input.device() && slope.scalar_type() == slope_type(input)),
              "linear_act slope must be what its forward kept");
  OptionalTensor dx, dw, db;
  if (!output_mask[0] && !output_mask[1] && !output_mask[2]) return {dx, dw, db};
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = as_apart_rows(input), dy = as_apart_rows(grad_output);
  const auto w = weight.contiguous();
  auto p = linear_problem(input, weight, x, act);
  p.grad_stride = dy.stride;
  if (output_mask[0]) dx = at::empty(input.sizes(), input.options());
  if (output_mask[1]) dw = at::empty(weight.sizes(), weight.options());
  if (output_mask[2]) db = at::empty({p.outputs}, weight.options());
  const auto dtype = sequence_dtype(input);
  const size_t bytes = convnd_hip_linear_backward_workspace_size(
      dtype, &p, dy.tensor.const_data_ptr(), x.tensor.const_data_ptr(), w.const_data_ptr(),
      output_mask[0], output_mask[1], output_mask[2]);
  at::Tensor workspace;
  if (bytes > 0)
    workspace = at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte));
  check_status(convnd_hip_linear_backward(
      dtype, &p, dy.tensor.const_data_ptr(), x.tensor.const_data_ptr(), w.const_data_ptr(),
      act != CONVND_HIP_ACT_NONE ? slope.const_data_ptr() : nullptr,
      dx.has_value() ? dx->mutable_data_ptr() : nullptr,
      dw.has_value() ? dw->mutable_data_ptr() : nullptr,
      db.has_value() ? db->mutable_data_ptr() : nullptr,
      bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, stream_of(input)));
  return {dx, dw, db};
}

const auto& linear_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::linear_act", "")
                             .typed<decltype(linear_act_device)>();
  return op;
}
const auto& linear_backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::linear_act_backward", "")
                             .typed<decltype(linear_act_backward_device)>();
  return op;
}

class LinearActFunction : public torch::autograd::Function<LinearActFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& input,
                               const at::Tensor& weight, const OptionalTensor& bias,
                               const OptionalTensor& residual, const std::string& activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [output, slope] = linear_op().call(input, weight, bias, residual, activation, true);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({input, weight, slope});
    ctx->mark_non_differentiable({slope});
    ctx->set_materialize_grads(false);
    return {output, slope};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("linear_act");
    if (!grads[0].defined()) return variable_list(5);
    at::AutoDispatchBelowADInplaceOrView below;
    const auto saved = ctx->get_saved_variables();
    const bool bias = ctx->saved_data["bias"].toBool();
    const bool residual = ctx->saved_data["residual"].toBool();
    const std::array<bool, 3> mask = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                      bias && ctx->needs_input_grad(2)};
    auto [dx, dw, db] =
        linear_backward_op().call(grads[0], saved[0], saved[1], saved[2],
                                  ctx->saved_data["activation"].toStringRef(), mask);
    return {dx.value_or(at::Tensor()), dw.value_or(at::Tensor()), db.value_or(at::Tensor()),
            residual ? grads[0] : at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> linear_act_autograd(const at::Tensor& input,
                                                       const at::Tensor& weight,
                                                       const OptionalTensor& bias,
                                                       const OptionalTensor& residual,
                                                       c10::string_view activation, bool keep_slope) {
  if (!at::GradMode::is_enabled() || !(wants_grad(input) || wants_grad(weight) ||
                                       wants_grad(bias) || wants_grad(residual))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_op().call(input, weight, bias, residual, activation, keep_slope);
  }
  auto out = LinearActFunction::apply(input, weight, bias, residual, std::string(activation));
  return {out[0], out[1]};
}

// ---- gated recurrence ------------------------------------------------------------------------

void check_recurrence_input(const at::Tensor& input, const at::Tensor& gate,
                            const OptionalTensor& lengths) {
  TORCH_CHECK(input.dim() == 3 && input.size(2) > 0,
              "gated_recurrence expects an input of [batch, tokens, channels]");
  TORCH_CHECK(native_type(input.scalar_type()),
              "native gated_recurrence supports float16, bfloat16 and float32");
  TORCH_CHECK(gate.sizes() == input.sizes() && gate.device() == input.device() &&
                  gate.scalar_type() == input.scalar_type(),
              "gated_recurrence gate must match the input's shape, device and dtype");
  if (lengths.has_value())
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == input.size(0) &&
                    lengths->device() == input.device() &&
                    (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong),
                "gated_recurrence lengths must be int32 or int64 of [batch] on the input's device");
}

void check_state(const OptionalTensor& state, const at::Tensor& input, const char* name) {
  if (!state.has_value()) return;
  TORCH_CHECK(state->dim() == 2 && state->size(0) == input.size(0) &&
                  state->size(1) == input.size(2) && state->device() == input.device() &&
                  state->scalar_type() == at::kFloat,
              "gated_recurrence ", name, " must be float32 of [batch, channels] on the input's device");
}

// The tensor itself where its channels are contiguous and its tokens neither overlap nor lie too
// far apart for the kernels' offsets, else a contiguous copy.
at::Tensor token_rows(const at::Tensor& t) {
  const bool direct = (t.stride(2) == 1 || t.size(2) == 1) && t.stride(1) >= t.size(2) &&
                      t.stride(1) < (int64_t{1} << 21);
  if (direct) return t;
  // A single token's stride may be anything, a copy's too.
  return t.size(1) == 1 ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}

convnd_hip_recurrence_problem recurrence_problem(const at::Tensor& x, const at::Tensor& g,
                                                 const OptionalTensor& lengths) {
  convnd_hip_recurrence_problem p{};
  p.batch = x.size(0);
  p.tokens = x.size(1);
  p.channels = x.size(2);
  p.input_batch = x.stride(0);
  p.input_token = x.stride(1);
  p.gate_batch = g.stride(0);
  p.gate_token = g.stride(1);
  p.wide_lengths = lengths.has_value() && lengths->scalar_type() == at::kLong;
  return p;
}

at::Tensor recurrence_workspace(const convnd_hip_recurrence_problem& p, const at::Tensor& input) {
  const size_t bytes = convnd_hip_recurrence_workspace_size(sequence_dtype(input), &p);
  if (bytes == 0) return at::Tensor();
  return at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_recurrence_device(
    const at::Tensor& input, const at::Tensor& gate, const OptionalTensor& first,
    const OptionalTensor& lengths, bool keep_carries) {
  check_recurrence_input(input, gate, lengths);
  check_state(first, input, "initial_state");
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = token_rows(input), g = token_rows(gate);
  const auto f = contiguous(first), n = contiguous(lengths);
  const auto p = recurrence_problem(x, g, lengths);
  const auto single = input.options().dtype(at::kFloat);
  auto output = at::empty(input.sizes(), input.options());
  auto last = at::empty({p.batch, p.channels}, single);
  auto carries = at::empty(
      {keep_carries ? p.batch : 0, convnd_hip_recurrence_carries(p.tokens), p.channels}, single);
  auto workspace = recurrence_workspace(p, input);
  check_status(convnd_hip_recurrence(
      sequence_dtype(input), &p, x.const_data_ptr(), g.const_data_ptr(),
      f.has_value() ? f->const_data_ptr<float>() : nullptr, data_or_null(n),
      output.mutable_data_ptr(), last.mutable_data_ptr<float>(),
      keep_carries && carries.numel() > 0 ? carries.mutable_data_ptr<float>() : nullptr,
      workspace.defined() ? workspace.mutable_data_ptr() : nullptr,
      workspace.defined() ? workspace.numel() : 0, stream_of(input)));
  return {output, last, carries};
}

std::tuple<at::Tensor, at::Tensor, OptionalTensor> gated_recurrence_backward_device(
    const at::Tensor& grad_output, const OptionalTensor& grad_last, const at::Tensor& input,
    const at::Tensor& gate, const OptionalTensor& lengths, const at::Tensor& carries,
    bool need_first) {
  check_recurrence_input(input, gate, lengths);
  check_state(grad_last, input, "grad_last");
  TORCH_CHECK(grad_output.sizes() == input.sizes() && grad_output.device() == input.device() &&
                  grad_output.scalar_type() == input.scalar_type(),
              "gated_recurrence grad_output must match the input's shape, device and dtype");
  TORCH_CHECK(carries.scalar_type() == at::kFloat && carries.is_contiguous() &&
                  carries.device() == input.device() &&
                  carries.numel() == input.size(0) * input.size(2) *
                                         convnd_hip_recurrence_carries(input.size(1)),
              "gated_recurrence carries must be those its forward kept");
  const c10::OptionalDeviceGuard guard(input.device());
  const auto x = token_rows(input), g = token_rows(gate);
  const auto dy = grad_output.contiguous();
  const auto dl = contiguous(grad_last), n = contiguous(lengths);
  const auto p = recurrence_problem(x, g, lengths);
  auto dx = at::empty(input.sizes(), input.options());
  auto dg = at::empty(input.sizes(), input.options());
  OptionalTensor df;
  if (need_first) df = at::empty({p.batch, p.channels}, input.options().dtype(at::kFloat));
  auto workspace = recurrence_workspace(p, input);
  check_status(convnd_hip_recurrence_backward(
      sequence_dtype(input), &p, dy.const_data_ptr(),
      dl.has_value() ? dl->const_data_ptr<float>() : nullptr, x.const_data_ptr(),
      g.const_data_ptr(), data_or_null(n), carries.const_data_ptr<float>(), dx.mutable_data_ptr(),
      dg.mutable_data_ptr(), df.has_value() ? df->mutable_data_ptr<float>() : nullptr,
      workspace.defined() ? workspace.mutable_data_ptr() : nullptr,
      workspace.defined() ? workspace.numel() : 0, stream_of(input)));
  return {dx, dg, df};
}

const auto& recurrence_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::gated_recurrence", "")
                             .typed<decltype(gated_recurrence_device)>();
  return op;
}
const auto& recurrence_backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::gated_recurrence_backward", "")
                             .typed<decltype(gated_recurrence_backward_device)>();
  return op;
}

class RecurrenceFunction : public torch::autograd::Function<RecurrenceFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& input,
                               const at::Tensor& gate, const OptionalTensor& first,
                               const OptionalTensor& lengths) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [output, last, carries] = recurrence_op().call(input, gate, first, lengths, true);
    ctx->saved_data["first"] = first.has_value() && first->defined();
    ctx->save_for_backward({input, gate, lengths.value_or(at::Tensor()), carries});
    ctx->mark_non_differentiable({carries});
    ctx->set_materialize_grads(false);
    return {output, last, carries};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_recurrence");
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
    at::AutoDispatchBelowADInplaceOrView below;
    const auto saved = ctx->get_saved_variables();
    const auto optional = [](const at::Tensor& t) {
      return t.defined() ? OptionalTensor(t) : std::nullopt;
    };
    const auto dy = grads[0].defined() ? grads[0] : at::zeros_like(saved[0]);
    const bool need_first = ctx->saved_data["first"].toBool() && ctx->needs_input_grad(2);
    auto [dx, dg, df] =
        recurrence_backward_op().call(dy, optional(grads[1]), saved[0], saved[1],
                                      optional(saved[2]), saved[3], need_first);
    return {dx, dg, df.value_or(at::Tensor()), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_recurrence_autograd(
    const at::Tensor& input, const at::Tensor& gate, const OptionalTensor& first,
    const OptionalTensor& lengths, bool keep_carries) {
  if (!at::GradMode::is_enabled() ||
      !(wants_grad(input) || wants_grad(gate) || wants_grad(first))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return recurrence_op().call(input, gate, first, lengths, keep_carries);
  }
  auto out = RecurrenceFunction::apply(input, gate, first, lengths);
  return {out[0], out[1], out[2]};
}

}  // namespace
}  // namespace torch_convnd_hip

TORCH_LIBRARY_IMPL(torch_convnd, Autograd, library) {
  library.impl("layer_norm", &torch_convnd_hip::layer_norm_autograd);
  library.impl("linear_act", &torch_convnd_hip::linear_act_autograd);
  library.impl("gated_recurrence", &torch_convnd_hip::gated_recurrence_autograd);
}

TORCH_LIBRARY_IMPL(torch_convnd, CUDA, library) {
  library.impl("layer_norm", &torch_convnd_hip::layer_norm_device);
  library.impl("layer_norm_backward", &torch_convnd_hip::layer_norm_backward_device);
  library.impl("linear_act", &torch_convnd_hip::linear_act_device);
  library.impl("linear_act_backward", &torch_convnd_hip::linear_act_backward_device);
  library.impl("gated_recurrence", &torch_convnd_hip::gated_recurrence_device);
  library.impl("gated_recurrence_backward", &torch_convnd_hip::gated_recurrence_backward_device);
}
