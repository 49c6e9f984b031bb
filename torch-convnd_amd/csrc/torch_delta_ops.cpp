// PyTorch dispatcher kernels of torch_convnd::gated_delta_rule and its backward operator, a thin layer
// over the C ABI. The schemas are defined from Python (torch_convnd/_operators.py); no counterpart in the
// reference.

#include "torch_sequence.h"

namespace torch_convnd_hip {
namespace {

void check_delta_inputs(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                        const at::Tensor& decay, const at::Tensor& beta, const OptionalTensor& lengths) {
  TORCH_CHECK(native_type(query.scalar_type()),
              "native gated_delta_rule supports float16, bfloat16 and float32");
  TORCH_CHECK(query.dim() == 4 && key.sizes() == query.sizes() && query.size(2) > 0 && query.size(3) > 0,
              "gated_delta_rule expects query and key of [batch, tokens, key_heads, key_size]");
  TORCH_CHECK(value.dim() == 4 && value.size(0) == query.size(0) && value.size(1) == query.size(1) &&
                  value.size(2) > 0 && value.size(3) > 0 && value.size(2) % query.size(2) == 0,
              "gated_delta_rule expects a value of [batch, tokens, heads, value_size], heads a multiple of "
              "key_heads");
  const at::IntArrayRef gates = value.sizes().slice(0, 3);
  TORCH_CHECK(decay.sizes() == gates && beta.sizes() == gates,
              "gated_delta_rule expects decay and beta of [batch, tokens, heads]");
  for (const auto* t : {&key, &value})
    TORCH_CHECK(t->device() == query.device() && t->scalar_type() == query.scalar_type(),
                "gated_delta_rule query, key and value must have the same device and dtype");
  TORCH_CHECK(decay.device() == query.device() && beta.device() == query.device() &&
                  beta.scalar_type() == decay.scalar_type() &&
                  (decay.scalar_type() == query.scalar_type() || decay.scalar_type() == at::kFloat),
              "gated_delta_rule decay and beta must be on the inputs' device, both of their dtype or float32");
  TORCH_CHECK(query.size(3) <= 128 && value.size(3) <= 65535,
              "native gated_delta_rule supports key sizes up to 128 and value sizes up to 65535; use "
              "backend='torch'");
  if (lengths.has_value())
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == query.size(0) && lengths->device() == query.device() &&
                    (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong),
                "gated_delta_rule lengths must be int32 or int64 of [batch] on the inputs' device");
}

void check_delta_state(const OptionalTensor& state, const at::Tensor& query, const at::Tensor& value,
                       const char* name) {
  if (!state.has_value()) return;
  TORCH_CHECK(state->dim() == 4 && state->size(0) == query.size(0) && state->size(1) == value.size(2) &&
                  state->size(2) == query.size(3) && state->size(3) == value.size(3) &&
                  state->device() == query.device() && state->scalar_type() == at::kFloat,
              "gated_delta_rule ", name,
              " must be float32 of [batch, heads, key_size, value_size] on the inputs' device");
}

// The tensor itself where its last axis is contiguous and its tokens lie near enough for the kernels'
// offsets, else a contiguous copy.
at::Tensor head_rows(const at::Tensor& t) {
  const bool direct = (t.stride(3) == 1 || t.size(3) == 1) && t.stride(1) < (int64_t{1} << 21);
  if (direct) return t;
  // A single token's stride may be anything, a copy's too.
  return t.size(1) == 1 ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}

// Inputs as the kernels read them, and their description.
struct DeltaCall {
  at::Tensor query, key, value;
  OptionalTensor lengths;
  convnd_hip_delta_problem problem{};
  convnd_hip_dtype dtype;

  DeltaCall(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& decay,
            const at::Tensor& beta, const OptionalTensor& n, double scale, bool normalize)
      : query(head_rows(q)), key(head_rows(k)), value(head_rows(v)), lengths(contiguous(n)),
        dtype(sequence_dtype(q)) {
    auto& p = problem;
    p.batch = q.size(0);
    p.tokens = q.size(1);
    p.key_heads = q.size(2);
    p.heads = v.size(2);
    p.key_size = q.size(3);
    p.value_size = v.size(3);
    strides(query, &p.query_batch);
    strides(key, &p.key_batch);
    strides(value, &p.value_batch);
    strides(decay, &p.decay_batch);
    strides(beta, &p.beta_batch);
    p.scale = scale;
    p.normalize = normalize;
    p.gate_dtype = sequence_dtype(decay);
    p.wide_lengths = n.has_value() && n->scalar_type() == at::kLong;
  }

  // Three strides that follow each other in the problem: of the batch, the tokens and the heads.
  static void strides(const at::Tensor& t, int64_t* at) {
    for (int i = 0; i < 3; ++i) at[i] = t.stride(i);
  }
};

at::Tensor workspace_of(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> delta_device(
    const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, const at::Tensor& decay,
    const at::Tensor& beta, const OptionalTensor& first, const OptionalTensor& lengths, double scale,
    bool normalize, bool keep) {
  check_delta_inputs(query, key, value, decay, beta, lengths);
  check_delta_state(first, query, value, "initial_state");
  const c10::OptionalDeviceGuard guard(query.device());
  const DeltaCall c(query, key, value, decay, beta, lengths, scale, normalize);
  const auto f = contiguous(first);
  const auto& p = c.problem;
  auto output = at::empty(value.sizes(), value.options());
  auto last = at::empty({p.batch, p.heads, p.key_size, p.value_size}, query.options().dtype(at::kFloat));
  auto saved = at::empty({keep ? convnd_hip_delta_saved(c.dtype, &p) : 0}, query.options());
  const bool saving = keep && saved.numel() > 0;
  const size_t bytes =
      convnd_hip_delta_workspace_size(c.dtype, &p, c.query.const_data_ptr(), c.key.const_data_ptr(),
                                      c.value.const_data_ptr(), saving);
  auto workspace = workspace_of(bytes, query);
  check_status(convnd_hip_delta(
      c.dtype, &p, c.query.const_data_ptr(), c.key.const_data_ptr(), c.value.const_data_ptr(),
      decay.const_data_ptr(), beta.const_data_ptr(), f.has_value() ? f->const_data_ptr<float>() : nullptr,
      data_or_null(c.lengths), output.mutable_data_ptr(), last.mutable_data_ptr<float>(),
      saving ? saved.mutable_data_ptr() : nullptr, bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes,
      stream_of(query)));
  return {output, last, saved};
}

using DeltaGrads = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, OptionalTensor>;

DeltaGrads delta_backward_device(const at::Tensor& grad_output, const OptionalTensor& grad_last,
                                 const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                                 const at::Tensor& decay, const at::Tensor& beta,
                                 const OptionalTensor& lengths, const at::Tensor& saved, double scale,
                                 bool normalize, bool need_first) {
  check_delta_inputs(query, key, value, decay, beta, lengths);
  check_delta_state(grad_last, query, value, "grad_last");
  TORCH_CHECK(grad_output.sizes() == value.sizes() && grad_output.device() == value.device() &&
                  grad_output.scalar_type() == value.scalar_type(),
              "gated_delta_rule grad_output must match the value's shape, device and dtype");
  const c10::OptionalDeviceGuard guard(query.device());
  DeltaCall c(query, key, value, decay, beta, lengths, scale, normalize);
  auto& p = c.problem;
  TORCH_CHECK(saved.scalar_type() == query.scalar_type() && saved.is_contiguous() &&
                  saved.device() == query.device() && saved.numel() == convnd_hip_delta_saved(c.dtype, &p),
              "gated_delta_rule saved must be what its forward kept");
  const auto dy = head_rows(grad_output);
  DeltaCall::strides(dy, &p.grad_batch);
  const auto dl = contiguous(grad_last);
  auto dq = at::empty(query.sizes(), query.options()), dk = at::empty(key.sizes(), key.options());
  auto dv = at::empty(value.sizes(), value.options());
  auto dg = at::empty(decay.sizes(), decay.options()), db = at::empty(beta.sizes(), beta.options());
  OptionalTensor df;
  if (need_first)
    df = at::empty({p.batch, p.heads, p.key_size, p.value_size}, query.options().dtype(at::kFloat));
  const size_t bytes = convnd_hip_delta_backward_workspace_size(
      c.dtype, &p, dy.const_data_ptr(), c.query.const_data_ptr(), c.key.const_data_ptr(),
      c.value.const_data_ptr());
  auto workspace = workspace_of(bytes, query);
  check_status(convnd_hip_delta_backward(
      c.dtype, &p, dy.const_data_ptr(), dl.has_value() ? dl->const_data_ptr<float>() : nullptr,
      c.query.const_data_ptr(), c.key.const_data_ptr(), c.value.const_data_ptr(), decay.const_data_ptr(),
      beta.const_data_ptr(), data_or_null(c.lengths), saved.const_data_ptr(), dq.mutable_data_ptr(),
      dk.mutable_data_ptr(), dv.mutable_data_ptr(), dg.mutable_data_ptr(), db.mutable_data_ptr(),
      df.has_value() ? df->mutable_data_ptr<float>() : nullptr,
      bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, stream_of(query)));
  return {dq, dk, dv, dg, db, df};
}

const auto& delta_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::gated_delta_rule", "")
                             .typed<decltype(delta_device)>();
  return op;
}
const auto& delta_backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("torch_convnd::gated_delta_rule_backward", "")
                             .typed<decltype(delta_backward_device)>();
  return op;
}

class DeltaFunction : public torch::autograd::Function<DeltaFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& query, const at::Tensor& key,
                               const at::Tensor& value, const at::Tensor& decay, const at::Tensor& beta,
                               const OptionalTensor& first, const OptionalTensor& lengths, double scale,
                               bool normalize) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [output, last, saved] =
        delta_op().call(query, key, value, decay, beta, first, lengths, scale, normalize, true);
    ctx->saved_data["first"] = first.has_value() && first->defined();
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["normalize"] = normalize;
    ctx->save_for_backward({query, key, value, decay, beta, lengths.value_or(at::Tensor()), saved});
    ctx->mark_non_differentiable({saved});
    ctx->set_materialize_grads(false);
    return {output, last, saved};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_delta_rule");
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(9);
    at::AutoDispatchBelowADInplaceOrView below;
    const auto saved = ctx->get_saved_variables();
    const auto optional = [](const at::Tensor& t) {
      return t.defined() ? OptionalTensor(t) : std::nullopt;
    };
    const auto dy = grads[0].defined() ? grads[0] : at::zeros_like(saved[2]);
    const bool need_first = ctx->saved_data["first"].toBool() && ctx->needs_input_grad(5);
    auto [dq, dk, dv, dg, db, df] = delta_backward_op().call(
        dy, optional(grads[1]), saved[0], saved[1], saved[2], saved[3], saved[4], optional(saved[5]), saved[6],
        ctx->saved_data["scale"].toDouble(), ctx->saved_data["normalize"].toBool(), need_first);
    return {dq, dk, dv, dg, db, df.value_or(at::Tensor()), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> delta_autograd(
    const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, const at::Tensor& decay,
    const at::Tensor& beta, const OptionalTensor& first, const OptionalTensor& lengths, double scale,
    bool normalize, bool keep) {
  if (!at::GradMode::is_enabled() || !(wants_grad(query) || wants_grad(key) || wants_grad(value) ||
                                       wants_grad(decay) || wants_grad(beta) || wants_grad(first))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return delta_op().call(query, key, value, decay, beta, first, lengths, scale, normalize, keep);
  }
  auto out = DeltaFunction::apply(query, key, value, decay, beta, first, lengths, scale, normalize);
  return {out[0], out[1], out[2]};
}

}  // namespace
}  // namespace torch_convnd_hip

TORCH_LIBRARY_IMPL(torch_convnd, Autograd, library) {
  library.impl("gated_delta_rule", &torch_convnd_hip::delta_autograd);
}

TORCH_LIBRARY_IMPL(torch_convnd, CUDA, library) {
  library.impl("gated_delta_rule", &torch_convnd_hip::delta_device);
  library.impl("gated_delta_rule_backward", &torch_convnd_hip::delta_backward_device);
}
