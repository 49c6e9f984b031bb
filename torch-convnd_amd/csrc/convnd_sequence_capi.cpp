// C ABI of the sequence operators (layer norm, gated recurrence): argument checks and launches.
#include <algorithm>
#include <limits>

#include "convnd_internal.h"

namespace convnd {
namespace {

int size_of(convnd_hip_dtype dtype) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return 4;
    case CONVND_HIP_FLOAT16:
    case CONVND_HIP_BFLOAT16:
      return 2;
    default:
      return 0;
  }
}

constexpr const char* kTypes = "supports float16, bfloat16 and float32";

int check_norm(convnd_hip_dtype dtype, convnd_hip_dtype param_dtype, int64_t rows,
               int64_t channels, int64_t input_stride) {
  if (size_of(dtype) == 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, std::string("layer_norm ") + kTypes);
  if (param_dtype != dtype && param_dtype != CONVND_HIP_FLOAT32)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "layer_norm parameters must have the input's dtype or float32");
  if (rows < 0 || channels <= 0 || channels >= (int64_t{1} << 30))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "layer_norm needs nonnegative rows and 1 to 2^30 - 1 channels");
  int64_t total = 0;
  if (input_stride < 0 || !mul_ok(rows, std::max(channels, input_stride), &total))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "layer_norm sizes overflow int64");
  return CONVND_HIP_SUCCESS;
}

int64_t norm_partials(int64_t rows, int64_t channels, convnd_hip_dtype dtype) {
  return plan_norm(rows, channels, size_of(dtype), true).blocks * 2 * channels;
}

constexpr int64_t kMaxTokenStride = int64_t{1} << 21;

int check_recurrence(convnd_hip_dtype dtype, const convnd_hip_recurrence_problem* r) {
  if (size_of(dtype) == 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, std::string("gated_recurrence ") + kTypes);
  if (r == nullptr || r->batch < 0 || r->tokens < 0 || r->channels <= 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_recurrence needs nonnegative batch and tokens and positive channels");
  int64_t rows = 0, total = 0, extent = 0;
  const int64_t steps[] = {r->input_batch, r->gate_batch, r->input_token, r->gate_token};
  for (int64_t step : steps)
    if (step < 0 || !mul_ok(step, std::max(r->batch, r->tokens), &extent))
      return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_recurrence strides overflow int64");
  if (!mul_ok(r->batch, r->tokens, &rows) || !mul_ok(rows, r->channels, &total) ||
      !mul_ok(r->batch, r->channels, &total))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_recurrence sizes overflow int64");
  // A lane's place in a tile of up to 256 tokens is a 32-bit byte offset.
  if (r->input_token < r->channels || r->gate_token < r->channels)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_recurrence needs tokens at least their channels apart");
  if (r->channels >= kMaxTokenStride || r->input_token >= kMaxTokenStride ||
      r->gate_token >= kMaxTokenStride)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_recurrence needs channels and token strides below 2^21 elements");
  return CONVND_HIP_SUCCESS;
}

RecurrenceArgs to_args(const convnd_hip_recurrence_problem& r) {
  RecurrenceArgs a{};
  a.batch = r.batch;
  a.tokens = r.tokens;
  a.channels = r.channels;
  a.input_batch = r.input_batch;
  a.input_token = r.input_token;
  a.gate_batch = r.gate_batch;
  a.gate_token = r.gate_token;
  a.grad_batch = r.tokens * r.channels;
  a.grad_token = r.channels;
  a.wide_lengths = r.wide_lengths;
  return a;
}

int64_t summary_floats(const RecurrenceArgs& a, const RecurrencePlan& p) {
  return p.splits > 1 ? a.batch * p.splits * 2 * a.channels : 0;
}

// Plans the call into `a` and checks the workspace and the size of the grid.
int plan_call(convnd_hip_dtype dtype, RecurrenceArgs* a, void* workspace, size_t workspace_size,
              RecurrencePlan* p) {
  *p = plan_recurrence(dtype, *a);
  a->splits = p->splits;
  a->split_tokens = p->split_tokens;
  const int64_t floats = summary_floats(*a, *p);
  if (floats > 0 && (workspace == nullptr || workspace_size < floats * sizeof(float)))
    return fail(CONVND_HIP_WORKSPACE_TOO_SMALL,
                "gated_recurrence needs a workspace of " + std::to_string(floats * sizeof(float)) +
                    " bytes");
  a->summary = static_cast<float*>(workspace);
  const int64_t strips = (a->channels + 15) / 16;
  if (strips * p->splits * a->batch > std::numeric_limits<int32_t>::max())
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_recurrence sizes are too large");
  return CONVND_HIP_SUCCESS;
}

}  // namespace
}  // namespace convnd

using namespace convnd;

extern "C" {

int convnd_hip_layer_norm(convnd_hip_dtype dtype, convnd_hip_dtype param_dtype, const void* input,
                          int64_t input_stride, const void* weight, const void* bias, void* output,
                          float* mean, float* rstd, int64_t rows, int64_t channels, double eps,
                          void* stream) {
  const int st = check_norm(dtype, param_dtype, rows, channels, input_stride);
  if (st != CONVND_HIP_SUCCESS) return st;
  if ((mean == nullptr) != (rstd == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "layer_norm writes both statistics or neither");
  if (rows == 0) return CONVND_HIP_SUCCESS;
  if (input == nullptr || output == nullptr)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "input and output must not be null");
  NormArgs a{};
  a.input = input;
  a.weight = weight;
  a.bias = bias;
  a.output = output;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.channels = channels;
  a.input_stride = input_stride;
  a.eps = static_cast<float>(eps);
  return hip_check(launch_norm(dtype, param_dtype == CONVND_HIP_FLOAT32, a, false,
                               plan_norm(rows, channels, size_of(dtype), false),
                               static_cast<hipStream_t>(stream)),
                   "layer norm launch");
}

size_t convnd_hip_layer_norm_backward_workspace_size(convnd_hip_dtype dtype, int64_t rows,
                                                     int64_t channels) {
  if (check_norm(dtype, dtype, rows, channels, channels) != CONVND_HIP_SUCCESS) return 0;
  return static_cast<size_t>(norm_partials(rows, channels, dtype)) * sizeof(float);
}

int convnd_hip_layer_norm_backward(convnd_hip_dtype dtype, convnd_hip_dtype param_dtype,
                                   const void* grad_output, int64_t grad_stride, const void* input,
                                   int64_t input_stride, const void* weight, const float* mean,
                                   const float* rstd, void* grad_input, void* grad_weight,
                                   void* grad_bias, int64_t rows, int64_t channels,
                                   void* workspace, size_t workspace_size, void* stream) {
  int st = check_norm(dtype, param_dtype, rows, channels, input_stride);
  if (st == CONVND_HIP_SUCCESS) st = check_norm(dtype, param_dtype, rows, channels, grad_stride);
  if (st != CONVND_HIP_SUCCESS) return st;
  const bool params = grad_weight != nullptr || grad_bias != nullptr;
  if (!params && (grad_input == nullptr || rows == 0)) return CONVND_HIP_SUCCESS;
  if (rows > 0 && (grad_output == nullptr || input == nullptr || mean == nullptr || rstd == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "grad_output, input and the statistics must not be null");
  const int64_t floats = norm_partials(rows, channels, dtype);
  if (params && floats > 0 && (workspace == nullptr || workspace_size < floats * sizeof(float)))
    return fail(CONVND_HIP_WORKSPACE_TOO_SMALL,
                "layer_norm backward needs a workspace of " +
                    std::to_string(floats * sizeof(float)) + " bytes");
  const NormPlan p = plan_norm(rows, channels, size_of(dtype), true);
  float* partial = params ? static_cast<float*>(workspace) : nullptr;
  if (rows > 0) {
    NormArgs a{};
    a.input = input;
    a.weight = weight;
    a.grad_output = grad_output;
    a.grad_input = grad_input;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.partial = partial;
    a.rows = rows;
    a.channels = channels;
    a.input_stride = input_stride;
    a.grad_stride = grad_stride;
    st = hip_check(launch_norm(dtype, param_dtype == CONVND_HIP_FLOAT32, a, true, p,
                               static_cast<hipStream_t>(stream)),
                   "layer norm backward launch");
    if (st != CONVND_HIP_SUCCESS) return st;
  }
  if (!params) return CONVND_HIP_SUCCESS;
  return hip_check(launch_norm_reduce(param_dtype, partial, p.blocks, channels, grad_weight,
                                      grad_bias, static_cast<hipStream_t>(stream)),
                   "layer norm reduction launch");
}

int64_t convnd_hip_recurrence_carries(int64_t tokens) {
  return tokens <= 0 ? 0 : (tokens + kRecurrenceTile - 1) / kRecurrenceTile;
}

size_t convnd_hip_recurrence_workspace_size(convnd_hip_dtype dtype,
                                            const convnd_hip_recurrence_problem* problem) {
  if (check_recurrence(dtype, problem) != CONVND_HIP_SUCCESS) return 0;
  const RecurrenceArgs a = to_args(*problem);
  return static_cast<size_t>(summary_floats(a, plan_recurrence(dtype, a))) *
         sizeof(float);
}

int convnd_hip_recurrence(convnd_hip_dtype dtype, const convnd_hip_recurrence_problem* problem,
                          const void* input, const void* gate, const float* first,
                          const void* lengths, void* output, float* last, float* carries,
                          void* workspace, size_t workspace_size, void* stream) {
  int st = check_recurrence(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  if (problem->batch == 0) return CONVND_HIP_SUCCESS;
  if (last == nullptr ||
      (problem->tokens > 0 && (input == nullptr || gate == nullptr || output == nullptr)))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "input, gate, output and last must not be null");
  RecurrenceArgs a = to_args(*problem);
  a.input = input;
  a.gate = gate;
  a.first = first;
  a.lengths = lengths;
  a.output = output;
  a.last = last;
  a.carries = carries;
  RecurrencePlan p;
  st = plan_call(dtype, &a, workspace, workspace_size, &p);
  if (st != CONVND_HIP_SUCCESS) return st;
  return hip_check(launch_recurrence(dtype, a, false, p, static_cast<hipStream_t>(stream)),
                   "gated recurrence launch");
}

int convnd_hip_recurrence_backward(convnd_hip_dtype dtype, const convnd_hip_recurrence_problem* problem,
                                   const void* grad_output, const float* grad_last,
                                   const void* input, const void* gate, const void* lengths,
                                   const float* carries, void* grad_input, void* grad_gate,
                                   float* grad_first, void* workspace, size_t workspace_size,
                                   void* stream) {
  int st = check_recurrence(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  if (problem->batch == 0) return CONVND_HIP_SUCCESS;
  if (problem->tokens > 0 && (grad_output == nullptr || input == nullptr || gate == nullptr ||
                              carries == nullptr || grad_input == nullptr || grad_gate == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "grad_output, input, gate, carries, grad_input and grad_gate must not be null");
  RecurrenceArgs a = to_args(*problem);
  a.grad_output = grad_output;
  a.grad_last = grad_last;
  a.input = input;
  a.gate = gate;
  a.lengths = lengths;
  a.carries = const_cast<float*>(carries);
  a.grad_input = grad_input;
  a.grad_gate = grad_gate;
  a.grad_first = grad_first;
  RecurrencePlan p;
  st = plan_call(dtype, &a, workspace, workspace_size, &p);
  if (st != CONVND_HIP_SUCCESS) return st;
  return hip_check(launch_recurrence(dtype, a, true, p, static_cast<hipStream_t>(stream)),
                   "gated recurrence backward launch");
}

}  // extern "C"
