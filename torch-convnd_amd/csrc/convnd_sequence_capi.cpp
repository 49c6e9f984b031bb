// C ABI of the sequence operators (layer norm, linear layer, gated recurrence): argument checks and launches.
#include <algorithm>
#include <cstring>
#include <string>

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

// A workspace of `needed` bytes, on a whole multiple of `align`.
int check_workspace(const void* workspace, size_t size, size_t needed, size_t align,
                    const char* what) {
  if (needed == 0) return CONVND_HIP_SUCCESS;
  if (workspace == nullptr || size < needed)
    return fail(CONVND_HIP_WORKSPACE_TOO_SMALL, std::string(what) + " needs a workspace of " +
                                                    std::to_string(needed) + " bytes");
  if (reinterpret_cast<uintptr_t>(workspace) % align != 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, std::string(what) + " needs a workspace aligned to " +
                                                 std::to_string(align) + " bytes");
  return CONVND_HIP_SUCCESS;
}

// Plans the call into `a` and checks the workspace and the size of the grid.
int plan_call(convnd_hip_dtype dtype, RecurrenceArgs* a, bool backward, void* workspace,
              size_t workspace_size, RecurrencePlan* p) {
  *p = plan_recurrence(dtype, *a, backward);
  const size_t bytes = static_cast<size_t>(p->word_count) * 8;
  const int st = check_workspace(workspace, workspace_size, bytes, 8, "gated_recurrence");
  if (st != CONVND_HIP_SUCCESS) return st;
  a->words = workspace;
  a->word_count = p->word_count;
  if (!launch_fits(p->workgroups, p->threads))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_recurrence sizes are too large: more than 2^32 threads");
  return CONVND_HIP_SUCCESS;
}

// ---- linear --------------------------------------------------------------------------------------

// A tile's 256 rows of an operand are addressed with 31-bit byte offsets.
constexpr int64_t kMaxLinear = int64_t{1} << 21;

int check_linear(convnd_hip_dtype dtype, const convnd_hip_linear_problem* p) {
  if (size_of(dtype) == 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, std::string("linear_act ") + kTypes);
  if (p == nullptr || p->rows < 0 || p->inputs <= 0 || p->outputs <= 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "linear_act needs nonnegative rows and positive inputs and outputs");
  if (p->activation < CONVND_HIP_ACT_NONE || p->activation > CONVND_HIP_ACT_GELU_TANH)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "activation must be 'none', 'relu', 'gelu' or 'gelu_tanh'");
  if (p->inputs >= kMaxLinear || p->outputs >= kMaxLinear || p->input_stride >= kMaxLinear ||
      p->grad_stride >= kMaxLinear || p->residual_stride >= kMaxLinear)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "linear_act needs inputs, outputs and strides below 2^21 elements");
  if (p->rows >= int64_t{1} << 31)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "linear_act needs fewer than 2^31 rows");
  const auto tiles = [](int64_t n) { return (n + 127) / 128; };
  const int64_t widest = std::max(tiles(p->inputs), tiles(p->outputs));
  if (tiles(p->rows) * widest >= (int64_t{1} << 26) ||
      tiles(p->inputs) * tiles(p->outputs) >= (int64_t{1} << 26))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "linear_act sizes are too large");
  if (p->input_stride < p->inputs)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "linear_act needs rows at least their length apart");
  return CONVND_HIP_SUCCESS;
}

// A workspace handed out in parts of whole 256 bytes; sizes only where there is none.
struct Parts {
  char* base;
  size_t used = 0;
  void* take(int64_t bytes) {
    void* p = base == nullptr ? nullptr : base + used;
    used += (static_cast<size_t>(bytes) + 255) & ~size_t{255};
    return p;
  }
};

// One operand as the product kernels want it: itself, or a padded copy in the workspace.
struct Padded {
  const void* data;
  int64_t stride;
  bool copy;
};
bool whole(const void* data, int64_t stride, int64_t columns, int size) {
  return (reinterpret_cast<uintptr_t>(data) | static_cast<uintptr_t>(stride * size) |
          static_cast<uintptr_t>(columns * size)) % 4 == 0;
}
int64_t padded_columns(int64_t columns, int size) {
  const int64_t vec = 16 / size;
  return (columns + vec - 1) / vec * vec;
}
Padded padded(const void* data, int64_t stride, int64_t rows, int64_t columns, int size, Parts* ws) {
  if (whole(data, stride, columns, size)) return {data, stride, false};
  const int64_t pitch = padded_columns(columns, size);
  return {ws->take(rows * pitch * size), pitch, true};
}
int fill_padded(convnd_hip_dtype dtype, const Padded& p, const void* data, int64_t stride,
                int64_t rows, int64_t columns, hipStream_t stream) {
  if (!p.copy) return CONVND_HIP_SUCCESS;
  return hip_check(launch_linear_pad(dtype, data, stride, rows, columns,
                                     const_cast<void*>(p.data), stream),
                   "linear operand copy");
}

float* partial_sums(const LinearPlan& p, int64_t m, int64_t n, Parts* ws) {
  return p.splits > 1 ? static_cast<float*>(ws->take(p.splits * m * n * sizeof(float))) : nullptr;
}

// Whether the sizes leave a plan that one launch can hold.
int check_plan(const LinearPlan& p) {
  if (p.few_rows || p.tile != 0) return CONVND_HIP_SUCCESS;
  return fail(CONVND_HIP_INVALID_ARGUMENT,
              "linear_act sizes are too large: more than 2^32 threads");
}

int check_parts(const Parts& ws, size_t size, const char* what) {
  return check_workspace(ws.base, size, ws.used, 16, what);
}

struct LinearForward {
  LinearPlan plan;
  Padded x, w;
  float* partial;
};
LinearForward lay_out(convnd_hip_dtype dtype, const convnd_hip_linear_problem& p, const void* input,
                      const void* weight, Parts* ws) {
  const int size = size_of(dtype);
  LinearForward f{};
  f.plan = plan_product(dtype, LinearProduct::kForward, p.rows, p.outputs, p.inputs);
  f.x = {input, p.input_stride, false};
  f.w = {weight, p.inputs, false};
  if (!f.plan.few_rows) {
    f.x = padded(input, p.input_stride, p.rows, p.inputs, size, ws);
    f.w = padded(weight, p.inputs, p.outputs, p.inputs, size, ws);
  }
  f.partial = partial_sums(f.plan, p.rows, p.outputs, ws);
  return f;
}

struct LinearBackward {
  LinearPlan input_plan, weight_plan;
  Padded dz, x, w;
  bool make_dz;     // dz = dy act'(z), or a padded copy of dy
  int64_t parts;    // rows of the bias gradient's sums
  float* sums;
  float* input_partial;   // of the products' splits, or null
  float* weight_partial;
};
LinearBackward lay_out_backward(convnd_hip_dtype dtype, const convnd_hip_linear_problem& p,
                                const void* grad_output, const void* input, const void* weight,
                                bool need_input, bool need_weight, bool need_bias, Parts* ws) {
  const int size = size_of(dtype);
  LinearBackward b{};
  b.dz = {grad_output, p.grad_stride, false};
  const bool products = need_input || need_weight;
  if (products) {
    if (p.activation != CONVND_HIP_ACT_NONE) {
      const int64_t pitch = padded_columns(p.outputs, size);
      b.dz = {ws->take(p.rows * pitch * size), pitch, true};
    } else {
      b.dz = padded(grad_output, p.grad_stride, p.rows, p.outputs, size, ws);
    }
  }
  b.make_dz = b.dz.copy;
  if (need_weight) b.x = padded(input, p.input_stride, p.rows, p.inputs, size, ws);
  if (need_input) b.w = padded(weight, p.inputs, p.outputs, p.inputs, size, ws);
  b.parts = linear_grad_parts(p.rows, p.outputs);
  if (need_bias) b.sums = static_cast<float*>(ws->take(b.parts * p.outputs * sizeof(float)));
  if (need_input && need_weight)
    plan_gradients(dtype, p.rows, p.inputs, p.outputs, &b.input_plan, &b.weight_plan);
  else if (need_input)
    b.input_plan = plan_product(dtype, LinearProduct::kGradInput, p.rows, p.inputs, p.outputs);
  else if (need_weight)
    b.weight_plan = plan_product(dtype, LinearProduct::kGradWeight, p.outputs, p.inputs, p.rows);
  if (need_input) b.input_partial = partial_sums(b.input_plan, p.rows, p.inputs, ws);
  if (need_weight) b.weight_partial = partial_sums(b.weight_plan, p.outputs, p.inputs, ws);
  return b;
}

// A plan's description as JSON; numbers only beside the kernel's name.
struct Description {
  std::string text;
  explicit Description(const char* kernel) : text(std::string("{\"kernel\":\"") + kernel + "\"") {}
  Description& add(const char* name, int64_t value) {
    text += std::string(",\"") + name + "\":" + std::to_string(value);
    return *this;
  }
  int write(char* buffer, size_t length) const {
    if (buffer == nullptr || length == 0) return CONVND_HIP_SUCCESS;
    const std::string whole = text + "}";
    const size_t n = std::min(length - 1, whole.size());
    std::memcpy(buffer, whole.data(), n);
    buffer[n] = '\0';
    return CONVND_HIP_SUCCESS;
  }
};

int64_t tiles_of(const LinearPlan& p, int64_t m, int64_t n) {
  return ((m + p.tile - 1) / p.tile) * ((n + p.tile - 1) / p.tile) * p.splits;
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
  if (params && channels >= int64_t{1} << 27)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "layer_norm parameter gradients need fewer than 2^27 channels");
  if (!params && (grad_input == nullptr || rows == 0)) return CONVND_HIP_SUCCESS;
  if (rows > 0 && (grad_output == nullptr || input == nullptr || mean == nullptr || rstd == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "grad_output, input and the statistics must not be null");
  const int64_t floats = norm_partials(rows, channels, dtype);
  if (params) {
    st = check_workspace(workspace, workspace_size, floats * sizeof(float), 16,
                         "layer_norm backward");
    if (st != CONVND_HIP_SUCCESS) return st;
  }
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
  return hip_check(launch_sum_rows(param_dtype, partial, p.blocks, 2 * channels, channels,
                                   grad_weight, grad_bias, static_cast<hipStream_t>(stream)),
                   "layer norm reduction launch");
}

int64_t convnd_hip_recurrence_carries(int64_t tokens) {
  return tokens <= 0 ? 0 : (tokens + kRecurrenceTile - 1) / kRecurrenceTile;
}

size_t convnd_hip_recurrence_workspace_size(convnd_hip_dtype dtype,
                                            const convnd_hip_recurrence_problem* problem) {
  if (check_recurrence(dtype, problem) != CONVND_HIP_SUCCESS) return 0;
  const RecurrenceArgs a = to_args(*problem);
  return static_cast<size_t>(std::max(plan_recurrence(dtype, a, false).word_count,
                                      plan_recurrence(dtype, a, true).word_count)) *
         8;
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
  st = plan_call(dtype, &a, false, workspace, workspace_size, &p);
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
  st = plan_call(dtype, &a, true, workspace, workspace_size, &p);
  if (st != CONVND_HIP_SUCCESS) return st;
  return hip_check(launch_recurrence(dtype, a, true, p, static_cast<hipStream_t>(stream)),
                   "gated recurrence backward launch");
}

size_t convnd_hip_linear_workspace_size(convnd_hip_dtype dtype,
                                        const convnd_hip_linear_problem* problem,
                                        const void* input, const void* weight) {
  if (check_linear(dtype, problem) != CONVND_HIP_SUCCESS || problem->rows == 0) return 0;
  Parts ws{nullptr};
  lay_out(dtype, *problem, input, weight, &ws);
  return ws.used;
}

int convnd_hip_linear(convnd_hip_dtype dtype, const convnd_hip_linear_problem* problem,
                      const void* input, const void* weight, const void* bias,
                      const void* residual, void* output, void* slope, void* workspace,
                      size_t workspace_size, void* stream) {
  int st = check_linear(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  const convnd_hip_linear_problem& p = *problem;
  if (p.rows == 0) return CONVND_HIP_SUCCESS;
  if (input == nullptr || weight == nullptr || output == nullptr)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "input, weight and output must not be null");
  if (residual != nullptr && p.residual_stride < p.outputs)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "linear_act needs rows at least their length apart");
  Parts ws{static_cast<char*>(workspace)};
  const LinearForward f = lay_out(dtype, p, input, weight, &ws);
  st = check_plan(f.plan);
  if (st == CONVND_HIP_SUCCESS) st = check_parts(ws, workspace_size, "linear_act");
  if (st != CONVND_HIP_SUCCESS) return st;
  const auto on = static_cast<hipStream_t>(stream);
  st = fill_padded(dtype, f.x, input, p.input_stride, p.rows, p.inputs, on);
  if (st == CONVND_HIP_SUCCESS)
    st = fill_padded(dtype, f.w, weight, p.inputs, p.outputs, p.inputs, on);
  if (st != CONVND_HIP_SUCCESS) return st;
  LinearArgs a{};
  a.a = f.x.data;
  a.b = f.w.data;
  a.lda = f.x.stride;
  a.ldb = f.w.stride;
  a.m = p.rows;
  a.n = p.outputs;
  a.k = p.inputs;
  a.bias = bias;
  a.residual = residual;
  a.residual_stride = p.residual_stride;
  a.output = output;
  a.slope = p.activation != CONVND_HIP_ACT_NONE ? slope : nullptr;
  a.activation = p.activation;
  return hip_check(launch_linear_product(dtype, a, LinearProduct::kForward, f.plan, f.partial, on),
                   "linear launch");
}

size_t convnd_hip_linear_backward_workspace_size(convnd_hip_dtype dtype,
                                                 const convnd_hip_linear_problem* problem,
                                                 const void* grad_output, const void* input,
                                                 const void* weight, int need_grad_input,
                                                 int need_grad_weight, int need_grad_bias) {
  if (check_linear(dtype, problem) != CONVND_HIP_SUCCESS || problem->rows == 0) return 0;
  Parts ws{nullptr};
  lay_out_backward(dtype, *problem, grad_output, input, weight, need_grad_input != 0,
                   need_grad_weight != 0, need_grad_bias != 0, &ws);
  return ws.used;
}

int convnd_hip_linear_backward(convnd_hip_dtype dtype, const convnd_hip_linear_problem* problem,
                               const void* grad_output, const void* input, const void* weight,
                               const void* slope, void* grad_input, void* grad_weight,
                               void* grad_bias, void* workspace, size_t workspace_size,
                               void* stream) {
  int st = check_linear(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  const convnd_hip_linear_problem& p = *problem;
  const auto on = static_cast<hipStream_t>(stream);
  if (p.rows == 0) {
    if (grad_weight != nullptr)
      st = hip_check(launch_fill_zero(grad_weight, p.outputs * p.inputs * size_of(dtype), on),
                     "linear backward launch");
    if (st == CONVND_HIP_SUCCESS && grad_bias != nullptr)
      st = hip_check(launch_fill_zero(grad_bias, p.outputs * size_of(dtype), on),
                     "linear backward launch");
    return st;
  }
  const bool activated = p.activation != CONVND_HIP_ACT_NONE;
  if (p.grad_stride < p.outputs)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "linear_act needs rows at least their length apart");
  if (grad_output == nullptr || (activated && slope == nullptr) ||
      (grad_input != nullptr && weight == nullptr) || (grad_weight != nullptr && input == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "grad_output, input, weight and (with an activation) slope must not be null");
  Parts ws{static_cast<char*>(workspace)};
  const LinearBackward b =
      lay_out_backward(dtype, p, grad_output, input, weight, grad_input != nullptr,
                       grad_weight != nullptr, grad_bias != nullptr, &ws);
  if (grad_input != nullptr) st = check_plan(b.input_plan);
  if (st == CONVND_HIP_SUCCESS && grad_weight != nullptr) st = check_plan(b.weight_plan);
  if (st == CONVND_HIP_SUCCESS) st = check_parts(ws, workspace_size, "linear_act backward");
  if (st != CONVND_HIP_SUCCESS) return st;
  const bool both = grad_input != nullptr && grad_weight != nullptr;
  if (b.make_dz || grad_bias != nullptr) {
    LinearGradArgs g{};
    g.grad_output = grad_output;
    g.slope = activated ? slope : nullptr;
    g.grad_pre = b.make_dz ? const_cast<void*>(b.dz.data) : nullptr;
    g.partial = b.sums;
    g.rows = p.rows;
    g.columns = p.outputs;
    g.grad_stride = p.grad_stride;
    g.pitch = b.dz.stride;
    st = hip_check(launch_linear_grad(dtype, g, b.parts, on), "linear gradient launch");
    if (st == CONVND_HIP_SUCCESS && grad_bias != nullptr && !both)
      st = hip_check(launch_sum_rows(dtype, b.sums, b.parts, p.outputs, p.outputs, grad_bias,
                                     nullptr, on),
                     "linear bias gradient launch");
    if (st != CONVND_HIP_SUCCESS) return st;
  }
  LinearArgs x{}, w{};
  if (grad_input != nullptr) {
    st = fill_padded(dtype, b.w, weight, p.inputs, p.outputs, p.inputs, on);
    if (st != CONVND_HIP_SUCCESS) return st;
    x.a = b.dz.data;
    x.lda = b.dz.stride;
    x.b = b.w.data;
    x.ldb = b.w.stride;
    x.m = p.rows;
    x.n = p.inputs;
    x.k = p.outputs;
    x.output = grad_input;
  }
  if (grad_weight != nullptr) {
    st = fill_padded(dtype, b.x, input, p.input_stride, p.rows, p.inputs, on);
    if (st != CONVND_HIP_SUCCESS) return st;
    w.a = b.dz.data;
    w.lda = b.dz.stride;
    w.b = b.x.data;
    w.ldb = b.x.stride;
    w.m = p.outputs;
    w.n = p.inputs;
    w.k = p.rows;
    w.output = grad_weight;
  }
  if (both)
    return hip_check(launch_linear_gradients(dtype, x, b.input_plan, b.input_partial, w,
                                             b.weight_plan, b.weight_partial,
                                             {b.sums, b.parts, p.outputs, grad_bias}, on),
                     "linear gradients launch");
  if (grad_input != nullptr)
    return hip_check(launch_linear_product(dtype, x, LinearProduct::kGradInput, b.input_plan,
                                           b.input_partial, on),
                     "linear input gradient launch");
  if (grad_weight != nullptr)
    return hip_check(launch_linear_product(dtype, w, LinearProduct::kGradWeight, b.weight_plan,
                                           b.weight_partial, on),
                     "linear weight gradient launch");
  return st;
}

int convnd_hip_linear_plan_describe(convnd_hip_dtype dtype,
                                    const convnd_hip_linear_problem* problem, int which,
                                    char* buffer, size_t length) {
  int st = check_linear(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  const convnd_hip_linear_problem& p = *problem;
  if (which < 0 || which > 3 || p.rows == 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "which must be 0 to 3, and rows positive");
  LinearPlan x{}, w{};
  if (which == 0)
    x = plan_product(dtype, LinearProduct::kForward, p.rows, p.outputs, p.inputs);
  else if (which == 1)
    x = plan_product(dtype, LinearProduct::kGradInput, p.rows, p.inputs, p.outputs);
  else if (which == 2)
    x = plan_product(dtype, LinearProduct::kGradWeight, p.outputs, p.inputs, p.rows);
  else
    plan_gradients(dtype, p.rows, p.inputs, p.outputs, &x, &w);
  st = check_plan(x);
  if (st != CONVND_HIP_SUCCESS) return st;
  if (x.few_rows)
    return Description("few_rows").add("workgroups", (p.outputs + 15) / 16).write(buffer, length);
  if (which == 3)
    return Description("both_gradients")
        .add("tile", x.tile)
        .add("input_splits", x.splits)
        .add("weight_splits", w.splits)
        .add("workgroups", tiles_of(x, p.rows, p.inputs) + tiles_of(w, p.outputs, p.inputs))
        .write(buffer, length);
  const int64_t m = which == 2 ? p.outputs : p.rows, n = which == 0 ? p.outputs : p.inputs;
  return Description("tiles")
      .add("tile", x.tile)
      .add("splits", x.splits)
      .add("workgroups", tiles_of(x, m, n))
      .write(buffer, length);
}

int convnd_hip_recurrence_plan_describe(convnd_hip_dtype dtype,
                                        const convnd_hip_recurrence_problem* problem, int backward,
                                        char* buffer, size_t length) {
  const int st = check_recurrence(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  const RecurrencePlan p = plan_recurrence(dtype, to_args(*problem), backward != 0);
  const bool step = p.waves == 1 && backward == 0;
  return Description(p.chain ? "chain" : step ? "step" : "whole")
      .add("channels_per_lane", p.channels_per_lane)
      .add("lanes", p.lanes)
      .add("waves", p.waves)
      .add("tile", p.tile)
      .add("workgroups", p.workgroups)
      .write(buffer, length);
}

}  // extern "C"
