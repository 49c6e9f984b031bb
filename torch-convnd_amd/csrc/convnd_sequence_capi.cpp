// C ABI of the sequence operators (layer norm, linear layer, gated recurrence, delta rule): argument checks
// and launches.
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
                      const void* weight, Parts* ws) {  // gated: of 2 outputs
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
                                bool need_input, bool need_weight, bool need_bias, Parts* ws,
                                bool gated = false) {  // gated: of 2 outputs
  const int size = size_of(dtype);
  LinearBackward b{};
  b.dz = {grad_output, p.grad_stride, false};
  const bool products = need_input || need_weight;
  if (products) {
    if (gated || p.activation != CONVND_HIP_ACT_NONE) {
      const int64_t pitch = padded_columns(p.outputs, size);
      b.dz = {ws->take(p.rows * pitch * size), pitch, true};
    } else {
      b.dz = padded(grad_output, p.grad_stride, p.rows, p.outputs, size, ws);
    }
  }
  b.make_dz = b.dz.copy;
  if (need_weight) b.x = padded(input, p.input_stride, p.rows, p.inputs, size, ws);
  if (need_input) b.w = padded(weight, p.inputs, p.outputs, p.inputs, size, ws);
  b.parts = linear_grad_parts(p.rows, gated ? p.outputs / 2 : p.outputs);
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

// ---- delta rule ----------------------------------------------------------------------------------

// Up to so many tokens run one by one.
constexpr int64_t kDeltaStepTokens = 8;

int check_delta(convnd_hip_dtype dtype, const convnd_hip_delta_problem* p) {
  if (size_of(dtype) == 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, std::string("gated_delta_rule ") + kTypes);
  if (p == nullptr || p->batch < 0 || p->tokens < 0 || p->key_heads <= 0 || p->heads <= 0 ||
      p->heads % p->key_heads != 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_delta_rule needs nonnegative batch and tokens, and heads that are a multiple of "
                "the key heads");
  if (p->key_size <= 0 || p->key_size > 128 || p->value_size <= 0 || p->value_size > 65535)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_delta_rule needs key sizes of 1 to 128 and value sizes of 1 to 65535");
  if (p->gate_dtype != dtype && p->gate_dtype != CONVND_HIP_FLOAT32)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_delta_rule decay and beta must have the inputs' dtype or float32");
  if (p->tokens >= (int64_t{1} << 31) - 64 || p->batch >= int64_t{1} << 31 || p->heads >= int64_t{1} << 31)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule needs fewer than 2^31 tokens, sequences and heads");
  int64_t rows = 0, total = 0, extent = 0;
  const int64_t steps[] = {p->query_batch, p->query_token, p->query_head, p->key_batch,   p->key_token,
                           p->key_head,    p->value_batch, p->value_token, p->value_head, p->decay_batch,
                           p->decay_token, p->decay_head,  p->beta_batch,  p->beta_token, p->beta_head,
                           p->grad_batch,  p->grad_token,  p->grad_head};
  const int64_t most = std::max({p->batch, p->tokens, p->heads});
  for (int64_t step : steps)
    if (step < 0 || !mul_ok(step, most, &extent))
      return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule strides overflow int64");
  if (!mul_ok(p->batch, p->heads, &rows) || !mul_ok(rows, p->tokens + 64, &total) ||
      !mul_ok(total, (p->value_size + 127) * 128, &total))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule sizes overflow int64");
  // A row's place in a chunk is a 32-bit byte offset.
  if (!mul_ok(p->heads, p->value_size, &extent) || extent >= int64_t{1} << 23)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule needs fewer than 2^23 values a token");
  if (p->query_token >= kMaxTokenStride || p->key_token >= kMaxTokenStride ||
      p->value_token >= kMaxTokenStride || p->grad_token >= kMaxTokenStride)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule needs token strides below 2^21 elements");
  return CONVND_HIP_SUCCESS;
}

DeltaArgs to_args(convnd_hip_dtype dtype, const convnd_hip_delta_problem& p) {
  DeltaArgs a{};
  a.batch = p.batch;
  a.tokens = p.tokens;
  a.key_heads = p.key_heads;
  a.heads = p.heads;
  a.key_size = p.key_size;
  a.value_size = p.value_size;
  const int64_t chunk = delta_chunk(size_of(dtype));
  a.chunks = (p.tokens + chunk - 1) / chunk;
  a.value_pad = (p.value_size + 15) / 16 * 16;
  a.groups = static_cast<int>(p.heads / p.key_heads);
  // Eight workgroups a compute unit, of a chunk at least.
  if (dtype == CONVND_HIP_FLOAT16)
    a.parts = static_cast<int>(
        std::clamp<int64_t>(2048 / std::max<int64_t>(p.batch * p.heads, 1), 1, std::clamp<int64_t>(a.chunks, 1, 64)));
  a.query_strides = {p.query_batch, p.query_token, p.query_head};
  a.key_strides = {p.key_batch, p.key_token, p.key_head};
  a.value_strides = {p.value_batch, p.value_token, p.value_head};
  a.decay_strides = {p.decay_batch, p.decay_token, p.decay_head};
  a.beta_strides = {p.beta_batch, p.beta_token, p.beta_head};
  a.grad_strides = {p.grad_batch, p.grad_token, p.grad_head};
  a.scale = static_cast<float>(p.scale);
  a.normalize = p.normalize;
  a.float_gates = p.gate_dtype == CONVND_HIP_FLOAT32;
  a.wide_lengths = p.wide_lengths;
  return a;
}

// Rows as the kernels take them: themselves, or a padded copy in the workspace.
bool delta_copied(const void* data, const DeltaStrides& s, int64_t columns, int size) {
  return (reinterpret_cast<uintptr_t>(data) |
          static_cast<uintptr_t>((s.batch | s.token | s.head) * size)) % 4 != 0 ||
         columns * size % 16 != 0;
}
struct DeltaRows {
  const void* data;
  DeltaStrides strides;
  DeltaCopy copy;
  bool copied;
};
DeltaRows delta_rows(const void* data, const DeltaStrides& s, const DeltaArgs& a, int64_t heads,
                     int64_t columns, int size, Parts* ws) {
  DeltaRows r{data, s, {}, delta_copied(data, s, columns, size)};
  if (!r.copied) return r;
  const int64_t pitch = padded_columns(columns, size);
  r.copy = {data, ws->take(a.batch * a.tokens * heads * pitch * size), s, a.batch, a.tokens, heads, columns, pitch};
  r.data = r.copy.to;
  r.strides = {a.tokens * heads * pitch, heads * pitch, pitch};
  return r;
}
int fill_rows(convnd_hip_dtype dtype, const DeltaRows& r, hipStream_t stream) {
  if (!r.copied) return CONVND_HIP_SUCCESS;
  return hip_check(launch_delta_copy(dtype, r.copy, stream), "delta rule operand copy");
}

int64_t delta_key_pad(const DeltaArgs& a) { return a.key_size <= 64 ? 64 : 128; }

// Segments of the chunks where walks over all of them would leave three quarters of the compute units idle: as
// many as fill them, of eight chunks at least. A segment is walked twice, once with the unit matrix's columns
// beside its own, and segments are joined one after another, so it takes 32 chunks, and as many as there are walks,
// to gain: forward and backward of 128 x 128 take 71 and 97 us where one walk takes 76 and 115 (16 walks of 32
// chunks), 147 and 296 for 154 and 302 (64 of 64), but 128 and 248 for 125 and 242 (64 of 50), 66 and 92 for 60 and
// 92 (16 of 24).
DeltaPlan plan_delta(const DeltaArgs& a, bool saving) {
  DeltaPlan p{};
  p.step = !saving && a.tokens <= kDeltaStepTokens;
  const int64_t columns = kDeltaStepColumns;  // of a walk's four waves too
  const int64_t walks = a.batch * a.heads * ((a.value_size + columns - 1) / columns);
  p.workgroups = walks;
  p.threads = 256;
  p.segments = 1;
  p.segment_chunks = static_cast<int>(a.chunks);
  if (p.step) return p;
  p.threads = 512;
  if (walks > 0 && walks <= 64 && a.chunks >= std::max<int64_t>(32, walks)) {
    const int64_t most = std::min<int64_t>(256 / walks, a.chunks / 8);
    p.segment_chunks = static_cast<int>((a.chunks + most - 1) / most);
    p.segments = static_cast<int>((a.chunks + p.segment_chunks - 1) / p.segment_chunks);
  }
  p.workgroups = std::max(p.workgroups, a.batch * a.key_heads * a.chunks);
  return p;
}

// The workspace of a forward, with the arguments that point into it.
struct DeltaLayout {
  DeltaRows query, key, value, grad;
};
DeltaLayout lay_out_delta(DeltaArgs* a, int size, const DeltaPlan& p, bool saving, const void* query,
                          const void* key, const void* value, Parts* ws) {
  DeltaLayout l{};
  l.query = {query, a->query_strides, {}, false};
  l.key = {key, a->key_strides, {}, false};
  l.value = {value, a->value_strides, {}, false};
  if (!p.step) {
    l.query = delta_rows(query, a->query_strides, *a, a->key_heads, a->key_size, size, ws);
    l.key = delta_rows(key, a->key_strides, *a, a->key_heads, a->key_size, size, ws);
    l.value = delta_rows(value, a->value_strides, *a, a->heads, a->value_size, size, ws);
    if (!saving) {
      const int64_t records = a->batch * a->heads * a->chunks;
      a->panels = static_cast<char*>(ws->take(records * delta_panel_bytes(size)));
      a->records = static_cast<char*>(ws->take(records * delta_record_bytes(size)));
    }
    if (saving && a->parts > 0)
      a->largest = static_cast<float*>(ws->take(a->batch * a->heads * a->parts * int64_t{sizeof(float)}));
    a->segments = p.segments;
    a->segment_chunks = p.segment_chunks;
    if (p.segments > 1) {
      const int64_t rows = a->batch * a->heads * p.segments * delta_key_pad(*a) * int64_t{sizeof(float)};
      a->transits = static_cast<float*>(ws->take(rows * delta_key_pad(*a)));
      a->partials = static_cast<float*>(ws->take(rows * a->value_pad));
      a->starts = static_cast<float*>(ws->take(rows * a->value_pad));
    }
  }
  a->query = l.query.data;
  a->key = l.key.data;
  a->value = l.value.data;
  a->query_strides = l.query.strides;
  a->key_strides = l.key.strides;
  a->value_strides = l.value.strides;
  return l;
}

// A copied row's place in a chunk is a 32-bit byte offset as well: strides of zero let rows be many where their
// tokens are near.
int check_copies(const DeltaLayout& l, int size) {
  for (const DeltaRows* r : {&l.query, &l.key, &l.value, &l.grad})
    if (r->copied && r->copy.heads > (int64_t{1} << 25) / (r->copy.pitch * size))
      return fail(CONVND_HIP_INVALID_ARGUMENT,
                  "gated_delta_rule rows that are no whole 16 bytes, or do not start on 4, need at most 2^25 bytes a token");
  return CONVND_HIP_SUCCESS;
}

// What a forward keeps: states, updates, and the chunks' panels and records. In bytes, whole 16 each.
int64_t saved_states(const DeltaArgs& a, int size) {
  return a.batch * a.heads * a.chunks * a.value_pad * delta_key_pad(a) * size;
}
int64_t saved_updates(const DeltaArgs& a, int size) {
  return a.batch * a.heads * a.chunks * a.value_pad * delta_chunk(size) * size;
}
int64_t saved_bytes(const DeltaArgs& a, int size) {
  return saved_states(a, size) + saved_updates(a, size) +
         a.batch * a.heads * a.chunks * (delta_panel_bytes(size) + delta_record_bytes(size));
}
void place_saved(DeltaArgs* a, int size, void* saved) {
  char* at = static_cast<char*>(saved);
  a->states = at;
  a->updates = at += saved_states(*a, size);
  a->panels = at += saved_updates(*a, size);
  a->records = at + a->batch * a->heads * a->chunks * delta_panel_bytes(size);
}

DeltaLayout lay_out_delta_backward(DeltaArgs* a, int size, const void* grad_output, const void* query,
                                   const void* key, const void* value, Parts* ws) {
  DeltaLayout l = lay_out_delta(a, size, plan_delta(*a, true), true, query, key, value, ws);
  l.grad = delta_rows(grad_output, a->grad_strides, *a, a->heads, a->value_size, size, ws);
  a->grad_output = l.grad.data;
  a->grad_strides = l.grad.strides;
  a->grad_states = ws->take(saved_states(*a, size));
  a->grad_updates = ws->take(saved_updates(*a, size));
  if (a->parts > 0) a->units = static_cast<float*>(ws->take(a->batch * a->heads * int64_t{sizeof(float)}));
  return l;
}

// The products of a backward from its dz.
int run_gradients(convnd_hip_dtype dtype, const convnd_hip_linear_problem& p, const LinearBackward& b,
                  const void* input, const void* weight, void* grad_input, void* grad_weight,
                  void* grad_bias, hipStream_t on) {
  int st = CONVND_HIP_SUCCESS;
  const bool both = grad_input != nullptr && grad_weight != nullptr;
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

// Zeros where there are no rows.
int fill_no_rows(convnd_hip_dtype dtype, const convnd_hip_linear_problem& p, void* grad_weight,
                 void* grad_bias, hipStream_t on) {
  int st = CONVND_HIP_SUCCESS;
  if (grad_weight != nullptr)
    st = hip_check(launch_fill_zero(grad_weight, p.outputs * p.inputs * size_of(dtype), on),
                   "linear backward launch");
  if (st == CONVND_HIP_SUCCESS && grad_bias != nullptr)
    st = hip_check(launch_fill_zero(grad_bias, p.outputs * size_of(dtype), on),
                   "linear backward launch");
  return st;
}

// The gated layer as a linear one of both halves' outputs.
int check_gated(convnd_hip_dtype dtype, const convnd_hip_linear_problem* p, convnd_hip_linear_problem* both) {
  if (size_of(dtype) == 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, std::string("gated_linear ") + kTypes);
  if (p == nullptr || p->outputs <= 0 || p->outputs >= kMaxLinear / 2)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_linear needs 1 to 2^20 - 1 outputs");
  if (p->activation < CONVND_HIP_ACT_RELU || p->activation > CONVND_HIP_ACT_SILU)
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "gated_linear activation must be 'silu', 'relu', 'gelu' or 'gelu_tanh'");
  *both = *p;
  both->outputs = 2 * p->outputs;
  both->residual_stride = 0;
  both->activation = CONVND_HIP_ACT_NONE;
  return check_linear(dtype, both);
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
  if (p.rows == 0) return fill_no_rows(dtype, p, grad_weight, grad_bias, on);
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
  return run_gradients(dtype, p, b, input, weight, grad_input, grad_weight, grad_bias, on);
}

int64_t convnd_hip_delta_saved(convnd_hip_dtype dtype, const convnd_hip_delta_problem* problem) {
  if (check_delta(dtype, problem) != CONVND_HIP_SUCCESS) return 0;
  const DeltaArgs a = to_args(dtype, *problem);
  return saved_bytes(a, size_of(dtype)) / size_of(dtype);
}

size_t convnd_hip_delta_workspace_size(convnd_hip_dtype dtype, const convnd_hip_delta_problem* problem,
                                       const void* query, const void* key, const void* value, int saving) {
  if (check_delta(dtype, problem) != CONVND_HIP_SUCCESS || problem->batch == 0) return 0;
  DeltaArgs a = to_args(dtype, *problem);
  Parts ws{nullptr};
  lay_out_delta(&a, size_of(dtype), plan_delta(a, saving != 0), saving != 0, query, key, value, &ws);
  return ws.used;
}

int convnd_hip_delta(convnd_hip_dtype dtype, const convnd_hip_delta_problem* problem, const void* query,
                     const void* key, const void* value, const void* decay, const void* beta,
                     const float* first, const void* lengths, void* output, float* last, void* saved,
                     void* workspace, size_t workspace_size, void* stream) {
  int st = check_delta(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  if (problem->batch == 0) return CONVND_HIP_SUCCESS;
  if (last == nullptr || (problem->tokens > 0 && (query == nullptr || key == nullptr || value == nullptr ||
                                                  decay == nullptr || beta == nullptr || output == nullptr)))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "query, key, value, decay, beta, output and last must not be null");
  if (reinterpret_cast<uintptr_t>(saved) % 16 != 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "saved must be aligned to 16 bytes");
  DeltaArgs a = to_args(dtype, *problem);
  const int size = size_of(dtype);
  const DeltaPlan p = plan_delta(a, saved != nullptr);
  Parts ws{static_cast<char*>(workspace)};
  const DeltaLayout l = lay_out_delta(&a, size, p, saved != nullptr, query, key, value, &ws);
  if (!launch_fits(p.workgroups, p.threads))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule sizes are too large: more than 2^32 threads");
  st = check_copies(l, size);
  if (st == CONVND_HIP_SUCCESS) st = check_parts(ws, workspace_size, "gated_delta_rule");
  if (st != CONVND_HIP_SUCCESS) return st;
  a.decay = decay;
  a.beta = beta;
  a.first = first;
  a.lengths = lengths;
  a.output = output;
  a.last = last;
  if (saved != nullptr) place_saved(&a, size, saved);
  const auto on = static_cast<hipStream_t>(stream);
  for (const DeltaRows* r : {&l.query, &l.key, &l.value}) {
    st = fill_rows(dtype, *r, on);
    if (st != CONVND_HIP_SUCCESS) return st;
  }
  return hip_check(launch_delta(dtype, a, p, on), "delta rule launch");
}

size_t convnd_hip_delta_backward_workspace_size(convnd_hip_dtype dtype,
                                                const convnd_hip_delta_problem* problem,
                                                const void* grad_output, const void* query,
                                                const void* key, const void* value) {
  if (check_delta(dtype, problem) != CONVND_HIP_SUCCESS || problem->batch == 0) return 0;
  DeltaArgs a = to_args(dtype, *problem);
  Parts ws{nullptr};
  lay_out_delta_backward(&a, size_of(dtype), grad_output, query, key, value, &ws);
  return ws.used;
}

int convnd_hip_delta_backward(convnd_hip_dtype dtype, const convnd_hip_delta_problem* problem,
                              const void* grad_output, const float* grad_last, const void* query,
                              const void* key, const void* value, const void* decay, const void* beta,
                              const void* lengths, const void* saved, void* grad_query, void* grad_key,
                              void* grad_value, void* grad_decay, void* grad_beta, float* grad_first,
                              void* workspace, size_t workspace_size, void* stream) {
  int st = check_delta(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  if (problem->batch == 0) return CONVND_HIP_SUCCESS;
  if (problem->tokens > 0 &&
      (grad_output == nullptr || query == nullptr || key == nullptr || value == nullptr || decay == nullptr ||
       beta == nullptr || saved == nullptr || grad_query == nullptr || grad_key == nullptr ||
       grad_value == nullptr || grad_decay == nullptr || grad_beta == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT,
                "grad_output, query, key, value, decay, beta, saved and their gradients must not be null");
  if (reinterpret_cast<uintptr_t>(saved) % 16 != 0)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "saved must be aligned to 16 bytes");
  DeltaArgs a = to_args(dtype, *problem);
  const int size = size_of(dtype);
  Parts ws{static_cast<char*>(workspace)};
  const DeltaLayout l = lay_out_delta_backward(&a, size, grad_output, query, key, value, &ws);
  const DeltaPlan p = plan_delta(a, true);
  if (!launch_fits(p.workgroups, p.threads))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_delta_rule sizes are too large: more than 2^32 threads");
  st = check_copies(l, size);
  if (st == CONVND_HIP_SUCCESS) st = check_parts(ws, workspace_size, "gated_delta_rule backward");
  if (st != CONVND_HIP_SUCCESS) return st;
  a.decay = decay;
  a.beta = beta;
  a.lengths = lengths;
  a.grad_last = grad_last;
  place_saved(&a, size, const_cast<void*>(saved));
  a.grad_query = grad_query;
  a.grad_key = grad_key;
  a.grad_value = grad_value;
  a.grad_decay = grad_decay;
  a.grad_beta = grad_beta;
  a.grad_first = grad_first;
  const auto on = static_cast<hipStream_t>(stream);
  for (const DeltaRows* r : {&l.query, &l.key, &l.value, &l.grad}) {
    st = fill_rows(dtype, *r, on);
    if (st != CONVND_HIP_SUCCESS) return st;
  }
  return hip_check(launch_delta_backward(dtype, a, on), "delta rule backward launch");
}

size_t convnd_hip_gated_linear_workspace_size(convnd_hip_dtype dtype,
                                              const convnd_hip_linear_problem* problem,
                                              const void* input, const void* weight) {
  convnd_hip_linear_problem both;
  if (check_gated(dtype, problem, &both) != CONVND_HIP_SUCCESS || both.rows == 0) return 0;
  Parts ws{nullptr};
  lay_out(dtype, both, input, weight, &ws);
  return ws.used;
}

size_t convnd_hip_gated_linear_kept_size(convnd_hip_dtype dtype, const convnd_hip_linear_problem* problem) {
  convnd_hip_linear_problem both;
  if (check_gated(dtype, problem, &both) != CONVND_HIP_SUCCESS) return 0;
  return static_cast<size_t>(both.rows) * both.outputs * (size_of(dtype) == 4 ? 4 : 3);
}

int convnd_hip_gated_linear(convnd_hip_dtype dtype, const convnd_hip_linear_problem* problem,
                            const void* input, const void* weight, const void* bias, void* output,
                            void* kept, void* workspace, size_t workspace_size, void* stream) {
  convnd_hip_linear_problem both;
  int st = check_gated(dtype, problem, &both);
  if (st != CONVND_HIP_SUCCESS) return st;
  const convnd_hip_linear_problem& p = *problem;
  if (p.rows == 0) return CONVND_HIP_SUCCESS;
  if (input == nullptr || weight == nullptr || output == nullptr)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "input, weight and output must not be null");
  Parts ws{static_cast<char*>(workspace)};
  const LinearForward f = lay_out(dtype, both, input, weight, &ws);
  st = check_plan(f.plan);
  if (st == CONVND_HIP_SUCCESS) st = check_parts(ws, workspace_size, "gated_linear");
  if (st != CONVND_HIP_SUCCESS) return st;
  const auto on = static_cast<hipStream_t>(stream);
  st = fill_padded(dtype, f.x, input, p.input_stride, p.rows, p.inputs, on);
  if (st == CONVND_HIP_SUCCESS)
    st = fill_padded(dtype, f.w, weight, p.inputs, both.outputs, p.inputs, on);
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
  a.output = output;
  a.slope = kept;
  a.activation = p.activation;
  return hip_check(launch_gated_product(dtype, a, f.plan, f.partial, on), "gated linear launch");
}

size_t convnd_hip_gated_linear_backward_workspace_size(convnd_hip_dtype dtype,
                                                       const convnd_hip_linear_problem* problem,
                                                       const void* input, const void* weight,
                                                       int need_grad_input, int need_grad_weight,
                                                       int need_grad_bias) {
  convnd_hip_linear_problem both;
  if (check_gated(dtype, problem, &both) != CONVND_HIP_SUCCESS || both.rows == 0) return 0;
  Parts ws{nullptr};
  lay_out_backward(dtype, both, nullptr, input, weight, need_grad_input != 0, need_grad_weight != 0,
                   need_grad_bias != 0, &ws, true);
  return ws.used;
}

int convnd_hip_gated_linear_backward(convnd_hip_dtype dtype, const convnd_hip_linear_problem* problem,
                                     const void* grad_output, const void* input, const void* weight,
                                     const void* kept, void* grad_input, void* grad_weight,
                                     void* grad_bias, void* workspace, size_t workspace_size,
                                     void* stream) {
  convnd_hip_linear_problem both;
  int st = check_gated(dtype, problem, &both);
  if (st != CONVND_HIP_SUCCESS) return st;
  const auto on = static_cast<hipStream_t>(stream);
  if (both.rows == 0) return fill_no_rows(dtype, both, grad_weight, grad_bias, on);
  if (problem->grad_stride < problem->outputs)
    return fail(CONVND_HIP_INVALID_ARGUMENT, "gated_linear needs rows at least their length apart");
  if (grad_input == nullptr && grad_weight == nullptr && grad_bias == nullptr) return CONVND_HIP_SUCCESS;
  if (grad_output == nullptr || kept == nullptr || (grad_input != nullptr && weight == nullptr) ||
      (grad_weight != nullptr && input == nullptr))
    return fail(CONVND_HIP_INVALID_ARGUMENT, "grad_output, input, weight and kept must not be null");
  Parts ws{static_cast<char*>(workspace)};
  const LinearBackward b =
      lay_out_backward(dtype, both, nullptr, input, weight, grad_input != nullptr, grad_weight != nullptr,
                       grad_bias != nullptr, &ws, true);
  if (grad_input != nullptr) st = check_plan(b.input_plan);
  if (st == CONVND_HIP_SUCCESS && grad_weight != nullptr) st = check_plan(b.weight_plan);
  if (st == CONVND_HIP_SUCCESS) st = check_parts(ws, workspace_size, "gated_linear backward");
  if (st != CONVND_HIP_SUCCESS) return st;
  LinearGradArgs g{};
  g.grad_output = grad_output;
  g.slope = kept;
  g.grad_pre = b.make_dz ? const_cast<void*>(b.dz.data) : nullptr;
  g.partial = b.sums;
  g.rows = both.rows;
  g.columns = problem->outputs;
  g.grad_stride = problem->grad_stride;
  g.pitch = b.make_dz ? b.dz.stride : both.outputs;
  g.gated = true;
  st = hip_check(launch_linear_grad(dtype, g, b.parts, on), "gated linear gradient launch");
  if (st == CONVND_HIP_SUCCESS && grad_bias != nullptr && (grad_input == nullptr || grad_weight == nullptr))
    st = hip_check(launch_sum_rows(dtype, b.sums, b.parts, both.outputs, both.outputs, grad_bias, nullptr, on),
                   "gated linear bias gradient launch");
  if (st != CONVND_HIP_SUCCESS) return st;
  return run_gradients(dtype, both, b, input, weight, grad_input, grad_weight, grad_bias, on);
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

int convnd_hip_delta_plan_describe(convnd_hip_dtype dtype, const convnd_hip_delta_problem* problem,
                                   int saving, char* buffer, size_t length) {
  const int st = check_delta(dtype, problem);
  if (st != CONVND_HIP_SUCCESS) return st;
  const DeltaPlan p = plan_delta(to_args(dtype, *problem), saving != 0);
  return Description(p.step ? "step" : "chunks")
      .add("chunk", p.step ? 1 : delta_chunk(size_of(dtype)))
      .add("segments", p.segments)
      .add("segment_chunks", p.segment_chunks)
      .write(buffer, length);
}

}  // extern "C"
