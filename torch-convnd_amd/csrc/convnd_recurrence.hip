// Gated linear recurrence over the token axis of [batch, tokens, channels], and its backward pass.
//
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  h_{-1} the first state
//   D_t = dy_t + E_{t+1},  E_t = a_t D_t,  E_T the last state's gradient (E_0 is the first state's)
//   dx_t = (1 - a_t) D_t,  dgate_t = D_t (h_{t-1} - x_t) a_t (1 - a_t)
//
// Tokens at and past a sequence's length change no state: a = 1, 1 - a = 0 there (which gate = +inf
// and x = dy = 0 give by themselves), their outputs and gradients are zeros.
//
// Bound by HBM: two elements read and one written per token and channel in the forward, three and
// two in the backward, which makes its states again from one saved state per tile of 128 tokens
// instead of reading h. A run of tokens acts on the state as h -> A h + B, and such maps compose:
//   * A lane owns a channel (or two) and walks 16 consecutive tokens of it in registers; a wave is
//     64 lanes of neighbouring channels, so every access is a whole row segment.
//   * The 8 waves of a workgroup take the 8 runs of a tile, exchange their (A, B) through LDS (one
//     barrier a tile, two buffers), apply the maps before their own to the carried state and walk
//     their tokens again from registers. The next tile's loads are in flight meanwhile.
//   * With few sequences and channels the token axis is also split over workgroups: a first launch
//     leaves every split's map, the second composes the maps before its split and goes on as above
//     (it reads the inputs again).
// Every sum is in fp32 and in a fixed order; 1 - a is computed as sigmoid(-gate), which keeps its
// relative precision where a is near 1.

#include <algorithm>

#include "convnd_internal.h"
#include "convnd_sequence.h"

namespace convnd {
namespace {

constexpr int kRun = 16;  // tokens of a wave's run

struct Gate {
  float keep, take;  // sigmoid(g), sigmoid(-g)
};
__device__ __forceinline__ Gate open_gate(float g) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896f * fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.f + e);
  const float s = e * r;
  return g >= 0.f ? Gate{r, s} : Gate{s, r};
}

// The place of this workgroup and wave in the problem.
template <int CPL>
struct Place {
  int64_t batch, length, begin, end;  // tokens [begin, end) of the split
  int split, lane_channel, channel;   // channel: lane_channel, or the last whole one past the edge
  bool valid;
  __device__ __forceinline__ explicit Place(const RecurrenceArgs& a) {
    const int strips = static_cast<int>((a.channels + 64 * CPL - 1) / (64 * CPL));
    int64_t id = blockIdx.x;
    const int strip = static_cast<int>(id % strips);
    id /= strips;
    split = static_cast<int>(id % a.splits);
    batch = id / a.splits;
    const int C = static_cast<int>(a.channels);
    lane_channel = strip * 64 * CPL + static_cast<int>(threadIdx.x & 63) * CPL;
    valid = lane_channel < C;
    channel = valid ? lane_channel : C - CPL;
    length = a.tokens;
    if (a.lengths != nullptr) {
      const int64_t n = a.wide_lengths ? static_cast<const int64_t*>(a.lengths)[batch]
                                       : static_cast<const int32_t*>(a.lengths)[batch];
      length = n < 0 ? 0 : (n < a.tokens ? n : a.tokens);
    }
    begin = split * a.split_tokens;
    end = begin + a.split_tokens < a.tokens ? begin + a.split_tokens : a.tokens;
  }
};

// Tokens of [first, first + kRun) before `stop`, 0 to kRun; the same for the whole wave.
__device__ __forceinline__ int tokens_before(int64_t first, int64_t stop) {
  const int64_t n = stop - first;
  return n <= 0 ? 0 : (n < kRun ? static_cast<int>(n) : kRun);
}

// kRun tokens of a wave's channels; from token `live` on, `fill`.
template <typename T, int CPL>
__device__ __forceinline__ void load_tokens(Run<T, CPL> (&r)[kRun], const T* base, int64_t first,
                                            int64_t stride, int channel, int live, float fill) {
  const T* p = base + first * stride;
  if (live == kRun) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) r[i] = load_run<CPL>(p + i * stride + channel);
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) r[i].v[j] = static_cast<T>(fill);
      if (i < live) r[i] = load_run<CPL>(p + i * stride + channel);
    }
  }
}

// `stored` tokens written, of which those from `live` on as zeros.
template <typename T, int CPL>
__device__ __forceinline__ void store_tokens(T* base, int64_t first, int64_t stride, int channel,
                                             bool valid, int live, int stored,
                                             const float (&v)[kRun][CPL]) {
  if (!valid) return;
  T* p = base + first * stride;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    if (i >= stored) break;
    Run<T, CPL> r;
#pragma unroll
    for (int j = 0; j < CPL; ++j) r.v[j] = static_cast<T>(i < live ? v[i][j] : 0.f);
    store_run<CPL>(p + i * stride + channel, r);
  }
}

// kSummary: only the split's map (A, B) is left, in a.summary.
template <typename T, int CPL, int NW, bool kSummary>
__global__ __launch_bounds__(64 * NW) void recurrence_forward(RecurrenceArgs a) {
  __shared__ float maps[2][NW][2][64 * CPL];
  const Place<CPL> at(a);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t C = a.channels;
  const T* x = static_cast<const T*>(a.input) + at.batch * a.input_batch;
  const T* g = static_cast<const T*>(a.gate) + at.batch * a.gate_batch;
  T* y = static_cast<T*>(a.output) + at.batch * a.tokens * C;
  float carry[CPL], total[CPL];  // state before the tile (of the split's map: B, and A in total)
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    carry[j] = 0.f;
    total[j] = 1.f;
  }
  if constexpr (!kSummary) {
    if (a.first != nullptr) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = a.first[at.batch * C + at.channel + j];
    }
    const float* sum = a.summary + at.batch * a.splits * 2 * C + at.channel;
#pragma unroll 4
    for (int s = 0; s < at.split; ++s, sum += 2 * C) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(sum[j], carry[j], sum[C + j]);
    }
  }
  Run<T, CPL> nx[kRun], ng[kRun];
  auto fetch = [&](int64_t first) __attribute__((always_inline)) {
    const int live = tokens_before(first, at.length);
    load_tokens<T, CPL>(ng, g, first, a.gate_token, at.channel, live, __builtin_inff());
    load_tokens<T, CPL>(nx, x, first, a.input_token, at.channel, live, 0.f);
  };
  if (at.begin < at.end) fetch(at.begin + wave * kRun);
  int buffer = 0;
  for (int64_t tile = at.begin; tile < at.end; tile += NW * kRun, buffer ^= 1) {
    const int64_t first = tile + wave * kRun;
    float keep[kRun][CPL], add[kRun][CPL], A[CPL], B[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      A[j] = 1.f;
      B[j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
        keep[i][j] = q.keep;
        add[i][j] = q.take * static_cast<float>(nx[i].v[j]);
        A[j] *= q.keep;
        B[j] = fmaf(q.keep, B[j], add[i][j]);
      }
    if (tile + NW * kRun < at.end) fetch(first + NW * kRun);
    if constexpr (!kSummary) {
      if (a.carries != nullptr && wave == 0 && at.valid) {
        const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
        float* c = a.carries + (at.batch * tiles + tile / kRecurrenceTile) * C + at.channel;
#pragma unroll
        for (int j = 0; j < CPL; ++j) c[j] = carry[j];
      }
    }
    float h[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) h[j] = carry[j];
    if constexpr (NW > 1) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        maps[buffer][wave][0][lane * CPL + j] = A[j];
        maps[buffer][wave][1][lane * CPL + j] = B[j];
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          if (w == wave) h[j] = carry[j];
          const float aw = maps[buffer][w][0][lane * CPL + j];
          carry[j] = fmaf(aw, carry[j], maps[buffer][w][1][lane * CPL + j]);
          if constexpr (kSummary) total[j] *= aw;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        carry[j] = fmaf(A[j], carry[j], B[j]);
        if constexpr (kSummary) total[j] *= A[j];
      }
    }
    if constexpr (!kSummary) {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          h[j] = fmaf(keep[i][j], h[j], add[i][j]);
          keep[i][j] = h[j];
        }
      store_tokens<T, CPL>(y, first, C, at.channel, at.valid, tokens_before(first, at.length),
                           tokens_before(first, at.end), keep);
    }
  }
  if (wave != 0 || !at.valid) return;
  if constexpr (kSummary) {
    float* sum = a.summary + (at.batch * a.splits + at.split) * 2 * C + at.channel;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      sum[j] = total[j];
      sum[C + j] = carry[j];
    }
  } else if (at.split == a.splits - 1) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) a.last[at.batch * C + at.channel + j] = carry[j];
  }
}

// The backward walks the tiles from the last. kSummary: only the split's map of E, (A, R), is left.
template <typename T, int CPL, int NW, bool kSummary>
__global__ __launch_bounds__(64 * NW) void recurrence_backward(RecurrenceArgs a) {
  __shared__ float maps[2][NW][3][64 * CPL];
  const Place<CPL> at(a);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t C = a.channels;
  const T* x = static_cast<const T*>(a.input) + at.batch * a.input_batch;
  const T* g = static_cast<const T*>(a.gate) + at.batch * a.gate_batch;
  const T* dy = static_cast<const T*>(a.grad_output) + at.batch * a.grad_batch;
  T* dx = static_cast<T*>(a.grad_input) + at.batch * a.tokens * C;
  T* dg = static_cast<T*>(a.grad_gate) + at.batch * a.tokens * C;
  const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
  float carry[CPL], total[CPL];  // E after the tile (of the split's map: R, and A in total)
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    carry[j] = 0.f;
    total[j] = 1.f;
  }
  if constexpr (!kSummary) {
    if (a.grad_last != nullptr) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = a.grad_last[at.batch * C + at.channel + j];
    }
    const float* sum = a.summary + ((at.batch + 1) * a.splits - 1) * 2 * C + at.channel;
#pragma unroll 4
    for (int s = a.splits - 1; s > at.split; --s, sum -= 2 * C) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(sum[j], carry[j], sum[C + j]);
    }
  }
  Run<T, CPL> nx[kRun], ng[kRun], nd[kRun];
  float nh[CPL];
  auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
    const int64_t first = tile + wave * kRun;
    const int live = tokens_before(first, at.length);
    load_tokens<T, CPL>(ng, g, first, a.gate_token, at.channel, live, __builtin_inff());
    load_tokens<T, CPL>(nd, dy, first, a.grad_token, at.channel, live, 0.f);
    if constexpr (!kSummary) {
      load_tokens<T, CPL>(nx, x, first, a.input_token, at.channel, live, 0.f);
      const float* c = a.carries + (at.batch * tiles + tile / kRecurrenceTile) * C + at.channel;
#pragma unroll
      for (int j = 0; j < CPL; ++j) nh[j] = c[j];
    }
  };
  const int64_t count = at.end > at.begin ? (at.end - at.begin + NW * kRun - 1) / (NW * kRun) : 0;
  int64_t tile = at.begin + (count - 1) * NW * kRun;
  if (count > 0) fetch(tile);
  int buffer = 0;
  for (int64_t n = 0; n < count; ++n, tile -= NW * kRun, buffer ^= 1) {
    const int64_t first = tile + wave * kRun;
    float keep[kRun][CPL], take[kRun][CPL], xv[kRun][CPL], dv[kRun][CPL];
    float A[CPL], F[CPL], R[CPL], h[CPL], e[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      A[j] = 1.f;
      F[j] = R[j] = 0.f;
      h[j] = kSummary ? 0.f : nh[j];
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
        keep[i][j] = q.keep;
        dv[i][j] = static_cast<float>(nd[i].v[j]);
        A[j] *= q.keep;
        if constexpr (!kSummary) {
          take[i][j] = q.take;
          xv[i][j] = static_cast<float>(nx[i].v[j]);
          F[j] = fmaf(q.keep, F[j], q.take * xv[i][j]);
        }
      }
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) R[j] = keep[i][j] * (dv[i][j] + R[j]);
    if (n + 1 < count) fetch(tile - NW * kRun);
#pragma unroll
    for (int j = 0; j < CPL; ++j) e[j] = carry[j];
    if constexpr (NW > 1) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        maps[buffer][wave][0][lane * CPL + j] = A[j];
        maps[buffer][wave][1][lane * CPL + j] = R[j];
        if constexpr (!kSummary) maps[buffer][wave][2][lane * CPL + j] = F[j];
      }
      __syncthreads();
#pragma unroll
      for (int w = NW - 1; w >= 0; --w)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          if (w == wave) e[j] = carry[j];
          const float aw = maps[buffer][w][0][lane * CPL + j];
          carry[j] = fmaf(aw, carry[j], maps[buffer][w][1][lane * CPL + j]);
          if constexpr (kSummary) total[j] *= aw;
        }
      if constexpr (!kSummary) {
#pragma unroll
        for (int w = 0; w < NW - 1; ++w)
#pragma unroll
          for (int j = 0; j < CPL; ++j)
            if (w < wave)
              h[j] = fmaf(maps[buffer][w][0][lane * CPL + j], h[j],
                          maps[buffer][w][2][lane * CPL + j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        carry[j] = fmaf(A[j], carry[j], R[j]);
        if constexpr (kSummary) total[j] *= A[j];
      }
    }
    if constexpr (!kSummary) {
      // xv becomes (h_before - x) a (1 - a), then dgate; take becomes dx.
#pragma unroll
      for (int i = 0; i < kRun; ++i)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const float xi = xv[i][j];
          xv[i][j] = (h[j] - xi) * (keep[i][j] * take[i][j]);
          h[j] = fmaf(keep[i][j], h[j], take[i][j] * xi);
        }
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const float d = dv[i][j] + e[j];
          e[j] = keep[i][j] * d;
          take[i][j] *= d;
          xv[i][j] *= d;
        }
      const int live = tokens_before(first, at.length), stored = tokens_before(first, at.end);
      store_tokens<T, CPL>(dx, first, C, at.channel, at.valid, live, stored, take);
      store_tokens<T, CPL>(dg, first, C, at.channel, at.valid, live, stored, xv);
    }
  }
  if (wave != 0 || !at.valid) return;
  if constexpr (kSummary) {
    float* sum = a.summary + (at.batch * a.splits + at.split) * 2 * C + at.channel;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      sum[j] = total[j];
      sum[C + j] = carry[j];
    }
  } else if (at.split == 0 && a.grad_first != nullptr) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) a.grad_first[at.batch * C + at.channel + j] = carry[j];
  }
}

template <typename T, int CPL, int NW>
hipError_t launch_shape(const RecurrenceArgs& a, bool backward, hipStream_t stream) {
  const int64_t strips = (a.channels + 64 * CPL - 1) / (64 * CPL);
  const dim3 grid(static_cast<unsigned>(strips * a.splits * a.batch)), block(64 * NW);
  if (a.splits > 1) {
    if (backward)
      hipLaunchKernelGGL((recurrence_backward<T, CPL, NW, true>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((recurrence_forward<T, CPL, NW, true>), grid, block, 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  if (backward)
    hipLaunchKernelGGL((recurrence_backward<T, CPL, NW, false>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((recurrence_forward<T, CPL, NW, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_recurrence_typed(const RecurrenceArgs& a, bool backward, const RecurrencePlan& p,
                                   hipStream_t stream) {
  if (p.channels_per_lane == 2)
    return p.waves == 1 ? launch_shape<T, 2, 1>(a, backward, stream)
                        : launch_shape<T, 2, 8>(a, backward, stream);
  return p.waves == 1 ? launch_shape<T, 1, 1>(a, backward, stream)
                      : launch_shape<T, 1, 8>(a, backward, stream);
}

}  // namespace

RecurrencePlan plan_recurrence(convnd_hip_dtype dtype, const RecurrenceArgs& a, bool backward) {
  (void)backward;
  RecurrencePlan p{};
  p.waves = a.tokens <= kRun ? 1 : 8;
  // Two channels a lane read 16-bit rows in 256-byte segments, where that leaves enough workgroups.
  const bool even = a.channels % 2 == 0;
  p.channels_per_lane =
      dtype != CONVND_HIP_FLOAT32 && even && a.batch * a.channels / 128 >= 512 ? 2 : 1;
  const int64_t strips = (a.channels + 64 * p.channels_per_lane - 1) / (64 * p.channels_per_lane);
  const int64_t groups = strips * std::max<int64_t>(1, a.batch);
  const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
  p.splits = 1;
  p.split_tokens = std::max<int64_t>(1, tiles) * kRecurrenceTile;
  if (groups < 256 && tiles >= 8) {
    const int64_t wanted = std::min<int64_t>((512 + groups - 1) / groups, tiles / 2);
    const int64_t per = (tiles + wanted - 1) / wanted;
    p.splits = static_cast<int>((tiles + per - 1) / per);
    p.split_tokens = per * kRecurrenceTile;
  }
  return p;
}

hipError_t launch_recurrence(convnd_hip_dtype dtype, const RecurrenceArgs& a, bool backward,
                             const RecurrencePlan& p, hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return launch_recurrence_typed<float>(a, backward, p, stream);
    case CONVND_HIP_FLOAT16:
      return launch_recurrence_typed<_Float16>(a, backward, p, stream);
    case CONVND_HIP_BFLOAT16:
      return launch_recurrence_typed<__bf16>(a, backward, p, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace convnd
