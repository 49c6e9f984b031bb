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
// two in the backward, which makes its states again from one saved state per 64 tokens instead of
// reading h. A run of tokens acts on the state as h -> A h + B, and such maps compose:
//   * A lane owns a channel (two of a 16-bit type) and walks 8 consecutive tokens of it in
//     registers, once for the run's map and, when the state before the run is known, again.
//   * The 64 lanes of a wave are one run, or two or four that follow each other, of as many times
//     fewer channels; the 8 waves of a workgroup take the next runs. The maps are scanned over the
//     runs of a wave with lane shuffles and over the waves through LDS (one barrier a tile, two
//     buffers), and the carried state goes on to the next tile, whose loads are in flight
//     meanwhile. Fewer channels make more workgroups of the same problem.
//   * Rows are addressed as buffers with a 32-bit lane offset, the tile's end being the buffer's:
//     64-bit row addresses cost more than the arithmetic (8 x 2048 x 1024 bf16 backward 51 -> 44 us).
//   * Where there are still few, the token axis is split over workgroups: a first launch leaves
//     every split's map, the second composes the maps before its split and goes on as above (it
//     reads the inputs again; the first walks each split from the end the second comes to last, so
//     that what is read again first is what was read last).
// Every sum is in fp32 and in a fixed order; 1 - a is computed as sigmoid(-gate), which keeps its
// relative precision where a is near 1.

#include <algorithm>
#include <type_traits>

#include "convnd_internal.h"
#include "convnd_sequence.h"

namespace convnd {
namespace {

constexpr int kRun = 8;  // tokens of a run

struct Gate {
  float keep, take;  // sigmoid(g), sigmoid(-g)
};
__device__ __forceinline__ Gate open_gate(float g) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896f * fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.f + e);
  const float s = e * r;
  return g >= 0.f ? Gate{r, s} : Gate{s, r};
}

// The maps v -> a v + b of one lane's channels.
template <int CPL>
struct Map {
  float a[CPL], b[CPL];
  // This map after `before`.
  __device__ __forceinline__ void after(const Map& before) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      b[j] = fmaf(a[j], before.b[j], b[j]);
      a[j] *= before.a[j];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      a[j] = 1.f;
      b[j] = 0.f;
    }
  }
};

// Scan over the 64 / LANES runs of a wave, in token order (kUp) or from the last run: `m` becomes
// the map up to and with the lane's run, `before` the one without it.
template <int CPL, int LANES, bool kUp>
__device__ __forceinline__ void scan_runs(Map<CPL>& m, Map<CPL>& before) {
  before.clear();
  if constexpr (LANES < 64) {
    const int run = (threadIdx.x & 63) / LANES;
    const int place = kUp ? run : 64 / LANES - 1 - run;
    auto shifted = [&](int runs) {
      Map<CPL> o;
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        o.a[j] = kUp ? __shfl_up(m.a[j], runs * LANES) : __shfl_down(m.a[j], runs * LANES);
        o.b[j] = kUp ? __shfl_up(m.b[j], runs * LANES) : __shfl_down(m.b[j], runs * LANES);
      }
      return o;
    };
#pragma unroll
    for (int d = 1; d < 64 / LANES; d *= 2) {
      const Map<CPL> o = shifted(d);
      if (place >= d) m.after(o);
    }
    const Map<CPL> o = shifted(1);
    if (place >= 1) before = o;
  }
}

// The place of this workgroup and lane in the problem.
template <int CPL, int LANES>
struct Place {
  int64_t batch, length, begin, end;  // tokens [begin, end) of the split
  int split, channel;  // the lane's first channel, or the last whole one past the edge
  bool valid;
  __device__ __forceinline__ explicit Place(const RecurrenceArgs& a) {
    const int strips = static_cast<int>((a.channels + LANES * CPL - 1) / (LANES * CPL));
    // Workgroup ids go round the eight XCDs: neighbouring strips, whose row segments may share a
    // cache line, are given to the same one.
    const unsigned per = gridDim.x >> 3, rest = gridDim.x & 7, xcd = blockIdx.x & 7;
    unsigned id = xcd * per + (xcd < rest ? xcd : rest) + (blockIdx.x >> 3);
    const int strip = static_cast<int>(id % strips);
    id /= strips;
    split = static_cast<int>(id % a.splits);
    batch = id / a.splits;
    const int C = static_cast<int>(a.channels);
    const int own = (strip * LANES + static_cast<int>(threadIdx.x) % LANES) * CPL;
    valid = own < C;
    channel = valid ? own : C - CPL;
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

// The lane's tokens of a tile before `stop`, 0 to kRun, given the tile's first token.
__device__ __forceinline__ int tokens_before(int64_t tile, int run_token, int64_t stop) {
  const int64_t n = stop - tile - run_token;
  return n <= 0 ? 0 : (n < kRun ? static_cast<int>(n) : kRun);
}

// The rows of a tile before token `stop` as a buffer: reads past it give zeros, writes are dropped.
template <int kTile, typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rows(const T* base, int64_t tile,
                                                            int64_t stop, int64_t stride,
                                                            int64_t channels) {
  const int64_t rows = stop - tile < kTile ? stop - tile : kTile;
  const int64_t bytes = rows > 0 ? ((rows - 1) * stride + channels) * sizeof(T) : 0;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + tile * stride), 0,
                                           static_cast<int>(bytes), 0x00020000);
}

// kRun tokens of the lane's channels, `step` bytes apart.
template <typename T, int CPL>
__device__ __forceinline__ void load_tokens(Run<T, CPL> (&r)[kRun], __amdgpu_buffer_rsrc_t rows,
                                            unsigned offset, unsigned step) {
  // Hidden, so that the kRun offsets are added up here and not kept over the loop of tiles.
  asm volatile("" : "+v"(offset));
#pragma unroll
  for (int i = 0; i < kRun; ++i, offset += step) {
    if constexpr (sizeof(T) * CPL == 4)
      r[i] = __builtin_bit_cast(Run<T, CPL>,
                                __builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, 0));
    else
      r[i] = __builtin_bit_cast(Run<T, CPL>,
                                __builtin_amdgcn_raw_buffer_load_b16(rows, offset, 0, 0));
  }
}

template <typename T, int CPL>
__device__ __forceinline__ void store_tokens(__amdgpu_buffer_rsrc_t rows, unsigned offset,
                                             unsigned step, const float (&v)[kRun][CPL]) {
  asm volatile("" : "+v"(offset));
#pragma unroll
  for (int i = 0; i < kRun; ++i, offset += step) {
    Run<T, CPL> r;
#pragma unroll
    for (int j = 0; j < CPL; ++j) r.v[j] = static_cast<T>(v[i][j]);
    if constexpr (sizeof(T) * CPL == 4)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, r), rows, offset, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, r), rows, offset, 0,
                                            0);
  }
}

// From token `live` on, `fill`.
template <typename T, int CPL>
__device__ __forceinline__ void fill_tokens(Run<T, CPL> (&r)[kRun], int live, float fill) {
#pragma unroll
  for (int i = 0; i < kRun; ++i)
#pragma unroll
    for (int j = 0; j < CPL; ++j) r[i].v[j] = i < live ? r[i].v[j] : static_cast<T>(fill);
}
template <int CPL>
__device__ __forceinline__ void clear_tokens(float (&v)[kRun][CPL], int live) {
#pragma unroll
  for (int i = 0; i < kRun; ++i)
#pragma unroll
    for (int j = 0; j < CPL; ++j) v[i][j] = i < live ? v[i][j] : 0.f;
}

// Byte offset of the lane's first token and channel in a tile's rows.
template <typename T>
__device__ __forceinline__ unsigned lane_offset(int run_token, int64_t stride, int channel) {
  return (run_token * static_cast<unsigned>(stride) + channel) * sizeof(T);
}
constexpr unsigned kNowhere = 0x80000000u;  // past every tile's rows (below 2^31 bytes)

// Hides the value from the compiler, which would else keep the converted floats (twice the
// registers) from its first use to this one.
template <typename T>
__device__ __forceinline__ void hold(Run<T, 2>& r) {
  if constexpr (sizeof(T) == 2) {
    unsigned bits = __builtin_bit_cast(unsigned, r);
    asm volatile("" : "+v"(bits));
    r = __builtin_bit_cast(Run<T, 2>, bits);
  }
}
template <typename T>
__device__ __forceinline__ void hold(Run<T, 1>&) {}

// kSummary: only the split's map is left, in a.summary.
template <typename T, int CPL, int LANES, int NW, bool kSummary>
__global__ __launch_bounds__(64 * NW) void recurrence_forward(RecurrenceArgs a) {
  constexpr int kTile = NW * (64 / LANES) * kRun;
  __shared__ float maps[2][NW][2][LANES * CPL];
  const Place<CPL, LANES> at(a);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int run_token = (static_cast<int>(threadIdx.x) / LANES) * kRun;
  const int slot = lane % LANES * CPL;
  const int64_t C = a.channels;
  const T* x = static_cast<const T*>(a.input) + at.batch * a.input_batch;
  const T* g = static_cast<const T*>(a.gate) + at.batch * a.gate_batch;
  T* y = static_cast<T*>(a.output) + at.batch * a.tokens * C;
  const unsigned x_lane = lane_offset<T>(run_token, a.input_token, at.channel);
  const unsigned g_lane = lane_offset<T>(run_token, a.gate_token, at.channel);
  const unsigned y_lane = at.valid ? lane_offset<T>(run_token, C, at.channel) : kNowhere;
  float carry[CPL];  // the state before the tile
  Map<CPL> total;    // the split's map (kSummary)
  total.clear();
#pragma unroll
  for (int j = 0; j < CPL; ++j) carry[j] = 0.f;
  if constexpr (!kSummary) {
    if (a.first != nullptr) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = a.first[at.batch * C + at.channel + j];
    }
    const float* sum = a.summary + at.batch * a.splits * 2 * C + at.channel;
#pragma unroll 8
    for (int s = 0; s < at.split; ++s, sum += 2 * C) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(sum[j], carry[j], sum[C + j]);
    }
  }
  Run<T, CPL> nx[kRun], ng[kRun];
  auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
    load_tokens<T, CPL>(ng, tile_rows<kTile>(g, tile, at.length, a.gate_token, C), g_lane,
                        static_cast<unsigned>(a.gate_token) * sizeof(T));
    load_tokens<T, CPL>(nx, tile_rows<kTile>(x, tile, at.length, a.input_token, C), x_lane,
                        static_cast<unsigned>(a.input_token) * sizeof(T));
  };
  const int64_t count = at.end > at.begin ? (at.end - at.begin + kTile - 1) / kTile : 0;
  // The summary goes from the last tile to the first.
  int64_t tile = kSummary ? at.begin + (count - 1) * kTile : at.begin;
  constexpr int64_t kNext = kSummary ? -kTile : kTile;
  if (count > 0) fetch(tile);
  int buffer = 0;
  for (int64_t n = 0; n < count; ++n, tile += kNext, buffer ^= 1) {
    float keep[kRun][CPL], add[kRun][CPL];
    Map<CPL> map, before;
    map.clear();
    // Tokens past the length: open gates (the buffers gave zeros).
    const bool cut = tile + kTile > at.length;
    const int live = tokens_before(tile, run_token, at.length);
    if (cut) fill_tokens(ng, live, __builtin_inff());
#pragma unroll
    for (int i = 0; i < kRun; ++i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
        keep[i][j] = q.keep;
        add[i][j] = q.take * static_cast<float>(nx[i].v[j]);
        map.a[j] *= q.keep;
        map.b[j] = fmaf(q.keep, map.b[j], add[i][j]);
      }
    if (n + 1 < count) fetch(tile + kNext);
    scan_runs<CPL, LANES, true>(map, before);
    float h[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) h[j] = carry[j];
    if constexpr (NW > 1) {
      if (lane >= 64 - LANES) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          maps[buffer][wave][0][slot + j] = map.a[j];
          maps[buffer][wave][1][slot + j] = map.b[j];
        }
      }
      __syncthreads();
      Map<CPL> whole;
      whole.clear();
#pragma unroll
      for (int w = 0; w < NW; ++w) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const float aw = maps[buffer][w][0][slot + j], bw = maps[buffer][w][1][slot + j];
          if constexpr (kSummary) {
            whole.b[j] = fmaf(aw, whole.b[j], bw);
            whole.a[j] *= aw;
          } else {
            if (w == wave) h[j] = carry[j];
            carry[j] = fmaf(aw, carry[j], bw);
          }
        }
      }
      if constexpr (kSummary) total.after(whole);  // the tiles before this one came later
    } else {
      static_assert(NW > 1 || (LANES == 64 && !kSummary), "one wave takes one run, without splits");
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(map.a[j], carry[j], map.b[j]);
    }
    if constexpr (!kSummary) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) h[j] = fmaf(before.a[j], h[j], before.b[j]);
      const int64_t first = tile + run_token;
      if (a.carries != nullptr && at.valid && first % kRecurrenceTile == 0 && first < at.end) {
        const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
        float* c = a.carries + (at.batch * tiles + first / kRecurrenceTile) * C + at.channel;
#pragma unroll
        for (int j = 0; j < CPL; ++j) c[j] = h[j];
      }
#pragma unroll
      for (int i = 0; i < kRun; ++i)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          h[j] = fmaf(keep[i][j], h[j], add[i][j]);
          keep[i][j] = h[j];
        }
      if (cut) clear_tokens(keep, live);
      store_tokens<T, CPL>(tile_rows<kTile>(y, tile, at.end, C, C), y_lane,
                           static_cast<unsigned>(C) * sizeof(T), keep);
    }
  }
  if (threadIdx.x >= LANES || !at.valid) return;
  if constexpr (kSummary) {
    float* sum = a.summary + (at.batch * a.splits + at.split) * 2 * C + at.channel;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      sum[j] = total.a[j];
      sum[C + j] = total.b[j];
    }
  } else if (at.split == a.splits - 1) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) a.last[at.batch * C + at.channel + j] = carry[j];
  }
}

// The backward walks the tiles from the last. kSummary: only the split's map of E is left.
template <typename T, int CPL, int LANES, int NW, bool kSummary>
__global__ __launch_bounds__(64 * NW) void recurrence_backward(RecurrenceArgs a) {
  constexpr int kTile = NW * (64 / LANES) * kRun;
  __shared__ float maps[2][NW][kSummary ? 2 : 3][LANES * CPL];
  const Place<CPL, LANES> at(a);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int run_token = (static_cast<int>(threadIdx.x) / LANES) * kRun;
  const int slot = lane % LANES * CPL;
  const int64_t C = a.channels;
  const T* x = static_cast<const T*>(a.input) + at.batch * a.input_batch;
  const T* g = static_cast<const T*>(a.gate) + at.batch * a.gate_batch;
  const T* dy = static_cast<const T*>(a.grad_output) + at.batch * a.grad_batch;
  T* dx = static_cast<T*>(a.grad_input) + at.batch * a.tokens * C;
  T* dg = static_cast<T*>(a.grad_gate) + at.batch * a.tokens * C;
  const unsigned x_lane = lane_offset<T>(run_token, a.input_token, at.channel);
  const unsigned g_lane = lane_offset<T>(run_token, a.gate_token, at.channel);
  const unsigned d_lane = lane_offset<T>(run_token, a.grad_token, at.channel);
  const unsigned out_lane = at.valid ? lane_offset<T>(run_token, C, at.channel) : kNowhere;
  const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
  float carry[CPL];  // E after the tile
  Map<CPL> total;    // the split's map (kSummary)
  total.clear();
#pragma unroll
  for (int j = 0; j < CPL; ++j) carry[j] = 0.f;
  if constexpr (!kSummary) {
    if (a.grad_last != nullptr) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = a.grad_last[at.batch * C + at.channel + j];
    }
    const float* sum = a.summary + ((at.batch + 1) * a.splits - 1) * 2 * C + at.channel;
#pragma unroll 8
    for (int s = a.splits - 1; s > at.split; --s, sum -= 2 * C) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(sum[j], carry[j], sum[C + j]);
    }
  }
  Run<T, CPL> nx[kRun], ng[kRun], nd[kRun];
  float nh[CPL];  // the state before the tile
  auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
    load_tokens<T, CPL>(ng, tile_rows<kTile>(g, tile, at.length, a.gate_token, C), g_lane,
                        static_cast<unsigned>(a.gate_token) * sizeof(T));
    load_tokens<T, CPL>(nd, tile_rows<kTile>(dy, tile, at.length, a.grad_token, C), d_lane,
                        static_cast<unsigned>(a.grad_token) * sizeof(T));
    if constexpr (!kSummary) {
      load_tokens<T, CPL>(nx, tile_rows<kTile>(x, tile, at.length, a.input_token, C), x_lane,
                          static_cast<unsigned>(a.input_token) * sizeof(T));
      const float* c = a.carries + (at.batch * tiles + tile / kRecurrenceTile) * C + at.channel;
#pragma unroll
      for (int j = 0; j < CPL; ++j) nh[j] = c[j];
    }
  };
  const int64_t count = at.end > at.begin ? (at.end - at.begin + kTile - 1) / kTile : 0;
  // The summary goes from the first tile to the last.
  int64_t tile = kSummary ? at.begin : at.begin + (count - 1) * kTile;
  constexpr int64_t kNext = kSummary ? kTile : -kTile;
  if (count > 0) fetch(tile);
  int buffer = 0;
  for (int64_t n = 0; n < count; ++n, tile += kNext, buffer ^= 1) {
    float keep[kRun][CPL], take[kRun][CPL];
    Run<T, CPL> cx[kRun], cd[kRun];  // this tile's x and dy, as loaded
    Map<CPL> states, states_before, grads, grads_before;
    float h[CPL], e[CPL];
    states.clear();
    grads.clear();
    const bool cut = tile + kTile > at.length;
    const int live = tokens_before(tile, run_token, at.length);
    if (cut) fill_tokens(ng, live, __builtin_inff());
#pragma unroll
    for (int j = 0; j < CPL; ++j) h[j] = kSummary ? 0.f : nh[j];
#pragma unroll
    for (int i = 0; i < kRun; ++i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
        keep[i][j] = q.keep;
        states.a[j] *= q.keep;
        if constexpr (!kSummary) {
          take[i][j] = q.take;
          states.b[j] = fmaf(q.keep, states.b[j], q.take * static_cast<float>(nx[i].v[j]));
        }
      }
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) grads.b[j] = keep[i][j] * (static_cast<float>(nd[i].v[j]) + grads.b[j]);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      cd[i] = nd[i];
      if constexpr (!kSummary) cx[i] = nx[i];
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) grads.a[j] = states.a[j];
    if (n + 1 < count) fetch(tile + kNext);
    scan_runs<CPL, LANES, false>(grads, grads_before);
    if constexpr (!kSummary) scan_runs<CPL, LANES, true>(states, states_before);
#pragma unroll
    for (int j = 0; j < CPL; ++j) e[j] = carry[j];
    if constexpr (NW > 1) {
      // The wave's maps: of E in its first run's lanes, of the state in its last run's.
      if (lane < LANES) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          maps[buffer][wave][0][slot + j] = grads.a[j];
          maps[buffer][wave][1][slot + j] = grads.b[j];
        }
      }
      if constexpr (!kSummary) {
        if (lane >= 64 - LANES) {
#pragma unroll
          for (int j = 0; j < CPL; ++j) maps[buffer][wave][2][slot + j] = states.b[j];
        }
      }
      __syncthreads();
      Map<CPL> whole;
      whole.clear();
#pragma unroll
      for (int w = NW - 1; w >= 0; --w)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const float aw = maps[buffer][w][0][slot + j], bw = maps[buffer][w][1][slot + j];
          if constexpr (kSummary) {
            whole.b[j] = fmaf(aw, whole.b[j], bw);
            whole.a[j] *= aw;
          } else {
            if (w == wave) e[j] = carry[j];
            carry[j] = fmaf(aw, carry[j], bw);
          }
        }
      if constexpr (kSummary) {
        total.after(whole);
      } else {
#pragma unroll
        for (int w = 0; w < NW - 1; ++w)
#pragma unroll
          for (int j = 0; j < CPL; ++j)
            if (w < wave)
              h[j] = fmaf(maps[buffer][w][0][slot + j], h[j], maps[buffer][w][2][slot + j]);
      }
    } else {
      static_assert(NW > 1 || (LANES == 64 && !kSummary), "one wave takes one run, without splits");
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(grads.a[j], carry[j], grads.b[j]);
    }
    if constexpr (!kSummary) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        h[j] = fmaf(states_before.a[j], h[j], states_before.b[j]);
        e[j] = fmaf(grads_before.a[j], e[j], grads_before.b[j]);
      }
      // slope is (h_before - x) a (1 - a), then dgate; take becomes dx.
      float slope[kRun][CPL];
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        hold(cx[i]);
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const float xi = static_cast<float>(cx[i].v[j]);
          slope[i][j] = (h[j] - xi) * (keep[i][j] * take[i][j]);
          h[j] = fmaf(keep[i][j], h[j], take[i][j] * xi);
        }
      }
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i) {
        hold(cd[i]);
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const float d = static_cast<float>(cd[i].v[j]) + e[j];
          e[j] = keep[i][j] * d;
          take[i][j] *= d;
          slope[i][j] *= d;
        }
      }
      if (cut) {
        clear_tokens(take, live);
        clear_tokens(slope, live);
      }
      const unsigned step = static_cast<unsigned>(C) * sizeof(T);
      store_tokens<T, CPL>(tile_rows<kTile>(dx, tile, at.end, C, C), out_lane, step, take);
      store_tokens<T, CPL>(tile_rows<kTile>(dg, tile, at.end, C, C), out_lane, step, slope);
    }
  }
  if (threadIdx.x >= LANES || !at.valid) return;
  if constexpr (kSummary) {
    float* sum = a.summary + (at.batch * a.splits + at.split) * 2 * C + at.channel;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      sum[j] = total.a[j];
      sum[C + j] = total.b[j];
    }
  } else if (at.split == 0 && a.grad_first != nullptr) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) a.grad_first[at.batch * C + at.channel + j] = carry[j];
  }
}

// Up to kRun tokens, as in decoding: a thread walks its channels' tokens from the state.
constexpr int kStepThreads = 64;
template <typename T, int CPL>
__global__ __launch_bounds__(kStepThreads) void recurrence_step(RecurrenceArgs a) {
  const int64_t C = a.channels, parts = (C + CPL - 1) / CPL;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kStepThreads + threadIdx.x;
  if (id >= parts * a.batch) return;
  const int64_t batch = id / parts, channel = id % parts * CPL;
  int64_t length = a.tokens;
  if (a.lengths != nullptr) {
    const int64_t n = a.wide_lengths ? static_cast<const int64_t*>(a.lengths)[batch]
                                     : static_cast<const int32_t*>(a.lengths)[batch];
    length = n < 0 ? 0 : (n < a.tokens ? n : a.tokens);
  }
  const T* x = static_cast<const T*>(a.input) + batch * a.input_batch + channel;
  const T* g = static_cast<const T*>(a.gate) + batch * a.gate_batch + channel;
  T* y = static_cast<T*>(a.output) + batch * a.tokens * C + channel;
  const int64_t state = batch * C + channel;
  float h[CPL];
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    h[j] = a.first != nullptr ? a.first[state + j] : 0.f;
    // One saved state per sequence: its first (so few tokens are one tile).
    if (a.carries != nullptr && a.tokens > 0) a.carries[state + j] = h[j];
  }
  for (int64_t t = 0; t < a.tokens; ++t) {
    Run<T, CPL> r;
#pragma unroll
    for (int j = 0; j < CPL; ++j) r.v[j] = static_cast<T>(0.f);
    if (t < length) {
      const Run<T, CPL> gv = load_run<CPL>(g + t * a.gate_token);
      const Run<T, CPL> xv = load_run<CPL>(x + t * a.input_token);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const Gate q = open_gate(static_cast<float>(gv.v[j]));
        h[j] = fmaf(q.keep, h[j], q.take * static_cast<float>(xv.v[j]));
        r.v[j] = static_cast<T>(h[j]);
      }
    }
    store_run<CPL>(y + t * C, r);
  }
#pragma unroll
  for (int j = 0; j < CPL; ++j) a.last[state + j] = h[j];
}

template <typename T, int CPL, int LANES, int NW>
hipError_t launch_shape(const RecurrenceArgs& a, bool backward, hipStream_t stream) {
  const int64_t strips = (a.channels + LANES * CPL - 1) / (LANES * CPL);
  const dim3 grid(static_cast<unsigned>(strips * a.splits * a.batch)), block(64 * NW);
  if constexpr (LANES == 64 && NW > 1) {
    if (a.splits > 1) {
      if (backward)
        hipLaunchKernelGGL((recurrence_backward<T, CPL, LANES, NW, true>), grid, block, 0, stream,
                           a);
      else
        hipLaunchKernelGGL((recurrence_forward<T, CPL, LANES, NW, true>), grid, block, 0, stream,
                           a);
      const hipError_t err = hipGetLastError();
      if (err != hipSuccess) return err;
    }
  }
  if (backward)
    hipLaunchKernelGGL((recurrence_backward<T, CPL, LANES, NW, false>), grid, block, 0, stream, a);
  else if constexpr (NW > 1)
    hipLaunchKernelGGL((recurrence_forward<T, CPL, LANES, NW, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T, int CPL>
hipError_t launch_channels(const RecurrenceArgs& a, bool backward, const RecurrencePlan& p,
                           hipStream_t stream) {
  if (p.waves == 1) {
    if (backward) return launch_shape<T, CPL, 64, 1>(a, true, stream);
    const int64_t threads = (a.channels + CPL - 1) / CPL * a.batch;
    hipLaunchKernelGGL((recurrence_step<T, CPL>),
                       dim3(static_cast<unsigned>((threads + kStepThreads - 1) / kStepThreads)),
                       dim3(kStepThreads), 0, stream, a);
    return hipGetLastError();
  }
  if (p.lanes == 64) return launch_shape<T, CPL, 64, 8>(a, backward, stream);
  if (p.lanes == 32) return launch_shape<T, CPL, 32, 8>(a, backward, stream);
  return launch_shape<T, CPL, 16, 8>(a, backward, stream);
}

template <typename T>
hipError_t launch_recurrence_typed(const RecurrenceArgs& a, bool backward, const RecurrencePlan& p,
                                   hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.channels_per_lane == 2) return launch_channels<T, 2>(a, backward, p, stream);
  }
  return launch_channels<T, 1>(a, backward, p, stream);
}

}  // namespace

RecurrencePlan plan_recurrence(convnd_hip_dtype dtype, const RecurrenceArgs& a) {
  RecurrencePlan p{};
  p.waves = a.tokens <= kRun ? 1 : 8;
  p.channels_per_lane = dtype != CONVND_HIP_FLOAT32 && a.channels % 2 == 0 ? 2 : 1;
  p.lanes = 64;
  p.splits = 1;
  const int64_t batch = std::max<int64_t>(1, a.batch);
  const auto groups = [&](int lanes) {
    const int64_t wide = lanes * p.channels_per_lane;
    return batch * ((a.channels + wide - 1) / wide);
  };
  const auto tile = [&](int lanes) { return int64_t{8} * (64 / lanes) * kRun; };
  // The widest lanes that give every compute unit a workgroup: forward / backward of
  // 8 x 4096 x 4096 fp16 (256 workgroups at 64 lanes) 163 / 315 us at 64, 189 / 340 at 32;
  // 4 x 4096 x 2048 fp32 102 / 151 at 64 (128 workgroups), 93 / 150 at 32;
  // 8 x 2048 x 1024 bf16 25 / 44 at 16 (128 workgroups), 39 / 52 at 64 in four splits;
  // 13 x 777 x 300 fp16 12 / 20 at 16 (130), 22 / 34 at 64 in four splits.
  while (p.waves > 1 && p.lanes > 16 && a.tokens > tile(p.lanes) && groups(p.lanes) < 256)
    p.lanes /= 2;
  p.split_tokens = std::max<int64_t>(a.tokens, 1);
  // Few workgroups and a long token axis: splits of at least 512 tokens at 64 lanes, one
  // workgroup for every compute unit (1 x 65536 x 512 fp32: 174 us forward at 128 workgroups, 118 at
  // 256, 117 at 512, 128 at 1024).
  if (groups(16) < 128 && a.tokens >= 2048) {
    p.lanes = 64;
    const int64_t tiles = (a.tokens + tile(64) - 1) / tile(64);
    const int64_t wanted = std::min<int64_t>((256 + groups(64) - 1) / groups(64), tiles / 8);
    const int64_t per = (tiles + wanted - 1) / wanted;
    p.splits = static_cast<int>((tiles + per - 1) / per);
    p.split_tokens = per * tile(64);
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
