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
//   * A lane owns a channel (or two of a 16-bit type) and walks 8 consecutive tokens of it in
//     registers, once for the run's map and, when the state before the run is known, again.
//   * The 64 lanes of a wave are one run, or two or four that follow each other, of as many times
//     fewer channels; the 8 waves of a workgroup take the next runs. The maps are scanned over the
//     runs of a wave with lane shuffles and over the waves through LDS (one barrier a tile, two
//     buffers), and the carried state goes on to the next tile, whose loads are in flight
//     meanwhile. Fewer channels make more workgroups of the same problem.
//   * Rows are addressed as buffers with a 32-bit lane offset, the tile's end being the buffer's:
//     64-bit row addresses cost more than the arithmetic (a seventh of a bf16 backward's time).
//   * With few sequences and channels and many tokens, workgroups take chunks of the token axis
//     instead and hand the state on (below).
// Every sum is in fp32 and in a fixed order; 1 - a is computed as sigmoid(-gate), which keeps its
// relative precision where a is near 1.

#include <algorithm>
#include <type_traits>

#include "convnd_internal.h"
#include "convnd_sequence.h"

namespace convnd {
namespace {

constexpr int kRun = 8;    // tokens of a run
constexpr int kWaves = 8;  // of a workgroup

struct Gate {
  float keep, take;  // sigmoid(g), sigmoid(-g)
};
// The larger of the two is 1 less the smaller and so rounded once. As a reciprocal it is off by up to
// an ulp, to the same side for the same gate, and products over thousands of tokens add that up (a
// first state's gradient over 8192 tokens in bfloat16 4.4e-6 off, so 0.7e-6).
__device__ __forceinline__ Gate open_gate(float g) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896f * fabsf(g));
  const float s = e * __builtin_amdgcn_rcpf(1.f + e);
  const float r = 1.f - s;
  return g >= 0.f ? Gate{r, s} : Gate{s, r};
}

// A product of gates, the smallest of them `least`. It stays above zero where none is zero, at the
// smallest value there is, so that an infinite state stays infinite over tokens whose gates' product
// passes below the type's range, as it does token by token (zero times infinity is NaN). To a finite
// state that adds less than 5e-7.
__device__ __forceinline__ float bound_gates(float product, float least) {
  return fmaxf(product, fminf(least, 1.401298464e-45f));
}
__device__ __forceinline__ float join_gates(float a, float b) {
  return bound_gates(a * b, fminf(a, b));
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
      a[j] = join_gates(a[j], before.a[j]);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      a[j] = 1.f;
      b[j] = 0.f;
    }
  }
  // Bounds `a`, the product of these gates. Apart from the product, whose multiplications wait for
  // each other (4 x 16384 x 1024 bf16 took 111 us with a bound at each of them, 99 so).
  template <int N>
  __device__ __forceinline__ void bound(const float (&gates)[N][CPL]) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      float least = gates[0][j];
#pragma unroll
      for (int i = 1; i < N; ++i) least = fminf(least, gates[i][j]);
      a[j] = bound_gates(a[j], least);
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
  int64_t batch, length;
  int channel;  // the lane's first, or the last whole one past the edge
  bool valid;
  __device__ __forceinline__ explicit Place(const RecurrenceArgs& a) {
    const int strips = static_cast<int>((a.channels + LANES * CPL - 1) / (LANES * CPL));
    // Workgroup ids go round the eight XCDs: neighbouring strips, whose row segments may share a
    // cache line, are given to the same one.
    const unsigned per = gridDim.x >> 3, rest = gridDim.x & 7, xcd = blockIdx.x & 7;
    const unsigned id = xcd * per + (xcd < rest ? xcd : rest) + (blockIdx.x >> 3);
    const int strip = static_cast<int>(id % strips);
    batch = id / strips;
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
  }
};

// The lane's tokens of a tile before `stop`, 0 to N, given the tile's first token.
template <int N = kRun>
__device__ __forceinline__ int tokens_before(int64_t tile, int run_token, int64_t stop) {
  const int64_t n = stop - tile - run_token;
  return n <= 0 ? 0 : (n < N ? static_cast<int>(n) : N);
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

// N tokens of the lane's channels, `step` bytes apart.
template <typename T, int CPL, int N>
__device__ __forceinline__ void load_tokens(Run<T, CPL> (&r)[N], __amdgpu_buffer_rsrc_t rows,
                                            unsigned offset, unsigned step) {
  // Hidden, so that the N offsets are added up here and not kept over the loop of tiles.
  asm volatile("" : "+v"(offset));
#pragma unroll
  for (int i = 0; i < N; ++i, offset += step) {
    if constexpr (sizeof(T) * CPL == 4)
      r[i] = __builtin_bit_cast(Run<T, CPL>,
                                __builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, 0));
    else
      r[i] = __builtin_bit_cast(Run<T, CPL>,
                                __builtin_amdgcn_raw_buffer_load_b16(rows, offset, 0, 0));
  }
}

template <typename T, int CPL, int N>
__device__ __forceinline__ void store_tokens(__amdgpu_buffer_rsrc_t rows, unsigned offset,
                                             unsigned step, const float (&v)[N][CPL]) {
  asm volatile("" : "+v"(offset));
#pragma unroll
  for (int i = 0; i < N; ++i, offset += step) {
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
template <typename T, int CPL, int N>
__device__ __forceinline__ void fill_tokens(Run<T, CPL> (&r)[N], int live, float fill) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < CPL; ++j) r[i].v[j] = i < live ? r[i].v[j] : static_cast<T>(fill);
}
template <int CPL, int N>
__device__ __forceinline__ void clear_tokens(float (&v)[N][CPL], int live) {
#pragma unroll
  for (int i = 0; i < N; ++i)
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

template <typename T, int CPL, int LANES>
__global__ __launch_bounds__(64 * kWaves) void recurrence_forward(RecurrenceArgs a) {
  constexpr int kTile = kWaves * (64 / LANES) * kRun;
  __shared__ float maps[2][kWaves][2][LANES * CPL];
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
#pragma unroll
  for (int j = 0; j < CPL; ++j)
    carry[j] = a.first != nullptr ? a.first[at.batch * C + at.channel + j] : 0.f;
  Run<T, CPL> nx[kRun], ng[kRun];
  auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
    load_tokens(ng, tile_rows<kTile>(g, tile, at.length, a.gate_token, C), g_lane,
                static_cast<unsigned>(a.gate_token) * sizeof(T));
    load_tokens(nx, tile_rows<kTile>(x, tile, at.length, a.input_token, C), x_lane,
                static_cast<unsigned>(a.input_token) * sizeof(T));
  };
  fetch(0);
  int buffer = 0;
  for (int64_t tile = 0; tile < a.tokens; tile += kTile, buffer ^= 1) {
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
    map.bound(keep);
    if (tile + kTile < a.tokens) fetch(tile + kTile);
    scan_runs<CPL, LANES, true>(map, before);
    float h[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) h[j] = carry[j];
    if (lane >= 64 - LANES) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        maps[buffer][wave][0][slot + j] = map.a[j];
        maps[buffer][wave][1][slot + j] = map.b[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        if (w == wave) h[j] = carry[j];
        carry[j] = fmaf(maps[buffer][w][0][slot + j], carry[j], maps[buffer][w][1][slot + j]);
      }
#pragma unroll
    for (int j = 0; j < CPL; ++j) h[j] = fmaf(before.a[j], h[j], before.b[j]);
    const int64_t first = tile + run_token;
    if (a.carries != nullptr && at.valid && first % kRecurrenceTile == 0 && first < a.tokens) {
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
    store_tokens<T, CPL>(tile_rows<kTile>(y, tile, a.tokens, C, C), y_lane,
                         static_cast<unsigned>(C) * sizeof(T), keep);
  }
  if (threadIdx.x >= LANES || !at.valid) return;
#pragma unroll
  for (int j = 0; j < CPL; ++j) a.last[at.batch * C + at.channel + j] = carry[j];
}

// The backward walks the tiles from the last. One channel a lane in 16 bits too: two take 200 registers,
// which leaves two waves a SIMD (8 x 4096 x 4096 fp16 320 us with two, 285 with one; 64 x 512 x 4096 bf16
// 322 and 278; 13 x 777 x 300 fp16 23 and 17).
template <typename T, int LANES, int NW>
__global__ __launch_bounds__(64 * NW) void recurrence_backward(RecurrenceArgs a) {
  constexpr int CPL = 1;
  constexpr int kTile = NW * (64 / LANES) * kRun;
  __shared__ float maps[2][NW][3][LANES * CPL];
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
#pragma unroll
  for (int j = 0; j < CPL; ++j)
    carry[j] = a.grad_last != nullptr ? a.grad_last[at.batch * C + at.channel + j] : 0.f;
  Run<T, CPL> nx[kRun], ng[kRun], nd[kRun];
  float nh[CPL];  // the state before the tile
  auto fetch = [&](int64_t tile) __attribute__((always_inline)) {
    load_tokens(ng, tile_rows<kTile>(g, tile, at.length, a.gate_token, C), g_lane,
                static_cast<unsigned>(a.gate_token) * sizeof(T));
    load_tokens(nd, tile_rows<kTile>(dy, tile, at.length, a.grad_token, C), d_lane,
                static_cast<unsigned>(a.grad_token) * sizeof(T));
    load_tokens(nx, tile_rows<kTile>(x, tile, at.length, a.input_token, C), x_lane,
                static_cast<unsigned>(a.input_token) * sizeof(T));
    const float* c = a.carries + (at.batch * tiles + tile / kRecurrenceTile) * C + at.channel;
#pragma unroll
    for (int j = 0; j < CPL; ++j) nh[j] = c[j];
  };
  int64_t tile = (a.tokens - 1) / kTile * kTile;
  if (a.tokens > 0) fetch(tile);
  int buffer = 0;
  for (; a.tokens > 0 && tile >= 0; tile -= kTile, buffer ^= 1) {
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
    for (int j = 0; j < CPL; ++j) h[j] = nh[j];
#pragma unroll
    for (int i = 0; i < kRun; ++i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
        keep[i][j] = q.keep;
        states.a[j] *= q.keep;
        take[i][j] = q.take;
        states.b[j] = fmaf(q.keep, states.b[j], q.take * static_cast<float>(nx[i].v[j]));
      }
    states.bound(keep);
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < CPL; ++j) grads.b[j] = keep[i][j] * (static_cast<float>(nd[i].v[j]) + grads.b[j]);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      cd[i] = nd[i];
      cx[i] = nx[i];
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) grads.a[j] = states.a[j];
    if (tile > 0) fetch(tile - kTile);
    scan_runs<CPL, LANES, false>(grads, grads_before);
    scan_runs<CPL, LANES, true>(states, states_before);
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
      if (lane >= 64 - LANES) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) maps[buffer][wave][2][slot + j] = states.b[j];
      }
      __syncthreads();
#pragma unroll
      for (int w = NW - 1; w >= 0; --w)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          if (w == wave) e[j] = carry[j];
          carry[j] = fmaf(maps[buffer][w][0][slot + j], carry[j], maps[buffer][w][1][slot + j]);
        }
#pragma unroll
      for (int w = 0; w < NW - 1; ++w)
#pragma unroll
        for (int j = 0; j < CPL; ++j)
          if (w < wave)
            h[j] = fmaf(maps[buffer][w][0][slot + j], h[j], maps[buffer][w][2][slot + j]);
    } else {
      static_assert(NW > 1 || LANES == 64, "a single wave takes one run");
#pragma unroll
      for (int j = 0; j < CPL; ++j) carry[j] = fmaf(grads.a[j], carry[j], grads.b[j]);
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      h[j] = fmaf(states_before.a[j], h[j], states_before.b[j]);
      e[j] = fmaf(grads_before.a[j], e[j], grads_before.b[j]);
    }
    // slope is (h_before - x) a (1 - a), then dgate; take becomes dx.
    float slope[kRun][CPL];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const float xi = static_cast<float>(cx[i].v[j]);
        slope[i][j] = (h[j] - xi) * (keep[i][j] * take[i][j]);
        h[j] = fmaf(keep[i][j], h[j], take[i][j] * xi);
      }
    }
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
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
    store_tokens<T, CPL>(tile_rows<kTile>(dx, tile, a.tokens, C, C), out_lane, step, take);
    store_tokens<T, CPL>(tile_rows<kTile>(dg, tile, a.tokens, C, C), out_lane, step, slope);
  }
  if (threadIdx.x >= LANES || !at.valid) return;
  if (a.grad_first != nullptr) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) a.grad_first[at.batch * C + at.channel + j] = carry[j];
  }
}

// ---- few sequences and channels: chunks of the token axis in one pass ------------------------------
//
// A workgroup takes a chunk of a strip's tokens, holds it in registers, leaves the chunk's map (A, B) in
// the workspace, composes the maps of the chunks before it in its group of kGroup with the state at
// the group's start, and finishes its tokens. The group's last chunk leaves the next group's state.
// So the inputs are read once, and what runs along the token axis is one hand-over a group, while
// many groups' chunks load and store. The maps are always composed in token order: the result does
// not depend on who came first.
//
// Every wait ends: a workgroup takes its chunk from a counter when it starts, chunks of earlier
// tokens first, so all that it waits for belongs to workgroups that have started, and those wait only
// for earlier ones still (a map is left before any wait). Should a word not come all the same, a
// wait gives up after kPatience looks and the state becomes NaN.
//
// A map or state is one 8-byte word, written and read whole by relaxed device-scope atomics, which
// pass the caches of the eight XCDs; it needs no order to anything else. Words are complemented:
// zero, to which a small kernel sets the workspace, is "not there yet", and the one value that would
// come out as zero (two NaNs of all ones) is replaced by another pair of NaNs.

constexpr int kGroup = 32;       // chunks of a group
constexpr int kPatience = 1 << 20;
// Tokens of a wave's run, times the channels of a lane.
constexpr int kForwardRun = 32, kBackwardRun = 16;

using Word = unsigned long long;

__device__ __forceinline__ void leave_word(Word* at, float a, float b) {
  Word w = (static_cast<Word>(__builtin_bit_cast(unsigned, b)) << 32) | __builtin_bit_cast(unsigned, a);
  w = w == ~Word{0} ? ~Word{1} : w;
  __hip_atomic_store(at, ~w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// CPL words of a lane, once all lanes of the wave have theirs.
template <int CPL>
__device__ __forceinline__ void await_words(const Word* at, float (&a)[CPL], float (&b)[CPL]) {
  Word w[CPL];
  for (int look = 0;; ++look) {
    bool there = true;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      w[j] = __hip_atomic_load(at + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      there = there && w[j] != 0;
    }
    if (__all(there) || look == kPatience) break;
    __builtin_amdgcn_s_sleep(2);
  }
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    const Word v = ~w[j];  // of a word that never came: NaN, NaN
    a[j] = __builtin_bit_cast(float, static_cast<unsigned>(v));
    b[j] = __builtin_bit_cast(float, static_cast<unsigned>(v >> 32));
  }
}

// Words of the workspace: the counter (the first of kChainHead), the groups' first states
// [rows][groups][64 CPL], the chunks' maps [rows][chunks][64 CPL]; a row is a strip of a sequence.
constexpr int64_t kChainHead = 8;

// What a ticket stands for: chunk `chunk` (counted in the direction of the walk) of a strip of a
// sequence.
template <int CPL, int kChunk>
struct ChainPlace {
  unsigned rows, chunks, groups, chunk, row, group, place;
  int64_t batch, length;
  int channel;  // the lane's first, or the last whole one past the edge
  bool valid;
  __device__ __forceinline__ ChainPlace(const RecurrenceArgs& a, unsigned ticket) {
    constexpr int kWide = 64 * CPL;
    const int C = static_cast<int>(a.channels);
    const unsigned strips = static_cast<unsigned>((C + kWide - 1) / kWide);
    rows = strips * static_cast<unsigned>(a.batch);
    chunks = static_cast<unsigned>((a.tokens + kChunk - 1) / kChunk);
    groups = (chunks + kGroup - 1) / kGroup;
    chunk = ticket / rows;
    row = ticket - chunk * rows;
    group = chunk / kGroup;
    place = chunk - group * kGroup;
    batch = row / strips;
    const int own = static_cast<int>(row % strips) * kWide + static_cast<int>(threadIdx.x & 63) * CPL;
    valid = own < C;
    channel = valid ? own : C - CPL;
    length = a.tokens;
    if (a.lengths != nullptr) {
      const int64_t n = a.wide_lengths ? static_cast<const int64_t*>(a.lengths)[batch]
                                       : static_cast<const int32_t*>(a.lengths)[batch];
      length = n < 0 ? 0 : (n < a.tokens ? n : a.tokens);
    }
  }
  __device__ __forceinline__ Word* states(Word* words) const {
    return words + kChainHead + static_cast<int64_t>(row) * groups * (64 * CPL);
  }
  __device__ __forceinline__ Word* left(Word* words) const {
    return words + kChainHead +
           (static_cast<int64_t>(rows) * groups + static_cast<int64_t>(row) * chunks) * (64 * CPL);
  }
};

template <typename T, int CPL, int N>
__global__ __launch_bounds__(64 * kWaves, 4) void recurrence_chain(RecurrenceArgs a) {
  constexpr int kChunk = kWaves * N, kWide = 64 * CPL;
  __shared__ float maps[kWaves][2][kWide];  // of the chunk's waves
  __shared__ float earlier[kGroup - 1][2][kWide];
  __shared__ float start[kWide];
  __shared__ unsigned taken;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = lane * CPL;
  const int64_t C = a.channels;
  Word* words = reinterpret_cast<Word*>(a.words);
  if (threadIdx.x == 0) taken = atomicAdd(reinterpret_cast<unsigned*>(words), 1u);
  __syncthreads();
  const ChainPlace<CPL, kChunk> at(a, __builtin_amdgcn_readfirstlane(taken));
  Word* states = at.states(words) + slot;
  Word* left = at.left(words) + slot;
  const int64_t tile = static_cast<int64_t>(at.chunk) * kChunk;
  const int run_token = wave * N;
  const T* x = static_cast<const T*>(a.input) + at.batch * a.input_batch;
  const T* g = static_cast<const T*>(a.gate) + at.batch * a.gate_batch;
  T* y = static_cast<T*>(a.output) + at.batch * a.tokens * C;
  Run<T, CPL> nx[N], ng[N];
  load_tokens(ng, tile_rows<kChunk>(g, tile, at.length, a.gate_token, C),
              lane_offset<T>(run_token, a.gate_token, at.channel),
              static_cast<unsigned>(a.gate_token) * sizeof(T));
  load_tokens(nx, tile_rows<kChunk>(x, tile, at.length, a.input_token, C),
              lane_offset<T>(run_token, a.input_token, at.channel),
              static_cast<unsigned>(a.input_token) * sizeof(T));
  const bool cut = tile + kChunk > at.length;
  const int live = tokens_before<N>(tile, run_token, at.length);
  if (cut) fill_tokens(ng, live, __builtin_inff());
  float keep[N][CPL], add[N][CPL];
  Map<CPL> map;
  map.clear();
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
      keep[i][j] = q.keep;
      add[i][j] = q.take * static_cast<float>(nx[i].v[j]);
      map.a[j] *= q.keep;
      map.b[j] = fmaf(q.keep, map.b[j], add[i][j]);
    }
  // Else the two are interleaved, which takes 128 registers and spills (108 without; 4 x 16384 x 1024
  // bf16 129 us).
  __builtin_amdgcn_sched_barrier(0);
  map.bound(keep);
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    maps[wave][0][slot + j] = map.a[j];
    maps[wave][1][slot + j] = map.b[j];
  }
  __syncthreads();
  const bool last_of_group = at.place == kGroup - 1 || at.chunk + 1 == at.chunks;
  if (wave == 0 && !last_of_group) {
    Map<CPL> whole;
    whole.clear();
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const float aw = maps[w][0][slot + j];
        whole.b[j] = fmaf(aw, whole.b[j], maps[w][1][slot + j]);
        whole.a[j] = join_gates(whole.a[j], aw);
      }
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      leave_word(left + static_cast<int64_t>(at.chunk) * kWide + j, whole.a[j], whole.b[j]);
  }
  for (unsigned e = wave; e < at.place; e += kWaves) {
    float wa[CPL], wb[CPL];
    await_words<CPL>(left + static_cast<int64_t>(at.group * kGroup + e) * kWide, wa, wb);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      earlier[e][0][slot + j] = wa[j];
      earlier[e][1][slot + j] = wb[j];
    }
  }
  if (wave == kWaves - 1) {
    float unused[CPL], h0[CPL];
    if (at.group == 0) {
#pragma unroll
      for (int j = 0; j < CPL; ++j)
        h0[j] = a.first != nullptr ? a.first[at.batch * C + at.channel + j] : 0.f;
    } else {
      await_words<CPL>(states + static_cast<int64_t>(at.group) * kWide, unused, h0);
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) start[slot + j] = h0[j];
  }
  __syncthreads();
  float h[CPL];
#pragma unroll
  for (int j = 0; j < CPL; ++j) h[j] = start[slot + j];
  for (unsigned e = 0; e < at.place; ++e)
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      h[j] = fmaf(earlier[e][0][slot + j], h[j], earlier[e][1][slot + j]);
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      if (w < wave) h[j] = fmaf(maps[w][0][slot + j], h[j], maps[w][1][slot + j]);
  if (wave == kWaves - 1 && last_of_group) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const float after = fmaf(map.a[j], h[j], map.b[j]);
      if (at.chunk + 1 < at.chunks)
        leave_word(states + static_cast<int64_t>(at.group + 1) * kWide + j, 0.f, after);
      else if (at.valid)
        a.last[at.batch * C + at.channel + j] = after;
    }
  }
  const int64_t first = tile + run_token;
  if (a.carries != nullptr && at.valid && first % kRecurrenceTile == 0 && first < a.tokens) {
    const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
    float* c = a.carries + (at.batch * tiles + first / kRecurrenceTile) * C + at.channel;
#pragma unroll
    for (int j = 0; j < CPL; ++j) c[j] = h[j];
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      h[j] = fmaf(keep[i][j], h[j], add[i][j]);
      keep[i][j] = h[j];
    }
  if (cut) clear_tokens(keep, live);
  store_tokens<T, CPL>(tile_rows<kChunk>(y, tile, a.tokens, C, C),
               at.valid ? lane_offset<T>(run_token, C, at.channel) : kNowhere,
               static_cast<unsigned>(C) * sizeof(T), keep);
}

// The backward's chunks, from the last token to the first: maps and words are those of E.
template <typename T, int CPL, int N>
__global__ __launch_bounds__(64 * kWaves) void recurrence_chain_backward(RecurrenceArgs a) {
  constexpr int kChunk = kWaves * N, kWide = 64 * CPL;
  __shared__ float maps[kWaves][3][kWide];  // A, R (of E) and F (of the state) of the waves
  __shared__ float later[kGroup - 1][2][kWide];
  __shared__ float start[kWide];
  __shared__ unsigned taken;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t C = a.channels;
  Word* words = reinterpret_cast<Word*>(a.words);
  if (threadIdx.x == 0) taken = atomicAdd(reinterpret_cast<unsigned*>(words), 1u);
  __syncthreads();
  const ChainPlace<CPL, kChunk> at(a, __builtin_amdgcn_readfirstlane(taken));
  const int slot = lane * CPL;
  Word* states = at.states(words) + slot;
  Word* left = at.left(words) + slot;
  const int64_t tile = static_cast<int64_t>(at.chunks - 1 - at.chunk) * kChunk;
  const int run_token = wave * N;
  const T* x = static_cast<const T*>(a.input) + at.batch * a.input_batch;
  const T* g = static_cast<const T*>(a.gate) + at.batch * a.gate_batch;
  const T* dy = static_cast<const T*>(a.grad_output) + at.batch * a.grad_batch;
  Run<T, CPL> nx[N], ng[N], nd[N];
  load_tokens(ng, tile_rows<kChunk>(g, tile, at.length, a.gate_token, C),
              lane_offset<T>(run_token, a.gate_token, at.channel),
              static_cast<unsigned>(a.gate_token) * sizeof(T));
  load_tokens(nd, tile_rows<kChunk>(dy, tile, at.length, a.grad_token, C),
              lane_offset<T>(run_token, a.grad_token, at.channel),
              static_cast<unsigned>(a.grad_token) * sizeof(T));
  load_tokens(nx, tile_rows<kChunk>(x, tile, at.length, a.input_token, C),
              lane_offset<T>(run_token, a.input_token, at.channel),
              static_cast<unsigned>(a.input_token) * sizeof(T));
  const int64_t tiles = (a.tokens + kRecurrenceTile - 1) / kRecurrenceTile;
  float h[CPL], e[CPL];
#pragma unroll
  for (int j = 0; j < CPL; ++j)
    h[j] = a.carries[(at.batch * tiles + tile / kRecurrenceTile) * C + at.channel + j];
  const bool cut = tile + kChunk > at.length;
  const int live = tokens_before<N>(tile, run_token, at.length);
  if (cut) fill_tokens(ng, live, __builtin_inff());
  Map<CPL> map;
  float state[CPL];
  map.clear();
#pragma unroll
  for (int j = 0; j < CPL; ++j) state[j] = 0.f;
  float keep[N][CPL], take[N][CPL];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const Gate q = open_gate(static_cast<float>(ng[i].v[j]));
      keep[i][j] = q.keep;
      take[i][j] = q.take;
      map.a[j] *= q.keep;
      state[j] = fmaf(q.keep, state[j], q.take * static_cast<float>(nx[i].v[j]));
    }
  map.bound(keep);
#pragma unroll
  for (int i = N - 1; i >= 0; --i)
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      map.b[j] = keep[i][j] * (static_cast<float>(nd[i].v[j]) + map.b[j]);
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    maps[wave][0][slot + j] = map.a[j];
    maps[wave][1][slot + j] = map.b[j];
    maps[wave][2][slot + j] = state[j];
  }
  __syncthreads();
  const bool last_of_group = at.place == kGroup - 1 || at.chunk + 1 == at.chunks;
  if (wave == 0 && !last_of_group) {
    Map<CPL> whole;
    whole.clear();
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w)
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const float aw = maps[w][0][slot + j];
        whole.b[j] = fmaf(aw, whole.b[j], maps[w][1][slot + j]);
        whole.a[j] = join_gates(whole.a[j], aw);
      }
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      leave_word(left + static_cast<int64_t>(at.chunk) * kWide + j, whole.a[j], whole.b[j]);
  }
  for (unsigned c = wave; c < at.place; c += kWaves) {
    float wa[CPL], wb[CPL];
    await_words<CPL>(left + static_cast<int64_t>(at.group * kGroup + c) * kWide, wa, wb);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      later[c][0][slot + j] = wa[j];
      later[c][1][slot + j] = wb[j];
    }
  }
  if (wave == kWaves - 1) {
    float unused[CPL], e0[CPL];
    if (at.group == 0) {
#pragma unroll
      for (int j = 0; j < CPL; ++j)
        e0[j] = a.grad_last != nullptr ? a.grad_last[at.batch * C + at.channel + j] : 0.f;
    } else {
      await_words<CPL>(states + static_cast<int64_t>(at.group) * kWide, unused, e0);
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) start[slot + j] = e0[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < CPL; ++j) e[j] = start[slot + j];
  for (unsigned c = 0; c < at.place; ++c)
#pragma unroll
    for (int j = 0; j < CPL; ++j) e[j] = fmaf(later[c][0][slot + j], e[j], later[c][1][slot + j]);
#pragma unroll
  for (int w = kWaves - 1; w > 0; --w)
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      if (w > wave) e[j] = fmaf(maps[w][0][slot + j], e[j], maps[w][1][slot + j]);
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      if (w < wave) h[j] = fmaf(maps[w][0][slot + j], h[j], maps[w][2][slot + j]);
  if (wave == 0 && last_of_group) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const float before = fmaf(map.a[j], e[j], map.b[j]);
      if (at.chunk + 1 < at.chunks)
        leave_word(states + static_cast<int64_t>(at.group + 1) * kWide + j, 0.f, before);
      else if (at.valid && a.grad_first != nullptr)
        a.grad_first[at.batch * C + at.channel + j] = before;
    }
  }
  // slope is (h_before - x) a (1 - a), then dgate; take becomes dx.
  float slope[N][CPL];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    hold(nx[i]);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const float xi = static_cast<float>(nx[i].v[j]);
      slope[i][j] = (h[j] - xi) * (keep[i][j] * take[i][j]);
      h[j] = fmaf(keep[i][j], h[j], take[i][j] * xi);
    }
  }
#pragma unroll
  for (int i = N - 1; i >= 0; --i) {
    hold(nd[i]);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const float d = static_cast<float>(nd[i].v[j]) + e[j];
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
  const unsigned out = at.valid ? lane_offset<T>(run_token, C, at.channel) : kNowhere;
  T* dx = static_cast<T*>(a.grad_input) + at.batch * a.tokens * C;
  T* dg = static_cast<T*>(a.grad_gate) + at.batch * a.tokens * C;
  store_tokens<T, CPL>(tile_rows<kChunk>(dx, tile, a.tokens, C, C), out, step, take);
  store_tokens<T, CPL>(tile_rows<kChunk>(dg, tile, a.tokens, C, C), out, step, slope);
}

__global__ __launch_bounds__(256) void clear_words(Word* words, int64_t count) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count;
       i += static_cast<int64_t>(gridDim.x) * 256)
    words[i] = 0;
}

template <typename T, int CPL>
hipError_t launch_chain(const RecurrenceArgs& a, bool backward, const RecurrencePlan& p,
                        hipStream_t stream) {
  constexpr int kForward = kForwardRun / CPL, kBackward = kBackwardRun / CPL;
  const dim3 grid(static_cast<unsigned>(p.workgroups)), block(static_cast<unsigned>(p.threads));
  const int64_t count = a.word_count;
  hipLaunchKernelGGL(clear_words,
                     dim3(static_cast<unsigned>(std::min<int64_t>((count + 255) / 256, 2048))),
                     dim3(256), 0, stream, reinterpret_cast<Word*>(a.words), count);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (backward)
    hipLaunchKernelGGL((recurrence_chain_backward<T, CPL, kBackward>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((recurrence_chain<T, CPL, kForward>), grid, block, 0, stream, a);
  return hipGetLastError();
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

template <typename T, int CPL, int LANES>
void launch_whole(const RecurrenceArgs& a, bool backward, const RecurrencePlan& p,
                  hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.workgroups)), block(static_cast<unsigned>(p.threads));
  if constexpr (CPL == 1) {
    if (backward) {
      hipLaunchKernelGGL((recurrence_backward<T, LANES, kWaves>), grid, block, 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((recurrence_forward<T, CPL, LANES>), grid, block, 0, stream, a);
}

template <typename T, int CPL>
hipError_t launch_channels(const RecurrenceArgs& a, bool backward, const RecurrencePlan& p,
                           hipStream_t stream) {
  if (p.chain) return launch_chain<T, CPL>(a, backward, p, stream);
  if (backward && CPL != 1) return hipErrorInvalidValue;  // no plan has it
  const dim3 grid(static_cast<unsigned>(p.workgroups)), block(static_cast<unsigned>(p.threads));
  if (p.waves == 1 && backward)
    hipLaunchKernelGGL((recurrence_backward<T, 64, 1>), grid, block, 0, stream, a);
  else if (p.waves == 1)
    hipLaunchKernelGGL((recurrence_step<T, CPL>), grid, block, 0, stream, a);
  else if (p.lanes == 64)
    launch_whole<T, CPL, 64>(a, backward, p, stream);
  else if (p.lanes == 32)
    launch_whole<T, CPL, 32>(a, backward, p, stream);
  else
    launch_whole<T, CPL, 16>(a, backward, p, stream);
  return hipGetLastError();
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

namespace {

// What a forward of 1024 tokens and more takes (us), in whole sequences at one workgroup or less a
// compute unit and in chunks of the token axis: a share of each 1024 tokens, which follow each other
// on 16, 32 or 64 lanes, and of each MB moved. Fitted to 87 sizes of 1024 to 4096 tokens and 32 to 256
// workgroups. What it takes is at most 8 % slower than the other there (7 x 1024 x 1024 bf16 whole 14.4 us, in
// chunks 19.4; 7 x 2048 x 1024 30.4 and 31.8; 7 x 4096 x 1024 58 and 51), at most 6 % in 44 sizes besides.
struct ForwardCost {
  float whole, tokens[3], bytes;
  float chain, chain_tokens, chain_bytes;
};
constexpr ForwardCost kOneChannel = {-0.9f, {6.4f, 7.1f, 12.0f}, 0.148f, 5.7f, 0.4f, 0.204f};
constexpr ForwardCost kTwoChannels = {1.0f, {9.6f, 15.8f, 26.6f}, 0.094f, 8.3f, 1.1f, 0.218f};

bool weigh_whole(convnd_hip_dtype dtype, const RecurrenceArgs& a, int channels_per_lane, int lanes) {
  const ForwardCost& c = channels_per_lane == 2 ? kTwoChannels : kOneChannel;
  const float thousands = static_cast<float>(a.tokens) / 1024.f;
  const float mb = static_cast<float>(a.batch) * static_cast<float>(a.tokens) *
                   static_cast<float>(a.channels) *
                   (dtype == CONVND_HIP_FLOAT32 ? 12e-6f : 6e-6f);
  const float turn = c.tokens[lanes == 16 ? 0 : lanes == 32 ? 1 : 2];
  return c.whole + turn * thousands + c.bytes * mb <
         c.chain + c.chain_tokens * thousands + c.chain_bytes * mb;
}

}  // namespace

RecurrencePlan plan_recurrence(convnd_hip_dtype dtype, const RecurrenceArgs& a, bool backward) {
  RecurrencePlan p{};
  p.waves = a.tokens <= kRun ? 1 : 8;
  // Two 16-bit channels a lane, where they fill more than half of a wave's lanes.
  p.channels_per_lane =
      dtype != CONVND_HIP_FLOAT32 && a.channels % 2 == 0 && a.channels > 64 ? 2 : 1;
  p.lanes = 64;
  const auto groups = [&](int lanes) {
    const int64_t wide = lanes * p.channels_per_lane;
    return std::max<int64_t>(1, a.batch) * ((a.channels + wide - 1) / wide);
  };
  // Whole sequences a workgroup where those fill the chip (8 x 4096 x 4096 fp16, 256 workgroups:
  // forward 163 us, in chunks 176) or are short (600 tokens of 256 channels, fp32: 7 us against 11); else
  // chunks of the token axis (forward / backward of 1 x 65536 x 512 fp32: 85 / 143 us, in splits with a
  // second reading of the inputs 130 / 180; 4 x 16384 x 1024 bf16: 97 / 174, whole sequences 202 / 404;
  // backward 8 x 2048 x 1024 51 and 77). The forward weighs the two: whole sequences on as few lanes as
  // leave a workgroup for each compute unit at most.
  if (a.tokens >= 1024 && groups(64) < 256) {
    int lanes = 16;
    while (lanes < 64 && groups(lanes) > 256) lanes *= 2;
    if (!backward && weigh_whole(dtype, a, p.channels_per_lane, lanes)) {
      p.lanes = lanes;
      p.tile = kWaves * (64 / lanes) * kRun;
      p.workgroups = groups(lanes);
      p.threads = 64 * kWaves;
      return p;
    }
    p.chain = true;
    const int64_t wide = 64 * p.channels_per_lane;
    p.tile = kWaves * (backward ? kBackwardRun : kForwardRun) / p.channels_per_lane;
    const int64_t chunks = (a.tokens + p.tile - 1) / p.tile;
    p.word_count = kChainHead + groups(64) * wide * (chunks + (chunks + kGroup - 1) / kGroup);
    p.workgroups = groups(64) * chunks;
    p.threads = 64 * kWaves;
    return p;
  }
  // The forward takes one channel a lane in 16 bits too where that makes workgroups for idle compute
  // units (13 x 777 x 300 fp16 14.3 us with two channels, 11.8 with one; 8 x 4096 x 4096, 256
  // workgroups of two, 164 and 154). Else two are loaded at half the cost (64 x 512 x 4096 bf16 154
  // and 173; 16 x 512 x 1024, 128 workgroups, 15 and 18).
  if (backward || groups(16) < 256 || (groups(64) >= 256 && groups(64) <= 512))
    p.channels_per_lane = 1;
  // The widest lanes that give every compute unit a workgroup, of those that one tile needs
  // (forward / backward of 4 x 4096 x 2048 fp32 at 32 lanes, 256 workgroups, 93 / 150 us, at 64
  // 102 / 151; 13 x 777 x 300 fp16 at 16 12 / 17, at 64 31 / 67).
  while (p.waves > 1 && p.lanes > 16 && a.tokens > int64_t{8} * (64 / p.lanes) * kRun &&
         groups(p.lanes) < 256)
    p.lanes /= 2;
  p.workgroups = groups(p.lanes);
  p.threads = 64 * p.waves;
  p.tile = p.waves * (64 / p.lanes) * kRun;
  if (p.waves == 1 && !backward) {  // the step kernel
    const int64_t each = (a.channels + p.channels_per_lane - 1) / p.channels_per_lane;
    p.workgroups = (each * a.batch + kStepThreads - 1) / kStepThreads;
    p.threads = kStepThreads;
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
