// Layer norm over the last axis of [rows, channels], forward and backward.
//
//   mean = sum(x) / C, rstd = 1 / sqrt(sum((x - mean)^2) / C + eps), xh = (x - mean) rstd
//   y  = xh w + b
//   dx = rstd (w dy - mean(w dy) - xh mean(w dy xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by HBM: the forward reads x and writes y, the backward reads x and dy and writes dx. So a
// row is read once and stays in registers: TPR threads (a part of a wave, a wave, or a workgroup)
// hold NCH runs of 16 bytes each, the statistics are sums over those registers (the variance
// about the mean, a second pass that costs no traffic), and the next row's loads are in flight
// meanwhile. A thread keeps the same channels for all its rows, so w and b are read once and the
// backward's dw and db are summed in registers (fp32) over the rows of the workgroup; the
// workgroups' sums go to a [workgroups, channels] buffer that a second launch adds in a fixed order.
// Rows of more channels than 1024 threads hold run on kernels that read the row three times.

#include <algorithm>

#include "convnd_internal.h"
#include "convnd_sequence.h"

namespace convnd {
namespace {

// Threads of a workgroup: one row above a wave's width, else four waves of rows.
template <int TPR>
constexpr int norm_threads = TPR > 64 ? TPR : 256;

// Sum over the TPR threads of a row; `slot` alternates between calls so that one barrier each is
// enough (a slot is written again only after the barrier of the call between).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*scratch)[16], int slot) {
  if constexpr (TPR <= 64) {
    return lanes_sum<TPR>(v);
  } else {
    v = lanes_sum<64>(v);
    if ((threadIdx.x & 63) == 0) scratch[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) s += scratch[slot][i];
    return s;
  }
}

// Two sums at once, for the backward: slots turn and turn + 1, the other pair on the next call.
template <int TPR>
__device__ __forceinline__ void row_sums(float& u, float& v, float (*scratch)[16], int turn) {
  u = lanes_sum<(TPR > 64 ? 64 : TPR)>(u);
  v = lanes_sum<(TPR > 64 ? 64 : TPR)>(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) {
      scratch[turn][threadIdx.x >> 6] = u;
      scratch[turn + 1][threadIdx.x >> 6] = v;
    }
    __syncthreads();
    u = v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) {
      u += scratch[turn][i];
      v += scratch[turn + 1][i];
    }
  }
}

// One run of `kVec` channels from c0: whole, cut at the row's end, or past it (zeros).
template <int kVec, typename T>
__device__ __forceinline__ Run<T, kVec> load_part(const T* row, int c0, int channels) {
  if (c0 + kVec <= channels) return load_run<kVec>(row + c0);
  Run<T, kVec> r;
#pragma unroll
  for (int i = 0; i < kVec; ++i) r.v[i] = c0 + i < channels ? row[c0 + i] : static_cast<T>(0.f);
  return r;
}
template <int kVec, typename T>
__device__ __forceinline__ void store_part(T* row, int c0, int channels, const Run<T, kVec>& r) {
  if (c0 + kVec <= channels) {
    store_run<kVec>(row + c0, r);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (c0 + i < channels) row[c0 + i] = r.v[i];
  }
}

// T: type of x and y, W: type of the parameters.
template <typename T, typename W, int TPR, int NCH>
__global__ __launch_bounds__(norm_threads<TPR>) void norm_forward_rows(NormArgs a) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kRows = norm_threads<TPR> / TPR;
  __shared__ float scratch[2][16];
  const int C = static_cast<int>(a.channels);
  const int t = threadIdx.x % TPR;
  const T* x = static_cast<const T*>(a.input);
  T* y = static_cast<T*>(a.output);
  const W* weight = static_cast<const W*>(a.weight);
  const W* bias = static_cast<const W*>(a.bias);
  Run<W, kVec> w[NCH], b[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c0 = (k * TPR + t) * kVec;
    if (weight != nullptr) {
      w[k] = load_part<kVec>(weight, c0, C);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) w[k].v[i] = static_cast<W>(1.f);
    }
    if (bias != nullptr) {
      b[k] = load_part<kVec>(bias, c0, C);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) b[k].v[i] = static_cast<W>(0.f);
    }
  }
  const float inv = 1.f / static_cast<float>(C);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  Run<T, kVec> next[NCH];
  if (row < a.rows) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      next[k] = load_part<kVec>(x + row * a.input_stride, (k * TPR + t) * kVec, C);
  }
  for (; row < a.rows; row += step) {
    float v[NCH][kVec];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[k][i] = static_cast<float>(next[k].v[i]);
        s += v[k][i];
      }
    if (row + step < a.rows) {
#pragma unroll
      for (int k = 0; k < NCH; ++k)
        next[k] = load_part<kVec>(x + (row + step) * a.input_stride, (k * TPR + t) * kVec, C);
    }
    const float mean = row_sum<TPR>(s, scratch, 0) / static_cast<float>(C);  // constant rows: exact
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c0 = (k * TPR + t) * kVec;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[k][i] = c0 + i < C ? v[k][i] - mean : 0.f;
        q = fmaf(v[k][i], v[k][i], q);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(q, scratch, 1) * inv + a.eps);
    if (t == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    T* out = y + row * a.channels;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      Run<T, kVec> r;
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        r.v[i] = static_cast<T>(fmaf(v[k][i] * rstd, static_cast<float>(w[k].v[i]),
                                     static_cast<float>(b[k].v[i])));
      store_part<kVec>(out, (k * TPR + t) * kVec, C, r);
    }
  }
}

template <typename T, typename W, int TPR, int NCH>
__global__ __launch_bounds__(norm_threads<TPR>) void norm_backward_rows(NormArgs a) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kRows = norm_threads<TPR> / TPR;
  __shared__ float scratch[4][16];
  // The workgroup's row groups hand their dw and db sums over here (TPR <= 64).
  __shared__ float sums[TPR <= 64 ? kRows * TPR * NCH * kVec : 1];
  const int C = static_cast<int>(a.channels);
  const int t = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  const T* x = static_cast<const T*>(a.input);
  const T* dy = static_cast<const T*>(a.grad_output);
  T* dx = static_cast<T*>(a.grad_input);
  const W* weight = static_cast<const W*>(a.weight);
  Run<W, kVec> w[NCH];
  float gw[NCH][kVec], gb[NCH][kVec];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    if (weight != nullptr) {
      w[k] = load_part<kVec>(weight, (k * TPR + t) * kVec, C);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) w[k].v[i] = static_cast<W>(1.f);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) gw[k][i] = gb[k][i] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(C);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + group;
  Run<T, kVec> nx[NCH], ny[NCH];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t r) {
    nmean = a.mean[r];
    nrstd = a.rstd[r];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      nx[k] = load_part<kVec>(x + r * a.input_stride, (k * TPR + t) * kVec, C);
      ny[k] = load_part<kVec>(dy + r * a.grad_stride, (k * TPR + t) * kVec, C);
    }
  };
  if (row < a.rows) fetch(row);
  int turn = 0;
  for (; row < a.rows; row += step) {
    const float mean = nmean, rstd = nrstd;
    Run<T, kVec> cx[NCH], cy[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      cx[k] = nx[k];
      cy[k] = ny[k];
    }
    if (row + step < a.rows) fetch(row + step);
    // Past the row's end dy is zero, so those lanes add nothing to any sum.
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float g = static_cast<float>(cy[k].v[i]);
        const float h = (static_cast<float>(cx[k].v[i]) - mean) * rstd;
        const float wg = g * static_cast<float>(w[k].v[i]);
        s1 += wg;
        s2 = fmaf(wg, h, s2);
        gw[k][i] = fmaf(g, h, gw[k][i]);
        gb[k][i] += g;
      }
    if (dx == nullptr) continue;
    row_sums<TPR>(s1, s2, scratch, turn);
    turn ^= 2;
    const float c1 = s1 * inv, c2 = s2 * inv;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      Run<T, kVec> r;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float h = (static_cast<float>(cx[k].v[i]) - mean) * rstd;
        const float wg = static_cast<float>(cy[k].v[i]) * static_cast<float>(w[k].v[i]);
        r.v[i] = static_cast<T>(rstd * (wg - c1 - h * c2));
      }
      store_part<kVec>(dx + row * a.channels, (k * TPR + t) * kVec, C, r);
    }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.channels;
#pragma unroll
  for (int which = 0; which < 2; ++which, out += a.channels) {
    if constexpr (TPR > 64) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        Run<float, kVec> r;
#pragma unroll
        for (int i = 0; i < kVec; ++i) r.v[i] = which == 0 ? gw[k][i] : gb[k][i];
        store_part<kVec>(out, (k * TPR + t) * kVec, C, r);
      }
    } else {
      constexpr int kRow = TPR * NCH * kVec;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          sums[group * kRow + (k * TPR + t) * kVec + i] = which == 0 ? gw[k][i] : gb[k][i];
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += norm_threads<TPR>) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) s += sums[r * kRow + c];
        out[c] = s;
      }
    }
  }
}

// Rows too long for registers: a workgroup per row, three reads of it (the later ones from L2).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_forward_long(NormArgs a) {
  __shared__ float scratch[2][16];
  const W* weight = static_cast<const W*>(a.weight);
  const W* bias = static_cast<const W*>(a.bias);
  const float inv = 1.f / static_cast<float>(a.channels);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.input) + row * a.input_stride;
    T* y = static_cast<T*>(a.output) + row * a.channels;
    float s = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < a.channels; c += 1024) s += static_cast<float>(x[c]);
    const float mean = row_sum<1024>(s, scratch, 0) / static_cast<float>(a.channels);
    for (int64_t c = threadIdx.x; c < a.channels; c += 1024) {
      const float d = static_cast<float>(x[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(q, scratch, 1) * inv + a.eps);
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < a.channels; c += 1024) {
      const float w = weight != nullptr ? static_cast<float>(weight[c]) : 1.f;
      const float b = bias != nullptr ? static_cast<float>(bias[c]) : 0.f;
      y[c] = static_cast<T>(fmaf((static_cast<float>(x[c]) - mean) * rstd, w, b));
    }
  }
}

// Its input gradient, and the rows' share of dw and db in one row of `partial` per workgroup.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_backward_long(NormArgs a) {
  __shared__ float scratch[4][16];
  const W* weight = static_cast<const W*>(a.weight);
  const float inv = 1.f / static_cast<float>(a.channels);
  float* gw = a.partial != nullptr ? a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.channels
                                   : nullptr;
  bool begun = false;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.input) + row * a.input_stride;
    const T* dy = static_cast<const T*>(a.grad_output) + row * a.grad_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < a.channels; c += 1024) {
      const float g = static_cast<float>(dy[c]);
      const float h = (static_cast<float>(x[c]) - mean) * rstd;
      const float wg = weight != nullptr ? g * static_cast<float>(weight[c]) : g;
      s1 += wg;
      s2 = fmaf(wg, h, s2);
      if (gw != nullptr) {  // this thread's own channels only
        gw[c] = begun ? fmaf(g, h, gw[c]) : g * h;
        gw[a.channels + c] = begun ? gw[a.channels + c] + g : g;
      }
    }
    begun = true;
    if (a.grad_input == nullptr) continue;
    row_sums<1024>(s1, s2, scratch, turn);
    turn ^= 2;
    const float c1 = s1 * inv, c2 = s2 * inv;
    T* dx = static_cast<T*>(a.grad_input) + row * a.channels;
    for (int64_t c = threadIdx.x; c < a.channels; c += 1024) {
      const float h = (static_cast<float>(x[c]) - mean) * rstd;
      const float wg = static_cast<float>(dy[c]) *
                       (weight != nullptr ? static_cast<float>(weight[c]) : 1.f);
      dx[c] = static_cast<T>(rstd * (wg - c1 - h * c2));
    }
  }
}

// Up to two results (dw and db) from the workgroups' sums, rows of `pitch` floats: 32 channels a
// workgroup, its 32 groups of 32 lanes add every 32nd row, then the groups' sums are added in order.
constexpr int kReduceChannels = 32, kReduceGroups = 32;
template <typename W>
__global__ __launch_bounds__(kReduceChannels* kReduceGroups) void sum_rows(
    const float* __restrict__ partial, int64_t rows, int64_t pitch, int64_t channels, W* dw, W* db) {
  __shared__ float sums[kReduceGroups][kReduceChannels + 1];
  const int lane = threadIdx.x % kReduceChannels, group = threadIdx.x / kReduceChannels;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kReduceChannels + lane;
  W* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;  // the same for the whole workgroup
  float s = 0.f;
  if (c < channels) {
    const float* p = partial + blockIdx.y * channels + c;
#pragma unroll 8
    for (int64_t r = group; r < rows; r += kReduceGroups) s += p[r * pitch];
  }
  sums[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < channels) {
    float total = 0.f;
#pragma unroll
    for (int g = 0; g < kReduceGroups; ++g) total += sums[g][lane];
    out[c] = static_cast<W>(total);
  }
}

template <typename T, typename W, int TPR, int NCH>
hipError_t launch_rows(const NormArgs& a, bool backward, int64_t blocks, hipStream_t stream) {
  if (backward)
    hipLaunchKernelGGL((norm_backward_rows<T, W, TPR, NCH>), dim3(blocks),
                       dim3(norm_threads<TPR>), 0, stream, a);
  else
    hipLaunchKernelGGL((norm_forward_rows<T, W, TPR, NCH>), dim3(blocks), dim3(norm_threads<TPR>),
                       0, stream, a);
  return hipGetLastError();
}

template <typename T, typename W>
hipError_t launch_norm_typed(const NormArgs& a, bool backward, const NormPlan& p,
                             hipStream_t stream) {
  if (p.threads_per_row == 0) {
    if (backward)
      hipLaunchKernelGGL((norm_backward_long<T, W>), dim3(p.blocks), dim3(1024), 0, stream, a);
    else
      hipLaunchKernelGGL((norm_forward_long<T, W>), dim3(p.blocks), dim3(1024), 0, stream, a);
    return hipGetLastError();
  }
  switch (p.threads_per_row * 16 + p.runs) {
    case 8 * 16 + 1: return launch_rows<T, W, 8, 1>(a, backward, p.blocks, stream);
    case 16 * 16 + 1: return launch_rows<T, W, 16, 1>(a, backward, p.blocks, stream);
    case 32 * 16 + 1: return launch_rows<T, W, 32, 1>(a, backward, p.blocks, stream);
    case 64 * 16 + 1: return launch_rows<T, W, 64, 1>(a, backward, p.blocks, stream);
    case 128 * 16 + 1: return launch_rows<T, W, 128, 1>(a, backward, p.blocks, stream);
    case 256 * 16 + 1: return launch_rows<T, W, 256, 1>(a, backward, p.blocks, stream);
    case 512 * 16 + 1: return launch_rows<T, W, 512, 1>(a, backward, p.blocks, stream);
    case 1024 * 16 + 1: return launch_rows<T, W, 1024, 1>(a, backward, p.blocks, stream);
    case 1024 * 16 + 2: return launch_rows<T, W, 1024, 2>(a, backward, p.blocks, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

NormPlan plan_norm(int64_t rows, int64_t channels, int element_size, bool backward) {
  const int64_t runs = (channels + 16 / element_size - 1) / (16 / element_size);
  NormPlan p{};
  // One run a thread: the backward's sums and next row are many registers, and a row over more
  // waves beats more runs a thread (65536 x 2048 fp16: forward 133 / backward 379 us with 64
  // threads of four runs, 110 / 227 with 128 of two, 99 / 179 with 256 of one).
  if (runs <= 1024) {
    p.threads_per_row = 8, p.runs = 1;
    while (p.threads_per_row < runs) p.threads_per_row *= 2;
  } else if (runs <= 2048) {
    p.threads_per_row = 1024, p.runs = 2;
  }
  const int threads = p.threads_per_row == 0 ? 1024 : (p.threads_per_row > 64 ? p.threads_per_row : 256);
  const int per_block = p.threads_per_row == 0 ? 1 : threads / std::min(threads, p.threads_per_row);
  const int64_t needed = (rows + per_block - 1) / per_block;
  // The forward fills the chip with rows in flight (32 waves a compute unit: 99 us above, 131 with
  // 16). Every workgroup of the backward leaves a row of sums to be added up, so there are as many as
  // run side by side (20 waves a compute unit by their registers, 16 in workgroups of 8 or 16 waves;
  // 65536 x 2048 fp16: 162 us with these 1280, 179 with 1024, 188 with 2048; 16384 x 4096 bf16: 95
  // with these 512, 118 with 768), and several rows each (5003 x 769 fp32: 17 us with 768, 23 with 2560).
  if (backward) {
    const int64_t resident = 256 * (threads > 256 ? 16 : 20) * 64 / threads;
    p.blocks = std::min(needed, std::min(resident, std::max<int64_t>(256, rows / 8)));
  } else {
    p.blocks = std::min<int64_t>(needed, 524288 / threads);
  }
  return p;
}

hipError_t launch_norm(convnd_hip_dtype dtype, bool float_params, const NormArgs& a, bool backward,
                       const NormPlan& p, hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return launch_norm_typed<float, float>(a, backward, p, stream);
    case CONVND_HIP_FLOAT16:
      return float_params ? launch_norm_typed<_Float16, float>(a, backward, p, stream)
                          : launch_norm_typed<_Float16, _Float16>(a, backward, p, stream);
    case CONVND_HIP_BFLOAT16:
      return float_params ? launch_norm_typed<__bf16, float>(a, backward, p, stream)
                          : launch_norm_typed<__bf16, __bf16>(a, backward, p, stream);
    default:
      return hipErrorInvalidValue;
  }
}

hipError_t launch_sum_rows(convnd_hip_dtype param_dtype, const float* partial, int64_t rows,
                           int64_t pitch, int64_t channels, void* dw, void* db,
                           hipStream_t stream) {
  const dim3 grid((channels + kReduceChannels - 1) / kReduceChannels, pitch > channels ? 2 : 1);
  const dim3 block(kReduceChannels * kReduceGroups);
  switch (param_dtype) {
    case CONVND_HIP_FLOAT32:
      hipLaunchKernelGGL(sum_rows<float>, grid, block, 0, stream, partial, rows, pitch, channels,
                         static_cast<float*>(dw), static_cast<float*>(db));
      break;
    case CONVND_HIP_FLOAT16:
      hipLaunchKernelGGL(sum_rows<_Float16>, grid, block, 0, stream, partial, rows, pitch, channels,
                         static_cast<_Float16*>(dw), static_cast<_Float16*>(db));
      break;
    case CONVND_HIP_BFLOAT16:
      hipLaunchKernelGGL(sum_rows<__bf16>, grid, block, 0, stream, partial, rows, pitch, channels,
                         static_cast<__bf16*>(dw), static_cast<__bf16*>(db));
      break;
    default:
      return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace convnd
