// Shared by the sequence kernels (layer norm, linear, gated recurrence): vector accesses of any
// alignment and reductions over the lanes of a wave.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "convnd_types.h"

namespace convnd {

// N elements at an address aligned to one element only. gfx950 runs in unaligned-access mode, so
// this is one wide load or store (16 bytes: dwordx4) whatever the row's alignment.
template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Run {
  T v[N];
};

template <int N, typename T>
__device__ __forceinline__ Run<T, N> load_run(const T* p) {
  return *reinterpret_cast<const Run<T, N>*>(p);
}
template <int N, typename T>
__device__ __forceinline__ void store_run(T* p, const Run<T, N>& r) {
  *reinterpret_cast<Run<T, N>*>(p) = r;
}
// Ends the element-by-element path of a row's end. Without it the compiler shares the last elements'
// accesses between that path and the whole run's and cuts the run's into pieces (three dwords and two
// elements: a linear layer's epilogue 74 -> 68 us at 8192 x 1024 -> 4096).
__device__ __forceinline__ void end_of_part() { asm volatile(""); }

template <int kControl>
__device__ __forceinline__ float dpp_read(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                       0, __builtin_bit_cast(int, v), kControl, 0xf, 0xf, true));
}

// Sum over aligned groups of N lanes (8, 16, 32 or 64); every lane gets its group's sum, added in
// the same order on every call. Up to 16 lanes the partner's value comes through DPP (quad
// permutations, then mirrors: the halves of a mirrored pair already hold equal sums).
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(N == 8 || N == 16 || N == 32 || N == 64, "group size");
  v += dpp_read<0xb1>(v);   // quad_perm 1,0,3,2
  v += dpp_read<0x4e>(v);   // quad_perm 2,3,0,1
  v += dpp_read<0x141>(v);  // row_half_mirror
  if constexpr (N >= 16) v += dpp_read<0x140>(v);  // row_mirror
  if constexpr (N >= 32) v += __shfl_xor(v, 16);
  if constexpr (N >= 64) v += __shfl_xor(v, 32);
  return v;
}

}  // namespace convnd
