// Shared by the sequence kernels (layer norm, linear, gated recurrence, delta rule): vector accesses of
// any alignment, reductions over the lanes of a wave, fragments of the matrix instructions, loads
// from memory straight into LDS, and LDS of more than 64 KB.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
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

typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr unsigned kNowhere = 0x80000000u;  // past every buffer (below 2^31 bytes)

// 16 bytes of a fragment: for 16-bit types 8 values of K for one MFMA, for float 4 for four.
template <typename T>
struct Fragment {
  static constexpr int kSteps = 1;
  using type = typename Mfma16<T>::frag;
  __device__ __forceinline__ static f32x4 mma(type a, type b, f32x4 c) {
    return Mfma16<T>::run(a, b, c);
  }
};
template <>
struct Fragment<float> {
  using type = f32x4;
  __device__ __forceinline__ static f32x4 mma(type a, type b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// 16 or 4 bytes per lane from the buffer straight into LDS: lane l writes dst + 16 l (4 l), dst the
// same for the whole wave. Inline assembly, so that the compiler does not take the LDS reads that
// follow, of other stages, to depend on them: whoever reads what they bring waits with wait_loads.
__device__ __forceinline__ void load_lds16(u32x4 rows, unsigned dst, unsigned offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst),
      "v"(offset), "s"(rows)
      : "m0");
}
__device__ __forceinline__ void load_lds4(u32x4 rows, unsigned dst, unsigned offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(dst),
               "v"(offset), "s"(rows)
               : "m0");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// More than 64 KB of LDS has to be asked for, once per device and kernel (`asked` is the kernel's).
template <typename Kernel>
inline hipError_t ask_lds(Kernel kernel, int bytes, std::atomic<uint64_t>& asked) {
  if (bytes <= 65536) return hipSuccess;
  int device = 0;
  hipError_t err = hipGetDevice(&device);
  if (err != hipSuccess) return err;
  const uint64_t bit = uint64_t{1} << (device & 63);
  if ((asked.load(std::memory_order_relaxed) & bit) != 0) return hipSuccess;
  err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == hipSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return err;
}

}  // namespace convnd
