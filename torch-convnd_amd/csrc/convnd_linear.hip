// Linear layer, y = act(x W^T + b) + r, and its backward pass: products on the matrix cores.
//
//   z = x W^T + b, y = act(z) + r
//   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum_rows dz (dr = dy needs no work)
//
// A product C[m][n] = sum_k A[m][k] B[n][k] takes each operand as it lies in memory: with K
// contiguous ("inner": x and W in the forward, dz for dx) or with K as the row index ("outer": W for
// dx, dz and x for dW). 16-bit types multiply on the 16x16x32 MFMA, float on the 16x16x4 one, both
// from 16-byte fragments and with float sums.
//   * Many rows: workgroups take tiles of 256 x 256 (8 waves of 128 x 64: half the LDS reads a
//     product of 64 x 64), 128 x 128 or 64 x 64 (4 waves) as plan_product weighs them. Stages of 128
//     bytes of K go straight from memory to LDS, a whole stage ahead; their 16-byte chunks are
//     permuted so that fragment reads meet no bank twice. An outer operand is read with the
//     transposing LDS read. The barrier of a stage falls between its two halves, whose fragments are
//     then in registers.
//   * Few tiles and a long K: K is split over workgroups, their float sums go to the workspace and
//     are added in order by a second launch with the epilogue.
//   * Up to 64 rows (decoding), not too long: bound by reading W once. A workgroup takes 16 rows of W, its waves
//     take parts of K and read fragments from memory into registers, all in flight at once.
// The bounds of a tile are those of the buffers it reads through; 16-bit rows of odd length or stride
// are first copied to the workspace with padding.

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "convnd_internal.h"
#include "convnd_sequence.h"

namespace convnd {
namespace {

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

// One operand of the product: `extent` rows (its side of the result) by K. Inner: row-major with K
// contiguous; outer: K rows of `extent` contiguous values. Staged in LDS as it lies in memory, 128 bytes
// of K (inner) or rows of EXT values (outer), its 16-byte chunks permuted within a row. Rows start
// on 4 bytes, and one whose length is no whole 4 bytes is padded with a zero: the buffer's bounds are
// checked by 4 bytes.
template <typename T, bool OUTER, int EXT, int W>
struct Operand {
  static constexpr int kK = 128 / sizeof(T);             // K values of a stage
  static constexpr int kBytes = EXT * 128;               // of a stage
  static constexpr int kLoads = kBytes / 1024 / W;       // loads of a wave (1 KB each)
  static constexpr int kPitch = OUTER ? EXT * int(sizeof(T)) : 128;
  static constexpr int kChunks = kPitch / 16;            // of a row
  static constexpr int kVec = 16 / sizeof(T);
  static_assert(kLoads >= 1, "at least one load a wave");
  const char* base;      // of the workgroup's rows or columns, at the first K value of the next stage
  int64_t ld;            // bytes of a row
  unsigned before_last;  // inner: bytes of the workgroup's rows but the last
  unsigned row_bytes;    // outer: bytes of a row from base on
  unsigned offset[kLoads];

  __device__ __forceinline__ static int swizzle(int row) {
    if constexpr (!OUTER) return (row >> 1) & 7;
    // A transposing read takes 32 bytes of rows r .. r + 3 and r + 8 .. r + 11 at a time.
    if constexpr (sizeof(T) == 2 && EXT >= 128) return ((row & 3) | ((row >> 1) & 4)) << 1;
    if constexpr (sizeof(T) == 2) return (((row >> 1) & 1) | ((row >> 2) & 2)) << 1;
    return 0;
  }

  __device__ __forceinline__ static unsigned whole_words(unsigned bytes) {
    return (bytes + 3) & ~3u;
  }

  __device__ __forceinline__ void init(const void* p, int64_t ld_elements, int64_t extent,
                                       int64_t at, int64_t k0) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    ld = ld_elements * sizeof(T);
    base = static_cast<const char*>(p) + (OUTER ? k0 * ld + at * int64_t{sizeof(T)}
                                                : at * ld + k0 * int64_t{sizeof(T)});
    const int64_t rows = extent - at < EXT ? extent - at : EXT;
    before_last = static_cast<unsigned>((rows - 1) * ld);
    row_bytes = whole_words(static_cast<unsigned>((extent - at) * sizeof(T)));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int chunk = (i * W + wave) * 64 + lane;  // in the stage
      const int row = chunk / kChunks;
      offset[i] = static_cast<unsigned>(row) * static_cast<unsigned>(ld) +
                  ((chunk % kChunks) ^ swizzle(row)) * 16;
    }
  }

  // The stage's rows up to K value k as a buffer.
  __device__ __forceinline__ u32x4 rows(int k) const {
    const unsigned bytes = OUTER ? static_cast<unsigned>((k - 1) * ld) + row_bytes
                                 : before_last + whole_words(static_cast<unsigned>(k) * unsigned{sizeof(T)});
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(at));
    r[1] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(at >> 32) & 0xffffu);
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00020000u;
    return r;
  }
  __device__ __forceinline__ void advance() { base += OUTER ? kK * ld : 128; }

  // Load i (of kLoads) of a whole stage into LDS at `dst`.
  __device__ __forceinline__ void load(u32x4 r, unsigned dst, int wave, int i) const {
    load_lds16(r, dst + (i * W + wave) * 1024, offset[i]);
  }

  // Loads the last stage, of k <= kK values of K; zeros follow them. An inner row goes on in the next
  // one there: whole chunks past k are sent nowhere, and where k ends inside a chunk the loads are of
  // 4 bytes.
  __device__ __forceinline__ void load_last(unsigned dst, int wave, int k) const {
    const int lane = threadIdx.x & 63;
    const u32x4 r = rows(k);
    if (OUTER || k % kVec == 0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int chunk = (i * W + wave) * 64 + lane;
        const bool inside =
            OUTER || (((chunk % kChunks) ^ swizzle(chunk / kChunks)) * kVec) < k;
        load_lds16(r, dst + (i * W + wave) * 1024, inside ? offset[i] : kNowhere);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kLoads * 4; ++i) {
        const int part = (i / 4 * W + wave) * 4 + i % 4;  // of 256 bytes
        const int word = part * 64 + lane;
        const int row = word / 32;
        const int column = ((word % 32 / 4) ^ swizzle(row)) * 16 + word % 4 * 4;
        const unsigned at = static_cast<unsigned>(row) * static_cast<unsigned>(ld) + column;
        load_lds4(r, dst + part * 256, column < k * int{sizeof(T)} ? at : kNowhere);
      }
    }
  }
};

// Fragment reads of a wave: COUNT fragments of 16 rows (or columns) from `first` on.
template <typename T, bool OUTER, int EXT, int COUNT>
struct Reader {
  using frag = typename Fragment<T>::type;
  unsigned at[OUTER ? COUNT : 2];
  __device__ __forceinline__ void init(int first) {
    const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
    if constexpr (!OUTER) {
      // Row first + l (+ 16 per fragment: the swizzle repeats every 16 rows).
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        at[ks] = (first + l) * 128 + (((ks * 4 + g) ^ ((l >> 1) & 7)) << 4);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int n = 0; n < COUNT; ++n) {
        const int swizzle = EXT >= 128 ? (l >> 2) | ((g & 1) << 2) : (l >> 3) | ((g & 1) << 1);
        const int pair = (first / 16 + n) ^ swizzle;
        at[n] = (8 * g + (l >> 2)) * (EXT * 2) + pair * 32 + (l & 3) * 8;
      }
    } else {
#pragma unroll
      for (int n = 0; n < COUNT; ++n) at[n] = 4 * g * (EXT * 4) + (first + n * 16 + l) * 4;
    }
  }
  // Fragment n of half ks of the stage at `lds`.
  __device__ __forceinline__ frag read(const unsigned char* lds, int ks, int n) const {
    frag f;
    if constexpr (!OUTER) {
      f = *reinterpret_cast<const frag*>(lds + at[ks] + n * 2048);
    } else if constexpr (sizeof(T) == 2) {
      // Transposing reads: each gives the lane 4 K values of its column.
      using lds_vec = __attribute__((address_space(3))) s16x4*;
      const unsigned char* p = lds + at[n] + ks * 32 * (EXT * 2);
      union {
        s16x4 part[2];
        frag whole;
      } u;
      u.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec)(p));
      u.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec)(p + 4 * (EXT * 2)));
      f = u.whole;
    } else {
      const unsigned char* p = lds + at[n] + ks * 16 * (EXT * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float*>(p + i * (EXT * 4));
    }
    return f;
  }
};

// 0.5 erfc(|z| / sqrt 2) and exp(-z^2 / 2) for 16-bit results: Abramowitz and Stegun's formula
// 7.1.26, off by at most 0.75e-7, at a third of erff's instructions (13 us of 8192 x 1024 -> 4096).
// float results take erff.
struct Normal {
  float tail, gauss;
};
__device__ __forceinline__ Normal gauss_tail(float z) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, fabsf(z), 1.f));
  const float gauss = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
  float p = fmaf(0.5307027145f, t, -0.7265760135f);
  p = fmaf(p, t, 0.7107068705f);
  p = fmaf(p, t, -0.142248368f);
  p = fmaf(p, t, 0.127414796f);
  return {p * t * gauss, gauss};
}

// The normal distribution's Phi(z) (as `tail`: the part below z), and exp(-z^2 / 2).
template <typename T>
__device__ __forceinline__ Normal normal(float z) {
  if constexpr (sizeof(T) == 2) {
    const Normal q = gauss_tail(z);
    return {z < 0.f ? q.tail : 1.f - q.tail, q.gauss};
  } else {
    return {0.5f * (1.f + erff(z * 0.70710678118654752f)),
            __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z)};
  }
}

// Activates v; with SLOPE, d is the activation's slope at v (of an infinite v NaN, as the formulas).
// An epilogue of this size is bound by its instructions: each one an element less is 0.9 us of
// 8192 x 1024 -> 4096.
template <typename T, bool SLOPE>
__device__ __forceinline__ void activate_all(float (&v)[8], float (&d)[8], int act) {
  if (act == CONVND_HIP_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d[e] = v[e] > 0.f ? 1.f : 0.f;
      v[e] = v[e] < 0.f ? 0.f : v[e];  // NaN stays
    }
  } else if (act == CONVND_HIP_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const auto [phi, gauss] = normal<T>(v[e]);
      if constexpr (SLOPE) d[e] = fmaf(v[e] * 0.39894228040143268f, gauss, phi);
      v[e] *= phi;
    }
  } else if (act == CONVND_HIP_ACT_GELU_TANH) {
    // 0.5 z (1 + tanh u) = z s, s = 1 / (1 + exp(-2 u)), u = c z (1 + q z^2) with c = sqrt(2 / pi)
    // and q = 0.044715; its slope s + 2 z s (1 - s) c (1 + 3 q z^2). The bound on z^2 keeps its
    // products with a vanished s (1 - s) finite.
    constexpr float c = 0.79788456080286536f, q = 0.044715f, to_base_2 = -2.88539008177792681f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float z2 = fminf(v[e] * v[e], 1e30f);
      const float u = v[e] * fmaf(to_base_2 * c * q, z2, to_base_2 * c);
      const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u));
      if constexpr (SLOPE) d[e] = fmaf(v[e] * fmaf(-s, s, s), fmaf(6.f * c * q, z2, 2.f * c), s);
      v[e] *= s;
    }
  }
}

// What the backward pass needs of the activation is its slope, within -0.13 and 1.13. Beside 16-bit
// values it is kept in 16 bits of fixed point, 1 / 28672 a step (1 is on the grid; the lowest code
// is NaN): at most 1.8e-5 off, where the sum before the activation in bfloat16 moved gradients by
// half of their own rounding, and read by one multiplication (8192 x 4096 with GELU 40 -> 27 us). What
// that costs is in the tail: 3 to 5 % of GELU's slope at z = -4, and all of it below z = -4.81 (-4.60 in
// the tanh form), where it is within 1.75e-5 of zero.
template <typename T>
using Slope = std::conditional_t<sizeof(T) == 2, int16_t, float>;
template <typename T>
__device__ __forceinline__ Run<Slope<T>, 8> keep_slopes(const float (&d)[8]) {
  Run<Slope<T>, 8> r;
  if constexpr (sizeof(T) == 2) {
    typedef short Pair __attribute__((ext_vector_type(2)));
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      // Rounded products with 32767.
      constexpr float step = 28672.f / 32767.f;
      const Pair q = __builtin_bit_cast(
          Pair, __builtin_amdgcn_cvt_pknorm_i16(d[e] * step, d[e + 1] * step));
      r.v[e] = q[0];
      r.v[e + 1] = q[1];
      nan |= __builtin_isunordered(d[e], d[e + 1]);
    }
    if (nan)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d[e] != d[e]) r.v[e] = -32768;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = d[e];
  }
  return r;
}
__device__ __forceinline__ float slope_of(int16_t q) {
  return q == -32768 ? __builtin_nanf("") : static_cast<float>(q) * (1.f / 28672.f);
}
__device__ __forceinline__ float slope_of(float d) { return d; }

// 16 bytes stored past the caches' order of use, for what is not read before much else is.
template <typename T>
__device__ __forceinline__ void stream_run(T* p, const Run<T, 8>& r) {
  static_assert(sizeof(T) == 2, "8 values of 16 bits");
  typedef unsigned Words __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(__builtin_bit_cast(Words, r), reinterpret_cast<Words*>(p));
}

// Outputs of this size and more are streamed past the caches: their reader finds little of them there
// either way. Training steps of three blocks (layer norm and two layers) in bfloat16 with outputs of
// 32 MB (4096 x 1024 -> 4096 -> 1024) 926 us plain and 980 streamed, of 64 MB (8192 rows) 1539 and
// 1567, (16384 x 2048 -> 2048) 2810 and 2762, of 128 MB (16384 x 1024 -> 4096) 2884 and 2799.
constexpr int64_t kStreamBytes = int64_t{96} << 20;

// Up to 8 neighbouring sums of row m from column n on: the partial sums of a split as they are, else
// bias, activation and residual in float and one rounding (and the activation's slope, where the
// backward pass is to have it).
template <typename T>
__device__ __forceinline__ void finish(const LinearArgs& a, float (&v)[8], const float (&bias)[8],
                                       int64_t split, int64_t m, int64_t n, int count) {
  const int64_t at = m * a.n + n;
  if (a.partial != nullptr) {
    float* p = a.partial + split * a.m * a.n + at;
    if (count == 8) {
      Run<float, 4> r[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e / 4].v[e % 4] = v[e];
      store_run<4>(p, r[0]);
      store_run<4>(p + 4, r[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) p[e] = v[e];
      end_of_part();
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += bias[e];
  T* out = static_cast<T*>(a.output) + at;
  float d[8];
  if (a.slope != nullptr) {
    activate_all<T, true>(v, d, a.activation);
    const Run<Slope<T>, 8> kept = keep_slopes<T>(d);
    Slope<T>* slope = static_cast<Slope<T>*>(a.slope) + at;
    if (count == 8) {
      // Read by the backward pass, long after.
      if constexpr (sizeof(T) == 2)
        stream_run(slope, kept);
      else
        store_run<8>(slope, kept);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) slope[e] = kept.v[e];
      end_of_part();
    }
  } else {
    activate_all<T, false>(v, d, a.activation);
  }
  if (a.residual != nullptr) {
    const T* residual = static_cast<const T*>(a.residual) + m * a.residual_stride + n;
    if (count == 8) {
      const Run<T, 8> r = load_run<8>(residual);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += static_cast<float>(r.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) v[e] += static_cast<float>(residual[e]);
      end_of_part();
    }
  }
  Run<T, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y.v[e] = static_cast<T>(v[e]);
  if (count == 8) {
    if constexpr (sizeof(T) == 2) {
      if (a.m * a.n * int64_t{sizeof(T)} >= kStreamBytes) {
        end_of_part();  // around it, else the two stores become one
        stream_run(out, y);
        end_of_part();
      } else {
        store_run<8>(out, y);
      }
    } else {
      store_run<8>(out, y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) out[e] = y.v[e];
    end_of_part();
  }
}

// C[m][n] = sum over K of A's row m and B's row n; a workgroup's tile is BM x BN, its WM x WN
// waves take MB x NB fragments each. This is workgroup `id` of `workgroups`.
template <typename T, bool AOUT, bool BOUT, int MB, int NB, int WM, int WN>
__device__ __forceinline__ void linear_tile(const LinearArgs& a, unsigned id, unsigned workgroups,
                                            unsigned char* lds) {
  constexpr int BM = WM * MB * 16, BN = WN * NB * 16;
  using OpA = Operand<T, AOUT, BM, WM * WN>;
  using OpB = Operand<T, BOUT, BN, WM * WN>;
  using frag = typename Fragment<T>::type;
  constexpr int kStage = OpA::kBytes + OpB::kBytes;
  constexpr int kK = OpA::kK;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;

  // Workgroup ids go round the eight XCDs: each takes a run of tiles, in bands of 8 tile rows, so
  // that what its workgroups read at a time stays in its L2.
  {
    const unsigned per = workgroups >> 3, rest = workgroups & 7, x = id & 7;
    id = x * per + (x < rest ? x : rest) + (id >> 3);
  }
  const unsigned tiles = a.tiles_m * a.tiles_n;
  const unsigned split = id / tiles;
  id -= split * tiles;
  constexpr unsigned kBand = 8;
  const unsigned band = id / (kBand * a.tiles_n), in_band = id - band * kBand * a.tiles_n;
  const unsigned height = a.tiles_m - band * kBand < kBand ? a.tiles_m - band * kBand : kBand;
  const int64_t m0 = static_cast<int64_t>(band * kBand + in_band % height) * BM;
  const int64_t n0 = static_cast<int64_t>(in_band / height) * BN;

  const int64_t k0 = split * a.split_k;
  const int64_t k_count = k0 + a.split_k < a.k ? a.split_k : a.k - k0;
  const int stages = static_cast<int>((k_count + kK - 1) / kK);
  const int k_last = static_cast<int>(k_count - int64_t{stages - 1} * kK);
  OpA opa;
  OpB opb;
  opa.init(a.a, a.lda, a.m, m0, k0);
  opb.init(a.b, a.ldb, a.n, n0, k0);
  Reader<T, AOUT, BM, MB> ra;
  Reader<T, BOUT, BN, NB> rb;
  ra.init(wm * MB * 16);
  rb.init(wn * NB * 16);

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  frag fa[2][MB], fb[2][NB];
  const unsigned lds_at = static_cast<unsigned>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)(lds)));
  auto load = [&](int s) __attribute__((always_inline)) {
    const unsigned dst = lds_at + (s & 1) * kStage;
    if (s + 1 < stages) {
      const u32x4 a_rows = opa.rows(kK), b_rows = opb.rows(kK);
#pragma unroll
      for (int i = 0; i < OpA::kLoads; ++i) opa.load(a_rows, dst, wave, i);
#pragma unroll
      for (int i = 0; i < OpB::kLoads; ++i) opb.load(b_rows, dst + OpA::kBytes, wave, i);
    } else {
      opa.load_last(dst, wave, k_last);
      opb.load_last(dst + OpA::kBytes, wave, k_last);
    }
    opa.advance();
    opb.advance();
  };
  // Fragments i of A and B (where there is one) of half ks.
  auto read = [&](int s, int ks, int i) __attribute__((always_inline)) {
    const unsigned char* src = lds + (s & 1) * kStage;
    if (i < MB) fa[ks][i] = ra.read(src, ks, i);
    if (i < NB) fb[ks][i] = rb.read(src + OpA::kBytes, ks, i);
  };
  auto multiply = [&](int ks, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = Fragment<T>::mma(fb[ks][j], fa[ks][i], acc[i][j]);
  };
  static_assert(NB <= MB, "the steps of a stage are fragment rows of A");
  // A stage: the products of its first half while its second half is read, a barrier (then the
  // stage is in registers everywhere, and the next in LDS), the products of the second half while
  // the loads of the stage after next go out and the next stage's first half is read. A wave issues
  // in order and many reads or loads in a row wait for their queues: they are spread over the rows of
  // products, in this order.
  auto stage = [&](int s, auto next, auto after) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      multiply(0, i);
      // The first products wait for the fragments read before, not for these too.
      if (i == 0) __builtin_amdgcn_sched_barrier(0);
      read(s, 1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    u32x4 a_rows, b_rows;
    if constexpr (decltype(after)::value) {
      a_rows = opa.rows(kK);
      b_rows = opb.rows(kK);
    }
    if constexpr (decltype(next)::value) {
      wait_loads();
      __syncthreads();
      if constexpr (!decltype(after)::value) {
        if (s + 2 < stages) load(s + 2);
      }
    }
    const unsigned dst = lds_at + (s & 1) * kStage;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      if constexpr (decltype(after)::value) {
        constexpr int kPer = (OpA::kLoads + MB - 1) / MB;
        constexpr int kPerB = (OpB::kLoads + MB - 1) / MB;
#pragma unroll
        for (int q = 0; q < kPer; ++q)
          if (i * kPer + q < OpA::kLoads) opa.load(a_rows, dst, wave, i * kPer + q);
#pragma unroll
        for (int q = 0; q < kPerB; ++q)
          if (i * kPerB + q < OpB::kLoads)
            opb.load(b_rows, dst + OpA::kBytes, wave, i * kPerB + q);
      }
      multiply(1, i);
      if constexpr (decltype(next)::value) read(s + 1, 0, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (decltype(after)::value) {
      opa.advance();
      opb.advance();
    }
  };
  load(0);
  wait_loads();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MB; ++i) read(0, 0, i);
  if (stages > 1) load(1);
  int s = 0;
  for (; s + 3 < stages; ++s) stage(s, std::true_type{}, std::true_type{});
#pragma unroll 1
  for (; s + 1 < stages; ++s) stage(s, std::true_type{}, std::false_type{});
  stage(s, std::false_type{}, std::false_type{});

  // Each wave turns its sums through its own part of LDS, two fragment rows at a time, so that a
  // lane finishes 8 columns of a row and a store covers whole segments of rows.
  __syncthreads();
  constexpr int kPitch = NB * 16 + 4;  // floats; 4 more keep the 16 rows off each other's banks
  constexpr int kLanes = NB * 2;       // lanes of a row
  float* turn = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
  const int l = lane & 15, g = lane >> 4;
  const int64_t n = n0 + wn * NB * 16 + lane % kLanes * 8;
  const int count = n >= a.n ? 0 : (a.n - n < 8 ? static_cast<int>(a.n - n) : 8);
  float bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    bias[e] = a.bias != nullptr && e < count ? static_cast<float>(static_cast<const T*>(a.bias)[n + e])
                                             : 0.f;
#pragma unroll
  for (int i = 0; i < MB; i += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        *reinterpret_cast<f32x4*>(turn + (h * 16 + l) * kPitch + j * 16 + g * 4) = acc[i + h][j];
    const int64_t m_first = m0 + (wm * MB + i) * 16;
#pragma unroll 1
    for (int r = lane / kLanes; r < 32; r += 64 / kLanes) {
      const int64_t m = m_first + r;
      if (m >= a.m || count == 0) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(turn + r * kPitch + lane % kLanes * 8 + q * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q * 4 + e] = t[e];
      }
      finish<T>(a, v, bias, split, m, n, count);
    }
  }
}

template <typename T, bool AOUT, bool BOUT, int MB, int NB, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_kernel(LinearArgs a) {
  extern __shared__ __align__(1024) unsigned char lds[];
  linear_tile<T, AOUT, BOUT, MB, NB, WM, WN>(a, blockIdx.x, gridDim.x, lds);
}

// 32 columns' sums of a bias gradient from their partial sums, in a fixed order.
template <typename T, int THREADS>
__device__ __forceinline__ void add_sums(const LinearSums& a, unsigned id, float* scratch) {
  constexpr int kGroups = THREADS / 32;
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const int64_t c = int64_t{id} * 32 + lane;
  float s = 0.f;
  if (c < a.columns) {
    const float* p = a.partial + c;
#pragma unroll 8
    for (int64_t r = group; r < a.parts; r += kGroups) s += p[r * a.columns];
  }
  scratch[group * 33 + lane] = s;
  __syncthreads();
  if (group != 0 || c >= a.columns) return;
  float total = 0.f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) total += scratch[g * 33 + lane];
  static_cast<T*>(a.output)[c] = static_cast<T>(total);
}

// Both gradients' products and the bias's sums in one launch: `first` workgroups of the product with
// more K values a tile, then the other's up to `products`. Workgroups of one fill the places that
// the other leaves free, and one plan weighs both (8192 x 1024 -> 4096 in bfloat16 142 -> 124 us, 1001
// x 333 -> 517 in float 31 -> 22; a launch each with plans of their own before).
template <typename T, int MB, int NB, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_gradients(LinearArgs x, LinearArgs w,
                                                                   LinearSums sums,
                                                                   unsigned first,
                                                                   unsigned products,
                                                                   bool weight_first) {
  extern __shared__ __align__(1024) unsigned char lds[];
  if (blockIdx.x >= products) {
    add_sums<T, 64 * WM * WN>(sums, blockIdx.x - products, reinterpret_cast<float*>(lds));
    return;
  }
  const bool in_first = blockIdx.x < first;
  const unsigned id = in_first ? blockIdx.x : blockIdx.x - first;
  const unsigned workgroups = in_first ? first : products - first;
  if (in_first == weight_first)
    linear_tile<T, true, true, MB, NB, WM, WN>(w, id, workgroups, lds);
  else
    linear_tile<T, false, true, MB, NB, WM, WN>(x, id, workgroups, lds);
}

// ---- few rows --------------------------------------------------------------------------------

// Rows m < 16 MF of x times 16 rows of W a workgroup; W waves share K. Fragment reads straight
// from memory, of any alignment; past K's end zeros.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::type load_fragment(const T* row, int64_t k,
                                                                    int64_t k_end) {
  constexpr int kVec = 16 / sizeof(T);
  using frag = typename Fragment<T>::type;
  if (k + kVec <= k_end) return __builtin_bit_cast(frag, load_run<kVec>(row + k));
  Run<T, kVec> r;
#pragma unroll
  for (int i = 0; i < kVec; ++i) r.v[i] = k + i < k_end ? row[k + i] : static_cast<T>(0.f);
  return __builtin_bit_cast(frag, r);
}

constexpr int kFewWaves = 8;
template <typename T, int MF>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_rows(LinearArgs a) {
  constexpr int kStep = 64 / sizeof(T);  // K values of a fragment over its four lane groups
  constexpr int kUnroll = MF == 4 ? 2 : 4;
  using frag = typename Fragment<T>::type;
  __shared__ float sums[kFewWaves][16][MF * 16 + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const T* x = static_cast<const T*>(a.a);
  const T* w = static_cast<const T*>(a.b);
  // Rows past the end read the last one; their sums are not used.
  const T* w_row = w + std::min<int64_t>(n0 + l, a.n - 1) * a.ldb;
  const T* x_row[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) x_row[f] = x + std::min<int64_t>(f * 16 + l, a.m - 1) * a.lda;
  f32x4 acc[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Every wave a run of K: whole steps, the last wave the rest.
  const int64_t steps = (a.k + kStep - 1) / kStep;
  const int64_t first = steps * wave / kFewWaves, last = steps * (wave + 1) / kFewWaves;
  int64_t s = first;
  for (; s + kUnroll <= last && (s + kUnroll) * kStep <= a.k; s += kUnroll) {
    frag fw[kUnroll], fx[kUnroll][MF];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = (s + u) * kStep + g * (16 / sizeof(T));
      fw[u] = __builtin_bit_cast(frag, load_run<16 / sizeof(T)>(w_row + k));
#pragma unroll
      for (int f = 0; f < MF; ++f)
        fx[u][f] = __builtin_bit_cast(frag, load_run<16 / sizeof(T)>(x_row[f] + k));
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int f = 0; f < MF; ++f) acc[f] = Fragment<T>::mma(fw[u], fx[u][f], acc[f]);
  }
  for (; s < last; ++s) {
    const int64_t k = s * kStep + g * (16 / sizeof(T));
    const frag fw = load_fragment(w_row, k, a.k);
#pragma unroll
    for (int f = 0; f < MF; ++f) acc[f] = Fragment<T>::mma(fw, load_fragment(x_row[f], k, a.k), acc[f]);
  }
  // acc[f][e]: column n0 + 4 g + e of row f * 16 + l.
#pragma unroll
  for (int f = 0; f < MF; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][g * 4 + e][f * 16 + l] = acc[f][e];
  __syncthreads();
  for (int i = threadIdx.x; i < MF * 16 * 2; i += 64 * kFewWaves) {
    const int m = i / 2, c = i % 2 * 8;
    const int64_t n = n0 + c;
    if (m >= a.m || n >= a.n) continue;
    const int count = a.n - n < 8 ? static_cast<int>(a.n - n) : 8;
    float v[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int q = 0; q < kFewWaves; ++q) v[e] += sums[q][c + e][m];
      bias[e] = a.bias != nullptr && e < count
                    ? static_cast<float>(static_cast<const T*>(a.bias)[n + e])
                    : 0.f;
    }
    finish<T>(a, v, bias, 0, m, n, count);
  }
}

// ---- sums of a split K, padding, the activation's gradient -----------------------------------------

// Adds the splits' sums of one or two products in order and finishes 8 columns of a row a thread.
struct LinearJoin {
  LinearArgs a;
  const float* partial;
  int64_t splits;
  unsigned workgroups;
};
template <typename T>
__global__ __launch_bounds__(256) void linear_join(LinearJoin one, LinearJoin two) {
  const bool second = blockIdx.x >= one.workgroups;
  const LinearArgs& a = second ? two.a : one.a;
  const int64_t splits = second ? two.splits : one.splits;
  const int64_t workgroups = second ? two.workgroups : one.workgroups;
  const int64_t parts = (a.n + 7) / 8, total = a.m * parts, step = a.m * a.n;
  for (int64_t id = static_cast<int64_t>(blockIdx.x - (second ? one.workgroups : 0)) * 256 +
                    threadIdx.x;
       id < total; id += workgroups * 256) {
    const int64_t m = id / parts, n = id % parts * 8;
    const int count = a.n - n < 8 ? static_cast<int>(a.n - n) : 8;
    float v[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
      bias[e] = a.bias != nullptr && e < count
                    ? static_cast<float>(static_cast<const T*>(a.bias)[n + e])
                    : 0.f;
    }
    const float* p = (second ? two.partial : one.partial) + m * a.n + n;
#pragma unroll 4
    for (int64_t s = 0; s < splits; ++s, p += step) {
      if (count == 8) {
        const Run<float, 4> lo = load_run<4>(p), hi = load_run<4>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += lo.v[e];
          v[e + 4] += hi.v[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < count) v[e] += p[e];
        end_of_part();
      }
    }
    finish<T>(a, v, bias, 0, m, n, count);
  }
}

// Rows copied with a pitch of whole 16 bytes, zeros past their end.
template <typename T>
__global__ __launch_bounds__(256) void linear_pad(const T* __restrict__ src, int64_t stride,
                                                  int64_t rows, int64_t columns, T* __restrict__ dst) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t parts = (columns + kVec - 1) / kVec, total = rows * parts;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = id / parts, c = id % parts * kVec;
    const T* p = src + r * stride + c;
    Run<T, kVec> v;
    if (c + kVec <= columns) {
      v = load_run<kVec>(p);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v.v[i] = c + i < columns ? p[i] : static_cast<T>(0.f);
    }
    store_run<kVec>(dst + id * kVec, v);
  }
}

// dz = dy act'(z) (with a pitch of whole 16 bytes, zeros past a row's end) and the sums of dz over
// each workgroup's rows, which follow each other. TPR threads a row, 8 columns a thread. dz is rounded
// to the element type, which the matrix cores multiply; the bias's sums take it unrounded. Beside GELU
// (relu's and no activation's dz are exact) that rounding is as large as the gradients' own: they
// are 1.41 of their rounding off (8192 x 1024 -> 4096 bf16 2.35e-3 for 1.66e-3). dz as two 16-bit
// terms would take products of twice the K, 72 -> 147 and 82 -> 138 us there of a step's 251.
template <typename T, int TPR>
__global__ __launch_bounds__(256) void linear_grad(LinearGradArgs a) {
  constexpr int kColumns = TPR * 8, kRows = 256 / TPR;
  __shared__ float sums[kRows][kColumns];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kColumns + lane * 8;
  const int count = n >= a.columns ? 0 : (a.columns - n < 8 ? static_cast<int>(a.columns - n) : 8);
  const T* dy = static_cast<const T*>(a.grad_output);
  const Slope<T>* slope = static_cast<const Slope<T>*>(a.slope);
  T* dz = static_cast<T*>(a.grad_pre);
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto finish_row = [&](int64_t m, Run<T, 8> d, const Run<Slope<T>, 8>& z)
                        __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float g = static_cast<float>(d.v[e]);
      if (slope != nullptr) g *= slope_of(z.v[e]);
      d.v[e] = static_cast<T>(g);
      sum[e] += g;
    }
    if (dz == nullptr) return;
    T* o = dz + m * a.pitch + n;
    if (n + 8 <= a.pitch) {
      store_run<8>(o, d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < a.pitch) o[e] = d.v[e];
      end_of_part();
    }
  };
  const int64_t first = a.rows * blockIdx.y / gridDim.y, last = a.rows * (blockIdx.y + 1) / gridDim.y;
  if (count == 8) {
    // Four rows' loads at a time.
    int64_t m = first + group;
    for (; m + 3 * kRows < last; m += 4 * kRows) {
      Run<T, 8> d[4];
      Run<Slope<T>, 8> z[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        d[u] = load_run<8>(dy + (m + u * kRows) * a.grad_stride + n);
        if (slope != nullptr) z[u] = load_run<8>(slope + (m + u * kRows) * a.columns + n);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) finish_row(m + u * kRows, d[u], z[u]);
    }
    for (; m < last; m += kRows) {
      const Run<T, 8> d = load_run<8>(dy + m * a.grad_stride + n);
      finish_row(m, d, slope != nullptr ? load_run<8>(slope + m * a.columns + n)
                                        : Run<Slope<T>, 8>{});
    }
  } else if (count > 0) {
    for (int64_t m = first + group; m < last; m += kRows) {
      Run<T, 8> d;
      Run<Slope<T>, 8> z;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        d.v[e] = e < count ? dy[m * a.grad_stride + n + e] : static_cast<T>(0.f);
        z.v[e] = slope != nullptr && e < count ? slope[m * a.columns + n + e] : Slope<T>(0);
      }
      finish_row(m, d, z);
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[group][lane * 8 + e] = sum[e];
  __syncthreads();
  for (int c = threadIdx.x; c < kColumns; c += 256) {
    const int64_t column = static_cast<int64_t>(blockIdx.x) * kColumns + c;
    if (column >= a.columns) break;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) s += sums[r][c];
    a.partial[blockIdx.y * a.columns + column] = s;
  }
}

// More than 64 KB of LDS has to be asked for, once per device and kernel (`asked` is the kernel's).
template <typename Kernel>
hipError_t ask_lds(Kernel kernel, int bytes, std::atomic<uint64_t>& asked) {
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

template <int MB, int NB, int WM, int WN>
constexpr int kTileBytes = 2 * (WM * MB + WN * NB) * 16 * 128;

template <typename T, bool AOUT, bool BOUT, int MB, int NB, int WM, int WN>
hipError_t launch_tiles(const LinearArgs& a, int64_t splits, hipStream_t stream) {
  constexpr int kBytes = kTileBytes<MB, NB, WM, WN>;
  const auto kernel = linear_kernel<T, AOUT, BOUT, MB, NB, WM, WN>;
  static std::atomic<uint64_t> asked{0};
  const hipError_t err = ask_lds(kernel, kBytes, asked);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.tiles_m * a.tiles_n * splits)),
                     dim3(64 * WM * WN), kBytes, stream, a);
  return hipGetLastError();
}

template <typename T, int MB, int NB, int WM, int WN>
hipError_t launch_gradients(const LinearArgs& x, unsigned x_groups, const LinearArgs& w,
                            unsigned w_groups, const LinearSums& sums, hipStream_t stream) {
  constexpr int kBytes = kTileBytes<MB, NB, WM, WN>;
  const auto kernel = linear_gradients<T, MB, NB, WM, WN>;
  static std::atomic<uint64_t> asked{0};
  const hipError_t err = ask_lds(kernel, kBytes, asked);
  if (err != hipSuccess) return err;
  const bool weight_first = w.split_k >= x.split_k;
  const unsigned products = x_groups + w_groups;
  const unsigned extra =
      sums.output != nullptr ? static_cast<unsigned>((sums.columns + 31) / 32) : 0;
  hipLaunchKernelGGL(kernel, dim3(products + extra), dim3(64 * WM * WN), kBytes, stream, x, w, sums,
                     weight_first ? w_groups : x_groups, products, weight_first);
  return hipGetLastError();
}

// The product's arguments with its tiles and, where K is split, the place of its sums.
LinearArgs planned(LinearArgs a, const LinearPlan& p, float* partial) {
  a.split_k = p.split_k;
  a.tiles_m = static_cast<unsigned>((a.m + p.tile - 1) / p.tile);
  a.tiles_n = static_cast<unsigned>((a.n + p.tile - 1) / p.tile);
  if (p.splits > 1) a.partial = partial;
  return a;
}

LinearJoin join_of(const LinearArgs& a, const LinearPlan& p, const float* partial) {
  const int64_t work = a.m * ((a.n + 7) / 8);
  return {a, partial, p.splits,
          p.splits > 1 ? static_cast<unsigned>(std::min<int64_t>((work + 255) / 256, 8192)) : 0};
}
template <typename T>
hipError_t launch_join(const LinearJoin& one, const LinearJoin& two, hipStream_t stream) {
  if (one.workgroups + two.workgroups == 0) return hipSuccess;
  hipLaunchKernelGGL(linear_join<T>, dim3(one.workgroups + two.workgroups), dim3(256), 0, stream,
                     one, two);
  return hipGetLastError();
}

template <typename T, bool AOUT, bool BOUT>
hipError_t launch_tiles_of(const LinearArgs& t, const LinearPlan& p, hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (p.tile == 256) return launch_tiles<T, AOUT, BOUT, 8, 4, 2, 4>(t, p.splits, stream);
  return p.tile == 128 ? launch_tiles<T, AOUT, BOUT, 4, 4, 2, 2>(t, p.splits, stream)
                       : launch_tiles<T, AOUT, BOUT, 2, 2, 2, 2>(t, p.splits, stream);
}

template <typename T, bool AOUT, bool BOUT>
hipError_t launch_product_typed(const LinearArgs& a, const LinearPlan& p, float* partial,
                                hipStream_t stream) {
  if constexpr (!AOUT && !BOUT) {
    if (p.few_rows) {
      const dim3 grid(static_cast<unsigned>((a.n + 15) / 16)), block(64 * kFewWaves);
      if (a.m <= 16)
        hipLaunchKernelGGL((linear_few_rows<T, 1>), grid, block, 0, stream, a);
      else if (a.m <= 32)
        hipLaunchKernelGGL((linear_few_rows<T, 2>), grid, block, 0, stream, a);
      else
        hipLaunchKernelGGL((linear_few_rows<T, 4>), grid, block, 0, stream, a);
      return hipGetLastError();
    }
  }
  const hipError_t err = launch_tiles_of<T, AOUT, BOUT>(planned(a, p, partial), p, stream);
  if (err != hipSuccess) return err;
  return launch_join<T>(join_of(a, p, partial), LinearJoin{}, stream);
}

template <typename T>
hipError_t launch_product(const LinearArgs& a, LinearProduct which, const LinearPlan& p,
                          float* partial, hipStream_t stream) {
  switch (which) {
    case LinearProduct::kForward:
      return launch_product_typed<T, false, false>(a, p, partial, stream);
    case LinearProduct::kGradInput:
      return launch_product_typed<T, false, true>(a, p, partial, stream);
    default:
      return launch_product_typed<T, true, true>(a, p, partial, stream);
  }
}

template <typename T>
hipError_t launch_both(const LinearArgs& x, const LinearPlan& xp, float* x_partial,
                       const LinearArgs& w, const LinearPlan& wp, float* w_partial,
                       const LinearSums& sums, hipStream_t stream) {
  const LinearArgs tx = planned(x, xp, x_partial), tw = planned(w, wp, w_partial);
  const auto gx = static_cast<unsigned>(tx.tiles_m * tx.tiles_n * xp.splits);
  const auto gw = static_cast<unsigned>(tw.tiles_m * tw.tiles_n * wp.splits);
  hipError_t err = hipErrorInvalidValue;
  if (xp.tile == 64)
    err = launch_gradients<T, 2, 2, 2, 2>(tx, gx, tw, gw, sums, stream);
  else if (xp.tile == 128)
    err = launch_gradients<T, 4, 4, 2, 2>(tx, gx, tw, gw, sums, stream);
  else if constexpr (sizeof(T) == 2)
    err = launch_gradients<T, 8, 4, 2, 4>(tx, gx, tw, gw, sums, stream);
  if (err != hipSuccess) return err;
  return launch_join<T>(join_of(x, xp, x_partial), join_of(w, wp, w_partial), stream);
}

// What a launch of a tile's workgroups takes (us), fitted to over a thousand timings (25 problems,
// forward and backward, 16-bit and float, every tile and number of parts): `slots`
// run side by side on the chip; a turn of them takes `turn` and `full` a K value, a workgroup alone
// `alone` a K value. (16-bit at 8192^3: 256 x 256 1370 TFLOP/s, 128 x 128 1160; float is bound by its
// MFMA rate at either tile, 130.)
struct TileCost {
  int tile, threads, slots;
  float set_up, alone, turn, full;
};
constexpr TileCost kTiles16[] = {{64, 256, 1280, 4.0f, 0.0046f, 2.7f, 0.0150f},
                                 {128, 256, 512, 5.0f, 0.0102f, 4.0f, 0.0140f},
                                 {256, 512, 256, 4.5f, 0.0210f, 6.0f, 0.0238f}};
constexpr TileCost kTiles32[] = {{64, 256, 1280, 3.9f, 0.0206f, 4.8f, 0.0772f},
                                 {128, 256, 512, 5.7f, 0.0656f, 7.9f, 0.1122f}};

// `groups` workgroups of `k` K values on the average, at most `most`: bound by the longest, or by what the
// busiest compute unit is given.
float tiles_time(const TileCost& c, uint32_t groups, float k, float most) {
  const float turns = static_cast<float>((groups + 255) / 256 * 256) / static_cast<float>(c.slots);
  return c.set_up + std::max(c.alone * most, turns * (c.turn + c.full * k));
}

// Writing, reading and joining splits' sums: `bytes`, at most `splits` of them in a row of loads.
float join_time(bool single, float bytes, uint32_t splits) {
  return 2.0f + (single ? 0.5f : 0.3f) * static_cast<float>(splits) +
         bytes / (single ? 8.5e6f : 4.6e6f);
}
float split_bytes(uint32_t m, uint32_t n, uint32_t splits) {
  return splits > 1 ? static_cast<float>(m) * static_cast<float>(n) *
                          static_cast<float>(4 * splits + 2)
                    : 0.f;
}

// A few parts only: this runs on every call.
constexpr uint32_t kParts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};

// K's stages in parts of at most `each`, as even as they come.
struct Split {
  uint32_t count, stages;
  Split(uint32_t all, uint32_t each) {
    stages = (all + (all + each - 1) / each - 1) / ((all + each - 1) / each);
    count = (all + stages - 1) / stages;
  }
};

LinearPlan plan_of(int tile, const Split& split, uint32_t stage, int64_t k) {
  LinearPlan p{};
  p.tile = tile;
  p.splits = static_cast<int>(split.count);
  p.split_k = split.count > 1 ? int64_t{split.stages} * stage : k;
  return p;
}

template <typename Visit>
void each_tile(bool single, Visit visit) {
  if (single)
    for (const TileCost& c : kTiles32) visit(c);
  else
    for (const TileCost& c : kTiles16) visit(c);
}

uint32_t over(int64_t n, int64_t by) { return static_cast<uint32_t>((n + by - 1) / by); }

}  // namespace

LinearPlan plan_product(convnd_hip_dtype dtype, LinearProduct which, int64_t m, int64_t n,
                        int64_t k) {
  LinearPlan p{};
  p.splits = 1;
  p.split_k = k;
  const bool single = dtype == CONVND_HIP_FLOAT32;
  // The few rows' kernel reads W once but its input once per 16 columns, and 16 rows of W through one
  // compute unit; from some length of K on tiles with K in parts are better off, sooner the more rows
  // there are, and with up to 16 only where columns are few (us of the few rows' kernel and of tiles
  // with cold weights: 64 x 4096 -> 4096 bf16 25 and 21, 64 x 1024 -> 4096 9 and 15; 32 x 8192 -> 4096
  // 29 and 25, 20 x 4096 -> 1024 13.6 and 15.4; 8 x 16384 -> 1024 33 and 25, 4 x 8192 -> 1024 17.2 and
  // 17.7, 2 x 16384 -> 4096 38 and 44).
  const int64_t row_bytes = k * (single ? 4 : 2);
  if (which == LinearProduct::kForward && m <= 64 &&
      (row_bytes < (m > 32 ? 8192 : m > 16 ? 16384 : 32768) || (m <= 16 && n >= 4096))) {
    p.few_rows = true;
    return p;
  }
  const uint32_t stage = single ? 32 : 64, stages = over(k, stage);
  float best = 0;
  each_tile(single, [&](const TileCost& c) {
    const int64_t tiles = int64_t{over(m, c.tile)} * over(n, c.tile);
    for (const uint32_t parts : kParts) {
      const Split split(stages, (stages + parts - 1) / parts);
      if (parts > 1 && split.stages < 4) break;
      if (!launch_fits(tiles * split.count, c.threads)) break;
      const float length = static_cast<float>(split.stages * stage);
      float us = tiles_time(c, static_cast<uint32_t>(tiles * split.count),
                            static_cast<float>(k) / static_cast<float>(split.count), length);
      if (split.count > 1)
        us += join_time(single, split_bytes(m, n, split.count), split.count);
      if (best == 0 || us < best) {
        best = us;
        p = plan_of(c.tile, split, stage, k);
      }
    }
  });
  return p;
}

// Both gradients' products in one launch, so of one tile: workgroups of both run side by side and take
// about as long each where K is cut into parts of about one length.
void plan_gradients(convnd_hip_dtype dtype, int64_t rows, int64_t inputs, int64_t outputs,
                    LinearPlan* x, LinearPlan* w) {
  const bool single = dtype == CONVND_HIP_FLOAT32;
  const uint32_t stage = single ? 32 : 64;
  const uint32_t x_stages = over(outputs, stage), w_stages = over(rows, stage);
  const uint32_t longest = std::max(x_stages, w_stages);
  float best = 0;
  each_tile(single, [&](const TileCost& c) {
    const uint32_t across = over(inputs, c.tile);
    const int64_t x_tiles = int64_t{over(rows, c.tile)} * across;
    const int64_t w_tiles = int64_t{over(outputs, c.tile)} * across;
    const float work = (static_cast<float>(x_tiles) * static_cast<float>(x_stages) +
                        static_cast<float>(w_tiles) * static_cast<float>(w_stages)) *
                       static_cast<float>(stage);
    for (const uint32_t parts : kParts) {
      const uint32_t each = (longest + parts - 1) / parts;
      if (parts > 1 && each < 4) break;
      const Split xs(x_stages, each), ws(w_stages, each);
      const int64_t groups = x_tiles * xs.count + w_tiles * ws.count;
      // With the bias's sums in the same launch.
      if (!launch_fits(groups + over(outputs, 32), c.threads)) break;
      float us = tiles_time(c, static_cast<uint32_t>(groups), work / static_cast<float>(groups),
                            static_cast<float>(std::max(xs.stages, ws.stages) * stage));
      if (xs.count > 1 || ws.count > 1)
        us += join_time(single,
                        split_bytes(rows, inputs, xs.count) + split_bytes(outputs, inputs, ws.count),
                        std::max(xs.count, ws.count));
      if (best == 0 || us < best) {
        best = us;
        *x = plan_of(c.tile, xs, stage, outputs);
        *w = plan_of(c.tile, ws, stage, rows);
      }
    }
  });
}

hipError_t launch_linear_product(convnd_hip_dtype dtype, const LinearArgs& a, LinearProduct which,
                                 const LinearPlan& p, float* partial, hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return launch_product<float>(a, which, p, partial, stream);
    case CONVND_HIP_FLOAT16:
      return launch_product<_Float16>(a, which, p, partial, stream);
    case CONVND_HIP_BFLOAT16:
      return launch_product<__bf16>(a, which, p, partial, stream);
    default:
      return hipErrorInvalidValue;
  }
}

hipError_t launch_linear_gradients(convnd_hip_dtype dtype, const LinearArgs& x,
                                   const LinearPlan& xp, float* x_partial, const LinearArgs& w,
                                   const LinearPlan& wp, float* w_partial, const LinearSums& sums,
                                   hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return launch_both<float>(x, xp, x_partial, w, wp, w_partial, sums, stream);
    case CONVND_HIP_FLOAT16:
      return launch_both<_Float16>(x, xp, x_partial, w, wp, w_partial, sums, stream);
    case CONVND_HIP_BFLOAT16:
      return launch_both<__bf16>(x, xp, x_partial, w, wp, w_partial, sums, stream);
    default:
      return hipErrorInvalidValue;
  }
}

hipError_t launch_linear_pad(convnd_hip_dtype dtype, const void* src, int64_t stride, int64_t rows,
                             int64_t columns, void* dst, hipStream_t stream) {
  const int vec = dtype == CONVND_HIP_FLOAT32 ? 4 : 8;
  const int64_t work = rows * ((columns + vec - 1) / vec);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((work + 255) / 256, 8192))), block(256);
  if (dtype == CONVND_HIP_FLOAT32)
    hipLaunchKernelGGL(linear_pad<float>, grid, block, 0, stream, static_cast<const float*>(src),
                       stride, rows, columns, static_cast<float*>(dst));
  else  // either 16-bit type: only zeros are made, the rest is moved
    hipLaunchKernelGGL(linear_pad<_Float16>, grid, block, 0, stream,
                       static_cast<const _Float16*>(src), stride, rows, columns,
                       static_cast<_Float16*>(dst));
  return hipGetLastError();
}

namespace {

int grad_threads(int64_t columns) { return columns <= 1024 ? 64 : 256; }

template <typename T>
void launch_grad(const LinearGradArgs& a, int64_t parts, hipStream_t stream) {
  const int threads = grad_threads(a.columns);
  const dim3 grid(static_cast<unsigned>((a.columns + threads * 8 - 1) / (threads * 8)),
                  static_cast<unsigned>(parts));
  if (threads == 64)
    hipLaunchKernelGGL((linear_grad<T, 64>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((linear_grad<T, 256>), grid, dim3(256), 0, stream, a);
}

}  // namespace

int64_t linear_grad_parts(int64_t rows, int64_t columns) {
  const int threads = grad_threads(columns);
  const int64_t wide = (columns + threads * 8 - 1) / (threads * 8), at_a_time = 256 / threads;
  const int64_t needed = (rows + at_a_time - 1) / at_a_time;
  return std::max<int64_t>(1, std::min<int64_t>(needed, std::max<int64_t>(1, 1024 / wide)));
}

hipError_t launch_linear_grad(convnd_hip_dtype dtype, const LinearGradArgs& a, int64_t parts,
                              hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      launch_grad<float>(a, parts, stream);
      break;
    case CONVND_HIP_FLOAT16:
      launch_grad<_Float16>(a, parts, stream);
      break;
    case CONVND_HIP_BFLOAT16:
      launch_grad<__bf16>(a, parts, stream);
      break;
    default:
      return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace convnd
