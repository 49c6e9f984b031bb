// Gated delta rule: a matrix state S [key_size, value_size] a head, corrected towards each token's value,
//
//   S_t = a_t S_(t-1) + k_t u_t^T,  u_t = beta_t (v_t - a_t S_(t-1)^T k_t),  a_t = exp(decay_t)
//   o_t = S_t^T q_t
//
// with q scaled (and q, k of unit length where asked for). Over a chunk of C tokens with the state S
// before it, the products G_ij = a_(j+1) .. a_i and their ends c_i = a_1 .. a_i, e_j = G_Cj,
//
//   A_ij = beta_i G_ij k_i.k_j (i > j),  T = (I + A)^-1,  U = T diag(beta) (V - diag(c) K S)
//   O = diag(c) Q S + P U,  P_ij = G_ij q_i.k_j (i >= j),  S' = c_C S + K^T diag(e) U
//
// T and P do not need the state: delta_prepare makes them for all chunks side by side, then
// delta_forward walks each head's chunks with S in registers; delta_backward walks back with S's gradient,
// and delta_gradients makes the rest of all chunks side by side. Of a step's few tokens delta_step
// computes the definition itself. Of 8 sequences of 2048 tokens and 8 heads of 128 x 128 in bfloat16:
// prepare 34 us, forward 92, backward 113, gradients 115 (token by token in torch 16 ms).
//
// Products run on the matrix cores: in 16 bits on chunks of 64 tokens, in float of 32 (128 bytes a row
// of T either way, the row of every panel in LDS). Decays' sums are kept in 64 bits and differences of
// them taken before exp, so that long chunks of strong decays lose nothing; a decay whose exp is zero
// in float (-inf, a packed document's start) is left out of the sums and its pairs masked. Unit lengths
// are factors of rows (rk, rq), never rounded into the operands.
//
// What is not an input is split into two 16-bit terms before a product (S, U, T, P and what they are
// made of), which doubles matrix instructions but not LDS reads of the shared operand, by which the
// walk is bound: the state stays within 1e-5 of the 64-bit one over thousands of tokens (one term:
// 3e-3) and outputs within their own rounding (1.65e-3 in bfloat16; one term 3.6e-3). What is kept for a
// backward, S and U (and D and Y for the gradients), is one term: a gradient of q, k or a gate that takes two
// of them is 2.5e-3 to 3.3e-3 off in bfloat16, where its own rounding is 1.65e-3; with the second terms the
// backward would move a half more. Of float16 that term is in units of the head's largest value or cotangent, and
// the backward's walk in those of the latter throughout (training 8 x 2048 tokens of 8 heads of 128 x 128: 23 us of
// 405 to find them, 4 in the walk).

#include <algorithm>
#include <type_traits>

#include "convnd_internal.h"
#include "convnd_sequence.h"

namespace convnd {
namespace {

constexpr float kNormEps = 1e-6f;

template <typename T>
struct Chunk {
  using frag = typename Fragment<T>::type;
  static constexpr int kTokens = delta_chunk(sizeof(T));
  static constexpr int kTerms = sizeof(T) == 2 ? 2 : 1;
  static constexpr int kTiles = kTokens / 16;    // of 16 rows
  static constexpr int kStep = 64 / sizeof(T);   // contraction values of a fragment
  static constexpr int kPer = kStep / 16;        // tiles a fragment is made of
  static constexpr int kPanel = kTokens * 128;   // bytes of kTokens rows of 128
};

template <typename T>
using Four = T __attribute__((ext_vector_type(4)));

// Panels: rows of 128 bytes whose 16-byte pieces are permuted by the row, so that reads of 16 rows at a
// piece, in order or as 8 (i / 4) + i % 4, and transposing reads meet no bank twice.
__device__ __forceinline__ int swizzle(int row) {
  return ((row >> 1) & 1) << 2 | ((row >> 3) & 1) << 1 | (((row >> 4) ^ (row >> 2)) & 1);
}

// Lane's place among 16 columns (or rows) and its group of contraction values.
struct Lane {
  int l, g;
  __device__ __forceinline__ Lane() : l(threadIdx.x & 15), g((threadIdx.x >> 4) & 3) {}
};

// The row that lane l of tile m reads as operand, so that results' registers are contraction values in
// order: register e of lane group g in tile m holds row first_row(m, g) + e, and the kPer tiles of a
// fragment together its 16 bytes.
template <typename T>
__device__ __forceinline__ int operand_row(int m, int l) {
  if constexpr (sizeof(T) == 2) return m / 2 * 32 + (l >> 2) * 8 + m % 2 * 4 + (l & 3);
  return m * 16 + l;
}
template <typename T>
__device__ __forceinline__ int first_row(int m, int g) {
  if constexpr (sizeof(T) == 2) return m / 2 * 32 + g * 8 + m % 2 * 4;
  return m * 16 + g * 4;
}

template <typename V>
__device__ __forceinline__ V lds_read(unsigned at) {
  return *reinterpret_cast<__attribute__((address_space(3))) const V*>(static_cast<uintptr_t>(at));
}
template <typename V>
__device__ __forceinline__ void lds_write(unsigned at, const V& v) {
  *reinterpret_cast<__attribute__((address_space(3))) V*>(static_cast<uintptr_t>(at)) = v;
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)(p)));
}

// Reads of panels by their LDS address. The swizzle of a place is the exclusive or of a part of the lane and
// one of the place, so a lane holds one address for each value of the latter and every read is one of them
// and a constant; computed place by place, the compiler kept hundreds of addresses (and spilled).
template <typename T>
struct Reader {
  using frag = typename Chunk<T>::frag;
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kPanel = Chunk<T>::kPanel;
  unsigned rows[4], operands[kHalf ? 4 : 1], columns[4], ordered[kHalf ? 8 : 1];

  // `flip` goes into the places of ordered columns (64: two tiles further in a panel).
  __device__ __forceinline__ explicit Reader(unsigned flip = 0, unsigned thread = threadIdx.x) {
    const unsigned l = thread & 15, g = (thread >> 4) & 3;
    const auto bit = [](unsigned v, int i) { return v >> i & 1; };
#pragma unroll
    for (unsigned x = 0; x < 4; ++x)  // halves of a panel's rows, odd tiles
      rows[x] = l * 128 + (((g ^ (bit(l, 1) << 2 | bit(l, 3) << 1 | bit(l, 2))) << 4) ^ (x >> 1 << 6) ^ ((x & 1) << 4));
    if constexpr (kHalf) {
#pragma unroll
      for (unsigned x = 0; x < 4; ++x) {
        operands[x] = (l >> 2) * 1024 + (l & 3) * 128 +
                      (((g ^ (bit(l, 1) << 2 | bit(l, 2) << 1 | bit(l, 3))) << 4) ^ (x >> 1 << 6) ^ ((x & 1) << 4));
        const unsigned row = bit(l, 3) << 2 | bit(g, 0) << 1 | bit(g, 1);  // odd pairs of tiles, second rows
        columns[x] = g * 1024 + (l >> 2) * 128 + ((((l & 3) ^ row) << 4) ^ (x >> 1 << 6) ^ ((x & 1) << 4));
      }
#pragma unroll
      for (unsigned x = 0; x < 8; ++x)  // tiles of a panel, second rows
        ordered[x] = g * 1024 + (l >> 2) * 128 + (l & 1) * 8 +
                     (flip ^ ((bit(l, 1) ^ (bit(l, 3) << 2 | bit(g, 0) << 1 | bit(g, 1))) << 4) ^ (x >> 1 << 5) ^ ((x & 1) << 4));
    } else {
#pragma unroll
      for (unsigned x = 0; x < 4; ++x)  // odd tiles and second rows, odd steps
        columns[x] = g * 512 + (l & 3) * 4 +
                     ((((l >> 2) ^ (bit(g, 1) << 1 | bit(g, 0))) << 4) ^ (x >> 1 << 6) ^ ((x & 1) << 4));
    }
  }

  // The same addresses `by` bytes on, as they are: were the sum known, the compiler would add each read's constant
  // to `by` and the lane's part to that, two instructions a read.
  __device__ __forceinline__ Reader moved(unsigned by) const {
    Reader r = *this;
    const auto move = [by](unsigned& at) __attribute__((always_inline)) {
      at += by;
      asm("" : "+v"(at));
    };
    for (unsigned& at : r.rows) move(at);
    for (unsigned& at : r.operands) move(at);
    for (unsigned& at : r.columns) move(at);
    for (unsigned& at : r.ordered) move(at);
    return r;
  }

  // Fragment of step ks (two a panel) of row 16 n + l.
  __device__ __forceinline__ frag row(unsigned panels, int n, int ks) const {
    return lds_read<frag>(panels + rows[ks % 2 * 2 + n % 2] + ks / 2 * kPanel + n * 2048);
  }
  // Of row operand_row(m, l).
  __device__ __forceinline__ frag operand(unsigned panels, int m, int ks) const {
    if constexpr (kHalf)
      return lds_read<frag>(panels + operands[ks % 2 * 2 + m % 2] + ks / 2 * kPanel + m / 2 * 4096 + m % 2 * 512);
    else
      return row(panels, m, ks);
  }
  // Fragments of the transposed panels: contraction values are rows kt * kStep .., the lane's row of the
  // operand is column operand_row(m, l).
  __device__ __forceinline__ frag column(unsigned panels, int m, int kt) const {
    if constexpr (kHalf) {
      const unsigned at = panels + m / 4 * kPanel + kt * 4096 + m % 2 * 8;
      return join(down(at + columns[m / 2 % 2 * 2]), down(at + columns[m / 2 % 2 * 2 + 1] + 512));
    } else {
      f32x4 f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[i] = lds_read<float>(panels + columns[(m % 2 ^ i / 2) * 2 + kt % 2] + m / 2 * kPanel + kt * 2048 + i * 128);
      return f;
    }
  }
  // Column 16 m + l.
  __device__ __forceinline__ frag ordered_column(unsigned panels, int m, int kt) const {
    if constexpr (kHalf) {
      const unsigned at = panels + m / 4 * kPanel + kt * 4096;
      return join(down(at + ordered[m % 4 * 2]), down(at + ordered[m % 4 * 2 + 1] + 512));
    } else {
      return column(panels, m, kt);
    }
  }
  // Four values down a column. The 16 lanes of a group read 4 rows of 4 pieces of 8 bytes; lane l gets value
  // l % 4 of piece l / 4 of each.
  __device__ __forceinline__ static s16x4 down(unsigned at) {
    using lds_vec = __attribute__((address_space(3))) s16x4*;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_vec>(static_cast<uintptr_t>(at)));
  }
  __device__ __forceinline__ static frag join(s16x4 a, s16x4 b) {
    union {
      s16x4 part[2];
      frag whole;
    } u;
    u.part[0] = a;
    u.part[1] = b;
    return u.whole;
  }
};

// The same for one tile that the wave has as its own (rows 16 tile + l, columns 16 tile + l of the panels).
template <typename T>
struct Own {
  using frag = typename Chunk<T>::frag;
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kPanel = Chunk<T>::kPanel;
  unsigned rows[2], columns[kHalf ? 2 : 4], place;

  __device__ __forceinline__ explicit Own(int tile, int thread = threadIdx.x) {
    const int l = thread & 15, g = (thread >> 4) & 3, r = tile * 16 + l;
#pragma unroll
    for (int x = 0; x < 2; ++x) rows[x] = r * 128 + (((x * 4 + g) ^ swizzle(r)) << 4);
    // Of the first four values of a lane's (tile 0 of 16, four a lane group).
    const int at = g * 4 * sizeof(T);
    place = r * 128 + (((at >> 4) ^ swizzle(r)) << 4) + at % 16;
    if constexpr (kHalf) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = g * 8 + x * 4 + (l >> 2);
        columns[x] = tile / 4 * kPanel + row * 128 + (((tile % 4 * 2 + (l >> 1 & 1)) ^ swizzle(row)) << 4) + (l & 1) * 8;
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) {  // second rows, odd steps
        const int row = x % 2 * 16 + g * 4 + x / 2 * 2;
        columns[x] = tile / 2 * kPanel + g * 512 + (((tile % 2 * 4 + (l >> 2)) ^ swizzle(row)) << 4) + (l & 3) * 4;
      }
    }
  }
  __device__ __forceinline__ Own moved(unsigned by) const {
    Own r = *this;
    for (unsigned& at : r.rows) at += by;
    for (unsigned& at : r.columns) at += by;
    r.place += by;
    return r;
  }
  __device__ __forceinline__ frag row(unsigned panels, int ks) const {
    return lds_read<frag>(panels + rows[ks % 2] + ks / 2 * kPanel);
  }
  // Values 16 m + 4 g to 16 m + 4 g + 3 of the lane's row.
  __device__ __forceinline__ f32x4 four(unsigned panels, int m) const {
    constexpr int kTilePieces = sizeof(T);  // 16-byte pieces of 16 values
    const Four<T> v = lds_read<Four<T>>(panels + (place ^ (m * kTilePieces % 8 << 4)) + m * kTilePieces / 8 * kPanel);
    return f32x4{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]), static_cast<float>(v[3])};
  }
  __device__ __forceinline__ frag column(unsigned panels, int kt) const {
    if constexpr (kHalf) {
      return Reader<T>::join(Reader<T>::down(panels + columns[0] + kt * 4096), Reader<T>::down(panels + columns[1] + kt * 4096));
    } else {
      f32x4 f;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = lds_read<float>(panels + columns[i / 2 * 2 + kt % 2] + kt * 2048 + i * 128);
      return f;
    }
  }
  // The column at the rows of result tile m.
  __device__ __forceinline__ f32x4 values(unsigned panels, int m) const {
    if constexpr (kHalf) {
      const Four<T> s = __builtin_bit_cast(Four<T>, Reader<T>::down(panels + columns[m % 2] + m / 2 * 4096));
      return f32x4{static_cast<float>(s[0]), static_cast<float>(s[1]), static_cast<float>(s[2]), static_cast<float>(s[3])};
    } else {
      return column(panels, m);
    }
  }
};

// The second terms of float16 values are kept 2^11 times as large, in sums of their own: as they are, those of
// values below 0.1 would end in the type's fixed-point range (states 1.4e-5 off where bfloat16's are 4e-6).
template <typename T>
constexpr float kRestScale = std::is_same_v<T, _Float16> ? 2048.f : 1.f;

// A sum of products, and that of their second terms.
template <typename T>
struct Sum {
  f32x4 whole;
  f32x4 rest = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ explicit Sum(f32x4 from = {0.f, 0.f, 0.f, 0.f}) : whole(from) {}
  __device__ __forceinline__ void add(typename Chunk<T>::frag a, typename Chunk<T>::frag b, bool second) {
    if (second && kRestScale<T> != 1.f)
      rest = Fragment<T>::mma(a, b, rest);
    else
      whole = Fragment<T>::mma(a, b, whole);
  }
  __device__ __forceinline__ f32x4 value() const {
    return kRestScale<T> != 1.f ? whole + rest * (1.f / kRestScale<T>) : whole;
  }
};

// Four values rounded. They are rounded once for every use: the compiler would otherwise take float16 values
// for the product from one instruction and for the difference from another (a fused multiply-add that rounds
// once where the first rounds twice), and a last place between the two would be lost.
template <typename T>
__device__ __forceinline__ Four<T> nearest(const f32x4& v) {
  Four<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = static_cast<T>(v[i]);
  if constexpr (sizeof(T) == 2) {
    typedef unsigned Words __attribute__((ext_vector_type(2)));
    Words w = __builtin_bit_cast(Words, r);
    asm("" : "+v"(w));
    r = __builtin_bit_cast(Four<T>, w);
  }
  return r;
}
// What rounding left, as the second terms have it.
template <typename T>
__device__ __forceinline__ f32x4 rest_of(const f32x4& v, const Four<T>& rounded) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (v[i] - static_cast<float>(rounded[i])) * kRestScale<T>;
  return r;
}

// kPer result tiles as a fragment: the nearest values, and (16 bits) what they leave.
template <typename T, int TERMS>
__device__ __forceinline__ void split(const f32x4* tiles, typename Chunk<T>::frag (&out)[TERMS]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Four<T> hi = nearest<T>(tiles[i]);
      Four<T> lo;
      if constexpr (TERMS > 1) lo = nearest<T>(rest_of<T>(tiles[i], hi));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        out[0][i * 4 + e] = hi[e];
        if constexpr (TERMS > 1) out[1][i * 4 + e] = lo[e];
      }
    }
  } else {
    out[0] = tiles[0];
  }
}

// Types whose range is less than that of their sums: their operands are scaled.
template <typename T>
constexpr bool kUnits = std::is_same_v<T, _Float16>;

// A power of two that brings values within float16's range before they are split, and its inverse, which goes to
// the sums of their products; one beside other types, which have float's range. Factors of rows make it needed: a key
// near zero has 1 / |k| of up to 1000 (of its unit length), so that what its token brings leaves the range where the
// product with the key is small. With the largest value from 2^14 on, what is 2^-27 of it keeps 11 bits.
template <typename T>
struct Power {
  float up = 1.f, down = 1.f;
  __device__ __forceinline__ explicit Power(float largest) {
    if constexpr (kUnits<T>) {
      // Bounded, so that states that are multiplied by it too, as they join the sums, stay within float's range.
      const int exponent = std::max(__builtin_amdgcn_frexp_expf(largest), -40);
      up = __builtin_bit_cast(float, (127 + 15 - exponent) << 23);
      down = __builtin_bit_cast(float, (127 - 15 + exponent) << 23);
    }
  }
};
// The largest size of N result tiles' values in this lane, and that over a column's lanes, 16 and 32 apart (not looked
// for beside other types).
template <typename T, int N>
__device__ __forceinline__ float largest_size(const f32x4* tiles, float most = 0.f) {
  if constexpr (kUnits<T>) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(tiles[i][e]));
  }
  return most;
}
__device__ __forceinline__ float largest_of_groups(float most) {
  unsigned v = __builtin_bit_cast(unsigned, most);  // as float: none is negative or NaN
  const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = std::max<unsigned>(rows[0], rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_bit_cast(float, std::max<unsigned>(halves[0], halves[1]));
}
template <typename T>
__device__ __forceinline__ float over_lane_groups(float most) {
  return kUnits<T> ? largest_of_groups(most) : most;
}
// Over all lanes.
__device__ __forceinline__ float lanes_largest(float most) {
  most = fmaxf(most, dpp_read<0xb1>(most));
  most = fmaxf(most, dpp_read<0x4e>(most));
  most = fmaxf(most, dpp_read<0x141>(most));
  most = fmaxf(most, dpp_read<0x140>(most));
  return largest_of_groups(most);
}

// What is kept of float16 for a backward, one term each, is in units of its head's largest value (S and U: of the
// values and the first state) or gradient (D and Y: of the outputs' and the last state's), a power of two that takes
// it into 4 to 8. As they are, D's values, a hundredth of the gradients or less, would end in the type's fixed-point
// range while those are normal numbers (gradients of 1e-5: those of beta 4% off), and sums of large ones past it.
__device__ __forceinline__ float unit_of(const DeltaArgs& a, int64_t bh) {
  const int lane = threadIdx.x & 63;
  const float most = lanes_largest(lane < a.parts ? a.largest[bh * a.parts + lane] : 0.f);
  // Bounded, so that the two units' product and its inverse stay within float's range.
  const int exponent = most > 0.f ? std::min(std::max(__builtin_amdgcn_frexp_expf(most), -40), 60) : 3;
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane((127 + 3 - exponent) << 23));
}
// Both terms of a fragment as one in `unit`.
template <typename T, int TERMS>
__device__ __forceinline__ typename Chunk<T>::frag in_unit(const typename Chunk<T>::frag (&terms)[TERMS], float unit) {
  if constexpr (!kUnits<T>) {
    return terms[0];
  } else {
    typename Chunk<T>::frag r;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r[e] = static_cast<T>(fmaf(static_cast<float>(terms[1][e]), 1.f / kRestScale<T>, static_cast<float>(terms[0][e])) * unit);
    return r;
  }
}

__device__ __forceinline__ u32x4 buffer_at(const void* p) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(at));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(at >> 32) & 0xffffu);
  r[2] = kNowhere;
  r[3] = 0x00020000u;
  return r;
}

// Loads panels of kTokens rows into LDS: `count` panels of 128 bytes from `column` on of rows `stride`
// bytes apart; zeros past `rows` rows and `bytes` bytes of a row. Waves take turns from wave `turn` on.
template <typename T>
__device__ __forceinline__ void load_panels(u32x4 buffer, unsigned dst, int count, unsigned column,
                                            unsigned stride, int rows, unsigned bytes, int wave, int waves) {
  constexpr int kLoads = Chunk<T>::kTokens / 8;
  const int lane = threadIdx.x & 63;
  for (int i = wave; i < count * kLoads; i += waves) {
    const int panel = i / kLoads, row = i % kLoads * 8 + lane / 8;
    const unsigned at = column + panel * 128 + (((lane % 8) ^ swizzle(row)) << 4);
    load_lds16(buffer, dst + i * 1024,
               row < rows && at < bytes ? static_cast<unsigned>(row) * stride + at : kNowhere);
  }
}
// The same with the lane's places made once, for a walk over chunks: COUNT panels by W waves.
template <typename T, int COUNT, int W>
struct PanelLoads {
  static constexpr int kLoads = Chunk<T>::kTokens / 8, kAll = COUNT * kLoads, kMine = (kAll + W - 1) / W;
  static_assert(kAll % W == 0 || kAll < W, "as many loads a wave, or one of some");
  unsigned offset[kMine];
  __device__ __forceinline__ static int row(int j, int wave) {
    return (j * W + wave) % kLoads * 8 + static_cast<int>(threadIdx.x & 63) / 8;
  }
  __device__ __forceinline__ PanelLoads(unsigned column, unsigned stride, unsigned bytes, int wave) {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int r = row(j, wave);
      const unsigned at = column + (j * W + wave) / kLoads * 128 + (((threadIdx.x % 8) ^ swizzle(r)) << 4);
      offset[j] = at < bytes ? static_cast<unsigned>(r) * stride + at : kNowhere;
    }
  }
  // Lower triangles that lie in memory one after another, without the quarter that no fragment reaches.
  __device__ __forceinline__ explicit PanelLoads(int wave) {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int r = row(j, wave), piece = (threadIdx.x % 8) ^ swizzle(r);
      offset[j] = r < Chunk<T>::kTokens / 2 && piece >= 4
                      ? kNowhere
                      : (j * W + wave) * 1024 + (threadIdx.x & 63) / 8 * 128 + (piece << 4);
    }
  }
  __device__ __forceinline__ void load(u32x4 buffer, unsigned dst, int wave, int rows) const {
    if (kAll < W && wave >= kAll) return;
    if (rows == Chunk<T>::kTokens) {
#pragma unroll
      for (int j = 0; j < kMine; ++j) load_lds16(buffer, dst + (j * W + wave) * 1024, offset[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kMine; ++j)
        load_lds16(buffer, dst + (j * W + wave) * 1024, row(j, wave) < rows ? offset[j] : kNowhere);
    }
  }
};

// Waits for loads with COUNT or more after them.
template <int COUNT>
__device__ __forceinline__ void wait_older_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory");
}

constexpr int kTurnPitch = 20;  // elements of a row of 16 columns

// Tokens of sequence b that count.
__device__ __forceinline__ int length_of(const DeltaArgs& a, int b) {
  if (a.lengths == nullptr) return static_cast<int>(a.tokens);
  const int64_t n = a.wide_lengths ? static_cast<const int64_t*>(a.lengths)[b]
                                   : static_cast<const int32_t*>(a.lengths)[b];
  return static_cast<int>(n < 0 ? 0 : n > a.tokens ? a.tokens : n);
}

// Up to four neighbouring values.
template <typename T>
__device__ __forceinline__ void store_four(T* p, const f32x4& v, int count) {
  Run<T, 4> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.v[e] = static_cast<T>(v[e]);
  if (count >= 4) {
    store_run<4>(p, r);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) p[e] = r.v[e];
    end_of_part();
  }
}

template <typename T>
__device__ __forceinline__ const T* at_token(const void* p, const DeltaStrides& s, int64_t batch, int64_t token,
                                             int64_t head) {
  return static_cast<const T*>(p) + batch * s.batch + token * s.token + head * s.head;
}

// A chunk's record beside its panels: factors of rows in float (one value a token each), the sums of
// decays in 64 bits, and a bit for each closed token.
template <typename T>
struct Record {
  static constexpr int kTokens = Chunk<T>::kTokens;
  float state_to_value[kTokens];  // beta c rk: what a row of K S takes from its value
  float beta[kTokens];
  float value_to_state[kTokens];  // e rk
  float state_to_output[kTokens];  // c rq
  float whole;                     // c of the last token
  float unit;                      // of the S and U that are kept
  float unused[2];
  float rk[kTokens];
  float rq[kTokens];
  float norm[kTokens];            // rq without the scale
  double sum[kTokens];
  uint64_t closed;
  uint64_t filler;
};

// ---- T, P and the factors of every chunk ----------------------------------------------------------

// exp of the decays between tokens j and i > j, none of them closed.
__device__ __forceinline__ bool open_between(uint64_t closed, int j, int i) {
  // Bits j + 1 .. i.
  return ((closed >> 1 >> j) & ((uint64_t{1} << (i - j)) - 1)) == 0;
}
__device__ __forceinline__ float decay_between(double later, double earlier) {
  return __builtin_amdgcn_exp2f(static_cast<float>(later - earlier) * 1.44269504088896341f);
}

// Bound by memory and the latency of its short steps, four workgroups a compute unit: 34 us for 2048 chunks of
// 128-wide heads, 64 KB each (4 TB/s). A workgroup takes a chunk of a key head and its value heads one after
// another; wave w makes rows 16 w
// to 16 w + 15. k.k and q.k are in registers for all heads. T: each wave inverts its 16 x 16 block of I
// + A by substitution, then makes its row of blocks from the right, T_ij = -(sum_k T_ik A_kj) T_jj, on
// the float matrix instructions, transposed so that a result is the next product's operand and a lane's
// four values neighbours in a row.
template <typename T, int DK>
__global__ __launch_bounds__(Chunk<T>::kTokens * 4, 4) void delta_prepare(DeltaArgs a) {
  using C = Chunk<T>;
  using frag = typename C::frag;
  constexpr int kTokens = C::kTokens, kTiles = C::kTiles, kPanels = DK / kTokens;
  constexpr int kSteps = DK / C::kStep;
  constexpr int kPitch = kTokens + 4, kBlockPitch = 20;
  __shared__ __align__(1024) union {
    unsigned char operands[2][kPanels * C::kPanel];
    struct {
      float rest[kTokens][kPitch];                // A transposed
      float block[kTiles][16][kBlockPitch];       // the diagonal blocks' inverses, transposed
    } solve;
  } lds;
  __shared__ float rk[kTokens], rq[kTokens], norm[kTokens], beta[kTokens];
  __shared__ double sum[kTokens];
  const Lane lane;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned row = blockIdx.x / static_cast<unsigned>(a.chunks);
  const int chunk = static_cast<int>(blockIdx.x - row * static_cast<unsigned>(a.chunks));
  const int b = static_cast<int>(row / static_cast<unsigned>(a.key_heads));
  const int kh = static_cast<int>(row) - b * static_cast<int>(a.key_heads);
  const int length = length_of(a, b), t0 = chunk * kTokens;
  if (t0 >= length) return;
  const int rows = length - t0 < kTokens ? length - t0 : kTokens;
  {
    const unsigned bytes = static_cast<unsigned>(a.key_size * sizeof(T));
    const u32x4 k = buffer_at(at_token<T>(a.key, a.key_strides, b, t0, kh));
    const u32x4 q = buffer_at(at_token<T>(a.query, a.query_strides, b, t0, kh));
    load_panels<T>(k, lds_address(lds.operands[0]), kPanels, 0,
                   static_cast<unsigned>(a.key_strides.token * sizeof(T)), rows, bytes, wave, kTiles);
    load_panels<T>(q, lds_address(lds.operands[1]), kPanels, 0,
                   static_cast<unsigned>(a.query_strides.token * sizeof(T)), rows, bytes, wave, kTiles);
    wait_loads();
    __syncthreads();
  }
  {
    // Four threads a row.
    float ss[2] = {1.f, 1.f};
    const int r = threadIdx.x / 4;
    if (a.normalize) {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        float s = 0.f;
        for (int c = threadIdx.x % 4; c < kPanels * 8; c += 4) {
          const frag f = *reinterpret_cast<const frag*>(lds.operands[o] + c / 8 * C::kPanel + r * 128 + c % 8 * 16);
#pragma unroll
          for (int i = 0; i < 16 / int(sizeof(T)); ++i) {
            const float v = static_cast<float>(f[i]);
            s = fmaf(v, v, s);
          }
        }
        s += dpp_read<0xb1>(s);
        s += dpp_read<0x4e>(s);
        ss[o] = 1.f / sqrtf(s + kNormEps);
      }
    }
    if (threadIdx.x % 4 == 0) {
      rk[r] = ss[0];
      rq[r] = ss[1] * a.scale;
      norm[r] = ss[1];
    }
  }
  const Reader<T> read;
  const Own<T> own(wave);
  const unsigned keys = lds_address(lds.operands[0]), queries = lds_address(lds.operands[1]);
  f32x4 kk[kTiles], qk[kTiles];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) kk[j] = qk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < kSteps; ++ks) {
    const frag own_k = own.row(keys, ks), own_q = own.row(queries, ks);
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      if (j > wave) continue;
      const frag k = read.row(keys, j, ks);
      kk[j] = Fragment<T>::mma(own_k, k, kk[j]);  // registers rows of this wave, lanes columns
      qk[j] = Fragment<T>::mma(k, own_q, qk[j]);  // registers columns, lanes rows of this wave
    }
  }
  const int groups = a.groups;
  for (int group = 0; group < groups; ++group) {
    const int h = kh * groups + group;
    int l = lane.l, g = lane.g;
    asm volatile("" : "+v"(l), "+v"(g));  // what follows from them is made again for each head
    const int64_t at = (static_cast<int64_t>(b) * a.heads + h) * a.chunks + chunk;
    // Every wave adds the decays up; the first one keeps them for the rows' use.
    const int token = threadIdx.x & 63;
    float decay = 0.f, factor = 0.f;
    if (token < rows) {
      const int64_t d = b * a.decay_strides.batch + (t0 + token) * a.decay_strides.token + h * a.decay_strides.head;
      const int64_t f = b * a.beta_strides.batch + (t0 + token) * a.beta_strides.token + h * a.beta_strides.head;
      if (a.float_gates) {
        decay = static_cast<const float*>(a.decay)[d];
        factor = static_cast<const float*>(a.beta)[f];
      } else {
        decay = static_cast<float>(static_cast<const T*>(a.decay)[d]);
        factor = static_cast<float>(static_cast<const T*>(a.beta)[f]);
      }
    }
    const bool shut = decay < kDeltaClosed;
    const uint64_t closed = __ballot(shut);
    double total = shut ? 0. : static_cast<double>(decay);
#pragma unroll
    for (int step = 1; step < kTokens; step *= 2) {
      const double before = __shfl_up(total, step);
      if (token >= step) total += before;
    }
    const double last = __shfl(total, kTokens - 1);
    float unit = 1.f;
    if constexpr (kUnits<T>)
      if (wave == 0 && a.largest != nullptr) unit = unit_of(a, static_cast<int64_t>(b) * a.heads + h);
    __syncthreads();  // rk and rq are there; the head before has read what follows
    if (wave == 0 && token < kTokens) {
      sum[token] = total;
      beta[token] = factor;
      Record<T>* r = reinterpret_cast<Record<T>*>(a.records) + at;
      const float c = (closed & (~uint64_t{0} >> (63 - token))) == 0 ? decay_between(total, 0.) : 0.f;
      const float e = open_between(closed, token, kTokens - 1) ? decay_between(last, total) : 0.f;
      r->state_to_value[token] = factor * c * rk[token];
      r->beta[token] = factor;
      r->value_to_state[token] = e * rk[token];
      r->state_to_output[token] = c * rq[token];
      r->rk[token] = rk[token];
      r->rq[token] = rq[token];
      r->norm[token] = norm[token];
      r->sum[token] = total;
      if (token == kTokens - 1) {
        r->closed = closed;
        r->whole = c;
        r->unit = unit;
      }
    }
    __syncthreads();
    T* panels = reinterpret_cast<T*>(a.panels + at * (2 * C::kTerms * C::kPanel));
    {
      // A, transposed: lane's column j, four rows of this wave.
      double later[4];
      float up[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = wave * 16 + g * 4 + e;
        later[e] = sum[i];
        up[e] = beta[i] * rk[i];
      }
#pragma unroll
      for (int jb = 0; jb < kTiles; ++jb) {
        if (jb > wave) continue;
        const int j = jb * 16 + l;
        const double earlier = sum[j];
        const float own_rk = rk[j];
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = wave * 16 + g * 4 + e;
          const float pair = up[e] * own_rk * decay_between(later[e], earlier) * kk[jb][e];
          v[e] = i > j ? pair : 0.f;
        }
        if (closed != 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = wave * 16 + g * 4 + e;
            if (i > j && !open_between(closed, j, i)) v[e] = 0.f;
          }
        }
        *reinterpret_cast<f32x4*>(&lds.solve.rest[j][wave * 16 + g * 4]) = v;
      }
    }
    {
      // P: lane's row i, four columns; blocks past the diagonal as far as a fragment reaches.
      const int i = wave * 16 + l;
      const double later = sum[i];
      const float own_rq = rq[i];
      T* p = panels + C::kTerms * kTokens * kTokens + i * kTokens + g * 4;
#pragma unroll
      for (int jb = 0; jb < kTiles; ++jb) {
        if (jb / C::kPer > wave / C::kPer) continue;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = jb * 16 + g * 4 + e;
          const float pair = own_rq * rk[j] * decay_between(later, sum[j]) * qk[jb][e];
          v[e] = i >= j ? pair : 0.f;
        }
        if (closed != 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = jb * 16 + g * 4 + e;
            if (i >= j && !open_between(closed, j, i)) v[e] = 0.f;
          }
        }
#pragma unroll
        for (int term = 0; term < C::kTerms; ++term) {
          const Four<T> hi = nearest<T>(v);
          *reinterpret_cast<Four<T>*>(p + term * kTokens * kTokens + jb * 16) = hi;
          v = rest_of<T>(v, hi);
        }
      }
    }
    __syncthreads();
    {
      // Column l of the inverse of this wave's diagonal block, x = e_l - (A - its diagonal) x.
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = i == l ? 1.f : 0.f;
#pragma unroll
      for (int k = 0; k < 15; ++k) {
        const float* column = &lds.solve.rest[wave * 16 + k][wave * 16];
#pragma unroll
        for (int i = k + 1; i < 16; ++i) x[i] = fmaf(-column[i], x[k], x[i]);
      }
      if (g == 0) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<f32x4*>(&lds.solve.block[wave][l][i]) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
      }
    }
    __syncthreads();
    {
      f32x4 t[kTiles];  // T_ij transposed: registers columns, lanes rows
#pragma unroll
      for (int j = kTiles - 1; j >= 0; --j) {
        if (j > wave) {
          t[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else if (j == wave) {
#pragma unroll
          for (int e = 0; e < 4; ++e) t[j][e] = lds.solve.block[wave][g * 4 + e][l];
        } else {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = j + 1; k < kTiles; ++k) {
            if (k > wave) continue;
            const f32x4 f = *reinterpret_cast<const f32x4*>(&lds.solve.rest[j * 16 + l][k * 16 + g * 4]);
            acc = Fragment<float>::mma(f, t[k], acc);
          }
          const f32x4 d = *reinterpret_cast<const f32x4*>(&lds.solve.block[j][l][g * 4]);
          t[j] = Fragment<float>::mma(-d, acc, f32x4{0.f, 0.f, 0.f, 0.f});
        }
      }
      T* p = panels + (wave * 16 + l) * kTokens + g * 4;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        if (j / C::kPer > wave / C::kPer) continue;
#pragma unroll
        for (int term = 0; term < C::kTerms; ++term) {
          const Four<T> hi = nearest<T>(t[j]);
          *reinterpret_cast<Four<T>*>(p + term * kTokens * kTokens + j * 16) = hi;
          t[j] = rest_of<T>(t[j], hi);
        }
      }
    }
  }
}

// ---- the walk over the chunks ------------------------------------------------------------------------

// Where a workgroup of a walk is: `columns` values of a head (or columns of the unit matrix) and a segment of its
// chunks. Workgroups of a head are a whole number of heads apart: where that is a multiple of eight they run on
// one XCD and share its L2.
struct WalkPlace {
  int64_t bh;
  int b, h, kh, v0, segment;
  bool unit;
  __device__ __forceinline__ WalkPlace(const DeltaArgs& a, int columns, int units) {
    const unsigned heads = static_cast<unsigned>(a.batch * a.heads), group = blockIdx.x / heads;
    bh = blockIdx.x - group * heads;
    b = static_cast<int>(static_cast<unsigned>(bh) / static_cast<unsigned>(a.heads));
    h = static_cast<int>(bh) - b * static_cast<int>(a.heads);
    kh = h / a.groups;
    const int tiles = (static_cast<int>(a.value_size) + columns - 1) / columns, all = tiles + units / columns;
    segment = static_cast<int>(group) / all;
    const int tile = static_cast<int>(group) - segment * all;
    unit = tile >= tiles;
    v0 = (unit ? tile - tiles : tile) * columns;
  }
};

// Block i of a lower triangle of tiles by steps of a fragment, its first steps before its second ones.
template <typename T>
struct Triangle {
  static constexpr int kTiles = Chunk<T>::kTiles, kPer = Chunk<T>::kPer, kBlocks = 2 * kTiles - kPer;
  int tile, step;
  __device__ __forceinline__ explicit Triangle(int i)
      : tile(i < kTiles ? i : i - kTiles + kPer), step(i < kTiles ? 0 : 1) {}
};
// Reads of LDS and matrix instructions stay in the order written; arithmetic and stores may move. Left to
// itself the compiler reads each fragment right before its product (a chunk took 8 us, and with this 4).
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x2 | 0x4 | 0x40); }
constexpr int kAhead = 10;  // of the 15 that may be under way

// LDS of the walks forward: Q (and, where both do not fit twice, T and P) once, the other panels of a chunk twice,
// and what a wave of states hands to its wave of outputs.
template <typename T, int DK, int W, bool OUTPUTS>
struct Walk {
  using C = Chunk<T>;
  static constexpr bool kTwice = W == 2 || !OUTPUTS;  // T and P
  static constexpr int kKeyBytes = DK / C::kTokens * C::kPanel, kPairBytes = C::kTerms * C::kPanel;
  static constexpr int kValuePanels = (W * 16 + C::kTokens - 1) / C::kTokens;
  // Once.
  static constexpr int kQuery = 0;
  static constexpr int kSolveOnce = kQuery + (OUTPUTS ? kKeyBytes : 0);
  static constexpr int kPairsOnce = kSolveOnce + (kTwice ? 0 : kPairBytes);
  static constexpr int kStages = kPairsOnce + (kTwice ? 0 : kPairBytes);
  // In a stage.
  static constexpr int kKeys = 0;
  static constexpr int kSolve = kKeys + kKeyBytes;
  static constexpr int kPairs = kSolve + (kTwice ? kPairBytes : 0);
  static constexpr int kValues = kPairs + (kTwice && OUTPUTS ? kPairBytes : 0);
  static constexpr int kFactors = kValues + kValuePanels * C::kPanel;
  static constexpr int kStage = kFactors + 2048;
  // Handed on, for each wave: fragments of S and of U.
  static constexpr int kState = kStages + 2 * kStage;
  static constexpr int kStateBytes = DK / C::kStep * C::kTerms * 1024, kUpdateBytes = 2 * C::kTerms * 1024;
  static constexpr int kUpdate = kState + W * kStateBytes;
  static constexpr int kBytes = OUTPUTS ? kUpdate + W * kUpdateBytes : kState;
  static_assert(W * 16 % C::kTokens == 0 || C::kTokens % (W * 16) == 0, "whole panels of values, or parts of one");
  static_assert(kFactors <= 65536 && kStages <= 65536 && kBytes <= 163840, "constants of reads, and LDS");
};

// Two waves share 16 columns. One keeps S in registers, as results [key, column] of the products that update it,
// and walks through all of them by itself: K S, T R and K^T U take its columns' values as one operand straight
// from the results before (operand_row puts them in order) and the shared panels as the other, from LDS. The
// other wave makes the outputs: while the first is at K S and T R it multiplies the S before the chunk, which it
// is handed through LDS, with Q, and while the first updates S, P with U; it also loads, and stores outputs and what
// is kept for a backward behind the next chunk's loads. Waves meet twice a chunk; panels load a chunk or half of one
// ahead. With few heads (W = 2) it is bound by the chain from S to the next S: 2.9 us a chunk of 64 tokens, where
// all in one wave took 3.9. With all compute units at work (W = 4) memory is near: 263 us for 4096 tokens of 128
// heads that keep S and U, 1.2 GB (4.6 TB/s); all in one wave 338.
template <typename T, int DK, int W, bool KEEP, bool TRANSIT>
__global__ __launch_bounds__(128 * W) __attribute__((amdgpu_waves_per_eu(W / 2, W / 2))) void delta_forward(DeltaArgs a) {
  using C = Chunk<T>;
  using frag = typename C::frag;
  using S = Walk<T, DK, W, !TRANSIT>;
  constexpr int kTokens = C::kTokens, kTiles = C::kTiles, kTerms = C::kTerms, kPer = C::kPer;
  constexpr int kSteps = DK / C::kStep, kStateTiles = DK / 16;
  constexpr bool kTwice = S::kTwice;
  extern __shared__ __align__(1024) unsigned char lds[];
  const Lane lane;
  const int thread = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % W;
  const WalkPlace w(a, W * 16, TRANSIT ? DK : 0);
  const int64_t bh = w.bh;
  const int b = w.b, h = w.h, kh = w.kh;
  const int value_size = static_cast<int>(a.value_size), key_size = static_cast<int>(a.key_size);
  const int v0 = w.v0, column = v0 + part * 16;  // of the workgroup and the wave
  const bool active = TRANSIT && w.unit ? true : column < value_size;
  const int mine = column + lane.l;
  const int length = length_of(a, b);
  const int all_chunks = (length + kTokens - 1) / kTokens;
  const int begin = w.segment * a.segment_chunks;
  const int end = all_chunks < begin + a.segment_chunks ? all_chunks : begin + a.segment_chunks;
  const int64_t first_chunk = bh * a.chunks, segment_at = bh * a.segments + w.segment;
  const unsigned lds_at = lds_address(lds);

  // Panels of values start at whole ones; the wave's columns lie within.
  const int from_panel = v0 % (S::kValuePanels * kTokens);
  const T* k_at = at_token<T>(a.key, a.key_strides, b, 0, kh);
  const T* q_at = at_token<T>(a.query, a.query_strides, b, 0, kh);
  const T* v_at = at_token<T>(a.value, a.value_strides, b, 0, h);
  const unsigned key_bytes = static_cast<unsigned>(key_size * sizeof(T));
  const PanelLoads<T, DK / kTokens, W> key_loads(0, static_cast<unsigned>(a.key_strides.token * sizeof(T)), key_bytes, part);
  const PanelLoads<T, DK / kTokens, W> query_loads(0, static_cast<unsigned>(a.query_strides.token * sizeof(T)), key_bytes, part);
  const PanelLoads<T, S::kValuePanels, W> value_loads(
      static_cast<unsigned>((v0 - from_panel) * sizeof(T)), static_cast<unsigned>(a.value_strides.token * sizeof(T)),
      TRANSIT && w.unit ? 0u : static_cast<unsigned>(value_size * sizeof(T)), part);
  const PanelLoads<T, kTerms, W> pair_loads(part);
  const auto rows_of = [&](int c) __attribute__((always_inline)) {
    const int64_t left = c < end ? length - static_cast<int64_t>(c) * kTokens : 0;
    return left < kTokens ? static_cast<int>(left) : kTokens;
  };
  const auto load_solve = [&](int c, unsigned dst) __attribute__((always_inline)) {
    pair_loads.load(buffer_at(a.panels + (first_chunk + c) * (2 * S::kPairBytes)), dst, part, c < end ? kTokens : 0);
  };
  const auto load_pairs = [&](int c, unsigned dst) __attribute__((always_inline)) {
    pair_loads.load(buffer_at(a.panels + (first_chunk + c) * (2 * S::kPairBytes) + S::kPairBytes), dst, part,
                    c < end ? kTokens : 0);
  };
  const auto load_query = [&](int c) __attribute__((always_inline)) {
    query_loads.load(buffer_at(q_at + static_cast<int64_t>(c) * kTokens * a.query_strides.token), lds_at + S::kQuery, part,
                     rows_of(c));
  };
  // As many loads whether there is a chunk or not, since waits count them (but the factors').
  constexpr int kStageLoads = (DK / kTokens + S::kValuePanels) * (kTokens / 8) / W;
  const auto load_stage = [&](int c) __attribute__((always_inline)) {
    const unsigned dst = lds_at + S::kStages + (c & 1) * S::kStage;
    const int64_t t0 = static_cast<int64_t>(c) * kTokens;
    const int rows = rows_of(c);
    key_loads.load(buffer_at(k_at + t0 * a.key_strides.token), dst + S::kKeys, part, rows);
    value_loads.load(buffer_at(v_at + t0 * a.value_strides.token), dst + S::kValues, part, rows);
    if constexpr (kTwice) {
      load_solve(c, dst + S::kSolve);
      if constexpr (!TRANSIT) load_pairs(c, dst + S::kPairs);
    }
    if (part < 2) {  // the factors, and after them `whole`
      const unsigned at = part * 16 * kTokens + thread * 16;
      load_lds16(buffer_at(reinterpret_cast<const Record<T>*>(a.records) + first_chunk + c),
                 dst + S::kFactors + part * 1024, c < end && at < (part == 0 ? 16 : 17) * kTokens ? at : kNowhere);
    }
  };
  if (wave >= W && begin < end) {  // the waves of outputs load
    load_stage(begin);
    if constexpr (!TRANSIT) load_query(begin);
    if constexpr (!kTwice) load_solve(begin, lds_at + S::kSolveOnce);
  }
  constexpr int kRows = kTiles * kSteps, kBlocks = Triangle<T>::kBlocks, kColumns = 2 * kStateTiles;
  const unsigned state_at = lds_at + S::kState + part * S::kStateBytes + thread * 16;
  const unsigned update_at = lds_at + S::kUpdate + part * S::kUpdateBytes + thread * 16;

  if (wave < W) {
    const Reader<T> places;
    const Own<T> own(from_panel / 16 + part);
    f32x4 state[kStateTiles];
#pragma unroll
    for (int m = 0; m < kStateTiles; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = first_row<T>(m, lane.g) + e;
        if constexpr (TRANSIT)
          state[m][e] = w.unit && d == mine ? 1.f : 0.f;
        else if (a.segments > 1)
          state[m][e] = active ? a.starts[(segment_at * DK + d) * a.value_pad + mine] : 0.f;
        else
          state[m][e] = a.first != nullptr && d < key_size && mine < value_size
                            ? a.first[(bh * key_size + d) * value_size + mine]
                            : 0.f;
      }
    frag s[kSteps][kTerms];
    const auto hand_state = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        split<T>(&state[ks * kPer], s[ks]);
        if constexpr (!TRANSIT) {
#pragma unroll
          for (int term = 0; term < kTerms; ++term) lds_write(state_at + (ks * kTerms + term) * 1024, s[ks][term]);
        }
      }
    };
    hand_state();
#pragma unroll 1
    for (int c = begin; c < end; ++c) {
      __syncthreads();  // the chunk is there, and the one before done with
      if (!active) {
        if constexpr (!TRANSIT) __syncthreads();
        continue;
      }
      const unsigned at = lds_at + S::kStages + (c & 1) * S::kStage;
      const Reader<T> read = places.moved(at);
      const Reader<T> solve_read = kTwice ? read : places.moved(lds_at);
      constexpr unsigned kSolve = kTwice ? S::kSolve : S::kSolveOnce;
      const float* factors = reinterpret_cast<const float*>(lds + S::kStages + (c & 1) * S::kStage + S::kFactors);
      const float whole = factors[256];
      // The chunk's fragments in the order of their products, read kAhead of them before: K, T, K^T.
      // Neighbouring products are of different sums, since one waits for the last of its own sum.
      frag kf[kRows], tf[kTerms * kBlocks], cf[kColumns];
      const auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i < kRows) {
          kf[i] = read.operand(S::kKeys, i % kTiles, i / kTiles);
        } else if ((i -= kRows) < kTerms * kBlocks) {
          const Triangle<T> b(i % kBlocks);
          tf[i] = solve_read.operand(kSolve + i / kBlocks * C::kPanel, b.tile, b.step);
        } else if ((i -= kTerms * kBlocks) < kColumns) {
          cf[i] = read.column(S::kKeys, i / 8 * 4 + i % 4, i / 4 % 2);
        }
      };
      constexpr int kFirstT = kRows, kFirstC = kFirstT + kTerms * kBlocks;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fetch(i);
      keep_order();

      // R = beta V - (beta c rk) K S.
      Sum<T> sums[kTiles];
#pragma unroll
      for (int i = 0; i < kRows; i += kTiles) {
#pragma unroll
        for (int m = 0; m < kTiles; ++m) fetch(i + m + kAhead);
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int m = 0; m < kTiles; ++m) sums[m].add(kf[i + m], s[i / kTiles][term], term > 0);
        keep_order();
      }
      f32x4 r[kTiles];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        const f32x4 acc = sums[m].value();
        const f32x4 v = own.values(at + S::kValues, m);
        const int row = first_row<T>(m, lane.g);
        const f32x4 take = *reinterpret_cast<const f32x4*>(factors + row);
        const f32x4 beta = *reinterpret_cast<const f32x4*>(factors + kTokens + row);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[m][e] = fmaf(beta[e], v[e], -take[e] * acc[e]);
        sums[m] = Sum<T>();
      }
      frag rf[2][kTerms], uf[2][kTerms], df[2][kTerms];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) split<T>(&r[kt * kPer], rf[kt]);
      // U = T R.
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) fetch(kFirstT + term * kBlocks + i + kAhead);
#pragma unroll
        for (int other = 0; other < kTerms - term; ++other)
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            const Triangle<T> b(i);
            sums[b.tile].add(tf[term * kBlocks + i], rf[b.step][other], term + other > 0);
          }
        keep_order();
      }
      f32x4 u[kTiles];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) u[m] = sums[m].value();
      if constexpr (!TRANSIT) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          split<T>(&u[kt * kPer], uf[kt]);
#pragma unroll
          for (int term = 0; term < kTerms; ++term) lds_write(update_at + (kt * kTerms + term) * 1024, uf[kt][term]);
        }
      }
      if constexpr (!TRANSIT) __syncthreads();  // U is handed on
      // S = c S + K^T (e rk U).
#pragma unroll
      for (int m = 0; m < kTiles; ++m) u[m] *= *reinterpret_cast<const f32x4*>(factors + 2 * kTokens + first_row<T>(m, lane.g));
      const Power<T> power(over_lane_groups<T>(largest_size<T, kTiles>(u)));
      const float faded = whole * power.up;
#pragma unroll
      for (int m = 0; m < kTiles; ++m) u[m] *= power.up;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) split<T>(&u[kt * kPer], df[kt]);
#pragma unroll
      for (int m0 = 0; m0 < kStateTiles; m0 += 4) {
        Sum<T> sum[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) sum[m].whole = state[m0 + m] * faded;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
          for (int m = 0; m < 4; ++m) fetch(kFirstC + m0 * 2 + kt * 4 + m + kAhead);
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int m = 0; m < 4; ++m) sum[m].add(cf[m0 * 2 + kt * 4 + m], df[kt][term], term > 0);
          keep_order();
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) state[m0 + m] = sum[m].value() * power.down;
      }
      hand_state();
    }
    if (!active) return;
    if (TRANSIT || a.segments == 1) {
#pragma unroll
      for (int m = 0; m < kStateTiles; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = first_row<T>(m, lane.g) + e;
          if constexpr (TRANSIT) {
            if (w.unit)
              a.transits[(segment_at * DK + d) * DK + mine] = state[m][e];
            else
              a.partials[(segment_at * DK + d) * a.value_pad + mine] = state[m][e];
          } else if (d < key_size && mine < value_size) {
            a.last[(bh * key_size + d) * value_size + mine] = state[m][e];
          }
        }
    }
    return;
  }

  if constexpr (TRANSIT) {
#pragma unroll 1
    for (int c = begin; c < end; ++c) {
      wait_loads();
      __syncthreads();
      load_stage(c + 1);
    }
    wait_loads();  // none into LDS that is another workgroup's by then
  } else {
    const Reader<T> places;
    const Reader<T> fixed = places.moved(lds_at);
    T* out = static_cast<T*>(a.output) + (static_cast<int64_t>(b) * a.tokens * a.heads + h) * value_size;
    const int64_t out_token = a.heads * value_size;
    const int store_at = column + lane.g * 4, store_count = value_size - store_at;
    const bool whole_rows = column + 16 <= value_size;
    unsigned out_place[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) out_place[n] = (n * 16 + lane.l) * static_cast<unsigned>(out_token) + store_at;
    const unsigned state_place = mine * DK + lane.g * (16 / sizeof(T));
    const unsigned update_place = mine * kTokens + lane.g * (16 / sizeof(T));
    // The wait for what was loaded is not for the stores after it, of which there are at least so many.
    constexpr int kKept = KEEP ? 2 + kSteps : 0;
    const float unit = KEEP && kUnits<T> ? unit_of(a, bh) : 1.f;
    bool all_stored = false;
#pragma unroll 1
    for (int c = begin; c < end; ++c) {
      if (c == begin)
        wait_loads();
      else if (all_stored)
        wait_older_loads<kTiles + kKept>();
      else if (active)
        wait_older_loads<kKept>();
      else
        wait_loads();
      __syncthreads();
      if constexpr (!kTwice) load_pairs(c, lds_at + S::kPairsOnce);
      load_stage(c + 1);
      frag s[kSteps][kTerms], qf[kRows];
      const auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i < kRows) qf[i] = fixed.row(S::kQuery, i % kTiles, i / kTiles);
      };
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
        for (int term = 0; term < kTerms; ++term) s[ks][term] = lds_read<frag>(state_at + (ks * kTerms + term) * 1024);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) fetch(i);
      keep_order();
      // O = c rq Q S + P U: its lanes are tokens and its registers columns.
      const float* factors = reinterpret_cast<const float*>(lds + S::kStages + (c & 1) * S::kStage + S::kFactors);
      Sum<T> o[kTiles];
#pragma unroll
      for (int i = 0; i < kRows; i += kTiles) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) fetch(i + n + kTiles);
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int n = 0; n < kTiles; ++n) o[n].add(s[i / kTiles][term], qf[i + n], term > 0);
        keep_order();
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const float factor = factors[3 * kTokens + n * 16 + lane.l];
        o[n].whole *= factor;
        o[n].rest *= factor;
      }
      if constexpr (!kTwice) wait_older_loads<kStageLoads>();  // P
      __syncthreads();
      load_query(c + 1);
      if constexpr (!kTwice) load_solve(c + 1, lds_at + S::kSolveOnce);
      if (!active) continue;
      asm volatile("" ::: "memory");  // the stores stay behind the loads
      const Reader<T> read = kTwice ? places.moved(lds_at + S::kStages + (c & 1) * S::kStage) : fixed;
      constexpr unsigned kPairs = kTwice ? S::kPairs : S::kPairsOnce;
      frag uf[2][kTerms], pf[kTerms * kBlocks];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int term = 0; term < kTerms; ++term) uf[kt][term] = lds_read<frag>(update_at + (kt * kTerms + term) * 1024);
#pragma unroll
      for (int i = 0; i < kTerms * kBlocks; ++i) {
        const Triangle<T> b(i % kBlocks);
        pf[i] = read.row(kPairs + i / kBlocks * C::kPanel, b.tile, b.step);
      }
#pragma unroll
      for (int term = 0; term < kTerms; ++term)
#pragma unroll
        for (int other = 0; other < kTerms - term; ++other)
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            const Triangle<T> b(i);
            o[b.tile].add(uf[b.step][other], pf[term * kBlocks + i], term + other > 0);
          }
      T* to = out + static_cast<int64_t>(c) * kTokens * out_token;
      all_stored = whole_rows && (c + 1) * kTokens <= a.tokens;
      if (all_stored) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) *reinterpret_cast<Run<T, 4>*>(to + out_place[n]) = __builtin_bit_cast(Run<T, 4>, nearest<T>(o[n].value()));
      } else {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          const Four<T> v = nearest<T>(o[n].value());
          if (static_cast<int64_t>(c) * kTokens + n * 16 + lane.l < a.tokens) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < store_count) to[out_place[n] + e] = v[e];
            end_of_part();
          }
        }
      }
      if constexpr (KEEP) {
        T* updates = static_cast<T*>(a.updates) + (first_chunk + c) * a.value_pad * kTokens;
        T* states = static_cast<T*>(a.states) + (first_chunk + c) * a.value_pad * DK;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) *reinterpret_cast<frag*>(updates + (update_place + kt * C::kStep)) = in_unit<T>(uf[kt], unit);
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) *reinterpret_cast<frag*>(states + (state_place + ks * C::kStep)) = in_unit<T>(s[ks], unit);
      }
    }
    wait_loads();  // none into LDS that is another workgroup's by then
    if (!active) return;
    // Tokens past the last chunk give zeros.
    const int64_t stop = a.tokens < int64_t{begin + a.segment_chunks} * kTokens
                             ? a.tokens
                             : int64_t{begin + a.segment_chunks} * kTokens;
    for (int64_t t = int64_t{end > begin ? end : begin} * kTokens + lane.l; t < stop; t += 16)
      if (store_count > 0) store_four(out + t * out_token + store_at, f32x4{0.f, 0.f, 0.f, 0.f}, store_count);
  }
}

// ---- segments of the chunks --------------------------------------------------------------------------------

// With few heads a walk over all chunks would leave most of the chip idle. What a segment of them makes of the
// state before it is linear, S' = M S + N: the walk without outputs gives N from a state of zeros and M's columns
// from those of the unit matrix (and no values), all segments side by side. Here they are put together, one after
// another in float32 for every state before a segment (REVERSE: from the last one, gradients), from which the
// walks of all segments then run side by side. A workgroup has 16 columns, a wave 16 rows. 16
// segments of 8 heads take 39 us, bound by the one's wait for the one before (with 32 rows a wave 45, and with loads
// two segments ahead of that 45 to 49). 32768 tokens in all take 0.3 ms, and in a single segment 1.9.
template <int DK, bool REVERSE>
__global__ __launch_bounds__(DK * 4) void delta_join(DeltaArgs a) {
  constexpr int kTiles = DK / 16;
  __shared__ f32x4 shared[2][kTiles][64];
  const int l = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3, at = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = wave * 16;
  const unsigned heads = static_cast<unsigned>(a.batch * a.heads), tile = blockIdx.x / heads;
  const int64_t bh = blockIdx.x - tile * heads;
  const int mine = static_cast<int>(tile) * 16 + l;
  const int value_size = static_cast<int>(a.value_size), key_size = static_cast<int>(a.key_size);
  const float* from = REVERSE ? a.grad_last : a.first;
  float* to = REVERSE ? a.grad_first : a.last;
  const float unit = REVERSE && a.largest != nullptr ? unit_of(a, bh) : 1.f;  // of gradients
  f32x4 state;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = first + g * 4 + e;
    state[e] = from != nullptr && d < key_size && mine < value_size ? from[(bh * key_size + d) * value_size + mine] * unit
                                                                    : 0.f;
  }
  // A segment's rows of M and its N, a segment ahead.
  f32x4 rows[kTiles], next;
  const auto load = [&](int s) __attribute__((always_inline)) {
    const int64_t segment = bh * a.segments + s;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      rows[t] = *reinterpret_cast<const f32x4*>(a.transits + (segment * DK + first + l) * DK + t * 16 + g * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) next[e] = a.partials[(segment * DK + first + g * 4 + e) * a.value_pad + mine];
  };
  load(REVERSE ? a.segments - 1 : 0);
#pragma unroll 1
  for (int i = 0; i < a.segments; ++i) {
    const int s = REVERSE ? a.segments - 1 - i : i;
    const int64_t segment = bh * a.segments + s;
    shared[i & 1][wave][at] = state;
#pragma unroll
    for (int e = 0; e < 4; ++e) a.starts[(segment * DK + first + g * 4 + e) * a.value_pad + mine] = state[e];
    __syncthreads();
    // A result's registers at a lane are an operand's of the same tile: rows 4 g to 4 g + 3 of a column.
    f32x4 part[2] = {next, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int t = 0; t < kTiles; ++t) part[t & 1] = Fragment<float>::mma(rows[t], shared[i & 1][t][at], part[t & 1]);
    state = part[0] + part[1];
    if (i + 1 < a.segments) load(REVERSE ? s - 1 : s + 1);
  }
  if (to == nullptr) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = first + g * 4 + e;
    if (d < key_size && mine < value_size) to[(bh * key_size + d) * value_size + mine] = state[e] / unit;
  }
}

// ---- the walk back ----------------------------------------------------------------------------------------

// With D the gradient of the state after a chunk and Y = T^T dU,
//
//   dU = P^T dO + diag(e rk) K D,  dV = diag(beta) Y
//   D' = c_C D + Q^T diag(c rq) dO - K^T diag(beta c rk) Y
//
// in the forward walk's form: of two waves with 16 columns one has D in registers, and walks from D to the next D,
// and the other makes P^T dO and Q^T dO, which do not need it, and stores. D and Y of every chunk are kept
// for delta_gradients. 3.5 us a chunk with few heads (all in one wave 4.4), 271 us where the forward takes 263 (350).
template <typename T, int DK, int W>
struct WalkBack {
  using C = Chunk<T>;
  static constexpr bool kTwice = W == 2;  // T and P
  static constexpr int kKeyBytes = DK / C::kTokens * C::kPanel, kPairBytes = C::kTerms * C::kPanel;
  static constexpr int kValuePanels = (W * 16 + C::kTokens - 1) / C::kTokens;
  // Once.
  static constexpr int kQuery = 0;
  static constexpr int kSolveOnce = kQuery + kKeyBytes;
  static constexpr int kPairsOnce = kSolveOnce + (kTwice ? 0 : kPairBytes);
  static constexpr int kStages = kPairsOnce + (kTwice ? 0 : kPairBytes);
  // In a stage.
  static constexpr int kKeys = 0;
  static constexpr int kSolve = kKeys + kKeyBytes;
  static constexpr int kPairs = kSolve + (kTwice ? kPairBytes : 0);
  static constexpr int kValues = kPairs + (kTwice ? kPairBytes : 0);
  static constexpr int kFactors = kValues + kValuePanels * C::kPanel;
  static constexpr int kStage = kFactors + 2048;
  // Handed on, for each pair of waves: what the chunk adds to D (then D itself), and P^T dO (then dV and Y).
  static constexpr int kAdded = kStages + 2 * kStage, kAddedBytes = DK / 16 * 1024;
  static constexpr int kToUpdate = kAdded + W * kAddedBytes;
  static constexpr int kTurnBytes = C::kTokens * kTurnPitch * int(sizeof(T)), kToUpdateBytes = kTurnBytes + 2048;
  static constexpr int kBytes = kToUpdate + W * kToUpdateBytes;
  static_assert(C::kTiles * 1024 <= kToUpdateBytes && DK / C::kStep * 1024 <= kAddedBytes, "in one's place");
  static_assert(kFactors <= 65536 && kStages <= 65536 && kBytes <= 163840, "constants of reads, and LDS");
};

template <typename T, int DK, int W, bool TRANSIT>
__global__ __launch_bounds__(128 * W) __attribute__((amdgpu_waves_per_eu(W / 2, W / 2))) void delta_backward(DeltaArgs a) {
  using C = Chunk<T>;
  using frag = typename C::frag;
  using S = WalkBack<T, DK, W>;
  constexpr int kTokens = C::kTokens, kTiles = C::kTiles, kTerms = C::kTerms, kPer = C::kPer;
  constexpr int kSteps = DK / C::kStep, kStateTiles = DK / 16;
  constexpr bool kTwice = S::kTwice;
  constexpr int kAheadBack = 6;  // of transposing reads, two instructions each
  constexpr int kRows = kTiles * kSteps, kBlocks = Triangle<T>::kBlocks, kColumns = 2 * kStateTiles;
  extern __shared__ __align__(1024) unsigned char lds[];
  const Lane lane;
  const int thread = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % W;
  const WalkPlace w(a, W * 16, TRANSIT ? DK : 0);
  const int64_t bh = w.bh;
  const int b = w.b, h = w.h, kh = w.kh;
  const int value_size = static_cast<int>(a.value_size), key_size = static_cast<int>(a.key_size);
  const int v0 = w.v0, column = v0 + part * 16;  // of the workgroup and the wave
  const bool active = TRANSIT && w.unit ? true : column < value_size;
  const int mine = column + lane.l;
  const int length = length_of(a, b);
  const int all_chunks = (length + kTokens - 1) / kTokens;
  const int begin = w.segment * a.segment_chunks;
  const int end = all_chunks < begin + a.segment_chunks ? all_chunks : begin + a.segment_chunks;
  const int64_t first_chunk = bh * a.chunks, segment_at = bh * a.segments + w.segment;
  const unsigned lds_at = lds_address(lds);
  // Panels of values start at whole ones; the wave's columns lie within.
  const int from_panel = v0 % (S::kValuePanels * kTokens);
  const unsigned added_at = lds_at + S::kAdded + part * S::kAddedBytes + thread * 16;
  const unsigned to_update = lds_at + S::kToUpdate + part * S::kToUpdateBytes;
  const unsigned update_at = to_update + S::kTurnBytes + thread * 16;

  const T* k_at = at_token<T>(a.key, a.key_strides, b, 0, kh);
  const T* q_at = at_token<T>(a.query, a.query_strides, b, 0, kh);
  const T* g_at = at_token<T>(a.grad_output, a.grad_strides, b, 0, h);
  const unsigned key_bytes = static_cast<unsigned>(key_size * sizeof(T));
  const PanelLoads<T, DK / kTokens, W> key_loads(0, static_cast<unsigned>(a.key_strides.token * sizeof(T)), key_bytes, part);
  const PanelLoads<T, DK / kTokens, W> query_loads(0, static_cast<unsigned>(a.query_strides.token * sizeof(T)), key_bytes, part);
  const PanelLoads<T, S::kValuePanels, W> value_loads(
      static_cast<unsigned>((v0 - from_panel) * sizeof(T)), static_cast<unsigned>(a.grad_strides.token * sizeof(T)),
      TRANSIT && w.unit ? 0u : static_cast<unsigned>(value_size * sizeof(T)), part);
  const PanelLoads<T, kTerms, W> pair_loads(part);
  // As many loads whether there is a chunk or not, since waits count them (but the factors').
  const auto rows_of = [&](int c) __attribute__((always_inline)) {
    const int64_t left = c >= begin ? length - static_cast<int64_t>(c) * kTokens : 0;
    return left < kTokens ? static_cast<int>(left) : kTokens;
  };
  const auto load_pair = [&](int c, int which, unsigned dst) __attribute__((always_inline)) {
    pair_loads.load(buffer_at(a.panels + (first_chunk + c) * (2 * S::kPairBytes) + which * S::kPairBytes), dst, part,
                    c >= begin ? kTokens : 0);
  };
  constexpr int kStageLoads = (DK / kTokens + S::kValuePanels) * (kTokens / 8) / W;
  const auto load_stage = [&](int c) __attribute__((always_inline)) {
    const unsigned dst = lds_at + S::kStages + (c & 1) * S::kStage;
    const int64_t t0 = static_cast<int64_t>(c) * kTokens;
    const int rows = rows_of(c);
    key_loads.load(buffer_at(k_at + t0 * a.key_strides.token), dst + S::kKeys, part, rows);
    value_loads.load(buffer_at(g_at + t0 * a.grad_strides.token), dst + S::kValues, part, rows);
    if constexpr (kTwice) {
      load_pair(c, 0, dst + S::kSolve);
      load_pair(c, 1, dst + S::kPairs);
    }
    if (part < 2) {  // the factors, and after them `whole`
      const unsigned at = part * 16 * kTokens + thread * 16;
      load_lds16(buffer_at(reinterpret_cast<const Record<T>*>(a.records) + first_chunk + c),
                 dst + S::kFactors + part * 1024, c >= begin && at < (part == 0 ? 16 : 17) * kTokens ? at : kNowhere);
    }
  };

  if (wave < W) {
    if (begin < end) load_stage(end - 1);
    const float unit = kUnits<T> ? unit_of(a, bh) : 1.f, to_whole = 1.f / unit;  // of D and Y
    const Reader<T> places;
    f32x4 state[kStateTiles];
#pragma unroll
    for (int m = 0; m < kStateTiles; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = first_row<T>(m, lane.g) + e;
        if constexpr (TRANSIT)
          state[m][e] = w.unit && d == mine ? 1.f : 0.f;
        else if (a.segments > 1)
          state[m][e] = active ? a.starts[(segment_at * DK + d) * a.value_pad + mine] : 0.f;
        else
          state[m][e] = a.grad_last != nullptr && d < key_size && mine < value_size
                            ? a.grad_last[(bh * key_size + d) * value_size + mine] * unit
                            : 0.f;
      }
    frag s[kSteps][kTerms];
    const auto hand_state = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        split<T>(&state[ks * kPer], s[ks]);
        if constexpr (!TRANSIT) lds_write(added_at + ks * 1024, s[ks][0]);
      }
    };
    hand_state();
#pragma unroll 1
    for (int c = end - 1; c >= begin; --c) {
      wait_loads();
      __syncthreads();  // the chunk is there, and the one before done with
      if constexpr (!kTwice) load_pair(c, 0, lds_at + S::kSolveOnce);
      load_stage(c - 1);
      if (!active) {
        if constexpr (!kTwice) wait_older_loads<kStageLoads>();
        __syncthreads();
        continue;
      }
      const unsigned at = lds_at + S::kStages + (c & 1) * S::kStage;
      const Reader<T> read = places.moved(at);
      const Reader<T> solve_read = kTwice ? read : places.moved(lds_at);
      constexpr unsigned kSolve = kTwice ? S::kSolve : S::kSolveOnce;
      const float* factors = reinterpret_cast<const float*>(lds + S::kStages + (c & 1) * S::kStage + S::kFactors);
      const float whole = factors[256];
      // dU = diag(e rk) K D + P^T dO, whose second part is handed.
      frag kf[kRows];
      const auto fetch_key = [&](int i) __attribute__((always_inline)) {
        if (i < kRows) kf[i] = read.operand(S::kKeys, i % kTiles, i / kTiles);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fetch_key(i);
      keep_order();
      Sum<T> sums[kTiles];
#pragma unroll
      for (int i = 0; i < kRows; i += kTiles) {
#pragma unroll
        for (int m = 0; m < kTiles; ++m) fetch_key(i + m + kAhead);
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int m = 0; m < kTiles; ++m) sums[m].add(kf[i + m], s[i / kTiles][term], term > 0);
        keep_order();
      }
      f32x4 y[kTiles];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        y[m] = sums[m].value() * *reinterpret_cast<const f32x4*>(factors + 2 * kTokens + first_row<T>(m, lane.g));
        sums[m] = Sum<T>();
      }
      if constexpr (!kTwice) wait_older_loads<kStageLoads>();  // T
      __syncthreads();  // what the other wave made
      // Fragments in the order of their products: T^T, K^T.
      frag tf[kTerms * kBlocks], cf[kColumns], yf[2][kTerms], uf[2][kTerms];
      const auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i < kTerms * kBlocks) {
          const Triangle<T> b(i % kBlocks);
          tf[i] = solve_read.column(kSolve + i / kBlocks * C::kPanel, kTiles - 1 - b.tile, 1 - b.step);
        } else if ((i -= kTerms * kBlocks) < kColumns) {
          cf[i] = read.column(S::kKeys, i / 8 * 4 + i % 4, i / 4 % 2);
        }
      };
      constexpr int kFirstC = kTerms * kBlocks;
#pragma unroll
      for (int m = 0; m < kTiles; ++m) y[m] += lds_read<f32x4>(to_update + m * 1024 + thread * 16) * unit;
#pragma unroll
      for (int i = 0; i < kAheadBack; ++i) fetch(i);
      keep_order();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) split<T>(&y[kt * kPer], uf[kt]);
      // Y = T^T dU.
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
#pragma unroll
        for (int other = 0; other < kTerms - term; ++other)
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            const Triangle<T> b(i);
            if (other == 0) fetch(term * kBlocks + i + kAheadBack);
            sums[kTiles - 1 - b.tile].add(tf[term * kBlocks + i], uf[1 - b.step][other], term + other > 0);
          }
        keep_order();
      }
#pragma unroll
      for (int m = 0; m < kTiles; ++m) y[m] = sums[m].value();
      // dV and Y for the other wave to store: dV as [token][column].
      if constexpr (!TRANSIT) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          frag hi[1];
          split<T>(&y[kt * kPer], hi);
          lds_write(update_at + kt * 1024, hi[0]);
        }
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
          const int row = first_row<T>(m, lane.g);
          const f32x4 dv = y[m] * (*reinterpret_cast<const f32x4*>(factors + kTokens + row) * to_whole);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            lds_write(to_update + static_cast<unsigned>(((row + e) * kTurnPitch + lane.l) * sizeof(T)), static_cast<T>(dv[e]));
        }
      }
#pragma unroll
      for (int m = 0; m < kTiles; ++m) y[m] *= -*reinterpret_cast<const f32x4*>(factors + first_row<T>(m, lane.g));
      const Power<T> power(over_lane_groups<T>(largest_size<T, kTiles>(y)));
#pragma unroll
      for (int m = 0; m < kTiles; ++m) y[m] *= power.up;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) split<T>(&y[kt * kPer], yf[kt]);
      // D = c D + Q^T (c rq dO), which is handed, - K^T (beta c rk Y).
#pragma unroll
      for (int m0 = 0; m0 < kStateTiles; m0 += 4) {
        Sum<T> sum[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) sum[m].whole = (state[m0 + m] * whole + lds_read<f32x4>(added_at + (m0 + m) * 1024)) * power.up;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
          for (int m = 0; m < 4; ++m) fetch(kFirstC + m0 * 2 + kt * 4 + m + kAheadBack);
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int m = 0; m < 4; ++m) sum[m].add(cf[m0 * 2 + kt * 4 + m], yf[kt][term], term > 0);
          keep_order();
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) state[m0 + m] = sum[m].value() * power.down;
      }
      hand_state();
    }
    wait_loads();  // none into LDS that is another workgroup's by then
    __syncthreads();  // the last dV and Y are handed on
    if (!active) return;
    if (TRANSIT || (a.segments == 1 && a.grad_first != nullptr)) {
#pragma unroll
      for (int m = 0; m < kStateTiles; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = first_row<T>(m, lane.g) + e;
          if constexpr (TRANSIT) {
            if (w.unit)
              a.transits[(segment_at * DK + d) * DK + mine] = state[m][e];
            else
              a.partials[(segment_at * DK + d) * a.value_pad + mine] = state[m][e];
          } else if (d < key_size && mine < value_size) {
            a.grad_first[(bh * key_size + d) * value_size + mine] = state[m][e] * to_whole;
          }
        }
    }
    return;
  }

  // The other waves: what does not need D, with its loads, and the stores.
  const auto load_once = [&](int c) __attribute__((always_inline)) {
    query_loads.load(buffer_at(q_at + static_cast<int64_t>(c) * kTokens * a.query_strides.token), lds_at + S::kQuery, part,
                     rows_of(c));
    if constexpr (!kTwice) load_pair(c, 1, lds_at + S::kPairsOnce);
  };
  if (begin < end) load_once(end - 1);
  const float unit = kUnits<T> ? unit_of(a, bh) : 1.f;
  if constexpr (kUnits<T> && !TRANSIT)
    if (v0 == 0 && w.segment == 0 && part == 0 && thread == 0) a.units[bh] = unit;
  const Reader<T> places;
  const Own<T> own(from_panel / 16 + part);
  const Reader<T> fixed = places.moved(lds_at);
  T* out = static_cast<T*>(a.grad_value) + (static_cast<int64_t>(b) * a.tokens * a.heads + h) * value_size;
  const int64_t out_token = a.heads * value_size;
  const int store_at = column + lane.g * 4, store_count = value_size - store_at;
  const unsigned state_place = mine * DK + lane.g * (16 / sizeof(T));
  const unsigned update_place = mine * kTokens + lane.g * (16 / sizeof(T));
  const bool whole_rows = column + 16 <= value_size;
  unsigned out_place[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) out_place[n] = (n * 16 + lane.l) * static_cast<unsigned>(out_token) + store_at;
  Four<T> held_value[kTiles];
  frag held_update[2];
  const auto take_held = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
      held_value[n] = lds_read<Four<T>>(to_update + static_cast<unsigned>(((n * 16 + lane.l) * kTurnPitch + lane.g * 4) * sizeof(T)));
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) held_update[kt] = lds_read<frag>(update_at + kt * 1024);
  };
  // Of chunk c; true if every store was made.
  const auto store_held = [&](int c) __attribute__((always_inline)) {
    T* to = out + static_cast<int64_t>(c) * kTokens * out_token;
    const bool all = whole_rows && (c + 1) * kTokens <= a.tokens;
    if (all) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n) *reinterpret_cast<Run<T, 4>*>(to + out_place[n]) = __builtin_bit_cast(Run<T, 4>, held_value[n]);
    } else {
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
        if (static_cast<int64_t>(c) * kTokens + n * 16 + lane.l < a.tokens) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < store_count) to[out_place[n] + e] = held_value[n][e];
          end_of_part();
        }
    }
    T* keep = static_cast<T*>(a.grad_updates) + (first_chunk + c) * a.value_pad * kTokens;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) *reinterpret_cast<frag*>(keep + (update_place + kt * C::kStep)) = held_update[kt];
    return all;
  };
  bool all_stored = false;
#pragma unroll 1
  for (int c = end - 1; c >= begin; --c) {
    // The wait for what was loaded is not for the stores after it, of which there are at least so many.
    if (TRANSIT || c == end - 1 || !active)
      wait_loads();
    else if (all_stored)
      wait_older_loads<kTiles + 2 + kSteps>();
    else
      wait_older_loads<kSteps>();
    __syncthreads();
    const unsigned at = lds_at + S::kStages + (c & 1) * S::kStage;
    const Reader<T> pair_read = kTwice ? places.moved(at) : fixed;
    constexpr unsigned kPairs = kTwice ? S::kPairs : S::kPairsOnce;
    const float* factors = reinterpret_cast<const float*>(lds + S::kStages + (c & 1) * S::kStage + S::kFactors);
    frag d[kSteps];
    if constexpr (!TRANSIT) {
      take_held();
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) d[ks] = lds_read<frag>(added_at + ks * 1024);
    }
    frag g[2], pf[kTerms * kBlocks], qf[kColumns];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) g[kt] = own.column(at + S::kValues, kt);
    const auto fetch = [&](int i) __attribute__((always_inline)) {
      if (i < kTerms * kBlocks) {
        const Triangle<T> b(i % kBlocks);
        pf[i] = pair_read.column(kPairs + i / kBlocks * C::kPanel, kTiles - 1 - b.tile, 1 - b.step);
      } else if ((i -= kTerms * kBlocks) < kColumns) {
        qf[i] = fixed.column(S::kQuery, i / 8 * 4 + i % 4, i / 4 % 2);
      }
    };
    constexpr int kFirstQ = kTerms * kBlocks;
#pragma unroll
    for (int i = 0; i < kAheadBack; ++i) fetch(i);
    keep_order();
    // P^T dO.
    Sum<T> sums[kTiles];
#pragma unroll
    for (int term = 0; term < kTerms; ++term) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const Triangle<T> b(i);
        fetch(term * kBlocks + i + kAheadBack);
        sums[kTiles - 1 - b.tile].add(pf[term * kBlocks + i], g[1 - b.step], term > 0);
      }
      keep_order();
    }
#pragma unroll
    for (int m = 0; m < kTiles; ++m) lds_write(to_update + m * 1024 + thread * 16, sums[m].value());
    // Q^T (c rq dO).
    frag gf[2][kTerms];
    f32x4 v[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const f32x4 factor = *reinterpret_cast<const f32x4*>(factors + 3 * kTokens + first_row<T>(i, lane.g));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = factor[e] * static_cast<float>(g[i / kPer][i % kPer * 4 + e]);
    }
    const Power<T> power(over_lane_groups<T>(largest_size<T, kTiles>(v)));
    const float to_unit = power.down * unit;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) v[i] *= power.up;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) split<T>(&v[kt * kPer], gf[kt]);
#pragma unroll
    for (int m0 = 0; m0 < kStateTiles; m0 += 4) {
      Sum<T> sum[4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int m = 0; m < 4; ++m) fetch(kFirstQ + m0 * 2 + kt * 4 + m + kAheadBack);
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int m = 0; m < 4; ++m) sum[m].add(qf[m0 * 2 + kt * 4 + m], gf[kt][term], term > 0);
        keep_order();
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) lds_write(added_at + (m0 + m) * 1024, sum[m].value() * to_unit);
    }
    __syncthreads();
    load_once(c - 1);
    asm volatile("" ::: "memory");  // the stores stay behind the loads
    if constexpr (!TRANSIT) {
      if (!active) continue;
      if (c < end - 1) all_stored = store_held(c + 1);
      T* states = static_cast<T*>(a.grad_states) + (first_chunk + c) * a.value_pad * DK;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) *reinterpret_cast<frag*>(states + (state_place + ks * C::kStep)) = d[ks];
    }
  }
  wait_loads();  // none into LDS that is another workgroup's by then
  __syncthreads();
  if constexpr (!TRANSIT) {
    if (!active) return;
    if (begin < end) {
      take_held();
      store_held(begin);
    }
    const int64_t stop = a.tokens < int64_t{begin + a.segment_chunks} * kTokens
                             ? a.tokens
                             : int64_t{begin + a.segment_chunks} * kTokens;
    for (int64_t t = int64_t{end > begin ? end : begin} * kTokens + lane.l; t < stop; t += 16)
      if (store_count > 0) store_four(out + t * out_token + store_at, f32x4{0.f, 0.f, 0.f, 0.f}, store_count);
  }
}

// ---- gradients within every chunk --------------------------------------------------------------------------

// With dP = dO U^T and dA = -Y U^T (i > j), N = G dA,
//
//   dq' = diag(c) dO S^T + (G dP rk) K                                   (q' the scaled and normalised q)
//   dk' = -diag(beta c) Y S^T + diag(e) U D^T + (G dP)^T q' + (beta N) k' + (beta N)^T k'
//   dbeta_i = Y_i.V_i - c_i k'_i.(Y S^T)_i + sum_j N_ij k'_i.k'_j
//
// and a decay's gradient is the sum over the pairs, and the states, that its token lies between: with the
// gradients of the sums of decays, their total from the token on. A workgroup takes a chunk of a key head and
// adds up its value heads. Two waves share 16 tokens, which are their lanes throughout: each makes half of the
// keys' gradients, and one makes the pairs with its token as the row i (registers j), the other those with it
// as the column j (registers i), so that either is the operand of the next products, which they exchange.
// 190 KB are read and written for a chunk of 128 x 128 in bfloat16; 2048 of them take 115 us (3.4 TB/s), the rest
// of the time goes to the steps between barriers that the one workgroup of a compute unit has nothing beside.
typedef double f64x2 __attribute__((ext_vector_type(2)));
template <typename T, int DK>
struct GradientsLds {
  using C = Chunk<T>;
  static constexpr int kWide = DK / C::kTokens * C::kPanel;
  static constexpr int kRecord = (sizeof(Record<T>) + 1023) / 1024 * 1024;
  struct Block {
    unsigned char wide[2][kWide];        // states and their gradients
    unsigned char narrow[3][C::kPanel];  // U and Y transposed, dO; then the pairs as fragments
    unsigned char record[kRecord];
  } blocks[2];
  unsigned char keys[kWide], queries[kWide];
  unsigned char values[C::kPanel];  // of the block at work
  float slope[2][C::kTokens], kept[2][C::kTokens], step[2][C::kTokens], inner[2 * C::kTiles];
};

// What a wave does that makes the pairs with its tokens as rows (HALF 0) or columns (1), of the first (SIDE 0) or
// the second fragment of the chunk's tokens: all of it is known to the compiler but the tokens.
template <typename T, int DK, bool GROUPED, int HALF, int SIDE>
__device__ __forceinline__ void gradients_of(const DeltaArgs& a, GradientsLds<T, DK>& lds) {
  using C = Chunk<T>;
  using frag = typename C::frag;
  constexpr int kTokens = C::kTokens, kTiles = C::kTiles, kPer = C::kPer, kWaves = 2 * kTiles;
  constexpr int kPanels = DK / kTokens, kSteps = DK / C::kStep, kKeyTiles = DK / 32;  // of a wave
  constexpr int kVec = 16 / sizeof(T);
  auto& slope = lds.slope;
  auto& kept = lds.kept;
  auto& step = lds.step;
  auto& inner = lds.inner;
  // This thread, as a value that the compiler takes for another one each time: what follows from a lane's place is
  // made where it is used. Kept from one chunk to the next (or one phase), it took registers that then spilled,
  // and a wait for a reload is one for the next block's loads too.
  const auto again = []() __attribute__((always_inline)) {
    int thread = threadIdx.x & 63;
    asm volatile("" : "+v"(thread));
    return thread;
  };
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int half = HALF;
  const int block = wave % kTiles;
  // The wave's keys: from a panel of its half on, or (64 keys of 16 bits) from the middle of the only one.
  constexpr bool kFlip = DK / 2 * sizeof(T) < 128;
  constexpr unsigned kWide = kPanels * C::kPanel, kNarrow = 2 * kWide, kHalf = kFlip ? 0 : half * (kWide / 2);
  const int groups = GROUPED ? a.groups : 1;
  const int key_size = static_cast<int>(a.key_size), value_size = static_cast<int>(a.value_size);
  const auto store_gate = [&](void* p, int64_t at, float v) __attribute__((always_inline)) {
    if (a.float_gates)
      static_cast<float*>(p)[at] = v;
    else
      static_cast<T*>(p)[at] = static_cast<T>(v);
  };
  // A key head's chunk. One past its sequence's length has only zeros to be written.
  struct Item {
    unsigned id;
    int chunk, kh, b, t0, rows;
  };
  const unsigned key_heads = static_cast<unsigned>(a.key_heads), chunks = static_cast<unsigned>(a.chunks);
  const unsigned items = static_cast<unsigned>(a.batch) * key_heads * chunks;
  const auto item_from = [&](unsigned id) __attribute__((always_inline)) {
    Item it{id, 0, 0, 0, 0, 0};
    const int thread = again(), own_token = block * 16 + (thread & 15), first_key = half * (DK / 2) + (thread >> 4) * 4;
    for (; it.id < items; it.id += gridDim.x) {
      const unsigned row = it.id / chunks, sequence = row / key_heads;
      it.chunk = static_cast<int>(it.id - row * chunks);
      it.kh = static_cast<int>(row - sequence * key_heads);
      it.b = static_cast<int>(sequence);
      it.t0 = it.chunk * kTokens;
      const int left = length_of(a, it.b) - it.t0;
      it.rows = left < kTokens ? left : kTokens;
      if (left > 0) break;
      if (it.t0 + own_token >= a.tokens) continue;
      const int64_t token = static_cast<int64_t>(it.b) * a.tokens + it.t0 + own_token;
#pragma unroll 1
      for (int m = 0; m < kKeyTiles; ++m) {
        const int d = first_key + m * 16;
        if (d >= key_size) continue;
        const int64_t to = (token * a.key_heads + it.kh) * key_size + d;
        store_four(static_cast<T*>(a.grad_query) + to, f32x4{0.f, 0.f, 0.f, 0.f}, key_size - d);
        store_four(static_cast<T*>(a.grad_key) + to, f32x4{0.f, 0.f, 0.f, 0.f}, key_size - d);
      }
      if (thread < 16 && half == 0)
        for (int group = 0; group < groups; ++group) {
          store_gate(a.grad_decay, token * a.heads + it.kh * groups + group, 0.f);
          store_gate(a.grad_beta, token * a.heads + it.kh * groups + group, 0.f);
        }
    }
    return it;
  };
  // Four neighbouring values of this lane's row, in the wave's tile m.
  const auto own_values = [&](const Own<T>& mine, unsigned panels, int m) __attribute__((always_inline)) {
    if constexpr (kFlip) return half == 0 ? mine.four(panels, m) : mine.four(panels, m + kKeyTiles);
    return mine.four(panels, m);
  };
  const auto over_groups = [](float v) __attribute__((always_inline)) {
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
  };
  // Whether tile m holds partners of this wave's tokens.
  const auto has = [](int m) __attribute__((always_inline)) {
    return HALF == 0 ? m / kPer <= SIDE : m / kPer >= SIDE;
  };
  // Tiles of the chunk's tokens that hold partners of this wave's, and the fragments of them that a step reads.
  constexpr int kFirstOther = HALF == 0 ? 0 : SIDE * kPer;
  constexpr int kPartners = HALF == 0 ? (SIDE + 1) * kPer : (2 - SIDE) * kPer, kOthers = kPartners * (HALF + 1);
  constexpr int kAheadGrad = 6;
  // Blocks of values, of one head after another and one item after another: the next one's operands load while
  // one is worked on.
  // Every wave loads 8 rows of each panel.
  static_assert(kWaves == kTokens / 8, "a load a wave");
  const auto load_set = [&](int thread, const void* from, unsigned dst, int count, unsigned column, unsigned stride,
                            int rows, unsigned bytes) __attribute__((always_inline)) {
    const int load_row = wave * 8 + thread / 8;
    const unsigned load_piece = ((thread % 8) ^ swizzle(load_row)) << 4;
    const u32x4 buffer = buffer_at(from);
    const unsigned at = load_row < rows ? load_row * stride : kNowhere;
#pragma unroll
    for (int p = 0; p < count; ++p) {
      const unsigned in_row = column + p * 128 + load_piece;
      load_lds16(buffer, dst + p * C::kPanel + wave * 1024, in_row < bytes ? at + in_row : kNowhere);
    }
  };
  // As many loads whether there is a block or not (zeros, then), since waits count them.
  constexpr int kLoads = 2 * kPanels + 3;
  const auto load = [&](const Item& it, int group, int v0, int into, bool live) __attribute__((always_inline)) {
    const int h = it.kh * groups + group, thread = again();
    const int64_t at = (static_cast<int64_t>(it.b) * a.heads + h) * chunks + it.chunk;
    auto& to = lds.blocks[into & 1];
    const int left = static_cast<int>(a.value_pad) - v0, v_rows = !live ? 0 : left < kTokens ? left : kTokens;
    const int64_t v_at = at * a.value_pad + v0;
    load_set(thread, static_cast<const T*>(a.states) + v_at * DK, lds_address(to.wide[0]), kPanels, 0, DK * sizeof(T), v_rows,
             DK * sizeof(T));
    load_set(thread, static_cast<const T*>(a.grad_states) + v_at * DK, lds_address(to.wide[1]), kPanels, 0, DK * sizeof(T),
             v_rows, DK * sizeof(T));
    load_set(thread, static_cast<const T*>(a.updates) + v_at * kTokens, lds_address(to.narrow[0]), 1, 0, 128, v_rows, 128);
    load_set(thread, static_cast<const T*>(a.grad_updates) + v_at * kTokens, lds_address(to.narrow[1]), 1, 0, 128, v_rows, 128);
    load_set(thread, at_token<T>(a.grad_output, a.grad_strides, it.b, it.t0, h), lds_address(to.narrow[2]), 1,
             static_cast<unsigned>(v0 * sizeof(T)), static_cast<unsigned>(a.grad_strides.token * sizeof(T)), live ? it.rows : 0,
             static_cast<unsigned>(value_size * sizeof(T)));
    if (wave < GradientsLds<T, DK>::kRecord / 1024) {
      const unsigned at_byte = wave * 1024 + thread * 16;
      load_lds16(buffer_at(reinterpret_cast<const Record<T>*>(a.records) + at), lds_address(to.record) + wave * 1024,
                 live && at_byte < sizeof(Record<T>) ? at_byte : kNowhere);
    }
  };
  const auto load_keys = [&](const Item& it) __attribute__((always_inline)) {
    const unsigned bytes = static_cast<unsigned>(key_size * sizeof(T));
    const int thread = again();
    load_set(thread, at_token<T>(a.key, a.key_strides, it.b, it.t0, it.kh), lds_address(lds.keys), kPanels, 0,
             static_cast<unsigned>(a.key_strides.token * sizeof(T)), it.rows, bytes);
    load_set(thread, at_token<T>(a.query, a.query_strides, it.b, it.t0, it.kh), lds_address(lds.queries), kPanels, 0,
             static_cast<unsigned>(a.query_strides.token * sizeof(T)), it.rows, bytes);
  };
  int index = 0;  // of the block, over all items
  Item it = item_from(blockIdx.x);
  if (it.id < items) load(it, 0, 0, 0, true);
  wait_loads();
#pragma unroll 1
  while (it.id < items) {
    const Item next = item_from(it.id + gridDim.x);
    const int t0 = it.t0, kh = it.kh, b = it.b, rows = it.rows;
    f32x4 dq_all[GROUPED ? kKeyTiles : 1], dk_all[GROUPED ? kKeyTiles : 1];
    if constexpr (GROUPED) {
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m) dq_all[m] = dk_all[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll 1
  for (int group = 0; group < groups; ++group) {
    const int h = kh * groups + group;
    float grad_unit = 1.f;
    if constexpr (kUnits<T>) grad_unit = a.units[static_cast<int64_t>(b) * a.heads + h];
    f32x4 dq[kKeyTiles], dk[kKeyTiles], back[kKeyTiles];  // dO S^T, Y S^T, U D^T
#pragma unroll
    for (int m = 0; m < kKeyTiles; ++m) dq[m] = dk[m] = back[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 pair_p[kTiles], pair_a[kTiles];  // dP and Y U^T
#pragma unroll
    for (int m = 0; m < kTiles; ++m) pair_p[m] = pair_a[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    float dbeta = 0.f, product = 0.f;
    unsigned here = 0;
    const int at_blocks = again();
    Reader<T> read(kFlip ? half * 64 : 0, at_blocks);
    Own<T> mine(block, at_blocks);
#pragma unroll 1
    for (int v0 = 0; v0 < a.value_pad; v0 += kTokens, ++index) {
      // What a first block needs was waited for before the results before it were stored.
      if (v0 > 0) wait_loads();
      __syncthreads();
      if constexpr (HALF == 0) {  // the wave's own rows of the values
        const u32x4 buffer = buffer_at(at_token<T>(a.value, a.value_strides, b, t0, h));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int thread = again(), row = block * 16 + i * 8 + thread / 8;
          const unsigned in_row = static_cast<unsigned>(v0 * sizeof(T)) + (((thread % 8) ^ swizzle(row)) << 4);
          load_lds16(buffer, lds_address(lds.values) + (block * 2 + i) * 1024,
                     row < rows && in_row < static_cast<unsigned>(value_size * sizeof(T))
                         ? row * static_cast<unsigned>(a.value_strides.token * sizeof(T)) + in_row
                         : kNowhere);
        }
      }
      if (group == 0 && v0 == 0) load_keys(it);
      {
        const bool more = v0 + kTokens < a.value_pad, stays = more || group + 1 < groups;
        load(stays ? it : next, more ? group : stays ? group + 1 : 0, more ? v0 + kTokens : 0, index + 1,
             stays || next.id < items);
      }
      const unsigned to = lds_address(&lds.blocks[index & 1]);
      read = read.moved(to - here);
      mine = mine.moved(to - here);
      here = to;
      // Fragments in the order of their products, read kAheadGrad before them.
      constexpr int kStep = 3 + 2 * kKeyTiles + kOthers;
      frag of[2 * kStep];
      const auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i >= 2 * kStep) return;
        const int kt = i / kStep, k = i % kStep, n = k - 3 - 2 * kKeyTiles;
        of[i] = k == 0   ? mine.row(kNarrow + 2 * C::kPanel, kt)
                : k == 1 ? mine.column(kNarrow, kt)
                : k == 2 ? mine.column(kNarrow + C::kPanel, kt)
                : n < 0  ? read.ordered_column((k - 3) % 2 * kWide + kHalf, (k - 3) / 2, kt)
                : HALF == 0  ? read.column(kNarrow, kFirstOther + n, kt)
                : n % 2 == 0 ? read.operand(kNarrow + 2 * C::kPanel, kFirstOther + n / 2, kt)
                             : read.column(kNarrow + C::kPanel, kFirstOther + n / 2, kt);
      };
#pragma unroll
      for (int i = 0; i < kAheadGrad; ++i) fetch(i);
      keep_order();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        fetch(kt * kStep + kAheadGrad);
        fetch(kt * kStep + kAheadGrad + 1);
        fetch(kt * kStep + kAheadGrad + 2);
        const frag g = of[kt * kStep], u = of[kt * kStep + 1], y = of[kt * kStep + 2];
#pragma unroll
        for (int m = 0; m < kKeyTiles; ++m) {
          const int i = kt * kStep + 3 + 2 * m;
          fetch(i + kAheadGrad);
          fetch(i + kAheadGrad + 1);
          dq[m] = Fragment<T>::mma(of[i], g, dq[m]);
          dk[m] = Fragment<T>::mma(of[i], y, dk[m]);
          back[m] = Fragment<T>::mma(of[i + 1], u, back[m]);
          keep_order();
        }
#pragma unroll
        for (int n = 0; n < kPartners; ++n) {
          const int m = kFirstOther + n, i = kt * kStep + 3 + 2 * kKeyTiles + n * (HALF + 1);
          fetch(i + kAheadGrad);
          if constexpr (HALF == 0) {
            pair_p[m] = Fragment<T>::mma(of[i], g, pair_p[m]);
            pair_a[m] = Fragment<T>::mma(of[i], y, pair_a[m]);
          } else {
            fetch(i + kAheadGrad + 1);
            pair_p[m] = Fragment<T>::mma(of[i], u, pair_p[m]);
            pair_a[m] = Fragment<T>::mma(of[i + 1], u, pair_a[m]);
          }
          keep_order();
        }
        if constexpr (HALF == 0) {
          if (kt == 0) wait_older_loads<kLoads>();
          const frag f = lds_read<frag>(lds_address(lds.values) - here + mine.rows[kt]);
#pragma unroll
          for (int i = 0; i < kVec; ++i) dbeta = fmaf(static_cast<float>(f[i]), static_cast<float>(y[i]), dbeta);
        }
      }
      // The state's product with its gradient.
      for (int i = threadIdx.x; i < kPanels * C::kPanel / 16; i += 64 * kWaves) {
        const frag s = lds_read<frag>(here + i * 16);
        const frag d = lds_read<frag>(here + kWide + i * 16);
#pragma unroll
        for (int e = 0; e < kVec; ++e) product = fmaf(static_cast<float>(s[e]), static_cast<float>(d[e]), product);
      }
    }
    // The products of either unit alone, in both.
    float value_unit = 1.f;
    if constexpr (kUnits<T>) value_unit = reinterpret_cast<const Record<T>*>(lds.blocks[(index - 1) & 1].record)->unit;
    const float to_whole = 1.f / (value_unit * grad_unit);
    dbeta *= value_unit;
#pragma unroll
    for (int m = 0; m < kKeyTiles; ++m) dq[m] *= grad_unit;
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
      if (has(m)) pair_p[m] *= grad_unit;
    if (group == 0 && a.value_pad <= kTokens) {  // the keys are under way still
      wait_older_loads<kLoads>();
      __syncthreads();
    }
    product = lanes_sum<64>(product);
    if ((threadIdx.x & 63) == 0) inner[wave] = product * to_whole;
    const auto* facts = reinterpret_cast<const Record<T>*>(lds.blocks[(index - 1) & 1].record);
    const double* sum = facts->sum;
    const float *beta = facts->beta, *rk = facts->rk, *rq = facts->rq;
    const uint64_t closed = facts->closed;
    const int thread = again(), own = block * 16 + (thread & 15), first = thread >> 4;
    const Reader<T> key_read = Reader<T>(kFlip ? half * 64 : 0, thread).moved(lds_address(lds.keys));
    const Own<T> key_mine = Own<T>(block, thread).moved(lds_address(lds.keys));
    constexpr unsigned keys = 0, queries = kWide;
    constexpr unsigned states = keys + kHalf, grads = queries + kHalf;  // of the wave's keys
    const double own_sum = sum[own];
    const float own_beta = beta[own], own_rk = rk[own], own_rq = rq[own], norm = facts->norm[own];

    dbeta = over_groups(dbeta);
    float dsum;
    {
      // What comes through the states.
      const float c = (closed & (~uint64_t{0} >> (63 - own))) == 0 ? decay_between(own_sum, 0.) : 0.f;
      const float e_own = open_between(closed, own, kTokens - 1) ? decay_between(sum[kTokens - 1], own_sum) : 0.f;
      float q_dot = 0.f, k_dot = 0.f, b_dot = 0.f;
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m) {
        const f32x4 q = own_values(key_mine, grads, m), k = own_values(key_mine, states, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q_dot = fmaf(q[e], dq[m][e], q_dot);
          k_dot = fmaf(k[e], dk[m][e], k_dot);
          b_dot = fmaf(k[e], back[m][e], b_dot);
          dq[m][e] *= c;
          dk[m][e] = fmaf(e_own, back[m][e], -own_beta * c * dk[m][e]);
        }
      }
      q_dot = over_groups(q_dot) * c * own_rq;
      k_dot = over_groups(k_dot) * c * own_rk;
      b_dot = over_groups(b_dot) * e_own * own_rk;
      dbeta -= k_dot;
      dsum = q_dot - own_beta * k_dot - b_dot;
      if (first == 0) kept[half][own] = b_dot * to_whole;
    }
    // Pairs.
    f32x4 kk[kTiles], qk[kTiles];
#pragma unroll
    for (int m = 0; m < kTiles; ++m) kk[m] = qk[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    {
      constexpr int kStep = 2 + kOthers;
      frag of[kSteps * kStep];
      const auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i >= kSteps * kStep) return;
        const int ks = i / kStep, k = i % kStep, n = k - 2;
        of[i] = k == 0       ? key_mine.row(keys, ks)
                : k == 1     ? key_mine.row(queries, ks)
                : HALF == 0  ? key_read.operand(keys, kFirstOther + n, ks)
                : n % 2 == 0 ? key_read.operand(keys, kFirstOther + n / 2, ks)
                             : key_read.operand(queries, kFirstOther + n / 2, ks);
      };
#pragma unroll
      for (int i = 0; i < kAheadGrad; ++i) fetch(i);
      keep_order();
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        fetch(ks * kStep + kAheadGrad);
        fetch(ks * kStep + kAheadGrad + 1);
        const frag k = of[ks * kStep], q = of[ks * kStep + 1];
#pragma unroll
        for (int n = 0; n < kPartners; ++n) {
          const int m = kFirstOther + n, i = ks * kStep + 2 + n * (HALF + 1);
          fetch(i + kAheadGrad);
          kk[m] = Fragment<T>::mma(of[i], k, kk[m]);
          if constexpr (HALF == 0) {
            qk[m] = Fragment<T>::mma(of[i], q, qk[m]);
          } else {
            fetch(i + kAheadGrad + 1);
            qk[m] = Fragment<T>::mma(of[i + 1], k, qk[m]);
          }
          keep_order();
        }
      }
    }
    // Which pairs no closed gate parts: a bit each.
    unsigned open_bits = ~0u;
    if (closed != 0) {
      open_bits = 0;
#pragma unroll
      for (int n = 0; n < 4 * kTiles; ++n) {
        const int other = first_row<T>(n / 4, first) + n % 4;
        const int i = half == 0 ? own : other, j = half == 0 ? other : own;
        if (j <= i && open_between(closed, j, i)) open_bits |= 1u << n;
      }
    }
    // Without branches: all is read and made, then chosen.
    float pairs = 0.f, steps = 0.f;
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
      if (!has(m)) continue;
      const int at = first_row<T>(m, first);
      const f32x4 other_rk = *reinterpret_cast<const f32x4*>(rk + at);
      const f32x4 other_rq = HALF == 0 ? other_rk : *reinterpret_cast<const f32x4*>(rq + at);
      const f32x4 other_beta = HALF == 0 ? other_rk : *reinterpret_cast<const f32x4*>(beta + at);
      const f64x2 other_sum[2] = {*reinterpret_cast<const f64x2*>(sum + at), *reinterpret_cast<const f64x2*>(sum + at + 2)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int other = at + e;
        const bool below = HALF == 0 ? own > other : other > own, open = (open_bits >> (m * 4 + e) & 1) != 0;
        const double to = other_sum[e / 2][e % 2];
        const float ratio = HALF == 0 ? decay_between(own_sum, to) : decay_between(to, own_sum);
        // The other token's factors; this one's are taken out of the sums.
        float p = ratio * (HALF == 0 ? other_rk[e] : other_rq[e]) * pair_p[m][e];
        float n = -ratio * other_rk[e] * pair_a[m][e];
        p = (open & (below | (own == other))) ? p : 0.f;
        n = (open & below) ? n : 0.f;
        const float weighed = HALF == 0 ? n : n * other_beta[e];
        pairs = fmaf(p, qk[m][e], pairs);
        steps = fmaf(weighed, kk[m][e], steps);
        pair_p[m][e] = p;
        pair_a[m][e] = HALF == 0 ? own_beta * n : weighed;
      }
    }
    pairs = over_groups(pairs);
    steps = over_groups(steps);
    if (half == 0) {
      dbeta += steps * own_rk;
      dsum += pairs * own_rq + own_beta * own_rk * steps;
    } else {
      dsum -= (pairs + steps) * own_rk;
    }
    // Of float16, the largest of the pairs with a token, over both waves: behind the record, whose place is larger.
    float* pair_sizes = reinterpret_cast<float*>(lds.blocks[(index - 1) & 1].record + sizeof(Record<T>));
    static_assert(!kUnits<T> || GradientsLds<T, DK>::kRecord - sizeof(Record<T>) >= 8 * kTokens);
    const float most = over_lane_groups<T>(largest_size<T, kTiles>(pair_a, largest_size<T, kTiles>(pair_p)));
    if (first == 0) {
      slope[half][own] = dsum * to_whole;
      step[half][own] = dbeta * to_whole;
      if constexpr (kUnits<T>) pair_sizes[half * kTokens + own] = most;
    }
    // The pairs as fragments, for both waves of these tokens: three of each kind.
    __syncthreads();  // all have read U, Y and dO
    float both = 0.f;
    if constexpr (kUnits<T>) both = fmaxf(pair_sizes[own], pair_sizes[kTokens + own]);
    const Power<T> power(both);
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
      if (!has(m)) continue;
      pair_p[m] *= power.up;
      pair_a[m] *= power.up;
    }
#pragma unroll
    for (int m = 0; m < kKeyTiles; ++m) {
      dq[m] *= power.up;
      dk[m] *= power.up;
    }
    frag* shared = reinterpret_cast<frag*>(lds.blocks[(index - 1) & 1].narrow[0]) + block * 6 * 64 + thread;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      if (!has(kt * kPer)) continue;
      frag f[1];
      split<T>(&pair_p[kt * kPer], f);
      shared[(kt + half) * 128] = f[0];
      split<T>(&pair_a[kt * kPer], f);
      shared[(kt + half) * 128 + 64] = f[0];
    }
    __syncthreads();
    {
      // k for rows and columns, q for columns of the first (SIDE 0) or the second fragment of tokens and on.
      frag of[4 * kKeyTiles];
      const auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i >= 4 * kKeyTiles) return;
        const int kt = i / (2 * kKeyTiles), m = i % (2 * kKeyTiles) / 2;
        if (i % 2 == 0)
          of[i] = key_read.ordered_column(states, m, kt);
        else if (kt >= SIDE)
          of[i] = key_read.ordered_column(grads, m, kt);
      };
      frag weights[2][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (w < 2 ? kt <= SIDE : kt >= SIDE) weights[kt][w] = shared[(kt + w / 2) * 128 + w % 2 * 64];
#pragma unroll
      for (int i = 0; i < kAheadGrad; ++i) fetch(i);
      keep_order();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const bool as_row = kt <= SIDE, as_column = kt >= SIDE;
#pragma unroll
        for (int m = 0; m < kKeyTiles; ++m) {
          const int i = (kt * kKeyTiles + m) * 2;
          fetch(i + kAheadGrad);
          fetch(i + kAheadGrad + 1);
          if (as_row) {
            dq[m] = Fragment<T>::mma(of[i], weights[kt][0], dq[m]);
            dk[m] = Fragment<T>::mma(of[i], weights[kt][1], dk[m]);
          }
          if (as_column) {
            dk[m] = Fragment<T>::mma(of[i], weights[kt][3], dk[m]);
            dk[m] = Fragment<T>::mma(of[i + 1], weights[kt][2], dk[m]);
          }
          keep_order();
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kKeyTiles; ++m) {
      dq[m] *= power.down * to_whole;
      dk[m] *= power.down * to_whole;
    }
    // The next block is there, long since: waited for here, so that no wait is for the stores that follow.
    wait_loads();
    // (By one wave, which the others need not wait for.)
    const auto store_gates = [&]() __attribute__((always_inline)) {
      if (wave != 0) return;
      // A token's decay: the gradients of the sums from it on, the last of which has the states' too.
      const int t = thread;
      float v = 0.f, k = 0.f;
      if (t < kTokens) {
        v = slope[0][t] + slope[1][t];
        k = kept[0][t] + kept[1][t];
      }
      k = lanes_sum<64>(k);
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += inner[w];
      if (t == kTokens - 1) v += k + facts->whole * s;
#pragma unroll
      for (int by = 1; by < kTokens; by *= 2) {
        const float after = __shfl_down(v, by);
        if (t + by < kTokens) v += after;
      }
      if (t < kTokens && t0 + t < a.tokens) {
        const int64_t to = (static_cast<int64_t>(b) * a.tokens + t0 + t) * a.heads + h;
        store_gate(a.grad_decay, to, t < rows && (closed >> t & 1) == 0 ? v : 0.f);
        store_gate(a.grad_beta, to, t < rows ? step[0][t] + step[1][t] : 0.f);
      }
    };
    if constexpr (GROUPED) {
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m) {
        dq_all[m] += dq[m];
        dk_all[m] += dk[m];
      }
    }
    if (GROUPED && group + 1 < groups) {
      store_gates();
      continue;
    }
    // q = q' / rq and k = k' / rk, with their lengths.
    const f32x4* dqs = GROUPED ? dq_all : dq;
    const f32x4* dks = GROUPED ? dk_all : dk;
    float q_dot = 0.f, k_dot = 0.f;
    if (a.normalize) {
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m) {
        const f32x4 q = own_values(key_mine, grads, m), k = own_values(key_mine, states, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q_dot = fmaf(q[e], dqs[m][e], q_dot);
          k_dot = fmaf(k[e], dks[m][e], k_dot);
        }
      }
      q_dot = over_groups(q_dot);
      k_dot = over_groups(k_dot);
      float* dots = reinterpret_cast<float*>(lds.values);  // [2][2][kTokens]
      if (first == 0) {
        dots[half * kTokens + own] = q_dot;
        dots[(2 + half) * kTokens + own] = k_dot;
      }
      __syncthreads();
      q_dot = (dots[own] + dots[kTokens + own]) * norm * norm;
      k_dot = (dots[2 * kTokens + own] + dots[3 * kTokens + own]) * own_rk * own_rk;
    }
    if (t0 + own < a.tokens) {
      const int64_t row = (static_cast<int64_t>(b) * a.tokens + t0 + own) * a.key_heads + kh;
      T* dq_out = static_cast<T*>(a.grad_query) + row * key_size;
      T* dk_out = static_cast<T*>(a.grad_key) + row * key_size;
      const int first_key = half * (DK / 2) + first * 4;
      const bool whole = key_size % 4 == 0;
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m) {
        const int d = first_key + m * 16;
        const f32x4 q = own_values(key_mine, grads, m), k = own_values(key_mine, states, m);
        const f32x4 to_q = own_rq * (dqs[m] - q_dot * q), to_k = own_rk * (dks[m] - k_dot * k);
        if (d >= key_size) continue;
        store_four(dq_out + d, to_q, whole ? 4 : key_size - d);
        store_four(dk_out + d, to_k, whole ? 4 : key_size - d);
      }
    }
    store_gates();
  }
    it = next;
  }
}

template <typename T, int DK, bool GROUPED>
__global__ __launch_bounds__(Chunk<T>::kTokens * 8, 2) void delta_gradients(DeltaArgs a) {
  extern __shared__ __align__(1024) unsigned char shared[];
  auto& lds = *reinterpret_cast<GradientsLds<T, DK>*>(shared);
  constexpr int kTiles = Chunk<T>::kTiles;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool second = wave % kTiles >= kTiles / 2;
  if (wave < kTiles) {
    if (second)
      gradients_of<T, DK, GROUPED, 0, 1>(a, lds);
    else
      gradients_of<T, DK, GROUPED, 0, 0>(a, lds);
  } else {
    if (second)
      gradients_of<T, DK, GROUPED, 1, 1>(a, lds);
    else
      gradients_of<T, DK, GROUPED, 1, 0>(a, lds);
  }
}

// ---- few tokens ----------------------------------------------------------------------------------------

// The definition, token by token: a workgroup keeps kDeltaStepColumns columns of a head's state, a
// thread four of them at DK / 16 keys. One pass over the state gives S^T k and S^T q together, since
// o = a S^T q + (k.q) u; a token costs one barrier. Bound by reading and writing the state: one token of 32
// sequences with 8 heads of 128 x 128, 34 MB, in 12.6 us (2.7 TB/s, its launch included).
template <typename T, int DK>
__global__ __launch_bounds__(256, 4) void delta_step(DeltaArgs a) {
  constexpr int kRows = DK / 16, kQuads = kDeltaStepColumns / 4;
  __shared__ float sums[2][4][kQuads][12];
  const int quad = threadIdx.x % kQuads, part = threadIdx.x / kQuads, wave = threadIdx.x >> 6;
  const unsigned heads = static_cast<unsigned>(a.batch * a.heads), tile = blockIdx.x / heads;
  const int64_t bh = blockIdx.x - tile * heads;
  const int b = static_cast<int>(static_cast<unsigned>(bh) / static_cast<unsigned>(a.heads));
  const int h = static_cast<int>(bh) - b * static_cast<int>(a.heads);
  const int kh = h / a.groups;
  const int value_size = static_cast<int>(a.value_size), key_size = static_cast<int>(a.key_size);
  const int v0 = static_cast<int>(tile) * kDeltaStepColumns + quad * 4;
  const int count = value_size - v0;  // columns of this thread, of four
  const int length = length_of(a, b);
  f32x4 state[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int d = part + i * 16;
    state[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.first == nullptr || d >= key_size || count <= 0) continue;
    const float* p = a.first + (bh * key_size + d) * value_size + v0;
    if (count >= 4) {
      state[i] = __builtin_bit_cast(f32x4, load_run<4>(p));
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < count) state[i][e] = p[e];
      end_of_part();
    }
  }
  T* out = static_cast<T*>(a.output) + (static_cast<int64_t>(b) * a.tokens * a.heads + h) * value_size + v0;
#pragma unroll 1
  for (int t = 0; t < length; ++t) {
    const T* kp = at_token<T>(a.key, a.key_strides, b, t, kh);
    const T* qp = at_token<T>(a.query, a.query_strides, b, t, kh);
    float k[kRows], q[kRows], v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int d = part + i * 16;
      k[i] = d < key_size ? static_cast<float>(kp[d]) : 0.f;
      q[i] = d < key_size ? static_cast<float>(qp[d]) : 0.f;
    }
    const T* vp = at_token<T>(a.value, a.value_strides, b, t, h) + v0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) v[e] = static_cast<float>(vp[e]);
    const int64_t d_at = b * a.decay_strides.batch + t * a.decay_strides.token + h * a.decay_strides.head;
    const int64_t f_at = b * a.beta_strides.batch + t * a.beta_strides.token + h * a.beta_strides.head;
    const float decay = a.float_gates ? static_cast<const float*>(a.decay)[d_at]
                                      : static_cast<float>(static_cast<const T*>(a.decay)[d_at]);
    const float beta = a.float_gates ? static_cast<const float*>(a.beta)[f_at]
                                     : static_cast<float>(static_cast<const T*>(a.beta)[f_at]);
    // S^T k, S^T q, then k.k, q.q, k.q.
    float s[11] = {};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = fmaf(state[i][e], k[i], s[e]);
        s[4 + e] = fmaf(state[i][e], q[i], s[4 + e]);
      }
      s[8] = fmaf(k[i], k[i], s[8]);
      s[9] = fmaf(q[i], q[i], s[9]);
      s[10] = fmaf(k[i], q[i], s[10]);
    }
#pragma unroll
    for (int j = 0; j < 11; ++j) {
      s[j] += __shfl_xor(s[j], 16);
      s[j] += __shfl_xor(s[j], 32);
    }
    if ((threadIdx.x & 63) < kQuads) {
#pragma unroll
      for (int j = 0; j < 11; ++j) sums[t & 1][wave][quad][j] = s[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 11; ++j) {
      s[j] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) s[j] += sums[t & 1][w][quad][j];
    }
    const float rk = a.normalize ? 1.f / sqrtf(s[8] + kNormEps) : 1.f;
    const float rq = a.scale * (a.normalize ? 1.f / sqrtf(s[9] + kNormEps) : 1.f);
    const float keep = decay < kDeltaClosed ? 0.f : expf(decay);
    f32x4 o;
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = beta * fmaf(-keep * rk, s[e], v[e]) * rk;
      o[e] = rq * fmaf(keep, s[4 + e], s[10] * u[e]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[i][e] = fmaf(k[i], u[e], keep * state[i][e]);
    if (part == 0 && count > 0) store_four(out + static_cast<int64_t>(t) * a.heads * value_size, o, count);
  }
  if (count <= 0) return;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int d = part + i * 16;
    if (d < key_size) store_four(a.last + (bh * key_size + d) * value_size + v0, state[i], count);
  }
  for (int t = length + part; t < a.tokens; t += 16)
    store_four(out + static_cast<int64_t>(t) * a.heads * value_size, f32x4{0.f, 0.f, 0.f, 0.f}, count);
}

// ---- the largest value of a head ------------------------------------------------------------------------------

// Of a head's values and its first state, or of its gradients of outputs and of the last state, over a part of the
// tokens and of the state; what is not finite, or past a sequence's length, does not count.
// Bound by memory: 33 MB in 14 us, 134 MB in 41 (3.3 TB/s); the walks that follow read the same.
template <typename T, bool GRADIENT>
__global__ __launch_bounds__(256) void delta_largest(DeltaArgs a) {
  constexpr unsigned kInfinity = 0x7c00;
  __shared__ float waves[4];
  // Heads of the same tokens, which lie side by side in memory, in workgroups that do.
  const unsigned heads = static_cast<unsigned>(a.batch * a.heads), part = blockIdx.x / heads, row = blockIdx.x - part * heads;
  const int b = static_cast<int>(row / static_cast<unsigned>(a.heads)), h = static_cast<int>(row) - b * static_cast<int>(a.heads);
  const DeltaStrides& strides = GRADIENT ? a.grad_strides : a.value_strides;
  const T* rows = at_token<T>(GRADIENT ? a.grad_output : a.value, strides, b, 0, h);
  const int64_t length = length_of(a, b), begin = length * part / a.parts, end = length * (part + 1) / a.parts;
  // Rows are whole 16 bytes long. Four loads a thread are under way (the last piece again where there are fewer).
  const int64_t pieces = (a.value_size + 7) / 8, all = (end - begin) * pieces;
  unsigned largest = 0;
  for (int64_t first = 0; first < all; first += 1024) {
    Run<uint16_t, 8> v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t i = std::min<int64_t>(first + k * 256 + threadIdx.x, all - 1);
      const int64_t t = static_cast<unsigned>(i) == i ? static_cast<unsigned>(i) / static_cast<unsigned>(pieces) : i / pieces;
      v[k] = load_run<8>(reinterpret_cast<const uint16_t*>(rows + (begin + t) * strides.token + (i - t * pieces) * 8));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned size = v[k].v[e] & 0x7fffu;
        largest = std::max(largest, size < kInfinity ? size : 0u);
      }
  }
  float most = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(largest)));
  const float* state = GRADIENT ? a.grad_last : a.first;
  if (state != nullptr) {
    const int64_t count = a.key_size * a.value_size;
    for (int64_t i = part * 256 + threadIdx.x; i < count; i += a.parts * 256) {
      const float size = fabsf(state[row * count + i]);
      most = fmaxf(most, size < __builtin_inff() ? size : 0.f);
    }
  }
  most = lanes_largest(most);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0) a.largest[row * a.parts + part] = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
}

// ---- launches --------------------------------------------------------------------------------------------

// Rows [batch, tokens, heads, size] copied with a pitch of whole 16 bytes, zeros past their end.
template <typename T>
__global__ __launch_bounds__(256) void delta_copy(DeltaCopy c) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t parts = c.pitch / kVec, total = c.batch * c.tokens * c.heads * parts;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t at = id % parts * kVec, row = id / parts;
    const int64_t h = row % c.heads, t = row / c.heads % c.tokens, b = row / c.heads / c.tokens;
    const T* p = at_token<T>(c.from, c.strides, b, t, h) + at;
    Run<T, kVec> v;
    if (at + kVec <= c.size) {
      v = load_run<kVec>(p);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v.v[i] = at + i < c.size ? p[i] : static_cast<T>(0.f);
    }
    store_run<kVec>(static_cast<T*>(c.to) + id * kVec, v);
  }
}

template <typename T, bool GRADIENT>
hipError_t launch_largest(const DeltaArgs& a, hipStream_t stream) {
  if (a.largest == nullptr) return hipSuccess;
  hipLaunchKernelGGL((delta_largest<T, GRADIENT>), dim3(static_cast<unsigned>(a.batch * a.heads * a.parts)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

template <typename T, int DK>
hipError_t launch_prepare(const DeltaArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((delta_prepare<T, DK>), dim3(static_cast<unsigned>(a.batch * a.key_heads * a.chunks)),
                     dim3(Chunk<T>::kTokens * 4), 0, stream, a);
  return hipGetLastError();
}

int64_t value_tiles(const DeltaArgs& a, int columns) { return (a.value_size + columns - 1) / columns; }

// Walks of 32 columns where those of 64 would leave half of the compute units idle: 2048 tokens of 48 and 64 heads
// of 128 x 128 (96 and 128 walks of 64 columns) take 83 and 89 us forward and 106 and 108 back where 64 columns take
// 109 and 112, 113 and 120. From 129 on two of 32 would share a compute unit's time: 72 heads 160 and 195 us for 122
// and 122.
bool narrow_walk(const DeltaArgs& a) { return a.segments == 1 && a.batch * a.heads * value_tiles(a, 64) <= 128; }

// One walk; TRANSIT: of its segments, with the columns of the unit matrix.
template <typename T, int DK, bool KEEP, bool TRANSIT, int W>
hipError_t launch_walk(const DeltaArgs& a, hipStream_t stream) {
  constexpr int kBytes = Walk<T, DK, W, !TRANSIT>::kBytes;
  const auto kernel = delta_forward<T, DK, W, KEEP, TRANSIT>;
  static std::atomic<uint64_t> asked{0};
  const hipError_t err = ask_lds(kernel, kBytes, asked);
  if (err != hipSuccess) return err;
  const int64_t tiles = value_tiles(a, W * 16) + (TRANSIT ? DK / (W * 16) : 0);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.batch * a.heads * tiles * a.segments)), dim3(128 * W), kBytes,
                     stream, a);
  return hipGetLastError();
}

template <typename T, int DK, bool TRANSIT, int W>
hipError_t launch_walk_back(const DeltaArgs& a, hipStream_t stream) {
  constexpr int kBytes = WalkBack<T, DK, W>::kBytes;
  const auto kernel = delta_backward<T, DK, W, TRANSIT>;
  static std::atomic<uint64_t> asked{0};
  const hipError_t err = ask_lds(kernel, kBytes, asked);
  if (err != hipSuccess) return err;
  const int64_t tiles = value_tiles(a, W * 16) + (TRANSIT ? DK / (W * 16) : 0);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.batch * a.heads * tiles * a.segments)), dim3(128 * W), kBytes,
                     stream, a);
  return hipGetLastError();
}

template <int DK, bool REVERSE>
hipError_t launch_join(const DeltaArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((delta_join<DK, REVERSE>), dim3(static_cast<unsigned>(a.batch * a.heads * value_tiles(a, 16))),
                     dim3(DK * 4), 0, stream, a);
  return hipGetLastError();
}

template <typename T, int DK>
hipError_t launch_forward(const DeltaArgs& a, const DeltaPlan& p, hipStream_t stream) {
  if (p.step) {
    hipLaunchKernelGGL((delta_step<T, DK>),
                       dim3(static_cast<unsigned>(a.batch * a.heads * value_tiles(a, kDeltaStepColumns))), dim3(256), 0,
                       stream, a);
    return hipGetLastError();
  }
  hipError_t err = hipSuccess;
  if constexpr (kUnits<T>) err = launch_largest<T, false>(a, stream);
  if (err == hipSuccess && a.chunks > 0) err = launch_prepare<T, DK>(a, stream);
  if (err == hipSuccess && a.segments > 1) {
    err = launch_walk<T, DK, false, true, 4>(a, stream);
    if (err == hipSuccess) err = launch_join<DK, false>(a, stream);
  }
  if (err != hipSuccess) return err;
  if (narrow_walk(a))
    return a.states != nullptr ? launch_walk<T, DK, true, false, 2>(a, stream) : launch_walk<T, DK, false, false, 2>(a, stream);
  return a.states != nullptr ? launch_walk<T, DK, true, false, 4>(a, stream) : launch_walk<T, DK, false, false, 4>(a, stream);
}

template <typename T, int DK, bool GROUPED>
hipError_t launch_gradients(const DeltaArgs& a, hipStream_t stream) {
  constexpr int kBytes = sizeof(GradientsLds<T, DK>);
  const auto kernel = delta_gradients<T, DK, GROUPED>;
  static std::atomic<uint64_t> asked{0};
  const hipError_t err = ask_lds(kernel, kBytes, asked);
  if (err != hipSuccess) return err;
  // As many workgroups as run side by side, each with one chunk after another.
  const int64_t items = a.batch * a.key_heads * a.chunks;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(items, 256 * (163840 / kBytes)))),
                     dim3(Chunk<T>::kTokens * 8), kBytes, stream, a);
  return hipGetLastError();
}

template <typename T, int DK>
hipError_t launch_backward(const DeltaArgs& a, hipStream_t stream) {
  hipError_t err = hipSuccess;
  if constexpr (kUnits<T>) err = launch_largest<T, true>(a, stream);
  if (err == hipSuccess && a.segments > 1) {
    err = launch_walk_back<T, DK, true, 4>(a, stream);
    if (err == hipSuccess) err = launch_join<DK, true>(a, stream);
  }
  if (err == hipSuccess) err = narrow_walk(a) ? launch_walk_back<T, DK, false, 2>(a, stream) : launch_walk_back<T, DK, false, 4>(a, stream);
  if (err != hipSuccess || a.chunks == 0) return err;
  return a.heads == a.key_heads ? launch_gradients<T, DK, false>(a, stream) : launch_gradients<T, DK, true>(a, stream);
}

template <typename T>
hipError_t backward_of(const DeltaArgs& a, hipStream_t stream) {
  return a.key_size <= 64 ? launch_backward<T, 64>(a, stream) : launch_backward<T, 128>(a, stream);
}

template <typename T>
hipError_t forward_of(const DeltaArgs& a, const DeltaPlan& p, hipStream_t stream) {
  return a.key_size <= 64 ? launch_forward<T, 64>(a, p, stream) : launch_forward<T, 128>(a, p, stream);
}

}  // namespace

int64_t delta_panel_bytes(int element_size) {
  const int64_t terms = element_size == 2 ? 2 : 1;
  return 2 * terms * delta_chunk(element_size) * 128;
}
int64_t delta_record_bytes(int element_size) {
  return element_size == 2 ? sizeof(Record<__bf16>) : sizeof(Record<float>);
}

hipError_t launch_delta_copy(convnd_hip_dtype dtype, const DeltaCopy& c, hipStream_t stream) {
  const int vec = dtype == CONVND_HIP_FLOAT32 ? 4 : 8;
  const int64_t work = c.batch * c.tokens * c.heads * (c.pitch / vec);
  if (work == 0) return hipSuccess;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((work + 255) / 256, 8192))), block(256);
  if (dtype == CONVND_HIP_FLOAT32)
    hipLaunchKernelGGL(delta_copy<float>, grid, block, 0, stream, c);
  else  // either 16-bit type: only zeros are made, the rest is moved
    hipLaunchKernelGGL(delta_copy<_Float16>, grid, block, 0, stream, c);
  return hipGetLastError();
}

hipError_t launch_delta(convnd_hip_dtype dtype, const DeltaArgs& a, const DeltaPlan& p, hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return forward_of<float>(a, p, stream);
    case CONVND_HIP_FLOAT16:
      return forward_of<_Float16>(a, p, stream);
    case CONVND_HIP_BFLOAT16:
      return forward_of<__bf16>(a, p, stream);
    default:
      return hipErrorInvalidValue;
  }
}

hipError_t launch_delta_backward(convnd_hip_dtype dtype, const DeltaArgs& a, hipStream_t stream) {
  switch (dtype) {
    case CONVND_HIP_FLOAT32:
      return backward_of<float>(a, stream);
    case CONVND_HIP_FLOAT16:
      return backward_of<_Float16>(a, stream);
    case CONVND_HIP_BFLOAT16:
      return backward_of<__bf16>(a, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace convnd
