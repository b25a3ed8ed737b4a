// Device helpers of the window and 8-bit cache kernels.
#pragma once

#include "common.hpp"
#include "launch.hpp"
#include "window.hpp"

namespace ifr {
namespace window {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int elt_bytes(int format) { return format == kBf16 ? 2 : 1; }

// Over the four 16-lane groups of a wave (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float groups_max(float x) { return pair_max32(pair_max16(x)); }
__device__ __forceinline__ float groups_sum(float x) { return pair_sum32(pair_sum16(x)); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {  // round to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}

// A wave-uniform f32 through the scalar cache.
__device__ __forceinline__ float sload_f32(const float* p) {
  return __int_as_float(sload(reinterpret_cast<const int32_t*>(p)));
}

// Bytes `lo` and `hi` (0 .. 3) of two words as a pair of bf16 (exact: e4m3 has 4
// significant bits, int8 8).
template <int kFormat, int kByte>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t a, uint32_t b) {
  static_assert(kFormat == kInt8, "e4m3 converts adjacent bytes");
  const float x = static_cast<float>(static_cast<int8_t>(a >> (8 * kByte)));
  const float y = static_cast<float>(static_cast<int8_t>(b >> (8 * kByte)));
  return pack_bf16(x, y);
}

// Four adjacent codes as two pairs of bf16.
template <int kFormat>
__device__ __forceinline__ u32x2_t codes4_bf16(uint32_t w) {
  if constexpr (kFormat == kE4m3) {
    return u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
  } else {
    return u32x2_t{pack_bf16(static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8))),
                   pack_bf16(static_cast<float>(static_cast<int8_t>(w >> 16)),
                             static_cast<float>(static_cast<int8_t>(w >> 24)))};
  }
}

// The same, times a power of two (or 0): exact where the product is a bf16 number, which a finite one
// above 2^-126 is.
template <int kFormat>
__device__ __forceinline__ u32x2_t codes4_scaled(uint32_t w, float scale) {
  if constexpr (kFormat == kE4m3) {
    return u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))};
  } else {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * scale;
    return u32x2_t{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
  }
}

// Non-finite values of V.  In a product of matrices they reach every column, also those
// that do not see them, as 0 * inf, and a weight's second part turns inf into NaN.  The
// sums show that; the walk is then done again with each fragment of V taken apart: its
// finite values, with 0 in the place of the others, go into the sum; 1 in the place of
// +inf and NaN, and of -inf and NaN, is multiplied by 1 for each position that a column
// sees, and what is above 0 there adds +inf, or -inf.
__device__ __forceinline__ bool all_finite(f32x4_t x) {
  bool f = true;
#pragma unroll
  for (int r = 0; r < 4; ++r) f = f && __builtin_fabsf(x[r]) < INFINITY;
  return f;
}
struct Parts {
  bf16x8_t finite, up, down;
};
__device__ __forceinline__ Parts taken_apart(const u32x4_t& v) {
  u32x4_t f, u, d;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = u[i] = d[i] = 0;
#pragma unroll
    for (int s = 0; s < 32; s += 16) {
      const uint32_t x = (v[i] >> s) & 0xFFFFu;
      const bool finite = (x & 0x7F80u) != 0x7F80u;
      f[i] |= (finite ? x : 0u) << s;
      u[i] |= (finite || x == 0xFF80u ? 0u : 0x3F80u) << s;
      d[i] |= (finite || x == 0x7F80u ? 0u : 0x3F80u) << s;
    }
  }
  return Parts{__builtin_bit_cast(bf16x8_t, f), __builtin_bit_cast(bf16x8_t, u), __builtin_bit_cast(bf16x8_t, d)};
}
template <typename Acc>
__device__ __forceinline__ Acc with_infinities(Acc acc, const Acc& up, const Acc& down) {
#pragma unroll
  for (int r = 0; r < static_cast<int>(sizeof(Acc) / 4); ++r) {
    acc[r] += up[r] > 0.0f ? INFINITY : 0.0f;
    acc[r] += down[r] > 0.0f ? -INFINITY : 0.0f;
  }
  return acc;
}
__device__ __forceinline__ f32x4_t add_infinities(f32x4_t acc, const Parts& v, bf16x8_t seen) {
  const f32x4_t none = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const f32x4_t up = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.up, seen, none, 0, 0, 0);
  const f32x4_t down = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.down, seen, none, 0, 0, 0);
  return with_infinities(acc, up, down);
}

// Whether a query at position p sees position j.
__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
  const int before = window == 0 ? -1 : p - window;  // no short circuits: they would be branches
  return (j <= p) & ((j > before) | (j < sinks));
}
// 1 for each of a lane's eight positions of a tile that a query at p sees, as P^T lies.
__device__ __forceinline__ bf16x8_t seen_ones(int p, int pos0, int g, int window, int sinks) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * i + e;
      w[i] |= (sees(p, pos0 + 16 * (j >> 2) + 4 * g + (j & 3), window, sinks) ? 0x3F80u : 0u) << (16 * e);
    }
  }
  return __builtin_bit_cast(bf16x8_t, w);
}
// Whether one of the queries p0 .. p1 sees a position of [j, j + n): any, or all of them all.
__device__ __forceinline__ bool any_seen(int p0, int p1, int j, int n, int window, int sinks) {
  return j <= p1 && (window == 0 || j + n - 1 > p0 - window || j < sinks);
}
__device__ __forceinline__ bool all_seen(int p0, int p1, int j, int n, int window, int sinks) {
  return j + n - 1 <= p0 && (window == 0 || j > p1 - window || j + n - 1 < sinks);
}

// Cache row of a tile's first position: tiles lie inside pages (of 32 rows at least).
__device__ __forceinline__ int64_t tile_row(const int32_t* rows, int pos0, int shift, int row_mask) {
  return static_cast<int64_t>(sload(rows + (pos0 >> shift))) + (pos0 & row_mask);
}

}  // namespace window
}  // namespace ifr
