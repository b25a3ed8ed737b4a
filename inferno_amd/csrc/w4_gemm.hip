// Products with 4-bit weights and group scales:
//   out[m][n] = bf16(sum_g scale[n][g] * sum_{k in group g} x[m][k] * value(code[n][k]))
// bf16 x [M][K], codes [N][K / 2] with the lower four bits first, bf16 scales
// [N][K / group].  Codes become bf16 numbers without rounding (int4: -8..7, e2m1:
// two significant bits), the matrix products sum a group in f32, and the group's scale
// multiplies that sum in f32: nothing is rounded before the result.
#include "common.hpp"
#include "step.hpp"

namespace ifr {
namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// What the products of a format have to be multiplied by at the end: int4 codes
// come out of v_cvt_off_f32_i4 as code / 16.
template <int kFmt>
constexpr float kUnit = kFmt == kW4Int4 ? 16.0f : 1.0f;

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  bf16x2_t p;
  p[0] = static_cast<__bf16>(lo);
  p[1] = static_cast<__bf16>(hi);
  return __builtin_bit_cast(uint32_t, p);
}

// The eight values of a word of codes, in order, over kUnit.
template <int kFmt>
__device__ __forceinline__ bf16x8_t w4_values(uint32_t w) {
  uint4 r;
  if constexpr (kFmt == kW4Int4) {
    const uint32_t h = w >> 4;
    r.x = pack_bf16(__builtin_amdgcn_cvt_off_f32_i4(w), __builtin_amdgcn_cvt_off_f32_i4(h));
    r.y = pack_bf16(__builtin_amdgcn_cvt_off_f32_i4(w >> 8),
                    __builtin_amdgcn_cvt_off_f32_i4(h >> 8));
    r.z = pack_bf16(__builtin_amdgcn_cvt_off_f32_i4(w >> 16),
                    __builtin_amdgcn_cvt_off_f32_i4(h >> 16));
    r.w = pack_bf16(__builtin_amdgcn_cvt_off_f32_i4(w >> 24),
                    __builtin_amdgcn_cvt_off_f32_i4(h >> 24));
  } else {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
  }
  return __builtin_bit_cast(bf16x8_t, r);
}

// One wave: 16 columns of the output for 16 tokens, all of k, straight from memory.
// v_mfma_f32_16x16x32_bf16 with x as A (lane l: token l % 16) and the weight as B (column
// l % 16), k 8 * (l / 16) .. + 7.
template <int kFmt>
__global__ __launch_bounds__(256) void w4_gemm_wave_kernel(
    const uint16_t* __restrict__ x, const uint8_t* __restrict__ codes,
    const uint16_t* __restrict__ scales, uint16_t* __restrict__ out, int M, int N, int K,
    int group) {
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int n0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
  if (n0 >= N) return;
  const int m0 = blockIdx.y * 16;
  const int64_t n = min(n0 + r, N - 1);
  const uint16_t* xp = x + static_cast<int64_t>(min(m0 + r, M - 1)) * K + 8 * q;
  const uint8_t* wp = codes + n * (K / 2) + 4 * q;
  const uint16_t* sp = scales + n * (K / group);
  f32x4_t sum{0.0f, 0.0f, 0.0f, 0.0f};
  for (int g = 0; g < K / group; ++g) {
    f32x4_t acc{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = g * group; k < (g + 1) * group; k += 32) {
      const uint4 a = *reinterpret_cast<const uint4*>(xp + k);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(wp + k / 2);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                    w4_values<kFmt>(w), acc, 0, 0, 0);
    }
    const float s = bf16_to_f32(sp[g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(s, acc[i], sum[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + 4 * q + i;
    if (m < M && n0 + r < N)
      out[static_cast<int64_t>(m) * N + n0 + r] =
          static_cast<uint16_t>(f32_to_bf16_bits(kUnit<kFmt> * sum[i]));
  }
}

}  // namespace

int64_t w4_gemm_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_w4_gemm(const W4Args& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.N + 63) / 64), static_cast<unsigned>((a.M + 15) / 16));
  const int m = static_cast<int>(a.M), n = static_cast<int>(a.N), k = static_cast<int>(a.K);
  if (a.format == kW4Int4)
    hipLaunchKernelGGL((w4_gemm_wave_kernel<kW4Int4>), grid, dim3(256), 0, stream, a.x, a.codes,
                       a.scales, a.out, m, n, k, a.group);
  else
    hipLaunchKernelGGL((w4_gemm_wave_kernel<kW4E2m1>), grid, dim3(256), 0, stream, a.x, a.codes,
                       a.scales, a.out, m, n, k, a.group);
  return hipGetLastError();
}

}  // namespace ifr
