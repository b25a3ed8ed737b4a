// Products with 4-bit weights and group scales:
//   out[m][n] = bf16(sum_g scale[n][g] * sum_{k in group g} x[m][k] * value(code[n][k]))
// bf16 x [M][K], codes [N][K / 2] with the lower four bits first, bf16 scales
// [N][K / group].  Codes become bf16 numbers without rounding (int4: -8..7, e2m1:
// two significant bits), the matrix products sum a group in f32, and the group's scale
// multiplies that sum in f32: nothing is rounded before the result.
#include <algorithm>
#include <type_traits>

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

// The low four bits of byte B as a number of two's complement over 16.  (The whole byte is asked
// for, though the conversion takes its low half, because that is one operand selection.)
template <int B>
__device__ __forceinline__ float code_byte(uint32_t w) {
  return __builtin_amdgcn_cvt_off_f32_i4((w >> (8 * B)) & 0xFFu);
}

// The eight values of a word of codes, in order, over kUnit.
template <int kFmt>
__device__ __forceinline__ bf16x8_t w4_values(uint32_t w) {
  uint4 r;
  if constexpr (kFmt == kW4Int4) {
    uint32_t h = w >> 4;
    asm("" : "+v"(h));  // no instruction: keeps the shift from being taken apart, byte by byte
    r.x = pack_bf16(code_byte<0>(w), code_byte<0>(h));
    r.y = pack_bf16(code_byte<1>(w), code_byte<1>(h));
    r.z = pack_bf16(code_byte<2>(w), code_byte<2>(h));
    r.w = pack_bf16(code_byte<3>(w), code_byte<3>(h));
  } else {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
  }
  return __builtin_bit_cast(bf16x8_t, r);
}

// A step is 128 columns of 16 weight rows: lane l holds 16 bytes, columns 32 q .. + 31 of row
// r, for r = l % 16 and q = l / 16, and v_mfma_f32_16x16x32_bf16 takes the weight as its B
// operand (column r of the output, eight k of quarter q), so that a lane holds codes of one
// row and one scale multiplies its sums.  A matrix product adds over the quarters, so groups
// of less than 128 have to be moved to one register first: swaps between the quarters
// (transposing words, four of a lane, with quarters) leave word j of all lanes in group
// 32 j / kGroup.  x has to come in the same order: x_offset is the k, within the step, of the
// eight values that lane quarter q multiplies with word j.
template <int kGroup>
__device__ __forceinline__ int x_offset(int j, int q) {
  if constexpr (kGroup == 128) return 32 * q + 8 * j;
  if constexpr (kGroup == 64) return 64 * (j >> 1) + 8 * (j & 1) + 32 * (q & 1) + 16 * (q >> 1);
  return 32 * j + 8 * q;
}
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
template <int kGroup>
__device__ __forceinline__ void order_words(uint4& w) {
  if constexpr (kGroup < 128) {
    swap32(w.x, w.z);
    swap32(w.y, w.w);
  }
  if constexpr (kGroup < 64) {
    swap16(w.x, w.y);
    swap16(w.z, w.w);
  }
}

// The scales of a step of one row: 128 / kGroup bf16 numbers.
template <int kGroup>
struct StepScales {
  uint32_t v[kGroup == 32 ? 2 : 1];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (kGroup == 128) v[0] = *p;
    if constexpr (kGroup == 64) v[0] = *reinterpret_cast<const uint32_t*>(p);
    if constexpr (kGroup == 32) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      v[0] = u.x, v[1] = u.y;
    }
  }
  __device__ __forceinline__ float get(int g) const {
    return g & 1 ? bf16_hi(v[g >> 1]) : bf16_lo(v[g >> 1]);
  }
};

// sum += the step's products, 16 tokens.  R: the values of a lane that stand for tokens (token t
// is row 4 (t / R) + t % R: with at most four tokens one value a lane has to be scaled, not four).
template <int kFmt, int kGroup, int R>
__device__ __forceinline__ void multiply_step(const bf16x8_t (&xf)[4], uint4 w,
                                              const StepScales<kGroup>& s, f32x4_t& sum) {
  order_words<kGroup>(w);
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
  constexpr int kPer = kGroup / 32;  // words of a group
#pragma unroll
  for (int g = 0; g < 4 / kPer; ++g) {
    f32x4_t acc{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[g * kPer + j], w4_values<kFmt>(word[g * kPer + j]),
                                                    acc, 0, 0, 0);
    const float sc = s.get(g);
#pragma unroll
    for (int i = 0; i < R; ++i) sum[i] = __builtin_fmaf(sc, acc[i], sum[i]);
  }
}

template <int R>
__device__ __forceinline__ int token_of_row(int row) {
  return (row >> 2) * R + min(row & 3, R - 1);
}

// Up to 16 tokens and few columns: a workgroup takes `cols` columns (NT tiles of 16), its waves
// take ST steps of k in turn, and their sums meet in LDS, added in wave order.  Every load of
// ST steps is under way before the first product; x comes from L2.
// Bound by latency: one token x 2,816 x 4,096 (int4, groups of 128; 6.1 MB) takes 5.1 us, one launch of
// 256 workgroups of 11 columns whose waves have one round of loads each.
template <int kFmt, int kGroup, int NT, int ST, int R>
__global__ __launch_bounds__(1024) void w4_few_kernel(W4Args a, int cols) {
  __shared__ float part[16][NT * R][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int M = static_cast<int>(a.M), N = static_cast<int>(a.N), K = static_cast<int>(a.K);
  const int n0 = blockIdx.x * cols, steps = K / 128;
  const uint16_t* xp = a.x + static_cast<int64_t>(min(token_of_row<R>(r), M - 1)) * K;
  const uint8_t* wp[NT];
  const uint16_t* sp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = min(n0 + min(16 * t + r, cols - 1), N - 1);
    wp[t] = a.codes + n * (K / 2) + 16 * q;
    sp[t] = a.scales + n * (K / kGroup);
  }
  f32x4_t sum[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) sum[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = wave * ST; s0 < steps; s0 += waves * ST) {
    uint4 w[ST][NT];
    StepScales<kGroup> sc[ST][NT];
    bf16x8_t xf[ST][4];
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      const int s = min(s0 + i, steps - 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[i][t] = *reinterpret_cast<const uint4*>(wp[t] + 64 * s);
        sc[i][t].load(sp[t] + s * (128 / kGroup));
      }
    }
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      const int s = min(s0 + i, steps - 1);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xf[i][j] = *reinterpret_cast<const bf16x8_t*>(xp + 128 * s + x_offset<kGroup>(j, q));
    }
    __builtin_amdgcn_sched_barrier(0);  // every load ahead of the first product
#pragma unroll
    for (int i = 0; i < ST; ++i)
      if (s0 + i < steps)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          multiply_step<kFmt, kGroup, R>(xf[i], w[i][t], sc[i][t], sum[t]);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < R; ++i) part[wave][t * R + i][lane] = sum[t][i];
  __syncthreads();
  for (int e = threadIdx.x; e < NT * R * 64; e += blockDim.x) {
    const int v = e >> 6, l = e & 63;
    const int m = (l >> 4) * R + v % R, c = 16 * (v / R) + (l & 15);
    if (m >= M || c >= cols || n0 + c >= N) continue;
    float total = part[0][v][l];
    for (int z = 1; z < waves; ++z) total = total + part[z][v][l];
    a.out[static_cast<int64_t>(m) * N + n0 + c] =
        static_cast<uint16_t>(pack_bf16(kUnit<kFmt> * total, 0.0f));
  }
}

// The scales of a tile's 16 rows, through LDS: a window of 64 bytes a row (kGroup / 4 steps) is one
// load of 16 bytes a lane, where a load for each step asks for the 16 rows' lines again every
// time (one token x 262,144 x 2,816, groups of 128: 93 us with a load a step).
constexpr int kScalePitch = 80;  // bytes of a row's window in LDS: 20 banks apart
template <int kGroup>
struct ScaleWindow {
  static constexpr int kSteps = kGroup / 4;
  static constexpr int kStepBytes = 256 / kGroup;
  // Row r's window from byte `at` of its scales (`row_bytes` a row; rows from n0).  Windows may
  // reach past a row's end, into the next rows, but not past the N rows.
  static __device__ __forceinline__ uint4 load(const W4Args& a, int64_t n0, int row_bytes, int at,
                                               int r, int q) {
    const uint8_t* base = reinterpret_cast<const uint8_t*>(a.scales);
    const int64_t total = a.N * row_bytes;
    const int64_t off = (n0 + r) * row_bytes + at + 16 * q;
    uint4 v = make_uint4(0, 0, 0, 0);
    if ((n0 + 15) * row_bytes + at + 64 <= total) {  // wave-uniform
      __builtin_memcpy(&v, base + off, 16);
    } else {
      uint32_t d[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (off + 2 * i + 2 <= total)
          d[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(base + off + 2 * i))
                      << (16 * (i % 2));
      v = make_uint4(d[0], d[1], d[2], d[3]);
    }
    return v;
  }
};

// Up to four tokens against many columns: a wave takes NT tiles of 16 columns over all of k, with x in
// LDS, a chunk of k at a time, and the codes straight from memory into registers, two steps
// ahead.
// Bound by HBM reads: one token x 262,144 x 2,816 (int4, groups of 128) takes 66 us, 5.8 TB/s, and reads
// 1.0 times its 381 MB.
constexpr int kStreamWaves = 8;
constexpr int kStreamTiles = 2;  // NT
constexpr int kStreamLds = 56 * 1024;  // x: two workgroups a CU
template <int kFmt, int kGroup>
__global__ __launch_bounds__(64 * kStreamWaves, 4) void w4_stream_kernel(W4Args a, int chunk_steps) {
  using Window = ScaleWindow<kGroup>;
  constexpr int NT = kStreamTiles;
  extern __shared__ __align__(16) uint8_t xs[];
  __shared__ __align__(16) uint8_t scale_lds[kStreamWaves * NT * 16 * kScalePitch];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int M = static_cast<int>(a.M), N = static_cast<int>(a.N), K = static_cast<int>(a.K);
  const int n0 = (blockIdx.x * kStreamWaves + wave) * 16 * NT;
  const int steps = K / 128;
  const int pitch = 256 * chunk_steps + 16;  // rows four banks apart
  uint8_t* my_scales = scale_lds + wave * NT * 16 * kScalePitch + r * kScalePitch;

  const uint8_t* wp[NT];
  uint4 w[2][NT], window[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = min(n0 + 16 * t + r, N - 1);
    wp[t] = a.codes + n * (K / 2) + 16 * q;
  }
  const int row_bytes = K / kGroup * 2;
  auto load_window = [&](int s) {
    if (s >= steps) return;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      window[t] = Window::load(a, n0 + 16 * t, row_bytes, s * Window::kStepBytes, r, q);
  };
  // Two steps, the halves of a row's 128-byte lines, behind each other: with a step of the first
  // half between them lines are fetched twice (75 us against 68 at 262,144 x 2,816).
  auto load = [&](int s) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h][t] = *reinterpret_cast<const uint4*>(wp[t] + 64 * min(s + h, steps - 1));
  };
  load_window(0);
  load(0);

  f32x4_t sum[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) sum[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const uint8_t* xrow = xs + min(token_of_row<1>(r), M - 1) * pitch;
  auto multiply = [&](const uint4 (&now)[NT], int s, int in_chunk) {
    bf16x8_t xf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      xf[j] = *reinterpret_cast<const bf16x8_t*>(xrow + 256 * in_chunk + 2 * x_offset<kGroup>(j, q));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      StepScales<kGroup> sc;
      sc.load(reinterpret_cast<const uint16_t*>(my_scales + t * 16 * kScalePitch +
                                                s % Window::kSteps * Window::kStepBytes));
      multiply_step<kFmt, kGroup, 1>(xf, now[t], sc, sum[t]);
    }
  };
  for (int c0 = 0; c0 < steps; c0 += chunk_steps) {
    const int here = min(chunk_steps, steps - c0);
    if (c0) __syncthreads();
    // Rows of `here` steps of 256 bytes, 16 bytes a thread.
    const int per = 16 * here;
    for (int i = threadIdx.x; i < M * per; i += 64 * kStreamWaves) {
      const int m = i / per, at = i - m * per;
      *reinterpret_cast<uint4*>(xs + m * pitch + 16 * at) = *reinterpret_cast<const uint4*>(
          a.x + static_cast<int64_t>(m) * K + 128 * c0 + 8 * at);
    }
    __syncthreads();
    for (int s = c0; s < c0 + here; s += 2) {
      if (s % Window::kSteps == 0) {  // the wave's own LDS: its accesses are in order
#pragma unroll
        for (int t = 0; t < NT; ++t)
          *reinterpret_cast<uint4*>(my_scales + t * 16 * kScalePitch + 16 * q) = window[t];
        load_window(s + Window::kSteps);
      }
      uint4 now[2][NT];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) now[h][t] = w[h][t];
      load(s + 2);
      multiply(now[0], s, s - c0);
      if (s + 1 < c0 + here) multiply(now[1], s + 1, s + 1 - c0);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = n0 + 16 * t + r;
    if (n < N && q < M)
      a.out[static_cast<int64_t>(q) * N + n] =
          static_cast<uint16_t>(pack_bf16(kUnit<kFmt> * sum[t][0], 0.0f));
  }
}

// 17 to 64 tokens, and 5 to 16 against many columns or from k past 4,096: as the stream kernel, with x in units of two steps that go
// from memory into LDS by themselves (global_load_lds), one unit ahead, so that W waves of NT tiles
// share it behind one barrier a unit.  The codes of a unit are loaded again as soon as the unit
// before is multiplied, two units ahead of their use.
//
// Bound by no one part: 64 tokens x 262,143 x 2,816 (e2m1, groups of 32) takes 160 us, 2.9 TB/s, with the matrix
// units busy for 26 %, a CU's vector instructions for about half of the time and 43 % of its waves'
// time spent waiting; without its stores, its loads of x or its reads of LDS it takes 4 to 13 % less.
//
// 16-byte chunk c of x row r lies at c ^ (r % 16), so that the 16 rows of a quarter of a
// fragment read lie in 16 different bank groups.
typedef __attribute__((address_space(3))) void lds_void_t;
template <int kFmt, int kGroup, int TM, int NT, int W, bool kSplit>
__global__ __launch_bounds__(64 * W, W == 16 ? 4 : 2) void w4_batch_kernel(W4Args a, int span_steps,
                                                              int64_t part_stride) {
  using Window = ScaleWindow<kGroup>;
  constexpr int kUnitBytes = TM * 16 * 512;
  constexpr int kLoads = (TM * 8 + W - 1) / W;  // 1 KiB loads (two rows) of a wave a unit
  __shared__ __align__(16) uint8_t x0[kUnitBytes];
  __shared__ __align__(16) uint8_t x1[kUnitBytes];
  __shared__ __align__(16) uint8_t scale_lds[W * NT * 16 * kScalePitch];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int M = static_cast<int>(a.M), N = static_cast<int>(a.N), K = static_cast<int>(a.K);
  const int n0 = (blockIdx.x * W + wave) * 16 * NT;
  const int first = blockIdx.y * span_steps;
  const int steps = min(span_steps, K / 128 - first);
  const int units = (steps + 1) / 2;
  uint8_t* my_scales = scale_lds + wave * NT * 16 * kScalePitch + r * kScalePitch;

  const uint8_t* wp[NT];
  uint4 w[2][2][NT], window[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = min(n0 + 16 * t + r, N - 1);
    wp[t] = a.codes + n * (K / 2) + 64 * first + 16 * q;
  }
  const int row_bytes = K / kGroup * 2;
  auto load_window = [&](int s) {
    if (s >= steps) return;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      window[t] = Window::load(a, n0 + 16 * t, row_bytes, (first + s) * Window::kStepBytes, r, q);
  };
  auto load_half = [&](int set, int u, int t) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[set][h][t] = *reinterpret_cast<const uint4*>(wp[t] + 64 * min(2 * u + h, steps - 1));
  };
  // x rows 2 i and 2 i + 1 of unit u; rows past M and k past K repeat others (not used).
  const uint16_t* xsrc[kLoads];
  int xcol[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = 2 * (wave + W * i) + (lane >> 5);
    xsrc[i] = a.x + static_cast<int64_t>(min(row, M - 1)) * K;
    xcol[i] = 128 * first + 8 * ((lane & 31) ^ (row & 15));
  }
  auto load_x = [&](int u, uint8_t* buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (TM * 8 % W == 0 || wave + W * i < TM * 8)
        __builtin_amdgcn_global_load_lds(
            static_cast<const void*>(xsrc[i] + min(xcol[i] + 256 * u, K - 8)),
            (lds_void_t*)(buf + 1024 * (wave + W * i)), 16, 0, 0);
  };

  f32x4_t sum[NT][TM];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < TM; ++m) sum[t][m] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto multiply = [&](uint4 (&now)[NT], int s, int half, const uint8_t* xb) {
    StepScales<kGroup> sc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      sc[t].load(reinterpret_cast<const uint16_t*>(my_scales + t * 16 * kScalePitch +
                                                   s % Window::kSteps * Window::kStepBytes));
#pragma unroll
    for (int t = 0; t < NT; ++t) order_words<kGroup>(now[t]);
    constexpr int kPer = kGroup / 32;  // words of a group
#pragma unroll
    for (int g = 0; g < 4 / kPer; ++g) {
      f32x4_t acc[NT][TM];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[t][m] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = g * kPer; j < (g + 1) * kPer; ++j) {
        bf16x8_t xf[TM];
#pragma unroll
        for (int m = 0; m < TM; ++m)
          xf[m] = *reinterpret_cast<const bf16x8_t*>(
              xb + 512 * (16 * m + r) + 256 * half + 16 * ((x_offset<kGroup>(j, q) / 8) ^ r));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t word = j == 0 ? now[t].x : j == 1 ? now[t].y : j == 2 ? now[t].z : now[t].w;
          const bf16x8_t b = w4_values<kFmt>(word);
#pragma unroll
          for (int m = 0; m < TM; ++m)
            acc[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[m], b, acc[t][m], 0, 0, 0);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float scale = sc[t].get(g);
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sum[t][m][i] = __builtin_fmaf(scale, acc[t][m][i], sum[t][m][i]);
      }
    }
  };

  load_window(0);
  load_x(0, x0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int set = 0; set < 2; ++set)
#pragma unroll
    for (int t = 0; t < NT; ++t) load_half(set, set, t);
  auto unit = [&](int set, int u, const uint8_t* cur, uint8_t* next) {
    // x of unit u has landed when only the codes loaded behind it are outstanding (2 NT loads at
    // least), and nobody reads the buffer of unit u - 1 any more.
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NT) : "memory");
    load_x(min(u + 1, units - 1), next);
    __builtin_amdgcn_sched_barrier(0);
    const int s = 2 * u;
    if (s % Window::kSteps == 0) {  // the wave's own LDS: its accesses are in order
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<uint4*>(my_scales + t * 16 * kScalePitch + 16 * q) = window[t];
      load_window(s + Window::kSteps);
    }
    multiply(w[set][0], s, 0, cur);
    if (s + 1 < steps) multiply(w[set][1], s + 1, 1, cur);
#pragma unroll
    for (int t = 0; t < NT; ++t) load_half(set, u + 2, t);
  };
  for (int u = 0; u < units; u += 2) {
    unit(0, u, x0, x1);
    if (u + 1 < units) unit(1, u + 1, x1, x0);
  }
  // No load may still be on its way into LDS when the workgroup ends.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = n0 + 16 * t + r;
    if (n >= N) continue;
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = 16 * m + 4 * q + i;
        if (token >= M) continue;
        const int64_t o = static_cast<int64_t>(token) * N + n;
        if constexpr (kSplit)
          a.workspace[blockIdx.y * part_stride + o] = sum[t][m][i];
        else
          a.out[o] = static_cast<uint16_t>(pack_bf16(kUnit<kFmt> * sum[t][m][i], 0.0f));
      }
  }
}

// out = bf16(unit * (part[0] + part[1] + ...)), four outputs a thread, added in order.
__global__ __launch_bounds__(256) void w4_reduce_kernel(const float* __restrict__ part,
                                                        uint16_t* __restrict__ out, int64_t count,
                                                        int64_t part_stride, int splits,
                                                        float unit) {
  const int64_t i = 4 * (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x);
  if (i >= count) return;
  float4 s = *reinterpret_cast<const float4*>(part + i);
#pragma unroll 4
  for (int z = 1; z < splits; ++z) {
    const float4 v = *reinterpret_cast<const float4*>(part + z * part_stride + i);
    s.x = s.x + v.x, s.y = s.y + v.y, s.z = s.z + v.z, s.w = s.w + v.w;
  }
  const uint2 p = make_uint2(pack_bf16(unit * s.x, unit * s.y), pack_bf16(unit * s.z, unit * s.w));
  if (i + 4 <= count) {
    *reinterpret_cast<uint2*>(out + i) = p;
  } else {
    const uint16_t v[4] = {static_cast<uint16_t>(p.x), static_cast<uint16_t>(p.x >> 16),
                           static_cast<uint16_t>(p.y), 0};
    for (int j = 0; i + j < count; ++j) out[i + j] = v[j];
  }
}

// More than 64 tokens: a workgroup of 4 waves (2 x 2) computes 64 MB tokens x 128 columns, each wave MB x 2
// blocks of v_mfma_f32_32x32x16_bf16.  x is A (lane l: token l % 32, eight k of half l / 32) and
// travels, 64 k a chunk, from memory into one of three LDS buffers (global_load_lds): while chunk c is
// multiplied c + 1 lands and c + 2 is issued, so one barrier a chunk publishes c and frees the buffer of
// c + 2.  The weight is B (column l % 32).  Its codes come the same way, 128 k (two chunks) a
// stage, two stages ahead, and become bf16 in registers; scales 16 bytes a row at a time.  Straight
// into registers a load would touch 32 lines for 1 KiB of codes, and again for the scales, which
// costs more of the CU's address unit than the products take (142 against 124 us at 4,099 x 2,816 x 4,096;
// now 115, 822 TFLOP/s, matrix units 34 % busy: the conversions of the codes and the fma of the scales take
// the time, on the same SIMDs).
//
// A group's products are summed by themselves and then scaled into the total: exact products, at
// the price of as many registers again and of an fma for each sum and group.  Rounding scale times
// code to bf16 instead would need neither, and put 2^-9 of every weight into the result.
//
// k within a chunk comes in the order in which a lane holds its words: word j of half h is k
// 32 h + 8 j; with groups of 32 two swaps between the halves move each group into two words, k
// 32 (j / 2) + 16 h + 8 (j % 2).
typedef float f32x16_t __attribute__((ext_vector_type(16)));
constexpr int kTileThreads = 256;
constexpr int kTileN = 128;
constexpr int kRowBytes = 128;  // of x in LDS: 64 k; 16-byte chunk q of row r lies at q ^ ((r / 2) % 8)
template <int kFmt, int kGroup, int MB, bool kSplit>
__global__ __launch_bounds__(kTileThreads) __attribute__((amdgpu_waves_per_eu(MB == 1 ? 3 : 2)))
void w4_tile_kernel(W4Args a, int span_steps, int64_t part_stride, int m_tiles, int n_tiles) {
  constexpr int BM = 64 * MB;
  constexpr int kLoads = BM / 32;             // 1 KiB loads (8 rows) of x by a wave a chunk
  __shared__ __align__(16) uint8_t buf0[BM * kRowBytes];
  __shared__ __align__(16) uint8_t buf1[BM * kRowBytes];
  __shared__ __align__(16) uint8_t buf2[BM * kRowBytes];
  __shared__ __align__(16) uint8_t codes0[kTileN * 64];
  __shared__ __align__(16) uint8_t codes1[kTileN * 64];
  __shared__ __align__(16) uint8_t codes2[kTileN * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = lane >> 5, r32 = lane & 31;
  const int M = static_cast<int>(a.M), N = static_cast<int>(a.N), K = static_cast<int>(a.K);

  // Workgroups go to the 8 XCDs round robin: XCD b % 8 takes a contiguous run of tiles, ordered in
  // bands of 8 token tiles (token tile fastest inside a band).
  const int tiles = m_tiles * n_tiles, per = (tiles + 7) / 8;
  const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || t >= tiles) return;  // block-uniform
  constexpr int kBand = 8;
  const int band = t / (kBand * n_tiles), in_band = t - band * kBand * n_tiles;
  const int height = min(kBand, m_tiles - band * kBand);
  const int m0 = (band * kBand + in_band % height) * BM;
  const int n0 = (in_band / height) * kTileN;
  const int k0 = blockIdx.y * span_steps * 128;
  const int nk = min(span_steps * 128, K - k0) / 64;  // chunks, an even number
  const int wm = (wave & 1) * (BM / 2), wn = (wave >> 1) * 64;

  const uint16_t* src[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = 8 * (wave + 4 * i) + (lane >> 3);
    src[i] = a.x + static_cast<int64_t>(min(m0 + r, M - 1)) * K + k0 + 8 * ((lane & 7) ^ ((r >> 1) & 7));
  }
  // Load i of this wave moves 16 weight rows, 64 bytes each: lane p row p / 4, 16-byte chunk p % 4,
  // which lies at (p % 4) ^ ((row / 4) % 4), so that 16 rows' chunks are in 16 bank groups.
  const uint8_t* csrc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = 16 * (wave + 4 * i) + (lane >> 2);
    csrc[i] = a.codes + static_cast<int64_t>(min(n0 + row, N - 1)) * (K / 2) + k0 / 2 +
              16 * ((lane & 3) ^ ((row >> 2) & 3));
  }
  auto load_codes = [&](int i, int stage, uint8_t* buf) {
    __builtin_amdgcn_global_load_lds(static_cast<const void*>(csrc[i] + 64 * min(stage, nk / 2 - 1)),
                                     (lds_void_t*)(buf + 1024 * (wave + 4 * i)), 16, 0, 0);
  };
  // Lane l loads the scales of column wn + l, a stage at a time.
  const uint16_t* sp = a.scales + static_cast<int64_t>(min(n0 + wn + lane, N - 1)) * (K / kGroup) + k0 / kGroup;
  StepScales<kGroup> sc[3];
  auto load_scales = [&](int set, int stage) { sc[set].load(sp + min(stage, nk / 2 - 1) * (128 / kGroup)); };
  auto load_x = [&](int c, uint8_t* buf) {
    c = min(c, nk - 1);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(src[i] + 64 * c),
                                       (lds_void_t*)(buf + 8 * (wave + 4 * i) * kRowBytes), 16, 0, 0);
  };

  f32x16_t sum[MB][2], acc[MB][2];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int v = 0; v < 16; ++v) sum[m][b][v] = 0.0f;

  const int lane_sw = (r32 >> 1) & 7;
  auto chunk = [&](int c, const uint8_t* cur, uint8_t* next, const uint8_t* codes, uint8_t* next_codes,
                   int set, auto even) {
    constexpr bool kEven = decltype(even)::value;
    constexpr bool kStarts = kEven || kGroup != 128;  // a group
    // Chunk c and its codes have landed when only what was loaded during chunk c - 1 is outstanding.
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kEven ? kLoads + 1 : kLoads + 2)
                 : "memory");
    if constexpr (kEven) load_scales((set + 2) % 3, c / 2 + 2);
    load_codes(kEven ? 0 : 1, c / 2 + 2, next_codes);
    load_x(c + 2, next);
    __builtin_amdgcn_sched_barrier(0);
    uint4 now[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int row = wn + 32 * b + r32;
      now[b] = *reinterpret_cast<const uint4*>(codes + 64 * row +
                                               16 * (((kEven ? 0 : 2) + half) ^ ((row >> 2) & 3)));
    }
    // The chunk's scales: those of the lower lanes are block 0's, those of the upper block 1's.
    const auto both = __builtin_amdgcn_permlane32_swap(sc[set].v[kGroup == 32 && !kEven ? 1 : 0],
                                                       sc[set].v[kGroup == 32 && !kEven ? 1 : 0], false, false);
    if constexpr (kGroup == 32)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        swap32(now[b].x, now[b].z);
        swap32(now[b].y, now[b].w);
      }
    bf16x8_t xf[2][MB], wf[2][2];
    auto fragments = [&](int j) {
      const int q = kGroup == 32 ? 4 * (j >> 1) + (j & 1) + 2 * half : 4 * half + j;
#pragma unroll
      for (int m = 0; m < MB; ++m)
        xf[j & 1][m] = *reinterpret_cast<const bf16x8_t*>(cur + (wm + 32 * m + r32) * kRowBytes +
                                                          16 * (q ^ lane_sw));
#pragma unroll
      for (int b = 0; b < 2; ++b)
        wf[j & 1][b] = w4_values<kFmt>(j == 0 ? now[b].x : j == 1 ? now[b].y : j == 2 ? now[b].z : now[b].w);
    };
    fragments(0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      if (j < 3) fragments(j + 1);
      const bool first = kGroup == 32 ? j % 2 == 0 : j == 0 && kStarts;
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          acc[m][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xf[j & 1][m], wf[j & 1][b],
                                                              first ? f32x16_t{} : acc[m][b], 0, 0, 0);
      const bool last = kGroup == 32 ? j % 2 == 1 : j == 3 && (kGroup == 64 || !kEven);
      if (last) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const bool upper = kGroup == 32 ? j == 3 : kGroup == 64 ? !kEven : false;
          const float scale = upper ? bf16_hi(both[b]) : bf16_lo(both[b]);
#pragma unroll
          for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int v = 0; v < 16; ++v) sum[m][b][v] = __builtin_fmaf(scale, acc[m][b][v], sum[m][b][v]);
        }
      }
    }
  };
  load_scales(0, 0);
  load_codes(0, 0, codes0);
  load_codes(1, 0, codes0);
  load_x(0, buf0);
  __builtin_amdgcn_sched_barrier(0);
  load_scales(1, 1);
  load_codes(0, 1, codes1);
  load_codes(1, 1, codes1);
  load_x(1, buf1);
  const std::true_type even;
  const std::false_type odd;
  int c = 0;
  for (; c + 6 <= nk; c += 6) {
    chunk(c, buf0, buf2, codes0, codes2, 0, even);
    chunk(c + 1, buf1, buf0, codes0, codes2, 0, odd);
    chunk(c + 2, buf2, buf1, codes1, codes0, 1, even);
    chunk(c + 3, buf0, buf2, codes1, codes0, 1, odd);
    chunk(c + 4, buf1, buf0, codes2, codes1, 2, even);
    chunk(c + 5, buf2, buf1, codes2, codes1, 2, odd);
  }
  if (c < nk) {
    chunk(c, buf0, buf2, codes0, codes2, 0, even);
    chunk(c + 1, buf1, buf0, codes0, codes2, 0, odd);
  }
  if (c + 2 < nk) {
    chunk(c + 2, buf2, buf1, codes1, codes0, 1, even);
    chunk(c + 3, buf0, buf2, codes1, codes0, 1, odd);
  }
  // The scales that the last chunks load are of no use, but the waits count those loads.
#pragma unroll
  for (int set = 0; set < 3; ++set)
#pragma unroll
    for (uint32_t v : sc[set].v) asm volatile("" ::"v"(v));
  // No load may still be on its way into LDS when the workgroup ends.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // C layout: value 4 j + i of a block is token 8 j + 4 half + i, column r32.
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int n = n0 + wn + 32 * b + r32;
      if (n >= N) continue;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int token = m0 + wm + 32 * m + 8 * (v >> 2) + 4 * half + (v & 3);
        if (token >= M) continue;
        const int64_t o = static_cast<int64_t>(token) * N + n;
        if constexpr (kSplit)
          a.workspace[blockIdx.y * part_stride + o] = sum[m][b][v];
        else
          a.out[o] = static_cast<uint16_t>(pack_bf16(kUnit<kFmt> * sum[m][b][v], 0.0f));
      }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

enum Kind : int { kFew, kStream, kBatch, kTile };
struct Plan {
  Kind kind;
  int nt, waves;  // tiles of 16 columns a wave, and waves of a workgroup; of kTile nt 64s of tokens
  int splits;     // spans of k with partial sums in the workspace
  int span;       // steps of 128 k in one
};

// From 32,768 columns there are 128 workgroups of 256 columns or more, and the kernels that
// stream them.  us for one token, columns over waves | streams: k of 2,816, int4 in groups of 128, 32,768 columns 15.9 | 17.8,
// 50,257 23.8 | 19.6, 128,256 51.6 | 38.2; k of 4,096 25.5 | 23.0, 41.7 | 24.1, 93.3 | 51.0.
constexpr int64_t kManyColumns = 32768;

// Tokens of a tile and spans of k past 64 tokens: the cheapest by a model of the launch, fitted to 65
// to 1,024 tokens, both tiles and 1 to 16 spans at N = 2,816, K = 4,096, int4 in groups of 128 alone: 32
// steps of up to 256 tiles take 33 us (64 tokens) or 45 (128), of each 256 of more tiles, of which a CU
// has several at once, 23 or 43; spans add a launch and the partial sums' way out and back.
// It picks the best measured or one within 13 % of it: 65 tokens 15.1 us (best 13.4), 256 20.4
// (19.6), 512 28.0 (28.0; one span of 128 tokens 48.3), 1,024 43.4 (43.4).
// Spans only up to 768 workgroups, which bounds the workspace for every M.
constexpr int kTileSpans = 16;
constexpr int64_t kTileBlocks = 768;
Plan tile_plan(int64_t M, int64_t N, int steps) {
  Plan best{kTile, 2, 4, 1, steps};
  double best_us = 1e30;
  for (int mb = 1; mb <= 2; ++mb) {
    const int64_t tiles = ceil_div(M, 64 * mb) * ceil_div(N, kTileN);
    for (int want = 1; want <= kTileSpans && (want == 1 || steps >= 4 * want); ++want) {
      const int span = static_cast<int>(ceil_div(steps, want));
      const int splits = static_cast<int>(ceil_div(steps, span));
      const int64_t blocks = tiles * splits;
      if (splits > 1 && blocks > kTileBlocks) break;
      const double tile = blocks <= 256 ? (mb == 1 ? 33.0 : 45.0)
                                        : (mb == 1 ? 23.0 : 43.0) * static_cast<double>(ceil_div(blocks, 256));
      double us = 2.5 + tile * span / 32.0;
      if (splits > 1) us += 3.0 + 0.9e-6 * static_cast<double>(splits) * static_cast<double>(M * N);
      if (us < best_us) {
        best_us = us;
        best = {kTile, mb, 4, splits, span};
      }
    }
  }
  return best;
}

Plan plan_of(int64_t M, int64_t N, int64_t K) {
  const int steps = static_cast<int>(K / 128);
  // Past four tokens each workgroup of the first reads all of x (16 x 2,816 x 8,192: 12.3 us against 10.0
  // in spans of k; at 4,096 7.6).
  // Columns of a workgroup, us at k of 2,816, 16 | 32 | 64: one token x 4,096 4.0 | 5.0 | 6.9, x 8,192 5.7 | 5.5 | 7.4,
  // x 30,000 16.3 | 12.7 | 14.3; 16 tokens x 4,096 5.9 | 6.9 | 9.1, x 8,192 9.4 | 7.5 | 9.4, x 30,000 29.5 | 23.2 | 19.1.
  if ((M <= 4 || (M <= 16 && K <= 4096)) && N < kManyColumns)
    return {kFew, N <= 4096 ? 1 : M <= 4 || N <= 8192 ? 2 : 4, 16, 1, steps};
  if (M <= 4) return {kStream, kStreamTiles, kStreamWaves, 1, steps};
  if (M <= 64) {
    const bool many = N >= kManyColumns;
    const int nt = M > 16 && M <= 32 && many ? 2 : 1;
    const int waves = !many ? 4 : M <= 32 ? 16 : 8;
    const int64_t blocks = ceil_div(N, 16 * nt * waves);
    // Spans of an even number of steps, six where there are that many, for 512 workgroups.  us in spans for
    // 256 | 352 | 512: 5 tokens x 8,192 x 8,192 17.5 | 16.1 | 14.6, 64 26.5 | 24.3 | 22.5; 61 x 2,816 x 4,096 in
    // spans of six steps 12.2, of four 12.9.  (Workgroups of 16 waves have other sums: 5 x 33,000 x 4,096 24.9 us for
    // 352, 27.7 for 512; of two tiles a wave, 20 tokens, 41.4 for 256 and 38.0 for 512.)
    const int64_t full = many && M <= 16 ? 352 : 512;
    const int64_t want = std::min<int64_t>(ceil_div(full, blocks), std::min(16, (steps + 4) / 5));
    const int span = static_cast<int>(ceil_div(ceil_div(steps, want), 2) * 2);
    return {kBatch, nt, waves, static_cast<int>(ceil_div(steps, span)), span};
  }
  return tile_plan(M, N, steps);
}
int64_t part_stride(int64_t M, int64_t N) { return (M * N + 3) / 4 * 4; }

template <int kFmt, int kGroup, int NT, int ST, int R>
hipError_t launch_few(const W4Args& a, hipStream_t stream) {
  const int cols = NT > 1 ? 16 * NT : static_cast<int>(std::min<int64_t>(16, ceil_div(a.N, 256)));
  const int64_t steps = a.K / 128;
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, cols)));
  const dim3 block(static_cast<unsigned>(64 * std::min<int64_t>(16, ceil_div(steps, ST))));
  hipLaunchKernelGGL((w4_few_kernel<kFmt, kGroup, NT, ST, R>), grid, block, 0, stream, a, cols);
  return hipGetLastError();
}

template <int kFmt, int kGroup>
hipError_t launch_stream(const W4Args& a, hipStream_t stream) {
  // The largest even number of steps of x that fits, all of them if they do.
  const int64_t room = (kStreamLds / a.M - 16) / 256 / 2 * 2;
  const int chunk = static_cast<int>(std::min<int64_t>(room, a.K / 128));
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, 16 * kStreamTiles * kStreamWaves)));
  hipLaunchKernelGGL((w4_stream_kernel<kFmt, kGroup>), grid, dim3(64 * kStreamWaves),
                     static_cast<size_t>(a.M * (256 * chunk + 16)), stream, a, chunk);
  return hipGetLastError();
}

template <int kFmt>
hipError_t launch_reduce(const W4Args& a, const Plan& p, hipStream_t stream) {
  const int64_t count = a.M * a.N;
  hipLaunchKernelGGL(w4_reduce_kernel, dim3(static_cast<unsigned>(ceil_div(count, 1024))),
                     dim3(256), 0, stream, a.workspace, a.out, count, part_stride(a.M, a.N), p.splits,
                     kUnit<kFmt>);
  return hipGetLastError();
}

template <int kFmt, int kGroup, int TM, int NT, int W>
hipError_t launch_batch(const W4Args& a, const Plan& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, 16 * NT * W)),
                  static_cast<unsigned>(p.splits));
  const int64_t stride = part_stride(a.M, a.N);
  if (p.splits == 1) {
    hipLaunchKernelGGL((w4_batch_kernel<kFmt, kGroup, TM, NT, W, false>), grid, dim3(64 * W), 0,
                       stream, a, p.span, stride);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((w4_batch_kernel<kFmt, kGroup, TM, NT, W, true>), grid, dim3(64 * W), 0, stream,
                     a, p.span, stride);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  return launch_reduce<kFmt>(a, p, stream);
}

template <int kFmt, int kGroup, int MB>
hipError_t launch_tile(const W4Args& a, const Plan& p, hipStream_t stream) {
  const int mt = static_cast<int>(ceil_div(a.M, 64 * MB)), nt = static_cast<int>(ceil_div(a.N, kTileN));
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(mt) * nt + 7) / 8 * 8),
                  static_cast<unsigned>(p.splits));
  const int64_t stride = part_stride(a.M, a.N);
  if (p.splits == 1) {
    hipLaunchKernelGGL((w4_tile_kernel<kFmt, kGroup, MB, false>), grid, dim3(kTileThreads), 0, stream, a,
                       p.span, stride, mt, nt);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((w4_tile_kernel<kFmt, kGroup, MB, true>), grid, dim3(kTileThreads), 0, stream, a,
                     p.span, stride, mt, nt);
  const hipError_t err = hipGetLastError();
  return err != hipSuccess ? err : launch_reduce<kFmt>(a, p, stream);
}

template <int kFmt, int kGroup>
hipError_t launch_group(const W4Args& a, hipStream_t stream) {
  const Plan p = plan_of(a.M, a.N, a.K);
  if (p.kind == kFew) {
    if (p.nt == 4) return launch_few<kFmt, kGroup, 4, 2, 4>(a, stream);
    if (p.nt == 2)
      return a.M <= 4 ? launch_few<kFmt, kGroup, 2, 2, 1>(a, stream) : launch_few<kFmt, kGroup, 2, 2, 4>(a, stream);
    if (a.K > 4096) return launch_few<kFmt, kGroup, 1, 4, 1>(a, stream);  // four tokens at most
    return a.M <= 4 ? launch_few<kFmt, kGroup, 1, 2, 1>(a, stream) : launch_few<kFmt, kGroup, 1, 2, 4>(a, stream);
  }
  if (p.kind == kStream) return launch_stream<kFmt, kGroup>(a, stream);
  if (p.kind == kBatch) {
    if (p.waves == 16 && p.nt == 1) return launch_batch<kFmt, kGroup, 1, 1, 16>(a, p, stream);
    if (p.waves == 16) return launch_batch<kFmt, kGroup, 2, 2, 16>(a, p, stream);
    if (p.waves == 8) return launch_batch<kFmt, kGroup, 4, 1, 8>(a, p, stream);
    if (a.M <= 16) return launch_batch<kFmt, kGroup, 1, 1, 4>(a, p, stream);
    if (a.M <= 32) return launch_batch<kFmt, kGroup, 2, 1, 4>(a, p, stream);
    return launch_batch<kFmt, kGroup, 4, 1, 4>(a, p, stream);
  }
  return p.nt == 1 ? launch_tile<kFmt, kGroup, 1>(a, p, stream) : launch_tile<kFmt, kGroup, 2>(a, p, stream);
}

template <int kFmt>
hipError_t launch_format(const W4Args& a, hipStream_t stream) {
  if (a.group == 32) return launch_group<kFmt, 32>(a, stream);
  if (a.group == 64) return launch_group<kFmt, 64>(a, stream);
  return launch_group<kFmt, 128>(a, stream);
}

}  // namespace

// For every number of tokens up to M: exact for each kind of plan up to 64, beyond the bound that
// kTileBlocks sets (of tiles of 128 x 128).
int64_t w4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  int64_t floats = 0;
  for (const int64_t up_to : {16, 32, 64}) {
    const int64_t m = std::min(M, up_to);
    const Plan p = plan_of(m, N, K);
    if (p.splits > 1) floats = std::max(floats, p.splits * part_stride(m, N));
  }
  if (M > 64 && K / 128 >= 8 && 2 * ceil_div(N, kTileN) <= kTileBlocks)
    floats = std::max(floats, std::min(kTileSpans * part_stride(M, N), kTileBlocks * 128 * kTileN));
  return floats * 4;
}

void w4_gemm_plan(int64_t M, int64_t N, int64_t K, int64_t* plan) {
  const Plan p = plan_of(M, N, K);
  plan[0] = p.kind, plan[1] = p.nt, plan[2] = p.waves, plan[3] = p.splits, plan[4] = p.span;
}

hipError_t launch_w4_gemm(const W4Args& a, hipStream_t stream) {
  return a.format == kW4Int4 ? launch_format<kW4Int4>(a, stream)
                             : launch_format<kW4E2m1>(a, stream);
}

}  // namespace ifr
