// RoPE and the quantising write into an 8-bit paged cache (gfx950): codes of OCP e4m3 or
// int8, a power-of-two scale for each block of rows and kv head.
//
// A scale is the smallest power of two with amax <= Q * scale (Q = 448 or 127).  Powers of
// two cost e4m3 nothing (its relative step does not depend on the scale) and int8 half a
// bit on average, and they make a block that grows cheap and safe: old codes are scaled by
// 2^-n, exactly in e4m3 above its subnormals, and a row is rounded again once for each
// doubling of the block's largest value, errors that halve each time, not once for each
// new largest value.  The values also are bf16 numbers, so that attention reads them
// without a further rounding.
//
// Grid: first the k and v of (write block, kv head), a workgroup each; then q, whole
// rows a workgroup.  A row of head_dim values is head_dim / 8 lanes.
//
// Bound by HBM for prompts (k, v, q once, codes once): 2 x 2,048 tokens of 16 q and 8 kv heads of 256
// take 25 us, 4.9 TB/s; by a launch's latency for single tokens: 64 of them 8 us.
#include <float.h>

#include "window_dev.hpp"

namespace ifr {
namespace {

using namespace window;

constexpr int kThreads = 256;

struct Chunk {
  float v[8];
};

__device__ __forceinline__ Chunk load_chunk(const uint16_t* p) {
  const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p);
  Chunk c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c.v[2 * i] = bf16_lo(w[i]);
    c.v[2 * i + 1] = bf16_hi(w[i]);
  }
  return c;
}
__device__ __forceinline__ void store_chunk(uint16_t* p, const Chunk& c) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16(c.v[2 * i], c.v[2 * i + 1]);
  *reinterpret_cast<u32x4_t*>(p) = w;
}
__device__ __forceinline__ Chunk load_table(const float* p) {
  Chunk c;
#pragma unroll
  for (int i = 0; i < 8; ++i) c.v[i] = p[i];
  return c;
}

// Dims d .. d + 7 of a rotated row: dims [0, half) pair with [pair, pair + half).
__device__ __forceinline__ Chunk rotated_chunk(const uint16_t* row, int d, int half, int pair, const float* cos_row,
                                               const float* sin_row) {
  Chunk x = load_chunk(row + d);
  const bool lo = d < half, hi = d >= pair && d < pair + half;
  if (lo || hi) {
    const int f = lo ? d : d - pair;
    const Chunk y = load_chunk(row + (lo ? d + pair : d - pair));
    const Chunk cs = load_table(cos_row + f), sn = load_table(sin_row + f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x.v[i] * cs.v[i], b = y.v[i] * sn.v[i];
      x.v[i] = lo ? a - b : a + b;
    }
  }
  return x;
}

// The exponent field of the smallest power of two s with amax <= Q s; 0 for amax 0.
template <int kFormat>
__device__ __forceinline__ uint32_t scale_bits(float amax) {
  constexpr uint32_t q = kFormat == kE4m3 ? 0x43E00000u : 0x42FE0000u;  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const uint32_t u = __float_as_uint(amax);
  if (u == 0) return 0;
  const int e = static_cast<int>(u >> 23) - static_cast<int>(q >> 23) + 127 + ((u & 0x7FFFFFu) > (q & 0x7FFFFFu) ? 1 : 0);
  return static_cast<uint32_t>(max(e, 1)) << 23;
}

// The largest code times `scale`, inv = 1 / scale, that f32 (and so bf16) holds: 240 under 2^120
// in e4m3, 63 under 2^122 in int8, where the nearest code of the largest bf16 values stands for 2^128.
template <int kFormat>
__device__ __forceinline__ float top_code(float inv) {
  if constexpr (kFormat == kE4m3) return fminf(448.0f, 0x1.Ep127f * inv);  // 240 * 2^120: 448 * 2^119 is less
  else return fminf(127.0f, __builtin_floorf(FLT_MAX * inv));
}

// x (already divided by the scale) to a code: nearest even, at most top; NaN stays (e4m3) or
// becomes 0 (int8).
template <int kFormat>
__device__ __forceinline__ uint32_t codes4(const float* x, float top) {
  if constexpr (kFormat == kE4m3) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i], -top, top);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    uint32_t r = static_cast<uint32_t>(w);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (x[i] != x[i]) r |= 0x7Fu << (8 * i);
    return r;
  } else {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = x[i] == x[i] ? __builtin_rintf(__builtin_amdgcn_fmed3f(x[i], -top, top)) : 0.0f;
      r |= (static_cast<uint32_t>(static_cast<int32_t>(y)) & 0xFFu) << (8 * i);
    }
    return r;
  }
}
template <int kFormat>
__device__ __forceinline__ void values4(uint32_t w, float* x) {
  const u32x2_t b = codes4_bf16<kFormat>(w);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[2 * i] = bf16_lo(b[i]);
    x[2 * i + 1] = bf16_hi(b[i]);
  }
}

template <int kD, int kFormat>
__global__ __launch_bounds__(kThreads) void kv8_write_kernel(const Kv8WriteArgs a) {
  constexpr int kLanes = kD / 8;              // threads of a row
  constexpr int kRows = kThreads / kLanes;    // rows of a pass
  constexpr int kHeld = 8;                    // passes whose values stay in registers
  const int64_t kv_groups = a.num_writes * a.num_kv * 2;

  if (static_cast<int64_t>(blockIdx.x) >= kv_groups) {
    // ---- q: a thread takes both chunks of a pair, or one that is not rotated ----
    const int half8 = a.half / 8, units = kLanes - half8, rows = kThreads / units;
    const int sub = threadIdx.x / units, i = threadIdx.x - sub * units;
    const int row = static_cast<int>(blockIdx.x - kv_groups) * rows + sub;
    if (sub >= rows || row >= a.seq_len * a.num_q) return;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(row) * kD;
    uint16_t* dst = static_cast<uint16_t*>(a.q_out) + static_cast<int64_t>(row) * kD;
    if (i < half8) {
      const int tok = row / a.num_q;
      const int32_t* rp = a.image + a.image[kHdrOffRuns] + 4 * a.image[a.image[kHdrOffTokRun] + tok];
      const int64_t pos = rp[1] + (tok - rp[0]);
      const Chunk cs = load_table(a.cos_table + pos * a.half + 8 * i), sn = load_table(a.sin_table + pos * a.half + 8 * i);
      Chunk x = load_chunk(src + 8 * i), y = load_chunk(src + a.pair_stride + 8 * i), lo, hi;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = x.v[e] * cs.v[e], r = y.v[e] * sn.v[e], s = y.v[e] * cs.v[e], t = x.v[e] * sn.v[e];
        lo.v[e] = p - r;
        hi.v[e] = s + t;
      }
      store_chunk(dst + 8 * i, lo);
      store_chunk(dst + a.pair_stride + 8 * i, hi);
    } else if (src != dst) {  // dims [half, pair) and [pair + half, D)
      const int d = 8 * i < a.pair_stride ? 8 * i : 8 * i + a.half;
      *reinterpret_cast<u32x4_t*>(dst + d) = *reinterpret_cast<const u32x4_t*>(src + d);
    }
    return;
  }

  __shared__ float sm_max[kThreads / 64];
  const int is_v = blockIdx.x & 1;
  const int64_t pair_id = blockIdx.x >> 1;
  const int h = static_cast<int>(pair_id % a.num_kv);
  const int32_t* wb = a.image + a.off_writes + (pair_id / a.num_kv) * kWriteBlockWords;
  const int tok = sload(wb + kWbToken), count = sload(wb + kWbCount), pos = sload(wb + kWbPos);
  const int64_t row0 = sload(wb + kWbRow);
  const int block_rows = 1 << a.block_shift;
  const int before = static_cast<int>(row0 & (block_rows - 1));  // rows of the block that are older
  const int tr = threadIdx.x / kLanes, d = 8 * (threadIdx.x % kLanes);
  const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.v : a.k) + (static_cast<int64_t>(tok) * a.num_kv + h) * kD;
  const int64_t src_stride = static_cast<int64_t>(a.num_kv) * kD;
  uint8_t* cache = static_cast<uint8_t*>(is_v ? a.v_cache : a.k_cache) + static_cast<int64_t>(h) * kD + d;
  float* scale = (is_v ? a.v_scale : a.k_scale) + (row0 >> a.block_shift) * a.num_kv + h;

  auto values = [&](int r) {
    const uint16_t* row = src + r * src_stride;
    if (is_v) return load_chunk(row + d);
    const int64_t t = (static_cast<int64_t>(pos) + r) * a.half;
    return rotated_chunk(row, d, a.half, a.pair_stride, a.cos_table + t, a.sin_table + t);
  };
  float amax = 0.0f;
  auto take_max = [&](const Chunk& c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __builtin_fabsf(c.v[i]);
      amax = x < INFINITY ? fmaxf(amax, x) : amax;
    }
  };
  // Values of the first passes stay in registers; a block of more rows than that reads the
  // others again, from L2.
  Chunk held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int r = i * kRows + tr;
    if (r < count) {
      held[i] = values(r);
      take_max(held[i]);
    }
  }
  for (int r = kHeld * kRows + tr; r < count; r += kRows) take_max(values(r));
  amax = wave_max_ref(amax);
  if ((threadIdx.x & 63) == 0) sm_max[threadIdx.x >> 6] = amax;
  const float old = before > 0 ? *scale : 0.0f;
  __syncthreads();
  amax = fmaxf(fmaxf(sm_max[0], sm_max[1]), fmaxf(sm_max[2], sm_max[3]));
  const float now = fmaxf(__uint_as_float(scale_bits<kFormat>(amax)), old);
  if (threadIdx.x == 0) *scale = now;  // every thread has read it: the barrier is behind

  // A power of two of at most 2^126: exact.  Under a scale of 0 every finite value is 0.
  const float inv = now > 0.0f ? 1.0f / now : 1.0f;
  const float top = top_code<kFormat>(inv);
  auto store = [&](int64_t row, const float* x) {
    u32x2_t w;
    w[0] = codes4<kFormat>(x, top);
    w[1] = codes4<kFormat>(x + 4, top);
    *reinterpret_cast<u32x2_t*>(cache + row * a.kv_stride) = w;
  };
  auto write = [&](int r, const Chunk& c) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c.v[i] * inv;
    store(row0 + r, x);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int r = i * kRows + tr;
    if (r < count) write(r, held[i]);
  }
  for (int r = kHeld * kRows + tr; r < count; r += kRows) write(r, values(r));
  // Older rows under a scale that grew.  From 0 it makes their codes 0: they were worth that (an
  // infinity among rows of zeros has the largest code).
  if (before > 0 && now > old) {
    const float ratio = old * inv;
    for (int r = tr; r < before; r += kRows) {
      const int64_t row = row0 - before + r;
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(cache + row * a.kv_stride);
      float x[8];
      values4<kFormat>(w[0], x);
      values4<kFormat>(w[1], x + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= ratio;
      store(row, x);
    }
  }
}

template <int kD>
hipError_t write_of(const Kv8WriteArgs& a, int format, hipStream_t stream) {
  const int64_t rows = kThreads / (kD / 8 - a.half / 8);  // of q, a workgroup
  const int64_t groups = a.num_writes * a.num_kv * 2 + (static_cast<int64_t>(a.seq_len) * a.num_q + rows - 1) / rows;
  if (groups > kMaxGroups) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<uint32_t>(groups));
  if (format == kE4m3) kv8_write_kernel<kD, kE4m3><<<grid, kThreads, 0, stream>>>(a);
  else kv8_write_kernel<kD, kInt8><<<grid, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_write(const Kv8WriteArgs& a, int format, int head_dim, hipStream_t stream) {
  if (head_dim == 128) return write_of<128>(a, format, stream);
  if (head_dim == 256) return write_of<256>(a, format, stream);
  return write_of<512>(a, format, stream);
}

}  // namespace ifr
