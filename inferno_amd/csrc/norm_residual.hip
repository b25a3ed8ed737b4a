// The norm behind a block, its gate and residual scale, and the norm ahead of the next
// block, in one pass over a token's row:
//   t  = y / sqrt(mean(y^2) + eps) * post_weight          (or y)
//   r' = residual_scale * residual + block_scale * (gate * t)
//   x  = r' / sqrt(mean(r'^2) + eps) * pre_weight
// in f32; r' and x are each rounded once, x from the unrounded r'.
#include <algorithm>

#include "common.hpp"
#include "step.hpp"

namespace ifr {
namespace {

__device__ __forceinline__ float wave_sum(float v) { return pair_sum32(pair_sum16(tree16_sum(v))); }

__device__ __forceinline__ void unpack8(uint4 p, float* v) {
  v[0] = bf16_lo(p.x), v[1] = bf16_hi(p.x), v[2] = bf16_lo(p.y), v[3] = bf16_hi(p.y);
  v[4] = bf16_lo(p.z), v[5] = bf16_hi(p.z), v[6] = bf16_lo(p.w), v[7] = bf16_hi(p.w);
}
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  bf16x2_t p;
  p[0] = static_cast<__bf16>(lo);
  p[1] = static_cast<__bf16>(hi);
  return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
}

// W waves a row, C chunks of 8 elements a lane: the row stays in registers between
// its reads and its writes, and each of the two sums is one reduction, so every byte moves once.
// 16,384 tokens x 2,816, bf16, a gate of the layer: 71 us, 5.2 TB/s, the rate of a copy.  A single token:
// 2.8 us, a read, two reductions over LDS and a write one after the other.
template <int W, int C, bool kF32>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_residual_kernel(NormResidualArgs a) {
  constexpr int kRowThreads = 64 * W;
  __shared__ float part[2][W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  if (row >= a.rows) return;  // W > 1: block-uniform
  const int t = W == 1 ? lane : threadIdx.x;
  const int hidden = static_cast<int>(a.hidden), chunks = hidden / 8;
  const float n = static_cast<float>(hidden);

  auto row_sum = [&](float v, int which) {
    v = wave_sum(v);
    if constexpr (W > 1) {
      if (lane == 0) part[which][wave] = v;
      __syncthreads();
      v = part[which][0];
#pragma unroll
      for (int w = 1; w < W; ++w) v = v + part[which][w];
    }
    return v;
  };

  // With eight chunks a lane its 128 registers hold y and r alone, and the gate and the weights are loaded where they
  // are used (2,048 tokens x 65,536, bf16: 249 us; all of them ahead, 372 B a lane in scratch memory: 592).
  constexpr bool kAhead = C <= 4;
  uint4 y[C], g[kAhead ? C : 1], pw[kAhead ? C : 1], qw[kAhead ? C : 1];
  float r[C][8];
  auto gate_at = [&](int at) { return reinterpret_cast<const uint4*>(a.gate + row * a.gate_stride)[at]; };
  auto post_at = [&](int at) { return reinterpret_cast<const uint4*>(a.post_weight)[at]; };
  auto pre_at = [&](int at) { return reinterpret_cast<const uint4*>(a.pre_weight)[at]; };
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = c * kRowThreads + t;
    if (at < chunks) {
      y[c] = reinterpret_cast<const uint4*>(a.y + row * hidden)[at];
      if constexpr (kF32) {
        const float4* p = reinterpret_cast<const float4*>(
                              static_cast<const float*>(a.residual) + row * hidden) + 2 * at;
        const float4 lo = p[0], hi = p[1];
        r[c][0] = lo.x, r[c][1] = lo.y, r[c][2] = lo.z, r[c][3] = lo.w;
        r[c][4] = hi.x, r[c][5] = hi.y, r[c][6] = hi.z, r[c][7] = hi.w;
      } else {
        unpack8(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.residual) +
                                               row * hidden)[at], r[c]);
      }
      if constexpr (kAhead) {
        if (a.gate) g[c] = gate_at(at);
        if (a.post_weight) pw[c] = post_at(at);
        if (a.pre_weight) qw[c] = pre_at(at);
      }
    }
  }
  float inv = 1.0f;
  if (a.post_norm) {
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (c * kRowThreads + t >= chunks) continue;
      float v[8];
      unpack8(y[c], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
    }
    inv = 1.0f / sqrtf(row_sum(ss, 0) / n + a.eps);
  }
  // (No instruction: keeps the addresses of the first loop from being held until here, in scratch memory.)
  int again = t;
  if constexpr (!kAhead) asm("" : "+v"(again));
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = c * kRowThreads + again;
    if (at >= chunks) continue;
    float v[8], w[8];
    unpack8(y[c], v);
    if (a.post_weight) {
      unpack8(kAhead ? pw[kAhead ? c : 0] : post_at(at), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * inv;
    }
    if (a.gate) {
      unpack8(kAhead ? g[kAhead ? c : 0] : gate_at(at), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * w[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[c][i] = __builtin_fmaf(a.block_scale, v[i], a.residual_scale * r[c][i]);
      ss = __builtin_fmaf(r[c][i], r[c][i], ss);
    }
    if constexpr (kF32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.residual_out) + row * hidden) +
                  2 * at;
      p[0] = make_float4(r[c][0], r[c][1], r[c][2], r[c][3]);
      p[1] = make_float4(r[c][4], r[c][5], r[c][6], r[c][7]);
    } else {
      reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.residual_out) + row * hidden)[at] =
          pack8(r[c]);
    }
  }
  if (!a.x_out) return;
  inv = 1.0f / sqrtf(row_sum(ss, 1) / n + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = c * kRowThreads + again;
    if (at >= chunks) continue;
    float v[8], w[8];
    if (a.pre_weight) unpack8(kAhead ? qw[kAhead ? c : 0] : pre_at(at), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a.pre_weight ? r[c][i] * inv * w[i] : r[c][i] * inv;
    reinterpret_cast<uint4*>(a.x_out + row * hidden)[at] = pack8(v);
  }
}

// One launch, but for millions of long rows as many as their threads need.
template <int W, int C>
hipError_t launch_wc(const NormResidualArgs& all, hipStream_t stream) {
  constexpr int kThreads = W == 1 ? 256 : 64 * W, kRows = W == 1 ? 4 : 1;  // of a workgroup
  constexpr int64_t kMaxRows = max_blocks(kThreads) * kRows;
  for (int64_t row0 = 0; row0 < all.rows; row0 += kMaxRows) {
    NormResidualArgs a = all;
    const int64_t at = row0 * a.hidden, res = at * (a.f32 ? 4 : 2);
    a.rows = std::min(all.rows - row0, kMaxRows);
    a.y += at;
    a.residual = static_cast<const char*>(a.residual) + res;
    a.residual_out = static_cast<char*>(a.residual_out) + res;
    if (a.x_out) a.x_out += at;
    if (a.gate) a.gate += row0 * a.gate_stride;
    const dim3 grid(static_cast<unsigned>((a.rows + kRows - 1) / kRows));
    if (a.f32)
      hipLaunchKernelGGL((norm_residual_kernel<W, C, true>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((norm_residual_kernel<W, C, false>), grid, dim3(kThreads), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace

// A wave a row to 1,024 elements, four waves to 8,192, 16 beyond, as few chunks a lane as that takes.  Both
// sides in us, bf16, both weights, replayed from a graph, one token | 16,384:
//   512   1 wave 2.3 | 12.0, 4 waves 2.5 | 17.2     1,024   1 wave 2.7 | 21.4, 4 waves 2.5 | 23.0
//   2,048 1 wave 3.8 | 48.1, 4 waves 2.6 | 42.0     4,096   4 waves 4.1 | 95, 16 waves 3.0 | 112
//   8,192 4 waves 4.4 | 189, 16 waves 3.7 | 194     16,384  16 waves 4.9 | 397, 4 waves 6.5 | 399
// Past 16,384 the chunks of 16 waves alone grow: one token | 2,048 of 32,768 8.1 | 118, of 65,536 12.4 | 249.
hipError_t launch_norm_residual(const NormResidualArgs& a, hipStream_t stream) {
  const int64_t chunks = a.hidden / 8;
  if (chunks <= 64) return launch_wc<1, 1>(a, stream);
  if (chunks <= 64 * 2) return launch_wc<1, 2>(a, stream);
  if (chunks <= 256) return launch_wc<4, 1>(a, stream);
  if (chunks <= 256 * 2) return launch_wc<4, 2>(a, stream);
  if (chunks <= 256 * 4) return launch_wc<4, 4>(a, stream);
  if (chunks <= 1024 * 2) return launch_wc<16, 2>(a, stream);
  if (chunks <= 1024 * 4) return launch_wc<16, 4>(a, stream);
  return launch_wc<16, 8>(a, stream);
}

}  // namespace ifr
