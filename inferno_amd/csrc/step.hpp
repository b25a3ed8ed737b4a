// Launches of the operators behind the attention: products with 4-bit weights
// (w4_gemm.hip), norms around a block (norm_residual.hip) and sampling (sample.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ifr {

// Workgroups of a launch, whose grid has less than 2^32 threads.
constexpr int64_t max_blocks(int threads) { return ((int64_t{1} << 32) - 1) / threads; }

constexpr int kW4Int4 = 1;  // IFR_W4_INT4
constexpr int kW4E2m1 = 2;  // IFR_W4_E2M1

struct W4Args {
  const uint16_t* x;       // [M][K] bf16
  const uint8_t* codes;    // [N][K / 2]
  const uint16_t* scales;  // [N][K / group] bf16
  uint16_t* out;           // [M][N] bf16
  float* workspace;
  int64_t M, N, K;
  int group, format;
};
int64_t w4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K);
// {kind, tiles, waves, spans of k, steps of a span}, as plan_of in w4_gemm.hip has them.
void w4_gemm_plan(int64_t M, int64_t N, int64_t K, int64_t* plan);
hipError_t launch_w4_gemm(const W4Args& a, hipStream_t stream);

struct NormResidualArgs {
  const uint16_t* y;
  const void* residual;
  void* residual_out;
  uint16_t* x_out;              // null: no second norm
  const uint16_t* post_weight;  // null: weights of one
  const uint16_t* gate;         // null: none
  const uint16_t* pre_weight;   // null: weights of one
  int64_t rows, hidden, gate_stride;
  bool f32, post_norm;
  float eps, residual_scale, block_scale;
};
hipError_t launch_norm_residual(const NormResidualArgs& a, hipStream_t stream);

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  bool f32;
  const float* temperature;  // each null: off
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int32_t* tokens;
  int64_t rows, vocab;
  void* workspace;
};
int64_t sample_workspace_bytes(int64_t rows, int64_t vocab);
// Workgroups of the first launch.
int64_t sample_scan_blocks(int64_t rows, int64_t vocab, bool f32);
constexpr int kScanThreads = 256;
hipError_t launch_sample(const SampleArgs& a, hipStream_t stream);

}  // namespace ifr
