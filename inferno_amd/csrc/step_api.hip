// Entry points of the operators behind the attention (declared in include/inferno_hip.h):
// products with 4-bit weights, norms around a block, sampling.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/inferno_hip.h"
#include "step.hpp"

namespace ifr {
int32_t abi_fail(int32_t code, const char* msg);  // api.hip
int32_t abi_ok();
}  // namespace ifr

namespace {

static_assert(ifr::kW4Int4 == IFR_W4_INT4 && ifr::kW4E2m1 == IFR_W4_E2M1, "formats");

int32_t fail(int32_t code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return ifr::abi_fail(code, buf);
}

int32_t launched(hipError_t err, const char* what) {
  if (err != hipSuccess) return fail(IFR_EHIP, "%s: %s", what, hipGetErrorString(err));
  return ifr::abi_ok();
}

// A buffer of a call; no two of which one is written may share memory.
struct Span {
  const void* at;
  int64_t bytes;
};
bool overlap(Span a, Span b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  if (!a.at || !b.at || a.bytes <= 0 || b.bytes <= 0) return false;
  return x < y ? y - x < static_cast<uint64_t>(a.bytes) : x - y < static_cast<uint64_t>(b.bytes);
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
hipStream_t as_stream(uint64_t s) { return reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(s)); }

constexpr int64_t kMaxW4Rows = int64_t{1} << 24, kMaxW4Cols = int64_t{1} << 20,
                  kMaxW4Tokens = int64_t{1} << 19;
constexpr int64_t kMaxVocab = int64_t{1} << 20, kMaxSampleRows = int64_t{1} << 20;

bool w4_shape(int64_t rows, int64_t cols, int64_t seq_len) {
  return rows > 0 && rows <= kMaxW4Rows && cols > 0 && cols % 128 == 0 && cols <= kMaxW4Cols &&
         seq_len >= 0 && seq_len <= kMaxW4Tokens;
}
bool sample_shape(int64_t num_rows, int64_t vocab) {
  return num_rows >= 0 && num_rows <= kMaxSampleRows && vocab >= 1 && vocab <= kMaxVocab;
}

}  // namespace

extern "C" {

int64_t ifr_w4_gemm_workspace_bytes(int64_t rows, int64_t cols, int64_t seq_len) {
  if (!w4_shape(rows, cols, seq_len)) return -1;
  return seq_len == 0 ? 0 : ifr::w4_gemm_workspace_bytes(seq_len, rows, cols);
}

// Not part of the C API: the launch that a shape takes, for the tests to hold on to.
int32_t ifr_internal_w4_plan(int64_t rows, int64_t cols, int64_t seq_len, int64_t* plan) {
  if (!w4_shape(rows, cols, seq_len) || seq_len == 0) return fail(IFR_EINVAL, "bad w4_gemm_cols shape");
  ifr::w4_gemm_plan(seq_len, rows, cols, plan);
  return ifr::abi_ok();
}

int32_t ifr_dispatch_w4_gemm_cols(const void* x, const void* codes, const void* scales,
                                  void* output, int64_t rows, int64_t cols, int64_t seq_len,
                                  int64_t group, int64_t w_format, void* workspace,
                                  int64_t workspace_bytes, uint64_t stream) {
  if (!w4_shape(rows, cols, seq_len))
    return fail(IFR_EINVAL, "rows must be in [1, 2^24], cols a multiple of 128 in [128, 2^20], "
                            "seq_len in [0, 2^19]");
  if (group != 32 && group != 64 && group != 128)
    return fail(IFR_EINVAL, "group must be 32, 64 or 128");
  if (w_format != IFR_W4_INT4 && w_format != IFR_W4_E2M1)
    return fail(IFR_EINVAL, "w_format must be IFR_W4_INT4 or IFR_W4_E2M1");
  if (seq_len == 0) return ifr::abi_ok();
  if (!x || !codes || !scales || !output) return fail(IFR_EINVAL, "null pointer");
  if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(output, 16))
    return fail(IFR_EINVAL, "x, codes, scales and output must be 16-byte aligned");
  const int64_t need = ifr::w4_gemm_workspace_bytes(seq_len, rows, cols);
  if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
    return fail(IFR_ESPACE, "workspace needs %lld bytes, 16-byte aligned", (long long)need);
  const Span out{output, 2 * seq_len * rows}, space{need > 0 ? workspace : nullptr, need};
  for (const Span in : {Span{x, 2 * seq_len * cols}, Span{codes, rows * (cols / 2)},
                        Span{scales, 2 * rows * (cols / group)}})
    if (overlap(out, in) || overlap(space, in))
      return fail(IFR_EINVAL, "output or workspace overlaps an input");
  if (overlap(out, space)) return fail(IFR_EINVAL, "output overlaps the workspace");
  const ifr::W4Args a{static_cast<const uint16_t*>(x), static_cast<const uint8_t*>(codes),
                      static_cast<const uint16_t*>(scales), static_cast<uint16_t*>(output),
                      static_cast<float*>(workspace), seq_len, rows, cols,
                      static_cast<int>(group), static_cast<int>(w_format)};
  return launched(ifr::launch_w4_gemm(a, as_stream(stream)), "w4_gemm_cols");
}

int32_t ifr_norm_residual(const void* y, const void* residual, void* residual_out, void* x_out,
                          const void* post_weight, const void* gate, const void* pre_weight,
                          int64_t hidden, int64_t seq_len, int64_t residual_type,
                          int64_t post_norm, int64_t gate_stride, float residual_scale,
                          float block_scale, float eps, uint64_t stream) {
  if (hidden <= 0 || hidden % 8 != 0 || hidden > 65536)
    return fail(IFR_EINVAL, "hidden must be a multiple of 8 in [8, 65536]");
  if (seq_len < 0 || seq_len > (int64_t{1} << 24))
    return fail(IFR_EINVAL, "seq_len must be in [0, 2^24]");
  if (residual_type != IFR_RESIDUAL_BF16 && residual_type != IFR_RESIDUAL_F32)
    return fail(IFR_EINVAL, "residual_type must be IFR_RESIDUAL_BF16 or IFR_RESIDUAL_F32");
  if (!(eps > 0.0f) || isinf(eps)) return fail(IFR_EINVAL, "eps must be above 0 and finite");
  if (gate && gate_stride != 0 && (gate_stride < hidden || gate_stride % 8 != 0))
    return fail(IFR_EINVAL, "gate_stride must be 0 or a multiple of 8 of at least hidden");
  if (gate && gate_stride > (int64_t{1} << 32)) return fail(IFR_EINVAL, "gate_stride too large");
  if (post_norm != 0 && post_norm != 1) return fail(IFR_EINVAL, "post_norm must be 0 or 1");
  if (post_weight && !post_norm) return fail(IFR_EINVAL, "post_weight without post_norm");
  if (pre_weight && !x_out) return fail(IFR_EINVAL, "pre_weight without x_out");
  if (seq_len == 0) return ifr::abi_ok();
  if (!y || !residual || !residual_out) return fail(IFR_EINVAL, "null pointer");
  for (const void* p : {y, residual, static_cast<const void*>(residual_out),
                        static_cast<const void*>(x_out), post_weight, gate, pre_weight})
    if (!aligned(p, 16)) return fail(IFR_EINVAL, "every pointer must be 16-byte aligned");
  const int64_t n = seq_len * hidden, res = residual_type == IFR_RESIDUAL_F32 ? 4 * n : 2 * n;
  const Span r_out{residual_out, res}, xs{x_out, 2 * n}, ys{y, 2 * n}, rs{residual, res};
  // In place, from its start, each output may be the input that it follows.
  if (overlap(r_out, xs) || overlap(r_out, ys) || overlap(xs, rs) ||
      (residual_out != residual && overlap(r_out, rs)) || (x_out != y && overlap(xs, ys)))
    return fail(IFR_EINVAL, "x_out and residual_out overlap, or an output another input than its own");
  const Span gates{gate, 2 * ((gate_stride ? (seq_len - 1) * gate_stride : 0) + hidden)};
  for (const Span in : {gates, Span{post_weight, 2 * hidden}, Span{pre_weight, 2 * hidden}})
    if (overlap(r_out, in) || overlap(xs, in)) return fail(IFR_EINVAL, "an output overlaps a gate or weight");
  const ifr::NormResidualArgs a{static_cast<const uint16_t*>(y), residual, residual_out,
                                static_cast<uint16_t*>(x_out),
                                static_cast<const uint16_t*>(post_weight),
                                static_cast<const uint16_t*>(gate),
                                static_cast<const uint16_t*>(pre_weight), seq_len, hidden,
                                gate_stride, residual_type == IFR_RESIDUAL_F32, post_norm == 1,
                                eps, residual_scale, block_scale};
  return launched(ifr::launch_norm_residual(a, as_stream(stream)), "norm_residual");
}

int64_t ifr_sample_workspace_bytes(int64_t num_rows, int64_t vocab) {
  if (!sample_shape(num_rows, vocab)) return -1;
  return num_rows == 0 ? 0 : ifr::sample_workspace_bytes(num_rows, vocab);
}

int32_t ifr_dispatch_sample_tokens(const void* logits, const float* uniform, int32_t* tokens,
                                   const float* temperature, const int32_t* top_k,
                                   const float* top_p, const float* min_p, int64_t num_rows,
                                   int64_t vocab, int64_t row_stride, int64_t logits_type,
                                   void* workspace, int64_t workspace_bytes, uint64_t stream) {
  if (!sample_shape(num_rows, vocab))
    return fail(IFR_EINVAL, "num_rows must be in [0, 2^20], vocab in [1, 2^20]");
  if (row_stride < vocab || row_stride > (int64_t{1} << 32))
    return fail(IFR_EINVAL, "row_stride must be in [vocab, 2^32]");
  if (logits_type != IFR_LOGITS_BF16 && logits_type != IFR_LOGITS_F32)
    return fail(IFR_EINVAL, "logits_type must be IFR_LOGITS_BF16 or IFR_LOGITS_F32");
  if (num_rows == 0) return ifr::abi_ok();
  if (!logits || !uniform || !tokens) return fail(IFR_EINVAL, "null pointer");
  if (!aligned(logits, logits_type == IFR_LOGITS_F32 ? 4 : 2))
    return fail(IFR_EINVAL, "logits must be aligned to their elements");
  for (const void* p : {static_cast<const void*>(uniform), static_cast<const void*>(tokens),
                        static_cast<const void*>(temperature), static_cast<const void*>(top_k),
                        static_cast<const void*>(top_p), static_cast<const void*>(min_p)})
    if (!aligned(p, 4)) return fail(IFR_EINVAL, "the rows' numbers must be 4-byte aligned");
  const int64_t need = ifr::sample_workspace_bytes(num_rows, vocab);
  if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
    return fail(IFR_ESPACE, "workspace needs %lld bytes, 16-byte aligned", (long long)need);
  if (ifr::sample_scan_blocks(num_rows, vocab, logits_type == IFR_LOGITS_F32) > ifr::max_blocks(ifr::kScanThreads))
    return fail(IFR_EINVAL, "the rows have 2^24 pieces of 16 KiB of logits or more");
  const Span out{tokens, 4 * num_rows}, space{need > 0 ? workspace : nullptr, need};
  const int64_t size = logits_type == IFR_LOGITS_F32 ? 4 : 2;
  for (const Span in : {Span{logits, size * ((num_rows - 1) * row_stride + vocab)}, Span{uniform, 4 * num_rows},
                        Span{temperature, 4 * num_rows}, Span{top_k, 4 * num_rows}, Span{top_p, 4 * num_rows},
                        Span{min_p, 4 * num_rows}})
    if (overlap(out, in) || overlap(space, in))
      return fail(IFR_EINVAL, "tokens or workspace overlap an input");
  if (overlap(out, space)) return fail(IFR_EINVAL, "tokens overlap the workspace");
  const ifr::SampleArgs a{logits, row_stride, logits_type == IFR_LOGITS_F32, temperature, top_k,
                          top_p, min_p, uniform, tokens, num_rows, vocab, workspace};
  return launched(ifr::launch_sample(a, as_stream(stream)), "sample_tokens");
}

}  // extern "C"
