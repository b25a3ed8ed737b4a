// Attention with a window and sinks for prompts (gfx950): blocks of many queries, over bf16
// and 8-bit caches.
//
// A block's waves share tiles of 32 positions of K and V in LDS.  A wave holds 16 x kNc
// columns, (token, q head) pairs, with all head_dim dims of their sums (kNc = 512 / D, so
// 128 accumulators and 64 registers of queries at every head_dim), as S^T = K . Q^T and
// O^T += V^T . P^T in 16x16x32 MFMAs: the weights stay in the lanes that computed them (see
// window_rows.hip), K fragments are 16 bytes of an LDS row, V^T fragments come from two
// transposing LDS reads.
//
// Rows in LDS are swizzled in 16-byte chunks: K's chunk x of row r lies at x ^ (r % 16),
// V's at x ^ 2 (r % 8), so that the reads of 16 rows spread over the banks.  bf16 tiles go
// straight from the cache into LDS, 8-bit ones through registers, where the codes become
// bf16 (exactly; the scales of the two half tiles multiply scores and weights instead).
//
// The maximum of a column's softmax is only moved when a score passes it by 2^8: the
// weights are then at most 2^8, which f32 sums and bf16's exponent hold with room, and the
// accumulators are rarely multiplied.
#include <type_traits>

#include "prefill_waves.hpp"
#include "window_dev.hpp"

namespace ifr {
namespace {

using namespace window;
using prefill::lds_barrier;
using prefill::load_lds2;
using prefill::load_lds4;
using prefill::lds_s16x4_t;
using prefill::s16x4_t;
using prefill::wait_loads;

constexpr float kSlack = 8.0f;  // how far scores may pass the maximum in use, in powers of two

template <int kD, int kFormat>
__global__ __launch_bounds__(64 * prompt_waves(kD)) __attribute__((amdgpu_waves_per_eu(2, 2)))
void window_prompt_kernel(const WindowArgs a, int off_items) {
  constexpr int kWaves = prompt_waves(kD);
  constexpr int kNc = 512 / kD;                 // column tiles of a wave
  constexpr int kRowBytes = 2 * kD;             // of a tile row in LDS
  constexpr int kTileBytes = kTileKeys * kRowBytes;
  constexpr int kSteps = kD / 32, kBlocks = kD / 16;
  constexpr int kWaveRows = kTileKeys / kWaves; // rows that a wave stages
  constexpr int kLoads = kWaveRows * kRowBytes / 1024;
  constexpr int kRowLanes = kRowBytes / 16;     // lanes of a row in one staging load
  constexpr int kCodes = kTileKeys * kD / (64 * kWaves);  // 8-bit: codes of a thread
  static_assert(kFormat != kBf16 || kLoads == 4 || kLoads == 2, "a staging load of this count");
  __shared__ __align__(16) uint8_t kbuf[2 * kTileBytes];
  __shared__ __align__(16) uint8_t vbuf[2 * kTileBytes];
  __shared__ int again;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % a.num_kv;
  const int32_t* it = a.image + off_items + static_cast<int64_t>(blockIdx.x / a.num_kv) * kWorkWords;
  const int t0 = sload(it + kItT0), ntok = sload(it + kItTokens), p0 = sload(it + kItPos);
  const int lo = sload(it + kItLo), hi = sload(it + kItHi), col0 = sload(it + kItCol);
  const int32_t* rows = a.image + sload(it + kItRows);
  const int p1 = p0 + ntok - 1;
  const Span span = visible_span(p0, a.window, a.sinks);

  // Columns; those past the last token repeat it and are not stored.
  const int wave_col = wave * 16 * kNc;
  const bool wave_live = wave_col / a.gqa < ntok;
  const int wp0 = p0 + min(wave_col / a.gqa, ntok - 1);  // the wave's first and last position
  const int wp1 = p0 + min((wave_col + 16 * kNc - 1) / a.gqa, ntok - 1);
  int pos_of[kNc];
  int64_t q_row[kNc];
  bool live[kNc];
  u32x4_t qf[kNc][kSteps];
#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    const int col = wave_col + 16 * n + c;
    const int tok = col / a.gqa;
    live[n] = tok < ntok;
    const int tk = min(tok, ntok - 1);
    pos_of[n] = p0 + tk;
    q_row[n] = static_cast<int64_t>(t0 + tk) * a.num_q + h * a.gqa + (live[n] ? col - tok * a.gqa : 0);
    const uint16_t* qr = static_cast<const uint16_t*>(a.q) + q_row[n] * kD + 8 * g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[n][s] = *reinterpret_cast<const u32x4_t*>(qr + 32 * s);
  }

  const int64_t row_bytes = a.kv_stride * elt_bytes(kFormat);
  const uint32_t rb32 = static_cast<uint32_t>(row_bytes);
  const char* kb = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * kD * elt_bytes(kFormat);
  const char* vb = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * kD * elt_bytes(kFormat);
  auto tile_pos = [&](int vt) { return kTileKeys * (vt < span.n_sink ? vt : vt - span.n_sink + span.first); };

  // ---- staging ----
  // bf16: load i of a wave moves its rows i * 64 / kRowLanes + lane / kRowLanes; LDS is
  // filled in order, so the swizzle is in the chunk that a lane fetches.
  // Rows that no query of the block sees: K's scores are masked, V's row is another one
  // that is seen (its weights are 0).
  auto stage_bf16 = [&](int vt, int buf) {
    const int pos0 = tile_pos(vt);
    const int64_t row = tile_row(rows, pos0, a.shift, a.row_mask);
    const int w_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
    const bool unseen = pos0 + kTileKeys - 1 > p1 || (pos0 < w_lo && pos0 + kTileKeys - 1 >= a.sinks);
    uint32_t ko[kLoads], vo[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = wave * kWaveRows + i * (64 / kRowLanes) + lane / kRowLanes;
      const uint32_t x = lane % kRowLanes;
      int rv = r;
      if (unseen) {
        const int j = pos0 + r;
        if (j > p1) rv = p1 - pos0;
        else if (j < w_lo && j >= a.sinks) rv = (w_lo < pos0 + kTileKeys ? w_lo : a.sinks - 1) - pos0;
      }
      const uint32_t shift = 1024u * (3 - i);  // the instruction's offset counts on both sides
      ko[i] = static_cast<uint32_t>(r) * rb32 + 16u * (x ^ (r & 15)) + shift;
      vo[i] = static_cast<uint32_t>(rv) * rb32 + 16u * (x ^ (2 * (r & 7))) + shift;
    }
    const char* kt = kb + row * row_bytes - 3072;
    const char* vt_ = vb + row * row_bytes - 3072;
    uint8_t* kd = kbuf + buf * kTileBytes + wave * kWaveRows * kRowBytes;
    uint8_t* vd = vbuf + buf * kTileBytes + wave * kWaveRows * kRowBytes;
    if constexpr (kLoads == 4) {
      load_lds4(kt, ko[0], ko[1], ko[2], ko[3], kd);
      load_lds4(vt_, vo[0], vo[1], vo[2], vo[3], vd);
    } else {
      load_lds2(kt, ko[0], ko[1], kd);
      load_lds2(vt_, vo[0], vo[1], vd);
    }
  };
  // 8-bit: a thread's kCodes codes of one row, to registers and later to LDS.
  constexpr int kRowThreads = kD / kCodes;
  const int sr = threadIdx.x / kRowThreads, sx = threadIdx.x % kRowThreads;
  u32x4_t kc[kCodes / 16], vc[kCodes / 16];
  auto fetch_codes = [&](int vt) {
    const int pos0 = tile_pos(vt);
    const int64_t row = tile_row(rows, pos0, a.shift, a.row_mask);
    const uint32_t off = static_cast<uint32_t>(sr) * rb32 + static_cast<uint32_t>(kCodes) * sx;
    const char* kt = kb + row * row_bytes;
    const char* vt_ = vb + row * row_bytes;
#pragma unroll
    for (int i = 0; i < kCodes / 16; ++i) {
      kc[i] = *reinterpret_cast<const u32x4_t*>(kt + off + 16 * i);
      vc[i] = *reinterpret_cast<const u32x4_t*>(vt_ + off + 16 * i);
    }
  };
  auto store_codes = [&](int vt, int buf) {
    const bool seen = any_seen(p0, p1, tile_pos(vt) + sr, 1, a.window, a.sinks);
    uint8_t* kd = kbuf + buf * kTileBytes + sr * kRowBytes;
    uint8_t* vd = vbuf + buf * kTileBytes + sr * kRowBytes;
#pragma unroll
    for (int i = 0; i < kCodes / 16; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = sx * (kCodes / 8) + 2 * i + e;
        const u32x2_t k0 = codes4_bf16<kFormat>(kc[i][2 * e]), k1 = codes4_bf16<kFormat>(kc[i][2 * e + 1]);
        const u32x2_t v0 = codes4_bf16<kFormat>(seen ? vc[i][2 * e] : 0u), v1 = codes4_bf16<kFormat>(seen ? vc[i][2 * e + 1] : 0u);
        *reinterpret_cast<u32x4_t*>(kd + 16 * (x ^ (sr & 15))) = u32x4_t{k0[0], k0[1], k1[0], k1[1]};
        *reinterpret_cast<u32x4_t*>(vd + 16 * (x ^ (2 * (sr & 7)))) = u32x4_t{v0[0], v0[1], v1[0], v1[1]};
      }
  };

  // ---- LDS reads ----
  // K fragment of half tile u, step s: chunk 4 s + g of row 16 u + c.
  int k_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) k_at[i] = c * kRowBytes + 16 * ((4 * i + g) ^ c);
  // V^T fragment of dims 16 b ..: rows 4 g + c / 4 of both halves, 8 bytes at dim 4 (c % 4).
  int v_at[8];
  {
    const int r = 4 * g + (c >> 2);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v_at[i] = r * kRowBytes + 16 * ((2 * i + ((c & 3) >> 1)) ^ (2 * (r & 7))) + 8 * (c & 1);
  }

  float m[kNc], l[kNc];
  f32x4_t acc[kBlocks][kNc];

  // careful: the second walk of a block whose first one ended with a sum that is not finite.
  auto compute = [&](auto careful, int vt, int buf) {
    constexpr bool kCareful = decltype(careful)::value;
    const int pos0 = tile_pos(vt);
    if (!wave_live || !any_seen(wp0, wp1, pos0, kTileKeys, a.window, a.sinks)) return;  // wave-uniform
    const bool masked = !all_seen(wp0, wp1, pos0, kTileKeys, a.window, a.sinks);
    float ks[2] = {1.0f, 1.0f}, vs[2] = {1.0f, 1.0f};
    if constexpr (kFormat != kBf16) {
      const int64_t row = tile_row(rows, pos0, a.shift, a.row_mask);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        ks[u] = vs[u] = 0.0f;
        if (!masked || any_seen(wp0, wp1, pos0 + 16 * u, 16, a.window, a.sinks)) {
          const int64_t s = ((row + 16 * u) >> a.block_shift) * a.num_kv + h;
          ks[u] = sload_f32(a.k_scale + s);
          vs[u] = sload_f32(a.v_scale + s);
        }
      }
    }
    const uint8_t* kt = kbuf + buf * kTileBytes;
    const uint8_t* vt_ = vbuf + buf * kTileBytes;
    f32x4_t s4[2][kNc];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < kNc; ++n) s4[u][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(kt + k_at[s & 3] + (s >> 2) * 256 + u * 16 * kRowBytes);
#pragma unroll
        for (int n = 0; n < kNc; ++n)
          s4[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, __builtin_bit_cast(bf16x8_t, qf[n][s]), s4[u][n], 0, 0, 0);
      }
    bf16x8_t pf[kNc];
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      float sc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j] = s4[j >> 2][n][j & 3] * (a.scale_log2 * ks[j >> 2]);
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sc[j] = sees(pos_of[n], pos0 + 16 * (j >> 2) + 4 * g + (j & 3), a.window, a.sinks) ? sc[j] : -INFINITY;
      }
      float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
      mx = groups_max(mx);
      if (__builtin_amdgcn_ballot_w64(mx > m[n] + kSlack) != 0) {  // wave-uniform
        const float m_new = mx > m[n] + kSlack ? mx : m[n];
        const float corr = m_new == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - m_new);
        m[n] = m_new;
        l[n] *= corr;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[b][n] *= corr;
      }
      const float ref = m[n] == -INFINITY ? 0.0f : m[n];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(sc[j] - ref);
        l[n] += w[j];
        if constexpr (kFormat != kBf16) w[j] *= vs[j >> 2];
      }
      // Rounded to bf16 for the product: off by 2^-9 of each weight at most, which
      // independent values average to less than the result's own rounding.
      u32x4_t ph;
#pragma unroll
      for (int j = 0; j < 4; ++j) ph[j] = pack_bf16(w[2 * j], w[2 * j + 1]);
      pf[n] = __builtin_bit_cast(bf16x8_t, ph);
    }
    auto v_frag = [&](int b) {
      const uint8_t* at = vt_ + v_at[b & 7] + (b >> 3) * 256;
      const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)at);
      const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(at + 16 * kRowBytes));
      return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    if constexpr (kCareful) {
      bf16x8_t ones[kNc];
#pragma unroll
      for (int n = 0; n < kNc; ++n) ones[n] = seen_ones(pos_of[n], pos0, g, a.window, a.sinks);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        __builtin_amdgcn_sched_barrier(0);  // one fragment at a time: registers
        const Parts v = taken_apart(v_frag(b));
#pragma unroll
        for (int n = 0; n < kNc; ++n) {
          acc[b][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.finite, pf[n], acc[b][n], 0, 0, 0);
          acc[b][n] = add_infinities(acc[b][n], v, ones[n]);
        }
      }
      return;
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, v_frag(b));
#pragma unroll
      for (int n = 0; n < kNc; ++n) acc[b][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n], acc[b][n], 0, 0, 0);
    }
  };

  auto walk = [&](auto careful) {
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) acc[b][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if constexpr (kFormat == kBf16) {
      stage_bf16(lo, 0);
    } else {
      fetch_codes(lo);
      store_codes(lo, 0);
    }
    wait_loads<0>();
    lds_barrier();
    // One barrier a tile: a buffer is filled again after the barrier that ended its reads.
    for (int vt = lo; vt < hi; ++vt) {
      const int buf = (vt - lo) & 1;
      const bool more = vt + 1 < hi;
      if (more) {
        if constexpr (kFormat == kBf16) stage_bf16(vt + 1, buf ^ 1);
        else fetch_codes(vt + 1);
      }
      compute(careful, vt, buf);
      if constexpr (kFormat != kBf16)
        if (more) store_codes(vt + 1, buf ^ 1);
      wait_loads<0>();
      lds_barrier();
    }
  };
  if (threadIdx.x == 0) again = 0;  // ahead of the walk's first barrier
  walk(std::false_type{});
  if constexpr (kFormat != kInt8) {  // int8 codes are finite
    bool odd = false;
#pragma unroll
    for (int n = 0; n < kNc; ++n)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) odd |= !all_finite(acc[b][n]);
    if (odd) again = 1;
    lds_barrier();
    // Read by every wave ahead of the second walk, which does not write it.
    if (__builtin_amdgcn_readfirstlane(again) != 0) walk(std::true_type{});
  }

  // ---- the result, or a partial column: value r of block b is dim 16 b + 4 g + r ----
#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    const float sum = groups_sum(l[n]);
    if (!live[n]) continue;
    if (col0 < 0) {
      const float inv = 1.0f / sum;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + q_row[n] * kD + 4 * g;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        *reinterpret_cast<u32x2_t*>(dst + 16 * b) = u32x2_t{pack_bf16(acc[b][n][0] * inv, acc[b][n][1] * inv),
                                                            pack_bf16(acc[b][n][2] * inv, acc[b][n][3] * inv)};
    } else {
      const int64_t col = col0 + static_cast<int64_t>(h) * prompt_cols(kD) + wave_col + 16 * n + c;
      float* dst = a.partials + col * kD + 4 * g;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<f32x4_t*>(dst + 16 * b) = acc[b][n];
      if (g == 0) {
        a.sums[2 * col] = m[n];
        a.sums[2 * col + 1] = sum;
      }
    }
  }
}

template <int kD>
hipError_t prompts_of(const WindowArgs& a, int format, int off_items, int64_t num_items, hipStream_t stream) {
  const int64_t groups = num_items * a.num_kv;
  if (groups > kMaxGroups) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<uint32_t>(groups)), block(64 * prompt_waves(kD));
  if (format == kBf16) window_prompt_kernel<kD, kBf16><<<grid, block, 0, stream>>>(a, off_items);
  else if (format == kE4m3) window_prompt_kernel<kD, kE4m3><<<grid, block, 0, stream>>>(a, off_items);
  else window_prompt_kernel<kD, kInt8><<<grid, block, 0, stream>>>(a, off_items);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_window_prompts(const WindowArgs& a, int format, int head_dim, int off_items, int64_t num_items,
                                 hipStream_t stream) {
  if (head_dim == 128) return prompts_of<128>(a, format, off_items, num_items, stream);
  if (head_dim == 256) return prompts_of<256>(a, format, off_items, num_items, stream);
  return prompts_of<512>(a, format, off_items, num_items, stream);
}

}  // namespace ifr
