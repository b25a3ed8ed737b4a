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
using prefill::raw_max;
using prefill::load_lds2;
using prefill::load_lds4;
using prefill::lds_s16x4_t;
using prefill::s16x4_t;
using prefill::wait_loads;

// One 1 KiB load into LDS (see load_lds4).
__device__ __forceinline__ void load_lds1(const char* base, uint32_t off, const uint8_t* lds) {
  uint32_t m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %2, %3\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(m0)
      : "s"(prefill::lds_addr(lds)), "v"(off), "s"(base)
      : "memory");
}
// The lane, counted anew: what follows from it in a tile would otherwise be kept in registers
// from the first tile on, and, as there are too few, in scratch memory.  Its reloads would
// wait for every load of the next tiles in flight.
__device__ __forceinline__ int lane_now() {
  int n;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(n));
  return n;
}
__device__ __forceinline__ float max4(const float* v) { return raw_max(prefill::max3_raw(v[0], v[1], v[2]), v[3]); }

// A wave's sums, 16x16 blocks of O^T, in accumulation registers from the first product to
// the last.  Held as ordinary values, the compiler moves them between the two halves of the
// register file for every tile, as the rare multiplication by a correction and the store
// are VALU work; so all that touches them is written as instructions here.  The compiler
// does not know that these are MFMAs: what VALU instructions wrote (a move of an operand
// that the compiler put there among them) is read two wait states later at the earliest,
// hence the s_nop 1, and the sums are read behind accs_settled().
__device__ __forceinline__ void acc_zero(f32x4_t& acc) {
  const u32x4_t none = u32x4_t{0u, 0u, 0u, 0u};
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(none));
}
__device__ __forceinline__ void acc_mfma(f32x4_t& acc, bf16x8_t x, bf16x8_t y) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
}
// Scores, in ordinary registers: as the compiler's own MFMAs they would be given accumulation
// registers, and the sums pushed out of them.
__device__ __forceinline__ void score_first(f32x4_t& s, bf16x8_t x, bf16x8_t y) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(x), "v"(y));
}
__device__ __forceinline__ void score_mfma(f32x4_t& s, bf16x8_t x, bf16x8_t y) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(x), "v"(y));
}
__device__ __forceinline__ void accs_settled() { asm volatile("s_nop 15\n\ts_nop 15"); }
// Two blocks to ordinary registers, and back, over 2 KiB of LDS that the wave has to itself
// (at: this lane's 16 bytes).
constexpr int kOwnBytes = 2048;
__device__ __forceinline__ void accs_out(f32x4_t* v, const f32x4_t& a0, const f32x4_t& a1, uint32_t at) {
  asm volatile(
      "ds_write_b128 %2, %3\n\tds_write_b128 %2, %4 offset:1024\n\ts_waitcnt lgkmcnt(0)\n\t"
      "ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1])
      : "v"(at), "a"(a0), "a"(a1)
      : "memory");
}
__device__ __forceinline__ void accs_in(f32x4_t& a0, f32x4_t& a1, const f32x4_t* v, uint32_t at) {
  asm volatile(
      "ds_write_b128 %2, %3\n\tds_write_b128 %2, %4 offset:1024\n\ts_waitcnt lgkmcnt(0)\n\t"
      "ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)"
      : "=&a"(a0), "=&a"(a1)
      : "v"(at), "v"(v[0]), "v"(v[1])
      : "memory");
}

constexpr float kSlack = 24.0f;  // how far scores may pass the maximum in use, in powers of two

// One block.  False if a sum came out that is not finite: the block is then done again with
// kCareful, which stores over it (two functions, so that the registers of one do not weigh
// on the other).
template <int kD, int kFormat>
struct Prompt {
  static constexpr int kNc = prompt_col_tiles(kD);        // column tiles of a wave
  static constexpr int kRowBytes = 2 * kD;                // of a tile row in LDS
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  static constexpr int kGroup = kD == 512 ? 1 : 2;        // tiles between two barriers
  static constexpr int kStageBytes = kTileKeys * kD * elt_bytes(kFormat);  // of K, or V, as it comes from the cache
  // bf16: the tiles at hand and the next ones.  8-bit: the tiles at hand, and their codes
  // and the next ones'.
  static constexpr int kRows = kGroup * 2 * kTileBytes, kRing = 2 * kGroup * 2 * kStageBytes;
  static constexpr int kTiles = kFormat == kBf16 ? kRing : kRows + kRing;
  static constexpr int kLds = kTiles + kPromptWaves * kOwnBytes;  // and what accs_out and accs_in use
};

template <int kD, int kFormat, bool kCareful>
__device__ __forceinline__ bool prompt_block(const WindowArgs& a, int off_items, uint8_t* lds, int* odd_flag) {
  using P = Prompt<kD, kFormat>;
  constexpr int kWaves = kPromptWaves;
  constexpr int kNc = P::kNc, kRowBytes = P::kRowBytes, kTileBytes = P::kTileBytes;
  constexpr int kSteps = kD / 32, kBlocks = kD / 16;
  constexpr int kEsz = elt_bytes(kFormat);
  constexpr int kStageBytes = P::kStageBytes, kGroup = P::kGroup;
  constexpr int kLoads = kStageBytes / kWaves / 1024;     // 1 KiB loads of a wave
  constexpr int kRowLanes = kD * kEsz / 16;               // lanes of a row in one of them
  constexpr bool kMayFail = !kCareful && kFormat != kInt8;  // int8 codes are finite

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
  const int wp0 = p0 + min(wave_col / a.gqa, ntok - 1);  // the wave's first and last position
  const int wp1 = p0 + min((wave_col + 16 * kNc - 1) / a.gqa, ntok - 1);
  auto column = [&](int n, bool* live) {  // the row of q and of the output
    const int col = wave_col + 16 * n + c;
    const int tok = col / a.gqa;
    *live = tok < ntok;
    return static_cast<int64_t>(t0 + min(tok, ntok - 1)) * a.num_q + h * a.gqa + (*live ? col - tok * a.gqa : 0);
  };
  int pos_of[kNc];
  u32x4_t qf[kNc][kSteps];
#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    bool live;
    const uint16_t* qr = static_cast<const uint16_t*>(a.q) + column(n, &live) * kD + 8 * g;
    pos_of[n] = p0 + min((wave_col + 16 * n + c) / a.gqa, ntok - 1);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[n][s] = *reinterpret_cast<const u32x4_t*>(qr + 32 * s);
  }

  const int64_t row_bytes = a.kv_stride * elt_bytes(kFormat);
  const uint32_t rb32 = static_cast<uint32_t>(row_bytes);
  const char* kb = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * kD * elt_bytes(kFormat);
  const char* vb = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * kD * elt_bytes(kFormat);
  auto tile_pos = [&](int vt) { return kTileKeys * (vt < span.n_sink ? vt : vt - span.n_sink + span.first); };

  // ---- staging ----
  // Load i of a wave moves its rows i * 64 / kRowLanes + lane / kRowLanes of the tile.  LDS
  // is filled in order, so bf16's swizzle is in the chunk that a lane fetches.
  // Rows that no query of the block sees: K's scores are masked, V's row is another one
  // that is seen (its weights are 0).
  const int w_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
  auto seen_row = [&](int pos0, int r) {  // r, or the row that stands in for it
    const bool all = pos0 + kTileKeys - 1 <= p1 && (pos0 >= w_lo || pos0 + kTileKeys - 1 < a.sinks);
    if (all) return r;  // wave-uniform
    const int j = pos0 + r;
    const int gap = (w_lo < pos0 + kTileKeys ? w_lo : a.sinks - 1) - pos0;
    return j > p1 ? p1 - pos0 : (j < w_lo && j >= a.sinks) ? gap : r;
  };
  auto stage = [&](int pos0, int64_t row, uint8_t* kd, uint8_t* vd) {
    const bool both = kLoads > 0;  // else the first half of the waves loads K, the second V
    constexpr int kN = kLoads > 0 ? kLoads : 1;
    constexpr uint32_t kAt = 1024u * (kN < 2 ? 0 : kN < 4 ? 1 : 3);
    const int first = both ? wave * kN : wave % (kWaves / 2);
    const int lane = lane_now();
    uint32_t ko[kN], vo[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = (first + i) * (64 / kRowLanes) + lane / kRowLanes;
      const uint32_t x = lane % kRowLanes;
      const int rv = seen_row(pos0, r);
      const uint32_t on = kAt - 1024u * (i & 3);  // the instruction's offset counts on both sides
      ko[i] = static_cast<uint32_t>(r) * rb32 + 16u * (kFormat == kBf16 ? x ^ (r & 15) : x) + on;
      vo[i] = static_cast<uint32_t>(rv) * rb32 + 16u * (kFormat == kBf16 ? x ^ (2 * (r & 7)) : x) + on;
    }
    const char* kt = kb + row * row_bytes - kAt;
    const char* vt = vb + row * row_bytes - kAt;
    kd += first * 1024;
    vd += first * 1024;
    if constexpr (kLoads == 4) {
      load_lds4(kt, ko[0], ko[1], ko[2], ko[3], kd);
      load_lds4(vt, vo[0], vo[1], vo[2], vo[3], vd);
    } else if constexpr (kLoads == 2) {
      load_lds2(kt, ko[0], ko[1], kd);
      load_lds2(vt, vo[0], vo[1], vd);
    } else {
      static_assert(kLoads == 1 || (kLoads == 0 && kStageBytes / 1024 == kWaves / 2));
      if (both || wave < kWaves / 2) load_lds1(kt, ko[0], kd);
      if (both || wave >= kWaves / 2) load_lds1(vt, vo[0], vd);
    }
  };
  // 8-bit: the staged codes become bf16 rows, times their blocks' scales (powers of two, so
  // exactly).  A thread takes 16 codes at a time, and has loaded their scale with them.
  constexpr int kTurns = kFormat == kBf16 ? 1 : 2 * kStageBytes / 16 / (64 * kWaves);
  auto fetch_scales = [&](int pos0, int64_t row, float* scale) {
    const int thread = 64 * wave + lane_now();
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = thread + 64 * kWaves * i;
      const bool is_v = at >= kStageBytes / 16;
      const int r = at / kRowLanes % kTileKeys;
      const int64_t block = (row + (is_v ? seen_row(pos0, r) : r)) >> a.block_shift;
      scale[i] = (is_v ? a.v_scale : a.k_scale)[block * a.num_kv + h];
    }
  };
  auto convert = [&](const uint8_t* codes, uint8_t* to, const float* scale) {
    const int thread = 64 * wave + lane_now();
    u32x4_t w[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      w[i] = *reinterpret_cast<const u32x4_t*>(codes + 16 * (thread + 64 * kWaves * i));
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = thread + 64 * kWaves * i;
      const int v = at >= kStageBytes / 16 ? 1 : 0;  // of K, of V
      const int r = at / kRowLanes % kTileKeys, x = 2 * (at % kRowLanes);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x2_t y = codes4_scaled<kFormat>(w[i][2 * e], scale[i]), z = codes4_scaled<kFormat>(w[i][2 * e + 1], scale[i]);
        *reinterpret_cast<u32x4_t*>(to + v * kTileBytes + r * kRowBytes + 16 * ((x + e) ^ (v ? 2 * (r & 7) : r & 15))) =
            u32x4_t{y[0], y[1], z[0], z[1]};
      }
    }
  };

  auto own_now = [&] { return prefill::lds_addr(lds + P::kTiles + kOwnBytes * wave) + 16 * lane_now(); };

  // ---- LDS reads ----
  // K fragment of half tile u, step s: chunk 4 s + g of row 16 u + c, that is k_at ^ 64 s.
  // V^T fragment of dims 16 b ..: rows 4 g + c / 4 of both halves, 8 bytes at dim 4 (c % 4),
  // that is v_at ^ 32 b.
  float m[kNc], l[kNc];
  f32x4_t acc[kBlocks][kNc];

  // No wave leaves out a tile that none of its columns sees: the others keep the block
  // there anyway, and the branch around the accumulators would cost a copy of them.
  // ---- a tile: scores of the K at LDS kt, then weights and sums over the V at vt ----
  constexpr int kAhead = 4;  // fragments that LDS reads run ahead of their MFMAs
  float sc[kNc][8], top[kNc];
  // Tiles whose first position lies in [seen_first, seen_last], or up to seen_sink, are seen
  // whole by every column of the wave.
  const int seen_last = wp0 - (kTileKeys - 1), seen_sink = a.sinks - kTileKeys;
  const int seen_first = a.window > 0 ? wp1 - a.window + 1 : 0;
  // True if some column's maximum has to be moved first.
  auto scores = [&](int pos0, const uint8_t* kt) {
    const bool masked = pos0 > seen_last || (pos0 < seen_first && pos0 > seen_sink);  // wave-uniform
    f32x4_t s4[2][kNc];
    const int lane = lane_now();
    const int k_at = (lane & 15) * kRowBytes + 16 * ((lane >> 4) ^ (lane & 15));
    // Fragment i: half tile i % 2 of step i / 2, kAhead reads ahead of its products.
    auto k_frag = [&](int i) {
      const int s = i >> 1, u = i & 1;
      return *reinterpret_cast<const bf16x8_t*>(kt + (k_at ^ (64 * (s & 3))) + (s >> 2) * 256 + u * 16 * kRowBytes);
    };
    bf16x8_t kf[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(i);
    __builtin_amdgcn_s_setprio(1);  // products ahead of the other wave's softmax
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < kNc; ++n) {
        const bf16x8_t y = __builtin_bit_cast(bf16x8_t, qf[n][i >> 1]);
        if (i < 2) score_first(s4[i][n], kf[i % kAhead], y);
        else score_mfma(s4[i & 1][n], kf[i % kAhead], y);
      }
      if (i + kAhead < 2 * kSteps) kf[i % kAhead] = k_frag(i + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    // The compiler knows nothing of the wait states between these MFMAs and their readers.
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < kNc; ++n) asm volatile("" : "+v"(s4[u][n]));
    asm volatile("s_nop 15");
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < kNc; ++n) {
        asm volatile("" : "+v"(s4[u][n]));
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[n][4 * u + r] = s4[u][n][r];
      }
    if (masked) {
      const int j0 = pos0 + 4 * (lane_now() >> 4);  // also keeps this a branch: few tiles take it
#pragma unroll
      for (int n = 0; n < kNc; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float& x = sc[n][j];
          x = sees(pos_of[n], j0 + 16 * (j >> 2) + (j & 3), a.window, a.sinks) ? x : -INFINITY;
        }
    }
    bool move = false;
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      top[n] = prefill::groups_max(raw_max(max4(sc[n]), max4(sc[n] + 4)) * a.scale_log2);
      move |= top[n] > m[n] + kSlack;
    }
    return __builtin_amdgcn_ballot_w64(move) != 0;  // wave-uniform
  };
  auto move_maxima = [&](bool first) {
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      const float m_new = top[n] > m[n] + kSlack ? top[n] : m[n];
      const float corr = m_new == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - m_new);
      m[n] = m_new;
      l[n] *= corr;
      if (first) continue;  // the sums are 0
      if constexpr (kCareful) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[b][n] *= corr;
      } else {
        accs_settled();
        const uint32_t own = own_now();
#pragma unroll
        for (int b = 0; b < kBlocks; b += 2) {
          f32x4_t v[2];
          accs_out(v, acc[b][n], acc[b + 1][n], own);
          v[0] *= corr;
          v[1] *= corr;
          accs_in(acc[b][n], acc[b + 1][n], v, own);
        }
      }
    }
  };
  auto sums = [&](int pos0, const uint8_t* vt) {
    bf16x8_t pf[kNc];
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      const float ref = m[n] == -INFINITY ? 0.0f : m[n];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][j], a.scale_log2, -ref));
        l[n] += w[j];
      }
      // Rounded to bf16 for the product: off by 2^-8 of each weight at most, which
      // independent values average to less than the result's own rounding.
      u32x4_t ph;
#pragma unroll
      for (int j = 0; j < 4; ++j) ph[j] = pack_bf16(w[2 * j], w[2 * j + 1]);
      pf[n] = __builtin_bit_cast(bf16x8_t, ph);
    }
    const int lane = lane_now(), v_row = lane >> 2;  // 4 g + c / 4
    const int v_at = v_row * kRowBytes + 16 * (((lane & 3) >> 1) ^ (2 * (v_row & 7))) + 8 * (lane & 1);
    auto v_frag = [&](int b) {
      const uint8_t* at = vt + (v_at ^ (32 * (b & 7))) + (b >> 3) * 256;
      const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)at);
      const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(at + 16 * kRowBytes));
      return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    if constexpr (kCareful) {
      bf16x8_t ones[kNc];
#pragma unroll
      for (int n = 0; n < kNc; ++n) ones[n] = seen_ones(pos_of[n], pos0, lane >> 4, a.window, a.sinks);
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
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t vf[kAhead];
#pragma unroll
    for (int b = 0; b < kAhead; ++b) vf[b] = v_frag(b);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      __builtin_amdgcn_sched_barrier(0);
      const bf16x8_t x = __builtin_bit_cast(bf16x8_t, vf[b % kAhead]);
#pragma unroll
      for (int n = 0; n < kNc; ++n) acc_mfma(acc[b][n], x, pf[n]);
      if (b + kAhead < kBlocks) vf[b % kAhead] = v_frag(b + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  };

#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      if constexpr (kCareful) acc[b][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      else acc_zero(acc[b][n]);
    }
  }
  if (kMayFail && threadIdx.x == 0) *odd_flag = 0;
  // Groups of tiles go to two places in turn, which are filled again after the barrier that
  // ended their reads: a group is loaded during the work on the one before it.
  auto row_of = [&](int vt) { return vt < hi ? tile_row(rows, tile_pos(vt), a.shift, a.row_mask) : 0; };
  uint8_t* ring = kFormat == kBf16 ? lds : lds + P::kRows;
  int64_t next[kGroup];  // rows of the group to be loaded
  float scale[kGroup][kTurns];
  auto stage_group = [&](int vt, uint8_t* to) {
#pragma unroll
    for (int e = 0; e < kGroup; ++e)
      if (vt + e < hi) {
        const int pos0 = tile_pos(vt + e);
        if constexpr (kFormat != kBf16) fetch_scales(pos0, next[e], scale[e]);
        stage(pos0, next[e], to + e * 2 * kStageBytes, to + e * 2 * kStageBytes + kStageBytes);
        next[e] = row_of(vt + kGroup + e);
      }
  };
#pragma unroll
  for (int e = 0; e < kGroup; ++e) next[e] = row_of(lo + e);
  stage_group(lo, ring);
  int place = 0;
  for (int vt = lo; vt < hi; vt += kGroup) {
    wait_loads<0>();
    lds_barrier();  // the group is there, and the one before it has no reader left
    const uint8_t* at = ring + place * (P::kRing / 2);
    place ^= 1;
    if constexpr (kFormat != kBf16) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e)
        if (vt + e < hi) convert(at + e * 2 * kStageBytes, lds + e * 2 * kTileBytes, scale[e]);
      lds_barrier();
      at = lds;
    }
    stage_group(vt + kGroup, ring + place * (P::kRing / 2));
#pragma unroll 1
    for (int e = 0; e < kGroup && vt + e < hi; ++e) {
      const int pos0 = tile_pos(vt + e);
      if (scores(pos0, at + e * 2 * kTileBytes)) move_maxima(vt + e == lo);
      sums(pos0, at + e * 2 * kTileBytes + kTileBytes);
    }
  }
  lds_barrier();  // ahead of a second walk

  // ---- the result, or a partial column: value r of block b is dim 16 b + 4 g + r ----
  if constexpr (!kCareful) accs_settled();
  const uint32_t own = own_now();
  bool odd = false;
#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    const float sum = groups_sum(l[n]);
    bool live;
    const int64_t out_row = column(n, &live);
    const int64_t col = col0 + static_cast<int64_t>(h) * prompt_cols(kD) + wave_col + 16 * n + c;
    const float inv = 1.0f / sum;
    uint16_t* dst = static_cast<uint16_t*>(a.out) + out_row * kD + 4 * g;
    float* part = a.partials + col * kD + 4 * g;
#pragma unroll
    for (int b = 0; b < kBlocks; b += 2) {
      f32x4_t v[2];
      if constexpr (kCareful) {
        v[0] = acc[b][n];
        v[1] = acc[b + 1][n];
      } else {
        accs_out(v, acc[b][n], acc[b + 1][n], own);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        odd |= !all_finite(v[i]);
        if (!live) continue;
        if (col0 < 0)
          *reinterpret_cast<u32x2_t*>(dst + 16 * (b + i)) =
              u32x2_t{pack_bf16(v[i][0] * inv, v[i][1] * inv), pack_bf16(v[i][2] * inv, v[i][3] * inv)};
        else
          *reinterpret_cast<f32x4_t*>(part + 16 * (b + i)) = v[i];
      }
    }
    if (live && col0 >= 0 && g == 0) {
      a.sums[2 * col] = m[n];
      a.sums[2 * col + 1] = sum;
    }
  }
  if constexpr (kMayFail) {
    if (odd) *odd_flag = 1;
    lds_barrier();
    return __builtin_amdgcn_readfirstlane(*odd_flag) == 0;
  }
  return true;
}

template <int kD, int kFormat>
__global__ __launch_bounds__(64 * kPromptWaves)
__attribute__((amdgpu_waves_per_eu(2, 2)))
void window_prompt_kernel(const WindowArgs a, int off_items) {
  __shared__ __align__(16) uint8_t lds[Prompt<kD, kFormat>::kLds];
  __shared__ int odd_flag;
  if (!prompt_block<kD, kFormat, false>(a, off_items, lds, &odd_flag)) {
    lds_barrier();  // every wave has read the flag
    prompt_block<kD, kFormat, true>(a, off_items, lds, &odd_flag);
  }
}

template <int kD>
hipError_t prompts_of(const WindowArgs& a, int format, int off_items, int64_t num_items, hipStream_t stream) {
  const int64_t groups = num_items * a.num_kv;
  if (groups > kMaxGroups) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<uint32_t>(groups)), block(64 * kPromptWaves);
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
