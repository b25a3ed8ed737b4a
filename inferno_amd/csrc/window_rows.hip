// Attention with a window and sinks for few queries (gfx950): single tokens and runs of a
// few tokens, over bf16 and 8-bit caches, and the merge of split sequences.
//
// A wave holds 16 columns, the (token, q head) pairs of one kv head, and walks tiles of
// 32 positions with the running maximum m and sum l of each column's softmax:
//
//   S^T[32 x 16] = K . Q^T          16x16x32 MFMA, K straight from the cache
//   p = exp2(c s - m), l += p       c = scale * log2 e, s times the block's scale
//   O^T[D x 16] += V^T . P^T
//
// A 16x16x32 MFMA gives lane (c, g) = (lane % 16, lane / 16) the scores of column c at
// positions 4 g .. 4 g + 3 of a half tile, and takes, for its column, eight positions of
// P^T.  With those eight chosen as the lane's own (4 g .. of both halves) the weights never
// leave their registers, and V is read for the same positions: a lane loads 16 bytes of
// each of its eight rows, the 16 lanes of a group one row's contiguous bytes, and the
// transposition is one v_perm_b32 for two elements.
//
// Bound by HBM: a position of a kv head is 4 D bytes (2 D in 8 bits) against 16 MFMA passes
// that the 14 idle columns of a two-head group do not make longer.  Measured: 64 single tokens, 16 q
// and 8 kv heads of 256, on 512 to 32,768 positions of e4m3: 634 us, 6.5 TB/s; with a window of 1,024
// on a bf16 cache 92 us, 5.8 TB/s.  At head_dim 512 the registers hold one workgroup a CU: 48 on 512 to
// 16,384 positions of int8 149 us, 5.4 TB/s, 33 on a window of 4,096 of bf16 149 us, 3.3 TB/s.  One
// token on 4,096 positions takes 16 us, 10 here (latency: item, page entry, K and V, the sum over
// LDS) and 6 in the merge.
#include <type_traits>

#include "window_dev.hpp"

namespace ifr {
namespace {

using namespace window;

constexpr int kWaves = 4;

// 16 columns' registers of one lane: bytes of a row that a lane loads at once (kVb), how
// many such chunks a row has (kVch), elements of a chunk (kVc).
template <int kD, int kFormat>
struct Shape {
  static constexpr int kEsz = elt_bytes(kFormat);
  static constexpr int kKl = kD * kEsz / 64;                               // 16-byte loads of a K row's lane
  static constexpr int kVb = kD * kEsz / 16 < 16 ? kD * kEsz / 16 : 16;
  static constexpr int kVch = kD * kEsz / (16 * kVb);
  static constexpr int kVc = kVb / kEsz;
  static constexpr int kSteps = kD / 32;                                   // score MFMAs of a half tile
  static constexpr int kBlocks = kD / 16;                                  // 16-dim blocks of O^T
};

template <int kD, int kFormat>
__global__ __launch_bounds__(64 * kWaves, kD == 512 ? 1 : 2)
void window_rows_kernel(const WindowArgs a, int off_items, int per_group) {
  using Sh = Shape<kD, kFormat>;
  // Where a wave's cache tile fills the registers, its queries stay in LDS (until the
  // waves' sums go there).
  constexpr bool kQueryLds = kD * Sh::kEsz >= 512;
  union Shared {
    float acc[kWaves][kRowCols][kD + 4];
    u32x4_t q[kQueryLds ? kWaves : 1][kQueryLds ? Sh::kSteps : 1][64];
  };
  __shared__ __align__(16) Shared sm;
  __shared__ float sm_ml[kWaves][kRowCols][2];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int head_groups = a.num_kv / per_group;
  const int item_id = blockIdx.x / head_groups;
  const int head0 = (blockIdx.x % head_groups) * per_group;
  const int h = head0 + wave % per_group;
  const int sub = wave / per_group, nsub = kWaves / per_group;

  const int32_t* it = a.image + off_items + static_cast<int64_t>(item_id) * kWorkWords;
  const int t0 = sload(it + kItT0), ntok = sload(it + kItTokens), p0 = sload(it + kItPos);
  const int lo = sload(it + kItLo), hi = sload(it + kItHi), col0 = sload(it + kItCol);
  const int32_t* rows = a.image + sload(it + kItRows);
  const int p1 = p0 + ntok - 1;
  const Span span = visible_span(p0, a.window, a.sinks);

  // Column c: token c / gqa, q head c % gqa; columns past the last repeat it.
  const int col_tok = c / a.gqa;
  const bool live = col_tok < ntok;
  const int tok = min(col_tok, ntok - 1);
  const int q_head = h * a.gqa + (live ? c - col_tok * a.gqa : 0);
  const int p = p0 + tok;
  const int64_t q_row = static_cast<int64_t>(t0 + tok) * a.num_q + q_head;

  // Score step s takes dims 32 s + 8 g .. + 7 of K; of 8-bit K 16 codes at a time, two
  // steps' worth: dims 64 (s / 2) + 16 g + 8 (s % 2) ...
  u32x4_t qf[kQueryLds ? 1 : Sh::kSteps];
  {
    const uint16_t* qr = static_cast<const uint16_t*>(a.q) + q_row * kD;
#pragma unroll
    for (int s = 0; s < Sh::kSteps; ++s) {
      const int d = kFormat == kBf16 ? 32 * s + 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(qr + d);
      if constexpr (kQueryLds) sm.q[wave][s][lane] = w;
      else qf[s] = w;
    }
  }
  auto query = [&](int s) {
    if constexpr (kQueryLds) return __builtin_bit_cast(bf16x8_t, sm.q[wave][s][lane]);
    else return __builtin_bit_cast(bf16x8_t, qf[s]);
  };

  const int64_t row_bytes = a.kv_stride * Sh::kEsz;
  const char* kb = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * kD * Sh::kEsz;
  const char* vb = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * kD * Sh::kEsz;
  const uint32_t k_lane = static_cast<uint32_t>(c) * static_cast<uint32_t>(row_bytes) + 16u * g;
  const uint32_t v_lane = 4u * g * static_cast<uint32_t>(row_bytes) + static_cast<uint32_t>(Sh::kVb) * c;

  u32x4_t kr[2][Sh::kKl];
  uint32_t vr[8][Sh::kVch][Sh::kVb / 4];
  float ks[2], vs[2];

  auto tile_pos = [&](int vt) { return kTileKeys * (vt < span.n_sink ? vt : vt - span.n_sink + span.first); };
  auto load_k = [&](int64_t row) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const char* base = kb + (row + 16 * u) * row_bytes;  // wave-uniform
#pragma unroll
      for (int i = 0; i < Sh::kKl; ++i)
        kr[u][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(base + k_lane + 64 * i));
    }
  };
  auto load_v = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* base = vb + (row + 16 * (j >> 2) + (j & 3)) * row_bytes;  // wave-uniform
#pragma unroll
      for (int x = 0; x < Sh::kVch; ++x) {
        if constexpr (Sh::kVb == 16) {
          const u32x4_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(base + v_lane + 256 * x));
#pragma unroll
          for (int i = 0; i < 4; ++i) vr[j][x][i] = w[i];
        } else {
          const u32x2_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(base + v_lane + 128 * x));
          vr[j][x][0] = w[0];
          vr[j][x][1] = w[1];
        }
      }
    }
  };

  float m, l;  // l: of this lane's positions alone, until the end
  f32x4_t acc[Sh::kBlocks];

  // careful: the second walk of a wave whose first one ended with a sum that is not finite.
  auto tile = [&](auto careful, int pos0, int64_t row, bool more, int64_t next) {
    constexpr bool kCareful = decltype(careful)::value;
    const bool masked = !all_seen(p0, p1, pos0, kTileKeys, a.window, a.sinks);  // wave-uniform
    // ---- scales of the two half tiles' blocks ----
    if constexpr (kFormat != kBf16) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        ks[u] = vs[u] = 0.0f;
        if (!masked || any_seen(p0, p1, pos0 + 16 * u, 16, a.window, a.sinks)) {
          const int64_t s = ((row + 16 * u) >> a.block_shift) * a.num_kv + h;
          ks[u] = sload_f32(a.k_scale + s);
          vs[u] = sload_f32(a.v_scale + s);
        }
      }
    }
    // ---- scores ----
    float sc[8];
    {
      f32x4_t s4[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) s4[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < Sh::kSteps; ++s) {
        const bf16x8_t qs = query(s);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32x4_t k4;
          if constexpr (kFormat == kBf16) {
            k4 = kr[u][s];
          } else {
            const u32x2_t x = codes4_bf16<kFormat>(kr[u][s / 2][2 * (s & 1)]);
            const u32x2_t y = codes4_bf16<kFormat>(kr[u][s / 2][2 * (s & 1) + 1]);
            k4 = u32x4_t{x[0], x[1], y[0], y[1]};
          }
          s4[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k4), qs, s4[u], 0, 0, 0);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // Not times a product of the two factors, which may pass f32's range where the scores do not.
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[4 * u + r] = (kFormat == kBf16 ? s4[u][r] : s4[u][r] * ks[u]) * a.scale_log2;
      }
    }
    if (masked) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sc[j] = sees(p, pos0 + 16 * (j >> 2) + 4 * g + (j & 3), a.window, a.sinks) ? sc[j] : -INFINITY;
    }
    // The scheduler left alone mixes the phases and runs out of registers.
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_k(next);
    __builtin_amdgcn_sched_barrier(0);
    // ---- softmax ----
    float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
    mx = groups_max(mx);
    if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {  // wave-uniform
      const float m_new = fmaxf(m, mx);
      const float corr = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= corr;
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b) acc[b] *= corr;
    }
    const float ref = m == -INFINITY ? 0.0f : m;  // a column that has seen nothing yet
    u32x4_t ph, pl;
    {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(sc[j] - ref);
        l += w[j];
        if constexpr (kFormat != kBf16) w[j] *= vs[j >> 2];
      }
      // The weights in two bf16 parts: 16 bits of each, so that the sum over V is about
      // as exact as its bf16 result needs, for MFMA passes that HBM leaves free.
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ph[j] = pack_bf16(w[2 * j], w[2 * j + 1]);
        pl[j] = pack_bf16(w[2 * j] - bf16_lo(ph[j]), w[2 * j + 1] - bf16_hi(ph[j]));
      }
    }
    const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, ph), pf_lo = __builtin_bit_cast(bf16x8_t, pl);
    // ---- O^T += V^T . P^T ----
    if (masked) {  // a weight of 0 does not stand up to a row of infinities
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool seen = any_seen(p0, p1, pos0 + 16 * (j >> 2) + 4 * g + (j & 3), 1, a.window, a.sinks);
#pragma unroll
        for (int x = 0; x < Sh::kVch; ++x)
#pragma unroll
          for (int i = 0; i < Sh::kVb / 4; ++i) vr[j][x][i] = seen ? vr[j][x][i] : 0u;
      }
    }
    auto product = [&](int b, const u32x4_t& v4) {
      if constexpr (kCareful) {
        __builtin_amdgcn_sched_barrier(0);  // one fragment at a time: registers
        const Parts v = taken_apart(v4);
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.finite, pf, acc[b], 0, 0, 0);
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.finite, pf_lo, acc[b], 0, 0, 0);
        acc[b] = add_infinities(acc[b], v, seen_ones(p, pos0, g, a.window, a.sinks));
      } else {
        const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, v4);
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, acc[b], 0, 0, 0);
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf_lo, acc[b], 0, 0, 0);
      }
    };
#pragma unroll
    for (int x = 0; x < Sh::kVch; ++x)
#pragma unroll
      for (int w = 0; w < Sh::kVb / 4; ++w) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kFormat == kBf16) {
          u32x4_t even, odd;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            even[j] = __builtin_amdgcn_perm(vr[2 * j + 1][x][w], vr[2 * j][x][w], 0x05040100u);
            odd[j] = __builtin_amdgcn_perm(vr[2 * j + 1][x][w], vr[2 * j][x][w], 0x07060302u);
          }
          product(x * Sh::kVc + 2 * w, even);
          product(x * Sh::kVc + 2 * w + 1, odd);
        } else {
          u32x4_t d[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t va = vr[2 * j][x][w], vb_ = vr[2 * j + 1][x][w];
            if constexpr (kFormat == kE4m3) {
              const u32x2_t lo2 = codes4_bf16<kE4m3>(__builtin_amdgcn_perm(vb_, va, 0x05010400u));
              const u32x2_t hi2 = codes4_bf16<kE4m3>(__builtin_amdgcn_perm(vb_, va, 0x07030602u));
              d[0][j] = lo2[0];
              d[1][j] = lo2[1];
              d[2][j] = hi2[0];
              d[3][j] = hi2[1];
            } else {
              d[0][j] = codes_bf16<kInt8, 0>(va, vb_);
              d[1][j] = codes_bf16<kInt8, 1>(va, vb_);
              d[2][j] = codes_bf16<kInt8, 2>(va, vb_);
              d[3][j] = codes_bf16<kInt8, 3>(va, vb_);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) product(x * Sh::kVc + 4 * w + e, d[e]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_v(next);
    __builtin_amdgcn_sched_barrier(0);
  };

  auto walk = [&](auto careful) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int b = 0; b < Sh::kBlocks; ++b) acc[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    int vt = lo + sub;
    if (vt >= hi) return;
    int64_t row = tile_row(rows, tile_pos(vt), a.shift, a.row_mask);
    load_k(row);
    load_v(row);
    while (vt < hi) {
      const bool more = vt + nsub < hi;
      const int64_t next = more ? tile_row(rows, tile_pos(vt + nsub), a.shift, a.row_mask) : row;
      tile(careful, tile_pos(vt), row, more, next);
      row = next;
      vt += nsub;
    }
  };
  walk(std::false_type{});
  if constexpr (kFormat != kInt8) {  // int8 codes are finite
    bool odd = false;
#pragma unroll
    for (int b = 0; b < Sh::kBlocks; ++b) odd |= !all_finite(acc[b]);
    if (__builtin_amdgcn_ballot_w64(odd) != 0) walk(std::true_type{});
  }
  l = groups_sum(l);

  // ---- the waves that shared a head's tiles, then the result or a partial column ----
  // Value r of block x kVc + i is dim (16 x + 4 g + r) kVc + i.
  uint16_t* out = static_cast<uint16_t*>(a.out);
  if (nsub == 1) {
    if (!live) return;
    if (col0 < 0) {
      const float inv = 1.0f / l;
      uint32_t* dst = reinterpret_cast<uint32_t*>(out + q_row * kD);
#pragma unroll
      for (int x = 0; x < Sh::kVch; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < Sh::kVc; i += 2)
            dst[((16 * x + 4 * g + r) * Sh::kVc + i) / 2] =
                pack_bf16(acc[x * Sh::kVc + i][r] * inv, acc[x * Sh::kVc + i + 1][r] * inv);
    } else {
      const int64_t col = col0 + static_cast<int64_t>(h) * kRowCols + c;
      f32x4_t* dst = reinterpret_cast<f32x4_t*>(a.partials + col * kD);
#pragma unroll
      for (int x = 0; x < Sh::kVch; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < Sh::kVc; i += 4) {
            const int b = x * Sh::kVc + i;
            dst[((16 * x + 4 * g + r) * Sh::kVc + i) / 4] = f32x4_t{acc[b][r], acc[b + 1][r], acc[b + 2][r], acc[b + 3][r]};
          }
      if (g == 0) {
        a.sums[2 * col] = m;
        a.sums[2 * col + 1] = l;
      }
    }
    return;
  }
  if (g == 0) {
    sm_ml[wave][c][0] = m;
    sm_ml[wave][c][1] = l;
  }
  __syncthreads();
  if (live) {
    float top = -INFINITY;
    for (int s = 0; s < nsub; ++s) top = fmaxf(top, sm_ml[wave % per_group + s * per_group][c][0]);
    const float f = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    float* dst = &sm.acc[wave][c][0];
#pragma unroll
    for (int x = 0; x < Sh::kVch; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < Sh::kVc; i += 4) {
          const int b = x * Sh::kVc + i;
          *reinterpret_cast<f32x4_t*>(dst + (16 * x + 4 * g + r) * Sh::kVc + i) =
              f32x4_t{acc[b][r] * f, acc[b + 1][r] * f, acc[b + 2][r] * f, acc[b + 3][r] * f};
        }
  }
  __syncthreads();
  const int cols = ntok * a.gqa;
  for (int i = threadIdx.x; i < per_group * cols * (kD / 4); i += 64 * kWaves) {
    const int d = 4 * (i % (kD / 4)), col_i = i / (kD / 4) % cols, ho = i / (kD / 4) / cols;
    float top = -INFINITY, sum = 0.0f;
    f32x4_t v = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < nsub; ++s) top = fmaxf(top, sm_ml[ho + s * per_group][col_i][0]);
    for (int s = 0; s < nsub; ++s) {
      const int w = ho + s * per_group;
      const float mw = sm_ml[w][col_i][0];
      sum += sm_ml[w][col_i][1] * (mw == top ? 1.0f : __builtin_amdgcn_exp2f(mw - top));
      v += *reinterpret_cast<const f32x4_t*>(&sm.acc[w][col_i][d]);
    }
    const int hh = head0 + ho;
    if (col0 < 0) {
      const float inv = 1.0f / sum;
      const int tk = col_i / a.gqa;
      const int64_t row = static_cast<int64_t>(t0 + tk) * a.num_q + hh * a.gqa + (col_i - tk * a.gqa);
      *reinterpret_cast<u32x2_t*>(out + row * kD + d) = u32x2_t{pack_bf16(v[0] * inv, v[1] * inv), pack_bf16(v[2] * inv, v[3] * inv)};
    } else {
      const int64_t col = col0 + static_cast<int64_t>(hh) * kRowCols + col_i;
      *reinterpret_cast<f32x4_t*>(a.partials + col * kD + d) = v;
      if (d == 0) {
        a.sums[2 * col] = top;
        a.sums[2 * col + 1] = sum;
      }
    }
  }
}

// The splits of a token's heads: o = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s.  A
// wave takes one q head, a lane D / 64 dims and, for the factors, one split.
template <int kD>
__global__ __launch_bounds__(64 * kWaves) void window_merge_kernel(const WindowArgs a, int off_units) {
  constexpr int kN = kD / 64;
  constexpr int kAhead = kD == 512 ? 8 : 16;  // splits' loads in flight together
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int groups = (a.num_q + kWaves - 1) / kWaves;
  const int head = (blockIdx.x % groups) * kWaves + wave;
  if (head >= a.num_q) return;
  const int32_t* un = a.image + off_units + static_cast<int64_t>(blockIdx.x / groups) * kMergeWords;
  const int n = sload(un + kUnCount);
  const int64_t step = sload(un + kUnStep);
  const int kv = head / a.gqa;
  const int64_t col = static_cast<int64_t>(sload(un + kUnCol)) + static_cast<int64_t>(kv) * sload(un + kUnHstep) + (head - kv * a.gqa);
  const float* src = a.partials + col * kD + lane * kN;
  float x[kAhead][kN];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const float* ps = src + min(s0 + e, n - 1) * step * kD;
#pragma unroll
      for (int i = 0; i < kN; ++i) x[e][i] = ps[i];
    }
  };
  float ms = -INFINITY, ls = 0.0f;
  if (lane < n) {
    ms = a.sums[2 * (col + lane * step)];
    ls = a.sums[2 * (col + lane * step) + 1];
  }
  fetch(0);  // ahead of the wait for the factors
  const float top = wave_max_ref(ms);
  const float f = ms == top ? 1.0f : __builtin_amdgcn_exp2f(ms - top);
  float sum = lane < n ? ls * f : 0.0f;
  sum = tree16_sum(sum);
  sum = pair_sum32(pair_sum16(sum));
  float v[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = 0.0f;
  for (int s0 = 0; s0 < n; s0 += kAhead) {
    if (s0 > 0) fetch(s0);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (s0 + e >= n) break;
      const float fs = readlane_f32(f, s0 + e);
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = __builtin_fmaf(x[e][i], fs, v[i]);
    }
  }
  const float inv = 1.0f / sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) +
                                              (static_cast<int64_t>(sload(un + kUnToken)) * a.num_q + head) * kD + lane * kN);
#pragma unroll
  for (int i = 0; i < kN; i += 2) dst[i / 2] = pack_bf16(v[i] * inv, v[i + 1] * inv);
}

template <int kD>
hipError_t rows_of(const WindowArgs& a, int format, int off_items, int64_t num_items, int per_group, hipStream_t stream) {
  const int64_t groups = num_items * (a.num_kv / per_group);
  if (groups > kMaxGroups) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<uint32_t>(groups));
  if (format == kBf16) window_rows_kernel<kD, kBf16><<<grid, 64 * kWaves, 0, stream>>>(a, off_items, per_group);
  else if (format == kE4m3) window_rows_kernel<kD, kE4m3><<<grid, 64 * kWaves, 0, stream>>>(a, off_items, per_group);
  else window_rows_kernel<kD, kInt8><<<grid, 64 * kWaves, 0, stream>>>(a, off_items, per_group);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_window_rows(const WindowArgs& a, int format, int head_dim, int off_items, int64_t num_items,
                              int heads_per_group, hipStream_t stream) {
  if (head_dim == 128) return rows_of<128>(a, format, off_items, num_items, heads_per_group, stream);
  if (head_dim == 256) return rows_of<256>(a, format, off_items, num_items, heads_per_group, stream);
  return rows_of<512>(a, format, off_items, num_items, heads_per_group, stream);
}

hipError_t launch_window_merge(const WindowArgs& a, int head_dim, int off_units, int64_t num_units, hipStream_t stream) {
  const int64_t groups = num_units * ((a.num_q + kWaves - 1) / kWaves);
  if (groups > kMaxGroups) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<uint32_t>(groups));
  if (head_dim == 128) window_merge_kernel<128><<<grid, 64 * kWaves, 0, stream>>>(a, off_units);
  else if (head_dim == 256) window_merge_kernel<256><<<grid, 64 * kWaves, 0, stream>>>(a, off_units);
  else window_merge_kernel<512><<<grid, 64 * kWaves, 0, stream>>>(a, off_units);
  return hipGetLastError();
}

}  // namespace ifr
