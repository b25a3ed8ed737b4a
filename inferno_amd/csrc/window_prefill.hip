// Attention with a window and sinks for prompts (gfx950): blocks of many queries, over bf16
// and 8-bit caches.
//
// A block's eight waves share tiles of 32 positions of K and V in LDS.  A wave holds some tiles of
// columns, (token, q head) pairs, with all head_dim dims of their sums, 128 accumulators a lane at each
// head_dim: S^T = K . Q^T and O^T += V^T . P^T in 32x32x16 MFMAs (at head_dim 512, where 32 columns
// do not fit, 16x16x32).  The weights stay in the lanes that computed
// them (the order of positions inside a product is free, and V^T is read in the order in which the
// scores lie), K fragments are 16 bytes of an LDS row, V^T fragments two transposing LDS reads.
//
// Rows in LDS are swizzled in 16-byte chunks: K's chunk x of row r lies at x ^ (r % 16), V's at
// x ^ S::v_swizzle(r), so that the rows that one read takes lie in different banks.  bf16 tiles go
// straight from the cache into LDS; of 8-bit ones the codes do, and become bf16 rows, times their
// scales, between the products of the tile before (exactly: a code has at most 8 significant bits
// and a scale is a power of two).
//
// Weights are 2^(score - m) with an m that lies up to 16 powers of two above the column's largest score
// so far, and is only moved when a score passes it: the accumulators are rarely multiplied, and the
// weights are at most 1, so that no sum passes what sum |v| over the positions seen does.  At the
// other end a weight below 2^-110 of the largest counts as 0, and a result below 2^-110 loses bits.
//
// Measured: 4 prompts of 2,048 new tokens, 16 q and 8 kv heads of 256, on up to 7,693 positions of
// an int8 cache: 704 us, 966 TFLOP/s of what the mask leaves; with a window of 1,024 on a bf16 cache
// 183 us.  With all waves at the same thing at the same time the first took 769 to 785 us, the sum
// of its parts, each at the rate of the pipe that does it (repeated calls, 735 us: without the products
// 430, without the softmax 690, without loading and converting 560); two waves a SIMD is what 256
// registers each leave.  The halves of the waves apart (see the walk) cost a longer start, 3 % of a
// piece of 29 tiles; at head_dim 128 they are not, as the registers that it takes there cost 2 to 5 %.
// Tried and slower, in that form: a second barrier in each step between the halves' parts (790 us
// against 735); scores of the next tile between the weights of this one (810); 16x16x32 products with
// two or three column tiles a wave (815).  A group of two tiles a barrier made no difference, nor did
// fewer instructions for addresses.  Stores of whole cache lines over LDS saved 15 us of the second's 206.
#include <float.h>

#include <type_traits>
#include <utility>

#include "prefill_waves.hpp"
#include "window_dev.hpp"

namespace ifr {
namespace {

using namespace window;
using prefill::f32x16_t;
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
__device__ __forceinline__ uint32_t lane_now() {
  uint32_t n;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(n));
  return n;
}

// f(0) ... f(n - 1), the numbers as types: loops whose bodies the compiler's own unrolling
// finds too long.
template <typename F, int... i>
__device__ __forceinline__ void counted(F f, std::integer_sequence<int, i...>) {
  (f(std::integral_constant<int, i>{}), ...);
}
template <int n, typename F>
__device__ __forceinline__ void counted(F f) {
  counted(f, std::make_integer_sequence<int, n>{});
}

// The two MFMA shapes: 32 columns a tile, or 16 (head_dim 512, whose sums leave no room for
// 32).  A lane's scores of a tile of 32 positions are kScores values of one column; value j is
// position position(lane, j).  In the order of j they are the B operands of kParts products.
template <int kM>
struct Shape;
template <>
struct Shape<32> {
  typedef f32x16_t Acc;
  static __device__ __forceinline__ int v_swizzle(int r) { return 4 * (r & 3); }
  static constexpr int kScores = 16, kParts = 2, kHalves = 1;  // kHalves: score products' row tiles
  static __device__ __forceinline__ int position(int lane, int j) { return 8 * (j >> 2) + 4 * (lane >> 5) + (j & 3); }
  static __device__ __forceinline__ float max_over_groups(float x) {
    float a, b;
    prefill::pair32(x, a, b);
    return raw_max(a, b);
  }
  static __device__ __forceinline__ float sum_over_groups(float x) { return pair_sum32(x); }
  static __device__ __forceinline__ Acc product(bf16x8_t x, bf16x8_t y, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  }
};
template <>
struct Shape<16> {
  typedef f32x4_t Acc;
  static __device__ __forceinline__ int v_swizzle(int r) { return 2 * (r & 7); }
  static constexpr int kScores = 8, kParts = 1, kHalves = 2;
  static __device__ __forceinline__ int position(int lane, int j) { return 16 * (j >> 2) + 4 * (lane >> 4) + (j & 3); }
  static __device__ __forceinline__ float max_over_groups(float x) { return prefill::groups_max(x); }
  static __device__ __forceinline__ float sum_over_groups(float x) { return groups_sum(x); }
  static __device__ __forceinline__ Acc product(bf16x8_t x, bf16x8_t y, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
};

// A wave's sums, blocks of O^T, stay in accumulation registers from the first product to the
// last.  Held as ordinary values, the compiler moves them between the two halves of the
// register file for every tile, as the rare multiplication by a correction and the store
// are VALU work; so the products are written as instructions here.  The compiler does not know
// that these are MFMAs: what VALU instructions wrote (a move of an operand that the compiler
// put there among them) may be read two wait states later at the earliest (mfma_ready), and
// results are read behind mfma_settled().
__device__ __forceinline__ void mfma_ready() { asm volatile("s_nop 1"); }
__device__ __forceinline__ void mfma_settled() { asm volatile("s_nop 15"); }
__device__ __forceinline__ void acc_zero(f32x4_t& acc) {
  const u32x4_t none = u32x4_t{0u, 0u, 0u, 0u};
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(none));
}
__device__ __forceinline__ void acc_zero(f32x16_t& acc) {
  const u32x4_t none = u32x4_t{0u, 0u, 0u, 0u};
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(none));
}
__device__ __forceinline__ void acc_mfma(f32x4_t& acc, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
}
__device__ __forceinline__ void acc_mfma(f32x16_t& acc, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
}
// Scores, in ordinary registers: as the compiler's own MFMAs they would be given accumulation
// registers, and the sums pushed out of them.
__device__ __forceinline__ void score_first(f32x4_t& s, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(x), "v"(y));
}
__device__ __forceinline__ void score_first(f32x16_t& s, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(x), "v"(y));
}
__device__ __forceinline__ void score_mfma(f32x4_t& s, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(x), "v"(y));
}
__device__ __forceinline__ void score_mfma(f32x16_t& s, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(x), "v"(y));
}

// How far m is put above the score that moves it, in powers of two.  4 prompts of 2,048 tokens with a
// window of 1,024 take 213 us at 10, 205 at 12, 193 at 14 and 189 at 16, where
// the moves no longer show.
constexpr float kSlack = 16.0f;

// One block.  False if a sum came out that is not finite: the block is then done again with
// kCareful, which stores over it.  Both are parts of one kernel, and what the second keeps in scratch
// memory counts for the kernel's; of the first walks' tiles only those at head_dim 128 over int8 read
// a value back from there.
template <int kD, int kFormat>
struct Prompt {
  static constexpr int kM = prompt_tile_cols(kD), kNc = prompt_col_tiles(kD);  // columns of a tile, tiles of a wave
  static constexpr int kRowBytes = 2 * kD;                                     // of a tile row in LDS
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  static constexpr int kStageBytes = kTileKeys * kD * elt_bytes(kFormat);  // of K, or V, as it comes from the cache
  // How the waves go over the tiles (see the walk): at head_dim 256 in two halves, at 512 the 8-bit
  // rows between two barriers of their own, as LDS holds no second place for them.
  static constexpr bool kApart = kFormat != kBf16 && kD == 512, kSkew = kD == 256;
  // Places of K and V: of rows, and of 8-bit codes.
  static constexpr int kRowPlaces =
      kFormat == kBf16 ? (kSkew ? 4 : kD == 512 ? 2 : 3) : kApart ? 1 : kSkew ? 3 : 2;
  static constexpr int kCodePlaces = kFormat == kBf16 ? 0 : kSkew ? 3 : 2;
  // A step on one tile loads the tile this far behind it, into the place of a tile whose readers
  // a barrier has seen end.
  static constexpr int kLead = kSkew ? (kFormat == kBf16 ? 3 : 4) : kFormat == kBf16 ? kRowPlaces - 1 : kApart ? 1 : 2;
  static constexpr int kCodesAt = 2 * kRowPlaces * kTileBytes;
  static constexpr int kPosAt = kCodesAt + 2 * kCodePlaces * kStageBytes;  // the columns' positions
  static constexpr int kLds = kPosAt + kPromptWaves * 256 * kNc;
};

template <int kD, int kFormat, bool kCareful>
__device__ __forceinline__ bool prompt_block(const WindowArgs& a, int off_items, uint8_t* lds, int* odd_flag) {
  using P = Prompt<kD, kFormat>;
  constexpr int kWaves = kPromptWaves;
  using S = Shape<P::kM>;
  using Acc = typename S::Acc;
  constexpr int kM = P::kM, kNc = P::kNc, kRowBytes = P::kRowBytes, kTileBytes = P::kTileBytes;
  constexpr int kFrags = kD / 16;           // fragments of a tile of K, and of V
  constexpr int kStep = 512 / kM;           // dims of a product of scores
  constexpr int kSteps = kD / kStep, kBlocks = kD / kM;
  constexpr int kEsz = elt_bytes(kFormat);
  constexpr int kStageBytes = P::kStageBytes;
  constexpr int kLoads = kStageBytes / kWaves / 1024;     // 1 KiB loads of a wave
  constexpr int kRowLanes = kD * kEsz / 16;               // lanes of a row in one of them
  constexpr bool kMayFail = !kCareful && kFormat != kInt8;  // int8 codes are finite

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.num_kv;
  const int32_t* it = a.image + off_items + static_cast<int64_t>(blockIdx.x / a.num_kv) * kWorkWords;
  const int t0 = sload(it + kItT0), ntok = sload(it + kItTokens), p0 = sload(it + kItPos);
  const int lo = sload(it + kItLo), hi = sload(it + kItHi), col0 = sload(it + kItCol);
  const int32_t* rows = a.image + sload(it + kItRows);
  const int p1 = p0 + ntok - 1;
  const Span span = visible_span(p0, a.window, a.sinks);

  // Columns; those past the last token repeat it and are not stored.
  const int wave_col = wave * kM * kNc;
  const int wp0 = p0 + min(wave_col / a.gqa, ntok - 1);  // the wave's first and last position
  const int wp1 = p0 + min((wave_col + kM * kNc - 1) / a.gqa, ntok - 1);
  auto column = [&](int n, int lane, bool* live) {  // the row of q and of the output
    const int col = wave_col + kM * n + lane % kM;
    const int tok = col / a.gqa;
    *live = tok < ntok;
    return static_cast<int64_t>(t0 + min(tok, ntok - 1)) * a.num_q + h * a.gqa + (*live ? col - tok * a.gqa : 0);
  };
  int* own_pos = reinterpret_cast<int*>(lds + P::kPosAt) + 64 * kNc * wave;  // [kNc][64]
  u32x4_t qf[kNc][kSteps];
#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    const uint32_t lane = lane_now();
    bool live;
    const uint16_t* qr = static_cast<const uint16_t*>(a.q) + column(n, lane, &live) * kD + 8 * (lane / kM);
    own_pos[64 * n + lane] = p0 + min((wave_col + kM * n + static_cast<int>(lane % kM)) / a.gqa, ntok - 1);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[n][s] = *reinterpret_cast<const u32x4_t*>(qr + kStep * s);
  }

  const uint32_t rb32 = static_cast<uint32_t>(a.kv_stride * elt_bytes(kFormat));
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
    // Uniform: the last row seen, and the rows between the sinks and the window.
    const int last = p1 - pos0, from = max(0, a.sinks - pos0), to = max(from, w_lo - pos0);
    int gap = to < kTileKeys ? to : from - 1;
    asm("" : "+s"(gap));  // a value: else its choice becomes a branch
    const int most = min(r, last);
    return static_cast<uint32_t>(r - from) < static_cast<uint32_t>(to - from) ? gap : most;
  };
  auto all_seen = [&](int pos0) {  // no row stands in for another; wave-uniform
    return pos0 + kTileKeys - 1 <= p1 && (pos0 >= w_lo || pos0 + kTileKeys <= a.sinks);
  };
  constexpr int kN = kLoads > 0 ? kLoads : 1;
  constexpr uint32_t kAt = 1024u * (kN - 1);  // the instruction's offset counts on both sides
  // Half a load a wave: the first half of the waves loads K, the second V.
  const int first_load = kLoads > 0 ? wave * kN : wave % (kWaves / 2);
  auto offset_of = [&](bool is_v, int i, int pos0) {
    const uint32_t lane = lane_now();
    const int r = (first_load + i) * (64 / kRowLanes) + lane / kRowLanes;
    const uint32_t x = lane % kRowLanes;
    const uint32_t chunk = kFormat != kBf16 ? x : x ^ (is_v ? S::v_swizzle(r) : r & 15);
    return static_cast<uint32_t>(pos0 >= 0 ? seen_row(pos0, r) : r) * rb32 + 16u * chunk + (kAt - 1024u * i);
  };
  uint32_t k_off[kN], v_off[kN];  // of tiles that are seen whole (8-bit: the same)
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    k_off[i] = offset_of(false, i, -1);
    v_off[i] = kFormat == kBf16 ? offset_of(true, i, -1) : k_off[i];
  }
  auto stage = [&](bool is_v, int pos0, uint64_t at, uint8_t* to) {  // at: the tile's byte in the cache
    if (kLoads == 0 && is_v != (wave >= kWaves / 2)) return;
    uint32_t off[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) off[i] = is_v ? v_off[i] : k_off[i];
    if (is_v && !all_seen(pos0)) {
#pragma unroll
      for (int i = 0; i < kN; ++i) off[i] = offset_of(true, i, pos0);
    }
    const char* from = (is_v ? vb : kb) + at - kAt;
    to += first_load * 1024;
    if constexpr (kN == 4) load_lds4(from, off[0], off[1], off[2], off[3], to);
    else if constexpr (kN == 2) load_lds2(from, off[0], off[1], to);
    else load_lds1(from, off[0], to);
    static_assert(kN == 1 || kN == 2 || kN == 4);
  };
  // 8-bit: the staged codes become bf16 rows, times their blocks' scales (powers of two, so
  // exactly).  A thread takes 16 codes of a row at a time, of K or of V, and stores them in two
  // halves.  A tile's rows lie in two blocks at most, of 16 rows or more.
  constexpr int kTurns = kFormat == kBf16 ? 0 : 2 * kStageBytes / 16 / (64 * kWaves);
  struct Scales {
    float s[2];
  };
  auto scales_of = [&](bool is_v, int32_t row) {
    const float* table = is_v ? a.v_scale : a.k_scale;
    Scales x;
#pragma unroll
    for (int i = 0; i < 2; ++i) x.s[i] = sload_f32(table + static_cast<int64_t>((row + 16 * i) >> a.block_shift) * a.num_kv + h);
    return x;
  };
  // The turns of K come first, and those of V; of a single turn, the first half of the waves has K.
  auto turn_is_v = [&](int turn) { return kTurns > 1 ? turn >= kTurns / 2 : wave >= kWaves / 2; };
  auto turn_row = [&](int turn, uint32_t lane) {
    return static_cast<int>((64 * kWaves * turn + 64 * wave) / kRowLanes % kTileKeys + lane / kRowLanes);
  };
  // A turn in hand: codes, their scale, and the byte of K's or V's rows where they go.
  struct Turn {
    u32x4_t code;
    float scale;
    uint32_t to;
  };
  auto take = [&](int turn, const uint8_t* kc, const uint8_t* vc, const Scales& ks, const Scales& vs, int pos0) {
    const bool is_v = turn_is_v(turn);
    const uint32_t lane = lane_now();
    const int at = (64 * kWaves * turn + 64 * wave) % (kStageBytes / 16), r = turn_row(turn, lane);
    Turn x;
    x.code = *reinterpret_cast<const u32x4_t*>((is_v ? vc : kc) + 16 * at + 16 * lane);
    const float s0 = is_v ? vs.s[0] : ks.s[0], s1 = is_v ? vs.s[1] : ks.s[1];  // values: a choice of two places would be memory
    x.scale = (is_v ? seen_row(pos0, r) : r) < 16 ? s0 : s1;
    x.to = r * kRowBytes + 16 * (2 * (lane % kRowLanes) ^ (is_v ? S::v_swizzle(r) : r & 15));
    return x;
  };
  auto put_row = [&](int turn, int e, const Turn& x, u32x2_t y, u32x2_t z, uint8_t* kr, uint8_t* vr) {
    *reinterpret_cast<u32x4_t*>((turn_is_v(turn) ? vr : kr) + (x.to ^ 16 * e)) = u32x4_t{y[0], y[1], z[0], z[1]};
  };

  float m[kNc], l[kNc];
  Acc acc[kBlocks][kNc];

  // No wave leaves out a tile that none of its columns sees: the others keep the block
  // there anyway, and the branch around the accumulators would cost a copy of them.
  constexpr int kAhead = kNc == 1 ? 4 : 2;  // fragments that LDS reads run ahead of their MFMAs
  // Tiles whose first position lies in [seen_first, seen_last], or up to seen_sink, are seen
  // whole by every column of the wave.
  const int seen_last = wp0 - (kTileKeys - 1), seen_sink = a.sinks - kTileKeys;
  const int seen_first = a.window > 0 ? wp1 - a.window + 1 : 0;

  // ---- scores: value j of a lane's column of tile n ----
  struct Scores {
    Acc s[S::kHalves][kNc];
    __device__ __forceinline__ float get(int n, int j) const {
      return S::kHalves == 1 ? s[0][n][j] : s[j >> 2][n][j & 3];
    }
  };
  // The products of a tile of K at kt; between(i) is called behind those of fragment i, for
  // work that fills the time they take.  Fragment i: 32 rows of 16 dims, or 16 rows, half
  // i % 2, of 32.
  auto score_tile = [&](const uint8_t* kt, Scores& to, auto between) {
    const uint32_t lane = lane_now();
    const uint32_t k_at = (lane % kM) * kRowBytes + 16 * ((lane / kM) ^ (lane & 15));
    constexpr int kTurn = 16 * kStep / 8;  // bytes from one step to the next
    auto k_frag = [&](int i) {
      const int u = i % S::kHalves, byte = i / S::kHalves * kTurn;
      return *reinterpret_cast<const bf16x8_t*>(kt + (k_at ^ (byte & 255)) + (byte & ~255) + u * 16 * kRowBytes);
    };
    bf16x8_t kf[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(i);
    if constexpr (!kCareful) mfma_ready();
    __builtin_amdgcn_s_setprio(1);  // products ahead of the other wave's softmax
    counted<kFrags>([&](auto number) {
      constexpr int i = number, u = i % S::kHalves, s = i / S::kHalves;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < kNc; ++n) {
        const bf16x8_t y = __builtin_bit_cast(bf16x8_t, qf[n][s]);
        if constexpr (kCareful) to.s[u][n] = S::product(kf[i % kAhead], y, s == 0 ? Acc{} : to.s[u][n]);
        else if constexpr (s == 0) score_first(to.s[u][n], kf[i % kAhead], y);
        else score_mfma(to.s[u][n], kf[i % kAhead], y);
      }
      if constexpr (i + kAhead < kFrags) kf[i % kAhead] = k_frag(i + kAhead);
      between(number);
    });
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if constexpr (!kCareful) {
      // The compiler knows nothing of the wait states between these MFMAs and their readers.
#pragma unroll
      for (int i = 0; i < S::kHalves * kNc; ++i) asm volatile("" : "+v"(to.s[i / kNc][i % kNc]));
      mfma_settled();
#pragma unroll
      for (int i = 0; i < S::kHalves * kNc; ++i) asm volatile("" : "+v"(to.s[i / kNc][i % kNc]));
    }
  };
  auto is_masked = [&](int pos0) {  // wave-uniform
    return pos0 > seen_last || (pos0 < seen_first && pos0 > seen_sink);
  };
  auto mask = [&](Scores& x, int pos0) {
    const uint32_t lane = lane_now();
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      const int p = own_pos[64 * n + lane];
#pragma unroll
      for (int j = 0; j < S::kScores; ++j) {
        const float v = sees(p, pos0 + S::position(lane, j), a.window, a.sinks) ? x.get(n, j) : -INFINITY;
        if constexpr (S::kHalves == 1) x.s[0][n][j] = v;
        else x.s[j >> 2][n][j & 3] = v;
      }
    }
  };
  auto top_of = [&](const Scores& x, int n) {
    float top = prefill::max3_raw(x.get(n, 0), x.get(n, 1), x.get(n, 2));
#pragma unroll
    for (int j = 3; j + 1 < S::kScores; j += 2) top = prefill::max3_raw(top, x.get(n, j), x.get(n, j + 1));
    return S::max_over_groups(raw_max(top, x.get(n, S::kScores - 1)) * a.scale_log2);
  };
  // The sums as values that were settled and lie in accumulation registers.
  auto sums_settled = [&] {
    mfma_settled();
#pragma unroll
    for (int i = 0; i < kBlocks * kNc; ++i) asm volatile("" : "+a"(acc[i / kNc][i % kNc]));
  };
  // Moves the references that a score passes.
  auto move_references = [&](const float* top, bool first) {
    float corr[kNc];
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      const float m_new = top[n] > m[n] ? top[n] + kSlack : m[n];
      corr[n] = m_new == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - m_new);
      m[n] = m_new;
      l[n] *= corr[n];
    }
    if (first) return;  // the sums are 0
    if constexpr (!kCareful) sums_settled();
#pragma unroll
    for (int i = 0; i < kBlocks * kNc; ++i) {
      if constexpr (kCareful) {
        acc[i / kNc][i % kNc] *= corr[i % kNc];
      } else {
        // One block at a time through ordinary registers.
        Acc v = acc[i / kNc][i % kNc];
        asm volatile("" : "+v"(v));
        v *= corr[i % kNc];
        asm volatile("" : "+a"(v));
        acc[i / kNc][i % kNc] = v;
      }
    }
  };

  // ---- weights, as P^T's fragments ----
  struct Weights {
    u32x4_t p[S::kParts][kNc];
  };
  // Rounded to bf16 for the product, each off by 2^-8 of itself at most.  The sum of weights takes them
  // rounded too: the result is the exact softmax of the rounded weights, off by 2^-8 sum p |v - o| at
  // most.  With the weights as they were in the sum a row of which one weight is nearly all, 2^-x with any
  // x below kSlack, was off by that weight's own rounding, up to another 2^-8 of the whole result.
  auto weigh = [&](const Scores& x, Weights& w) {
    const bf16x2_t ones = bf16x2_t{1.0f, 1.0f};
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      float even = 0.0f;
#pragma unroll
      for (int j = 0; j < S::kScores; ++j) {
        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(x.get(n, j), a.scale_log2, -m[n]));
        if (j & 1) {
          const uint32_t two = pack_bf16(even, v);
          w.p[j >> 3][n][(j & 7) >> 1] = two;
          l[n] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), ones, l[n], false);
        } else {
          even = v;
        }
      }
    }
  };

  // ---- sums over a tile of V at vt; between(i) as in score_tile ----
  // Fragment i: of block i / kParts the positions of part i % kParts, 8 a lane in the order of
  // the weights, from two transposing reads of 16 lanes' 4 rows of 16 dims each.
  auto v_base = [&] {
    const int lane = lane_now();
    const int r = 4 * (lane / kM) + ((lane & 15) >> 2), x = (lane % kM / 16) * 2 + ((lane & 3) >> 1);
    return r * kRowBytes + 16 * (x ^ S::v_swizzle(r)) + 8 * (lane & 1);
  };
  auto v_frag = [&](const uint8_t* vt, int v_at, int i) {
    const int byte = i / S::kParts * 2 * kM;
    const uint8_t* at = vt + (v_at ^ (byte & 255)) + (byte & ~255) + i % S::kParts * 16 * kRowBytes;
    const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)at);
    const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(at + (kM == 32 ? 8 : 16) * kRowBytes));
    return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto sum_tile = [&](const uint8_t* vt, const Weights& w, auto between) {
    const int v_at = v_base();
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t vf[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vf[i] = v_frag(vt, v_at, i);
    mfma_ready();
    __builtin_amdgcn_s_setprio(1);
    counted<kFrags>([&](auto number) {
      constexpr int i = number, part = i % S::kParts, b = i / S::kParts;
      __builtin_amdgcn_sched_barrier(0);
      const bf16x8_t x = __builtin_bit_cast(bf16x8_t, vf[i % kAhead]);
#pragma unroll
      for (int n = 0; n < kNc; ++n) acc_mfma(acc[b][n], x, __builtin_bit_cast(bf16x8_t, w.p[part][n]));
      if constexpr (i + kAhead < kFrags) vf[i % kAhead] = v_frag(vt, v_at, i + kAhead);
      between(number);
    });
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  };
  auto careful_sums = [&](const uint8_t* vt, const Weights& w, int pos0) {
    const int lane = lane_now(), v_at = v_base();
#pragma unroll
    for (int i = 0; i < kFrags; ++i) {
      __builtin_amdgcn_sched_barrier(0);  // one fragment at a time: registers
      const Parts v = taken_apart(v_frag(vt, v_at, i));
#pragma unroll
      for (int n = 0; n < kNc; ++n) {
        // 1 for each of the fragment's positions that the column sees.
        const int p = own_pos[64 * n + lane], part = i % S::kParts;
        u32x4_t ones;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint32_t one = sees(p, pos0 + S::position(lane, 8 * part + e), a.window, a.sinks) ? 0x3F80u : 0u;
          const uint32_t two = sees(p, pos0 + S::position(lane, 8 * part + e + 1), a.window, a.sinks) ? 0x3F80u : 0u;
          ones[e / 2] = one | two << 16;
        }
        const bf16x8_t seen = __builtin_bit_cast(bf16x8_t, ones);
        Acc& sum = acc[i / S::kParts][n];
        sum = S::product(v.finite, __builtin_bit_cast(bf16x8_t, w.p[part][n]), sum);
        sum = with_infinities(sum, S::product(v.up, seen, Acc{}), S::product(v.down, seen, Acc{}));
      }
    }
  };

#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    m[n] = -FLT_MAX;  // not -inf: scores that are take it away from them
    l[n] = 0.0f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      if constexpr (kCareful) acc[b][n] = Acc{};
      else acc_zero(acc[b][n]);
    }
  }
  if (kMayFail && wave == 0) *odd_flag = 0;

  // ---- the walk over tiles ----
  auto rows_at = [&](bool is_v, int place) { return lds + (is_v * P::kRowPlaces + place) * kTileBytes; };
  auto codes_at = [&](bool is_v, int place) { return lds + P::kCodesAt + (is_v * P::kCodePlaces + place) * kStageBytes; };
  const int num = hi - lo;  // tiles
  auto pos_at = [&](int t) { return tile_pos(lo + t); };
  auto entry_at = [&](int t) { return sload(rows + (pos_at(min(t, num - 1)) >> a.shift)); };
  auto row_at = [&](int t, int32_t entry) { return entry + (pos_at(t) & a.row_mask); };  // cache rows are below 2^31
  auto load_k = [&](int t, int32_t row, int place) {
    if (t < num) stage(false, pos_at(t), static_cast<uint64_t>(static_cast<uint32_t>(row)) * rb32, kFormat == kBf16 ? rows_at(false, place) : codes_at(false, place));
  };
  auto load_v = [&](int t, int32_t row, int place) {
    if (t < num) stage(true, pos_at(t), static_cast<uint64_t>(static_cast<uint32_t>(row)) * rb32, kFormat == kBf16 ? rows_at(true, place) : codes_at(true, place));
  };
  // Scores to weights.
  auto soften = [&](Scores& x, Weights& w, int t) {
    const int pos0 = pos_at(t);
    if (is_masked(pos0)) mask(x, pos0);
    float top[kNc];
    bool move = false;
#pragma unroll
    for (int n = 0; n < kNc; ++n) {
      top[n] = top_of(x, n);
      move |= top[n] > m[n];
    }
    if (__builtin_amdgcn_ballot_w64(move) != 0) move_references(top, t == 0);
    weigh(x, w);
  };
  auto begin = [&] {
    wait_loads<0>();
    lds_barrier();
  };
  // All codes at a place become rows.
  auto rows_from = [&](int code_place, int row_place, int32_t row, int t) {
    const Scales ks = scales_of(false, row), vs = scales_of(true, row);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const Turn x = take(i, codes_at(false, code_place), codes_at(true, code_place), ks, vs, pos_at(t));
#pragma unroll
      for (int e = 0; e < 2; ++e)
        put_row(i, e, x, codes4_scaled<kFormat>(x.code[2 * e], x.scale), codes4_scaled<kFormat>(x.code[2 * e + 1], x.scale),
                rows_at(false, row_place), rows_at(true, row_place));
    }
  };

  if constexpr (kCareful) {
    // One tile at a time.
    for (int t = 0; t < num; ++t) {
      const int32_t row = row_at(t, entry_at(t));
      lds_barrier();  // the tile before it has no reader left
      load_k(t, row, 0);
      load_v(t, row, 0);
      begin();
      if constexpr (kFormat != kBf16) {
        rows_from(0, 0, row, t);
        lds_barrier();
      }
      Scores x;
      score_tile(rows_at(false, 0), x, [](auto) {});
      Weights w;
      soften(x, w, t);
      careful_sums(rows_at(true, 0), w, pos_at(t));
    }
  } else {
    // Between the products of a step's scores the loads of a later tile are started, and between
    // those of its sums the codes of the next tile become rows.
    //
    // At head_dim 256 the second half of the waves, the others of the first half's SIMDs, has its
    // barrier of a step behind the scores instead of ahead of them, so that one wave of a SIMD has
    // products to do while the other is at its softmax.  Between barriers t and t + 1 the first half
    // reads K and V of tile t, the second V of tile t and K of tile t + 1.  What is written there,
    // between the products of the sums: bf16, the loads of tile t + 3, to the place of tile t - 1,
    // whole by barrier t + 2; 8-bit, the rows of tile t + 2, to the place of tile t - 1, from codes
    // that were whole by barrier t, and the loads of the codes of tile t + 4, to the place of those of
    // tile t + 1.
    constexpr int kLead = P::kLead;
    constexpr bool kCodes = kFormat != kBf16, kApart = P::kApart, kSkew = P::kSkew;
    constexpr int kTileLoads = 2 * kLoads;  // of a wave
    constexpr int kLoadPlaces = kCodes ? P::kCodePlaces : P::kRowPlaces;
    int32_t row = row_at(0, entry_at(0)), row_next = row;  // of the tile loaded next; of the one that a step converts
    int32_t entry = entry_at(1);
    auto advance = [&](int t) {  // behind the loads of tile t
      row_next = row;
      row = row_at(t + 1, entry);
      entry = entry_at(t + 2);
    };
    int load_place = 0, row_place = 0;
    auto next_place = [](int& place, int places) { place = place + 1 == places ? 0 : place + 1; };
    auto load_next = [&](int t) {
      load_k(t, row, load_place);
      load_v(t, row, load_place);
      advance(t);
      next_place(load_place, kLoadPlaces);
    };
#pragma unroll
    for (int t = 0; t < (kLead < 3 ? kLead : 3); ++t) load_next(t);
    if constexpr (kSkew) {  // the first two tiles have come
      if (2 < num) wait_loads<kTileLoads>();
      else wait_loads<0>();
      lds_barrier();
    } else if constexpr (kCodes && !kApart) {
      begin();
    }
    if constexpr (kCodes && !kApart) {
      rows_from(0, 0, row_at(0, entry_at(0)), 0);
      if constexpr (kSkew) {
        rows_from(1, 1, row_at(1, entry_at(1)), 1);
        lds_barrier();
        load_next(3);
      }
    }
    int32_t entry_2 = kCodes && kSkew ? entry_at(2) : 0;  // of the tile that a step converts
    // What a step needs has come: all loads but those of the last tile, if they were started.
    auto step_begin = [&](int t) {
      constexpr int kMore = kSkew ? (kCodes ? 3 : 2) : kLead == 2 && !kCodes ? 1 : 0;
      if (kMore > 0 && t + kMore < num) wait_loads<kTileLoads>();
      else wait_loads<0>();
      lds_barrier();
    };
    const bool late = kSkew && wave >= kWaves / 2;

    for (int t = 0; t < num; ++t) {
      if (!late) step_begin(t);
      if constexpr (kApart) {
        const int32_t row_here = row_next;
        load_next(t + 1);
        rows_from(load_place, 0, row_here, t);
        lds_barrier();
      }
      Scores x;
      Scales ks{}, vs{};
      score_tile(rows_at(false, row_place), x, [&](auto number) {
        constexpr int i = number;
        if constexpr (kSkew && kCodes && i == 4) {
          const int32_t row_2 = row_at(t + 2, entry_2);
          ks = scales_of(false, row_2);
          vs = scales_of(true, row_2);
          entry_2 = entry_at(t + 3);
        }
        if constexpr (!kSkew && !kApart) {
          if constexpr (i == 1) load_k(t + kLead, row, load_place);
          if constexpr (i == 3) load_v(t + kLead, row, load_place);
          if constexpr (i == 4) {
            if constexpr (kCodes) {
              ks = scales_of(false, row_next);
              vs = scales_of(true, row_next);
            }
            advance(t + kLead);
          }
        }
      });
      if (late) step_begin(t);
      Weights w;
      soften(x, w, t);
      Turn turn;
      u32x2_t half;
      sum_tile(rows_at(true, row_place), w, [&](auto number) {
        constexpr int i = number;
        if constexpr (kTurns > 0 && !kApart) {
          // A word of a turn's four at a time, two products behind their read.
          static_assert(kFrags >= 6 * kTurns);
          constexpr int kTurn = i / 6, kWord = i % 6 - 2;
          const int tile = kSkew ? t + 2 : t + 1;
          const int rows = kSkew ? (row_place == 0 ? 2 : row_place - 1) : row_place ^ 1;
          const int codes = kSkew ? rows : load_place ^ 1;  // both rings of three: tile t + 2's place is that of t - 1
          if constexpr (kTurn < kTurns && kWord == -2)
            turn = take(kTurn, codes_at(false, codes), codes_at(true, codes), ks, vs, pos_at(tile));
          if constexpr (kTurn < kTurns && kWord >= 0) {
            const u32x2_t y = codes4_scaled<kFormat>(turn.code[kWord], turn.scale);
            if constexpr (kWord % 2 == 0) half = y;
            else put_row(kTurn, kWord / 2, turn, half, y, rows_at(false, rows), rows_at(true, rows));
          }
        }
        if constexpr (kSkew) {
          constexpr int kFrom = kCodes ? 6 * kTurns : 1;
          if constexpr (i == kFrom) load_k(t + kLead, row, load_place);
          if constexpr (i == kFrom + 1) load_v(t + kLead, row, load_place);
          if constexpr (i == kFrags - 1) advance(t + kLead);
        }
      });
      if constexpr (!kApart) next_place(load_place, kLoadPlaces);
      next_place(row_place, P::kRowPlaces);
    }
  }
  lds_barrier();  // ahead of a second walk

  // ---- the result, or a partial column: value r of block b is dim kM b + S::position(lane, r) ----
  if constexpr (!kCareful) sums_settled();
  // 128 bytes of each column at a time go over LDS, of which a wave has a part to itself, so that
  // stores fill whole cache lines: as the sums lie, one would touch 32 of them (19 us a block of
  // 256 columns of 256 dims, all of it waiting).
  constexpr int kOutRow = 128 + 16;
  static_assert(kPromptWaves * kM * kOutRow <= P::kPosAt);
  uint8_t* mine = lds + wave * kM * kOutRow;
  float check = 0.0f;  // NaN behind a sum that is not finite
  const int lane = lane_now();
#pragma unroll
  for (int n = 0; n < kNc; ++n) {
    const float sum = S::sum_over_groups(l[n]);
    const int64_t col = col0 + static_cast<int64_t>(h) * prompt_cols(kD) + wave_col + kM * n;
    char* to[kM / 8];  // where lane / 8 of row 8 i stores 16 bytes at a time
    bool live[kM / 8];
#pragma unroll
    for (int i = 0; i < kM / 8; ++i) {
      const int r = 8 * i + lane / 8;
      const int64_t out_row = column(n, r, &live[i]);
      to[i] = (col0 < 0 ? static_cast<char*>(a.out) + out_row * (2 * kD) : reinterpret_cast<char*>(a.partials + (col + r) * kD)) +
              16 * (lane % 8);
    }
    const auto through = [&](auto bytes, auto put) {  // of a value
      constexpr int kDims = 128 / bytes;
#pragma unroll
      for (int d = 0; d < kD; d += kDims) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = d / kM; b < (d + kDims) / kM; ++b)
#pragma unroll
          for (int r = 0; r < kM * kM / 64; r += 4) {
            const f32x4_t v = f32x4_t{acc[b][n][r], acc[b][n][r + 1], acc[b][n][r + 2], acc[b][n][r + 3]};
#pragma unroll
            for (int e = 0; e < 4; ++e) check = __builtin_fmaf(v[e], 0.0f, check);
            put(mine + lane % kM * kOutRow + bytes * (kM * b - d + S::position(lane, r)), v);
          }
#pragma unroll
        for (int i = 0; i < kM / 8; ++i) {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(mine + (8 * i + lane / 8) * kOutRow + 16 * (lane % 8));
          if (live[i]) *reinterpret_cast<u32x4_t*>(to[i] + bytes * d) = w;
        }
      }
    };
    if (col0 < 0) {
      const float inv = 1.0f / sum;
      through(std::integral_constant<int, 2>{}, [&](uint8_t* at, f32x4_t v) {
        *reinterpret_cast<u32x2_t*>(at) = u32x2_t{pack_bf16(v[0] * inv, v[1] * inv), pack_bf16(v[2] * inv, v[3] * inv)};
      });
    } else {
      through(std::integral_constant<int, 4>{}, [&](uint8_t* at, f32x4_t v) { *reinterpret_cast<f32x4_t*>(at) = v; });
      bool mine_live;
      column(n, lane, &mine_live);
      if (mine_live && lane < kM) {
        a.sums[2 * (col + lane)] = sum == 0.0f ? -INFINITY : m[n];
        a.sums[2 * (col + lane) + 1] = sum;
      }
    }
  }
  const bool odd = !(check == 0.0f);
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
