// A token a row from its logits z, with temperature T, top-k, top-p, min-p and a given u:
//   w_i = exp((z_i - max z) / T)
//   K   = the first top_k tokens by (z descending, index ascending)
//   P   = the shortest prefix of K with sum w >= top_p * sum over K of w, one token at least
//   M   = { i in P : w_i >= min_p }
//   the token is the first i of M, by index, with sum over j <= i in M of w_j > u * sum over M of w
//
// A draw lands next to a border between two tokens as often as the sums are wrong there: with
// 2^18 tokens of equal weight f32 sums would give another token in 2 to 3 % of draws.  So the
// weights and sums have 64 bits (f64 adds run at the rate of f32 ones on this card), and every sum is
// taken in an order that does not depend on timing.  Where atomics add, the weights are integers, of a
// unit of 2^-51 of the largest or, in the third launch, of at most 2^-55 of the row's sum if that is more
// (unit_bits): each is off by half a unit, which moves a border by less than 2^-31 of the whole in
// rows of up to 2^20 tokens, and a weight below half a unit counts as nothing.
//
// Three launches.  The first reads every logit once and leaves, for each 64 places, the
// largest key and, for rows that need it, the sum of weights relative to it.  The second has a
// workgroup a row, which in most cases reads a few of those 64 again and is done:
//  - without any limit, the sums give the 64 tokens in which the draw lands;
//  - a top-k of up to 1,024: the k-th largest of the 64s' largest is at most the k-th largest
//    logit, so the candidates are the tokens above it, little more than k, and histograms of them
//    say where the cuts and the draw lie (Crossing);
//  - top-p alone: the same with 128 and then 1,024, if the cut lies above; min-p alone has its
//    threshold.
// The third, with larger workgroups, takes the rows that are left: a cut among very many tokens in one
// pass (sample_wide), in parts of the row where few are left; a larger top-k or very many equal logits
// by descending through the keys, 11, 11 and 10 bits at a time, in histograms of counts or weights of
// the row.
#include <algorithm>

#include "common.hpp"
#include "step.hpp"

namespace ifr {
namespace {

constexpr int kThreads = 1024;  // of a row in the third launch
constexpr int kPickThreads = 512;
constexpr int kBins = 2048;
constexpr int kMaxSubs = 4096;  // sub-chunks of a row

// Logits in order as unsigned keys, 0 for those that are never drawn (-inf, NaN).
__device__ __forceinline__ uint32_t key_of(float z) {
  if (!(z > -__builtin_inff())) return 0;
  const uint32_t u = __float_as_uint(z + 0.0f);  // -0 is 0
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template <bool kF32>
__device__ __forceinline__ float load_logit(const void* row, int64_t i) {
  if constexpr (kF32)
    return static_cast<const float*>(row)[i];
  else
    return bf16_to_f32(static_cast<const uint16_t*>(row)[i]);
}

// 2^t for t <= 0: 2^n times the Taylor sum of 2^f = e^(f ln 2), |f| <= 1/2, up to the eleventh
// power (the next term is below 2^-47 of the result); 0 below 2^-1000, and for NaN.
constexpr double kLn2 = 0.693147180559945309417;
template <int n>
constexpr double kTaylor = kTaylor<n - 1> * kLn2 / n;
template <>
constexpr double kTaylor<0> = 1.0;
__device__ __forceinline__ double exp2_neg(double t) {
  const double n = __builtin_rint(t);
  const double f = t - n;
  double p = kTaylor<11>;
  p = __builtin_fma(p, f, kTaylor<10>);
  p = __builtin_fma(p, f, kTaylor<9>);
  p = __builtin_fma(p, f, kTaylor<8>);
  p = __builtin_fma(p, f, kTaylor<7>);
  p = __builtin_fma(p, f, kTaylor<6>);
  p = __builtin_fma(p, f, kTaylor<5>);
  p = __builtin_fma(p, f, kTaylor<4>);
  p = __builtin_fma(p, f, kTaylor<3>);
  p = __builtin_fma(p, f, kTaylor<2>);
  p = __builtin_fma(p, f, kTaylor<1>);
  p = __builtin_fma(p, f, 1.0);
  return t > -1000.0 ? __builtin_ldexp(p, static_cast<int>(n)) : 0.0;
}

// Bits behind the point of the integers that stand for weights of at most 1, of which a row has `sum`, at
// least 1: their sums stay below 2^62 and half a unit for each.
__device__ __forceinline__ int unit_bits(double sum) {
  const int log2_sum = static_cast<int>(__builtin_bit_cast(unsigned long long, sum) >> 52) - 1023;  // rounded down
  return min(51, 61 - log2_sum);
}

struct Weights {
  uint32_t top;  // the largest key
  double zmax, rate, unit;  // rate: log2 e / T; unit: of the integers of the descent
  __device__ __forceinline__ double real(uint32_t key) const {
    if (key == top) return 1.0;
    return exp2_neg((static_cast<double>(logit_of(key)) - zmax) * rate);  // inf * 0: NaN, so 0
  }
  __device__ __forceinline__ unsigned long long fixed(uint32_t key) const { return units(real(key)); }
  // weight * unit, at most 2^51, to the nearest integer: the low bits of its sum with 2^52.
  __device__ __forceinline__ unsigned long long units(double weight) const {
    return __builtin_bit_cast(unsigned long long, weight * unit + 0x1p52) & 0xFFFFFFFFFFFFFull;
  }
};

// A value of the lane that a DPP control names, 0 (or the lane's own nothing) where there is none.
template <int kCtrl, int kRows, typename T>
__device__ __forceinline__ T dpp_or_zero(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl,
                                                             kRows, 0xF, true));
  } else {
    const uint2 u = __builtin_bit_cast(uint2, v);
    uint2 r;
    r.x = __builtin_amdgcn_update_dpp(0, static_cast<int>(u.x), kCtrl, kRows, 0xF, true);
    r.y = __builtin_amdgcn_update_dpp(0, static_cast<int>(u.y), kCtrl, kRows, 0xF, true);
    return __builtin_bit_cast(T, r);
  }
}
// Sums over the lanes up to each: within rows of 16, then the rows before.
template <typename T>
__device__ __forceinline__ T wave_inclusive(T v) {
  v += dpp_or_zero<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v += dpp_or_zero<0x112, 0xF>(v);
  v += dpp_or_zero<0x114, 0xF>(v);
  v += dpp_or_zero<0x118, 0xF>(v);
  v += dpp_or_zero<0x142, 0xA>(v);  // lane 15 of a row to the next, rows 1 and 3
  v += dpp_or_zero<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
  return v;
}
template <typename T>
__device__ __forceinline__ T block_inclusive(T v, T* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_inclusive(v);
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  T before = 0;
  for (int w = 0; w < wave; ++w) before += waves[w];
  __syncthreads();
  return v + before;
}

struct Found {
  uint32_t bin;
  unsigned long long above;  // the sum over the bins above
};

// The bin, from the highest, in which the sum reaches target (1 <= target <= the sum of all).
__device__ __forceinline__ Found find_from_top(const unsigned long long* bins,
                                               unsigned long long target,
                                               unsigned long long* waves, Found* found) {
  const int hi = kBins - 1 - 2 * threadIdx.x;
  const unsigned long long a = bins[hi], b = bins[hi - 1];
  const unsigned long long incl = block_inclusive<unsigned long long>(a + b, waves);
  const unsigned long long before = incl - a - b;
  if (before < target && target <= incl) {
    const bool first = target <= before + a;
    *found = {static_cast<uint32_t>(first ? hi : hi - 1), first ? before : before + a};
  }
  __syncthreads();
  const Found f = *found;
  __syncthreads();
  return f;
}

struct Cut {
  uint32_t key;                // keys above are kept, and of this one
  unsigned long long ties;     // that many, the lowest indexes first
};

constexpr double kLog2E = 1.44269504088896340736;

// What a row asks for; k 0: no limit.
struct Asked {
  float t, top_p, min_p;
  int64_t k;
  __device__ __forceinline__ Asked(const SampleArgs& a, int64_t row) {
    t = a.temperature ? a.temperature[row] : 1.0f;
    k = a.top_k ? a.top_k[row] : 0;
    if (k < 0 || k >= a.vocab) k = 0;
    if (!(t > 0.0f)) k = a.vocab > 1 ? 1 : 0;
    top_p = a.top_p ? a.top_p[row] : 1.0f;
    if (!(top_p < 1.0f)) top_p = 1.0f;
    if (!(top_p > 0.0f)) top_p = 0.0f;
    min_p = a.min_p ? a.min_p[row] : 0.0f;
    if (!(min_p > 0.0f)) min_p = 0.0f;
    if (min_p >= 1.0f) min_p = 2.0f;  // the largest alone: a weight next to 1 rounds to 1
  }
  __device__ __forceinline__ double rate() const {
    return t > 0.0f ? kLog2E / static_cast<double>(t) : kLog2E;
  }
  // The sums of the first launch are those of the whole row.
  __device__ __forceinline__ bool needs_sums() const {
    return k == 0 && (top_p < 1.0f || min_p == 0.0f);
  }
};

// A row's logits in vectors of 16 bytes from the last aligned address at or before it: place p
// holds token p - shift.
template <bool kF32>
struct RowView {
  static constexpr int kPer = kF32 ? 4 : 8;  // logits of a vector
  const void* z;
  int shift, vocab;
  __device__ __forceinline__ RowView(const SampleArgs& a, int64_t row) {
    const char* p = static_cast<const char*>(a.logits) + row * a.row_stride * (kF32 ? 4 : 2);
    z = p;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / (kF32 ? 4 : 2);
    vocab = static_cast<int>(a.vocab);
  }
  __device__ __forceinline__ uint32_t key(int place) const {
    const int i = place - shift;
    return i >= 0 && i < vocab ? key_of(load_logit<kF32>(z, i)) : 0;
  }
  // Vectors [first_full, end_full) lie within the row.
  __device__ __forceinline__ int first_full() const { return shift ? 1 : 0; }
  __device__ __forceinline__ int end_full() const { return (shift + vocab) / kPer; }
  __device__ __forceinline__ uint4 full(int vector) const {
    return *reinterpret_cast<const uint4*>(static_cast<const char*>(z) +
                                           (static_cast<int64_t>(vector) * kPer - shift) * (kF32 ? 4 : 2));
  }
  // A vector's bits; those of -inf behind the row's ends.
  __device__ __forceinline__ uint4 raw(int place) const {
    const int i = place - shift;
    if (i >= 0 && i + kPer <= vocab) {
      if constexpr (kF32)
        return *reinterpret_cast<const uint4*>(static_cast<const float*>(z) + i);
      else
        return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(z) + i);
    }
    uint32_t b[4];
    if constexpr (kF32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        b[j] = i + j >= 0 && i + j < vocab ? static_cast<const uint32_t*>(z)[i + j] : 0xFF800000u;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t v = i + j >= 0 && i + j < vocab ? static_cast<const uint16_t*>(z)[i + j] : 0xFF80u;
        b[j / 2] |= v << (16 * (j % 2));
      }
    }
    return make_uint4(b[0], b[1], b[2], b[3]);
  }
  static __device__ __forceinline__ void split(uint4 u, float (&v)[kPer]) {
    if constexpr (kF32) {
      v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y);
      v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
    } else {
      v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
      v[4] = bf16_lo(u.z), v[5] = bf16_hi(u.z), v[6] = bf16_lo(u.w), v[7] = bf16_hi(u.w);
    }
  }
  // Its logits; -inf in the place of NaN.
  static __device__ __forceinline__ void unpack(uint4 u, float (&v)[kPer]) {
    split(u, v);
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = __builtin_fmaxf(v[j], -__builtin_inff());
  }
  __device__ __forceinline__ void logits(int place, float (&v)[kPer]) const { unpack(raw(place), v); }
};

constexpr int kSub = 64;             // places of a sub-chunk
constexpr int kScanVectors = 4;      // of a thread

// subs[row][s]: the largest key of sub-chunk s; sums[row][s]: its weights relative to that key.
// 16 lanes (f32) or 8 (bf16) have a sub-chunk, one load of 16 bytes each, four sub-chunks after each other.
// Without sums it is bound by its loads; with them, by some 20 instructions in 64 bits for each logit:
// 256 rows of 2^18 f32 logits take 84 us, 3.2 TB/s (54 at the rate of a copy), 64 mixed rows of bf16 17.
template <bool kF32>
__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(SampleArgs a, uint32_t* subs,
                                                                   double* sums, uint32_t* num_left,
                                                                   int num_subs, int chunks) {
  constexpr int kPer = RowView<kF32>::kPer;
  constexpr int kLanes = kSub / kPer;  // of a sub-chunk
  if (blockIdx.x == 0 && threadIdx.x == 0) *num_left = 0;  // for the second launch
  const int64_t row = blockIdx.x / static_cast<unsigned>(chunks);
  const int chunk = static_cast<int>(blockIdx.x - row * chunks);
  const RowView<kF32> view(a, row);
  float z[kScanVectors][kPer];
  const int v0 = chunk * kScanVectors * kScanThreads;
  if (v0 >= view.first_full() && v0 + kScanVectors * kScanThreads <= view.end_full()) {
#pragma unroll
    for (int v = 0; v < kScanVectors; ++v)
      RowView<kF32>::unpack(view.full(v0 + v * kScanThreads + static_cast<int>(threadIdx.x)), z[v]);
  } else {
#pragma unroll
    for (int v = 0; v < kScanVectors; ++v)
      view.logits((v0 + v * kScanThreads + static_cast<int>(threadIdx.x)) * kPer, z[v]);
  }
  const Asked asked(a, row);
  const bool with_sums = asked.needs_sums();
  const double rate = asked.rate();
#pragma unroll
  for (int v = 0; v < kScanVectors; ++v) {
    float top = z[v][0];
#pragma unroll
    for (int j = 1; j < kPer; ++j) top = __builtin_fmaxf(top, z[v][j]);
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
    const int s = ((chunk * kScanVectors + v) * kScanThreads + static_cast<int>(threadIdx.x)) / kLanes;
    const bool writes = threadIdx.x % kLanes == 0 && s < num_subs;
    if (writes) subs[row * num_subs + s] = key_of(top);
    if (!with_sums) continue;
    const double zmax = static_cast<double>(top);
    double sum = 0.0;
    if (__any(top == __builtin_inff())) {  // equal infinities weigh 1, though their difference is NaN
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        sum += z[v][j] == top && top > -__builtin_inff()
                   ? 1.0
                   : exp2_neg((static_cast<double>(z[v][j]) - zmax) * rate);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        sum += exp2_neg((static_cast<double>(z[v][j]) - zmax) * rate);
    }
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) sum += __shfl_xor(sum, d);
    if (writes) sums[row * num_subs + s] = sum;
  }
}

__device__ __forceinline__ double uniform_of(const SampleArgs& a, int64_t row) {
  const float u = a.uniform[row];
  return u > 0.0f ? (u < 1.0f ? static_cast<double>(u) : 1.0 - 0x1p-24) : 0.0;
}

// One lane's atomic for the wave where all its lanes have one bin and weight, as in a row of few
// different logits: 64 atomics at one address run one after the other.
__device__ __forceinline__ void add_to_bin(unsigned long long* bins, int bin, unsigned long long v) {
  if (!v) return;
  const int one = uniform_i32(bin);
  const unsigned long long here = __ballot(true), same = __ballot(bin == one);
  if (here != same) {
    atomicAdd(&bins[bin], v);
    return;
  }
  const uint32_t low = uniform_i32(static_cast<int>(v)), high = uniform_i32(static_cast<int>(v >> 32));
  const unsigned long long first = (static_cast<unsigned long long>(high) << 32) | low;
  if (__ballot(v == first) == here) {  // equal weights too
    if (__lane_id() == __ffsll(here) - 1) atomicAdd(&bins[bin], first * __popcll(here));
  } else {
    atomicAdd(&bins[bin], v);
  }
}

// The row by its keys' bits: a pass over it for each of the three digits of each cut, and one for the
// draw.  What bounds it is the one CU's instructions on every logit of each pass: 217 us for a top-k of 1,025
// of 2^18 f32 logits, 473 for a top-p of 0.5 of as many equal ones (318 and 958 with one load ahead).
template <bool kF32>
__device__ __forceinline__ void sample_descent(const SampleArgs& a, int64_t row, const RowView<kF32>& view,
                                               const Asked& asked, const Weights& w, int num_subs,
                                               unsigned long long* bins, uint32_t* tie_counts,
                                               unsigned long long* waves, Found* found) {
  constexpr int kPer = RowView<kF32>::kPer;
  const int tid = threadIdx.x, lane = tid & 63;
  const int vectors = num_subs * kSub / kPer;
  __shared__ unsigned long long s_total;
  // visit(keys, first place) for every vector of the row, in no order.
  auto each_vector = [&](auto visit) {
    constexpr int kAhead = 4;
    for (int v0 = tid; v0 - tid < vectors; v0 += kAhead * kThreads) {
      uint4 raw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) raw[i] = view.raw(min(v0 + i * kThreads, vectors) * kPer);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        float z[kPer];
        RowView<kF32>::unpack(raw[i], z);
        uint32_t key[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) key[j] = v0 + i * kThreads < vectors ? key_of(z[j]) : 0;
        visit(key, (v0 + i * kThreads) * kPer);
      }
    }
  };
  auto sum_of_all = [&](unsigned long long mine) {
    const unsigned long long incl = block_inclusive<unsigned long long>(mine, waves);
    if (tid == kThreads - 1) s_total = incl;
    __syncthreads();
    const unsigned long long all = s_total;
    __syncthreads();
    return all;
  };
  // The key in which the sum of value(key), from the largest key on, reaches target_of(the sum of
  // all), and the sum above that key; key 0 if the target is 0.
  auto descend = [&](auto value, auto target_of) {
    uint32_t prefix = 0;
    unsigned long long above = 0, target = 0;
    for (int level = 0; level < 3; ++level) {
      const int lo = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int width = level == 2 ? 10 : 11;
      for (int b = tid; b < kBins; b += kThreads) bins[b] = 0;
      __syncthreads();
      each_vector([&](const uint32_t (&key)[kPer], int) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (key[j] != 0 && (level == 0 || (key[j] >> (lo + width)) == prefix))
            add_to_bin(bins, (key[j] >> lo) & ((1u << width) - 1), value(key[j]));
      });
      __syncthreads();
      if (level == 0) {
        target = target_of(sum_of_all(bins[2 * tid] + bins[2 * tid + 1]));
        if (target == 0) return Found{0, 0};  // block-uniform
      }
      const Found f = find_from_top(bins, target - above, waves, found);
      above += f.above;
      prefix = (prefix << width) | f.bin;
    }
    return Found{prefix, above};
  };
  Cut cut{1, 0};  // key 1 stands for no logit: everything that can be drawn
  if (asked.k > 0) {
    const unsigned long long k = static_cast<unsigned long long>(asked.k);
    const Found f = descend([](uint32_t) { return 1ull; },
                            [&](unsigned long long alive) { return k < alive ? k : 0; });
    if (f.bin) cut = {f.bin, k - f.above};
  }
  if (asked.top_p < 1.0f) {
    // The kept ties of the top-k cut, all of one weight, count as one sum behind the rest.
    const unsigned long long tie = cut.ties ? w.fixed(cut.key) : 0;
    unsigned long long target = 0;
    bool in_ties = false;
    const Found f = descend([&](uint32_t key) { return key > cut.key ? w.fixed(key) : 0; },
                            [&](unsigned long long strict) {
      const unsigned long long all = strict + cut.ties * tie;
      const double want = __builtin_ceil(static_cast<double>(asked.top_p) * static_cast<double>(all));
      target = want < 1.0 ? 1 : static_cast<unsigned long long>(want);
      target = target < all ? target : all;
      in_ties = target > strict;
      if (in_ties) cut.ties = (target - strict + tie - 1) / tie;
      return in_ties ? 0ull : target;
    });
    if (!in_ties) {
      const unsigned long long each = w.fixed(f.bin);
      cut = {f.bin, (target - f.above + each - 1) / each};
    }
  }

  // By place: the weight and the ties of each of up to kMaxSubs parts of the row.
  int part = 6;  // log2 of a part's places
  while (((num_subs * kSub - 1) >> part) + 1 > kMaxSubs) ++part;
  const double floor_w = static_cast<double>(asked.min_p);
  auto kept = [&](uint32_t key) -> unsigned long long {
    const double v = w.real(key);
    return v >= floor_w || key == w.top ? w.units(v) : 0;
  };
  const unsigned long long tie = kept(cut.key);
  __syncthreads();
  for (int s = tid; s < kMaxSubs; s += kThreads) bins[s] = 0, tie_counts[s] = 0;
  __syncthreads();
  each_vector([&](const uint32_t (&key)[kPer], int place) {
    unsigned long long sum = 0;
    uint32_t ties = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (key[j] > cut.key) sum += kept(key[j]);
      ties += key[j] == cut.key;
    }
    if (sum) atomicAdd(&bins[place >> part], sum);
    if (ties) atomicAdd(&tie_counts[place >> part], ties);
  });
  __syncthreads();
  // Thread t has parts 4t .. 4t + 3.
  constexpr int kEach = kMaxSubs / kThreads;
  unsigned long long ties = 0, sum = 0;
  for (int j = 0; j < kEach; ++j) ties += tie_counts[kEach * tid + j];
  const unsigned long long ties_before = block_inclusive<unsigned long long>(ties, waves) - ties;
  unsigned long long first_ties = ties_before;
  for (int j = 0; j < kEach; ++j) {
    const int s = kEach * tid + j;
    const unsigned long long left = first_ties < cut.ties ? cut.ties - first_ties : 0;
    const unsigned long long here = tie_counts[s] < left ? tie_counts[s] : left;
    first_ties += tie_counts[s];
    bins[s] += here * tie;
    sum += bins[s];
  }
  const unsigned long long incl = block_inclusive<unsigned long long>(sum, waves);
  if (tid == kThreads - 1) s_total = incl;
  __syncthreads();
  const unsigned long long total = s_total;
  unsigned long long goal = static_cast<unsigned long long>(uniform_of(a, row) * static_cast<double>(total));
  if (goal >= total) goal = total - 1;  // total >= 1: the largest logit is kept
  __shared__ int s_part;
  __shared__ unsigned long long s_before, s_ties;
  if (incl - sum <= goal && goal < incl) {
    unsigned long long before = incl - sum;
    unsigned long long ties_at = ties_before;
    for (int j = 0; j < kEach; ++j) {
      const int s = kEach * tid + j;
      if (goal < before + bins[s]) {
        s_part = s;
        s_before = before;
        s_ties = ties_at;
        break;
      }
      before += bins[s];
      ties_at += tie_counts[s];
    }
  }
  __syncthreads();
  if (tid >= 64) return;
  unsigned long long before = s_before, ties_at = s_ties;
  const int end = (s_part + 1) << part;
  for (int p0 = s_part << part; p0 < end; p0 += 64) {
    const uint32_t key = view.key(p0 + lane);
    const unsigned long long is_tie = __ballot(key == cut.key);
    const unsigned long long order = ties_at + __popcll(is_tie & ((1ull << lane) - 1));
    const unsigned long long v = wave_inclusive(
        key > cut.key ? kept(key) : key == cut.key && order < cut.ties ? tie : 0);
    const unsigned long long hit = __ballot(before + v > goal);
    if (hit) {
      if (lane == 0) a.tokens[row] = p0 + static_cast<int>(__ffsll(hit)) - 1 - view.shift;
      return;
    }
    before += __shfl(v, 63);
    ties_at += __popcll(is_tie);
  }
}

constexpr int kMaxK = 1024;     // candidates that are sought
constexpr int kMaxTaken = 2048;  // and at most taken

// The entry in which a sum over the workgroup's entries, the largest `order` first, reaches target_of(the
// sum of all): its order, 0 if the target is 0.  Entry j of a thread has order[j] and weight[j], 0
// for none; bin_of(j) < 2 kT falls as the order rises, and the sums of the bins say in which one it lies.
template <int kT, int E>
struct Crossing {
  unsigned long long sums[2 * kT];
  unsigned long long orders[kT * E], weights[kT * E];  // of that bin's entries
  unsigned long long waves[kT / 64];
  unsigned long long total, above, result;
  int bin, count;

  template <typename Bin, typename Target>
  __device__ __forceinline__ unsigned long long find(const unsigned long long (&order)[E],
                                                     const unsigned long long (&weight)[E],
                                                     Bin bin_of, Target target_of) {
    const int tid = threadIdx.x;
    sums[2 * tid] = 0, sums[2 * tid + 1] = 0;
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (weight[j]) atomicAdd(&sums[bin_of(j)], weight[j]);
    __syncthreads();
    const unsigned long long a = sums[2 * tid], b = sums[2 * tid + 1];
    const unsigned long long incl = block_inclusive<unsigned long long>(a + b, waves);
    if (tid == kT - 1) total = incl;
    __syncthreads();
    const unsigned long long target = target_of(total);
    if (target == 0) return 0;  // block-uniform
    const unsigned long long before = incl - a - b;
    if (before < target && target <= incl) {
      const bool first = target <= before + a;
      bin = 2 * tid + !first;
      above = first ? before : before + a;
    }
    __syncthreads();
    const int at = bin;
    const unsigned long long ahead = above;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (weight[j] && bin_of(j) == at) {
        const int slot = atomicAdd(&count, 1);
        orders[slot] = order[j];
        weights[slot] = weight[j];
      }
    __syncthreads();
    const int n = count;
    for (int i = tid; i < n; i += kT) {
      const unsigned long long mine = orders[i];
      unsigned long long sum = ahead;
      for (int q = 0; q < n; ++q) sum += orders[q] > mine ? weights[q] : 0;
      if (sum < target && target <= sum + weights[i]) result = mine;
    }
    __syncthreads();
    return result;
  }
};

constexpr int kMaxBand = 11264;
constexpr int kMaxEqual = 1024;  // entries of a fine bin of the band: about as many equal logits
constexpr uint32_t kInfKey = 0xFF800000u;  // of +inf

// What the second launch leaves for the third.
struct RowRest {
  double total;       // the sum of the row's weights, if it has one
  uint32_t top;       // its largest key
  int32_t unit_bits;  // of the integers of its weights
  // Of the parts of a row: parts that are done, entries of the band, the weights above it.
  uint32_t done, listed;
  unsigned long long above;
};

constexpr uint32_t kJoinRows = 128;  // that may be in parts

// A row in parts, of whole groups of sub-chunks; the last one to end joins them.
struct Parts {
  int count, mine;
  RowRest* rest;
  unsigned long long* band;      // [kMaxBand]
  unsigned long long* sub_sums;  // [kMaxSubs]
};

// A row without a top-k that keeps very many tokens: one pass over its logits.
//
// min-p alone: the pass adds the weights of the kept ones by sub-chunk.  top-p: first a sample (about
// 16,000 of the logits, lines of 128 bytes evenly spread) says where the weights below add up to about
// 1 - top_p of all; those are many small ones, so a sample of them is good to a few percent.  Tokens
// above that band go to the sums, those within it to a list, in which the cut is then found.
// False if it is not there (or the list is full, or very many are equal): the caller descends.
//
// A CU takes 2 us for each instruction on all of 2^18 logits, so the pass does little for each:
// those at or above the band are moved together, 64 at a time, before their weights are taken.
template <bool kF32>
__device__ __forceinline__ bool sample_wide(const SampleArgs& a, int64_t row, const RowView<kF32>& view,
                                         const Asked& asked, const Weights& w, double total,
                                         int num_subs, const Parts& parts, unsigned long long* sub_sums,
                                         unsigned long long* digits, unsigned long long* band,
                                         unsigned long long* waves, Found* found, bool* joined) {
  unsigned long long* queues = digits;  // between the two uses of the digits
  __shared__ unsigned long long order[kMaxEqual];
  constexpr int kPer = RowView<kF32>::kPer;
  constexpr int kBand = 1024;  // bins of the sample
  __shared__ int s_n, s_a, s_b, s_place;
  __shared__ unsigned long long s_u64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int vectors = num_subs * kSub / kPer;
  const float zmax = logit_of(w.top);
  const bool nucleus = asked.top_p < 1.0f;
  const float rate = static_cast<float>(w.rate);
  const double floor_w = static_cast<double>(asked.min_p);
  // Bins of (zmax - z) * per, of which `above` is the first of the band; logits from z_from on are looked at.
  float per, z_from;
  int above, end = 0;  // of the band's bins
  double goal = 0.0;  // in units
  if (nucleus) {
    goal = static_cast<double>(asked.top_p) * total * w.unit;
    const double rest = (1.0 - static_cast<double>(asked.top_p)) * total;
    // Tokens of less than rest / vocab add up to less than rest: the cut is above.  (f32 will do for
    // what the band is found by.)
    const float depth = -__builtin_amdgcn_logf(static_cast<float>(rest) / static_cast<float>(view.vocab)) / rate;
    if (!(depth > 0.0f && depth < 1e30f)) return false;
    per = static_cast<float>(kBand - 1) / depth;
    if (!(per > 0.0f && per < 1e30f)) return false;
    for (int i = tid; i < kBins; i += kThreads) digits[i] = 0;
    __syncthreads();
    const int stride = max(1, vectors / (16384 / kPer));
    unsigned long long tail_sum = 0;  // of the last bin
    constexpr int kLoads = 16 / kPer;  // all of most threads'
    // Whole lines of 128 bytes, one of `stride`.
    auto sampled = [&](int i) { return i / 8 * (8 * stride) + i % 8; };
    for (int i0 = tid; sampled(i0) < vectors; i0 += kLoads * kThreads) {
      uint4 raw[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) raw[i] = view.raw(min(sampled(i0 + i * kThreads), vectors) * kPer);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        float z[kPer];
        RowView<kF32>::unpack(raw[i], z);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float x = zmax - z[j];
          const unsigned long long f = w.units(static_cast<double>(__builtin_amdgcn_exp2f(-x * rate)));
          if (x * per < kBand - 1)
            atomicAdd(&digits[static_cast<int>(x * per)], f);
          else
            tail_sum += f;  // what lies below the looked-at bins
        }
      }
    }
    tail_sum = wave_inclusive(tail_sum);
    if (lane == 63) atomicAdd(&digits[kBand - 1], tail_sum);
    if (tid == 0) s_a = 0, s_b = kBand - 1;
    __syncthreads();
    const double mine = tid < kBand ? static_cast<double>(digits[tid]) : 0.0;
    const double incl = block_inclusive<double>(mine, reinterpret_cast<double*>(waves));
    if (tid == kThreads - 1) s_u64 = static_cast<unsigned long long>(incl);
    __syncthreads();
    // Below bin tid, over the row; its error: each of the small tokens there is seen or not, and
    // weighs at most what its bin does.
    const double seen = static_cast<double>(s_u64);
    const double below = (seen - (incl - mine)) * stride, after = (seen - incl) * stride;
    const double rest_u = rest * w.unit;
    const float weight = __builtin_amdgcn_exp2f(-static_cast<float>(tid) / per * rate) * static_cast<float>(w.unit);
    const float spread = stride == 1 ? 0.0f : 2.5f * sqrtf(static_cast<float>(stride) * weight) *
                                                  sqrtf(static_cast<float>(rest_u));
    const double slack = static_cast<double>(spread) + rest_u / 128.0;
    // The band: from the last bin above which too little can be cut off, to the first below which
    // too much would be.
    if (below > rest_u + slack) atomicMax(&s_a, tid);
    if (after < rest_u - slack) atomicMin(&s_b, tid);
    __syncthreads();
    above = s_a;
    end = max(s_a, s_b) + 1;
    if (end >= kBand) return false;
    z_from = zmax - static_cast<float>(end) / per;
  } else {
    const double depth = -log2(floor_w) / w.rate;
    if (!(depth < 1e30)) return false;
    per = depth > 0.0 ? static_cast<float>((kBand - 2) / depth) : static_cast<float>(kBand);
    above = kBand;
    z_from = zmax - static_cast<float>(kBand - 1) / per;  // a bin past the exact border
  }

  if (!(per > 0.0f && per < 1e30f)) return false;

  int group = 0;
  while (((num_subs - 1) >> group) + 1 > kMaxSubs) ++group;
  for (int i = tid; i < kMaxSubs; i += kThreads) sub_sums[i] = 0;
  if (tid == 0) s_n = 0;
  __syncthreads();
  unsigned long long* queue = queues + 128 * wave;
  int head = 0, tail = 0;  // wave-uniform
  unsigned long long my_above = 0;
  auto take = [&](int n) {  // the next n of the queue, one a lane
    if (lane < n) {
      const unsigned long long e = queue[(head + lane) & 127];
      const uint32_t key = key_of(__uint_as_float(static_cast<uint32_t>(e >> 32)));
      const int place = static_cast<int>(static_cast<uint32_t>(e));
      const double v = w.real(key);
      const unsigned long long f = w.units(v);
      const float x = (zmax - logit_of(key)) * per;
      if (x < static_cast<float>(above)) {
        my_above += f;
        if (v >= floor_w || key == w.top) atomicAdd(&sub_sums[place / kSub >> group], f);
      } else {
        const int slot = atomicAdd(&s_n, 1);
        if (slot < kMaxBand)
          band[slot] = (static_cast<unsigned long long>(key) << 32) |
                       (0xFFFFFFFFu - static_cast<uint32_t>(place - view.shift));
      }
    }
    head += n;
  };
  auto push = [&](float z, float from, int place) {
    const bool in = z >= from;
    const unsigned long long m = __ballot(in);
    if (!m) return;
    if (in)
      queue[__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(m >> 32),
                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(m), tail)) & 127] =
          (static_cast<unsigned long long>(__float_as_uint(z)) << 32) | static_cast<uint32_t>(place);
    tail += __popcll(m);
    __builtin_amdgcn_wave_barrier();
    if (tail - head >= 64) take(64);
  };
  const int groups = ((num_subs - 1) >> group) + 1;
  const int first_group = static_cast<int>(static_cast<int64_t>(groups) * parts.mine / parts.count);
  const int end_group = static_cast<int>(static_cast<int64_t>(groups) * (parts.mine + 1) / parts.count);
  const int v_first = max(view.first_full(), (first_group << group) * (kSub / kPer));
  const int v_end = min(view.end_full(), (end_group << group) * (kSub / kPer));
  // (Few loads ahead: each place where the queue is emptied is a copy of that code, and 32 and more
  // of them no longer fit the instruction cache.)
  constexpr int kAhead = kF32 ? 4 : 2;
  if (v_first < v_end) {
    uint4 next[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) next[i] = view.full(min(v_first + tid + i * kThreads, v_end - 1));
    for (int v = v_first + tid; v - tid < v_end; v += kAhead * kThreads) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int at = v + i * kThreads;
        const float from = at < v_end ? z_from : __builtin_inff();  // no logit here is +inf
        float z[kPer];
        RowView<kF32>::split(next[i], z);
        next[i] = view.full(min(at + kAhead * kThreads, v_end - 1));
#pragma unroll
        for (int j = 0; j < kPer; ++j) push(z[j], from, at * kPer + j);
      }
    }
  }
  if (wave == 0) {  // the row's ends: less than two vectors
    const int row_end = max(view.end_full(), view.first_full()) * kPer;
    const int place = lane < kPer ? lane : row_end + lane - kPer;
    const bool end = lane < kPer ? parts.mine == 0 && view.first_full() > 0
                                 : parts.mine == parts.count - 1 && lane < 2 * kPer;
    const uint32_t key = end ? view.key(place) : 0;
    push(key ? logit_of(key) : -__builtin_inff(), z_from, place);
  }
  take(tail - head);
  const unsigned long long above_incl = block_inclusive<unsigned long long>(my_above, waves);
  if (tid == kThreads - 1) s_u64 = above_incl;
  __syncthreads();
  int listed = s_n;
  unsigned long long sum_above = s_u64;
  __syncthreads();
  if (parts.count > 1) {
    if (tid == 0) {
      s_a = static_cast<int>(atomicAdd(&parts.rest->listed, static_cast<uint32_t>(listed)));
      atomicAdd(&parts.rest->above, sum_above);
    }
    __syncthreads();
    const int slot = s_a;
    for (int i = tid; i < min(listed, kMaxBand - slot); i += kThreads) parts.band[slot + i] = band[i];
    for (int i = first_group + tid; i < end_group; i += kThreads) parts.sub_sums[i] = sub_sums[i];
    // All that this workgroup wrote is seen by the one that counts last: each wave's stores have reached the L2
    // ahead of the barrier, and the release of thread 0 behind it takes them on from there.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
      s_b = __hip_atomic_fetch_add(&parts.rest->done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
            static_cast<uint32_t>(parts.count - 1);
    __syncthreads();
    if (!s_b) return true;  // block-uniform
    if (tid == 0) {
      s_n = static_cast<int>(__hip_atomic_load(&parts.rest->listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      s_u64 = __hip_atomic_load(&parts.rest->above, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    listed = s_n;
    sum_above = s_u64;
    for (int i = tid; i < min(listed, kMaxBand); i += kThreads) band[i] = parts.band[i];
    for (int i = tid; i < groups; i += kThreads) sub_sums[i] = parts.sub_sums[i];
    __syncthreads();
  }
  *joined = true;
  const double mass_above = static_cast<double>(sum_above);
  uint32_t cut_key = 0, cut_index = 0xFFFFFFFFu;  // kept: above the key, or it up to that index
  if (nucleus) {
    if (listed > kMaxBand) return false;
    const double left = __builtin_ceil(goal - mass_above);
    if (!(left >= 1.0)) return false;  // the cut lies above the band
    const unsigned long long target = static_cast<unsigned long long>(left);
    // Finer bins of the band, the highest for its top; then the entries of the one bin by themselves.
    const float fine = static_cast<float>(kBins) / static_cast<float>(end - above);
    auto bin_of = [&](unsigned long long e) {
      const float x = (zmax - logit_of(static_cast<uint32_t>(e >> 32))) * per - static_cast<float>(above);
      return kBins - 1 - min(max(static_cast<int>(x * fine), 0), kBins - 1);
    };
    for (int b = tid; b < kBins; b += kThreads) digits[b] = 0;
    if (tid == 0) found->bin = kBins, s_n = 0;
    __syncthreads();
    for (int i = tid; i < listed; i += kThreads)
      atomicAdd(&digits[bin_of(band[i])], w.fixed(static_cast<uint32_t>(band[i] >> 32)));
    __syncthreads();
    const Found f = find_from_top(digits, target, waves, found);
    if (f.bin == kBins) return false;  // the cut lies below the band
    unsigned long long* weights = digits;
    for (int i = tid; i < listed; i += kThreads)
      if (bin_of(band[i]) == static_cast<int>(f.bin)) {
        const int slot = atomicAdd(&s_n, 1);
        if (slot < kMaxEqual) {
          order[slot] = band[i];
          weights[slot] = w.fixed(static_cast<uint32_t>(band[i] >> 32));
        }
      }
    __syncthreads();
    const int equal = s_n;
    if (equal > kMaxEqual) return false;
    if (tid < equal) {
      const unsigned long long mine = order[tid];
      unsigned long long sum = f.above;
      for (int j = 0; j < equal; ++j) sum += order[j] > mine ? weights[j] : 0;
      if (sum < target && target <= sum + weights[tid]) s_u64 = mine;
    }
    __syncthreads();
    cut_key = static_cast<uint32_t>(s_u64 >> 32);
    cut_index = 0xFFFFFFFFu - static_cast<uint32_t>(s_u64);
    __syncthreads();
  }
  for (int i = tid; i < min(listed, kMaxBand); i += kThreads) {
    const uint32_t key = static_cast<uint32_t>(band[i] >> 32);
    const uint32_t index = 0xFFFFFFFFu - static_cast<uint32_t>(band[i]);
    if (key < cut_key || (key == cut_key && index > cut_index)) continue;
    if (w.real(key) >= floor_w || key == w.top)
      atomicAdd(&sub_sums[(static_cast<int>(index) + view.shift) / kSub >> group], w.fixed(key));
  }
  __syncthreads();
  // The sub-chunks (of `group` doublings) in which the draw lands; thread t has 4t .. 4t + 3.
  constexpr int kEach = kMaxSubs / kThreads;
  unsigned long long sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) sum += sub_sums[kEach * tid + j];
  const unsigned long long incl = block_inclusive<unsigned long long>(sum, waves);
  if (tid == kThreads - 1) s_u64 = incl;
  __syncthreads();
  const unsigned long long all = s_u64;
  unsigned long long want = static_cast<unsigned long long>(uniform_of(a, row) * static_cast<double>(all));
  if (want >= all) want = all - 1;
  __syncthreads();
  if (incl - sum <= want && want < incl) {
    unsigned long long before = incl - sum;
    int at = kEach * tid;
    while (want >= before + sub_sums[at]) before += sub_sums[at++];
    s_place = at;
    s_u64 = want - before;
  }
  __syncthreads();
  if (wave != 0) return true;
  unsigned long long left = s_u64;
  for (int place = (s_place << group) * kSub + lane; ; place += 64) {
    const uint32_t key = view.key(place);
    const uint32_t index = static_cast<uint32_t>(place - view.shift);
    unsigned long long v = 0;
    if (key > cut_key || (key != 0 && key == cut_key && index <= cut_index))
      if (w.real(key) >= floor_w || key == w.top) v = w.fixed(key);
    unsigned long long run = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const unsigned long long o = __shfl_up(run, d);
      if (lane >= d) run += o;
    }
    const unsigned long long hit = __ballot(run > left);
    if (hit) {
      const int l = __ffsll(hit) - 1;
      if (lane == l) a.tokens[row] = static_cast<int32_t>(index);
      return true;
    }
    left -= __shfl(run, 63);
    if (place - lane >= view.vocab + view.shift) return true;  // not reached: the sums are the same
  }
}

// left[0]: how many rows are left; left[1 ..]: which, in no order.  Where the grid has several workgroups
// for each, they take parts of it.
template <bool kF32>
__global__ __launch_bounds__(kThreads) void sample_rest_kernel(SampleArgs a, RowRest* rest,
                                                               const uint32_t* __restrict__ left,
                                                               unsigned long long* joins, int max_parts,
                                                               int num_subs) {
  __shared__ unsigned long long bins[kMaxSubs];
  __shared__ unsigned long long digits[kBins];
  __shared__ unsigned long long band[kMaxBand];
  __shared__ unsigned long long waves[kThreads / 64];
  __shared__ Found found;
  const uint32_t num_left = left[0];
  const uint32_t num_parts =
      num_left > kJoinRows ? 1 : min(static_cast<uint32_t>(max_parts), gridDim.x / max(num_left, 1u));
  const uint32_t slot = blockIdx.x / num_parts;
  if (slot >= num_left) return;  // block-uniform
  const int64_t row = left[1 + slot];
  const Asked asked(a, row);
  const RowView<kF32> view(a, row);
  const uint32_t top = rest[row].top;
  const Weights w{top, static_cast<double>(logit_of(top)), asked.rate(),
                  static_cast<double>(1ull << rest[row].unit_bits)};
  unsigned long long* join = joins + static_cast<int64_t>(slot) * (kMaxBand + kMaxSubs);
  const Parts parts{static_cast<int>(num_parts), static_cast<int>(blockIdx.x - slot * num_parts), rest + row, join,
                    join + kMaxBand};
  // What sample_wide finds before its parts join is the same in all of them.
  const bool wide = asked.k == 0 && top != kInfKey;
  bool joined = false;
  if (wide && sample_wide<kF32>(a, row, view, asked, w, rest[row].total, num_subs, parts, bins, digits, band,
                                waves, &found, &joined))
    return;
  if (!joined && parts.mine != 0) return;
  sample_descent<kF32>(a, row, view, asked, w, num_subs, bins, reinterpret_cast<uint32_t*>(digits), waves, &found);
}

// The first thread by number whose condition holds, or else the last whose `or_else` does.
__device__ __forceinline__ int first_thread(bool holds, bool or_else, int* first, int* last) {
  if (threadIdx.x == 0) *first = 0x7FFFFFFF, *last = -1;
  __syncthreads();
  if (holds) atomicMin(first, static_cast<int>(threadIdx.x));
  if (or_else) atomicMax(last, static_cast<int>(threadIdx.x));
  __syncthreads();
  const int f = *first, l = *last;
  __syncthreads();
  return f != 0x7FFFFFFF ? f : l;
}

// One workgroup a row.  PER: sub-chunks a thread looks at.
// A chain of short steps, each behind a barrier, and of two reads of memory: for one row of 2^18 f32 logits
// under a top-k of 64 and a top-p the largest keys take 2.2 us, a threshold 3.5, listing and reading the
// candidates 4.4, the three histograms of them 6.  512 threads; a row of which 1,024 sub-chunks are read takes
// about 16 us more.  With 33 sub-chunks a thread (vocabularies past 294,905) up to 324 B a lane lie in scratch
// memory: a call for one row of 294,000 | 295,500 takes 21.4 | 26.3 us as above, 24.2 | 37.6 under a top-p alone.
template <bool kF32, int PER>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(
    SampleArgs a, const uint32_t* __restrict__ subs, const double* __restrict__ sums,
    RowRest* __restrict__ rest, uint32_t* left, int num_subs) {
  constexpr int kWaves = kPickThreads / 64;
  constexpr int kPickBins = 2 * kPickThreads;
  constexpr int kEach = kMaxTaken / kPickThreads;  // entries of a thread
  __shared__ unsigned long long cand[kMaxTaken];
  __shared__ uint32_t list[kMaxTaken];
  __shared__ Crossing<kPickThreads, kEach> crossing;
  __shared__ uint32_t bins[kPickBins];
  __shared__ unsigned long long waves[kWaves];
  __shared__ unsigned long long s_counts[2][kWaves];
  __shared__ int s_num, s_at, s_last;
  __shared__ uint32_t s_key;
  __shared__ double s_sum;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const Asked asked(a, row);
  const double u = uniform_of(a, row);
  const RowView<kF32> view(a, row);

  // Thread t has sub-chunks PER t .. PER t + PER - 1.
  uint32_t sub[PER];
  uint32_t top = 0, low = 0xFFFFFFFFu;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int s = PER * tid + j;
    sub[j] = s < num_subs ? subs[row * num_subs + s] : 0;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    top = max(top, sub[j]);
    low = min(low, sub[j] - 1);  // key 0, no logit, passes for the largest
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    top = max(top, static_cast<uint32_t>(__shfl_xor(top, d)));
    low = min(low, static_cast<uint32_t>(__shfl_xor(low, d)));
  }
  if (lane == 0) s_counts[0][wave] = (static_cast<unsigned long long>(low) << 32) | top;
  for (int i = tid; i < kPickBins; i += kPickThreads) bins[i] = 0;
  if (tid == 0) s_at = 0x7FFFFFFF;
  __syncthreads();
  const unsigned long long both = s_counts[0][lane % kWaves];
  top = static_cast<uint32_t>(both), low = static_cast<uint32_t>(both >> 32);
#pragma unroll
  for (int d = 1; d < kWaves; d *= 2) {
    top = max(top, static_cast<uint32_t>(__shfl_xor(top, d)));
    low = min(low, static_cast<uint32_t>(__shfl_xor(low, d)));
  }
  low += 1;
  if (top == 0 || asked.k == 1) {  // block-uniform
    // The first of the largest logits: the first sub-chunk that has it.
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j)
      if (sub[j] == top) at = PER * tid + j;
    if (top != 0 && at != 0x7FFFFFFF) atomicMin(&s_at, at);
    __syncthreads();
    if (wave == 0) {
      const unsigned long long m = top ? __ballot(view.key(s_at * kSub + lane) == top) : 0;
      if (lane == 0) a.tokens[row] = top ? s_at * kSub + __ffsll(m) - 1 - view.shift : -1;
    }
    return;
  }
  const Weights w{top, static_cast<double>(logit_of(top)), asked.rate(), 0x1p51};
  double mass[PER];
  double my_mass = 0.0, mass_incl = 0.0, total = 0.0;
  if (asked.needs_sums()) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int s = PER * tid + j;
      mass[j] = sub[j] ? sums[row * num_subs + s] : 0.0;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      mass[j] = sub[j] ? mass[j] * w.real(sub[j]) : 0.0;
      my_mass += mass[j];
    }
    mass_incl = block_inclusive<double>(my_mass, reinterpret_cast<double*>(waves));
    if (tid == kPickThreads - 1) s_sum = mass_incl;
    __syncthreads();
    total = s_sum;
    __syncthreads();
  }

  if (asked.k == 0 && asked.top_p == 1.0f && asked.min_p == 0.0f) {
    // Sums of different threads are added in different orders, so that by rounding none may pass
    // the goal: then the last with any weight has it.
    const double goal = u * total;
    if (tid == first_thread(my_mass > 0.0 && mass_incl > goal, my_mass > 0.0, &s_at, &s_last)) {
      int at = -1;
      double before = mass_incl - my_mass, at_before = 0.0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (mass[j] > 0.0 && (at < 0 || goal >= before)) at = PER * tid + j, at_before = before;
        before += mass[j];
      }
      s_num = at;
      s_sum = goal - at_before;
    }
    __syncthreads();
    if (wave != 0) return;
    const int place = s_num * kSub + lane;
    const uint32_t key = view.key(place);
    const double v = key ? w.real(key) : 0.0;
    double sum = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const unsigned long long hit = __ballot(v > 0.0 && sum > s_sum);
    const unsigned long long any = __ballot(v > 0.0);
    const int l = hit ? __ffsll(hit) - 1 : 63 - __clzll(any);
    if (lane == 0) a.tokens[row] = s_num * kSub + l - view.shift;
    return;
  }

  bool leaves = asked.k > kMaxK;  // to the third launch; block-uniform
  const float zmax = logit_of(top), zlow = logit_of(low);
  const double floor_w = static_cast<double>(asked.min_p);
  const bool by_floor = asked.k == 0 && asked.top_p == 1.0f;

  // The sub-chunks' largest in bins of equal width, from the top.
  const float per = static_cast<float>(kPickBins - 1) / (zmax - zlow);
  const bool binned = per > 0.0f && per < 1e30f;
  auto bin_of = [&](uint32_t key) {
    return binned ? min(static_cast<int>((zmax - logit_of(key)) * per), kPickBins - 1) : 0;
  };
  if (!by_floor && !leaves) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (sub[j]) atomicAdd(&bins[bin_of(sub[j])], 1u);
    __syncthreads();
  }

  int want = asked.k > 0 ? static_cast<int>(asked.k) : 128;
  // Thread t has the candidates t, t + kPickThreads, ..: (key, lowest index first), weight.
  unsigned long long entry[kEach], weight[kEach];
  while (!leaves) {
    // A key t0 with `want` sub-chunks or more at or above it, and not many more; 1 (every token that
    // can be drawn) if there are not as many.
    uint32_t t0 = 1;
    if (by_floor) {
      // Weights below min_p are below this by more than rounding.
      const double depth = -log2(floor_w) / w.rate;
      const float z = static_cast<float>(w.zmax - depth - 1e-5 * (__builtin_fabs(w.zmax) + depth));
      t0 = min(max(key_of(z), 1u), top);
    } else if (num_subs * kSub > kMaxTaken) {
      const int b0 = static_cast<int>(bins[2 * tid]), b1 = static_cast<int>(bins[2 * tid + 1]);
      const int incl = block_inclusive<int>(b0 + b1, reinterpret_cast<int*>(waves));
      if (tid == 0) s_at = -1, s_key = 0xFFFFFFFFu;
      __syncthreads();
      if (incl - b0 - b1 < want && want <= incl) {
        const bool first = incl - b1 >= want;
        s_at = 2 * tid + !first;
        s_num = first ? incl - b1 : incl;
      }
      __syncthreads();
      const int bin = s_at, count = s_num;
      if (bin >= 0) {
        if (count <= min(2 * want + 64, 1536)) {
          uint32_t least = 0xFFFFFFFFu;
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (sub[j] && bin_of(sub[j]) <= bin) least = min(least, sub[j]);
#pragma unroll
          for (int d = 1; d < 64; d *= 2) least = min(least, static_cast<uint32_t>(__shfl_xor(least, d)));
          if (lane == 0) atomicMin(&s_key, least);
          __syncthreads();
          t0 = s_key;
        } else {
          // Too many of one bin (a few logits far below or above the rest, or equal ones): bisection.
          uint32_t lo = 1, hi = top;  // at least want at lo
          int round = 0;
          const int enough = want + want / 4 + 16;
          while (lo < hi) {
            const uint32_t span = hi - lo;  // thresholds in (lo, hi]
            const uint32_t t[3] = {lo + max(span / 4, 1u), lo + max(span / 2, 1u), lo + span - span / 4};
            unsigned long long c = 0;  // three counts of 21 bits
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
              for (int j = 0; j < PER; ++j)
                c += static_cast<unsigned long long>(__popcll(__ballot(sub[j] >= t[i]))) << (21 * i);
            if (lane == 0) s_counts[round & 1][wave] = c;
            __syncthreads();
            c = s_counts[round & 1][lane % kWaves];
#pragma unroll
            for (int d = 1; d < kWaves; d *= 2) c += __shfl_xor(c, d);
            ++round;
            int at = -1, n_at = 0;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
              const int ci = static_cast<int>(c >> (21 * i)) & 0x1FFFFF;
              if (ci >= want) at = i, n_at = ci;
            }
            if (at < 2) hi = t[at + 1] - 1;
            if (at >= 0) lo = t[at];
            if (at >= 0 && n_at <= enough) break;
          }
          t0 = lo;
        }
      }
    }
    // Sub-chunks with candidates, then the candidates: (key, lowest index first) as one number.
    __syncthreads();
    if (tid == 0) s_num = 0, s_last = 0;
    __syncthreads();
    int my_subs = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) my_subs += sub[j] >= t0;
    if (__any(my_subs != 0)) {
      const int incl = wave_inclusive(my_subs);
      int base = 0;
      if (lane == 63) base = atomicAdd(&s_num, incl);
      int at = __shfl(base, 63) + incl - my_subs;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (sub[j] >= t0) {
          if (at < kMaxTaken) list[at] = PER * tid + j;
          ++at;
        }
    }
    __syncthreads();
    const int lists = s_num;
    bool fits = lists <= kMaxTaken;
    if (fits) {
      // A load of 16 bytes a lane takes kGroup sub-chunks.
      constexpr int kPer = RowView<kF32>::kPer, kLanes = kSub / kPer, kGroup = 64 / kLanes;
      constexpr int kAhead = kF32 ? 8 : 4;
      for (int i0 = wave * kGroup; i0 < lists; i0 += kAhead * kWaves * kGroup) {
        uint4 raw[kAhead];
        int at[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int l = i0 + i * kWaves * kGroup + lane / kLanes;
          at[i] = l < lists ? static_cast<int>(list[l]) * kSub + lane % kLanes * kPer : -kPer - 16;
          raw[i] = view.raw(at[i]);
        }
        uint32_t key[kAhead][kPer];
        int found = 0;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          float z[kPer];
          RowView<kF32>::unpack(raw[i], z);
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            key[i][j] = key_of(z[j]);
            found += key[i][j] >= t0;
          }
        }
        const int incl = wave_inclusive(found);
        int base = 0;
        if (lane == 63) base = atomicAdd(&s_last, incl);
        int slot = __shfl(base, 63) + incl - found;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (key[i][j] >= t0) {
              if (slot < kMaxTaken)
                cand[slot] = (static_cast<unsigned long long>(key[i][j]) << 32) |
                             (0xFFFFFFFFu - static_cast<uint32_t>(at[i] + j - view.shift));
              ++slot;
            }
      }
      __syncthreads();
      fits = s_last <= kMaxTaken;
    }
    if (!fits) {  // block-uniform
      leaves = true;
      break;
    }
    const int n = s_last;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = tid + kPickThreads * j;
      entry[j] = i < n ? cand[i] : 0;
    }
    // Bins of the candidates' logits, from the largest down to t0.  Without a t0, where every token of a vocabulary of
    // up to 2,048 is one, down to the smallest, or bins of the keys if that lies far below (a mask of the type's
    // lowest value): the entries of a bin are compared with each other, and 1,000 of them in one bin took 150 us.
    uint32_t bottom = t0;
    if (t0 == 1) {  // block-uniform
      bottom = top;
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (entry[j]) bottom = min(bottom, static_cast<uint32_t>(entry[j] >> 32));
      if (tid == 0) s_key = top;
      __syncthreads();
      atomicMin(&s_key, bottom);
      __syncthreads();
      bottom = s_key;
    }
    const float range = zmax - logit_of(bottom), per_logit = static_cast<float>(kPickBins - 1) / range;
    const bool linear = per_logit > 0.0f && per_logit < 1e30f && (t0 > 1 || range * w.rate < 256.0);
    const int key_shift = max(0, 22 - __builtin_clz((top - bottom) | 1u));  // to 1,024 bins
    auto entry_bin = [&](int j) {
      const uint32_t key = static_cast<uint32_t>(entry[j] >> 32);
      return linear ? min(static_cast<int>((zmax - logit_of(key)) * per_logit), kPickBins - 1)
                    : static_cast<int>((top - key) >> key_shift);
    };
    auto keep_from = [&](unsigned long long cut) {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (entry[j] < cut) entry[j] = 0, weight[j] = 0;
    };
    if (asked.k > 0 && n > asked.k) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) weight[j] = entry[j] != 0;
      keep_from(crossing.find(entry, weight, entry_bin, [&](unsigned long long) {
        return static_cast<unsigned long long>(asked.k);
      }));
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) weight[j] = entry[j] ? w.fixed(static_cast<uint32_t>(entry[j] >> 32)) : 0;
    if (by_floor || asked.top_p == 1.0f) break;
    bool below = false, guess = false;
    const unsigned long long cut = crossing.find(entry, weight, entry_bin, [&](unsigned long long listed) {
      const double all = asked.k > 0 ? static_cast<double>(listed) : total * w.unit;
      const double goal = __builtin_ceil(static_cast<double>(asked.top_p) * all);
      const double have = static_cast<double>(listed);
      if (asked.k == 0 && t0 > 1 && have < goal) {  // the cut lies below t0
        below = true;
        // The next ones' weights, if they fell as 1 / rank up to ten times as many, would not do
        // either: only a guess at what is faster.
        guess = have + 2.3 * n * w.real(t0) * w.unit < goal;
        return 0ull;
      }
      if (goal >= have) return 0ull;  // all of them
      return goal < 1.0 ? 1ull : static_cast<unsigned long long>(goal);
    });
    if (below) {
      leaves = want == kMaxK || guess;
      want = kMaxK;
      __syncthreads();
      continue;
    }
    keep_from(cut);
    break;
  }
  if (leaves) {
    double most = total;  // the sum of the row's weights, or what it cannot pass
    if (!asked.needs_sums()) {
      double mine = 0.0;  // (read again: a rolled loop over them needs no registers)
#pragma unroll 2
      for (int s = tid; s < num_subs; s += kPickThreads) {
        const uint32_t key = subs[row * num_subs + s];
        mine += key ? kSub * w.real(key) : 0.0;
      }
      most = block_inclusive<double>(mine, reinterpret_cast<double*>(waves));
    }
    if (tid == kPickThreads - 1) {
      rest[row] = {total, top, unit_bits(most), 0, 0, 0};
      left[1 + atomicAdd(&left[0], 1u)] = static_cast<uint32_t>(row);
    }
    return;
  }
  if (asked.min_p > 0.0f) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint32_t key = static_cast<uint32_t>(entry[j] >> 32);
      if (entry[j] && !(w.real(key) >= floor_w || key == top)) weight[j] = 0;
    }
  }
  // The draw, by index.
  int by = 0;
  while ((view.vocab - 1) >> by >= kPickBins) ++by;
#pragma unroll
  for (int j = 0; j < kEach; ++j) entry[j] &= 0xFFFFFFFFull;  // 2^32 - 1 - index
  __syncthreads();
  const unsigned long long drawn = crossing.find(
      entry, weight, [&](int j) { return static_cast<int>((0xFFFFFFFFu - static_cast<uint32_t>(entry[j])) >> by); },
      [&](unsigned long long listed) {  // the first whose sum passes u of all
        const unsigned long long goal = static_cast<unsigned long long>(u * static_cast<double>(listed));
        return min(goal, listed - 1) + 1;
      });
  if (tid == 0) a.tokens[row] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(drawn));
}

// Workgroups of the third launch: as many as rows, or the 256 CUs with up to eight a row, each of 64
// sub-chunks or more.  Of a batch few rows are left for it: 42 of 256 rows of 2^18 under a top-p of 0.95, which take
// 44 us in six parts each (the workgroups start and sample for 12, pass for 8, meet for 10 and cut and draw for 8)
// where a workgroup each took 75; and for one such row all three launches take 58 us where they took 102.
int64_t rest_parts(int64_t vocab) { return std::clamp<int64_t>(vocab / (64 * kSub), 1, 8); }
int64_t rest_blocks(int64_t rows, int64_t vocab) {
  return std::max(rows, std::min<int64_t>(rows * rest_parts(vocab), 256));
}

int64_t sub_chunks(int64_t vocab) { return (vocab + 7 + kSub - 1) / kSub; }

// Where the parts of a row meet.
int64_t join_longs(int64_t rows, int64_t vocab) {
  return rest_parts(vocab) > 1 ? std::min<int64_t>(rows, kJoinRows) * (kMaxBand + kMaxSubs) : 0;
}

template <bool kF32>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
  const int subs = static_cast<int>(sub_chunks(a.vocab));
  double* sums = static_cast<double*>(a.workspace);
  RowRest* rest = reinterpret_cast<RowRest*>(sums + a.rows * subs);
  const int parts = static_cast<int>(rest_parts(a.vocab));
  unsigned long long* joins = reinterpret_cast<unsigned long long*>(rest + a.rows);
  uint32_t* left = reinterpret_cast<uint32_t*>(joins + join_longs(a.rows, a.vocab));
  uint32_t* tops = left + 1 + a.rows;
  const int64_t blocks = sample_scan_blocks(a.rows, a.vocab, kF32);
  hipLaunchKernelGGL(sample_scan_kernel<kF32>, dim3(static_cast<unsigned>(blocks)), dim3(kScanThreads), 0, stream,
                     a, tops, sums, left, subs, static_cast<int>(blocks / a.rows));
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const dim3 grid(static_cast<unsigned>(a.rows));
  if (subs <= kPickThreads)
    hipLaunchKernelGGL((sample_pick_kernel<kF32, 1>), grid, dim3(kPickThreads), 0, stream, a, tops,
                       sums, rest, left, subs);
  else if (subs <= 9 * kPickThreads)
    hipLaunchKernelGGL((sample_pick_kernel<kF32, 9>), grid, dim3(kPickThreads), 0, stream, a, tops,
                       sums, rest, left, subs);
  else
    hipLaunchKernelGGL((sample_pick_kernel<kF32, 33>), grid, dim3(kPickThreads), 0, stream, a, tops,
                       sums, rest, left, subs);
  err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(sample_rest_kernel<kF32>, dim3(static_cast<unsigned>(rest_blocks(a.rows, a.vocab))),
                     dim3(kThreads), 0, stream, a, rest, left, joins, parts, subs);
  return hipGetLastError();
}

}  // namespace

int64_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
  return (rows * (sub_chunks(vocab) * 12 + static_cast<int64_t>(sizeof(RowRest)) + 4) + 4 +
          join_longs(rows, vocab) * 8 + 15) / 16 * 16;
}

// Each row has workgroups of its own, of 16 KiB of logits each.
int64_t sample_scan_blocks(int64_t rows, int64_t vocab, bool f32) {
  const int64_t chunk = kScanThreads * kScanVectors * (f32 ? RowView<true>::kPer : RowView<false>::kPer);
  return rows * ((sub_chunks(vocab) * kSub + chunk - 1) / chunk);
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  return a.f32 ? launch<true>(a, stream) : launch<false>(a, stream);
}

}  // namespace ifr
