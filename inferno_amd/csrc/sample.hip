// A token a row from its logits z, with temperature T, top-k, top-p, min-p and a given u:
//   w_i = exp((z_i - max z) / T)
//   K   = the first top_k tokens by (z descending, index ascending)
//   P   = the shortest prefix of K with sum w >= top_p * sum over K of w, one token at least
//   M   = { i in P : w_i >= min_p }
//   the token is the first i of M, by index, with sum over j <= i in M of w_j > u * sum over M of w
//
// A draw lands next to a border between two tokens as often as the sums are wrong there: with
// 2^18 tokens of equal weight f32 sums would give another token in 2 to 3 % of draws.
// The weights are f64 exponentials, taken as integers of 2^-shift (44 bits at 2^18 tokens) and
// added as 64-bit integers: the sums do not depend on their order.
//
// K and P are prefixes of the order by z, that is all keys above a key and the first few tokens of
// that key: the key is found 11, 11 and 10 bits at a time from histograms of counts or weights.
#include "common.hpp"
#include "step.hpp"

namespace ifr {
namespace {

constexpr int kThreads = 1024;
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

struct Weights {
  uint32_t top;  // the largest key
  double zmax, inv_t, unit;
  __device__ __forceinline__ double real(uint32_t key) const {
    if (key == top) return 1.0;
    const double a = (static_cast<double>(logit_of(key)) - zmax) * inv_t;
    return a > -745.0 ? exp(a) : 0.0;  // NaN (inf - inf, inf * 0): 0
  }
  __device__ __forceinline__ uint64_t fixed(uint32_t key) const {
    return static_cast<uint64_t>(__builtin_rint(real(key) * unit));
  }
};

template <typename T>
__device__ __forceinline__ T block_inclusive(T v, T* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
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

template <bool kF32>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a, int shift) {
  __shared__ unsigned long long bins[kMaxSubs];
  __shared__ uint32_t tie_counts[kMaxSubs];
  __shared__ unsigned long long waves[kThreads / 64];
  __shared__ Found found;
  __shared__ uint32_t s_top;
  const int64_t row = blockIdx.x;
  const int vocab = static_cast<int>(a.vocab);
  const void* z = static_cast<const char*>(a.logits) + row * a.row_stride * (kF32 ? 4 : 2);
  const int tid = threadIdx.x, lane = tid & 63;

  if (tid == 0) s_top = 0;
  __syncthreads();
  uint32_t top = 0;
  int valid = 0;
  for (int i = tid; i < vocab; i += kThreads) {
    const uint32_t k = key_of(load_logit<kF32>(z, i));
    top = max(top, k);
    valid += k != 0;
  }
  atomicMax(&s_top, top);
  unsigned long long count = block_inclusive<unsigned long long>(valid, waves);
  if (tid == kThreads - 1) found.above = count;
  __syncthreads();
  top = s_top;
  count = found.above;
  __syncthreads();
  if (count == 0) {  // block-uniform
    if (tid == 0) a.tokens[row] = -1;
    return;
  }

  const float t = a.temperature ? a.temperature[row] : 1.0f;
  int64_t k = a.top_k ? a.top_k[row] : 0;
  if (!(t > 0.0f)) k = 1;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  const float min_p = a.min_p ? a.min_p[row] : 0.0f;
  const Weights w{top, static_cast<double>(logit_of(top)), t > 0.0f ? 1.0 / static_cast<double>(t) : 1.0,
                  static_cast<double>(1ull << shift)};

  // Keys of `digit` bits at a time: the histogram of value(key) over the keys that
  // agree with `prefix` above the digit.
  Cut cut{1, count};  // key 1 stands for no logit: everything that can be drawn
  auto descend = [&](unsigned long long target, auto value) {
    uint32_t prefix = 0;
    unsigned long long above = 0;
    for (int level = 0; level < 3; ++level) {
      const int lo = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int width = level == 2 ? 10 : 11;
      for (int b = tid; b < kBins; b += kThreads) bins[b] = 0;
      __syncthreads();
      for (int i = tid; i < vocab; i += kThreads) {
        const uint32_t key = key_of(load_logit<kF32>(z, i));
        if (key == 0 || (level > 0 && (key >> (lo + width)) != prefix)) continue;
        const unsigned long long v = value(key);
        if (v) atomicAdd(&bins[(key >> lo) & ((1u << width) - 1)], v);
      }
      __syncthreads();
      const Found f = find_from_top(bins, target - above, waves, &found);
      above += f.above;
      prefix = (prefix << width) | f.bin;
      __syncthreads();
    }
    return Found{prefix, above};
  };
  if (k > 0 && static_cast<unsigned long long>(k) < count) {
    const Found f = descend(static_cast<unsigned long long>(k),
                            [](uint32_t) -> unsigned long long { return 1; });
    cut = {f.bin, static_cast<unsigned long long>(k) - f.above};
  }
  // The kept ties of the top-k cut, all of one weight, count as one sum behind the rest.
  if (top_p < 1.0f) {
    const unsigned long long tie = w.fixed(cut.key);
    auto value = [&](uint32_t key) -> unsigned long long {
      return key > cut.key ? w.fixed(key) : 0;
    };
    unsigned long long mine = 0;
    for (int i = tid; i < vocab; i += kThreads) {
      const uint32_t key = key_of(load_logit<kF32>(z, i));
      if (key) mine += value(key);
    }
    mine = block_inclusive<unsigned long long>(mine, waves);
    if (tid == kThreads - 1) found.above = mine;
    __syncthreads();
    const unsigned long long strict = found.above;
    __syncthreads();
    const unsigned long long total = strict + cut.ties * tie;
    const double p = top_p > 0.0f ? static_cast<double>(top_p) : 0.0;  // NaN: off, by the test above
    const double want = __builtin_ceil(p * static_cast<double>(total));
    unsigned long long target = want < 1.0 ? 1 : static_cast<unsigned long long>(want);
    target = target < total ? target : total;
    if (target > strict) {  // within the ties of the top-k cut
      cut.ties = (target - strict + tie - 1) / tie;
    } else {
      const Found f = descend(target, value);
      const unsigned long long each = w.fixed(f.bin);
      cut = {f.bin, (target - f.above + each - 1) / each};
    }
  }

  // By index: the weight and the ties of each sub-chunk of 2^sub tokens.
  int sub = 8;
  while (((vocab - 1) >> sub) + 1 > kMaxSubs) ++sub;
  const int subs = ((vocab - 1) >> sub) + 1;
  const double floor_w = min_p > 0.0f ? static_cast<double>(min_p) : 0.0;
  auto kept = [&](uint32_t key) -> unsigned long long {
    if (key == 0) return 0;
    const double v = w.real(key);
    return v >= floor_w || key == top ? static_cast<unsigned long long>(__builtin_rint(v * w.unit)) : 0;
  };
  const unsigned long long tie = kept(cut.key);
  for (int s = tid; s < kMaxSubs; s += kThreads)
    if (s >= subs) {
      bins[s] = 0;
      tie_counts[s] = 0;
    }
  for (int s = tid >> 6; s < subs; s += kThreads / 64) {
    unsigned long long sum = 0;
    uint32_t ties = 0;
    const int end = min(vocab, (s + 1) << sub);
    for (int i = (s << sub) + lane; i < end; i += 64) {
      const uint32_t key = key_of(load_logit<kF32>(z, i));
      if (key > cut.key) sum += kept(key);
      ties += key == cut.key;
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
      sum += __shfl_xor(sum, d);
      ties += __shfl_xor(ties, d);
    }
    if (lane == 0) {
      bins[s] = sum;
      tie_counts[s] = ties;
    }
  }
  __syncthreads();
  // Thread t has sub-chunks 4t .. 4t + 3.
  constexpr int kPer = kMaxSubs / kThreads;
  unsigned long long ties = 0, sum = 0;
  for (int j = 0; j < kPer; ++j) ties += tie_counts[kPer * tid + j];
  unsigned long long ties_before = block_inclusive<unsigned long long>(ties, waves) - ties;
  unsigned long long first_ties = ties_before;
  for (int j = 0; j < kPer; ++j) {
    const int s = kPer * tid + j;
    const unsigned long long left = first_ties < cut.ties ? cut.ties - first_ties : 0;
    const unsigned long long here = tie_counts[s] < left ? tie_counts[s] : left;
    first_ties += tie_counts[s];
    bins[s] += here * tie;
    sum += bins[s];
  }
  const unsigned long long incl = block_inclusive<unsigned long long>(sum, waves);
  if (tid == kThreads - 1) found.above = incl;
  __syncthreads();
  const unsigned long long total = found.above;
  __syncthreads();
  const float u = a.uniform[row];
  const double ud = u > 0.0f ? (u < 1.0f ? static_cast<double>(u) : 1.0 - 0x1p-24) : 0.0;
  unsigned long long goal = static_cast<unsigned long long>(ud * static_cast<double>(total));
  if (goal >= total) goal = total - 1;  // total >= 1: the largest logit is kept
  __shared__ int s_sub;
  __shared__ unsigned long long s_before, s_ties;
  if (incl - sum <= goal && goal < incl) {
    unsigned long long before = incl - sum;
    unsigned long long ties_at = ties_before;
    for (int j = 0; j < kPer; ++j) {
      const int s = kPer * tid + j;
      if (goal < before + bins[s]) {
        s_sub = s;
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
  const int end = min(vocab, (s_sub + 1) << sub);
  for (int i0 = s_sub << sub; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const uint32_t key = i < end ? key_of(load_logit<kF32>(z, i)) : 0;
    const unsigned long long is_tie = __ballot(key == cut.key && key != 0);
    const unsigned long long order =
        ties_at + __popcll(is_tie & ((1ull << lane) - 1));
    unsigned long long v = key > cut.key ? kept(key) : key == cut.key && order < cut.ties ? tie : 0;
    if (key == 0) v = 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const unsigned long long o = __shfl_up(v, d);
      if (lane >= d) v += o;
    }
    const unsigned long long hit = __ballot(before + v > goal);
    if (hit) {
      if (lane == 0) a.tokens[row] = i0 + static_cast<int>(__ffsll(hit)) - 1;
      return;
    }
    before += __shfl(v, 63);
    ties_at += __popcll(is_tie);
  }
}

// Bits of the integers that stand for weights of at most 1: sums of a row stay below 2^63.
int weight_shift(int64_t vocab) {
  int bits = 0;
  while ((int64_t{1} << bits) < vocab) ++bits;
  return bits < 10 ? 52 : 62 - bits;
}

}  // namespace

int64_t sample_workspace_bytes(int64_t, int64_t) { return 0; }

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  const int shift = weight_shift(a.vocab);
  if (a.f32)
    hipLaunchKernelGGL(sample_row_kernel<true>, dim3(static_cast<unsigned>(a.rows)),
                       dim3(kThreads), 0, stream, a, shift);
  else
    hipLaunchKernelGGL(sample_row_kernel<false>, dim3(static_cast<unsigned>(a.rows)),
                       dim3(kThreads), 0, stream, a, shift);
  return hipGetLastError();
}

}  // namespace ifr
