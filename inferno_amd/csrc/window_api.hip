// Planning and entry points of the attention with a window and sinks and of the 8-bit
// block-scaled cache (declared in include/inferno_hip.h).
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <array>
#include <functional>
#include <new>
#include <queue>
#include <utility>
#include <vector>

#include "../../include/inferno_hip.h"
#include "common.hpp"
#include "launch.hpp"
#include "window.hpp"

namespace ifr {
int32_t abi_fail(int32_t code, const char* msg);  // api.hip
int32_t abi_ok();
}  // namespace ifr

namespace {

using namespace ifr::window;

int32_t fail(int32_t code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return ifr::abi_fail(code, buf);
}

bool is_pow2(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
int64_t shift_of(int64_t pow2) {
  int64_t s = 0;
  while ((int64_t{1} << s) < pow2) ++s;
  return s;
}

// Words of info beyond those that every plan has (include/inferno_hip.h).
enum Info : int {
  kInItems = 0,
  kInUnits = 1,
  kInMode = 2,
  kInCols = 3,
  kInBytes = 4,
  kInSeq = 5,
  kInRuns = 6,
  kInShift = 7,
  kInRowMask = 8,
  kInPageMask = 9,
  kInCacheRows = 10,
  kInKind = 11,
  kInWindow = 12,
  kInMaxPos = 13,
  kInPrompts = 14,
  kInWrites = 15,
  kInSinks = 16,
  kInNumQ = 17,
  kInNumKv = 18,
  kInHeadDim = 19,
  kInBlock = 20,
  kInWorkspace = 21,
  kInOffPrompts = 22,
  kInOffWrites = 23,
  kInOffUnits = 24,
  kInHeadsPerGroup = 25,
  kInSharedWrites = 26,
};
static_assert(kInSharedWrites < IFR_WINDOW_INFO_LEN, "info holds every word");

// The work of a step in row items and prompt blocks.
//
// Row items take 16 columns, a (token, q head) each, and the cache at the rate that HBM
// gives it; prompt blocks take 8 to 32 times the columns and the cache through LDS.  A run
// of few columns would leave most of a prompt block idle, and one of many would have row items
// read the cache once for each 16 of them.  Runs of up to kRowItemCols columns are row items
// always, runs of up to kRowItemMost if what all of those read stays below kRowItemBytes: so a run
// of 33 to 128 columns has weights of two bf16 parts or of one by what else is in the step.
// Measured as row items and as prompt blocks, on 4,096 positions of an e4m3 cache (us):
//   head_dim 256, 8 kv heads, 1 run:   32 columns 20 and 37, 64 columns 28 and 38, 128 columns 30 and 39
//   the same, 16 runs:                 32 columns 111 and 162, 64 columns (1.1 GB) 195 and 165
//   head_dim 128, 4 kv heads, 16 runs: 32 columns 35 and 93, 64 columns (270 MB) 60 and 94, 128 (550 MB) 105 and 95
constexpr int64_t kRowItemCols = 32, kRowItemMost = 128;
constexpr int64_t kRowItemBytes = int64_t{400} << 20;
// Workgroups that run at once, of row items: two of four waves on each of 256 CUs, at
// head_dim 512 one; of prompt blocks: one of eight waves.
constexpr int64_t resident_groups(int64_t head_dim) { return head_dim == 512 ? 256 : 512; }
constexpr int64_t kPromptGroups = 256;
constexpr int64_t kBlockTiles = 3, kPieceTiles = 7;  // what a prompt block, and a piece of one, costs besides its tiles
constexpr int64_t kLeastPiece = 4;                   // tiles
constexpr int64_t kItemTiles = 4;                    // what a row item costs besides a wave's tiles
constexpr int64_t kMergePieces = 8;                  // pieces of a token whose merging costs as much as a tile
constexpr int64_t kMaxRounds = 4;
// Pieces at most that splits make: of row items all rounds, of prompt blocks two a CU more than there are.
constexpr int64_t kSplitPieces = kMaxRounds * resident_groups(256) + 2 * kPromptGroups;

constexpr int64_t kMostTokens = int64_t{1} << 24, kMostRows = INT32_MAX / 4;  // of a step, and of its run table

struct Work {
  std::array<int32_t, kWorkWords> words;
  int64_t len() const { return words[kItHi] - words[kItLo]; }
};

struct Builder {
  int64_t num_kv, gqa, window, sinks;
  std::vector<Work> items, prompts;
  std::vector<std::array<int32_t, kMergeWords>> units;
  int64_t cols = 0;

  int64_t tiles(int64_t p0, int64_t ntok) const {
    const Span s = visible_span(static_cast<int>(p0), static_cast<int>(window), static_cast<int>(sinks));
    return s.n_sink + (p0 + ntok - 1) / kTileKeys - s.first + 1;
  }
  // Splits the tiles of one set of tokens into n items of `width` columns a kv head.
  void put(std::vector<Work>& to, int64_t t0, int64_t ntok, int64_t rows_off, int64_t p0, int64_t n, int64_t width) {
    const int64_t all = tiles(p0, ntok);
    const int64_t step = width * num_kv;
    for (int64_t s = 0; s < n; ++s) {
      Work w{};
      w.words[kItT0] = static_cast<int32_t>(t0);
      w.words[kItTokens] = static_cast<int32_t>(ntok);
      w.words[kItRows] = static_cast<int32_t>(rows_off);
      w.words[kItPos] = static_cast<int32_t>(p0);
      w.words[kItLo] = static_cast<int32_t>(all * s / n);
      w.words[kItHi] = static_cast<int32_t>(all * (s + 1) / n);
      w.words[kItCol] = n > 1 ? static_cast<int32_t>(cols + s * step) : -1;
      to.push_back(w);
    }
    if (n == 1) return;
    for (int64_t t = 0; t < ntok; ++t) {
      std::array<int32_t, kMergeWords> u{};
      u[kUnToken] = static_cast<int32_t>(t0 + t);
      u[kUnCount] = static_cast<int32_t>(n);
      u[kUnCol] = static_cast<int32_t>(cols + t * gqa);
      u[kUnStep] = static_cast<int32_t>(step);
      u[kUnHstep] = static_cast<int32_t>(width);
      units.push_back(u);
    }
    cols += n * step;
  }
};

struct Part {
  int64_t run, t0, ntok, p0, tiles;
};

// How many pieces each prompt block's tiles are split into.  One workgroup of prompt blocks
// fits a CU, so what counts is the longest sum of pieces that one CU gets: 256 workgroups
// of n tiles take as long as n tiles, 257 twice that.  Splits that bring the pieces up to one
// or two workgroups a CU are compared with none, at their lengths and what a piece costs
// besides (its start, and where it is split its sums in memory and their merging).
std::vector<int64_t> prompt_splits(const std::vector<Part>& parts, int64_t num_kv) {
  const std::vector<int64_t> whole(parts.size(), 1);
  std::vector<int64_t> best = whole;
  const int64_t want = static_cast<int64_t>(parts.size()) * num_kv;
  if (parts.empty() || want >= 2 * kPromptGroups) return best;
  auto makespan = [&](const std::vector<int64_t>& n) {
    std::vector<int64_t> pieces;
    for (size_t i = 0; i < parts.size(); ++i)
      for (int64_t s = 0; s < n[i]; ++s)
        pieces.push_back(parts[i].tiles * (s + 1) / n[i] - parts[i].tiles * s / n[i] + (n[i] > 1 ? kPieceTiles : kBlockTiles));
    std::sort(pieces.begin(), pieces.end(), std::greater<int64_t>());
    std::priority_queue<int64_t, std::vector<int64_t>, std::greater<int64_t>> cus;
    for (int64_t i = 0; i < kPromptGroups; ++i) cus.push(0);
    int64_t end = 0;
    for (int64_t piece : pieces)
      for (int64_t h = 0; h < num_kv; ++h) {
        const int64_t t = cus.top() + piece;
        cus.pop();
        cus.push(t);
        end = std::max(end, t);
      }
    return end;
  };
  int64_t least = makespan(best);
  for (int64_t most : {kPromptGroups, 2 * kPromptGroups}) {
    std::vector<int64_t> n = whole;
    std::priority_queue<std::pair<int64_t, int64_t>> longest;  // piece, and the smaller index first
    for (size_t i = 0; i < parts.size(); ++i) longest.push({parts[i].tiles, -static_cast<int64_t>(i)});
    for (int64_t total = want; total + num_kv <= most; total += num_kv) {
      const auto [len, i] = longest.top();
      if (len < 2 * kLeastPiece) break;
      longest.pop();
      if (++n[-i] < kMaxStripes) longest.push({ceil_div(parts[-i].tiles, n[-i]), i});
      if (longest.empty()) break;
    }
    const int64_t t = makespan(n);
    if (t < least) {
      least = t;
      best = n;
    }
  }
  return best;
}

// Tiles of a row item at most.  Workgroups run `slots` at a time, so the time is about the rounds
// that they come to times an item's tiles (a wave's share of them) and what it costs besides, and
// the merging of the most pieces that a token has.  For each number of rounds the shortest items
// that keep to it are tried, and such of twice and four times the tiles.
int64_t row_chunk(const std::vector<Part>& parts, int64_t heads, int64_t subs, int64_t slots) {
  int64_t longest = subs;
  for (const Part& p : parts) longest = std::max(longest, p.tiles);
  auto rounds = [&](int64_t chunk) {
    int64_t n = 0;
    for (const Part& p : parts) n += std::min<int64_t>(ceil_div(p.tiles, chunk), kMaxStripes);
    return ceil_div(n * heads, slots);
  };
  int64_t best = longest, least = INT64_MAX;
  for (int64_t r = 1; r <= kMaxRounds; ++r) {
    int64_t lo = subs, hi = longest;  // the shortest chunk of r rounds, if there is one
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (rounds(mid) <= r) hi = mid;
      else lo = mid + 1;
    }
    if (rounds(lo) > r) continue;
    for (int64_t chunk = lo; chunk <= 4 * lo; chunk *= 2) {
      const int64_t pieces = ceil_div(longest, chunk);
      const int64_t cost = rounds(chunk) * (ceil_div(chunk, subs) + kItemTiles) + (pieces > 1 ? 1 + pieces / kMergePieces : 0);
      if (cost < least) {
        least = cost;
        best = chunk;
      }
    }
    if (lo == subs) break;  // no shorter items
  }
  return best;
}

// Longest first: workgroups start in order as earlier ones end.
void longest_first(std::vector<Work>& v) {
  std::stable_sort(v.begin(), v.end(), [](const Work& a, const Work& b) { return a.len() > b.len(); });
}

int64_t most_words(int64_t num_runs, int64_t num_rows, int64_t seq_len, int64_t block_len) {
  // A part a token at most; splits add kSplitPieces (with one kv head).
  const int64_t items = std::min(seq_len * kMaxStripes, seq_len + kSplitPieces);
  const int64_t writes = block_len > 0 ? seq_len / block_len + 2 * num_runs + 1 : 0;
  return ifr::kHdrWords + kWorkWords * items + 4 * num_runs + num_rows + seq_len + kMergeWords * seq_len + kWriteBlockWords * writes;
}

int32_t check_shape(int64_t num_q, int64_t num_kv, int64_t head_dim) {
  if (num_q <= 0 || num_kv <= 0 || num_q % num_kv != 0)
    return fail(IFR_EINVAL, "num_q must be a positive multiple of num_kv");
  if (num_q / num_kv > kRowCols) return fail(IFR_EUNSUPPORTED, "more than %d q heads a kv head", kRowCols);
  if (num_q > 1024) return fail(IFR_EUNSUPPORTED, "num_q > 1024");
  if (head_dim != 128 && head_dim != 256 && head_dim != 512)
    return fail(IFR_EUNSUPPORTED, "head_dim %lld is not compiled (128, 256, 512)", (long long)head_dim);
  return IFR_OK;
}

int32_t plan(int32_t* img, int64_t img_words, const int32_t* runs, int64_t num_runs, const int32_t* base_rows,
             int64_t num_rows, int64_t seq_len, int64_t window, int64_t sinks, int64_t page_len, int64_t cache_rows,
             int64_t num_q, int64_t num_kv, int64_t head_dim, int64_t block_len, int64_t* info) {
  using namespace ifr;
  if (!img || !info) return fail(IFR_EINVAL, "null image or info");
  if (seq_len <= 0 || seq_len > kMostTokens) return fail(IFR_EINVAL, "seq_len must be in [1, 2^24]");
  if (num_runs <= 0 || num_runs > seq_len) return fail(IFR_EINVAL, "num_runs must be in [1, seq_len]");
  if (num_rows < 0 || num_rows > kMostRows) return fail(IFR_EINVAL, "num_rows out of range");
  if (!runs || !base_rows) return fail(IFR_EINVAL, "null run table");
  if (window < 0 || window > INT32_MAX / 4) return fail(IFR_EINVAL, "window must be in [0, 2^29)");
  if (sinks < 0 || sinks > INT32_MAX / 4) return fail(IFR_EINVAL, "sinks must be in [0, 2^29)");
  if (sinks > 0 && window == 0) return fail(IFR_EINVAL, "sinks need a window (window 0 sees every position)");
  if (!is_pow2(page_len) || page_len < kTileKeys || page_len > (1 << 24))
    return fail(IFR_EINVAL, "page_len %lld is not a power of two in [32, 2^24]", (long long)page_len);
  if (cache_rows <= 0 || cache_rows > INT32_MAX) return fail(IFR_EINVAL, "cache_rows must be in [1, 2^31)");
  if (int32_t st = check_shape(num_q, num_kv, head_dim)) return st;
  if (seq_len * num_q > INT32_MAX) return fail(IFR_EUNSUPPORTED, "more than 2^31 rows of q");
  if (block_len != 0 && (!is_pow2(block_len) || block_len < 16 || block_len > page_len))
    return fail(IFR_EINVAL, "block_len must be 0 (bf16) or a power of two in [16, page_len]");
  if (runs[0] != 0) return fail(IFR_EINVAL, "runs[0].buf_start must be 0");

  const int64_t shift = shift_of(page_len), row_mask = page_len - 1;
  int64_t max_pos = 0;
  for (int64_t i = 0; i < num_runs; ++i) {
    const int64_t start = runs[4 * i], base = runs[4 * i + 1], off = runs[4 * i + 2], pages = runs[4 * i + 3];
    const int64_t next = i + 1 < num_runs ? runs[4 * (i + 1)] : seq_len;
    if (start < 0 || next > seq_len || next <= start)
      return fail(IFR_EINVAL, "run %lld holds no token or is out of order (buf_start %lld, next run at %lld)", (long long)i,
                  (long long)start, (long long)next);
    if (base < 0) return fail(IFR_EINVAL, "run %lld: negative base_pos", (long long)i);
    const int64_t last = base + next - start - 1;
    if (last > INT32_MAX / 4) return fail(IFR_EINVAL, "run %lld: position overflow", (long long)i);
    if (off < 0 || pages < 0 || off + pages > num_rows)
      return fail(IFR_EINVAL, "run %lld: rows [%lld, +%lld) outside base_rows[%lld]", (long long)i, (long long)off,
                  (long long)pages, (long long)num_rows);
    if ((last >> shift) >= pages)
      return fail(IFR_EINVAL, "run %lld needs %lld pages, has %lld", (long long)i, (long long)((last >> shift) + 1),
                  (long long)pages);
    max_pos = std::max(max_pos, last);
    // Pages that the kernels read: those with a position that some query sees.  The
    // others may be anything.
    auto check_page = [&](int64_t j) -> int32_t {
      const int64_t row = base_rows[off + j];
      if (row < 0 || row + page_len > cache_rows)
        return fail(IFR_EINVAL, "run %lld page %lld: base row %lld outside cache of %lld rows", (long long)i, (long long)j,
                    (long long)row, (long long)cache_rows);
      if (block_len > 0 && row % block_len != 0)
        return fail(IFR_EINVAL, "run %lld page %lld: base row %lld is not at a block of %lld rows", (long long)i, (long long)j,
                    (long long)row, (long long)block_len);
      return IFR_OK;
    };
    const int64_t head_end = window > 0 ? ceil_div(std::min(sinks, last + 1), page_len) : 0;
    const int64_t tail = window > 0 ? std::max<int64_t>(0, base - window + 1) >> shift : 0;
    for (int64_t j = 0; j < head_end; ++j)
      if (int32_t e = check_page(j)) return e;
    for (int64_t j = std::max(tail, head_end); j <= (last >> shift); ++j)
      if (int32_t e = check_page(j)) return e;
  }

  // ---- parts: 16-column row tiles of short runs, prompt blocks of the others ----
  const int64_t gqa = num_q / num_kv;
  const int64_t row_tokens = kRowCols / gqa;
  const int64_t block_cols = prompt_cols(static_cast<int>(head_dim));
  const int64_t block_tokens = block_cols / gqa;
  Builder b{num_kv, gqa, window, sinks, {}, {}, {}, 0};
  std::vector<Part> few, many;
  int64_t few_tiles = 0, between = 0;
  const int64_t tile_bytes = 2 * kTileKeys * head_dim * (block_len > 0 ? 1 : 2);
  for (int64_t i = 0; i < num_runs; ++i) {
    const int64_t n = (i + 1 < num_runs ? runs[4 * (i + 1)] : seq_len) - runs[4 * i], cols = n * gqa;
    if (cols > kRowItemCols && cols <= kRowItemMost)
      between += b.tiles(runs[4 * i + 1], n) * ceil_div(cols, kRowCols) * num_kv * tile_bytes;
  }
  const int64_t row_cols = between <= kRowItemBytes ? kRowItemMost : kRowItemCols;
  for (int64_t i = 0; i < num_runs; ++i) {
    const int64_t start = runs[4 * i], base = runs[4 * i + 1];
    const int64_t n = (i + 1 < num_runs ? runs[4 * (i + 1)] : seq_len) - start;
    const bool rows = n * gqa <= row_cols;
    const int64_t width = rows ? row_tokens : block_tokens;
    for (int64_t t = 0; t < n; t += width) {
      const int64_t c = std::min(width, n - t);
      const Part p{i, start + t, c, base + t, b.tiles(base + t, c)};
      (rows ? few : many).push_back(p);
      few_tiles += rows ? p.tiles : 0;
    }
  }
  // A row item's four waves take a kv head each, or two of them or all four share the tiles of one.
  // Sharing costs a sum over LDS, and gives items of a half or a quarter the length.  Single tokens,
  // 1, 2 and 4 heads an item (us), by tiles times kv heads for each workgroup that runs at once:
  //   2 (1 sequence of 4,096, e4m3, 256 dims)     16, 18 and 22
  //   32 (16 of 4,096; 64 of 1,024)               56, 54 and 57; 53, 51 and 52
  //   33 (33 of 700 to 20,000, window 4,096, bf16, 512 dims, 2 heads)   149 and 155
  //   48 (48 of 4,096, int8, 512 dims, 2 heads)   94 and 82
  //   129 (64 of 4,096)                           188, 177 and 170
  // Two heads from 40 on: at 32 they gain 2 us of 55, at 33 in 512 dims they lose 6 of 149.
  const int64_t groups = resident_groups(head_dim);
  const int64_t load = few_tiles * num_kv / groups;
  int64_t per_group = 1;
  if (load >= 64 && num_kv % 4 == 0) per_group = 4;
  else if (load >= 40 && num_kv % 2 == 0) per_group = 2;
  const int64_t subs = 4 / per_group;
  const int64_t few_chunk = row_chunk(few, num_kv / per_group, subs, groups);
  const int64_t rows_base = 0;  // filled below: offsets are relative to the row table
  for (const Part& p : few) {
    const int64_t n = std::min<int64_t>(ceil_div(p.tiles, few_chunk), kMaxStripes);
    b.put(b.items, p.t0, p.ntok, rows_base + runs[4 * p.run + 2], p.p0, std::max<int64_t>(n, 1), kRowCols);
  }
  const std::vector<int64_t> splits = prompt_splits(many, num_kv);
  for (size_t i = 0; i < many.size(); ++i)
    b.put(b.prompts, many[i].t0, many[i].ntok, rows_base + runs[4 * many[i].run + 2], many[i].p0, splits[i], block_cols);
  longest_first(b.items);
  longest_first(b.prompts);

  // ---- write blocks of an 8-bit cache ----
  std::vector<std::array<int32_t, kWriteBlockWords>> writes;
  bool shared = false;
  if (block_len > 0) {
    std::vector<int64_t> pages_written;
    for (int64_t i = 0; i < num_runs; ++i) {
      const int64_t start = runs[4 * i], base = runs[4 * i + 1], off = runs[4 * i + 2];
      const int64_t n = (i + 1 < num_runs ? runs[4 * (i + 1)] : seq_len) - start;
      for (int64_t pg = base >> shift; pg <= ((base + n - 1) >> shift); ++pg) pages_written.push_back(base_rows[off + pg]);
      for (int64_t p = base; p < base + n;) {
        const int64_t end = std::min((p / block_len + 1) * block_len, base + n);
        writes.push_back({static_cast<int32_t>(start + p - base), static_cast<int32_t>(end - p),
                          static_cast<int32_t>(base_rows[off + (p >> shift)] + (p & row_mask)), static_cast<int32_t>(p)});
        p = end;
      }
    }
    // Pages lie where their base rows say, aligned to blocks and not to pages, so two
    // written pages overlap where their rows are less than a page apart.
    std::sort(pages_written.begin(), pages_written.end());
    for (size_t i = 1; i < pages_written.size(); ++i) shared |= pages_written[i] - pages_written[i - 1] < page_len;
  }

  // ---- the image ----
  const int64_t n_items = static_cast<int64_t>(b.items.size()), n_prompts = static_cast<int64_t>(b.prompts.size());
  const int64_t n_units = static_cast<int64_t>(b.units.size()), n_writes = static_cast<int64_t>(writes.size());
  const int64_t off_items = kHdrWords, off_prompts = off_items + kWorkWords * n_items;
  const int64_t off_units = off_prompts + kWorkWords * n_prompts, off_writes = off_units + kMergeWords * n_units;
  const int64_t off_runs = off_writes + kWriteBlockWords * n_writes, off_rows = off_runs + 4 * num_runs;
  const int64_t off_tok = off_rows + num_rows, total = off_tok + seq_len;
  if (total > INT32_MAX || b.cols > INT32_MAX) return fail(IFR_EINVAL, "plan too large");
  if (total > img_words)
    return fail(IFR_ESPACE, "plan image needs %lld bytes, have %lld", (long long)(total * 4), (long long)(img_words * 4));
  memset(img, 0, sizeof(int32_t) * kHdrWords);
  auto put_items = [&](int64_t off, const std::vector<Work>& v) {
    for (size_t i = 0; i < v.size(); ++i) {
      int32_t* w = img + off + static_cast<int64_t>(i) * kWorkWords;
      memcpy(w, v[i].words.data(), sizeof(int32_t) * kWorkWords);
      w[kItRows] += static_cast<int32_t>(off_rows);
    }
  };
  put_items(off_items, b.items);
  put_items(off_prompts, b.prompts);
  for (int64_t i = 0; i < n_units; ++i) memcpy(img + off_units + i * kMergeWords, b.units[i].data(), sizeof(int32_t) * kMergeWords);
  for (int64_t i = 0; i < n_writes; ++i)
    memcpy(img + off_writes + i * kWriteBlockWords, writes[i].data(), sizeof(int32_t) * kWriteBlockWords);
  memcpy(img + off_runs, runs, sizeof(int32_t) * 4 * num_runs);
  memcpy(img + off_rows, base_rows, sizeof(int32_t) * num_rows);
  for (int64_t i = 0; i < num_runs; ++i) {
    const int64_t next = i + 1 < num_runs ? runs[4 * (i + 1)] : seq_len;
    for (int64_t t = runs[4 * i]; t < next; ++t) img[off_tok + t] = static_cast<int32_t>(i);
  }
  img[kHdrMagic] = kPlanMagic;
  img[kHdrNumRuns] = static_cast<int32_t>(num_runs);
  img[kHdrNumRows] = static_cast<int32_t>(num_rows);
  img[kHdrSeqLen] = static_cast<int32_t>(seq_len);
  img[kHdrNumItems] = static_cast<int32_t>(n_items);
  img[kHdrNumUnits] = static_cast<int32_t>(n_units);
  img[kHdrMode] = IFR_PLAN_WINDOW;
  img[kHdrOffRuns] = static_cast<int32_t>(off_runs);
  img[kHdrOffRows] = static_cast<int32_t>(off_rows);
  img[kHdrOffTokRun] = static_cast<int32_t>(off_tok);
  img[kHdrOffItems] = static_cast<int32_t>(off_items);
  img[kHdrOffUnits] = static_cast<int32_t>(off_units);
  img[kHdrTotalWords] = static_cast<int32_t>(total);
  img[kHdrOffQBlocks] = static_cast<int32_t>(off_prompts);
  img[kHdrNumQBlocks] = static_cast<int32_t>(n_prompts);

  memset(info, 0, sizeof(int64_t) * IFR_WINDOW_INFO_LEN);
  info[kInItems] = n_items;
  info[kInUnits] = n_units;
  info[kInMode] = IFR_PLAN_WINDOW;
  info[kInCols] = b.cols;
  info[kInBytes] = total * 4;
  info[kInSeq] = seq_len;
  info[kInRuns] = num_runs;
  info[kInShift] = shift;
  info[kInRowMask] = row_mask;
  info[kInPageMask] = -1;
  info[kInCacheRows] = cache_rows;
  info[kInKind] = 2;
  info[kInWindow] = window;
  info[kInMaxPos] = max_pos;
  info[kInPrompts] = n_prompts;
  info[kInWrites] = n_writes;
  info[kInSinks] = sinks;
  info[kInNumQ] = num_q;
  info[kInNumKv] = num_kv;
  info[kInHeadDim] = head_dim;
  info[kInBlock] = block_len;
  info[kInWorkspace] = b.cols * (head_dim + 2) * 4;
  info[kInOffPrompts] = off_prompts;
  info[kInOffWrites] = off_writes;
  info[kInOffUnits] = off_units;
  info[kInHeadsPerGroup] = per_group;
  info[kInSharedWrites] = shared ? 1 : 0;
  return ifr::abi_ok();
}

int32_t check_info(const int64_t* info, int64_t num_q, int64_t num_kv, int64_t head_dim, int64_t kv_stride, int64_t elt_bytes) {
  if (!info) return fail(IFR_EINVAL, "null info");
  if (info[kInMode] != IFR_PLAN_WINDOW) return fail(IFR_EINVAL, "info does not describe a window plan (ifr_plan_window)");
  if (num_q != info[kInNumQ] || num_kv != info[kInNumKv] || head_dim != info[kInHeadDim])
    return fail(IFR_EINVAL, "heads (%lld, %lld, %lld) differ from the plan's (%lld, %lld, %lld)", (long long)num_q,
                (long long)num_kv, (long long)head_dim, (long long)info[kInNumQ], (long long)info[kInNumKv],
                (long long)info[kInHeadDim]);
  if (kv_stride < num_kv * head_dim || (kv_stride * elt_bytes) % 16 != 0)
    return fail(IFR_EINVAL, "kv_stride must cover num_kv*head_dim and keep rows 16-byte aligned");
  if (kv_stride > (int64_t{1} << 24)) return fail(IFR_EUNSUPPORTED, "kv_stride > 2^24");
  return IFR_OK;
}

int32_t attention(int format, const void* image, const int64_t* info, const void* q, const void* k, const float* k_scale,
                  const void* v, const float* v_scale, void* output, void* workspace, int64_t workspace_bytes,
                  int64_t num_q, int64_t num_kv, int64_t head_dim, int64_t kv_stride, float scale, uint64_t stream) {
  if (int32_t st = check_info(info, num_q, num_kv, head_dim, kv_stride, format == kBf16 ? 2 : 1)) return st;
  if (!image || !q || !k || !v || !output || (format != kBf16 && (!k_scale || !v_scale))) return fail(IFR_EINVAL, "null pointer");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(output, 16))
    return fail(IFR_EINVAL, "q, the caches and output must be 16-byte aligned");
  if (format != kBf16 && info[kInBlock] == 0) return fail(IFR_EINVAL, "the plan has no block_len: it was made for a bf16 cache");
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.0f) || !isfinite(scale_log2)) return fail(IFR_EINVAL, "scale must be positive, and finite times log2 e");
  if (info[kInWorkspace] > 0) {
    if (!workspace || workspace_bytes < info[kInWorkspace])
      return fail(IFR_ESPACE, "workspace of %lld bytes, the plan needs %lld", (long long)(workspace ? workspace_bytes : 0),
                  (long long)info[kInWorkspace]);
    if (!aligned(workspace, 16)) return fail(IFR_EINVAL, "workspace must be 16-byte aligned");
  }
  ifr::WindowArgs a{};
  a.image = static_cast<const int32_t*>(image);
  a.q = q;
  a.k = k;
  a.v = v;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.out = output;
  a.partials = static_cast<float*>(workspace);
  a.sums = a.partials ? a.partials + info[kInCols] * head_dim : nullptr;
  a.kv_stride = kv_stride;
  a.num_q = static_cast<int>(num_q);
  a.num_kv = static_cast<int>(num_kv);
  a.gqa = static_cast<int>(num_q / num_kv);
  a.shift = static_cast<int>(info[kInShift]);
  a.row_mask = static_cast<int>(info[kInRowMask]);
  a.block_shift = info[kInBlock] > 0 ? static_cast<int>(shift_of(info[kInBlock])) : 0;
  a.window = static_cast<int>(info[kInWindow]);
  a.sinks = static_cast<int>(info[kInSinks]);
  a.scale_log2 = scale_log2;
  const hipStream_t s = reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(stream));
  const int dim = static_cast<int>(head_dim);
  hipError_t e = hipSuccess;
  if (info[kInPrompts] > 0)
    e = ifr::launch_window_prompts(a, format, dim, static_cast<int>(info[kInOffPrompts]), info[kInPrompts], s);
  if (e == hipSuccess && info[kInItems] > 0)
    e = ifr::launch_window_rows(a, format, dim, ifr::kHdrWords, info[kInItems], static_cast<int>(info[kInHeadsPerGroup]), s);
  if (e == hipSuccess && info[kInUnits] > 0)
    e = ifr::launch_window_merge(a, dim, static_cast<int>(info[kInOffUnits]), info[kInUnits], s);
  if (e != hipSuccess) return fail(IFR_EHIP, "window attention: %s", hipGetErrorString(e));
  return ifr::abi_ok();
}

}  // namespace

extern "C" {

int64_t ifr_plan_window_bytes(int64_t num_runs, int64_t num_rows, int64_t seq_len, int64_t block_len) {
  if (num_runs < 0 || num_rows < 0 || seq_len < 0 || block_len < 0) return -1;
  if (num_runs > kMostTokens || num_rows > kMostRows || seq_len > kMostTokens) return -1;  // the plan refuses them
  return 4 * most_words(num_runs, num_rows, seq_len, block_len);
}

int32_t ifr_plan_window(void* image, int64_t image_bytes, const int32_t* runs, int64_t num_runs, const int32_t* base_rows,
                        int64_t num_rows, int64_t seq_len, int64_t window, int64_t sinks, int64_t page_len,
                        int64_t cache_rows, int64_t num_q, int64_t num_kv, int64_t head_dim, int64_t block_len,
                        int64_t* info) {
  try {
    return plan(static_cast<int32_t*>(image), image_bytes / 4, runs, num_runs, base_rows, num_rows, seq_len, window, sinks,
                page_len, cache_rows, num_q, num_kv, head_dim, block_len, info);
  } catch (const std::bad_alloc&) {  // no exception passes a C entry
    return fail(IFR_ENOMEM, "no host memory to plan %lld tokens in", (long long)seq_len);
  }
}

int32_t ifr_window_attention_bf16(const void* image_dev, const int64_t* info, const void* q, const void* k_base,
                                  const void* v_base, void* output, void* workspace, int64_t workspace_bytes,
                                  int64_t num_q, int64_t num_kv, int64_t head_dim, int64_t kv_stride, float scale,
                                  uint64_t stream) {
  return attention(kBf16, image_dev, info, q, k_base, nullptr, v_base, nullptr, output, workspace, workspace_bytes, num_q,
                   num_kv, head_dim, kv_stride, scale, stream);
}

int32_t ifr_kv8_attention(const void* image_dev, const int64_t* info, const void* q, const void* k_base,
                          const float* k_scale, const void* v_base, const float* v_scale, void* output, void* workspace,
                          int64_t workspace_bytes, int64_t num_q, int64_t num_kv, int64_t head_dim, int64_t kv_stride,
                          float scale, int64_t kv_format, uint64_t stream) {
  if (kv_format != IFR_KV8_E4M3 && kv_format != IFR_KV8_INT8) return fail(IFR_EINVAL, "kv_format must be IFR_KV8_E4M3 or IFR_KV8_INT8");
  return attention(static_cast<int>(kv_format), image_dev, info, q, k_base, k_scale, v_base, v_scale, output, workspace,
                   workspace_bytes, num_q, num_kv, head_dim, kv_stride, scale, stream);
}

int32_t ifr_kv8_cache_write(const void* image_dev, const int64_t* info, const void* q_src, const void* k_src,
                            const void* v_src, void* q_out, void* k_cache, float* k_scale, void* v_cache, float* v_scale,
                            const float* cos_table, const float* sin_table, int64_t num_q, int64_t num_kv, int64_t seq_len,
                            int64_t half, int64_t pair_stride, int64_t head_dim, int64_t kv_stride, int64_t kv_format,
                            uint64_t stream) {
  if (kv_format != IFR_KV8_E4M3 && kv_format != IFR_KV8_INT8) return fail(IFR_EINVAL, "kv_format must be IFR_KV8_E4M3 or IFR_KV8_INT8");
  if (int32_t st = check_info(info, num_q, num_kv, head_dim, kv_stride, 1)) return st;
  if (seq_len != info[kInSeq]) return fail(IFR_EINVAL, "seq_len differs from the plan");
  if (info[kInBlock] == 0) return fail(IFR_EINVAL, "the plan has no block_len: it was made for a bf16 cache");
  if (info[kInSharedWrites]) return fail(IFR_EINVAL, "two pages that the step writes to share rows");
  if (!image_dev || !q_src || !k_src || !v_src || !q_out || !k_cache || !k_scale || !v_cache || !v_scale || !cos_table || !sin_table)
    return fail(IFR_EINVAL, "null pointer");
  if (!aligned(q_src, 16) || !aligned(k_src, 16) || !aligned(v_src, 16) || !aligned(q_out, 16) || !aligned(k_cache, 16) ||
      !aligned(v_cache, 16) || !aligned(cos_table, 16) || !aligned(sin_table, 16))
    return fail(IFR_EINVAL, "q, k, v, the caches and the tables must be 16-byte aligned");
  if (half <= 0 || half > pair_stride || pair_stride + half > head_dim) return fail(IFR_EINVAL, "bad rope geometry");
  if (half % 8 != 0 || pair_stride % 8 != 0) return fail(IFR_EUNSUPPORTED, "half and pair_stride must be multiples of 8");
  ifr::Kv8WriteArgs a{};
  a.image = static_cast<const int32_t*>(image_dev);
  a.q = q_src;
  a.k = k_src;
  a.v = v_src;
  a.q_out = q_out;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.cos_table = cos_table;
  a.sin_table = sin_table;
  a.kv_stride = kv_stride;
  a.num_q = static_cast<int>(num_q);
  a.num_kv = static_cast<int>(num_kv);
  a.seq_len = static_cast<int>(seq_len);
  a.half = static_cast<int>(half);
  a.pair_stride = static_cast<int>(pair_stride);
  a.block_shift = static_cast<int>(shift_of(info[kInBlock]));
  a.off_writes = static_cast<int>(info[kInOffWrites]);
  a.num_writes = info[kInWrites];
  const hipError_t e = ifr::launch_kv8_write(a, static_cast<int>(kv_format), static_cast<int>(head_dim),
                                             reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(stream)));
  if (e != hipSuccess) return fail(IFR_EHIP, "kv8 cache write: %s", hipGetErrorString(e));
  return ifr::abi_ok();
}

}  // extern "C"
