// Attention with a window and sinks over bf16 and 8-bit caches: what the planner
// (window_api.hip) and the kernels (window_rows.hip, window_prefill.hip, kv8_write.hip)
// share.
//
// A query at position p sees the positions j <= p with window == 0, j > p - window or
// j < sinks.  The cache is walked in tiles of 32 positions that start at multiples of 32;
// the tiles that some query of a work item sees are numbered from 0: `sink tiles` 0 ..
// n_sink - 1 of the sequence, then the tiles from the window's first one on.
#pragma once

#include <stdint.h>

namespace ifr {
namespace window {

constexpr int kTileKeys = 32;  // positions of a tile: one K = 32 product of P.V
// Formats of a cache.
enum Format : int { kBf16 = 0, kE4m3 = 1, kInt8 = 2 };

// Work item (image words): query tokens [t0, t0 + ntok) of one run against its visible
// tiles [lo, hi).  col0: the first of its partial columns (kv head 0), or -1 where the
// item covers everything its queries see and writes the output itself.
enum Item : int { kItT0, kItTokens, kItRows, kItPos, kItLo, kItHi, kItCol, kItPad, kWorkWords };
// Merge unit: a token whose tiles were split over n items.  Its columns of item s and kv
// head h start at col + s * step + h * hstep.
enum Unit : int { kUnToken, kUnCount, kUnCol, kUnStep, kUnHstep, kUnPad0, kUnPad1, kUnPad2, kMergeWords };
// Write block: `count` of the step's tokens in one block of the 8-bit cache: the first
// token, the cache row and the position of it.
enum WriteBlock : int { kWbToken, kWbCount, kWbRow, kWbPos, kWriteBlockWords };

constexpr int64_t kMaxGroups = (1 << 23) - 1;  // a launch's threads fit 32 bits at up to 512 a workgroup
constexpr int kMaxStripes = 64;  // splits of a token: one lane each in the merge kernel
constexpr int kRowCols = 16;     // columns of a row item: (token, q head of the kv head)

// A prompt block: eight waves, each with some tiles of 32 columns, at head_dim 512 of 16.
constexpr int kPromptWaves = 8;
constexpr int prompt_tile_cols(int head_dim) { return head_dim == 512 ? 16 : 32; }
constexpr int prompt_col_tiles(int head_dim) { return head_dim == 128 ? 2 : 1; }
constexpr int prompt_cols(int head_dim) { return kPromptWaves * prompt_tile_cols(head_dim) * prompt_col_tiles(head_dim); }

struct Span {
  int n_sink;  // sink tiles ahead of the window's first tile
  int first;   // the window's first tile
};
// Of queries whose first position is p0.
#ifdef __HIPCC__
__host__ __device__
#endif
inline Span visible_span(int p0, int window, int sinks) {
  Span s{0, 0};
  if (window > 0) {
    const int lo = p0 - window + 1;
    s.first = lo > 0 ? lo / kTileKeys : 0;
    const int head = (sinks + kTileKeys - 1) / kTileKeys;
    s.n_sink = head < s.first ? head : s.first;
  }
  return s;
}

}  // namespace window
}  // namespace ifr
