// attn_plan.hpp -- how swamp_attn_paged cuts a call into workgroups: blocks of rows
// and pieces of the keys.  Host-only arithmetic on sizes, so that it can be checked
// without a GPU.
#pragma once
#include <math.h>

#include <algorithm>

#include "paging.hpp"

namespace swamp_attn {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRows = 128;     // rows of a block
constexpr int kFew = 32;       // rows up to which a block's waves share the rows instead
constexpr int kTile = 64;      // keys of a workgroup's tile

}  // namespace swamp_attn

namespace swamp {

using swamp_attn::kFew;
using swamp_attn::kRows;
using swamp_attn::kTile;
using swamp_attn::kWaves;

// Workgroups that one launch can have: its threads are counted in 32 bits.
constexpr int64_t kMaxGroups = (int64_t(1) << 32) / swamp_attn::kThreads - 1;
// Positions from here on are not walked, so that a tile's end is still an int.
constexpr int64_t kLastPosition = (int64_t(1) << 31) - 512;

// Pieces of a call that is cut for evenness rather than to fill the card, and bytes
// of partial sums that a call may ask the stream's scratch for.  Pieces are written
// and read once each, 256 dim bytes a block of 32 rows against 4 dim bytes a key:
// a few percent of the time wherever the lengths are near max_len.
constexpr int kMostPieces = 16;
constexpr size_t kPartBytes = size_t(256) << 20;

// Positions that a page table holds and that are walked.
SWAMP_HD int64_t walked(int64_t pages_stride, int page_shift) {
  const int64_t cols = int64_t(1) << 31;
  const int64_t room = (pages_stride < cols ? pages_stride : cols) << page_shift;
  return room < kLastPosition ? room : kLastPosition;
}

struct AttnPlan {
  int blocks, one_block, few, splits, chunk;
};

// Pieces of the keys that make attn_many_kernel shortest, by a model of its time
// on this card, us: a tile takes 0.55 + 0.007 dim where a CU has one workgroup
// and 0.6 more for each further one (heads of 128: 1.45 and 2.06 us measured), a
// workgroup's start and end three tiles, and a join 4 us and its sums' way
// through memory.  A last round that is not full costs its share, as most rows
// see less than the longest sequence, and a little more: without it 45
// workgroups of 256 dims go in 6 pieces instead of 5, 38.8 us and 30.8.  Down
// to one tile a piece pays (7 workgroups, 256 dims, 554 keys: pieces of four
// tiles 34.8 us, of one 23.7).
inline int many_splits(int64_t base, int64_t rows, int64_t keys, int dim, int cus) {
  const int most = dim <= 64 ? 3 : dim <= 128 ? 2 : 1;  // workgroups of a CU
  const double tiles = double(keys) / kTile;
  double best = 0;
  int want = 1;
  for (int n = 1; n <= kMostPieces && n <= std::max<int64_t>(1, keys / kTile); n++) {
    const int64_t load = std::min<int64_t>(most, (base * n + cus - 1) / cus);
    const double rounds = std::max(1.0, double(base) * n / (double(cus) * most));
    double t = (0.95 * rounds + 0.05 * std::ceil(rounds)) * (tiles / n + 3) * (0.55 + 0.007 * dim + 0.6 * double(load - 1));
    if (n > 1) t += 4 + n * double(rows) * dim * 8 / 6e6;
    if (n == 1 || t < best) best = t, want = n;
  }
  return want;
}

inline size_t attn_part_bytes(const AttnCall &c, int splits) {
  return size_t(splits) * c.batch.n_tok * c.n_heads * c.cache.dim * 4;
}
inline size_t attn_stat_bytes(const AttnCall &c, int splits) {
  return size_t(splits) * c.batch.n_tok * c.n_heads * 8;
}

// Sums and statistics of one piece.
inline size_t attn_piece_bytes(const AttnCall &c) {
  return attn_part_bytes(c, 1) + attn_stat_bytes(c, 1);
}

// Blocks of rows of a cache head, of a sequence at most `most`, of all sequences at
// most this many, whatever the rows' distribution.
inline int64_t attn_blocks(const AttnCall &c, int64_t &most) {
  const int group = c.n_heads / c.cache.n_kv;
  const int64_t rows = int64_t(c.batch.n_tok) * group;
  most = (int64_t(c.max_new) * group + kRows - 1) / kRows;
  return most <= 1 ? c.batch.n_seq
                   : std::min((rows + int64_t(kRows - 1) * c.batch.n_seq) / kRows,
                              most * c.batch.n_seq);
}
// One launch holds the call.
inline bool attn_fits(const AttnCall &c) {
  int64_t most;
  return attn_blocks(c, most) * c.cache.n_kv <= kMaxGroups;
}

// Of a call that attn_fits.
inline AttnPlan plan_attn(const AttnCall &c, int cus) {
  const int group = c.n_heads / c.cache.n_kv;
  const int64_t rows = int64_t(c.batch.n_tok) * group;  // of a cache head
  int64_t most;
  AttnPlan p;
  p.blocks = int(attn_blocks(c, most));
  p.few = int64_t(c.max_new) * group <= kFew;
  p.one_block = most <= 1;
  const int64_t base = std::max<int64_t>(1, int64_t(p.blocks) * c.cache.n_kv);
  const int64_t seen = int64_t(c.window) + (p.few ? c.max_new : kRows / group) + kTile;
  const int64_t held = std::min<int64_t>(
      c.max_len, walked(c.batch.pages_stride, c.cache.page_shift));
  const int64_t keys = c.window ? std::min(held, seen) : held;
  int64_t want;
  if (p.few) {
    // one workgroup a CU, of short heads two while a piece keeps two steps (64
    // workgroups of 128 dims over 4001 keys: 256 in all 22.4 us, 512 25.2, 64 60;
    // 22 of 64 dims over up to 22634 keys: 528 in all 27.5, 242 41.5; 2 over 20345:
    // 160 in all 13.3, 318 14.8)
    want = cus / base;
    if (c.cache.dim <= 64) want = std::max(want, std::min(2 * cus / base, keys / (64 * kWaves)));
    // sequences of unequal length in a piece or two each: pieces of 2048 keys even
    // them out (256 workgroups over up to 6000 keys 39.9 us, whole 47.0; 115 over
    // up to 14540: 68.5, in two 78.9); where there are more pieces these are too
    // many (70 of 256 dims over up to 13260 keys: 124 us, in three 109)
    // (kMostPieces at most, as max_len may be far above the lengths: 64 sequences of
    // 1000 tokens, 512 workgroups, under a max_len of 131072: in 64 pieces 164 us, in
    // 16 43, while 11 of up to 36000 keep their 105 and 186 at 64 and 128 dims)
    if (want < 3) want = std::max(want, std::min<int64_t>(kMostPieces, keys / 2048));
    // none below the time of the join (8 workgroups, 128 dims, 512 keys: whole 9.6
    // us, in pieces 11.1; 1024 keys: 14.2 and 10.8; 64 dims, 1024 keys: 10.6 and 11)
    if (keys * c.cache.dim <= 65536) want = 1;
  } else {
    want = many_splits(base, rows * c.cache.n_kv, keys, c.cache.dim, cus);
  }
  want = std::min(want, int64_t(kPartBytes / std::max<size_t>(1, attn_piece_bytes(c))));
  // what one launch holds, and the join's, which has a row a workgroup at worst
  want = std::min(want, kMaxGroups / base);
  if (int64_t(c.batch.n_tok) * c.n_heads > kMaxGroups) want = 1;
  // a piece is whole tiles; of a few rows one for each wave at least
  const int64_t step = p.few ? 32 * kWaves : kTile;
  want = std::max<int64_t>(1, want);
  const int64_t chunk = std::max(((keys + want - 1) / want + step - 1) / step * step, step);
  p.chunk = int(chunk);  // (kLastPosition is whole steps)
  p.splits = int(std::max<int64_t>(1, (keys + chunk - 1) / chunk));
  return p;
}

}  // namespace swamp
