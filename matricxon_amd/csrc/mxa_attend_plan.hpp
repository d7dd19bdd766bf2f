// How attention over the 4-bit cache shares its work out, in plain C++. (std::min and std::max by their full names: HIP's own
// take ints on the host.)
#pragma once

#include <limits.h>
#include <stddef.h>

#include <algorithm>

#include "mxa_kv4_shape.hpp"

namespace mxa {

constexpr int kAttendMaxSplits = 768;

// Floats of a split's part of a tile's rows: 16 rows of 32 w values, 16 references, 16 sums.
inline size_t part_floats(int w) { return 16 * 32 * (size_t)w + 32; }

// Shares of `least` to `most` blocks for the workgroups that the CUs hold at once. At least two blocks a wave: 1000 places
// of one reply took 13.8 us in shares of 4 blocks, 11.8 of 8, 12.2 of 16 (9.5 since their join is faster). At most 128
// blocks where several sequences end at places that the host does not know: 64 replies of up to 16384 places 188 us without,
// 149 us with that bound, 160 of 96. More of them where the parts would not fit into what there is for them.
inline void share_out(long long blocks, long long workgroups, long long slots, int least, int most, int most_splits,
                      int& splits, int& chunk) {
  const long long want = std::max<long long>(1, slots / workgroups);
  chunk = (int)std::max<long long>(least, std::min<long long>(most, (blocks + want - 1) / want));
  most_splits = std::min<int>(most_splits, kAttendMaxSplits);
  chunk = (int)std::max<long long>(chunk, (blocks + most_splits - 1) / most_splits);
  splits = (int)((blocks + chunk - 1) / chunk);
  chunk = (int)((blocks + splits - 1) / splits);
}

// How the places of up to `most` tokens of each sequence are shared out. Sequences of up to kFewRows rows a key head go in
// tiles of 16 rows (attend_kernel), others in those of attend_tile_kernel, which widens a place once for
// all of them; a call without query_starts has one kind. 16 sequences of 2048 places take, of 64 rows a key head, 32 us in
// tiles of 16 and 41 in the others; of 96 rows 39 and 43; of 128 rows 51 and 45, and with lengths of all sizes up to 2048
// 36 and 43.
constexpr int kFewRows = 128, kTileSplits = 16, kFewParts = 16, kLeastBlocks = 8, kMostBlocks = 128;
constexpr long long kMostFloats = 64 << 20;  // of a call's parts, of both kinds together
struct Plan {
  bool few, many;       // the kinds that there may be
  long long pairs[2];   // (tile of 16 rows, key head) of a sequence
  int splits[2], chunk[2];
  int rows;             // of a workgroup, for many rows
  long long tiles;      // of the call, for many rows
  long long slots;      // tiles of 16 rows of the call, at most
  int per[2];           // tiles that the parts have room for of each sequence, or 0: for all of the call's as they lie in it
  long long floats[2];  // of the tiles' parts, one each
};

inline Plan plan_of(int n_seq, int n_tokens, bool ragged, int kv_heads, int group, int max_length, long long window,
                    int dim) {
  Plan p{};
  const long long most = (long long)(ragged ? n_tokens : n_tokens / n_seq) * group;
  p.few = ragged || most <= kFewRows;
  p.many = most > kFewRows;
  const long long reach = window > 0 ? std::min<long long>(max_length, window + most / group) : max_length;
  const long long blocks = reach / kKvBlock + 2;
  const bool narrow = kv_groups(dim) <= 4;
  const long long part = kv_heads * (long long)part_floats(kv_groups(dim));
  p.slots = (long long)n_tokens * group / 16 + n_seq;
  if (p.many) {
    p.pairs[1] = (most + 15) / 16 * kv_heads;
    p.floats[1] = p.slots * part;
    // Workgroups of 256 rows widen a place once for all; where they are too few for the CUs and their places few as well,
    // two of 128 rows hide each other's waits: 128 tokens x 32 heads of 128, window 1024: 27.9 and 22.3 us; without, over
    // 8192 places, 52.7 and 57.2.
    const auto span_of = [&](int rows) {
      return window > 0 ? std::min<long long>(max_length, window + rows / group) / kKvBlock + 2 : blocks;
    };
    const bool fill = (most + 255) / 256 * kv_heads * (ragged ? 1 : n_seq) >= 256;
    p.rows = narrow && most > 128 && (fill || span_of(256) > 48) ? 256 : 128;
    p.tiles = ragged ? most / p.rows + std::min<long long>(n_seq, most / (kFewRows + 1)) : (most + p.rows - 1) / p.rows * n_seq;
    const long long span = span_of(p.rows);
    const long long groups = p.tiles * kv_heads, slots = narrow && p.rows == 128 ? 512 : 256;
    // Parts of a tile's places, by what they cost: as many rounds of the CUs as the workgroups take, each a part's blocks
    // and some 10 blocks' time to begin and end, and the join. Half of the room, where there may be few rows as well.
    const long long room = p.few ? kMostFloats / 2 : kMostFloats;
    double least = 0;
    for (int n = 1; n <= kTileSplits && (n == 1 || (span / n >= 8 && p.floats[1] * n <= room)); ++n) {
      const double cost = (double)((groups * n + slots - 1) / slots) * ((double)span / n + 10) + (n > 1 ? 8 : 0);
      if (n == 1 || cost < 0.95 * least) least = cost, p.splits[1] = n;
    }
    p.chunk[1] = 0;
  }
  if (p.few) {
    const long long tiles = (std::min<long long>(most, kFewRows) + 15) / 16;  // of a sequence
    p.pairs[0] = tiles * kv_heads;
    // Room for the tiles of sequences of few rows alone: a long chunk in the call leaves the replies beside it their shares
    // (three replies of 131072 places beside 8192 tokens, 32 + 8 heads of 128: shares of 128 blocks; with room for all tiles
    // of the call there would be one share of all 4098).
    p.per[0] = tiles * n_seq <= p.slots ? (int)tiles : 0;
    p.floats[0] = std::min<long long>(tiles * n_seq, p.slots) * part;
    const long long room = kMostFloats - (p.many && p.splits[1] > 1 ? p.floats[1] * p.splits[1] : 0);
    const long long slots = 256 * (narrow ? 3 : 2);  // workgroups that the CUs hold at once
    // pairs that have rows: with query_starts the grid has room for any sequence to have all of them, and those of many rows
    // are not here
    const long long pairs = std::min<long long>(p.pairs[0] * n_seq,
                                                kv_heads * std::max<long long>(std::min(n_seq, n_tokens), (long long)n_tokens * group / 16));
    share_out(blocks, pairs, slots, kLeastBlocks, n_seq > 1 ? kMostBlocks : INT_MAX,
              (int)std::max<long long>(1, room / p.floats[0]), p.splits[0], p.chunk[0]);
  }
  return p;
}

inline size_t part_bytes(const Plan& p, int kind) {
  return p.splits[kind] <= 1 ? 0 : (size_t)(p.floats[kind] * p.splits[kind]) * sizeof(float);
}
inline size_t parts_bytes(const Plan& p) { return part_bytes(p, 0) + part_bytes(p, 1); }

}  // namespace mxa
