// What a block of the packed causal attention in tensor memory covers, usable on the host
// and the device (a plain C++ compiler reads this file too).
#pragma once
#include "pages.cuh"

namespace oasis {

constexpr int kPromptTile = 128;  // query rows of a tile, keys of a block

// The block's two tiles. Every role works it out alike from cu.
struct PromptUnit {
  int head[2], r0[2];       // tile t: its head and first row
  int begin;                // first key of block 0
  int first[2], last[2];    // tile t takes key blocks [first, last)
  int blocks;

  // Whether tile t has a key block. Its Q is fetched only then: the warp that issues the
  // products waits for it ahead of the tile's first one, and nobody does for a tile without
  // any, whose copy could then still be on its way when the block gives its memory back.
  OASIS_HD bool has(int t) const { return first[t] < last[t]; }
};

// Row tiles (or pairs) `rt` of head (or pair of heads) x; rows of sequences end at `end`.
OASIS_HD PromptUnit prompt_unit(const int* cu, int n, bool pair_heads, int end, int x, int rt) {
  constexpr int kNone = 0x7fffffff;
  PromptUnit u;
  const int rows = pair_heads ? kPromptTile : 2 * kPromptTile;
  int low[2];
  u.begin = kNone;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    u.head[t] = pair_heads ? 2 * x + t : x;
    u.r0[t] = rt * rows + (pair_heads ? 0 : t * kPromptTile);
    // the first row of the tile that belongs to a sequence, and that sequence's start
    int lo = kNone;
    if (t == 1 && pair_heads) {
      lo = low[0];
    } else if (u.r0[t] < end) {
      const int a = cu[last_not_above(cu, n, u.r0[t])];
      if (a > u.r0[t]) {
        if (a < u.r0[t] + kPromptTile && a < end) lo = a;
      } else if (a >= 0) {
        lo = a;
      }
    }
    low[t] = lo;
    u.begin = lo < u.begin ? lo : u.begin;
  }
  u.blocks = 0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    u.first[t] = u.last[t] = 0;
    if (low[t] != kNone) {
      const int to = u.r0[t] + kPromptTile < end ? u.r0[t] + kPromptTile : end;
      u.first[t] = (low[t] - u.begin) / kPromptTile;
      u.last[t] = (to - u.begin + kPromptTile - 1) / kPromptTile;
      u.blocks = u.last[t] > u.blocks ? u.last[t] : u.blocks;
    }
  }
  return u;
}

}  // namespace oasis
