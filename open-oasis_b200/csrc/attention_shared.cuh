// Arguments and index helpers of the attention over the paged cache.
#pragma once
#include <cuda_runtime.h>

#include "pages.cuh"

namespace oasis {

constexpr int kUnit = 16;  // keys of a step of a warp: always inside one page

struct SharedParams {
  PageGeometry g;
  const void *q, *pool;
  void* out;
  long long q_row, q_head, o_row, o_head;
  const int *table, *lengths, *seqs, *group_start, *prefix_pages;
  int* status;
  float* part_o;   // [rows heads][splits][D]
  float2* part_ml; // [rows heads][splits] (what sum and values are relative to, sum): base-2 exponent of
                   // the maximum less the kernel's lift of its probabilities
  int rows, groups, heads, per, layer;  // per: heads of a key head
  int prefix_splits, own_splits, own_units, tiles, head_tiles, whole;  // own_units: of a split but the last
  int team;    // warps of an item of own keys: 1 or 4
  int tensor;  // the prefix runs on the tensor-memory kernel
  int reach;   // (row, head) queries of a group and key head that the prefix kernel takes
  float scale_log2;
};

// Length of row b's sequence, 0 where there is none; `s` its slot.
__device__ __forceinline__ int row_length(const SharedParams& p, int b, int* s) {
  const int x = p.seqs[b];
  *s = x;
  if (x < 0 || x >= p.g.slots) return 0;
  return held_tokens(p.lengths[x], p.g.page_size, p.g.width);
}

// Queries of a key head in the order (row, head of the key head): the tile's first one
// by 64-bit division once, those behind it by 32-bit ones.
struct Queries {
  long long row;   // row of the tile's first query
  unsigned head, per;
  __device__ __forceinline__ Queries(long long first, int per_) : row(first / per_), head((unsigned)(first % per_)), per(per_) {}
  __device__ __forceinline__ long long row_of(int r) const { return row + (head + r) / per; }
  __device__ __forceinline__ int head_of(int r) const { return (int)((head + r) % per); }
};

// Group of row b, by the whole warp: the last one that starts at or before b; -1
// where b lies outside of them.
__device__ __forceinline__ int row_group(const SharedParams& p, int b) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = p.groups;  // the answer is in [lo, lo + n)
  if (n < 1 || p.group_start[0] > b || p.group_start[p.groups] <= b) return -1;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const bool ok = i < n && p.group_start[lo + i] <= b;
    const int c = 32 - __clz(__ballot_sync(0xffffffffu, ok) | 1u);  // probes that hold: a run from lane 0
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  return lo;
}

// Tokens of a group's prefix.
__device__ __forceinline__ int group_tokens(const SharedParams& p, int group) {
  return group < 0 ? 0 : held_tokens(p.prefix_pages[group], 1, p.g.width) * p.g.page_size;
}

// The group whose prefix ranges row b takes, by the whole warp: -1 where it lies outside
// of the groups or behind the rows that the prefix kernel takes (a group larger than the
// caller's hint); its prefix is then part of its own keys.
__device__ __forceinline__ int served_group(const SharedParams& p, int b) {
  if (!p.prefix_splits) return -1;
  const int group = row_group(p, b);
  if (group < 0) return -1;
  return ((long long)b - max(0, p.group_start[group]) + 1) * p.per <= p.reach ? group : -1;
}

// The prefix ranges of every group on the tensor-memory kernel; `half` chooses the type.
int shared_prefix_tc_launch(const SharedParams& p, bool half, cudaStream_t s);
int read_device_error_shared(int reset);

}  // namespace oasis
