// Index arithmetic of the paged session cache, usable on the host and the device
// (a plain C++ compiler reads this file too).
//
// Pool: [pages][layers][2][kv_heads][page_size][head_dim] 2-byte elements, so a
// page is one contiguous block and a (page, layer, k or v, head) tile is
// page_size consecutive rows. Table row of a sequence: its pages in order;
// lengths[s] tokens are held, so ceil(length / page_size) entries count. Every
// entry and length read from device memory is checked against its bounds before
// it becomes an address.
#pragma once

#if defined(__CUDACC__)
#define OASIS_HD __host__ __device__ inline
#else
#define OASIS_HD inline
#endif

namespace oasis {

struct PageGeometry {
  int pages = 0, layers = 0, kv_heads = 0, page_size = 0, head_dim = 0;
  int slots = 0, width = 0;  // page table [slots][width]
};

// Pages that `tokens` tokens take (0 for a negative count).
OASIS_HD long long pages_of(long long tokens, int page_size) {
  return tokens > 0 ? (tokens + page_size - 1) / page_size : 0;
}

// Entries of a table row that a stored length makes valid: never more than the row.
OASIS_HD int used_entries(int length, int page_size, int width) {
  const long long p = pages_of(length, page_size);
  return p < width ? (int)p : width;
}

// Tokens of a row that may be read: a stored length clipped to what the row holds.
OASIS_HD int held_tokens(int length, int page_size, int width) {
  const long long room = (long long)width * page_size;
  return length < 0 ? 0 : (length < room ? length : (int)room);
}

OASIS_HD bool page_ok(int page, int pages) { return page >= 0 && page < pages; }

// 16-byte vectors of one page's (layer, k or v, head) tile row, tile and page.
OASIS_HD int row_vectors(const PageGeometry& g) { return g.head_dim / 8; }
OASIS_HD long long tile_vectors(const PageGeometry& g) { return (long long)g.page_size * row_vectors(g); }
OASIS_HD int page_tiles(const PageGeometry& g) { return g.layers * 2 * g.kv_heads; }
OASIS_HD long long page_vectors(const PageGeometry& g) { return page_tiles(g) * tile_vectors(g); }

// Vector offset in the pool of the first row of a tile (which: 0 keys, 1 values).
OASIS_HD long long tile_offset(const PageGeometry& g, int page, int layer, int which, int head) {
  return page * page_vectors(g) + ((long long)(layer * 2 + which) * g.kv_heads + head) * tile_vectors(g);
}

// The last index i in [0, n) with starts[i] <= at, for non-decreasing starts with
// starts[0] <= at; 0 where there is none. Stays inside [0, n) whatever starts holds.
OASIS_HD int last_not_above(const int* starts, int n, int at) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (starts[mid] <= at)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

}  // namespace oasis
