// Management of the paged session cache: extending sequences (reserve + write),
// forking and copying them, freeing them, and compacting the pool.
//
// A page is free while refs[page] == 0. The bookkeeping is whole numbers that one
// thread block works out in order (a prefix sum over the requests' page needs and
// one over the free pages), so its result does not depend on scheduling: request i
// takes the lowest free pages that requests before it left. Then a grid over every
// SM moves the bytes, its units found from the same prefix sums on the device, so
// no call reads anything back and all of them can be captured into a graph.
//
// Bound: what is copied, read and written once (HBM), and for small calls the two
// launches; the planning block reads refs up to the last page it hands out, and takes 6
// to 7 us for its chain of searches and sums. Full copies of six sessions, 165 MB read
// and written: 40 us (4.1 TB/s); 60 forks of four sessions, 49 MB: 23 us; 24 sessions
// ended, compacted, reserved and written in four layers, twice, 356 MB: 108 us.
#include <limits.h>

#include "../../include/oasis_b200.h"
#include "common.cuh"
#include "gemm.cuh"
#include "pages.cuh"
#include "status.h"

namespace oasis {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = 16;       // pages a thread looks at per round of the free-page search
constexpr int kFewSlots = 8192;    // up to this many sequences, requests' targets are told apart in shared memory
constexpr int kCopyThreads = 256;
constexpr int kWriteVectors = 4;   // of 16 bytes, of a thread at a time
constexpr int kCounters = 16;      // [0] new pages granted, [1] pages moved, [2] live pages

struct PageArgs {
  PageGeometry g;
  uint4* pool;
  int* table;
  int* lengths;
  int* refs;
  int* status;
  int* ws;  // [kCounters][owner: slots][base: slots][len: slots][list: pages][from: pages][map: pages]
};

__device__ __forceinline__ int* ws_owner(const PageArgs& c) { return c.ws + kCounters; }
__device__ __forceinline__ int* ws_base(const PageArgs& c) { return ws_owner(c) + c.g.slots; }
__device__ __forceinline__ int* ws_len(const PageArgs& c) { return ws_base(c) + c.g.slots; }
__device__ __forceinline__ int* ws_list(const PageArgs& c) { return ws_len(c) + c.g.slots; }
__device__ __forceinline__ int* ws_from(const PageArgs& c) { return ws_list(c) + c.g.pages; }
__device__ __forceinline__ int* ws_map(const PageArgs& c) { return ws_from(c) + c.g.pages; }

size_t workspace_bytes(const PageGeometry& g) {
  return sizeof(int) * ((size_t)kCounters + 3 * (size_t)g.slots + 3 * (size_t)g.pages);
}

// Exclusive prefix sum over the block; `total` gets the sum. All threads call it.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the previous scan's readers are done with part
  if (lane == 31) part[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int p = lane < (blockDim.x >> 5) ? part[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, p, d);
      if (lane >= d) p += y;
    }
    part[lane] = p;
  }
  __syncthreads();
  *total = part[31];
  return x - v + (warp ? part[warp - 1] : 0);
}

// Grants pages to n requests, one block. FORK: request i copies sequence a[i] into
// the empty sequence b[i] (base = new pages it needs: its partial last page, or all
// of them when deep). Otherwise request i extends sequence a[i] by cu[i + 1] - cu[i]
// tokens and start[i] gets its old length (-1 where it is refused). A sequence that
// two requests name as their target goes to the lower i.
template <bool FORK>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PageArgs c, const int* __restrict__ a,
                                                            const int* __restrict__ b, const int* __restrict__ cu,
                                                            int n, int deep, int* __restrict__ start) {
  pdl_trigger();
  pdl_wait();
  __shared__ int few_owners[kFewSlots];
  const int tid = threadIdx.x;
  const int P = c.g.page_size;
  int *base = ws_base(c), *len = ws_len(c), *list = ws_list(c);
  int* owner = c.g.slots <= kFewSlots ? few_owners : ws_owner(c);
  const int* target = FORK ? b : a;
  int bad = 0;
  auto free_pages = [&](long long p) {  // of the kPlanPer pages from p on, a bit each
    unsigned mask = 0;
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k)
      if (p + k < c.g.pages && c.refs[p + k] == 0) mask |= 1u << k;
    return mask;
  };
  const unsigned first_free = free_pages((long long)tid * kPlanPer);  // on its way beside the requests
  for (int i = tid; i < n; i += kPlanThreads) {
    const int t = target[i];
    if (t >= 0 && t < c.g.slots) owner[t] = INT_MAX;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) {
    const int t = target[i];
    if (t >= 0 && t < c.g.slots) atomicMin(&owner[t], i);
  }
  __syncthreads();
  // needs, in request order
  int wanted = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int need = 0;
    if (i < n) {
      const int t = target[i];
      int keep = -1;  // tokens that the request starts from, -1: refused
      if (t < 0 || t >= c.g.slots) {
        bad |= OASIS_PAGES_BAD_SEQUENCE;
      } else if (*(volatile int*)&owner[t] != i) {
        bad |= OASIS_PAGES_IN_USE;
      } else if (FORK) {
        const int s = a[i];
        if (s < 0 || s >= c.g.slots) {
          bad |= OASIS_PAGES_BAD_SEQUENCE;
        } else if (c.lengths[t] != 0) {
          bad |= OASIS_PAGES_IN_USE;
        } else {
          keep = held_tokens(c.lengths[s], P, c.g.width);
          need = (int)pages_of(keep, P) - (deep ? 0 : keep / P);
        }
      } else {
        const long long more = (long long)cu[i + 1] - cu[i];
        const int begin = held_tokens(c.lengths[t], P, c.g.width);
        if (more < 0) {
          bad |= OASIS_PAGES_BAD_SEQUENCE;
        } else if (begin + more > (long long)c.g.width * P) {
          bad |= OASIS_PAGES_TOO_LONG;
        } else {
          keep = begin;
          need = (int)(pages_of(begin + more, P) - pages_of(begin, P));
        }
      }
      len[i] = keep;
    }
    int sum;
    const int before = block_scan(need, &sum);
    if (i < n) base[i] = wanted + before;
    wanted += sum;
  }
  // the lowest free pages, in order
  int found = 0;
  for (long long p0 = 0; p0 < c.g.pages && found < wanted; p0 += kPlanThreads * kPlanPer) {
    const long long p = p0 + (long long)tid * kPlanPer;
    const unsigned free_mask = p0 == 0 ? first_free : free_pages(p);
    int sum;
    int at = found + block_scan(__popc(free_mask), &sum);
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k)
      if (free_mask >> k & 1) {
        if (at < wanted) list[at] = (int)(p + k);
        ++at;
      }
    found += sum;
  }
  const int granted = min(found, wanted);
  __syncthreads();
  // a request that would pass the last free page, and every later one that needs a page, is refused
  for (int i = tid; i < n; i += kPlanThreads) {
    int keep = len[i];
    if (keep >= 0) {
      const int t = target[i];
      const long long more = FORK ? 0 : (long long)cu[i + 1] - cu[i];
      const int need = FORK ? (int)pages_of(keep, P) - (deep ? 0 : keep / P)
                            : (int)(pages_of(keep + more, P) - pages_of(keep, P));
      if (need > 0 && base[i] + need > granted) {
        bad |= OASIS_PAGES_NO_PAGES;
        keep = len[i] = -1;
      } else {
        c.lengths[t] = keep + (int)more;
      }
    }
    if (!FORK) start[i] = keep;
  }
  __syncthreads();
  // page k of the list belongs to the last request whose base is not above k
  for (int k = tid; k < granted; k += kPlanThreads) {
    const int i = last_not_above(base, n, k);
    if (len[i] < 0) continue;
    const int page = list[k];
    c.refs[page] = 1;
    if (!FORK) {
      const long long at = pages_of(len[i], P) + k - base[i];
      if (at >= 0 && at < c.g.width) c.table[(long long)a[i] * c.g.width + at] = page;
    }
  }
  if (bad) atomicOr(c.status, bad);
  if (tid == 0) c.ws[0] = granted;
}

// Copies the first `fill` rows of every tile of page `from` into page `to`, part
// `part` of `parts`, with the whole block.
__device__ __forceinline__ void copy_page(const PageArgs& c, int from, int to, int fill, int part, int parts) {
  const int rv = row_vectors(c.g);
  const unsigned tile = (unsigned)tile_vectors(c.g), used = (unsigned)(fill * rv);
  const long long all = (long long)page_tiles(c.g) * used;
  const long long lo = all * part / parts, hi = all * (part + 1) / parts;
  const uint4* src = c.pool + from * page_vectors(c.g);
  uint4* dst = c.pool + to * page_vectors(c.g);
  constexpr int U = 4;  // loads in flight per thread
  for (long long v0 = lo + threadIdx.x; v0 < hi; v0 += U * kCopyThreads) {
    uint4 x[U];
    long long at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long v = v0 + u * kCopyThreads;
      at[u] = -1;
      if (v < hi) {
        if (used == tile) {
          at[u] = v;
        } else {
          const unsigned w = (unsigned)v, q = w / used;  // a page has fewer than 2^32 vectors
          at[u] = (long long)q * tile + (w - q * used);
        }
        x[u] = __ldcs(src + at[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] >= 0) __stcs(dst + at[u], x[u]);
  }
}

// Parts that each of `pages` pages' copies is cut into, so that every block of the grid
// has a part, or several where there are many pages. A unit begins with a chain of
// lookups (request, sequence, table), so there should be few of them.
__device__ __forceinline__ int copy_parts(const PageArgs& c, int pages) {
  const long long want = pages > 0 ? (gridDim.x + pages - 1LL) / pages : 1, most = page_vectors(c.g) / kCopyThreads;
  const long long parts = want < 4 ? 4 : want;
  return (int)(parts < most ? parts : most < 1 ? 1 : most);
}

// After plan_kernel<true>: the targets' table rows, the shared pages' counts and
// the copies. Sources are not targets of the same call unless they were empty. A source's
// entry outside the pool is the target's too, and the page that was meant for its copy is
// free again: there is nothing to copy, and what the page holds is not the sequence's.
__global__ void __launch_bounds__(kCopyThreads) fork_kernel(PageArgs c, const int* __restrict__ src,
                                                            const int* __restrict__ dst, int n, int deep) {
  pdl_trigger();
  pdl_wait();
  const int P = c.g.page_size, W = c.g.width;
  const int *base = ws_base(c), *len = ws_len(c), *list = ws_list(c);
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int L = len[i];
    if (L < 0) continue;
    const int* from = c.table + (long long)src[i] * W;
    int* to = c.table + (long long)dst[i] * W;
    const int whole = deep ? 0 : L / P, last = (int)pages_of(L, P);
    for (int k = threadIdx.x; k < last; k += kCopyThreads) {
      int page = from[k];
      const bool ok = page_ok(page, c.g.pages);
      if (!ok) atomicOr(c.status, OASIS_PAGES_BAD_PAGE);
      if (k < whole) {
        if (ok) atomicAdd(&c.refs[page], 1);
      } else {
        const int own = list[base[i] + k - whole];
        if (ok)
          page = own;
        else
          c.refs[own] = 0;
      }
      to[k] = page;
    }
  }
  const int parts = copy_parts(c, c.ws[0]);
  const long long units = (long long)c.ws[0] * parts;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int k = (int)(u / parts);
    const int i = last_not_above(base, n, k);
    const int L = len[i];
    if (L < 0) continue;
    const int at = (deep ? 0 : L / P) + k - base[i];
    if (at >= W) continue;
    const int from = c.table[(long long)src[i] * W + at];
    if (!page_ok(from, c.g.pages)) continue;
    copy_page(c, from, list[k], min(P, L - at * P), (int)(u - (long long)k * parts), parts);
  }
}

// One block per sequence. The length is swapped for 0 by one thread, so a sequence
// that is named twice is freed once.
__global__ void __launch_bounds__(128) free_kernel(PageArgs c, const int* __restrict__ seqs, int n) {
  pdl_trigger();
  pdl_wait();
  __shared__ int held;
  const int s = seqs[blockIdx.x];
  if (s < 0 || s >= c.g.slots) {
    if (threadIdx.x == 0) atomicOr(c.status, OASIS_PAGES_BAD_SEQUENCE);
    return;
  }
  if (threadIdx.x == 0) held = atomicExch(&c.lengths[s], 0);
  __syncthreads();
  int* row = c.table + (long long)s * c.g.width;
  const int last = used_entries(held, c.g.page_size, c.g.width);
  for (int k = threadIdx.x; k < last; k += blockDim.x) {
    const int page = row[k];
    row[k] = -1;
    if (page_ok(page, c.g.pages))
      atomicSub(&c.refs[page], 1);
    else
      atomicOr(c.status, OASIS_PAGES_BAD_PAGE);
  }
}

// Pairs the k-th live page at or above the live count with the k-th hole below it.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(PageArgs c) {
  pdl_trigger();
  pdl_wait();
  const long long pages = c.g.pages;
  const long long per = (pages + kPlanThreads - 1) / kPlanThreads;
  const long long lo = min(pages, threadIdx.x * per), hi = min(pages, lo + per);
  int *to = ws_list(c), *from = ws_from(c), *map = ws_map(c);
  int mine = 0;
  for (long long p = lo; p < hi; ++p) mine += c.refs[p] > 0;
  int live;
  int seen = block_scan(mine, &live);  // live pages before this thread's
  int below = 0;
  for (long long p = lo; p < hi && p < live; ++p) below += c.refs[p] > 0;
  int low;  // live pages below the live count
  block_scan(below, &low);
  for (long long p = lo; p < hi; ++p) {
    const bool held = c.refs[p] > 0;
    if (p < live && !held) to[p - seen] = (int)p;
    if (p >= live && held) from[seen - low] = (int)p;
    seen += held;
  }
  __syncthreads();
  const int moves = live - low;
  for (int k = threadIdx.x; k < moves; k += kPlanThreads) {
    const int s = from[k], t = to[k];
    c.refs[t] = c.refs[s];
    c.refs[s] = 0;
    map[s] = t;
  }
  if (threadIdx.x == 0) {
    c.ws[1] = moves;
    c.ws[2] = live;
  }
}

__global__ void __launch_bounds__(kCopyThreads) compact_kernel(PageArgs c) {
  pdl_trigger();
  pdl_wait();
  const int moves = c.ws[1], live = c.ws[2];
  const int *to = ws_list(c), *from = ws_from(c), *map = ws_map(c);
  if (moves == 0) return;
  for (int s = blockIdx.x; s < c.g.slots; s += gridDim.x) {
    int* row = c.table + (long long)s * c.g.width;
    const int last = used_entries(c.lengths[s], c.g.page_size, c.g.width);
    for (int k = threadIdx.x; k < last; k += kCopyThreads) {
      const int page = row[k];
      if (!page_ok(page, c.g.pages)) {
        atomicOr(c.status, OASIS_PAGES_BAD_PAGE);
      } else if (page >= live) {
        const int t = map[page];
        if (t >= 0 && t < live) row[k] = t;
      }
    }
  }
  const int parts = copy_parts(c, moves);
  const long long units = (long long)moves * parts;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int k = (int)(u / parts);
    copy_page(c, from[k], to[k], c.g.page_size, (int)(u - (long long)k * parts), parts);
  }
}

// New key and value rows of one layer into their pages: four 16-byte vectors per thread,
// loaded before the chain of lookups that says where they go (9 us a layer of 18 MB with
// the loads behind it and one vector per thread),
// row r of the packed rows at position start[i] + r - cu[i] of sequence seqs[i].
// V: 1 where that many threads still fit the GPU at once, else kWriteVectors.
template <int V>
__global__ void __launch_bounds__(kCopyThreads) write_kernel(PageArgs c, int layer, const uint4* __restrict__ k,
                                                             const uint4* __restrict__ v, long long k_row,
                                                             long long k_head, long long v_row, long long v_head,
                                                             const int* __restrict__ seqs, const int* __restrict__ cu,
                                                             const int* __restrict__ start, int n, int rows) {
  pdl_trigger();
  pdl_wait();
  const int rv = row_vectors(c.g), K = c.g.kv_heads;
  const unsigned per = (unsigned)(2 * K * rv);
  const int last = min(rows, cu[n]);
  // `width` threads to a row, so `group` rows at a time; longer rows in several rounds
  const unsigned width = min((per + V - 1) / V, (unsigned)kCopyThreads), group = kCopyThreads / width;
  const unsigned in_row = threadIdx.x % width, first = threadIdx.x / width;
  if (first >= group) return;
  for (long long r0 = (long long)blockIdx.x * group + first; r0 < last; r0 += (long long)gridDim.x * group) {
    const int r = (int)r0;
    const uint4 *k_at = k + r * k_row, *v_at = v + r * v_row;
    uint4 data[V];
    auto fetch = [&](unsigned w0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const unsigned w = w0 + j * width;
        if (w >= per) continue;
        const unsigned tile_row = w / rv, d = w - tile_row * rv;  // (keys or values, head)
        data[j] = tile_row >= (unsigned)K ? v_at[(tile_row - K) * v_head + d] : k_at[tile_row * k_head + d];
      }
    };
    fetch(in_row);
    const int i = last_not_above(cu, n, r);
    const int s = seqs[i], begin = start[i];
    if (begin < 0 || s < 0 || s >= c.g.slots) continue;
    const long long pos = (long long)begin + r - cu[i];
    if (pos < begin || pos >= held_tokens(c.lengths[s], c.g.page_size, c.g.width)) continue;
    const int at = (int)(pos / c.g.page_size), slot = (int)(pos - (long long)at * c.g.page_size);
    const int page = c.table[(long long)s * c.g.width + at];
    if (!page_ok(page, c.g.pages)) {
      atomicOr(c.status, OASIS_PAGES_BAD_PAGE);
      continue;
    }
    uint4* to = c.pool + tile_offset(c.g, page, layer, 0, 0) + (long long)slot * rv;
    const long long tile = tile_vectors(c.g);
    for (unsigned w0 = in_row; w0 < per; w0 += V * width) {
      if (w0 != in_row) fetch(w0);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const unsigned w = w0 + j * width;
        if (w >= per) continue;
        const unsigned tile_row = w / rv, d = w - tile_row * rv;
        to[tile_row * tile + d] = data[j];
      }
    }
  }
}

int check_cache(const OasisPageCache* c, PageArgs* p, const char* what, bool plans) {
  OASIS_REQUIRE(c, "%s: null cache", what);
  OASIS_REQUIRE(c->pool && c->table && c->lengths && c->refs && c->status, "%s: null pointer in the cache", what);
  OASIS_REQUIRE((reinterpret_cast<uintptr_t>(c->pool) & 15) == 0, "%s: pool not 16-byte aligned", what);
  OASIS_REQUIRE(c->dtype == OASIS_DTYPE_BF16 || c->dtype == OASIS_DTYPE_F16, "%s: dtype=%d", what, c->dtype);
  OASIS_REQUIRE(c->pages >= 1 && c->layers >= 1 && c->kv_heads >= 1 && c->slots >= 1 && c->width >= 1,
                "%s: pages=%d layers=%d kv_heads=%d slots=%d width=%d", what, c->pages, c->layers, c->kv_heads,
                c->slots, c->width);
  OASIS_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && c->page_size % 16 == 0,
                "%s: page_size=%d is not a multiple of 16 up to 256", what, c->page_size);
  OASIS_REQUIRE(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0,
                "%s: head_dim=%d is not a multiple of 8 up to 256", what, c->head_dim);
  OASIS_REQUIRE((long long)c->slots * c->width < (1LL << 31) && (long long)c->width * c->page_size < (1LL << 31),
                "%s: page table of %d x %d entries is too large", what, c->slots, c->width);
  PageGeometry g;
  g.pages = c->pages;
  g.layers = c->layers;
  g.kv_heads = c->kv_heads;
  g.page_size = c->page_size;
  g.head_dim = c->head_dim;
  g.slots = c->slots;
  g.width = c->width;
  OASIS_REQUIRE((long long)c->layers * c->kv_heads < (1LL << 24) && page_vectors(g) < (1LL << 31),
                "%s: a page of %d layers x %d heads is too large", what, c->layers, c->kv_heads);
  if (plans) {
    const size_t want = workspace_bytes(g);
    if (!c->workspace || c->workspace_bytes < want)
      return set_error(OASIS_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, c->workspace_bytes, want);
    OASIS_REQUIRE((reinterpret_cast<uintptr_t>(c->workspace) & 3) == 0, "%s: workspace not 4-byte aligned", what);
  }
  p->g = g;
  p->pool = static_cast<uint4*>(c->pool);
  p->table = c->table;
  p->lengths = c->lengths;
  p->refs = c->refs;
  p->status = c->status;
  p->ws = static_cast<int*>(c->workspace);
  return OASIS_OK;
}

// Blocks that one page's copy can keep busy.
int page_parts(const PageGeometry& g) {
  const long long parts = page_vectors(g) / (4 * kCopyThreads);
  return (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
}

// Grid of a copy of at most `units` units: eight blocks of 256 threads fill an SM.
unsigned copy_blocks(long long units) {
  const long long most = 8LL * num_sms();
  return (unsigned)(units < most ? units : most);
}

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace
}  // namespace oasis

using namespace oasis;

extern "C" {

size_t oasis_pages_workspace_size(int pages, int slots) {
  if (pages < 1 || slots < 1) return 0;
  PageGeometry g;
  g.pages = pages;
  g.slots = slots;
  return workspace_bytes(g);
}

int oasis_pages_reserve(const OasisPageCache* cache, const int* seqs, const int* cu, int n, int* start,
                        oasis_stream_t stream) {
  PageArgs p;
  OASIS_TRY(check_cache(cache, &p, "pages_reserve", true));
  OASIS_REQUIRE(n >= 0 && n <= p.g.slots, "pages_reserve: n=%d requests for %d sequences", n, p.g.slots);
  if (n == 0) return OASIS_OK;
  OASIS_REQUIRE(seqs && cu && start, "pages_reserve: null pointer");
  return launched(launch_pdl(plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), p,
                             seqs, static_cast<const int*>(nullptr), cu, n, 0, start),
                  "pages_reserve");
}

int oasis_pages_write(const OasisPageCache* cache, int layer, const void* k, const void* v, long long k_row_stride,
                      long long k_head_stride, long long v_row_stride, long long v_head_stride, const int* seqs,
                      const int* cu, const int* start, int n, int rows, oasis_stream_t stream) {
  PageArgs p;
  OASIS_TRY(check_cache(cache, &p, "pages_write", false));
  OASIS_REQUIRE(layer >= 0 && layer < p.g.layers, "pages_write: layer=%d of %d", layer, p.g.layers);
  OASIS_REQUIRE(n >= 0 && n <= p.g.slots && rows >= 0, "pages_write: n=%d rows=%d", n, rows);
  if (n == 0 || rows == 0) return OASIS_OK;
  OASIS_REQUIRE(k && v && seqs && cu && start, "pages_write: null pointer");
  OASIS_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
                "pages_write: keys or values not 16-byte aligned");
  OASIS_REQUIRE(((k_row_stride | k_head_stride | v_row_stride | v_head_stride) & 7) == 0,
                "pages_write: strides %lld %lld %lld %lld are not multiples of 8 elements", k_row_stride, k_head_stride,
                v_row_stride, v_head_stride);
  const long long per = 2LL * p.g.kv_heads * row_vectors(p.g), each = per * rows > 4LL * kCopyThreads * num_sms() ? kWriteVectors : 1;
  const long long width = (per + each - 1) / each, group = width < kCopyThreads ? kCopyThreads / width : 1;  // rows of a block
  const long long blocks = (rows + group - 1) / group;
  const long long most = 16LL * num_sms();
  return launched(launch_pdl(each == 1 ? write_kernel<1> : write_kernel<kWriteVectors>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(kCopyThreads), 0,
                             static_cast<cudaStream_t>(stream), p, layer, static_cast<const uint4*>(k),
                             static_cast<const uint4*>(v), k_row_stride / 8, k_head_stride / 8, v_row_stride / 8,
                             v_head_stride / 8, seqs, cu, start, n, rows),
                  "pages_write");
}

int oasis_pages_fork(const OasisPageCache* cache, const int* src, const int* dst, int n, int deep,
                     oasis_stream_t stream) {
  PageArgs p;
  OASIS_TRY(check_cache(cache, &p, "pages_fork", true));
  OASIS_REQUIRE(n >= 0 && n <= p.g.slots, "pages_fork: n=%d requests for %d sequences", n, p.g.slots);
  if (n == 0) return OASIS_OK;
  OASIS_REQUIRE(src && dst, "pages_fork: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  OASIS_TRY(launched(launch_pdl(plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, st, p, src, dst,
                                static_cast<const int*>(nullptr), n, deep ? 1 : 0, static_cast<int*>(nullptr)),
                     "pages_fork (plan)"));
  return launched(launch_pdl(fork_kernel, dim3(copy_blocks((long long)n * (deep ? p.g.width : 1) * page_parts(p.g))),
                             dim3(kCopyThreads), 0, st, p, src, dst, n, deep ? 1 : 0),
                  "pages_fork");
}

int oasis_pages_free(const OasisPageCache* cache, const int* seqs, int n, oasis_stream_t stream) {
  PageArgs p;
  OASIS_TRY(check_cache(cache, &p, "pages_free", false));
  OASIS_REQUIRE(n >= 0 && n <= p.g.slots, "pages_free: n=%d requests for %d sequences", n, p.g.slots);
  if (n == 0) return OASIS_OK;
  OASIS_REQUIRE(seqs, "pages_free: null pointer");
  return launched(
      launch_pdl(free_kernel, dim3(n), dim3(128), 0, static_cast<cudaStream_t>(stream), p, seqs, n), "pages_free");
}

int oasis_pages_compact(const OasisPageCache* cache, oasis_stream_t stream) {
  PageArgs p;
  OASIS_TRY(check_cache(cache, &p, "pages_compact", true));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  OASIS_TRY(launched(launch_pdl(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p), "pages_compact (plan)"));
  return launched(launch_pdl(compact_kernel, dim3(copy_blocks((long long)(p.g.pages / 2 + 1) * page_parts(p.g))),
                             dim3(kCopyThreads), 0, st, p),
                  "pages_compact");
}

}  // extern "C"
