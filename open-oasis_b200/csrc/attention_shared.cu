// Attention of one query per row over the paged cache, for batches whose rows share a
// prefix. Row b, head h, sequence s = seqs[b] with length t:
//   o = sum_{j < t} exp(x_j - m) v_j / sum_{j < t} exp(x_j - m),  x_j = scale q . k_j,  m = max x_j
// Keys split into ranges; a range gives (m_r, l_r, o~_r) with l_r and o~_r relative to
// its own maximum, and ranges join as m = max m_r, l = sum l_r e^(m_r - m),
// o = sum e^(m_r - m) o~_r / l.
//
// shared_prefix_kernel: the keys that a group's rows have in common, read once for all
// of them: 64 (row, head) queries of one key head per block, 64 keys a step, mma.sync; for
// short prefixes (attention_shared_tc.cu has the others). Bound by latency: a block of few
// steps loads its rows' lengths, the table and the keys one behind the other.
// shared_own_kernel: each row's keys behind the prefix: four warps (or one) per (row, key
// head, range), 16 keys a step, the heads of a key head as the eight columns of a fragment.
// The least is reading the keys and values once: 32 rows of up to 4096 tokens, 32 / 8 heads
// of 128, 97 MB: 29 us (3.4 TB/s) with the join; a block's lookups before its first load,
// two steps of keys in flight per warp and the rows' different lengths are the rest. It
// runs beside the prefix kernel. With one range it joins the prefix's and
// writes the result; otherwise shared_join_kernel does, a warp per (row, head).
// 64 rows behind 8192 shared tokens, up to 1024 own ones, 32 / 8 heads of 128: 48 us, about
// 25 for the prefix, the own keys beside and behind it and 8 to 10 for the join; the bytes
// alone would take 10.
// shared_whole_kernel: both in one pass where rows are many and short.
// Small batches run the own kernel alone, their prefixes read with the rows' own keys.
#include "../../include/oasis_b200.h"
#include "attention_rows.cuh"
#include "attention_shared.cuh"
#include "gemm.cuh"
#include "status.h"

namespace oasis {
namespace {

constexpr int kPrefixRows = 64;     // (row, head) queries of a block
constexpr int kPrefixKeys = 64;     // keys of a step
constexpr int kWholeRows = 32;      // queries of a block of the one-pass kernel
constexpr int kThreads = 128;
constexpr int kOwnWarps = 4;
// Prefixes of at least this many tokens run on the tensor-memory kernel. Where each of its
// blocks has at most 64 of its 256 queries and they come in several waves (an SM holds
// one), it is one token more for each block behind the first wave, up to the second
// number. Tensor memory / mma.sync, us, own keys included: 8 groups of up to 128 rows, 16
// heads of 64: 46.7 / 46.0 for up to 128 tokens, 47.3 / 48.1 for 256, 61.5 / 90.9 for 2048;
// 32 / 8 heads of 128: 49.7 / 47.8, 51.8 / 56.7, 77 / 182. 36 groups of up to 16 rows, 16
// heads of 64: 60.4 / 41.5 for 256, 63.3 / 53.0 for 512, 77 / 121 for 2048; 20 groups of up to
// 8 rows: 39.3 / 42.7 for 500.
constexpr int kTensorKeys = 256, kTensorKeysMost = 700;
constexpr int kMostSplits = 64;    // of a prefix, and of a row's own keys
constexpr int kMostRanges = 2 * kMostSplits;

template <int D>
constexpr int prefix_smem() {
  return (kPrefixRows + 4 * kPrefixKeys) * D * 2;
}
template <int D>
constexpr int whole_smem() {
  return (kWholeRows + 4 * kPrefixKeys) * D * 2;  // Q, then two steps' K and V or four rings of two units
}
template <int D>
constexpr int own_smem() {
  return kOwnWarps * 4 * kUnit * D * 2;
}

// One running-softmax step of a warp: 16 queries x 16 keys. `see(e, key)` masks; x
// holds the scores of key tiles 0 and 1 in fragment order and becomes P.
struct Running {
  float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
};

template <typename T>
__device__ __forceinline__ void softmax_step(float (&x)[2][4], Running& r, float& fa, float& fb, uint32_t (&pa)[4]) {
  float na = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
  float nb = fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3]));
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    na = fmaxf(na, __shfl_xor_sync(0xffffffffu, na, w));
    nb = fmaxf(nb, __shfl_xor_sync(0xffffffffu, nb, w));
  }
  na = fmaxf(na, r.ma);
  nb = fmaxf(nb, r.mb);
  float sa = softmax_shift(na), sb = softmax_shift(nb);
  fa = ex2_approx(r.ma - sa);
  fb = ex2_approx(r.mb - sb);
  sa -= kLift<T>;
  sb -= kLift<T>;
  r.ma = na;
  r.mb = nb;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    x[t][0] = ex2_approx(x[t][0] - sa);
    x[t][1] = ex2_approx(x[t][1] - sa);
    x[t][2] = ex2_approx(x[t][2] - sb);
    x[t][3] = ex2_approx(x[t][3] - sb);
  }
  r.la = r.la * fa + ((x[0][0] + x[0][1]) + (x[1][0] + x[1][1]));  // this lane's share
  r.lb = r.lb * fb + ((x[0][2] + x[0][3]) + (x[1][2] + x[1][3]));
  // P as the 16-bit operand: the one rounding inside the sum
  pa[0] = Elem<T>::pack(x[0][0], x[0][1]);
  pa[1] = Elem<T>::pack(x[0][2], x[0][3]);
  pa[2] = Elem<T>::pack(x[1][0], x[1][1]);
  pa[3] = Elem<T>::pack(x[1][2], x[1][3]);
}

template <typename T, int D>
__device__ __forceinline__ void scores(const uint8_t* sk, int row0, const uint32_t (&qa)[D / 16][4], float (&x)[2][4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    uint32_t b[4];
    ldsm_x4(b, sk + tile_at<D>(row0 + (lane & 7) + ((lane >> 4) << 3), s * 2 + ((lane >> 3) & 1)));
    Elem<T>::mma(x[0], qa[s], b[0], b[1]);
    Elem<T>::mma(x[1], qa[s], b[2], b[3]);
  }
}

template <typename T, int D>
__device__ __forceinline__ void add_values(const uint8_t* sv, int row0, const uint32_t (&pa)[4], float fa, float fb,
                                           float (&o)[D / 8][4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int t = 0; t < D / 8; t += 2) {
    uint32_t b[4];
    ldsm_x4_t(b, sv + tile_at<D>(row0 + (lane & 15), t + (lane >> 4)));
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      o[t + u][0] *= fa;
      o[t + u][1] *= fa;
      o[t + u][2] *= fb;
      o[t + u][3] *= fb;
      Elem<T>::mma(o[t + u], pa, b[2 * u], b[2 * u + 1]);
    }
  }
}

__device__ __forceinline__ void join_lanes(Running& r) {
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    r.la += __shfl_xor_sync(0xffffffffu, r.la, w);
    r.lb += __shfl_xor_sync(0xffffffffu, r.lb, w);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) shared_prefix_kernel(SharedParams p) {
  constexpr int CH = D / 8, KS = D / 16, NT = D / 8, TILE = kPrefixKeys * D * 2;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int limit[kPrefixRows];  // keys that a query sees; -1: no query
  __shared__ int lead_len[4], lead_row[4];
  __shared__ int unit_ok[2][4];
  pdl_wait();
  pdl_trigger();  // behind the wait: the kernel of the own keys starts without one
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int x = blockIdx.x;
  const int tile = x % p.tiles;
  x /= p.tiles;
  const int split = x % p.prefix_splits;
  x /= p.prefix_splits;
  const int kvh = x % p.g.kv_heads, group = x / p.g.kv_heads;
  const int b0 = max(0, p.group_start[group]), b1 = min(p.rows, p.group_start[group + 1]);
  const int P = p.g.page_size;
  const int tokens = group_tokens(p, group);
  const long long queries = (long long)max(0, b1 - b0) * p.per;
  if ((long long)tile * kPrefixRows >= queries) return;

  // The prefix is read through the table row of the longest sequence (the first of
  // them): a shorter one need not have all of its pages.
  int len = -1, row = b1;
  for (int b = b0 + tid; b < b1; b += kThreads) {
    int s;
    const int t = row_length(p, b, &s);
    if (t > len) {
      len = t;
      row = b;
    }
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    const int l2 = __shfl_xor_sync(0xffffffffu, len, w), r2 = __shfl_xor_sync(0xffffffffu, row, w);
    if (l2 > len || (l2 == len && r2 < row)) {
      len = l2;
      row = r2;
    }
  }
  if (lane == 0) {
    lead_len[warp] = len;
    lead_row[warp] = row;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (lead_len[w] > len || (lead_len[w] == len && lead_row[w] < row)) {
      len = lead_len[w];
      row = lead_row[w];
    }
  const int common = min(tokens, len);  // whole and valid pages but for the last
  const int* lead = p.table + (long long)(len > 0 ? p.seqs[row] : 0) * p.g.width;
  const int units = (max(common, 0) + kUnit - 1) / kUnit;
  const int u0 = (int)((long long)units * split / p.prefix_splits), u1 = (int)((long long)units * (split + 1) / p.prefix_splits);
  const int steps = (u1 - u0 + 3) / 4;

  for (long long m0 = (long long)tile * kPrefixRows; m0 < queries; m0 += (long long)p.tiles * kPrefixRows) {
    __syncthreads();
    const Queries at(m0, p.per);
    if (tid < kPrefixRows) {
      int lim = -1, s;
      if (m0 + tid < queries) lim = min(common, row_length(p, b0 + (int)at.row_of(tid), &s));
      limit[tid] = lim;
    }
    const T* q = static_cast<const T*>(p.q);
    for (int i = tid; i < kPrefixRows * CH; i += kThreads) {
      const int r = i / CH, c = i % CH;
      const bool ok = m0 + r < queries;
      const long long b = b0 + at.row_of(ok ? r : 0);
      const int h = kvh * p.per + at.head_of(ok ? r : 0);
      cp_async16(sm + tile_at<D>(r, c), q + b * p.q_row + h * p.q_head + c * 8, ok);
    }
    auto load = [&](int j) {
      uint8_t* kd = sm + kPrefixRows * D * 2 + (j & 1) * 2 * TILE;
      const uint4* pool = static_cast<const uint4*>(p.pool);
      for (int i = tid; i < kPrefixKeys * CH; i += kThreads) {
        const int r = i / CH, c = i % CH;
        const int u = u0 + j * 4 + r / kUnit;
        const int t = u * kUnit;
        const int page = u < u1 ? lead[t / P] : -1;
        const bool ok = page_ok(page, p.g.pages);
        const bool in = ok && t + r % kUnit < common;  // rows behind the sequences hold anything: zero instead
        const long long at = tile_offset(p.g, ok ? page : 0, p.layer, 0, kvh) + (long long)(t % P + r % kUnit) * CH + c;
        cp_async16(kd + tile_at<D>(r, c), pool + at, in);
        cp_async16(kd + TILE + tile_at<D>(r, c), pool + at + p.g.kv_heads * tile_vectors(p.g), in);
        if (c == 0 && r % kUnit == 0) {
          unit_ok[j & 1][r / kUnit] = ok;
          if (!ok && u < u1) atomicOr(p.status, OASIS_PAGES_BAD_PAGE);
        }
      }
      cp_async_commit();
    };
    if (steps > 0) load(0);
    const int wr = warp * 16, ra = wr + (lane >> 2);
    uint32_t qa[KS][4];
    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    Running run;
    int lim_a = -1, lim_b = -1;
    for (int j = 0; j < steps; ++j) {
      if (j + 1 < steps) {
        load(j + 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      if (j == 0) {
#pragma unroll
        for (int s = 0; s < KS; ++s) ldsm_x4(qa[s], sm + tile_at<D>(wr + (lane & 15), s * 2 + (lane >> 4)));
        lim_a = limit[ra];
        lim_b = limit[ra + 8];
      }
      const uint8_t* sk = sm + kPrefixRows * D * 2 + (j & 1) * 2 * TILE;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (!unit_ok[j & 1][h]) continue;
        const int kb = (u0 + j * 4 + h) * kUnit;
        float s[2][4] = {};
        scores<T, D>(sk, h * kUnit, qa, s);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = kb + t * 8 + (lane & 3) * 2 + (e & 1);
            s[t][e] = key < (e < 2 ? lim_a : lim_b) ? s[t][e] * p.scale_log2 : -INFINITY;
          }
        float fa, fb;
        uint32_t pa[4];
        softmax_step<T>(s, run, fa, fb, pa);
        add_values<T, D>(sk + TILE, h * kUnit, pa, fa, fb, o);
      }
      __syncthreads();
    }
    cp_async_wait_all();  // a range without keys has only Q in flight
    join_lanes(run);
    const int splits = p.prefix_splits + p.own_splits;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (m0 + ra + half * 8 >= queries) continue;
      const long long b = b0 + at.row_of(ra + half * 8);
      const int h = kvh * p.per + at.head_of(ra + half * 8);
      const long long slot = (b * p.heads + h) * splits + split;
      const float mm = half ? run.mb : run.ma, ll = half ? run.lb : run.la;
      if ((lane & 3) == 0) p.part_ml[slot] = make_float2(mm - kLift<T>, ll);
      if (mm == -INFINITY && ll == 0.f) continue;  // nothing in this range: its sums are not read
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<float2*>(p.part_o + slot * D + t * 8 + (lane & 3) * 2) =
            make_float2(o[t][2 * half], o[t][2 * half + 1]);
    }
  }
}

// Steps of a warp with eight queries as the columns of the product and 16 keys as its
// rows: a row of the batch has few heads to a key head, so that the other way round most
// of a fragment's 16 query rows would be idle through the softmax. A lane holds columns
// 2 (lane % 4) and the next of S^T (keys x queries) and of O^T (dims x queries).
template <int D>
struct Columns {
  float m[2], l[2];  // l: this lane's keys' share until join()
  float o[D / 16][4];
  __device__ __forceinline__ Columns() {
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
  }
  __device__ __forceinline__ void join() {
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], w);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], w);
    }
  }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The 16 keys at rows row0 of a tile, the first of them key `key0`; a column sees keys
// below its limit. `fresh`: the columns that see any have no keys yet.
template <typename T, int D>
__device__ __forceinline__ void column_step(Columns<D>& c, const uint8_t* sk, const uint8_t* sv, int row0, int key0,
                                            const uint32_t (&qb)[D / 16][2], int lim_a, int lim_b, bool fresh,
                                            float scale_log2) {
  const int lane = threadIdx.x & 31;
  float x[4] = {};
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    uint32_t a[4];
    ldsm_x4(a, sk + tile_at<D>(row0 + (lane & 15), s * 2 + (lane >> 4)));
    Elem<T>::mma(x, a, qb[s][0], qb[s][1]);
  }
  const int key = key0 + (lane >> 2);
  if (key >= lim_a) x[0] = -INFINITY;
  if (key >= lim_b) x[1] = -INFINITY;
  if (key + 8 >= lim_a) x[2] = -INFINITY;
  if (key + 8 >= lim_b) x[3] = -INFINITY;
  float na = fmaxf(x[0], x[2]) * scale_log2, nb = fmaxf(x[1], x[3]) * scale_log2;
#pragma unroll
  for (int w = 4; w < 32; w <<= 1) {
    na = fmaxf(na, __shfl_xor_sync(0xffffffffu, na, w));
    nb = fmaxf(nb, __shfl_xor_sync(0xffffffffu, nb, w));
  }
  na = fmaxf(na, c.m[0]);
  nb = fmaxf(nb, c.m[1]);
  float sa = softmax_shift(na), sb = softmax_shift(nb);
  const float fa = ex2_approx(c.m[0] - sa), fb = ex2_approx(c.m[1] - sb);
  sa -= kLift<T>;
  sb -= kLift<T>;
  c.m[0] = na;
  c.m[1] = nb;
  x[0] = ex2_approx(fmaf(x[0], scale_log2, -sa));
  x[1] = ex2_approx(fmaf(x[1], scale_log2, -sb));
  x[2] = ex2_approx(fmaf(x[2], scale_log2, -sa));
  x[3] = ex2_approx(fmaf(x[3], scale_log2, -sb));
  c.l[0] = c.l[0] * fa + (x[0] + x[2]);
  c.l[1] = c.l[1] * fb + (x[1] + x[3]);
  // P^T (keys x queries) turned into the second operand: the one rounding inside the sum
  const uint32_t b0 = transpose8(Elem<T>::pack(x[0], x[1])), b1 = transpose8(Elem<T>::pack(x[2], x[3]));
#pragma unroll
  for (int t = 0; t < D / 16; ++t) {
    uint32_t a[4];
    ldsm_x4_t(a, sv + tile_at<D>(row0 + (lane & 7) + ((lane >> 4) << 3), t * 2 + ((lane >> 3) & 1)));
    if (!fresh) {
      c.o[t][0] *= fa;
      c.o[t][1] *= fb;
      c.o[t][2] *= fa;
      c.o[t][3] *= fb;
    }
    Elem<T>::mma(c.o[t], a, b0, b1);
  }
}

// A row's result where the joined ranges are not finite: key by key, so that masked
// places, sums that overflow and the formula's own NaN come out as they should; zeros where
// no page of it lies in the pool. Whole warp.
template <typename T, int D>
__device__ __noinline__ void row_again(const SharedParams& p, int b, int h) {
  int s;
  const int len = row_length(p, b, &s), lane = threadIdx.x & 31, P = p.g.page_size;
  const int* table = p.table + (long long)s * p.g.width;
  const T* pool = static_cast<const T*>(p.pool);
  const int kvh = h / p.per;
  auto at = [&](long long j, int which) -> const T* {
    const int page = table[j / P];
    if (!page_ok(page, p.g.pages)) return nullptr;
    return pool + (tile_offset(p.g, page, p.layer, which, kvh) + (j % P) * (D / 8)) * 8;
  };
  float acc[D / 32];
  row_by_keys<T, D, 4>(static_cast<const T*>(p.q) + b * p.q_row + h * p.q_head, p.scale_log2, len,
                    [&](long long j) { return at(j, 0); }, [&](long long j) { return at(j, 1); }, acc);
  T* out = static_cast<T*>(p.out) + b * p.o_row + h * p.o_head;
#pragma unroll
  for (int d = 0; d < D / 32; d += 2)
    *reinterpret_cast<uint32_t*>(out + lane * (D / 32) + d) = Elem<T>::pack(acc[d], acc[d + 1]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kOwnWarps * 32) shared_own_kernel(SharedParams p) {
  constexpr int CH = D / 8, KS = D / 16, MT = D / 16, TILE = kUnit * D * 2;
  extern __shared__ __align__(128) uint8_t sm[];
  // Behind a prefix kernel this one starts when every block of that one is past its own
  // wait, so that all before it is done; its ranges are waited for where they are joined.
  pdl_trigger();
  if (!p.prefix_splits) pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = sm + warp * 4 * TILE;
  // an item is a warp's, or a team of four warps takes its units in turn
  const int member = p.team > 1 ? warp : 0;
  long long x = p.team > 1 ? (long long)blockIdx.x : (long long)blockIdx.x * kOwnWarps + warp;
  // every row's first range comes before the second ones, which few rows may have
  const int ht = (int)(x % p.head_tiles);
  x /= p.head_tiles;
  const int kvh = (int)(x % p.g.kv_heads);
  x /= p.g.kv_heads;
  const int split = (int)(x / p.rows), b = (int)(x % p.rows);
  if (split >= p.own_splits) {  // whole warps, and whole teams
    pdl_wait();
    return;
  }
  int s = p.seqs[b];
  const int P = p.g.page_size;
  const bool known = s >= 0 && s < p.g.slots;
  const int len = known ? held_tokens(p.lengths[s], P, p.g.width) : 0;
  if (split > 0 && (long long)split * p.own_units * kUnit >= len) {  // not even without a prefix
    pdl_wait();
    return;
  }
  const int group = served_group(p, b);
  const int begin = group_tokens(p, group);
  if (!known) {
    if (lane == 0) atomicOr(p.status, OASIS_PAGES_BAD_SEQUENCE);
    s = 0;
  }
  const int units = len > begin ? (len - begin + kUnit - 1) / kUnit : 0;
  const int u0 = min(units, split * p.own_units), u1 = split + 1 < p.own_splits ? min(units, u0 + p.own_units) : units;
  if (split > 0 && u0 == units) {  // a shorter row has fewer ranges
    pdl_wait();
    return;
  }
  const int* table = p.table + (long long)s * p.g.width;
  const uint4* pool = static_cast<const uint4*>(p.pool);
  const int nh = min(8, p.per - ht * 8), h0 = kvh * p.per + ht * 8;  // heads: the columns

  unsigned ok_bits = 0;  // of the two units in flight
  auto load = [&](int u, int n) {
    uint8_t* kd = ring + (n & 1) * 2 * TILE;
    const int t = begin + u * kUnit;
    const int page = table[t / P];
    const bool ok = page_ok(page, p.g.pages);
    ok_bits = (ok_bits & ~(1u << (n & 1))) | ((unsigned)ok << (n & 1));
    if (!ok && lane == 0) atomicOr(p.status, OASIS_PAGES_BAD_PAGE);
    const long long at = tile_offset(p.g, ok ? page : 0, p.layer, 0, kvh) + (long long)(t % P) * CH;
    const long long to_v = p.g.kv_heads * tile_vectors(p.g);
#pragma unroll
    for (int i = 0; i < kUnit * CH / 32; ++i) {
      const int y = i * 32 + lane, r = y / CH, c = y % CH;
      const bool in = ok && t + r < len;  // rows behind the sequence hold anything: zero instead
      cp_async16(kd + tile_at<D>(r, c), pool + at + y, in);
      cp_async16(kd + TILE + tile_at<D>(r, c), pool + at + to_v + y, in);
    }
    cp_async_commit();
  };
  if (u0 + member < u1) load(u0 + member, 0);

  const int ca = (lane & 3) * 2;  // this lane's columns: ca and ca + 1
  const T* q = static_cast<const T*>(p.q) + b * p.q_row + h0 * p.q_head;
  uint32_t qb[KS][2];
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = lane >> 2, c = k * 16 + e * 8 + (lane & 3) * 2;
      qb[k][e] = r < nh ? *reinterpret_cast<const uint32_t*>(q + r * p.q_head + c) : 0u;
    }
  Columns<D> run;
  for (int u = u0 + member, n = 0; u < u1; u += p.team, ++n) {
    if (u + p.team < u1) {
      load(u + p.team, n + 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncwarp();
    if (ok_bits >> (n & 1) & 1) {
      const uint8_t* sk = ring + (n & 1) * 2 * TILE;
      column_step<T, D>(run, sk, sk + TILE, 0, begin + u * kUnit, qb, len, len, n == 0, p.scale_log2);
    }
    __syncwarp();  // the stage may be loaded again
  }
  run.join();

  if (p.team > 1) {  // the team's sums, in fragment order, to its first warp
    float* mine = reinterpret_cast<float*>(ring) + lane;
    __shared__ float4 stats[kOwnWarps][32];
    if (member > 0) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[(t * 4 + e) * 32] = run.o[t][e];
      stats[member][lane] = make_float4(run.m[0], run.m[1], run.l[0], run.l[1]);
    }
    __syncthreads();
    if (member > 0) {
      pdl_wait();
      return;
    }
    float ma = run.m[0], mb = run.m[1];
#pragma unroll
    for (int w = 1; w < kOwnWarps; ++w) {
      ma = fmaxf(ma, stats[w][lane].x);
      mb = fmaxf(mb, stats[w][lane].y);
    }
    const float sa = softmax_shift(ma), sb = softmax_shift(mb);
    const float ka = ex2_approx(run.m[0] - sa), kb = ex2_approx(run.m[1] - sb);
    run.l[0] *= ka;
    run.l[1] *= kb;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      run.o[t][0] *= ka;
      run.o[t][1] *= kb;
      run.o[t][2] *= ka;
      run.o[t][3] *= kb;
    }
#pragma unroll
    for (int w = 1; w < kOwnWarps; ++w) {
      const float4 st = stats[w][lane];
      const float fa = ex2_approx(st.x - sa), fb = ex2_approx(st.y - sb);
      run.l[0] = fmaf(st.z, fa, run.l[0]);
      run.l[1] = fmaf(st.w, fb, run.l[1]);
      const float* other = reinterpret_cast<const float*>(sm + w * 4 * TILE) + lane;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        run.o[t][0] = fmaf(other[(t * 4 + 0) * 32], fa, run.o[t][0]);
        run.o[t][1] = fmaf(other[(t * 4 + 1) * 32], fb, run.o[t][1]);
        run.o[t][2] = fmaf(other[(t * 4 + 2) * 32], fa, run.o[t][2]);
        run.o[t][3] = fmaf(other[(t * 4 + 3) * 32], fb, run.o[t][3]);
      }
    }
    run.m[0] = ma;
    run.m[1] = mb;
  }

  const int splits = p.prefix_splits + p.own_splits;
  const int dim = lane >> 2;  // of a 16-dim tile: this one and the one eight behind it
  if (p.own_splits > 1) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (ca + half >= nh) continue;
      const long long slot = ((long long)b * p.heads + h0 + ca + half) * splits + p.prefix_splits + split;
      if (dim == 0) p.part_ml[slot] = make_float2(run.m[half] - kLift<T>, run.l[half]);
      if (run.m[half] == -INFINITY && run.l[half] == 0.f) continue;  // its sums are not read
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        p.part_o[slot * D + t * 16 + dim] = run.o[t][half];
        p.part_o[slot * D + t * 16 + dim + 8] = run.o[t][half + 2];
      }
    }
    pdl_wait();  // nobody ends before the prefix kernel does: what follows waits for this one alone
    return;
  }
  // the prefix ranges of these heads join here, each relative to its maximum less its lift
  pdl_wait();
  unsigned bad = 0;
  float inv[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const bool mine = ca + half < nh;
    const long long slot = ((long long)b * p.heads + h0 + (mine ? ca + half : 0)) * splits;
    const float m = run.m[half] - kLift<T>;
    float l = run.l[half];
    if (group >= 0 && mine) {
      // the joint maximum first, so that the ranges' loads do not wait for one another
      float top = m;
#pragma unroll 4
      for (int i = 0; i < p.prefix_splits; ++i) top = fmaxf(top, p.part_ml[slot + i].x);
      const float sh = softmax_shift(top), fo = ex2_approx(m - sh);
      l *= fo;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        run.o[t][half] *= fo;
        run.o[t][half + 2] *= fo;
      }
#pragma unroll 4
      for (int i = 0; i < p.prefix_splits; ++i) {
        const float2 ml = p.part_ml[slot + i];
        const float f = ex2_approx(ml.x - sh);
        l = fmaf(ml.y, f, l);
        const bool some = !(ml.x == -INFINITY && ml.y == 0.f);  // its sums were written
        const float* y = p.part_o + (slot + i) * D + dim;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          run.o[t][half] = fmaf(some ? y[t * 16] : 0.f, f, run.o[t][half]);
          run.o[t][half + 2] = fmaf(some ? y[t * 16 + 8] : 0.f, f, run.o[t][half + 2]);
        }
      }
    }
    inv[half] = len > 0 ? 1.f / l : 0.f;  // an empty sequence gives zeros
    bool ok = len == 0 || (l > 0.f && finite_f(l));
#pragma unroll
    for (int t = 0; t < MT; ++t) ok = ok && finite_f(run.o[t][half]) && finite_f(run.o[t][half + 2]);
    const unsigned votes = __ballot_sync(0xffffffffu, mine && !ok);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (votes & (0x11111111u << i)) bad |= 1u << (2 * i + half);
  }
  // O^T turned back, a pair of dims of query lane / 4 in a register
  T* out = static_cast<T*>(p.out) + b * p.o_row + (h0 + (lane >> 2)) * p.o_head + ca;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t y = transpose8(Elem<T>::pack(run.o[t][2 * e] * inv[0], run.o[t][2 * e + 1] * inv[1]));
      if ((lane >> 2) < nh) *reinterpret_cast<uint32_t*>(out + t * 16 + e * 8) = y;
    }
  __syncwarp();
  for (int r = 0; bad >> r; ++r)
    if (bad >> r & 1) row_again<T, D>(p, b, h0 + r);
}

// Prefix and own keys in one pass, for many rows with few keys each (forks of a short
// prompt: a group per patch, a few frames behind it): 32 (row, head) queries of one key
// head per block, whatever groups they belong to. First each warp goes through the own
// keys of its eight queries' rows, 16 keys at a time: the product is taken with all eight
// and the other rows' scores are masked, so that the softmax and O stay in one fragment;
// a row's first 16 keys find its O empty and need no rescaling. Then each
// group's prefix is read once for the rows of the tile that are in it. Bound by issue:
// about 200 instructions for each row's 16 keys, and by the latency of their loads.
// 9216 rows in 144 groups, 16 + up to 16 tokens each, 16 heads of 64, 255 MB: 108 us (2.4
// TB/s; one warp per row and head in two kernels 124 us). 64 queries and 8 warps a block,
// for groups of 16 rows: 35 -> 45 us.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, D == 64 ? 6 : 3) shared_whole_kernel(SharedParams p) {
  constexpr int CH = D / 8, KS = D / 16, MT = D / 16, TILE = kPrefixKeys * D * 2, UNIT = kUnit * D * 2;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int row_of[kWholeRows];    // row of a query, -1: none
  __shared__ int seq_of[kWholeRows];    // its sequence
  __shared__ int len_of[kWholeRows];    // its tokens
  __shared__ int begin_of[kWholeRows];  // its first own token
  __shared__ int page_of[kWholeRows];   // and that token's page
  __shared__ int group_of[kWholeRows];
  __shared__ int near_starts[kThreads];  // group starts from the first query's group on
  __shared__ int lead_len[4], lead_row[4];
  __shared__ int unit_ok[2][4];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % p.g.kv_heads;
  const long long m0 = (long long)(blockIdx.x / p.g.kv_heads) * kWholeRows, queries = (long long)p.rows * p.per;
  const Queries at_query(m0, p.per);
  const int P = p.g.page_size;
  const uint4* pool = static_cast<const uint4*>(p.pool);
  const long long to_v = p.g.kv_heads * tile_vectors(p.g);
  const T* q = static_cast<const T*>(p.q);
  for (int i = tid; i < kWholeRows * CH; i += kThreads) {
    const int r = i / CH, c = i % CH;
    const bool ok = m0 + r < queries;
    const long long b = at_query.row_of(ok ? r : 0);
    const int h = kvh * p.per + at_query.head_of(ok ? r : 0);
    cp_async16(sm + tile_at<D>(r, c), q + b * p.q_row + h * p.q_head + c * 8, ok);
  }
  const int g0 = max(0, row_group(p, (int)at_query.row));
  near_starts[tid] = p.groups > 0 ? p.group_start[min(g0 + tid, p.groups)] : 0;
  __syncthreads();
  if (tid < kWholeRows) {
    int b = -1, s = 0, len = 0, group = -1, begin = 0;
    if (m0 + tid < queries) {
      b = (int)at_query.row_of(tid);
      len = row_length(p, b, &s);
      if (s < 0 || s >= p.g.slots) {
        atomicOr(p.status, OASIS_PAGES_BAD_SEQUENCE);
        s = 0;
      }
      if (p.groups > 0) {
        const int k = last_not_above(near_starts, kThreads, b);
        if (k + 1 < kThreads && near_starts[k] <= b && near_starts[k + 1] > b && g0 + k < p.groups)
          group = g0 + k;
        else if (p.group_start[0] <= b && p.group_start[p.groups] > b)  // behind the starts at hand
          group = last_not_above(p.group_start, p.groups, b);
      }
      begin = group_tokens(p, group);
    }
    row_of[tid] = b;
    seq_of[tid] = s;
    len_of[tid] = len;
    begin_of[tid] = begin;
    group_of[tid] = group;
    page_of[tid] = len > begin ? p.table[(long long)s * p.g.width + begin / P] : -1;
  }
  cp_async_wait_all();
  __syncthreads();

  const int wr = warp * 8, ca = wr + (lane & 3) * 2, cb = ca + 1;  // this warp's queries, this lane's columns
  uint32_t qb[KS][2];
#pragma unroll
  for (int s = 0; s < KS; s += 2) {
    uint32_t r[4];
    ldsm_x4(r, sm + tile_at<D>(wr + (lane & 7), s * 2 + (lane >> 3)));
    qb[s][0] = r[0];
    qb[s][1] = r[1];
    qb[s + 1][0] = r[2];
    qb[s + 1][1] = r[3];
  }
  Columns<D> run;

  // ---- own keys: this warp's rows in turn. Lane x % 8 holds what query x's row needs.
  uint8_t* ring = sm + kWholeRows * D * 2 + warp * 4 * UNIT;
  const int qx = wr + (lane & 7), row_x = row_of[qx], len_x = len_of[qx], begin_x = begin_of[qx], page_x = page_of[qx];
  const bool leads = row_x >= 0 && (qx == wr || row_of[qx - 1] != row_x);  // the row's first query in this warp
  const int units_x = leads && len_x > begin_x ? (len_x - begin_x + kUnit - 1) / kUnit : 0;
  const long long at_x = page_ok(page_x, p.g.pages) ? tile_offset(p.g, page_x, p.layer, 0, kvh) : -1;
  const int row_a = row_of[ca], row_b = row_of[cb];
  unsigned todo = __ballot_sync(0xffffffffu, lane < 8 && units_x > 0);
  struct Step {
    int row, len, key;  // the row, its tokens, the first of the 16 keys
    bool fresh, there;
  };
  int x = 0, u = 0, units = 0;  // where the loads are
  long long at_first = 0;
  Step next = {-1, 0, 0, true, false};
  auto load = [&](int n) {
    uint8_t* kd = ring + (n & 1) * 2 * UNIT;
    next.key += u ? kUnit : 0;
    next.fresh = u == 0;
    int slot = u * kUnit;  // a prefix is whole pages: own tokens begin with one
    long long at = at_first;
    if (slot >= P) {
      const int page = p.table[(long long)seq_of[wr + x] * p.g.width + next.key / P];
      slot %= P;
      at = page_ok(page, p.g.pages) ? tile_offset(p.g, page, p.layer, 0, kvh) : -1;
    }
    next.there = at >= 0;
    if (!next.there && lane == 0) atomicOr(p.status, OASIS_PAGES_BAD_PAGE);
    const uint4* from = pool + (next.there ? at + slot * CH : 0) + lane;
    const int left = next.there ? next.len - next.key : 0;  // rows behind the sequence hold anything: zero instead
#pragma unroll
    for (int i = 0; i < kUnit * CH / 32; ++i) {
      const int y = i * 32 + lane, r = y / CH, c = y % CH;
      cp_async16(kd + tile_at<D>(r, c), from + i * 32, r < left);
      cp_async16(kd + UNIT + tile_at<D>(r, c), from + to_v + i * 32, r < left);
    }
    cp_async_commit();
  };
  auto advance = [&]() {  // to the next 16 keys; false behind the last ones
    if (++u < units) return true;
    if (!todo) return false;
    x = __ffs(todo) - 1;
    todo &= todo - 1;
    u = 0;
    units = __shfl_sync(0xffffffffu, units_x, x);
    at_first = __shfl_sync(0xffffffffu, at_x, x);
    next.row = __shfl_sync(0xffffffffu, row_x, x);
    next.len = __shfl_sync(0xffffffffu, len_x, x);
    next.key = __shfl_sync(0xffffffffu, begin_x, x);
    return true;
  };
  bool more = advance();
  if (more) load(0);
  for (int n = 0; more; ++n) {
    const Step now = next;
    more = advance();
    if (more) {
      load(n + 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncwarp();
    if (now.there) {
      const uint8_t* sk = ring + (n & 1) * 2 * UNIT;
      column_step<T, D>(run, sk, sk + UNIT, 0, now.key, qb, row_a == now.row ? now.len : 0, row_b == now.row ? now.len : 0,
                        now.fresh, p.scale_log2);
    }
    __syncwarp();  // the stage may be loaded again
  }
  __syncthreads();  // the rings' place is the prefix tiles'
  // ---- prefixes: the groups of the tile's rows in turn
  for (int x = 0; x < kWholeRows;) {
    const int group = group_of[x];
    const int tokens = begin_of[x];
    if (row_of[x] < 0) break;
    // up to the first row of another group (rows of none lie before the groups and behind them)
    static_assert(kWholeRows == 32, "a lane for each query");
    const unsigned others = __ballot_sync(0xffffffffu, lane > x && (group_of[lane] != group || row_of[lane] < 0));
    const int after = others ? __ffs(others) - 1 : kWholeRows;
    if (tokens == 0) {
      x = after;
      continue;
    }
    // read through the longest of the group's sequences (the first of them)
    const int b0 = max(0, p.group_start[group]), b1 = min(p.rows, p.group_start[group + 1]);
    int len = -1, row = b1;
    for (int b = b0 + tid; b < b1; b += kThreads) {
      int s;
      const int t = row_length(p, b, &s);
      if (t > len) {
        len = t;
        row = b;
      }
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) {
      const int l2 = __shfl_xor_sync(0xffffffffu, len, w), r2 = __shfl_xor_sync(0xffffffffu, row, w);
      if (l2 > len || (l2 == len && r2 < row)) {
        len = l2;
        row = r2;
      }
    }
    if (lane == 0) {
      lead_len[warp] = len;
      lead_row[warp] = row;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (lead_len[w] > len || (lead_len[w] == len && lead_row[w] < row)) {
        len = lead_len[w];
        row = lead_row[w];
      }
    const int common = max(0, min(tokens, len));
    const int* lead = p.table + (long long)(len > 0 ? p.seqs[row] : 0) * p.g.width;
    const int units = (common + kUnit - 1) / kUnit, steps = (units + 3) / 4;
    auto load = [&](int j) {
      uint8_t* kd = sm + kWholeRows * D * 2 + (j & 1) * 2 * TILE;
      const int keys = min(4, units - j * 4) * kUnit;
      for (int i = tid; i < keys * CH; i += kThreads) {
        const int r = i / CH, c = i % CH;
        const int t = (j * 4 + r / kUnit) * kUnit;
        const int page = lead[t / P];
        const bool ok = page_ok(page, p.g.pages);
        const long long at = tile_offset(p.g, ok ? page : 0, p.layer, 0, kvh) + (long long)(t % P + r % kUnit) * CH + c;
        const bool in = ok && t + r % kUnit < common;  // rows behind the sequences hold anything: zero instead
        cp_async16(kd + tile_at<D>(r, c), pool + at, in);
        cp_async16(kd + TILE + tile_at<D>(r, c), pool + at + to_v, in);
        if (c == 0 && r % kUnit == 0) {
          unit_ok[j & 1][r / kUnit] = ok;
          if (!ok) atomicOr(p.status, OASIS_PAGES_BAD_PAGE);
        }
      }
      cp_async_commit();
    };
    if (steps > 0) load(0);
    const int lim_a = ca >= x && ca < after ? min(common, len_of[ca]) : 0;
    const int lim_b = cb >= x && cb < after ? min(common, len_of[cb]) : 0;
    for (int j = 0; j < steps; ++j) {
      if (j + 1 < steps) {
        load(j + 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      const uint8_t* sk = sm + kWholeRows * D * 2 + (j & 1) * 2 * TILE;
      if (__any_sync(0xffffffffu, lim_a > 0 || lim_b > 0))
        for (int h = 0; h < min(4, units - j * 4); ++h)
          if (unit_ok[j & 1][h])
            column_step<T, D>(run, sk, sk + TILE, h * kUnit, (j * 4 + h) * kUnit, qb, lim_a, lim_b, false, p.scale_log2);
      __syncthreads();
    }
    __syncthreads();  // lead_len is free again
    x = after;
  }
  run.join();

  // ---- result, O^T turned back through this warp's own rows of Q
  const float ia = len_of[ca] > 0 ? 1.f / run.l[0] : 0.f, ib = len_of[cb] > 0 ? 1.f / run.l[1] : 0.f;
  bool ok_a = len_of[ca] == 0 || (run.l[0] > 0.f && finite_f(run.l[0]));
  bool ok_b = len_of[cb] == 0 || (run.l[1] > 0.f && finite_f(run.l[1]));
  const int qr = wr + (lane >> 2);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    ok_a = ok_a && finite_f(run.o[t][0]) && finite_f(run.o[t][2]);
    ok_b = ok_b && finite_f(run.o[t][1]) && finite_f(run.o[t][3]);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<uint32_t*>(sm + tile_at<D>(qr, t * 2 + e) + (lane & 3) * 4) =
          transpose8(Elem<T>::pack(run.o[t][2 * e] * ia, run.o[t][2 * e + 1] * ib));
  }
  const unsigned bad_a = __ballot_sync(0xffffffffu, !ok_a), bad_b = __ballot_sync(0xffffffffu, !ok_b);
  __syncwarp();
#pragma unroll
  for (int i = lane; i < 8 * CH; i += 32) {
    const int r = wr + i / CH, c = i % CH, b = row_of[r];
    if (b < 0) continue;
    const int h = kvh * p.per + at_query.head_of(r);
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + b * p.o_row + h * p.o_head + c * 8) =
        *reinterpret_cast<const uint4*>(sm + tile_at<D>(r, c));
  }
  if ((bad_a | bad_b) == 0) return;
  __syncwarp();
  for (int r = 0; r < 8; ++r)
    if (((r & 1 ? bad_b : bad_a) & (0x11111111u << (r >> 1))) && row_of[wr + r] >= 0)
      row_again<T, D>(p, row_of[wr + r], kvh * p.per + at_query.head_of(wr + r));
}

// Joins the ranges of each (row, head): a warp each, D / 32 dims per lane.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) shared_join_kernel(SharedParams p) {
  constexpr int DV = D / 32;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (kThreads / 32) + warp;
  if (item >= (long long)p.rows * p.heads) return;
  const int b = (int)(item / p.heads), h = (int)(item - (long long)b * p.heads);
  const int splits = p.prefix_splits + p.own_splits;
  const int group = served_group(p, b), first = group >= 0 ? 0 : p.prefix_splits;
  int s;
  const int len = row_length(p, b, &s);
  // the row's ranges: the prefix ones and as many own ones as its length has
  const int begin = group_tokens(p, group);
  const int units = len > begin ? (len - begin + kUnit - 1) / kUnit : 0;
  const int last = p.prefix_splits + min(p.own_splits, max(1, (units + p.own_units - 1) / p.own_units));
  const float2* ml = p.part_ml + item * splits;
  // all maxima and sums at once, four ranges per lane
  float2 mine[kMostRanges / 32];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMostRanges / 32; ++k) {
    const int i = first + k * 32 + lane;
    mine[k] = i < last ? ml[i] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, mine[k].x);
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
  const float sh = softmax_shift(m);
  float l = 0.f, o[DV] = {};
#pragma unroll
  for (int k = 0; k < kMostRanges / 32; ++k) {
    const float f = ex2_approx(mine[k].x - sh);
    l += mine[k].y * f;
    const bool some = !(mine[k].x == -INFINITY && mine[k].y == 0.f);  // its sums were written
    unsigned todo = __ballot_sync(0xffffffffu, some);
    while (todo) {  // eight ranges' loads in flight
      float4 y[8];
      float g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = todo ? __ffs(todo) - 1 : -1;
        todo &= todo - 1;
        g[e] = i >= 0 ? __shfl_sync(0xffffffffu, f, i) : 0.f;
        y[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i >= 0) {
          const float* at = p.part_o + (item * splits + first + k * 32 + i) * D + lane * DV;
          if constexpr (DV == 4) {
            y[e] = *reinterpret_cast<const float4*>(at);
          } else {
            const float2 z = *reinterpret_cast<const float2*>(at);
            y[e].x = z.x;
            y[e].y = z.y;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v[4] = {y[e].x, y[e].y, y[e].z, y[e].w};
#pragma unroll
        for (int d = 0; d < DV; ++d) o[d] = fmaf(v[d], g[e], o[d]);
      }
    }
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  bool ok = len == 0 || (l > 0.f && finite_f(l));
#pragma unroll
  for (int d = 0; d < DV; ++d) ok = ok && finite_f(o[d]);
  if (__any_sync(0xffffffffu, !ok)) {
    row_again<T, D>(p, b, h);
    return;
  }
  const float inv = len > 0 ? 1.f / l : 0.f;
  T* out = static_cast<T*>(p.out) + b * p.o_row + h * p.o_head + lane * DV;
#pragma unroll
  for (int d = 0; d < DV; d += 2) *reinterpret_cast<uint32_t*>(out + d) = Elem<T>::pack(o[d] * inv, o[d + 1] * inv);
}

// Splits and tiles of a call, from the shapes and the caller's hints alone.
void plan(const OasisSharedArgs* a, SharedParams* p) {
  const int sms = num_sms();
  const int K = a->cache->kv_heads;
  p->per = a->heads / K;
  p->head_tiles = (p->per + 7) / 8;
  bool prefix = a->groups > 0 && a->prefix_pages_hint > 0;
  long long own = a->own_tokens_hint;
  long long keys = prefix ? (long long)a->prefix_pages_hint * a->cache->page_size : 0;
  // Where sharing would save little reading (and what is read again comes from L2), each
  // row reads its prefix with its own keys: one kernel, and nothing waits for another. Shared
  // / alone, us, up to 40 own tokens, 16 heads of 64: 3 rows behind 144 tokens 12.0 / 5.6, 8
  // behind 500 (14 MB saved) 11.2 / 11.7, 16 behind 500 (31 MB) 11.4 / 14.7; 32 / 8 heads of
  // 128: 16 behind 500 14.5 / 12.7, 32 behind 500 (63 MB) 15.5 / 19.0. Groups cost the prefix
  // kernel more: 16 of up to 4 rows, 500 tokens, 29.8 / 15.7.
  const double saved = ((double)a->rows - a->groups) * keys * K * a->cache->head_dim * 4;  // bytes
  if (prefix && saved <= ((a->cache->head_dim == 64 ? 24 : 48) + 2 * (a->groups < 16 ? a->groups : 16)) * 1048576.0) {
    own += keys;
    keys = 0;
    prefix = false;
  }
  const long long room = (long long)a->cache->width * a->cache->page_size;  // of a sequence, below 2^31
  if (own > room) own = room;
  p->groups = prefix ? a->groups : 0;
  // A group has no more rows than the batch, whatever the hint; and what tiles do not cover is
  // covered all the same (they go on behind their last one, or leave rows to the own keys),
  // so that a launch has at most 2^30 of them.
  const long long hint = a->group_rows_hint < 1 ? 1 : a->group_rows_hint, group_rows = hint < a->rows ? hint : a->rows;
  const long long most_tiles = prefix ? (1LL << 30) / ((long long)a->groups * K) : 1;
  auto tiles = [&](int queries) {
    const long long n = (group_rows * p->per + queries - 1) / queries;
    return (int)(n < most_tiles ? n : most_tiles > 1 ? most_tiles : 1);
  };
  p->tiles = tiles(kPrefixRows);
  p->prefix_splits = 0;
  p->tensor = 0;
  p->reach = 0x7fffffff;
  if (prefix) {
    const long long pool_rows = (long long)a->cache->pages * a->cache->layers * 2 * K * a->cache->page_size;
    long long least = kTensorKeys;
    if (p->tiles == 1 && (long long)a->groups * K > sms) least += (long long)a->groups * K - sms;
    p->tensor = keys >= (least < kTensorKeysMost ? least : kTensorKeysMost) && pool_rows < (1LL << 31);
  }
  // A row's own keys go to teams of four warps in ranges of one length, so that a row
  // longer than the others only has more of them. Where the hinted length is small for the
  // number of items (row, key head, eight heads), an item is one warp's: a block's lookups
  // and its end then serve four items, and the longest row's warp takes four times as long.
  // One warp / four, us, ragged rows in groups, so many items with rows
  // of up to so many tokens behind their prefix: heads of 64: 272 items 12.6 / 13.6 (64), 20.5 /
  // 13.8 (256); 2512 items 19.5 / 28.8 (64), 30.4 / 32.6 (256), 80 / 47 (1024); 12544 items 47 /
  // 109 (64), 138 / 159 (1024). Heads of 128, where an SM holds half as many blocks: 536
  // items 18.9 / 23.1 (64), 24.1 / 25.2 (256), 83 / 54 (4096); 6272 items 56 / 117 (64), 138 / 165 (1024).
  const long long items = (long long)a->rows * K * p->head_tiles;
  const long long units = (own + kUnit - 1) / kUnit;
  p->team = units <= 8 + items * a->cache->head_dim / 8192 ? 1 : kOwnWarps;
  // Ranges: as many as make 12 teams for each SM (heads of 128: 6) where all rows have the
  // hinted length, up to twice as many where they would be longer than 1024 keys (and the
  // hint is not long for another group's prefix, 33.8 -> 41.2 us), each of at least 256. 12 / 24 teams, us: 64 rows alone, 16 heads of 64: 50.9 / 48.9 with up to
  // 2000 tokens, 118 / 88 with 8000; behind 2048 shared ones 35.9 / 40.1 with 1000. 6 / 12,
  // 32 / 8 heads of 128: 45.9 / 47.3, 98 / 78, 41.8 / 44.9. One range where a long prefix
  // takes as long: 8 rows behind 2048 tokens, up to 1000 own ones, 25.7 -> 20.6 us.
  const long long teams = 768 / a->cache->head_dim * sms;
  long long n = own >= 2 * keys ? (units + 63) / 64 : 1, most = (2 * teams + items - 1) / items;
  if (n > most) n = most;
  if (n * items < teams) n = (teams + items - 1) / items;
  if (n > kMostSplits) n = kMostSplits;
  long long each = (units + n - 1) / n;
  if (each < 16) each = 16;
  if (p->team == 1 || (p->tensor && keys >= 2048 && units <= 64 && items <= 2LL * sms)) each = units > 16 ? units : 16;
  p->own_units = (int)each;
  p->own_splits = (int)(units > each ? (units + each - 1) / each : 1);
  if (prefix) {
    if (p->tensor) {
      // One block for each SM, and at least 128 keys for each block; two thirds of them where
      // the own keys, in one range, can run beside them on the SMs that this leaves, since a
      // block takes all of its SM's registers. All / two thirds, us: 64 rows behind 8192
      // tokens, 16 heads of 64: 28.0 / 27.8 with up to 16 own tokens, 41.2 / 27.9 with 256;
      // 32 / 8 heads of 128: 38.1 / 33.7, 49.8 / 34.2; 256 rows of 16 heads of 64: 53.8 / 56.1
      // behind 8192 tokens, 43.2 / 41.3 behind 2048; with own keys in ranges, up to 2048 of
      // them: 57.1 / 62.1.
      const long long pairs = tiles(256);
      p->tiles = (int)pairs;
      p->reach = (int)(pairs * 256 < 0x7fffffff ? pairs * 256 : 0x7fffffff);
      const long long blocks = (long long)a->groups * K * pairs;
      long long n = sms / blocks;
      if (p->own_splits == 1 && n >= 6) n = n * 2 / 3;
      if (n > keys / 128) n = keys / 128;
      p->prefix_splits = (int)(n < 1 ? 1 : n > kMostSplits ? kMostSplits : n);
    } else {
      // two blocks for each SM, and at least 128 keys for each block
      const long long blocks = (long long)a->groups * K * p->tiles;
      long long n = (2LL * sms + blocks - 1) / blocks;
      if (n > keys / 128) n = keys / 128;
      p->prefix_splits = (int)(n < 1 ? 1 : n > kMostSplits ? kMostSplits : n);
    }
  }
  // One pass where its blocks fill the GPU and a warp has at most 32 steps of own keys
  // for its eight queries and 16 of a prefix, one behind the other.
  const long long blocks = ((long long)a->rows * p->per + kWholeRows - 1) / kWholeRows * K;
  const long long rows = (8 + p->per - 1) / p->per, steps = rows * ((own + kUnit - 1) / kUnit);
  p->whole = blocks >= 4LL * sms && steps <= 32 &&
             keys <= 16 * kPrefixKeys;
}

size_t partial_bytes(const OasisSharedArgs* a, const SharedParams& p) {
  if (p.whole || (p.prefix_splits == 0 && p.own_splits == 1)) return 0;
  const size_t slots = (size_t)a->rows * a->heads * (p.prefix_splits + p.own_splits);
  return slots * (sizeof(float2) + sizeof(float) * a->cache->head_dim);
}

template <typename T, int D>
int launch(const SharedParams& p, cudaStream_t s) {
  static std::atomic<bool> attr[64];  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaError_t e =
        cudaFuncSetAttribute(shared_prefix_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, prefix_smem<D>());
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(shared_whole_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, whole_smem<D>());
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(shared_own_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, own_smem<D>());
    if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr[dev & 63] = true;
  }
  if (p.whole) {
    const long long blocks = ((long long)p.rows * p.per + kWholeRows - 1) / kWholeRows * p.g.kv_heads;
    launch_pdl(shared_whole_kernel<T, D>, dim3((unsigned)blocks), dim3(kThreads), whole_smem<D>(), s, p);
    return check_launch("shared_whole_kernel");
  }
  if (p.prefix_splits && p.tensor) {
    OASIS_TRY(shared_prefix_tc_launch(p, Elem<T>::kHalf, s));
  } else if (p.prefix_splits) {
    const long long blocks = (long long)p.groups * p.g.kv_heads * p.prefix_splits * p.tiles;
    launch_pdl(shared_prefix_kernel<T, D>, dim3((unsigned)blocks), dim3(kThreads), prefix_smem<D>(), s, p);
    OASIS_TRY(check_launch("shared_prefix_kernel"));
  }
  const long long items = (long long)p.rows * p.g.kv_heads * p.head_tiles * p.own_splits, in_block = kOwnWarps / p.team;
  launch_pdl(shared_own_kernel<T, D>, dim3((unsigned)((items + in_block - 1) / in_block)), dim3(kOwnWarps * 32),
             own_smem<D>(), s, p);
  OASIS_TRY(check_launch("shared_own_kernel"));
  if (p.own_splits > 1) {
    const long long rows = (long long)p.rows * p.heads;
    launch_pdl(shared_join_kernel<T, D>, dim3((unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32))), dim3(kThreads),
               0, s, p);
    OASIS_TRY(check_launch("shared_join_kernel"));
  }
  return OASIS_OK;
}

int check_shared(const OasisSharedArgs* a) {
  OASIS_REQUIRE(a && a->cache, "attention_shared: null args");
  const OasisPageCache* c = a->cache;
  OASIS_REQUIRE(c->dtype == OASIS_DTYPE_BF16 || c->dtype == OASIS_DTYPE_F16, "attention_shared: dtype=%d", c->dtype);
  OASIS_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "attention_shared: head_dim=%d is not 64 or 128", c->head_dim);
  OASIS_REQUIRE(c->pages >= 1 && c->layers >= 1 && c->kv_heads >= 1 && c->slots >= 1 && c->width >= 1,
                "attention_shared: pages=%d layers=%d kv_heads=%d slots=%d width=%d", c->pages, c->layers, c->kv_heads,
                c->slots, c->width);
  OASIS_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && c->page_size % 16 == 0,
                "attention_shared: page_size=%d is not a multiple of 16 up to 256", c->page_size);
  OASIS_REQUIRE((long long)c->slots * c->width < (1LL << 31) && (long long)c->width * c->page_size < (1LL << 31),
                "attention_shared: page table of %d x %d entries is too large", c->slots, c->width);
  OASIS_REQUIRE(a->layer >= 0 && a->layer < c->layers, "attention_shared: layer=%d of %d", a->layer, c->layers);
  OASIS_REQUIRE(a->heads >= c->kv_heads && a->heads <= 1024 && a->heads % c->kv_heads == 0,
                "attention_shared: heads=%d kv_heads=%d", a->heads, c->kv_heads);
  OASIS_REQUIRE(a->rows >= 0 && a->groups >= 0, "attention_shared: rows=%d groups=%d", a->rows, a->groups);
  OASIS_REQUIRE((long long)a->rows * c->kv_heads * ((a->heads / c->kv_heads + 7) / 8) < (1LL << 31),
                "attention_shared: %d rows of %d heads are too many", a->rows, a->heads);
  OASIS_REQUIRE(a->scale > 0.f && a->scale <= 3e38f, "attention_shared: scale=%g", (double)a->scale);
  return OASIS_OK;
}

}  // namespace
}  // namespace oasis

using namespace oasis;

extern "C" {

size_t oasis_attention_shared_workspace_size(const OasisSharedArgs* a) {
  if (check_shared(a) != OASIS_OK || a->rows == 0) return 0;
  SharedParams p;
  plan(a, &p);
  return partial_bytes(a, p);
}

int oasis_attention_shared(const OasisSharedArgs* a, oasis_stream_t stream) {
  OASIS_TRY(check_shared(a));
  if (a->rows == 0) return OASIS_OK;
  const OasisPageCache* c = a->cache;
  OASIS_REQUIRE(a->q && a->out && a->seqs && c->pool && c->table && c->lengths && c->status,
                "attention_shared: null pointer");
  OASIS_REQUIRE(a->groups == 0 || (a->group_start && a->prefix_pages), "attention_shared: null group arrays");
  const uintptr_t at = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out) |
                       reinterpret_cast<uintptr_t>(c->pool);
  OASIS_REQUIRE((at & 15) == 0, "attention_shared: operands not 16-byte aligned");
  const long long strides[4] = {a->q_row_stride, a->q_head_stride, a->out_row_stride, a->out_head_stride};
  for (long long s : strides)
    OASIS_REQUIRE(s > 0 && s % 8 == 0 && s < (1LL << 36),
                  "attention_shared: stride %lld is not a positive multiple of 8 elements", s);
  SharedParams p;
  plan(a, &p);
  const long long blocks = (long long)p.groups * c->kv_heads * p.prefix_splits * p.tiles;
  const long long items = (long long)a->rows * c->kv_heads * p.head_tiles * p.own_splits;
  OASIS_REQUIRE(blocks < (1LL << 31) && items < (1LL << 31), "attention_shared: %d rows of %d heads are too many",
                a->rows, a->heads);
  const size_t want = partial_bytes(a, p);
  if (want && (!a->workspace || a->workspace_bytes < want))
    return set_error(OASIS_ERR_WORKSPACE, "attention_shared: workspace of %zu bytes, %zu needed", a->workspace_bytes,
                     want);
  OASIS_REQUIRE((reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0, "attention_shared: workspace not 16-byte aligned");
  p.g.pages = c->pages;
  p.g.layers = c->layers;
  p.g.kv_heads = c->kv_heads;
  p.g.page_size = c->page_size;
  p.g.head_dim = c->head_dim;
  p.g.slots = c->slots;
  p.g.width = c->width;
  p.q = a->q;
  p.out = a->out;
  p.pool = c->pool;
  p.q_row = strides[0];
  p.q_head = strides[1];
  p.o_row = strides[2];
  p.o_head = strides[3];
  p.table = c->table;
  p.lengths = c->lengths;
  p.seqs = a->seqs;
  p.group_start = a->group_start;
  p.prefix_pages = a->prefix_pages;
  p.status = c->status;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)a->rows * a->heads * (p.prefix_splits + p.own_splits) *
                                                       c->head_dim);
  p.rows = a->rows;
  p.heads = a->heads;
  p.layer = a->layer;
  p.scale_log2 = a->scale * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->dtype == OASIS_DTYPE_BF16)
    return c->head_dim == 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
  return c->head_dim == 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
}

}  // extern "C"
