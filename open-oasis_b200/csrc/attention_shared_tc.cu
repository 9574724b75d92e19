// The keys that a group's rows have in common, on the 5th-generation tensor cores: the
// prefix ranges of attention_shared.cu (which has the formula) for longer prefixes.
//
// A block takes 256 (row, head) queries of one group and key head, as two tiles of 128,
// and a range of the prefix in blocks of 128 keys; the products, the softmax and the
// roles of the warps are those of attention_prompt_tc.cu, without a causal mask: a
// query sees the keys below its limit. K and V blocks come by TMA from the pages, a box
// of a page's rows at a time (16 where pages do not divide 128), the pool seen as rows
// of one head; what lies behind the prefix or outside the pool is fetched from behind
// the pool's last row, which reads zero, and masked. The result is the range's maximum,
// sum and unnormalised O.
//
// Bound: for a group of at least 256 queries the softmax's pipes, as there; for small
// ones the latency of a range's blocks, S, softmax and P V one behind the other. 64 rows
// of 32 / 8 heads of 128 behind 8192 tokens: about 25 us with 18 ranges for each key head,
// of which 6 are the block's start (the longest row, Q, the first pages).
#include "../../include/oasis_b200.h"
#include "attention_shared.cuh"
#include "attention_tc.cuh"
#include "gemm.cuh"
#include "status.h"

namespace oasis {
namespace {

constexpr int kSharedThreads = 384;
// Of every eight pairs of exponentials this many go to the FMA pipe.
constexpr int kPoly = 2;

template <int D>
struct Cfg {
  static constexpr int CHUNKS = D / 64;               // 64-column chunks: 128 bytes of a row
  static constexpr int CHUNK_BYTES = kTile * 128;
  static constexpr int TILE_BYTES = CHUNKS * CHUNK_BYTES;
  static constexpr int STAGES = D == 64 ? 8 : 5;
  static constexpr int BAR_BYTES = 512;               // barriers, page words, the search for the longest sequence
  static constexpr int SMEM = 1024 + (2 + STAGES) * TILE_BYTES + BAR_BYTES;
  static_assert(SMEM <= 232448, "shared memory");
  static constexpr bool kApart = D == 64;             // S and P in columns of their own
  static constexpr int S_COL = 0;                     // + 128 per tile
  static constexpr int P_COL = kApart ? 256 : 0;      // + P_STEP per tile
  static constexpr int P_STEP = kApart ? 64 : 128;
  static constexpr int O_COL = kApart ? 384 : 256;    // + D per tile
};

template <typename T, int D>
__global__ void __launch_bounds__(kSharedThreads, 1)
    shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap pool_map, const __grid_constant__ SharedParams p,
                            int box_rows, int pool_rows) {
  using C = Cfg<D>;
  using E = Elem<T>;
  extern __shared__ uint8_t smem_raw[];
  pdl_wait();
  int x = blockIdx.x;
  const int pair = x % p.tiles;
  x /= p.tiles;
  const int split = x % p.prefix_splits;
  x /= p.prefix_splits;
  const int kvh = x % p.g.kv_heads, group = x / p.g.kv_heads;
  const int b0 = max(0, p.group_start[group]), b1 = min(p.rows, p.group_start[group + 1]);
  const long long queries = (long long)max(0, b1 - b0) * p.per, m0 = (long long)pair * 2 * kTile;
  if (m0 >= queries) return;  // the whole block
  const Queries at_query(m0, p.per);
  const int P = p.g.page_size;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + 2 * C::TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + C::STAGES * C::TILE_BYTES);
  uint64_t* s_full = bars + 2;     // [2]
  uint64_t* s_read = bars + 4;     // [2] softmax has S in registers (kApart)
  uint64_t* p_full = bars + 6;     // [2]
  uint64_t* pv_done = bars + 8;    // [2]
  uint64_t* drain = bars + 10;     // [2]
  uint64_t* kv_full = bars + 16;   // [STAGES <= 8]
  uint64_t* kv_empty = bars + 24;  // [STAGES <= 8]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);
  // Which groups of 16 keys of a block are there, of the last eight blocks: a block's
  // word is written again once S of the fourth block after it is done, when its own
  // softmax is long past it.
  unsigned* page_bits = reinterpret_cast<unsigned*>(bars + 40);
  int* lead_len = reinterpret_cast<int*>(bars + 48);              // [12]
  int* lead_row = lead_len + 12;                                  // [12]

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_read[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&pv_done[t], 1);
      mbar_init(&drain[t], 1);
    }
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], C::kApart ? 2 : 1);
    }
    fence_barrier_init();
  }
  if (warp == 9) {
    // The trigger is behind the wait, since the kernel of the own keys starts without one,
    // and behind the allocation: a kernel that took TMEM first and then waited for this
    // grid would never get to give it back.
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    pdl_trigger();
  }
  // The prefix is read through the table row of the longest sequence (the first of
  // them): a shorter one need not have all of its pages.
  int len = -1, lead = b1;
  for (int b = b0 + threadIdx.x; b < b1; b += kSharedThreads) {
    int s;
    const int t = row_length(p, b, &s);
    if (t > len) {
      len = t;
      lead = b;
    }
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    const int l2 = __shfl_xor_sync(0xffffffffu, len, w), r2 = __shfl_xor_sync(0xffffffffu, lead, w);
    if (l2 > len || (l2 == len && r2 < lead)) {
      len = l2;
      lead = r2;
    }
  }
  if (lane == 0) {
    lead_len[warp] = len;
    lead_row[warp] = lead;
  }
  // Q: the two tiles' rows, as TMA would lay them out
  for (int i = threadIdx.x; i < 2 * kTile * (D / 8); i += kSharedThreads) {
    const int r = i / (D / 8), ch = i % (D / 8);
    uint4 y = make_uint4(0, 0, 0, 0);
    if (m0 + r < queries) {
      const T* at = static_cast<const T*>(p.q) + (b0 + at_query.row_of(r)) * p.q_row +
                    (kvh * p.per + at_query.head_of(r)) * p.q_head;
      y = *reinterpret_cast<const uint4*>(at + ch * 8);
    }
    *reinterpret_cast<uint4*>(sQ + (r / kTile) * C::TILE_BYTES + (ch / 8) * C::CHUNK_BYTES + tile_at<64>(r % kTile, ch % 8)) = y;
  }
  fence_proxy_async();  // the products read Q through the async proxy
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = 0;  // all 512 columns are this block's, so they begin at 0
#pragma unroll
  for (int w = 0; w < 12; ++w)
    if (lead_len[w] > len || (lead_len[w] == len && lead_row[w] < lead)) {
      len = lead_len[w];
      lead = lead_row[w];
    }
  const int common = max(0, min(group_tokens(p, group), len));
  const int* table = p.table + (long long)(len > 0 ? p.seqs[lead] : 0) * p.g.width;
  const int all = (common + kTile - 1) / kTile;  // key blocks of the prefix, and this range's
  const int begin = (int)((long long)all * split / p.prefix_splits), blocks = (int)((long long)all * (split + 1) / p.prefix_splits) - begin;
  const int tiles_here = queries > m0 + kTile ? 2 : 1;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      // ---------------- TMA ----------------
      // A lane per box, with its page looked up one block ahead.
      const int total = 2 * blocks, boxes = kTile / box_rows;
      const long long tile_rows = (long long)p.g.kv_heads * P;  // pool rows of a page's layer's keys, or values
      auto page_at = [&](int block) {  // of this lane's box; -1: behind the prefix or not in the pool
        const int t = block * kTile + lane * box_rows;
        if (lane >= boxes || t >= common) return -1;
        const int page = table[t / P];
        if (page_ok(page, p.g.pages)) return page;
        atomicOr(p.status, OASIS_PAGES_BAD_PAGE);
        return -1;
      };
      int issued = 0, page = blocks > 0 ? page_at(begin) : -1;
      bool ok = true;
      while (issued < total && ok) {
        const int block = begin + (issued >> 1);
        const int ahead = (issued & 1) == 0 && issued + 2 < total ? page_at(block + 1) : -1;
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
        unsigned bits = 0;
        for (int i = 0; i < boxes; ++i)
          if (there >> i & 1) bits |= ((1u << (box_rows / kUnit)) - 1) << (i * (box_rows / kUnit));
        const int slot = (block * kTile + lane * box_rows) % P;
        int next_page = ahead;
        for (int which = 0; which < 2 && ok; ++which, ++issued) {
          const int st = issued % C::STAGES;
          if (issued >= C::STAGES)
            ok = __all_sync(0xffffffffu, wait_for(&kv_empty[st], ((issued / C::STAGES) & 1) ^ 1, kDevTimeoutSmemEmpty));
          if (!ok) break;
          if (lane == 0) {
            if (which == 0) {
              page_bits[(issued >> 1) & 7] = bits;
              __threadfence_block();
            }
            mbar_arrive_expect_tx(&kv_full[st], C::TILE_BYTES);
          }
          __syncwarp();  // the bytes are expected before they come
          if (lane < boxes) {
            uint8_t* dst = sKV + st * C::TILE_BYTES + lane * box_rows * 128;
            const int row = page >= 0 ? (int)((((long long)page * p.g.layers + p.layer) * 2 + which) * tile_rows +
                                              (long long)kvh * P + slot)
                                      : pool_rows;
#pragma unroll
            for (int c = 0; c < C::CHUNKS; ++c)
              tma_load_3d(dst + c * C::CHUNK_BYTES, &pool_map, &kv_full[st], c * 64, row, 0);
          }
        }
        page = next_page;
      }
      if (!ok)  // gave up: the copies in flight land before the block ends
        for (int i = max(0, issued - C::STAGES); i < issued; ++i)
          wait_for(&kv_full[i % C::STAGES], (i / C::STAGES) & 1, kDevTimeoutTmaFull);
    }
    if (warp == 9 || (C::kApart && warp == 10)) {
      // ---------------- MMA ----------------
      // D = 64: a warp per tile; with one warp for both, issuing 24 MMAs and waiting
      // for six barriers in turn took as long as the softmax. D = 128: one warp, so
      // that a tile's P V and next S run one behind the other and the tiles take turns;
      // issued by two warps they mixed and both tiles waited for all four.
      // The whole warp walks the loop with values that are the same in all lanes, so
      // that descriptors live in uniform registers, and one elected lane issues: from
      // a single-lane branch each tcgen05.mma took about 100 cycles to issue.
      constexpr uint32_t idS = idesc_16<T>(kTile, false);
      constexpr uint32_t idPV = idesc_16<T>(D, true);
      const bool one = elect_one();
      const int t0 = warp - 9, t1 = C::kApart ? t0 + 1 : 2;  // this warp's tiles
      const uint64_t q_desc = smem_desc_sw128(smem_u32(sQ)), k_desc = smem_desc_sw128(smem_u32(sKV)),
                     v_desc0 = v_desc(smem_u32(sKV));
      bool ok = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, wait_for(bar, parity, code)) != 0;
      };
      auto stage_off = [&](int i) { return (uint64_t)(i % C::STAGES * (C::TILE_BYTES >> 4)); };
      auto arrived = [&](int i) { return wait_all(&kv_full[i % C::STAGES], (i / C::STAGES) & 1, kDevTimeoutTmaFull); };
      // K or V block i, which has arrived, is not needed by this warp any more once the
      // MMAs issued so far are done
      auto release = [&](int i) {
        if (one) tc_commit(&kv_empty[i % C::STAGES]);
      };
      auto active = [&](int t) { return t < tiles_here; };
      auto issue_s = [&](int t, int j) {
        tc_fence_after();
        const uint64_t qa = q_desc + (uint64_t)(t * (C::TILE_BYTES >> 4)), ka = k_desc + stage_off(2 * j);
        const uint32_t d = C::S_COL + t * kTile;
        if (one) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t off = ((k >> 2) * C::CHUNK_BYTES + (k & 3) * 32) >> 4;
            tc_mma_bf16(d, qa + off, ka + off, idS, k > 0);
          }
          tc_commit(&s_full[t]);
        }
      };
      auto issue_pv = [&](int t, int j) {
        tc_fence_after();
        const uint64_t va = v_desc0 + stage_off(2 * j + 1);
        const uint32_t more = j > 0, d = C::O_COL + t * D, pa = C::P_COL + t * C::P_STEP;
        if (one) {
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k) mma_ts(d, pa + k * 8, va + (uint64_t)(k * 2048 >> 4), idPV, k > 0 ? 1u : more);
          tc_commit(&pv_done[t]);
        }
      };
      // Rows of V block j behind the longest sequence, where that ends inside a box, hold
      // anything: zeros instead, like their probabilities, since an infinity or NaN there would
      // send every row to the repair. It is the prefix's last block, so that its stage is
      // not loaded again; with two warps both write the same zeros, each ahead of its own products.
      auto clear = [&](int j) {
        const int row = common - (begin + j) * kTile;
        uint8_t* stage = sKV + (2 * j + 1) % C::STAGES * C::TILE_BYTES;
        for (int c = 0; c < C::CHUNKS; ++c)
          for (int i = row * 8 + lane; i < kTile * 8; i += 32)
            *reinterpret_cast<uint4*>(stage + c * C::CHUNK_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();  // the products read V through the async proxy
        __syncwarp();
      };
      auto next_s = [&](int t, int j) {  // K block j has arrived
        if (!ok || !active(t)) return;
        if (C::kApart && j > 0) ok = wait_all(&s_read[t], (j - 1) & 1, kDevTimeoutAccEmpty);
        if (ok) issue_s(t, j);
      };
      if (blocks > 0) {
        ok = arrived(0);
        for (int t = t0; t < t1; ++t) next_s(t, 0);
        if (ok) release(0);
      }
      for (int j = 0; j < blocks && ok; ++j) {
        const bool more = j + 1 < blocks;
        if (more) ok = arrived(2 * (j + 1));
        if (C::kApart && more) {
          next_s(t0, j + 1);
          if (ok) release(2 * (j + 1));
        }
        ok = ok && arrived(2 * j + 1);
        if (ok && (begin + j + 1) * kTile > common && common % box_rows) clear(j);
        for (int t = t0; t < t1; ++t) {
          if (ok && active(t)) {
            ok = wait_all(&p_full[t], j & 1, kDevTimeoutAccFull);
            if (ok) issue_pv(t, j);
          }
          if (!C::kApart && more) next_s(t, j + 1);  // behind P V in the same pipe: P's columns are free
        }
        if (ok) {
          release(2 * j + 1);
          if (!C::kApart && more) release(2 * (j + 1));
        }
      }
      if (!ok) {
        if (one) tc_commit(&drain[t0]);
        wait_for(&drain[t0], 0, kDevTimeoutAccFull);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---------------- softmax and output ----------------
    const int t = warp >> 2, quarter = warp & 3;
    const int first_query = t * kTile + quarter * 32;  // of this warp, from the tiles' first one
    const bool mine = m0 + first_query + lane < queries && t < tiles_here;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lane_base + C::S_COL + t * kTile, p_at = lane_base + C::P_COL + t * C::P_STEP,
                   o_at = lane_base + C::O_COL + t * D;
    int limit = 0;  // keys that the query sees
    if (mine) {
      int s;
      limit = min(common, row_length(p, b0 + (int)at_query.row_of(first_query + lane), &s));
    }
    const float sc = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    bool ok = t < tiles_here;
    for (int c = 0; c < blocks && ok; ++c) {
      if (!wait_for(&s_full[t], c & 1, kDevTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const unsigned there = page_bits[c & 7];
      uint32_t s[4][32];
#pragma unroll
      for (int x = 0; x < 4; ++x) tmem_ld32_issue(s_at + x * 32, s[x]);
#pragma unroll
      for (int x = 0; x < 4; ++x) tmem_wait_ld(s[x]);
      if constexpr (C::kApart) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_read[t]);
      }
      const int left = limit - (begin + c) * kTile;  // keys of this block that the query sees
      if (__any_sync(0xffffffffu, left < kTile || there != 0xffu)) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (x * 32 + k >= left || !(there >> (x * 2 + k / 16) & 1)) s[x][k] = 0xff800000u;  // -inf
      }
      float top[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        top[x] = fmaxf(__uint_as_float(s[x][0]), __uint_as_float(s[x][1]));
#pragma unroll
        for (int k = 2; k < 32; k += 2) top[x] = max3(top[x], __uint_as_float(s[x][k]), __uint_as_float(s[x][k + 1]));
      }
      const float bm = max3(fmaxf(top[0], top[1]), top[2], top[3]) * sc;
      uint64_t sum[4];
      uint32_t pk[64];
      const uint64_t sc2 = pair2(sc, sc);
      auto quarter_of_p = [&](int x, float shift) {
        const uint64_t shift2 = pair2(-shift, -shift);
        sum[x] = 0;
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const uint64_t e = fma2(pair2(__uint_as_float(s[x][k]), __uint_as_float(s[x][k + 1])), sc2, shift2);
          float2 y;
          if ((k / 2) % 8 < kPoly) {
            y = exp2_pair<E::kHalf>(e);
          } else {
            y = split2(e);
            y = make_float2(ex2_approx(y.x), ex2_approx(y.y));
          }
          sum[x] = add2(sum[x], pair2(y.x, y.y));
          pk[x * 16 + k / 2] = E::pack(y.x, y.y);  // the one rounding inside the sum, half a step per term
        }
      };
      const bool raise = bm > m + kRaise<T>;  // -inf + 8 is -inf: any finite score raises it
      const bool any_raise = __any_sync(0xffffffffu, raise);
      float alpha = 1.f;
      if (raise) {
        alpha = ex2_approx(m - bm);
        m = bm;
        l *= alpha;
      }
      auto rescale = [&]() {  // O of the blocks so far, whose P V is done
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          uint32_t o[32];
          tmem_ld32_issue(o_at + x * 32, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tmem_st32(o_at + x * 32, o);
        }
      };
      const float shift = softmax_shift(m) - kTileLift<T>;
#pragma unroll
      for (int x = 0; x < 4; ++x) quarter_of_p(x, shift);
      const float2 part = split2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
      l += part.x + part.y;
      if (c > 0) {
        if (!wait_for(&pv_done[t], (c - 1) & 1, kDevTimeoutAccFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (any_raise) rescale();
      }
      tmem_st32(p_at, pk);
      tmem_st32(p_at + 32, pk + 32);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    const int splits = p.prefix_splits + p.own_splits;
    auto slot_of = [&](int r) {  // range `split` of the query r behind the warp's first one
      return ((b0 + at_query.row_of(first_query + r)) * p.heads + kvh * p.per + at_query.head_of(first_query + r)) * splits + split;
    };
    if (blocks == 0) {
      if (mine) p.part_ml[slot_of(lane)] = make_float2(-INFINITY, 0.f);
    } else if (ok && wait_for(&pv_done[t], (blocks - 1) & 1, kDevTimeoutAccFull)) {
      tc_fence_after();
      // No score above -inf: the masked keys left at most 2^-136 each in the sum. Only a score of
      // NaN, which the maximum passes over, leaves more (or NaN), and then the row is NaN.
      if (m == -INFINITY) l = l < 1.f ? 0.f : __int_as_float(0x7fffffff);
      if (mine) p.part_ml[slot_of(lane)] = make_float2(m - kTileLift<T>, l);
      // O through this tile's Q, which no product reads any more: 32 columns of 32 rows,
      // so that a store covers four rows' 128 bytes
      const unsigned mine_rows = __ballot_sync(0xffffffffu, mine && !(m == -INFINITY && l == 0.f));
      uint8_t* stage = sQ + t * C::TILE_BYTES + quarter * (32 * 128);
      long long to[8];  // this lane's rows of a store
#pragma unroll
      for (int i = 0; i < 8; ++i) to[i] = slot_of(i * 4 + (lane >> 3)) * D + (lane & 7) * 4;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint32_t o[32];
        tmem_ld32_issue(o_at + x * 32, o);
        tmem_wait_ld(o);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<uint4*>(stage + tile_at<64>(lane, q)) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3), ch = lane & 7;
          const uint4 y = *reinterpret_cast<const uint4*>(stage + tile_at<64>(r, ch));
          if (mine_rows >> r & 1) *reinterpret_cast<uint4*>(p.part_o + to[i] + x * 32) = y;
        }
        __syncwarp();
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(*tmem_slot, 512);
}

template <typename T, int D>
int launch(const SharedParams& p, cudaStream_t s) {
  using C = Cfg<D>;
  static std::atomic<bool> attr[64];  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaError_t e =
        cudaFuncSetAttribute(shared_prefix_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr[dev & 63] = true;
  }
  const int P = p.g.page_size;
  const int box_rows = P % kTile == 0 ? kTile : kTile % P == 0 ? P : kUnit;  // rows of one page, dividing a block
  const long long pool_rows = (long long)p.g.pages * page_tiles(p.g) * P;
  CUtensorMap map;
  OASIS_TRY(make_tma_16bit_3d(&map, p.pool, Elem<T>::kHalf, D, pool_rows, 1, D, pool_rows * D, 64, box_rows, 1));
  const long long blocks = (long long)p.groups * p.g.kv_heads * p.prefix_splits * p.tiles;
  cudaError_t e = launch_pdl(shared_prefix_tc_kernel<T, D>, dim3((unsigned)blocks), dim3(kSharedThreads), C::SMEM, s, map, p,
                             box_rows, (int)pool_rows);
  if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "shared_prefix_tc_kernel: %s", cudaGetErrorString(e));
  return check_launch("shared_prefix_tc_kernel");
}

}  // namespace

int shared_prefix_tc_launch(const SharedParams& p, bool half, cudaStream_t s) {
  if (half) return p.g.head_dim == 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
  return p.g.head_dim == 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
}

int read_device_error_shared(int reset) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_wait_error, sizeof(int));
  if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "device_error: %s", cudaGetErrorString(e));
  if (reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_wait_error, &zero, sizeof(int));
    if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "device_error reset: %s", cudaGetErrorString(e));
  }
  return v;
}

}  // namespace oasis
