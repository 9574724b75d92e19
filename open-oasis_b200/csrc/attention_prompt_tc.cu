// Causal attention over packed prompts on the 5th-generation tensor cores: the kernel
// for sequences that are not short (attention_prompt.cu has the formula and the
// kernel for short ones).
//
// A block takes two tiles of 128 query rows that read the same keys: the same rows of
// two heads of one key head where heads come in even groups (both tiles then see the
// same key range), otherwise 256 consecutive rows of one head. Keys come in blocks of
// 128 from the first key that the first row sees; per tile and block
//   S = Q K^T        tcgen05.mma 128 x 128 x D, fp32 in TMEM
//   P = exp2(S c - m) one TMEM lane (query row) per thread, S read once into
//                    registers, P written back to TMEM as the 16-bit A operand
//   O += P V         tcgen05.mma 128 x D x 128 accumulating in TMEM, V as it lies in
//                    memory (MN-major B)
// While one tile is in the softmax the other one's products run. The maximum m that is
// subtracted is only raised when a row exceeds it by more than 2^8 (fp16: 2^6): P stays below
// 2^8 (fp16, where it is lifted besides: 2^15), the sum is exact to fp32 either way, and O in
// TMEM is rescaled a few times per row instead of once per block. With D = 64 TMEM holds S, P
// and O of both tiles apart, so the next S is computed during the softmax; with D = 128 P
// takes S's columns.
//
// Warps 0-3 and 4-7: softmax and output of tile 0 and 1. Warp 8 loads Q, K and V by TMA
// (128-byte swizzle, K and V blocks in one ring). Warps 9 and 10 (D = 128: 9 alone) issue
// the MMAs, warp 9 owns TMEM. Their warpgroup gives registers to the other two: 168 per
// thread at launch become 208, 208 and 88 (a row's 128 scores stay in registers).
// Every wait is bounded and leaves a code in this file's error word.
//
// Bound: with D = 64 the exponentials (one per score, 16 per clock and SM) take twice
// the tensor time, with D = 128 as long as it. 16384 tokens, 16 heads of 64: 674 us,
// 815 TFLOP/s; 16 heads of 128: 1005 us, 1094 TFLOP/s; 6042 tokens in 4 sequences, 32 / 8
// heads of 128: 261 us, 1129 TFLOP/s (up to 316 us where the power cap holds the clock at 1.55
// of 1.97 GHz); 9216 tokens in 8 sequences, 16 heads of 64: 94 us. With D = 64 a pair of tiles
// takes about 2800 clocks a key block where the exponentials left to the special-function unit
// take 1536: S's load, maximum, exponentials and P's store follow one another in a warp.
// Measured slower: all exponentials on that unit, or 3 and 4 of 8 on the FMA pipe; a row
// in two threads (16 softmax warps); the two tiles held half a block apart; P handed over
// in halves (D = 128, 271 -> 276 us); the rescaling ahead of the exponentials (spills at
// D = 128); one block per SM that takes tiles in turn, in snake order or as SMs fall free.
#include "../../include/oasis_b200.h"
#include "attention_prompt.cuh"
#include "attention_tc.cuh"
#include "gemm.cuh"
#include "prompt_unit.cuh"
#include "status.h"

namespace oasis {
namespace {

constexpr int kPromptThreads = 384;
// Of every eight pairs of exponentials this many go to the FMA pipe, the others to the
// special-function unit, which alone would be the bound.
constexpr int kPoly = 2;

template <int D>
struct Cfg {
  static constexpr int CHUNKS = D / 64;               // 64-column chunks: 128 bytes of a row
  static constexpr int CHUNK_BYTES = kTile * 128;
  static constexpr int TILE_BYTES = CHUNKS * CHUNK_BYTES;
  static constexpr int STAGES = D == 64 ? 8 : 5;
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM = 1024 + (2 + STAGES) * TILE_BYTES + BAR_BYTES;
  static_assert(SMEM <= 232448, "shared memory");
  static constexpr bool kApart = D == 64;             // S and P in columns of their own
  static constexpr int S_COL = 0;                     // + 128 per tile
  static constexpr int P_COL = kApart ? 256 : 0;      // + P_STEP per tile
  static constexpr int P_STEP = kApart ? 64 : 128;
  static constexpr int O_COL = kApart ? 384 : 256;    // + D per tile
};

static_assert(kPromptTile == kTile, "tiles");

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PromptParams p, int pair_heads) {
  using C = Cfg<D>;
  using E = Elem<T>;
  extern __shared__ uint8_t smem_raw[];
  pdl_wait();
  const int end = min(p.rows, p.cu[p.n]);
  // Work: a row tile (pair) x a head (pair), the last rows first: in a sequence those
  // see the most keys, and the blocks that finish last should be short.
  const int head_units = pair_heads ? p.heads / 2 : p.heads;
  const int tile_rows = pair_heads ? kTile : 2 * kTile;
  const int at = blockIdx.x / head_units;
  const PromptUnit u = prompt_unit(p.cu, p.n, pair_heads, end, blockIdx.x - at * head_units,
                                   (p.rows + tile_rows - 1) / tile_rows - 1 - at);
  if (u.blocks == 0) return;  // the whole block

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + 2 * C::TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + C::STAGES * C::TILE_BYTES);
  uint64_t* q_full = bars;         // [2]
  uint64_t* s_full = bars + 2;     // [2]
  uint64_t* s_read = bars + 4;     // [2] softmax has S in registers (kApart)
  uint64_t* p_full = bars + 6;     // [2]
  uint64_t* pv_done = bars + 8;    // [2]
  uint64_t* drain = bars + 10;     // [2]
  uint64_t* kv_full = bars + 16;   // [STAGES <= 8]
  uint64_t* kv_empty = bars + 24;  // [STAGES <= 8]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
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
    // What follows starts early only once this block has its TMEM: a kernel that took some
    // of it first and then waited for this grid would never get to give it back.
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    pdl_trigger();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = 0;  // all 512 columns are this block's, so they begin at 0
  const int kvh0 = u.head[0] / (p.heads / p.kv_heads);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8 && lane == 0) {
      // ---------------- TMA ----------------
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row) {
        mbar_arrive_expect_tx(bar, C::TILE_BYTES);
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) tma_load_3d(dst + c * C::CHUNK_BYTES, map, bar, c * 64, head, row);
      };
      const int total = 2 * u.blocks;
      int issued = 0;
      bool ok = true;
      auto next = [&]() {
        const int st = issued % C::STAGES;
        if (issued >= C::STAGES && !wait_for(&kv_empty[st], ((issued / C::STAGES) & 1) ^ 1, kDevTimeoutSmemEmpty))
          return false;
        load(sKV + st * C::TILE_BYTES, issued & 1 ? &tmV : &tmK, &kv_full[st], kvh0, u.begin + (issued >> 1) * kTile);
        ++issued;
        return true;
      };
      if (u.has(0)) load(sQ, &tmQ, &q_full[0], u.head[0], u.r0[0]);
      ok = next();
      if (u.has(1)) load(sQ + C::TILE_BYTES, &tmQ, &q_full[1], u.head[1], u.r0[1]);
      while (ok && issued < total) ok = next();
      if (!ok) {  // gave up: the copies in flight land before the block ends
        for (int t = 0; t < 2; ++t)
          if (u.has(t)) wait_for(&q_full[t], 0, kDevTimeoutTmaFull);
        for (int i = max(0, issued - C::STAGES); i < issued; ++i)
          wait_for(&kv_full[i % C::STAGES], (i / C::STAGES) & 1, kDevTimeoutTmaFull);
      }
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
      const int blocks = uniform(u.blocks);
      const int first[2] = {uniform(u.first[0]), uniform(u.first[1])}, last[2] = {uniform(u.last[0]), uniform(u.last[1])};
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
      auto active = [&](int t, int j) { return j >= first[t] && j < last[t]; };
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
        const uint32_t more = j > first[t], d = C::O_COL + t * D, pa = C::P_COL + t * C::P_STEP;
        if (one) {
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k) mma_ts(d, pa + k * 8, va + (uint64_t)(k * 2048 >> 4), idPV, k > 0 ? 1u : more);
          tc_commit(&pv_done[t]);
        }
      };
      // Rows of V block j behind the last sequence hold anything: zeros instead, like their
      // probabilities, since an infinity or NaN there would send the tile's rows to the
      // repair. It is the unit's last block, so that its stage is not loaded again; with two
      // warps both write the same zeros, each ahead of its own products.
      auto clear = [&](int j) {
        const int row = max(0, end - (u.begin + j * kTile));
        uint8_t* stage = sKV + (2 * j + 1) % C::STAGES * C::TILE_BYTES;
        for (int c = 0; c < C::CHUNKS; ++c)
          for (int i = row * 8 + lane; i < kTile * 8; i += 32)
            *reinterpret_cast<uint4*>(stage + c * C::CHUNK_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();  // the products read V through the async proxy
        __syncwarp();
      };
      auto next_s = [&](int t, int j) {  // K block j has arrived
        if (!ok || !active(t, j)) return;
        if (j == first[t]) ok = wait_all(&q_full[t], 0, kDevTimeoutTmaFull);
        if (ok && C::kApart && j > first[t]) ok = wait_all(&s_read[t], (j - 1 - first[t]) & 1, kDevTimeoutAccEmpty);
        if (ok) issue_s(t, j);
      };
      ok = arrived(0);
      for (int t = t0; t < t1; ++t) next_s(t, 0);
      if (ok) release(0);
      for (int j = 0; j < blocks && ok; ++j) {
        const bool more = j + 1 < blocks;
        if (more) ok = arrived(2 * (j + 1));
        if (C::kApart && more) {
          next_s(t0, j + 1);
          if (ok) release(2 * (j + 1));
        }
        ok = ok && arrived(2 * j + 1);
        if (ok && u.begin + (j + 1) * kTile > end) clear(j);
        for (int t = t0; t < t1; ++t) {
          if (ok && active(t, j)) {
            ok = wait_all(&p_full[t], (j - first[t]) & 1, kDevTimeoutAccFull);
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
    const int row = u.r0[t] + quarter * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lane_base + C::S_COL + t * kTile, p_at = lane_base + C::P_COL + t * C::P_STEP,
                   o_at = lane_base + C::O_COL + t * D;
    int lo = 0x3fffffff;  // first key that the row sees; beyond all keys where the row is nobody's
    if (row < end) {
      const int i = last_not_above(p.cu, p.n, row);
      const int a = p.cu[i];
      if (a >= 0 && a <= row && row < p.cu[i + 1]) lo = a;
    }
    const unsigned span = lo <= row ? row - lo : 0;  // sees keys lo .. lo + span
    const float sc = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = u.first[t]; j < u.last[t]; ++j) {
      const int c = j - u.first[t];
      if (!wait_for(&s_full[t], c & 1, kDevTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
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
      const int kb = u.begin + j * kTile;
      if (__any_sync(0xffffffffu, kb < lo || kb + kTile - 1 > row)) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if ((unsigned)(kb - lo + x * 32 + k) > span) s[x][k] = 0xff800000u;  // -inf
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
    const int blocks = u.last[t] - u.first[t];
    if (ok && blocks > 0 && wait_for(&pv_done[t], (blocks - 1) & 1, kDevTimeoutAccFull)) {
      tc_fence_after();
      const bool mine = lo <= row;
      bool good = l > 0.f && finite_f(l) && m != -INFINITY;
      const float inv = 1.f / l;
      // Through this tile's Q, which no product reads any more, so that a store covers
      // four rows' 128 bytes: a thread per row writing its own 16 bytes at a time
      // touched 32 lines a store and took 2 to 3.5 us a tile.
      const unsigned mine_rows = __ballot_sync(0xffffffffu, mine);
      uint8_t* stage = sQ + t * C::TILE_BYTES + quarter * (32 * 128);
      T* out = static_cast<T*>(p.out) + u.head[t] * p.o_head + (long long)(u.r0[t] + quarter * 32) * p.o_row;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint32_t o[32];
        tmem_ld32_issue(o_at + x * 32, o);
        tmem_wait_ld(o);
#pragma unroll
        for (int k = 0; k < 32; ++k) good = good && finite_f(__uint_as_float(o[k]));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = E::pack(__uint_as_float(o[8 * q + 2 * e]) * inv, __uint_as_float(o[8 * q + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + tile_at<64>(lane, (x & 1) * 4 + q)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (x & 1) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3), ch = lane & 7;
            const uint4 y = *reinterpret_cast<const uint4*>(stage + tile_at<64>(r, ch));
            if (mine_rows >> r & 1) *reinterpret_cast<uint4*>(out + r * p.o_row + (x >> 1) * 64 + ch * 8) = y;
          }
          __syncwarp();
        }
      }
      unsigned bad = __ballot_sync(0xffffffffu, mine && !good);
      const T* k0 = static_cast<const T*>(p.k) + kvh0 * p.k_head;
      const T* v0 = static_cast<const T*>(p.v) + kvh0 * p.v_head;
      while (bad) {  // rows to be done key by key
        const int r = __ffs(bad) - 1;
        bad &= bad - 1;
        const int at = u.r0[t] + quarter * 32 + r, from = __shfl_sync(0xffffffffu, lo, r);
        float acc[D / 32];
        __syncwarp();  // the row's first result is written
        row_by_keys<T, D, 8>(
            static_cast<const T*>(p.q) + u.head[t] * p.q_head + at * p.q_row, sc, at - from + 1,
            [&](long long x) { return k0 + (from + x) * p.k_row; }, [&](long long x) { return v0 + (from + x) * p.v_row; },
            acc);
        T* o = static_cast<T*>(p.out) + u.head[t] * p.o_head + at * p.o_row;
#pragma unroll
        for (int d = 0; d < D / 32; d += 2)
          *reinterpret_cast<uint32_t*>(o + lane * (D / 32) + d) = E::pack(acc[d], acc[d + 1]);
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
int launch(const PromptParams& p, cudaStream_t s) {
  using C = Cfg<D>;
  static std::atomic<bool> attr[64];  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(prompt_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr[dev & 63] = true;
  }
  const bool half = Elem<T>::kHalf;
  CUtensorMap tq, tk, tv;
  OASIS_TRY(make_tma_16bit_3d(&tq, p.q, half, D, p.heads, p.rows, p.q_head, p.q_row, 64, 1, kTile));
  OASIS_TRY(make_tma_16bit_3d(&tk, p.k, half, D, p.kv_heads, p.rows, p.k_head, p.k_row, 64, 1, kTile));
  OASIS_TRY(make_tma_16bit_3d(&tv, p.v, half, D, p.kv_heads, p.rows, p.v_head, p.v_row, 64, 1, kTile));
  const int pair_heads = (p.heads / p.kv_heads) % 2 == 0;
  const int rows = pair_heads ? kTile : 2 * kTile;
  const long long blocks = ((long long)p.rows + rows - 1) / rows * (pair_heads ? p.heads / 2 : p.heads);
  cudaError_t e = launch_pdl(prompt_tc_kernel<T, D>, dim3((unsigned)blocks), dim3(kPromptThreads), C::SMEM, s, tq, tk, tv,
                             p, pair_heads);
  if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "prompt_tc_kernel: %s", cudaGetErrorString(e));
  return check_launch("prompt_tc_kernel");
}

}  // namespace

int prompt_tc_launch(const PromptParams& p, cudaStream_t s) {
  if (p.dtype == OASIS_DTYPE_BF16)
    return p.head_dim == 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
  return p.head_dim == 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
}

int read_device_error_prompt(int reset) {
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
