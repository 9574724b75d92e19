// Causal attention over whole prompts: packed sequences of different lengths, grouped
// heads. Row i of sequence rows [a, b), head h, key head h / (heads / kv_heads):
//   x_j = scale q_i . k_j for a <= j <= i;  o_i = sum_j exp(x_j - max x) v_j / sum_j exp(x_j - max x)
//
// Both kernels tile the packed row stream, not the sequences: a tile of query rows
// takes the keys from the first key that its first row sees up to its own last row,
// and a per-row bound masks keys of earlier sequences. So sequences of a few tokens
// share tiles and there is no tile that is mostly empty.
//
// prompt_rows_kernel: 64 query rows x one head per block, a warp per 16 rows, mma.sync
// fragments with the running softmax in registers. For short sequences, where a tile
// sees little more than its own rows and the least is reading q, k, v and writing o:
// 37584 rows of 9216 sequences of 1 to 8 tokens, 16 heads of 64, 308 MB: 77 us (4.0 TB/s;
// a copy of as many bytes 47 us). What is left is issue, 51 % of the cycles, and the
// latency of a block's offsets and loads: six blocks an SM (D = 128: three) hide part of
// it; seven or eight with fewer registers, and several heads per block with the next
// one's loads ahead (115 us), were slower.
#include "../../include/oasis_b200.h"
#include "attention_prompt.cuh"
#include "attention_rows.cuh"
#include "gemm.cuh"
#include "pages.cuh"
#include "status.h"

namespace oasis {
namespace {

constexpr int kRowsTile = 64;   // query rows of a block
// Keys of a step. The first step's are the tile's own rows and 16 before them: they are
// loaded before it is known which sequences the rows belong to, and sequences of up to
// 17 tokens need no other. Further steps go back from there. One buffer: what hides the
// loads is the other blocks of the SM.
constexpr int kRowsBefore = 16;
constexpr int kRowsKeys = kRowsTile + kRowsBefore;
constexpr int kRowsThreads = 128;

// Up to this length the rows kernel is taken. 8192 tokens, 16 heads of 64, this kernel
// against the tcgen05 one: 20.9 / 30.2 us at length 64, 33.1 / 35.9 at 192, 39.7 / 32.4 at
// 256; 32 / 8 heads of 128: 65.4 / 77.8 us at 48, 79.1 / 75.6 at 96, 82.7 / 63.9 at 128.
constexpr int short_length(int head_dim) { return head_dim == 64 ? 192 : 96; }

template <int D>
constexpr int rows_smem() {
  return (kRowsTile + 2 * kRowsKeys) * D * 2;  // Q (then O), K and V
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowsThreads, D == 64 ? 6 : 3) prompt_rows_kernel(PromptParams p) {
  using E = Elem<T>;
  constexpr int CH = D / 8;   // 16-byte chunks of a row
  constexpr int KS = D / 16;  // k steps of Q K^T
  constexpr int NT = D / 8;   // 8-wide column tiles of O
  constexpr int Q_BYTES = kRowsTile * D * 2, K_BYTES = kRowsKeys * D * 2;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int first[kRowsTile];  // first key that a row sees; row + 1 where the row is nobody's
  __shared__ int lowest[2];
  __shared__ int starts[kRowsThreads];  // offsets from the first row's sequence on
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x % p.heads, r0 = (int)(blockIdx.x / p.heads) * kRowsTile;
  const T* q = static_cast<const T*>(p.q) + head * p.q_head;
  const int kvh = head / (p.heads / p.kv_heads);
  const T* k = static_cast<const T*>(p.k) + kvh * p.k_head;
  const T* v = static_cast<const T*>(p.v) + kvh * p.v_head;

  uint8_t* const sk = sm + Q_BYTES;
  uint8_t* const sv = sk + K_BYTES;
  // A thread's 16-byte chunks lie STEP rows apart, in the same swizzled column.
  constexpr int STEP = kRowsThreads / CH;
  static_assert(16 % STEP == 0 && STEP % 8 == 0 && kRowsTile % STEP == 0 && kRowsKeys % STEP == 0, "chunks of a thread");
  const int tr = tid / CH, tc = tid % CH;
  {
    const T* from = q + (long long)(r0 + tr) * p.q_row + tc * 8;
    uint8_t* to = sm + tile_at<D>(tr, tc);
#pragma unroll
    for (int i = 0; i < kRowsTile / STEP; ++i) {
      const bool ok = r0 + tr + i * STEP < p.rows;
      cp_async16(to + i * STEP * D * 2, ok ? from : q, ok);
      from += STEP * p.q_row;
    }
  }
  auto load = [&](int at) {
    const T *k_from = k + (long long)(at + tr) * p.k_row + tc * 8, *v_from = v + (long long)(at + tr) * p.v_row + tc * 8;
    uint8_t* to = sk + tile_at<D>(tr, tc);
#pragma unroll
    for (int i = 0; i < kRowsKeys / STEP; ++i) {
      const bool ok = (unsigned)(at + tr + i * STEP) < (unsigned)p.rows;
      cp_async16(to + i * STEP * D * 2, ok ? k_from : k, ok);
      cp_async16(to + K_BYTES + i * STEP * D * 2, ok ? v_from : v, ok);
      k_from += STEP * p.k_row;
      v_from += STEP * p.v_row;
    }
  };
  load(r0 - kRowsBefore);
  const int end = min(p.rows, p.cu[p.n]);
  if (r0 >= end) {
    cp_async_wait_all();
    return;
  }
  // Rows behind the last sequence hold anything: their values become zeros, like their
  // probabilities, since an infinity or NaN there would send the tile's rows to the repair.
  // A row of a sequence meets those of its own 16 keys only.
  if (r0 + kRowsTile > end) {
    cp_async_wait_all();
#pragma unroll
    for (int i = 0; i < 16 / STEP; ++i) {
      const int row = kRowsBefore + (end - r0) / 16 * 16 + i * STEP + tr;
      if (r0 - kRowsBefore + row >= end) *reinterpret_cast<uint4*>(sv + tile_at<D>(row, tc)) = make_uint4(0, 0, 0, 0);
    }
  }
  // The first row's sequence, a warp probing 32 places at a time; the other rows of the
  // tile belong to it or to the ones behind it.
  int i0 = 0;
  for (int n = p.n; n > 1;) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const bool ok = i < n && p.cu[i0 + i] <= r0;
    const int c = 32 - __clz(__ballot_sync(0xffffffffu, ok) | 1u);  // probes that hold: a run from lane 0
    i0 += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  starts[tid] = p.cu[min(i0 + tid, p.n)];
  __syncthreads();
  if (tid < kRowsTile) {
    const int r = r0 + tid;
    const int k = last_not_above(starts, kRowsThreads, r);
    int i = i0 + k, a = starts[k];
    int b = k + 1 < kRowsThreads ? starts[k + 1] : 0;
    if (k + 1 == kRowsThreads || i >= p.n) {  // behind the offsets at hand, or the last row's
      i = last_not_above(p.cu, p.n, r);
      a = p.cu[i];
      b = p.cu[i + 1];
    }
    const bool mine = r < end && a >= 0 && a <= r && r < b;
    first[tid] = mine ? a : r + 1;
    const int low = __reduce_min_sync(0xffffffffu, first[tid]);
    if (lane == 0) lowest[warp] = low;
  }
  __syncthreads();
  const int k_begin = min(lowest[0], lowest[1]);
  const int wr = warp * 16;  // this warp's first row in the tile
  const int ra = wr + (lane >> 2), rb = ra + 8;
  const int lo_a = first[ra], lo_b = first[rb];
  // keys lo .. lo + span are seen; a row of nobody sees none, its lo lies behind all keys
  const unsigned span_a = lo_a <= r0 + ra ? r0 + ra - lo_a : 0, span_b = lo_b <= r0 + rb ? r0 + rb - lo_b : 0;
  const int from_a = lo_a <= r0 + ra ? lo_a : 0x3fffffff, from_b = lo_b <= r0 + rb ? lo_b : 0x3fffffff;
  const int low = __reduce_min_sync(0xffffffffu, min(lo_a, lo_b)), high = __reduce_max_sync(0xffffffffu, max(lo_a, lo_b));
  uint32_t qa[KS][4];
  float o[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
  float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;

  for (int at = r0 - kRowsBefore, j = 0; j == 0 || at + kRowsKeys > k_begin; at -= kRowsKeys, ++j) {
    if (j) {
      __syncthreads();  // the keys before are done with
      load(at);
    }
    cp_async_wait_all();
    __syncthreads();
    if (j == 0) {
#pragma unroll
      for (int s = 0; s < KS; ++s) ldsm_x4(qa[s], sm + tile_at<D>(wr + (lane & 15), s * 2 + (lane >> 4)));
    }
    // 16 keys at a time: the visible range of this warp's rows is [low, r0 + wr + 15]
#pragma unroll
    for (int h = 0; h < kRowsKeys / 16; ++h) {
      const int kb = at + h * 16;
      if (kb > r0 + wr + 15 || kb + 15 < low) continue;
      float x[2][4] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint32_t b[4];
        ldsm_x4(b, sk + tile_at<D>(h * 16 + (lane & 7) + ((lane >> 4) << 3), s * 2 + ((lane >> 3) & 1)));
        E::mma(x[0], qa[s], b[0], b[1]);
        E::mma(x[1], qa[s], b[2], b[3]);
      }
      const bool whole = kb >= high && kb + 15 <= r0 + wr;
      if (!whole) {
        const int key = kb + (lane & 3) * 2;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((unsigned)(key - (e < 2 ? from_a : from_b) + t * 8 + (e & 1)) > (e < 2 ? span_a : span_b)) x[t][e] = -INFINITY;
      }
      float na = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])) * p.scale_log2;
      float nb = fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3])) * p.scale_log2;
#pragma unroll
      for (int w = 1; w < 4; w <<= 1) {
        na = fmaxf(na, __shfl_xor_sync(0xffffffffu, na, w));
        nb = fmaxf(nb, __shfl_xor_sync(0xffffffffu, nb, w));
      }
      na = fmaxf(na, ma);
      nb = fmaxf(nb, mb);
      float sa = softmax_shift(na), sb = softmax_shift(nb);
      const float fa = ex2_approx(ma - sa), fb = ex2_approx(mb - sb);
      sa -= kLift<T>;
      sb -= kLift<T>;
      ma = na;
      mb = nb;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        x[t][0] = ex2_approx(fmaf(x[t][0], p.scale_log2, -sa));
        x[t][1] = ex2_approx(fmaf(x[t][1], p.scale_log2, -sa));
        x[t][2] = ex2_approx(fmaf(x[t][2], p.scale_log2, -sb));
        x[t][3] = ex2_approx(fmaf(x[t][3], p.scale_log2, -sb));
      }
      la = la * fa + ((x[0][0] + x[0][1]) + (x[1][0] + x[1][1]));  // this lane's share; joined at the end
      lb = lb * fb + ((x[0][2] + x[0][3]) + (x[1][2] + x[1][3]));
      // P as the 16-bit operand: the one rounding inside the sum, half a step of the type per term
      const uint32_t pa[4] = {E::pack(x[0][0], x[0][1]), E::pack(x[0][2], x[0][3]), E::pack(x[1][0], x[1][1]),
                              E::pack(x[1][2], x[1][3])};
#pragma unroll
      for (int t = 0; t < NT; t += 2) {
        uint32_t b[4];
        ldsm_x4_t(b, sv + tile_at<D>(h * 16 + (lane & 15), t + (lane >> 4)));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          o[t + u][0] *= fa;
          o[t + u][1] *= fa;
          o[t + u][2] *= fb;
          o[t + u][3] *= fb;
          E::mma(o[t + u], pa, b[2 * u], b[2 * u + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    la += __shfl_xor_sync(0xffffffffu, la, w);
    lb += __shfl_xor_sync(0xffffffffu, lb, w);
  }
  const float ia = 1.f / la, ib = 1.f / lb;
  bool ok_a = la > 0.f && finite_f(la), ok_b = lb > 0.f && finite_f(lb);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    ok_a = ok_a && finite_f(o[t][0]) && finite_f(o[t][1]);
    ok_b = ok_b && finite_f(o[t][2]) && finite_f(o[t][3]);
    const int c = t ^ (ra & 7);  // ra and rb have the same low bits
    uint8_t* at = sm + ra * (D * 2) + (c << 4) + (lane & 3) * 4;
    *reinterpret_cast<uint32_t*>(at) = E::pack(o[t][0] * ia, o[t][1] * ia);
    *reinterpret_cast<uint32_t*>(at + 8 * D * 2) = E::pack(o[t][2] * ib, o[t][3] * ib);
  }
  const unsigned bad_a = __ballot_sync(0xffffffffu, !ok_a), bad_b = __ballot_sync(0xffffffffu, !ok_b);
  __syncwarp();
  T* out = static_cast<T*>(p.out) + head * p.o_head;
  T* to = out + (long long)(r0 + wr + lane / CH) * p.o_row + lane % CH * 8;
#pragma unroll
  for (int i = 0; i < 16 * CH / 32; ++i) {
    const int r = wr + i * (32 / CH) + lane / CH;
    if (first[r] <= r0 + r) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(sm + tile_at<D>(r, lane % CH));
    to += (32 / CH) * p.o_row;
  }
  if ((bad_a | bad_b) == 0) return;
  __syncwarp();
  for (int r = 0; r < 16; ++r) {  // rows to be done key by key
    if (((r < 8 ? bad_a : bad_b) >> ((r & 7) * 4) & 0xf) == 0) continue;
    const int row = r0 + wr + r, lo = first[wr + r];
    if (lo > row) continue;
    float acc[D / 32];
    row_by_keys<T, D, 2>(
        q + row * p.q_row, p.scale_log2, row - lo + 1, [&](long long x) { return k + (lo + x) * p.k_row; },
        [&](long long x) { return v + (lo + x) * p.v_row; }, acc);
#pragma unroll
    for (int d = 0; d < D / 32; d += 2)
      *reinterpret_cast<uint32_t*>(out + row * p.o_row + lane * (D / 32) + d) = E::pack(acc[d], acc[d + 1]);
  }
}

template <typename T, int D>
int launch_rows(const PromptParams& p, cudaStream_t s) {
  static std::atomic<bool> attr[64];  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaError_t e =
        cudaFuncSetAttribute(prompt_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, rows_smem<D>());
    if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr[dev & 63] = true;
  }
  const long long blocks = ((long long)p.rows + kRowsTile - 1) / kRowsTile * p.heads;
  cudaError_t e = launch_pdl(prompt_rows_kernel<T, D>, dim3((unsigned)blocks), dim3(kRowsThreads), rows_smem<D>(), s, p);
  if (e != cudaSuccess) return set_error(OASIS_ERR_CUDA, "prompt_rows_kernel: %s", cudaGetErrorString(e));
  return check_launch("prompt_rows_kernel");
}

}  // namespace

int prompt_rows_launch(const PromptParams& p, cudaStream_t s) {
  if (p.dtype == OASIS_DTYPE_BF16)
    return p.head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(p, s) : launch_rows<__nv_bfloat16, 128>(p, s);
  return p.head_dim == 64 ? launch_rows<__half, 64>(p, s) : launch_rows<__half, 128>(p, s);
}

}  // namespace oasis

using namespace oasis;

extern "C" int oasis_attention_prompt(const OasisPromptArgs* a, oasis_stream_t stream) {
  OASIS_REQUIRE(a, "attention_prompt: null args");
  OASIS_REQUIRE(a->rows >= 0 && a->n >= 0, "attention_prompt: rows=%d n=%d", a->rows, a->n);
  OASIS_REQUIRE(a->dtype == OASIS_DTYPE_BF16 || a->dtype == OASIS_DTYPE_F16, "attention_prompt: dtype=%d", a->dtype);
  OASIS_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "attention_prompt: head_dim=%d is not 64 or 128", a->head_dim);
  OASIS_REQUIRE(a->kv_heads >= 1 && a->heads >= a->kv_heads && a->heads <= 1024 && a->heads % a->kv_heads == 0,
                "attention_prompt: heads=%d kv_heads=%d", a->heads, a->kv_heads);
  OASIS_REQUIRE(a->scale > 0.f && a->scale <= 3e38f, "attention_prompt: scale=%g", (double)a->scale);
  if (a->rows == 0 || a->n == 0) return OASIS_OK;
  OASIS_REQUIRE(a->q && a->k && a->v && a->out && a->cu, "attention_prompt: null pointer");
  const uintptr_t at = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                       reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->out);
  OASIS_REQUIRE((at & 15) == 0, "attention_prompt: operands not 16-byte aligned");
  const long long strides[8] = {a->q_row_stride, a->q_head_stride, a->k_row_stride,   a->k_head_stride,
                                a->v_row_stride, a->v_head_stride, a->out_row_stride, a->out_head_stride};
  for (long long s : strides)
    OASIS_REQUIRE(s > 0 && s % 8 == 0 && s < (1LL << 36), "attention_prompt: stride %lld is not a positive multiple of 8 elements",
                  s);
  OASIS_REQUIRE(((long long)a->rows + kRowsTile - 1) / kRowsTile * a->heads < (1LL << 31),
                "attention_prompt: %d rows of %d heads are too many", a->rows, a->heads);
  PromptParams p;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.q_row = strides[0];
  p.q_head = strides[1];
  p.k_row = strides[2];
  p.k_head = strides[3];
  p.v_row = strides[4];
  p.v_head = strides[5];
  p.o_row = strides[6];
  p.o_head = strides[7];
  p.rows = a->rows;
  p.cu = a->cu;
  p.n = a->n;
  p.longest = a->longest;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.dtype = a->dtype;
  p.scale_log2 = a->scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->longest <= short_length(a->head_dim) ? prompt_rows_launch(p, st) : prompt_tc_launch(p, st);
}
