// Pieces shared by the attention kernels over packed sequences and paged caches:
// 16-bit matrix fragments for both element types, swizzled shared-memory tiles, and
// one query row worked out key by key.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace oasis {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Every copy of this thread, committed to a group or not.
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}

// Element type of a kernel: conversions and the m16n8k16 product.
template <typename T>
struct Elem;

template <>
struct Elem<__nv_bfloat16> {
  static constexpr bool kHalf = false;
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Elem<__half> {
  static constexpr bool kHalf = true;
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Probabilities of the mma.sync kernels, and so their sums, are 2^kLift times those relative to
// the running maximum. fp16's normal numbers end at 2^-14, and a weight below that is
// rounded by more than half a step of its own: where one key outweighs the others by 14 to 16
// nats, what those add was off by 17 to 67 half steps. 2^15 is the most that the type holds of
// the largest weight; weights are whole down to 2^-29 of it. bf16 has fp32's exponents.
template <typename T>
constexpr float kLift = Elem<T>::kHalf ? 15.f : 0.f;

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile of D-element rows whose
// chunks are XOR-swizzled by the row, so that eight rows' same chunk hits all banks.
template <int D>
__device__ __forceinline__ int tile_at(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ (row & 7)) << 4);
}

// What a running softmax subtracts for maximum m: m, or 0 while every value was -inf.
__device__ __forceinline__ float softmax_shift(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ bool finite_f(float x) { return fabsf(x) <= 3.402823466e38f; }

// One query row of D = 32 DV dims by a whole warp (lane holds dims [lane DV, lane DV + DV)).
// `key(j)` and `val(j)` give the row pointers of the j-th visible key or null for one to skip.
// The tiled kernels multiply a masked probability of zero with whatever the masked value row
// holds, which is wrong where that is an infinity or NaN, and their sum of values is divided
// only at the end, so that it overflows where values are near bf16's largest; rows whose
// result is not finite are done again here, where only visible keys take part and o is the
// weighted mean of the keys so far: never larger than they are. Zeros without a key; NaN
// where keys score -inf all of them, as the formula's 0 / 0, and from the first score of
// NaN or +inf on, where every further sum is NaN.
// 32 keys at a time, a lane for each one's score, BATCH 16-byte loads of a key and BATCH
// value rows in flight (2 where the calling kernel has few registers): key by key through the
// whole warp, each one's loads behind the shuffles of the one before, a row of 2000 keys
// took 0.55 us a key.
template <typename T, int D, int BATCH, typename Key, typename Val>
__device__ __noinline__ void row_by_keys(const T* q, float scale_log2, long long keys, Key key, Val val,
                                         float (&o)[D / 32]) {
  constexpr int DV = D / 32;
  const float nan = __int_as_float(0x7fffffff);
  const int lane = threadIdx.x & 31;
  float qv[DV], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < DV; d += 2) {
    const float2 x = Elem<T>::unpack(*reinterpret_cast<const uint32_t*>(q + lane * DV + d));
    qv[d] = x.x;
    qv[d + 1] = x.y;
    o[d] = o[d + 1] = 0.f;
  }
  bool any = false;
  for (long long j0 = 0; j0 < keys; j0 += 32) {
    const long long j = j0 + lane;
    const T *kp = nullptr, *vp = nullptr;
    if (j < keys) kp = key(j), vp = val(j);
    const unsigned there = __ballot_sync(0xffffffffu, kp != nullptr);
    if (!there) continue;
    any = true;
    float s = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < D / 8; c0 += BATCH) {
      uint4 x[BATCH];
#pragma unroll
      for (int c = 0; c < BATCH; ++c)
        x[c] = kp ? reinterpret_cast<const uint4*>(kp)[c0 + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < BATCH; ++c) {
        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 y = Elem<T>::unpack(w[e]);
          const int d = 2 * e % DV, from = ((c0 + c) * 8 + 2 * e) / DV;
          s = fmaf(__shfl_sync(0xffffffffu, qv[d], from), y.x, s);
          s = fmaf(__shfl_sync(0xffffffffu, qv[d + 1], from), y.y, s);
        }
      }
    }
    s = kp ? s * scale_log2 : -INFINITY;
    if (__any_sync(0xffffffffu, !(s < INFINITY))) {
#pragma unroll
      for (int d = 0; d < DV; ++d) o[d] = nan;
      return;
    }
    float mn = fmaxf(m, s);
#pragma unroll
    for (int w = 16; w; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
    const float sh = softmax_shift(mn), a = l * exp2f(m - sh), p = exp2f(s - sh);
    float sum = p;
#pragma unroll
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    m = mn;
    l = a + sum;
    // 0: no score above -inf yet; their weight is zero, which an infinite value makes NaN
    const float keep = l == 0.f ? 1.f : a / l, weight = l == 0.f ? 0.f : p / l;
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] *= keep;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += BATCH) {
      uint32_t y[BATCH][DV / 2];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const T* v = reinterpret_cast<const T*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vp), i0 + i));
        const bool in = there >> (i0 + i) & 1;
#pragma unroll
        for (int d = 0; d < DV / 2; ++d) y[i][d] = in ? reinterpret_cast<const uint32_t*>(v + lane * DV)[d] : 0u;
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float f = __shfl_sync(0xffffffffu, weight, i0 + i);
#pragma unroll
        for (int d = 0; d < DV / 2; ++d) {
          const float2 x = Elem<T>::unpack(y[i][d]);
          o[2 * d] = fmaf(f, x.x, o[2 * d]);
          o[2 * d + 1] = fmaf(f, x.y, o[2 * d + 1]);
        }
      }
    }
  }
  if (any && l == 0.f)
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] = nan;
}

}  // namespace oasis
