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

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile of D-element rows whose
// chunks are XOR-swizzled by the row, so that eight rows' same chunk hits all banks.
template <int D>
__device__ __forceinline__ int tile_at(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ (row & 7)) << 4);
}

// What a running softmax subtracts for maximum m: m, or 0 while every value was -inf.
__device__ __forceinline__ float softmax_shift(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ bool finite_f(float x) { return fabsf(x) <= 3.402823466e38f; }

// One query row of D = 32 DV dims, key by key, by a whole warp (lane holds dims
// [lane DV, lane DV + DV)). `key(j)` and `val(j)` give lane-independent row pointers
// of the j-th visible key or null for one to skip. The tiled kernels multiply a
// masked probability of zero with whatever the masked value row holds, which is
// wrong where that is an infinity or NaN, and their sum of values is divided only at the
// end, so that it overflows where values are near bf16's largest; rows whose result is not
// finite are done again here, where only visible keys take part and o is the weighted mean
// of the keys so far: never larger than they are. Zeros without a key; NaN where keys
// score -inf all of them, as the formula's 0 / 0.
template <typename T, int D, typename Key, typename Val>
__device__ __noinline__ void row_by_keys(const T* q, float scale_log2, long long keys, Key key, Val val,
                                         float (&o)[D / 32]) {
  constexpr int DV = D / 32;
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
  for (long long j = 0; j < keys; ++j) {
    const T* kp = key(j);
    if (!kp) continue;
    any = true;
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < DV; d += 2) {
      const float2 x = Elem<T>::unpack(*reinterpret_cast<const uint32_t*>(kp + lane * DV + d));
      s = fmaf(qv[d], x.x, fmaf(qv[d + 1], x.y, s));
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= scale_log2;
    const float mn = (s != s) ? s : fmaxf(m, s);  // a NaN score makes the row NaN
    const float sh = softmax_shift(mn), a = l * exp2f(m - sh), p = exp2f(s - sh);
    const T* vp = val(j);
    m = mn;
    l = a + p;
    const float keep = l == 0.f ? 1.f : a / l, add = l == 0.f ? 0.f : p / l;  // 0: no score above -inf yet
#pragma unroll
    for (int d = 0; d < DV; d += 2) {
      const float2 x = Elem<T>::unpack(*reinterpret_cast<const uint32_t*>(vp + lane * DV + d));
      o[d] = o[d] * keep + add * x.x;
      o[d + 1] = o[d + 1] * keep + add * x.y;
    }
  }
  if (any && l == 0.f)
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] = __int_as_float(0x7fffffff);
}

}  // namespace oasis
