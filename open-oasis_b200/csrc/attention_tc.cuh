// Pieces of the attention kernels whose products run on the 5th-generation tensor cores
// with P in tensor memory: bounded waits, operands, exponentials of register pairs.
#pragma once
#include "attention_rows.cuh"

namespace oasis {

constexpr int kTile = 128;  // query rows of a tile, keys of a block
// Base-2 exponents that a score may exceed the subtracted maximum by, and those that P is
// lifted by besides (see kLift): together 15 at most in fp16, where weights are whole down to
// 2^-23 of the largest. A smaller margin rescales O more often: 3 with a lift of 12, 5 with 10,
// 6 with 9 and 8 with 7 took 334.8 / 323.0 / 317.5 / 315.1 us for 6042 tokens in 4 sequences, 32 / 8
// heads of 128.
template <typename T>
constexpr float kRaise = Elem<T>::kHalf ? 6.f : 8.f;
template <typename T>
constexpr float kTileLift = Elem<T>::kHalf ? 9.f : 0.f;

// One word per translation unit, read by its own host function.
static __device__ int g_wait_error = 0;

__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int code) {
  const uint32_t addr = smem_u32(bar);
  if (mbar_try_wait(addr, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(addr, parity)) {
    if (clock64() - t0 > kWaitClockLimit) {
      atomicCAS(&g_wait_error, 0, code);
      return false;
    }
  }
  return true;
}

// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 values in a register pair: one instruction for both on sm_100.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The larger of two, NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of two values on the FMA pipe, for x <= 15:
// x = n + f with n the nearest whole number (Cody and Waite's reduction: adding
// 1.5 2^23 leaves n in the low bits), 2^f on [-1/2, 1/2] by the polynomial of least
// relative error (Remez), n added to the exponent field. Relative error 7.5e-5 in
// degree 3 for bf16 results (half a step 3.9e-3) and 2.7e-6 in degree 4 for fp16 (4.9e-4).
// Below the normal numbers the absolute error is less than 2^-126. What lies below
// -126.999, -inf included, counts as that: there n = -127 and 2^f is 1.0007, so that the
// exponent field is zero and the word a subnormal of 2^-136.5, which is zero in either
// 16-bit type. A masked key, whose x is -inf, must not keep any weight in P: bf16 has
// fp32's exponents, and its largest finite value times 2^-125 is 8. Measured beside
// it: a select of zero behind the exponent, 0.8 % (D = 64) to 2.8 % (128) of the time of
// long prompts.
// NaN gives the largest finite number, infinite as a 16-bit P, so that the row's result
// is not finite and the row is done again key by key.
template <bool FINE>
__device__ __forceinline__ float2 exp2_pair(uint64_t x2) {
  const float2 x = split2(x2);
  const uint64_t c = pair2(max_nan(x.x, -126.999f), max_nan(x.y, -126.999f));
  const uint64_t r = add2(c, pair2(12582912.f, 12582912.f));
  const uint64_t n = add2(r, pair2(-12582912.f, -12582912.f));
  const uint64_t f = fma2(n, pair2(-1.f, -1.f), c);
  uint64_t y;
  if constexpr (FINE) {
    y = fma2(f, pair2(0.009570102207362652f, 0.009570102207362652f), pair2(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(f, y, pair2(0.240247443318367f, 0.240247443318367f));
    y = fma2(f, y, pair2(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(f, y, pair2(0.9999992847442627f, 0.9999992847442627f));
  } else {
    y = fma2(f, pair2(0.0551716685295105f, 0.0551716685295105f), pair2(0.2426111251115799f, 0.2426111251115799f));
    y = fma2(f, y, pair2(0.6932609677314758f, 0.6932609677314758f));
    y = fma2(f, y, pair2(0.9999280571937561f, 0.9999280571937561f));
  }
  const float2 m = split2(y), b = split2(r);
  return make_float2(__uint_as_float(__float_as_uint(m.x) + (__float_as_uint(b.x) << 23)),
                     __uint_as_float(__float_as_uint(m.y) + (__float_as_uint(b.y) << 23)));
}

// V block as an MN-major operand: its 64-column chunks of 128 keys are 16 KB apart (the
// leading offset), groups of eight keys 1024 bytes.
__device__ __forceinline__ uint64_t v_desc(uint32_t addr) {
  return (smem_desc_sw128(addr) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(kTile * 128 >> 4) << 16);
}

template <typename T>
__host__ __device__ constexpr uint32_t idesc_16(int n, bool b_mn_major) {
  return (1u << 4) | (Elem<T>::kHalf ? 0u : (1u << 7) | (1u << 10)) | (b_mn_major ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// A value that all lanes of a warp hold, told to the compiler.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

}  // namespace oasis
