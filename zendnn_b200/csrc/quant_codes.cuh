// Scale and codes of the symmetric s8 quantisation of a row, shared by every kernel that writes such rows.
//
// Arithmetic contract: abs-max over finite values, clamp to 1e-10, scale = absmax / 127 (IEEE
// division), clamp to 1e-10, q = rne(v / scale) with IEEE division; non-finite inputs give 0.
#pragma once
#include "common.cuh"

namespace b200 {

__device__ __forceinline__ float scale_from_absmax(float absmax) {
  if (absmax < 1e-10f) absmax = 1e-10f;
  float s = __fdiv_rn(absmax, 127.0f);
  if (s < 1e-10f) s = 1e-10f;
  return s;
}
__device__ __forceinline__ int8_t quant_sym(float v, float scale) {
  if (!finite_f32(v)) return 0;
  return (int8_t)__float2int_rn(__fdiv_rn(v, scale));
}
// Codes without a division.  q0 = v * rinv (rinv = __frcp_rn(scale)) is a few units in the last place off the quotient; a correction step
// r = v - q0 * scale (one fused operation, exact), q1 = q0 + r * rinv gives the correctly rounded quotient (Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990); adding 1.5 * 2^23 rounds it to the nearest (even) integer and leaves that
// integer's two's complement in the low mantissa byte.  Needs a scale that comes from the abs-max of the row itself, so that
// |v / scale| <= 127 up to rounding.  bf16 elements: one step; all pairs of significands of element and abs-max, at every distance of
// exponents, were compared with the IEEE quotient, and the clamped scale as well.  f32 elements: two steps, after which the quotient's error before the
// last rounding is at most half a unit times 2^-24, less than the distance of any quotient from the middle of two floats.
// No branch: bf16 rows meet exact ties often (v / scale = 127 a / b with 8-bit a and b), and a form that sent vectors with an element near a tie
// through the division ran 237 instructions a vector of eight.
// A non-finite element makes the quotient NaN: bit 28 of the sum, clear for every code, is then set.
constexpr uint32_t kCodeNaN = 0x10000000u;
template <typename T>
__device__ __forceinline__ uint32_t quant_code(float v, float scale, float rinv) {
  float q = __fmul_rn(v, rinv);
  q = __fmaf_rn(__fmaf_rn(-q, scale, v), rinv, q);
  if (sizeof(T) == 4) q = __fmaf_rn(__fmaf_rn(-q, scale, v), rinv, q);
  return __float_as_uint(__fadd_rn(q, 12582912.0f));
}
template <typename T>
__device__ __forceinline__ int8_t quant_sym_r(float v, float scale, float rinv) {
  return finite_f32(v) ? (int8_t)(quant_code<T>(v, scale, rinv) & 0xFF) : (int8_t)0;
}

// The same for a whole 16-byte vector, on packed f32x2 arithmetic.
__device__ __forceinline__ uint64_t f32x2_pack(float lo, float hi) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ void f32x2_unpack(uint64_t r, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(r)); }
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) { uint64_t d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) { uint64_t d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) { uint64_t d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }

// STEPS: correction steps (1 for values that came from bf16, 2 otherwise).  False: an element is not finite, and its code is not valid.
template <int PAIRS, int STEPS>
__device__ __forceinline__ bool quant_pairs(const float (&v)[2 * PAIRS], float scale, float rinv, uint32_t (&m_bits)[2 * PAIRS]) {
  const uint64_t rinv2 = f32x2_pack(rinv, rinv), nscale2 = f32x2_pack(-scale, -scale), magic2 = f32x2_pack(12582912.0f, 12582912.0f);
  uint32_t any = 0u;
#pragma unroll
  for (int p = 0; p < PAIRS; ++p) {
    const uint64_t v2 = f32x2_pack(v[2 * p], v[2 * p + 1]);
    uint64_t q2 = f32x2_mul(v2, rinv2);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q2 = f32x2_fma(f32x2_fma(q2, nscale2, v2), rinv2, q2);
    float m0, m1;
    f32x2_unpack(f32x2_add(q2, magic2), m0, m1);
    m_bits[2 * p] = __float_as_uint(m0); m_bits[2 * p + 1] = __float_as_uint(m1);
    any |= m_bits[2 * p] | m_bits[2 * p + 1];
  }
  return (any & kCodeNaN) == 0u;
}
// low bytes of four words -> one word
__device__ __forceinline__ uint32_t low_bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace b200
