// e4m3 <-> f16/f32 helpers of the 8-bit KV cache.
//
// A cache row (one token, one KV head) is 128 e4m3 codes and one f32 scale:
//   scale = max|y| / 448, code = e4m3(y * 448 / max|y|),
// the scale rounded to f32 once, the code to nearest even and saturated.
// The row's largest value so uses e4m3's whole range; its smaller values keep
// 3 mantissa bits down to max|y| / 28672 (the smallest normal code, 2^-6) and
// a fixed step of max|y| / 229376 below that.  A row whose values an f16 cache would all round to
// zero (max|y| <= 2^-25) is stored as zero codes with scale 0.  A NaN stays a NaN
// code; a row with an infinity gets an infinite scale, so it reads back as NaN.
#pragma once
#include <cuda_fp16.h>

#include <cstdint>

#include "norm_rope.cuh"

namespace grout {

constexpr float kE4m3Max = 448.0f;
constexpr float kFp8ZeroRow = 2.98023223876953125e-8f;  // 2^-25

// Two f32 -> two e4m3 codes (lo in the low byte), nearest even, saturating.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
// The low / high two of four e4m3 codes -> packed f16 pair (exact; low byte -> low half).
__device__ __forceinline__ uint32_t f16x2_of_e4m3_lo(uint32_t codes) {
  uint32_t r;
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l; }" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3_hi(uint32_t codes) {
  uint32_t r;
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h; }" : "=r"(r) : "r"(codes));
  return r;
}
// Quantises an octet's row: lane j holds elements 8j..8j+7 (lo) and
// 64+8j..64+8j+7 (hi).  codes_lo/hi are the lane's 8-byte chunks; returns the
// row's scale (the same in every lane).  q = y * f32(448 f32(1 / max)) carries
// three roundings, which now and then turn a value next to a tie between two
// codes to the wrong side.  kExact (for V: f16 values, 448 y is exact): the
// residual 448 y - q * max, exact in one fused operation, corrects it to the
// quotient rounded once (Markstein's correction: "Computation of elementary
// functions on the IBM RISC System/6000 processor", IBM J. Res. Dev. 34, 1990), so
// the codes are the formula's bit for bit.  K's f32 values carry the norm's roundings, which
// do the same as often: there the correction would buy nothing.  (4096
// tokens, 64/8 heads: 32.0 us without, 33.3 on V, 33.5 on both.)
template <bool kExact>
__device__ __forceinline__ float octet_quantise(const float2 (&lo)[4], const float2 (&hi)[4],
                                                float2 nz, unsigned mask, uint2& codes_lo,
                                                uint2& codes_hi) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    top = fmaxf(top, fmaxf(fmaxf(fabsf(lo[e].x), fabsf(lo[e].y)), fmaxf(fabsf(hi[e].x), fabsf(hi[e].y))));
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, off, 8));
  const bool zero = top <= kFp8ZeroRow;
  const float rcp = zero ? 0.f : __frcp_rn(top);
  const float inv = __fmul_rn(rcp, kE4m3Max);
  const float2 inv2 = make_float2(inv, inv), nrcp2 = make_float2(-rcp, -rcp), top2 = make_float2(top, top),
               nmost = make_float2(-kE4m3Max, -kE4m3Max);
  const auto quotient = [&](const float2& y) {  // (the residual negated: -0 stays -0)
    const float2 q = mul2(y, inv2, nz);
    return kExact ? fma2(fma2(q, top2, mul2(y, nmost, nz)), nrcp2, q) : q;
  };
  float2 a[4], b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    a[e] = quotient(lo[e]);
    b[e] = quotient(hi[e]);
  }
  codes_lo = make_uint2(e4m3x4(a[0].x, a[0].y, a[1].x, a[1].y), e4m3x4(a[2].x, a[2].y, a[3].x, a[3].y));
  codes_hi = make_uint2(e4m3x4(b[0].x, b[0].y, b[1].x, b[1].y), e4m3x4(b[2].x, b[2].y, b[3].x, b[3].y));
  return zero ? 0.f : __fdiv_rn(top, kE4m3Max);
}

}  // namespace grout
