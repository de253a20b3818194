// e4m3 <-> f16/f32 helpers of the 8-bit KV cache.
//
// A cache row (one token, one KV head) is 128 e4m3 codes and one f32 scale:
//   scale = max|y| / 448, code = e4m3(y * (448 / max|y|)),
// both divisions and the product rounded to f32 once, the code rounded to
// nearest even and saturated (the product may pass 448 by one f32 rounding).
// The row's largest value so uses e4m3's whole range; its smaller values keep
// 3 mantissa bits down to max|y| / 28672 (the smallest normal code, 2^-6) and
// a fixed step of max|y| / 229376 below that.  A row whose values an f16 cache would all round to
// zero (max|y| <= 2^-25) is stored as zero codes with scale 0.  A NaN stays a NaN
// code; a row with an infinity gets an infinite scale, so it reads back as NaN.
#pragma once
#include <cuda_fp16.h>

#include <cstdint>

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
// row's scale (the same in every lane).
__device__ __forceinline__ float octet_quantise(const float (&lo)[8], const float (&hi)[8],
                                                unsigned mask, uint2& codes_lo, uint2& codes_hi) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, off, 8));
  const bool zero = top <= kFp8ZeroRow;
  const float inv = zero ? 0.f : __fdiv_rn(kE4m3Max, top);
  float a[8], b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    a[e] = __fmul_rn(lo[e], inv);
    b[e] = __fmul_rn(hi[e], inv);
  }
  codes_lo = make_uint2(e4m3x4(a[0], a[1], a[2], a[3]), e4m3x4(a[4], a[5], a[6], a[7]));
  codes_hi = make_uint2(e4m3x4(b[0], b[1], b[2], b[3]), e4m3x4(b[4], b[5], b[6], b[7]));
  return zero ? 0.f : __fdiv_rn(top, kE4m3Max);
}

}  // namespace grout
