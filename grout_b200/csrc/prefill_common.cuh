// Pieces that the prefill kernels share: packed f32x2 softmax arithmetic, the
// polynomial exponential, and tcgen05 MMA issue with precomputed descriptor
// words.
#pragma once
#include <cstdint>

#include "ptx.cuh"

namespace grout {

constexpr int kTile = 128 * 128 * 2;  // bytes of one 128x128 f16 tile (two 64-col boxes)
constexpr int kBox = kTile / 2;

// ---- packed f32x2 arithmetic (sm_100a): two softmax elements per instruction
__device__ __forceinline__ uint64_t f2pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2unpack(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x (x <= 0) for a pair, on the FMA/ALU pipes, used for a share of the
// softmax exponentials so the MUFU unit is not the only path.  Range
// reduction x = n + f, n = round(x) via the 1.5*2^23 magic constant,
// f in [-1/2, 1/2]; 2^f by a degree-3 polynomial fitted for minimum relative
// error (max 7.6e-5, below the f16 rounding P gets next); 2^n added into the
// exponent field.  Inputs below -125 clamp to ~2^-125 (P rounds to 0 in
// f16); the clamp keeps n + exponent(p) >= 1, so the sum never reaches the
// sign bit (p can be slightly below 1 when f < 0).
__device__ __forceinline__ void ex2_poly2(uint64_t x2, float& r0, float& r1) {
  float x0, x1;
  f2unpack(x2, x0, x1);
  x2 = f2pack(fmaxf(x0, -125.0f), fmaxf(x1, -125.0f));
  const uint64_t t2 = fadd2(x2, f2pack(12582912.0f, 12582912.0f));
  const uint64_t n2 = fadd2(t2, f2pack(-12582912.0f, -12582912.0f));
  const uint64_t f2 = ffma2(n2, f2pack(-1.0f, -1.0f), x2);
  uint64_t p2 = ffma2(f2pack(0.05517090484f, 0.05517090484f), f2,
                      f2pack(0.24260953069f, 0.24260953069f));
  p2 = ffma2(p2, f2, f2pack(0.69326096773f, 0.69326096773f));
  p2 = ffma2(p2, f2, f2pack(0.99992817640f, 0.99992817640f));
  float p0, p1, t0, t1;
  f2unpack(p2, p0, p1);
  f2unpack(t2, t0, t1);
  r0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  r1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

// Element pairs (of the 16 per 32-column chunk) whose exponentials run on
// ex2_poly2: one in four, so MUFU carries 3/4 of the exponentials.
__device__ __forceinline__ constexpr bool poly_pair(int i) { return (i & 3) == 3; }

// Online-softmax rescaling threshold (log2 units): the reference max a row
// exponentiates against moves only when the row max grows by more than this,
// so P stays <= 2^8 and O is rescaled rarely.
constexpr float kRescaleThreshold = 8.0f;

// Low/high words of the SW128 shared-memory descriptor (matches
// smem_desc_sw128): low = start address >> 4 | LBO >> 4 << 16;
// high = SBO (1024) >> 4 | version 1 << 14 | layout SW128 (2) << 29.
constexpr uint32_t kDescLboK = (16u >> 4) << 16;
constexpr uint32_t kDescLboV = ((uint32_t)kBox >> 4) << 16;
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
static_assert(((uint64_t)kDescHi << 32) == ((uint64_t)(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61),
              "descriptor high word");
__device__ __forceinline__ void mma_ss_lo(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc,
                                          uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 da, db; setp.ne.u32 p, %4, 0;"
      " mov.b64 da, {%1, %5}; mov.b64 db, {%2, %5};"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p; }" ::"r"(d),
      "r"(alo), "r"(blo), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts_lo(uint32_t d, uint32_t a_tmem, uint32_t blo, uint32_t idesc,
                                          uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 db; setp.ne.u32 p, %4, 0;"
      " mov.b64 db, {%2, %5};"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p; }" ::"r"(d),
      "r"(a_tmem), "r"(blo), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}

}  // namespace grout
