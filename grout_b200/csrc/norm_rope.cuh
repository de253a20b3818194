// The per-row arithmetic of the fused Q/K RMSNorm + RoPE write, shared by the
// standalone kernel (norm_rope.cu) and the fused decode kernel (decode.cu) so
// that both produce the same bits by construction.
//
// One octet (8 lanes) holds a 128-element head row: lane j of the octet owns
// the RoPE pairs i = 8j..8j+7, i.e. x[8j..8j+8) ("lo") and x[64+8j..64+8j+8)
// ("hi"), so rotate-half needs no shuffle and every access is 16 bytes.  The
// arithmetic is pinned so that the CPU oracle reproduces it bit for bit: no
// FMA contraction (explicit _rn intrinsics), a fixed sum order (lane sum
// ((t0+t1)+(t2+t3))+((t4+t5)+(t6+t7)), then an xor butterfly 4,2,1 over the
// octet), rsqrt as a correctly rounded reciprocal of a correctly rounded
// sqrt, and cos/sin read from a table of correctly rounded values of the
// reference's f32 angle f32(pos) * inv_freq[i] (src/kernels.rs:5012-5084).
#pragma once
#include <cuda_fp16.h>

#include <cstdint>

namespace grout {

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
    float2 v = __half22float2(h);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 ldg16(const void* p) {
  return __ldg(reinterpret_cast<const uint4*>(p));
}

// Lane j's cos (cs) and sin (sn) values of table row `trow` ([2][64] f32).
__device__ __forceinline__ void load_cos_sin(const float* trow, int j, float (&cs)[8],
                                             float (&sn)[8]) {
  const float4 c0 = __ldg(reinterpret_cast<const float4*>(trow + 8 * j));
  const float4 c1 = __ldg(reinterpret_cast<const float4*>(trow + 8 * j + 4));
  const float4 s0 = __ldg(reinterpret_cast<const float4*>(trow + 64 + 8 * j));
  const float4 s1 = __ldg(reinterpret_cast<const float4*>(trow + 64 + 8 * j + 4));
  cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w;
  cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
  sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w;
  sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
}

// RMSNorm of the octet's row (x = [xl | xh] as lane j's 16-byte chunks),
// scaled by the norm weight (wl, wh), rotated by (cs, sn) and rounded to f16
// once.  `mask` is the octet's lane mask for the butterfly.
__device__ __forceinline__ void octet_norm_rope(const uint4& xl, const uint4& xh,
                                                const float (&wl)[8], const float (&wh)[8],
                                                const float (&cs)[8], const float (&sn)[8],
                                                float eps, unsigned mask, uint4& out_lo,
                                                uint4& out_hi) {
  float lo[8], hi[8];
  unpack8(xl, lo);
  unpack8(xh, hi);
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = __fadd_rn(__fmul_rn(lo[e], lo[e]), __fmul_rn(hi[e], hi[e]));
  float ss = __fadd_rn(__fadd_rn(__fadd_rn(t[0], t[1]), __fadd_rn(t[2], t[3])),
                       __fadd_rn(__fadd_rn(t[4], t[5]), __fadd_rn(t[6], t[7])));
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(mask, ss, off, 8));
  // ss / 128 is an exact power-of-two scaling; the correctly rounded
  // reciprocal equals the IEEE quotient 1.0f / x.
  const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 0.0078125f), eps)));
  float ylo[8], yhi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float nlo = __fmul_rn(__fmul_rn(lo[e], inv), wl[e]);
    const float nhi = __fmul_rn(__fmul_rn(hi[e], inv), wh[e]);
    ylo[e] = __fsub_rn(__fmul_rn(nlo, cs[e]), __fmul_rn(nhi, sn[e]));
    yhi[e] = __fadd_rn(__fmul_rn(nhi, cs[e]), __fmul_rn(nlo, sn[e]));
  }
  out_lo = pack8(ylo);
  out_hi = pack8(yhi);
}

// ---- The same, without the rounding to f16, on f32x2 pairs: two correctly rounded operations an
// instruction, so the same bits at half the instructions.  A product is formed
// as a * b + nz with nz = -0 (exact, whatever the product's sign): mul.rn.f32x2
// followed by add.rn.f32x2 came out contracted to one rounding; with an nz that
// the compiler cannot know to be zero it cannot.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{ .reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7};"
      " fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b, float2 nz) { return fma2(a, b, nz); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 d, a, b;"
      " mov.b64 {%0, %1}, d; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; sub.rn.f32x2 d, a, b;"
      " mov.b64 {%0, %1}, d; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ void unpack4(const uint4& u, float2 (&f)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
__device__ __forceinline__ uint4 pack4(const float2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void load_cos_sin(const float* trow, int j, float2 (&cs)[4], float2 (&sn)[4]) {
  const float4 c0 = __ldg(reinterpret_cast<const float4*>(trow + 8 * j));
  const float4 c1 = __ldg(reinterpret_cast<const float4*>(trow + 8 * j + 4));
  const float4 s0 = __ldg(reinterpret_cast<const float4*>(trow + 64 + 8 * j));
  const float4 s1 = __ldg(reinterpret_cast<const float4*>(trow + 64 + 8 * j + 4));
  cs[0] = make_float2(c0.x, c0.y), cs[1] = make_float2(c0.z, c0.w);
  cs[2] = make_float2(c1.x, c1.y), cs[3] = make_float2(c1.z, c1.w);
  sn[0] = make_float2(s0.x, s0.y), sn[1] = make_float2(s0.z, s0.w);
  sn[2] = make_float2(s1.x, s1.y), sn[3] = make_float2(s1.z, s1.w);
}
__device__ __forceinline__ void octet_norm_rope_f32x2(const uint4& xl, const uint4& xh,
                                                      const uint4& wl, const uint4& wh,
                                                      const float2 (&cs)[4], const float2 (&sn)[4],
                                                      float eps, float2 nz, unsigned mask, float2 (&ylo)[4],
                                                      float2 (&yhi)[4]) {
  float2 lo[4], hi[4], w[4], t[4];
  unpack4(xl, lo);
  unpack4(xh, hi);
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = add2(mul2(lo[e], lo[e], nz), mul2(hi[e], hi[e], nz));
  float ss = __fadd_rn(__fadd_rn(__fadd_rn(t[0].x, t[0].y), __fadd_rn(t[1].x, t[1].y)),
                       __fadd_rn(__fadd_rn(t[2].x, t[2].y), __fadd_rn(t[3].x, t[3].y)));
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(mask, ss, off, 8));
  const float r = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 0.0078125f), eps)));
  const float2 inv = make_float2(r, r);
  unpack4(wl, w);
#pragma unroll
  for (int e = 0; e < 4; ++e) lo[e] = mul2(mul2(lo[e], inv, nz), w[e], nz);
  unpack4(wh, w);
#pragma unroll
  for (int e = 0; e < 4; ++e) hi[e] = mul2(mul2(hi[e], inv, nz), w[e], nz);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    ylo[e] = sub2(mul2(lo[e], cs[e], nz), mul2(hi[e], sn[e], nz));
    yhi[e] = add2(mul2(hi[e], cs[e], nz), mul2(lo[e], sn[e], nz));
  }
}

}  // namespace grout
