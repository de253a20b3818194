// Pieces of the merges of split softmax results: warp-wide maximum and sum,
// four-value accumulation and the rounding of a row's four values to f16.
#pragma once
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace grout {

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ void store_row4(__half* p, const float4& v, float scale) {
  uint2 u;
  u.x = pack_half2(v.x * scale, v.y * scale);
  u.y = pack_half2(v.z * scale, v.w * scale);
  *reinterpret_cast<uint2*>(p) = u;
}
__device__ __forceinline__ void fma4(float4& acc, float w, const float4& v) {
  acc.x += w * v.x;
  acc.y += w * v.y;
  acc.z += w * v.z;
  acc.w += w * v.w;
}

}  // namespace grout
