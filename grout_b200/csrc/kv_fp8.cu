// The 8-bit paged KV cache: the fused Q/K RMSNorm + RoPE write that quantises
// K and V as it stores them, and the read-back to f16 rows.
//
// No counterpart in the reference, whose caches are f16 (src/model.rs:
// 1587-1599); the norm and rotation are those of norm_rope.cu (reference
// src/kernels.rs:4845-5452) with the same bits, fp8.cuh says how a row is
// quantised.  Pools: codes [num_pages][hkv][page_size][128] e4m3, scales
// [num_pages][hkv][page_size] f32.  Both kernels are bound by HBM: every byte is read once and written once.
#include "fp8.cuh"
#include "internal.h"
#include "norm_rope.cuh"
#include "ptx.cuh"

namespace grout {
namespace {

// One octet (8 lanes) per 128-element row of the token's [Q | K | V] heads,
// as in norm_rope.cu.  Q rows are normalised, rotated and rounded to f16; K
// rows are normalised, rotated and quantised from f32 (one rounding, not an
// f16 one first); V rows are quantised.
template <bool kDecode>
__global__ void __launch_bounds__(256) qk_norm_rope_kv_fp8_kernel(const NormRopeFp8Args a) {
  const int j = threadIdx.x & 7;  // lane within the octet
  const unsigned mask = 0xFFu << (threadIdx.x & 24);
  const uint32_t heads = (uint32_t)(a.hq + 2 * a.hkv);
  const uint64_t ntask = (uint64_t)a.rows * heads;
  const uint32_t step = (gridDim.x * blockDim.x) >> 3;
  for (uint64_t task = (blockIdx.x * blockDim.x + threadIdx.x) >> 3; task < ntask; task += step) {
    const uint32_t s = (uint32_t)(task / heads);
    const int hh = (int)(task - (uint64_t)s * heads);
    const bool is_q = hh < a.hq;
    const bool is_v = hh >= a.hq + a.hkv;
    const int kh = hh - a.hq - (is_v ? a.hkv : 0);
    int64_t pos;
    const __half* src;
    if (kDecode) {
      pos = a.d_position[s];
      if (pos >= a.max_seq) {
        if (j == 0 && hh == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_POSITION);
        continue;
      }
      src = a.q + (int64_t)s * a.q_row_stride + (int64_t)hh * kHeadDim;
    } else {
      pos = (int64_t)a.pos0 + s;
      src = is_q ? a.q + (int64_t)s * a.q_row_stride + (int64_t)hh * kHeadDim
                 : (is_v ? a.v : a.k) + (int64_t)s * a.kv_row_stride + (int64_t)kh * kHeadDim;
    }
    const uint4 xl = ldg16(src + 8 * j);
    const uint4 xh = ldg16(src + 64 + 8 * j);
    int64_t slot = 0;  // cache row: (page * hkv + kh) * page_size + row in page
    if (!is_q) {
      const int64_t pg = pos / a.page_size;
      const int32_t page = a.page_table[(kDecode ? (int64_t)s * a.table_stride : 0) + pg];
      if (page < 0 || page >= a.num_pages) {
        if (j == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
        continue;
      }
      slot = ((int64_t)page * a.hkv + kh) * a.page_size + (pos - pg * a.page_size);
    }
    float lo[8], hi[8];
    if (is_v) {
      unpack8(xl, lo);
      unpack8(xh, hi);
    } else {
      float wl[8], wh[8], cs[8], sn[8];
      const __half* w = is_q ? a.q_w : a.k_w;
      unpack8(ldg16(w + 8 * j), wl);
      unpack8(ldg16(w + 64 + 8 * j), wh);
      load_cos_sin(a.table + pos * kHeadDim, j, cs, sn);
      octet_norm_rope_f32(xl, xh, wl, wh, cs, sn, a.eps, mask, lo, hi);
    }
    if (is_q) {
      __half* dst = a.q_out + (kDecode ? ((int64_t)s * a.hq + hh) * kHeadDim
                                       : (int64_t)s * a.q_row_stride + (int64_t)hh * kHeadDim);
      *reinterpret_cast<uint4*>(dst + 8 * j) = pack8(lo);
      *reinterpret_cast<uint4*>(dst + 64 + 8 * j) = pack8(hi);
    } else {
      uint2 clo, chi;
      const float scale = octet_quantise(lo, hi, mask, clo, chi);
      uint8_t* dst = (is_v ? a.pages.v : a.pages.k) + slot * kHeadDim;
      *reinterpret_cast<uint2*>(dst + 8 * j) = clo;
      *reinterpret_cast<uint2*>(dst + 64 + 8 * j) = chi;
      if (j == 0) (is_v ? a.pages.v_scales : a.pages.k_scales)[slot] = scale;
    }
  }
}

// Read-back: packed output row r of sequence b (cu[b] <= r < cu[b+1]) is cache
// position first[b] + r - cu[b].  One octet per (row, KV head): lane j turns
// 16 codes of K and 16 of V into f16(code * scale) and stores 32 bytes of each.
constexpr int kReadRows = 32;  // octets of a 256-thread block
__global__ void __launch_bounds__(256) kv_read_fp8_kernel(const KvReadFp8Args a) {
  const int j = threadIdx.x & 7;
  const uint64_t task = (uint64_t)blockIdx.x * kReadRows + (threadIdx.x >> 3);
  const int64_t row = (int64_t)(task / (uint32_t)a.hkv);
  const int kh = (int)(task - (uint64_t)row * (uint32_t)a.hkv);
  if (row >= a.rows) return;
  // last sequence whose first row is <= row (empty sequences own no row)
  int lo = 0, hi = a.batch;  // cu[lo] <= row < cu[hi] if the row has an owner
  if (row < a.cu[0] || row >= a.cu[a.batch]) return;  // rows of no sequence stay as they are
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int64_t pos = (a.first ? (int64_t)a.first[lo] : 0) + (row - a.cu[lo]);
  int64_t slot = -1;
  if (pos < 0 || pos >= a.max_seq) {
    if (j == 0 && kh == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_POSITION);
  } else {
    const int64_t pg = pos / a.page_size;
    const int32_t page = __ldg(a.page_table + (int64_t)lo * a.table_stride + pg);
    if (page < 0 || page >= a.num_pages) {
      if (j == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
    } else {
      slot = ((int64_t)page * a.hkv + kh) * a.page_size + (pos - pg * a.page_size);
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};  // a row that cannot be read is zero
    if (slot >= 0) {
      const uint4 c = ldg16((kv ? a.pages.v : a.pages.k) + slot * kHeadDim + 16 * j);
      const float scale = __ldg((kv ? a.pages.v_scales : a.pages.k_scales) + slot);
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
      uint32_t h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t p = f16x2_of_e4m3x2(w[i >> 1] >> (16 * (i & 1)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
        h[i] = pack_half2(__fmul_rn(f.x, scale), __fmul_rn(f.y, scale));
      }
      o[0] = make_uint4(h[0], h[1], h[2], h[3]);
      o[1] = make_uint4(h[4], h[5], h[6], h[7]);
    }
    __half* dst = (kv ? a.v_out : a.k_out) + row * a.out_row_stride + (int64_t)kh * kHeadDim + 16 * j;
    *reinterpret_cast<uint4*>(dst) = o[0];
    *reinterpret_cast<uint4*>(dst + 8) = o[1];
  }
}

}  // namespace

cudaError_t launch_qk_norm_rope_kv_fp8(const NormRopeFp8Args& a, int num_sms, cudaStream_t s) {
  const int64_t ntask = (int64_t)a.rows * (a.hq + 2 * a.hkv);
  if (ntask == 0) return cudaSuccess;
  const int per_block = 256 / 8;
  int64_t blocks = (ntask + per_block - 1) / per_block;
  const int64_t cap = (int64_t)num_sms * 8;  // 8 resident 256-thread blocks per SM
  if (blocks > cap) blocks = cap;
  if (a.d_position)
    qk_norm_rope_kv_fp8_kernel<true><<<(unsigned)blocks, 256, 0, s>>>(a);
  else
    qk_norm_rope_kv_fp8_kernel<false><<<(unsigned)blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv_read_fp8(const KvReadFp8Args& a, cudaStream_t s) {
  const int64_t blocks = (a.rows * a.hkv + kReadRows - 1) / kReadRows;
  if (blocks == 0) return cudaSuccess;
  kv_read_fp8_kernel<<<(unsigned)blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace grout
