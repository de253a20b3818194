// The 8-bit paged KV cache: the fused Q/K RMSNorm + RoPE write that quantises
// K and V as it stores them, and the read-back to f16 rows.
//
// No counterpart in the reference, whose caches are f16 (src/model.rs:
// 1587-1599); the norm and rotation are those of norm_rope.cu (reference
// src/kernels.rs:4845-5452) with the same bits, fp8.cuh says how a row is
// quantised.  Pools: codes [num_pages][hkv][page_size][128] e4m3, scales
// [num_pages][hkv][page_size] f32.  Every byte is read once and written once;
// long calls are bound by HBM, a single token by latency.
#include "fp8.cuh"
#include "internal.h"
#include "norm_rope.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace grout {
namespace {

// One token of each sequence: an octet (8 lanes) per 128-element row of the
// token's [Q | K | V] heads, as in norm_rope.cu.  Q rows are normalised,
// rotated and rounded to f16; K rows are normalised, rotated and quantised
// from f32 (one rounding, not an f16 one first); V rows are quantised.  One
// token of 64/8 heads: 2.6 us, a launch and three dependent loads (position,
// page, nothing behind it): latency.
__global__ void __launch_bounds__(256) qk_norm_rope_kv_fp8_kernel(const NormRopeFp8Args a) {
  const int j = threadIdx.x & 7;  // lane within the octet
  const unsigned mask = 0xFFu << (threadIdx.x & 24);
  const uint32_t heads = (uint32_t)(a.hq + 2 * a.hkv);
  const uint32_t ntask = (uint32_t)a.rows * heads;  // the host keeps it and the last step below 2^32
  const uint32_t step = (gridDim.x * blockDim.x) >> 3;
  const float2 nz = make_float2(a.neg_zero, a.neg_zero);
  for (uint32_t task = (blockIdx.x * blockDim.x + threadIdx.x) >> 3; task < ntask; task += step) {
    const uint32_t s = task / heads;
    const int hh = (int)(task - s * heads);
    const bool is_q = hh < a.hq;
    const bool is_v = hh >= a.hq + a.hkv;
    const int64_t pos = a.d_position[s];
    if (pos >= a.max_seq) {
      if (j == 0 && hh == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_POSITION);
      continue;
    }
    const __half* src = a.q + (int64_t)s * a.q_row_stride + (int64_t)hh * kHeadDim;
    const uint4 xl = ldg16(src + 8 * j);
    const uint4 xh = ldg16(src + 64 + 8 * j);
    int64_t slot = 0;  // cache row: (page * hkv + kh) * page_size + row in page
    if (!is_q) {
      const int kh = hh - a.hq - (is_v ? a.hkv : 0);
      const uint32_t pg = (uint32_t)pos / (uint32_t)a.page_size;
      const int32_t page = a.page_table[(int64_t)s * a.table_stride + pg];
      if (page < 0 || page >= a.num_pages) {
        if (j == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
        continue;
      }
      slot = ((int64_t)page * a.hkv + kh) * a.page_size + (uint32_t)pos - pg * (uint32_t)a.page_size;
    }
    float2 lo[4], hi[4];
    if (is_v) {
      unpack4(xl, lo);
      unpack4(xh, hi);
    } else {
      float2 cs[4], sn[4];
      const __half* w = is_q ? a.q_w : a.k_w;
      load_cos_sin(a.table + pos * kHeadDim, j, cs, sn);
      octet_norm_rope_f32x2(xl, xh, ldg16(w + 8 * j), ldg16(w + 64 + 8 * j), cs, sn, a.eps,
                            nz, mask, lo, hi);
    }
    if (is_q) {
      __half* dst = a.q_out + ((int64_t)s * a.hq + hh) * kHeadDim;
      *reinterpret_cast<uint4*>(dst + 8 * j) = pack4(lo);
      *reinterpret_cast<uint4*>(dst + 64 + 8 * j) = pack4(hi);
    } else {
      uint2 clo, chi;
      const float scale = is_v ? octet_quantise<true>(lo, hi, nz, mask, clo, chi)
                               : octet_quantise<false>(lo, hi, nz, mask, clo, chi);
      uint8_t* dst = (is_v ? a.pages.v : a.pages.k) + slot * kHeadDim;
      *reinterpret_cast<uint2*>(dst + 8 * j) = clo;
      *reinterpret_cast<uint2*>(dst + 64 + 8 * j) = chi;
      if (j == 0) (is_v ? a.pages.v_scales : a.pages.k_scales)[slot] = scale;
    }
  }
}

// A chunk of one sequence's tokens.  An octet keeps its unit, two query heads
// or K and V of a KV head, over every per-th token: the norm weights stay in
// registers, the angles are read once for two rows, and the next token's rows
// are loaded while this one's are worked on.  4096 tokens of 64/8 heads (161
// MB): 32.2 us in a graph, 5.0 TB/s (34.8 us a call in a stream); a row per octet
// and scalar arithmetic took 35.1 us, the schedulers issuing in 72 % of the cycles
// and L1 busy with angles for 61 %.  Now they issue in 50 % and L1 is busy for 49 %:
// what is left is latency, four warps a scheduler that wait for loads a third of
// their time, and more of them want the registers: 5 blocks of 128 threads (96
// registers) are 4 % faster than 4, 10 % than 6 (spills).
constexpr int kChunkThreads = 128;
constexpr int kChunkBlocks = 5;  // per SM
__global__ void __launch_bounds__(kChunkThreads, kChunkBlocks)
    qk_norm_rope_kv_fp8_chunk_kernel(const NormRopeFp8Args a, int per) {
  const int j = threadIdx.x & 7;  // lane within the octet
  const unsigned mask = 0xFFu << (threadIdx.x & 24);
  const uint32_t q_units = (uint32_t)(a.hq + 1) >> 1;
  const uint32_t units = q_units + (uint32_t)a.hkv;
  const uint32_t octet = (blockIdx.x * blockDim.x + threadIdx.x) >> 3;
  const uint32_t first = octet / units;
  if (first >= (uint32_t)per) return;
  const int unit = (int)(octet - first * units);
  const bool is_q = unit < (int)q_units;
  const int h0 = is_q ? 2 * unit : unit - (int)q_units;
  const bool second = !is_q || h0 + 1 < a.hq;
  const int64_t stride = is_q ? a.q_row_stride : a.kv_row_stride;
  const __half* src0 = (is_q ? a.q : a.k) + (int64_t)h0 * kHeadDim + 8 * j;
  const __half* src1 = is_q ? src0 + (second ? kHeadDim : 0) : a.v + (int64_t)h0 * kHeadDim + 8 * j;
  const __half* w = is_q ? a.q_w : a.k_w;
  const uint4 wl = ldg16(w + 8 * j), wh = ldg16(w + 64 + 8 * j);
  const float2 nz = make_float2(a.neg_zero, a.neg_zero);

  uint4 nx[4];
  auto fetch = [&](int s) {
    const int64_t off = (int64_t)s * stride;
    nx[0] = ldg16(src0 + off);
    nx[1] = ldg16(src0 + off + 64);
    nx[2] = ldg16(src1 + off);
    nx[3] = ldg16(src1 + off + 64);
  };
  int s = (int)first;
  if (s < a.rows) fetch(s);
  for (; s < a.rows; s += per) {
    const uint4 x0 = nx[0], x1 = nx[1], x2 = nx[2], x3 = nx[3];
    const int pos = a.pos0 + s;
    float2 cs[4], sn[4];
    load_cos_sin(a.table + (int64_t)pos * kHeadDim, j, cs, sn);
    int32_t page = 0;
    uint32_t in_page = 0;
    if (!is_q) {
      const uint32_t pg = (uint32_t)pos / (uint32_t)a.page_size;
      in_page = (uint32_t)pos - pg * (uint32_t)a.page_size;
      page = __ldg(a.page_table + pg);
    }
    if (s + per < a.rows) fetch(s + per);
    float2 lo[4], hi[4];
    octet_norm_rope_f32x2(x0, x1, wl, wh, cs, sn, a.eps, nz, mask, lo, hi);
    if (is_q) {
      __half* dst = a.q_out + (int64_t)s * a.q_row_stride + (int64_t)h0 * kHeadDim + 8 * j;
      *reinterpret_cast<uint4*>(dst) = pack4(lo);
      *reinterpret_cast<uint4*>(dst + 64) = pack4(hi);
      octet_norm_rope_f32x2(x2, x3, wl, wh, cs, sn, a.eps, nz, mask, lo, hi);
      if (second) {
        *reinterpret_cast<uint4*>(dst + kHeadDim) = pack4(lo);
        *reinterpret_cast<uint4*>(dst + kHeadDim + 64) = pack4(hi);
      }
    } else if (page < 0 || page >= a.num_pages) {
      if (j == 0 && a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
    } else {
      const int64_t slot = ((int64_t)page * a.hkv + h0) * a.page_size + in_page;
#pragma unroll
      for (int row = 0; row < 2; ++row) {
        if (row == 1) {
          unpack4(x2, lo);
          unpack4(x3, hi);
        }
        uint2 clo, chi;
        const float scale = row ? octet_quantise<true>(lo, hi, nz, mask, clo, chi)
                                : octet_quantise<false>(lo, hi, nz, mask, clo, chi);
        uint8_t* dst = (row ? a.pages.v : a.pages.k) + slot * kHeadDim + 8 * j;
        *reinterpret_cast<uint2*>(dst) = clo;
        *reinterpret_cast<uint2*>(dst + 64) = chi;
        if (j == 0) (row ? a.pages.v_scales : a.pages.k_scales)[slot] = scale;
      }
    }
  }
}

// Read-back: packed output row r of sequence b (cu[b] <= r < cu[b+1]) is cache
// position first[b] + r - cu[b].  A warp takes kReadTasks neighbouring (row, KV
// head) pairs: a lane each finds their sequence and cache row, then half-warps
// turn them, K in the lower and V in the upper half, 8 codes a lane (8-byte
// loads, 16-byte stores: both rows' 128 and 256 bytes are whole lines), all
// loads first.  Sixteen histories, 90,000 rows of 8 heads (0.56 GB): 89.5 us, 6.25
// TB/s (a row at a time per half-warp, its sequence searched there: 109 us).
constexpr int kReadTasks = 8;
constexpr int kReadWarps = 8;
__global__ void __launch_bounds__(32 * kReadWarps) kv_read_fp8_kernel(const KvReadFp8Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t task0 = ((int64_t)blockIdx.x * kReadWarps + (threadIdx.x >> 5)) * kReadTasks;
  int64_t slot_l = -1, out_l = -1;  // of task0 + lane: cache row (-1: zeros), output offset (-1: none)
  if (lane < kReadTasks && task0 + lane < a.rows * a.hkv) {
    const int64_t row = (task0 + lane) / a.hkv;
    const int kh = (int)(task0 + lane - row * a.hkv);
    if (row >= a.cu[0] && row < a.cu[a.batch]) {  // rows of no sequence stay as they are
      // the last sequence whose first row is <= row (empty sequences own no row)
      int lo = 0, hi = a.batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= row) lo = mid;
        else hi = mid;
      }
      out_l = row * a.out_row_stride + (int64_t)kh * kHeadDim;
      const int64_t pos = (a.first ? (int64_t)a.first[lo] : 0) + (row - a.cu[lo]);
      if (pos < 0 || pos >= a.max_seq) {
        if (a.err) atomicCAS(a.err, 0, DEV_ERR_POSITION);
      } else {
        const uint32_t pg = (uint32_t)pos / (uint32_t)a.page_size;
        const int32_t page = __ldg(a.page_table + (int64_t)lo * a.table_stride + pg);
        if (page < 0 || page >= a.num_pages) {
          if (a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
        } else {
          slot_l = ((int64_t)page * a.hkv + kh) * a.page_size + (uint32_t)pos - pg * (uint32_t)a.page_size;
        }
      }
    }
  }
  const bool v = lane >= 16;
  const int j = lane & 15;
  const uint8_t* codes = (v ? a.pages.v : a.pages.k) + 8 * j;
  const float* scales = v ? a.pages.v_scales : a.pages.k_scales;
  __half* out = (v ? a.v_out : a.k_out) + 8 * j;
  uint2 c[kReadTasks];
  float scale[kReadTasks];
#pragma unroll
  for (int u = 0; u < kReadTasks; ++u) {
    const int64_t slot = __shfl_sync(0xffffffffu, slot_l, u);
    c[u] = make_uint2(0, 0);  // a row that cannot be read is zero
    scale[u] = 0.f;
    if (slot >= 0) {
      c[u] = __ldg(reinterpret_cast<const uint2*>(codes + slot * kHeadDim));
      scale[u] = __ldg(scales + slot);
    }
  }
#pragma unroll
  for (int u = 0; u < kReadTasks; ++u) {
    const int64_t off = __shfl_sync(0xffffffffu, out_l, u);
    const uint32_t p[4] = {f16x2_of_e4m3_lo(c[u].x), f16x2_of_e4m3_hi(c[u].x), f16x2_of_e4m3_lo(c[u].y),
                           f16x2_of_e4m3_hi(c[u].y)};
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[i]));
      h[i] = pack_half2(__fmul_rn(f.x, scale[u]), __fmul_rn(f.y, scale[u]));
    }
    if (off >= 0) *reinterpret_cast<uint4*>(out + off) = make_uint4(h[0], h[1], h[2], h[3]);
  }
}

}  // namespace

cudaError_t launch_qk_norm_rope_kv_fp8(const NormRopeFp8Args& args, int num_sms, cudaStream_t s) {
  NormRopeFp8Args a = args;
  a.neg_zero = -0.0f;
  if (!a.d_position && a.rows > 0) {
    const int64_t units = ((int64_t)a.hq + 1) / 2 + a.hkv;
    const int64_t resident = (int64_t)num_sms * kChunkBlocks * (kChunkThreads / 8);  // octets
    const int64_t per = std::max<int64_t>(1, std::min<int64_t>(a.rows, resident / units));
    qk_norm_rope_kv_fp8_chunk_kernel<<<(unsigned)((per * units + kChunkThreads / 8 - 1) / (kChunkThreads / 8)), kChunkThreads, 0, s>>>(a, (int)per);
    return cudaGetLastError();
  }
  const int64_t ntask = (int64_t)a.rows * (a.hq + 2 * a.hkv);
  if (ntask == 0) return cudaSuccess;
  const int per_block = 256 / 8;
  int64_t blocks = (ntask + per_block - 1) / per_block;
  const int64_t cap = (int64_t)num_sms * 8;  // 8 resident 256-thread blocks per SM
  if (blocks > cap) blocks = cap;
  qk_norm_rope_kv_fp8_kernel<<<(unsigned)blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv_read_fp8(const KvReadFp8Args& a, cudaStream_t s) {
  const int64_t per = kReadWarps * kReadTasks;
  const int64_t blocks = (a.rows * a.hkv + per - 1) / per;
  if (blocks == 0) return cudaSuccess;
  kv_read_fp8_kernel<<<(unsigned)blocks, 32 * kReadWarps, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace grout
