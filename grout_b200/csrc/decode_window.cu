// Split-K GQA decode attention of a single token over a window of its cache,
// over f16 caches (contiguous or paged) and over the 8-bit paged cache (where
// the window may also be the whole context).
//
// No counterpart in the reference, whose decode attends to the whole f16 cache
// (src/kernels.rs:4016-4304); the serving extension next to decode.cu.
//
// A query at position p = kv_len - 1 sees key n if n <= p and
// (n >= kv_len - window or n < sinks); window 0 sees every n <= p.  With
// m a running maximum, per key  s = q . k * scale / ln 2,  p = 2^(s - m),
// l = sum p,  O = sum p v,  out = O / l: one pass over the visible keys, and
// only the 64-key tiles that hold one are read (sink tiles, then the window's).
//
// 8-bit rows are k = kc * ks, v = vc * vs with e4m3 codes and one f32 scale a
// row.  ks multiplies the score; vs is folded into the weight,
// w = 2^(s + log2 vs - m) with m the running maximum of s + log2 vs, so that
// the f16 weights of the PV product use f16's range whatever the scales are,
// and l sums w / vs = 2^(s - m) in f32.  Codes become f16 exactly.
//
// Structure as decode.cu (HBM-bound; one CTA per split, KV head and sequence;
// a producer warp fills a TMA ring, four consumer warps run mma.sync with the
// GQA group on the 8-wide N side, up to 16 splits merge in a thread-block
// cluster).  A stage of the ring holds 32 KB: 64 f16 keys or 128 8-bit keys
// (two 64-key tiles, which need not be neighbours: the sinks' last tile and
// the window's first one share a stage).
//
// Keys that are not seen get no weight and their V rows are zeroed before the
// product, so that whatever they hold (an unwritten page, a NaN) stays out.
//
// Range checks on the device as in decode.cu: a position >= max_seq records
// 0x200 and the row is zero; a page-table entry outside the pool that holds a
// visible key records 0x201 and its tile is left out of the softmax.
#include "fp8.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace grout {
namespace {

constexpr int kKeys = 64;  // keys per tile (one TMA box per 128 bytes of a row)
constexpr int kStages = 3;
constexpr int kStageBytes = 32768;  // K and V of one f16 tile, or of two 8-bit tiles
constexpr int kThreads = 160;
constexpr int kRingBytes = kStages * kStageBytes;
constexpr int kScaleFloats = 4 * kKeys;  // per stage: K scales of both tiles, V scales of both
constexpr int kCtlBytes = 128;           // full/empty barriers, abort flag, per-stage tile masks
constexpr int kSmemF16 = kRingBytes + 1024 + kCtlBytes;
constexpr int kSmemFp8 = kSmemF16 + kStages * kScaleFloats * 4;

struct RedSmem {
  float o[4][128][9];  // padded: the per-dimension merge reads are conflict-free
  float m[4][8];
  float l[4][8];
};
// A CTA's final split result, read by the other CTAs of its cluster.
struct FinSmem {
  float o[8][128];
  float lse[8];
};
constexpr int kFinOffset = 20480;
static_assert(sizeof(RedSmem) <= kFinOffset, "reduction area overlaps the split result");
static_assert(kFinOffset + sizeof(FinSmem) <= kRingBytes, "merge areas must fit in the ring");

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_dsmem_f32(const float* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// w_s = 2^(lse_s - max) / sum, out = sum_s w_s * O_s, rounded to f16.  Splits
// without a visible key have lse = -inf and O = 0; if all have, the row is 0.
// A NaN lse passes into the row.  get(s, want_lse) returns lse_s or O_s[d].
template <typename Get>
__device__ __forceinline__ __half merge_splits(int nks, Get get) {
  float M = -INFINITY;
  bool any = false;
  for (int s = 0; s < nks; ++s) {
    const float lse = get(s, true);
    any |= lse != -INFINITY;
    M = fmaxf(M, lse);
  }
  if (!any) return __float2half_rn(0.f);
  float W = 0.f, O = 0.f;
  for (int s = 0; s < nks; ++s) {
    const float lse = get(s, true);
    const float w = lse == -INFINITY ? 0.f : ex2(lse - M);
    W += w;
    O += w * get(s, false);
  }
  return __float2half_rn(O / W);
}

// The 64-key tiles that hold a visible key: the sinks' tiles, then those from
// the window's first key on.  Entry i is tile i or, past the sinks, i + skip.
struct TileList {
  int kv_len, lo, sinks, sink_tiles, skip, n;
  __device__ __forceinline__ TileList(int len, int window, int nsinks) {
    kv_len = len;
    sinks = nsinks;
    lo = window > 0 ? max(0, len - window) : 0;
    const int first = lo / kKeys;
    sink_tiles = min(first, (int)(((int64_t)nsinks + kKeys - 1) / kKeys));
    skip = first - sink_tiles;
    n = sink_tiles + (len + kKeys - 1) / kKeys - first;
  }
  __device__ __forceinline__ int key0(int i) const { return (i < sink_tiles ? i : i + skip) * kKeys; }
  __device__ __forceinline__ bool sees(int key) const {
    return key < kv_len && (key >= lo || key < sinks);
  }
  // whether some of the 16 keys from `base` on are not seen
  __device__ __forceinline__ bool partial(int base) const {
    return base + 16 > kv_len || (base < lo && base + 16 > sinks);
  }
};

template <bool kFp8, bool kPaged, bool kCluster>
__global__ void __launch_bounds__(kThreads, 2)
    decode_window_kernel(const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const DecodeWindowArgs a) {
  constexpr int kTiles = kFp8 ? 2 : 1;                   // 64-key tiles per stage
  constexpr int kTileBytes = kKeys * 128 * (kFp8 ? 1 : 2);
  constexpr int kVOff = kTiles * kTileBytes;             // V tiles follow the K tiles
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kRingBytes);  // full[3], empty[3]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * kStages);
  volatile int* bad_tile = abort_flag + 1;  // [kStages][2]: a page outside the pool
  float* scales = reinterpret_cast<float*>(smem + kRingBytes + kCtlBytes);  // [kStages][K0 K1 V0 V1][64]

  const int split = blockIdx.x;
  const int kh = blockIdx.y;
  const int b = blockIdx.z;
  const int G = a.hq / a.hkv;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const uint32_t pos = a.d_position[b];
  const bool pos_ok = pos < (uint32_t)a.max_seq;
  if (!pos_ok && split == 0 && kh == 0 && threadIdx.x == 0 && a.err)
    atomicCAS(a.err, 0, DEV_ERR_POSITION);
  const TileList list(pos_ok ? (int)pos + 1 : 0, a.window, a.sinks);
  const int tps = (list.n + a.nks - 1) / a.nks;
  const int t0 = min(split * tps, list.n);
  const int nt = min(tps, list.n - t0);
  const int n_stages = (nt + kTiles - 1) / kTiles;
  const int64_t head0 = (int64_t)b * a.hq + (int64_t)kh * G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&bars[i]), 1);
      mbar_init(smem_u32(&bars[kStages + i]), 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  // Consumer state lives at function scope so it survives the CTA barrier
  // that frees the ring for the cross-warp merge.
  const int g = lane >> 2;  // MMA row group: key (S^T) / dim (O^T) offset; head for Q
  const int t = lane & 3;   // MMA column pair: heads 2t, 2t+1
  float m0 = -1.0e30f, m1 = -1.0e30f, l0 = 0.f, l1 = 0.f;
  float o[8][4];
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    if (lane == 0 && nt > 0) {
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      int issued = 0;
      for (int it = 0; it < n_stages; ++it) {
        const int st = it % kStages;
        const int r = it / kStages;
        if (r > 0 && !mbar_wait(smem_u32(&bars[kStages + st]), (r - 1) & 1, a.err, 1, abort_flag))
          break;
        const int live = min(kTiles, nt - it * kTiles);
        const uint32_t full = smem_u32(&bars[st]);
        const uint32_t kb = smem_u32(smem + st * kStageBytes);
        int row[kTiles], outer[kTiles];
#pragma unroll
        for (int x = 0; x < kTiles; ++x) {
          if (x >= live) break;
          row[x] = list.key0(t0 + it * kTiles + x);
          outer[x] = b;  // sequence (contiguous caches) or page (paged pool)
          int bad = 0;
          if (kPaged) {
            // a 64-key tile never straddles a page (page_size % 64 == 0)
            const int pg = row[x] / a.page_size;
            outer[x] = __ldg(a.page_table + (int64_t)b * a.table_stride + pg);
            row[x] -= pg * a.page_size;
            if (outer[x] < 0 || outer[x] >= a.num_pages) {
              // load page 0 instead and leave the tile out of the softmax
              if (a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
              outer[x] = 0;
              bad = 1;
            }
          }
          bad_tile[st * 2 + x] = bad;
        }
        mbar_arrive_expect_tx(full, live * (2 * kTileBytes + (kFp8 ? 2 * kKeys * 4 : 0)));
#pragma unroll
        for (int x = 0; x < kTiles; ++x) {
          if (x >= live) break;
          const uint32_t kx = kb + x * kTileBytes, vx = kx + kVOff;
          tma_load_4d(kx, &tm_k, full, 0, row[x], kh, outer[x]);
          if (!kFp8) tma_load_4d(kx + kTileBytes / 2, &tm_k, full, 64, row[x], kh, outer[x]);
          tma_load_4d(vx, &tm_v, full, 0, row[x], kh, outer[x]);
          if (!kFp8) tma_load_4d(vx + kTileBytes / 2, &tm_v, full, 64, row[x], kh, outer[x]);
          if (kFp8) {
            // 64 scales of a page row range: 256-byte aligned (row % 64 == 0)
            const int64_t off = ((int64_t)outer[x] * a.hkv + kh) * a.page_size + row[x];
            const uint32_t sb = smem_u32(scales + st * kScaleFloats + x * kKeys);
            bulk_load(sb, a.k_scales + off, kKeys * 4, full);
            bulk_load(sb + 2 * kKeys * 4, a.v_scales + off, kKeys * 4, full);
          }
        }
        issued = it + 1;
      }
      // a wait gave up: let the copies in flight land before the CTA leaves
      if (*abort_flag)
        for (int it = max(0, issued - kStages); it < issued; ++it)
          for (int i = 0; i < (1 << 20); ++i)
            if (mbar_try_wait(smem_u32(&bars[it % kStages]), (it / kStages) & 1)) break;
    }
  } else {
    // ----------------------------------------------------------- consumers
    // B operand of the QK product: an 8-bit row delivers 4 neighbouring dims
    // a lane (dims 4t..4t+3 of a 16-dim chunk), so the MMA's k slots 2t, 2t+1
    // and 2t+8, 2t+9 stand for those; f16 rows keep the natural order.
    uint32_t qb[8][2];
    {
      const __half* qp = a.q + (head0 + g) * 128;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const int d0 = 16 * kk + (kFp8 ? 4 * t : 2 * t);
        const int d1 = d0 + (kFp8 ? 2 : 8);
        qb[kk][0] = g < G ? __ldg(reinterpret_cast<const uint32_t*>(qp + d0)) : 0u;
        qb[kk][1] = g < G ? __ldg(reinterpret_cast<const uint32_t*>(qp + d1)) : 0u;
      }
    }
    const float sl2 = a.scale_log2;
    const int a_row = 16 * warp + (lane & 7) + ((lane >> 3) & 1) * 8;
    const int a_chs = lane >> 4;
    const int v_row = 16 * warp + (lane & 7) + ((lane >> 4) & 1) * 8;
    const int v_chs = (lane >> 3) & 1;

    for (int it = 0; it < n_stages; ++it) {
      const int st = it % kStages;
      if (!mbar_wait(smem_u32(&bars[st]), (it / kStages) & 1, a.err, 2, abort_flag)) break;
      const uint32_t kb = smem_u32(smem + st * kStageBytes);
      const uint32_t vb = kb + kVOff;
      const float* sc_st = scales + st * kScaleFloats;

      // Scores of this warp's 16 keys of each tile: x = tile; [0],[1] key g
      // (heads 2t, 2t+1); [2],[3] key g+8.
      float s[kTiles][4], inv_vs[kTiles][2];
      bool masked = false;
      uint32_t keep[kTiles][2];  // V halves to keep: keys 2t, 2t+1 / 2t+8, 2t+9
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        float sc[4] = {0.f, 0.f, 0.f, 0.f};
        if (kFp8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = 2 * i + a_chs;
            const uint32_t addr = kb + x * kTileBytes + a_row * 128 + ((c ^ (a_row & 7)) << 4);
            uint32_t r0, r1, r2, r3;
            ldsm_x4(addr, r0, r1, r2, r3);
            mma16816(sc, f16x2_of_e4m3x2(r0), f16x2_of_e4m3x2(r1), f16x2_of_e4m3x2(r0 >> 16),
                     f16x2_of_e4m3x2(r1 >> 16), qb[2 * i][0], qb[2 * i][1]);
            mma16816(sc, f16x2_of_e4m3x2(r2), f16x2_of_e4m3x2(r3), f16x2_of_e4m3x2(r2 >> 16),
                     f16x2_of_e4m3x2(r3 >> 16), qb[2 * i + 1][0], qb[2 * i + 1][1]);
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const int c = 2 * kk + a_chs;
            const uint32_t addr =
                kb + (c >> 3) * (kTileBytes / 2) + a_row * 128 + (((c & 7) ^ (a_row & 7)) << 4);
            uint32_t a0, a1, a2, a3;
            ldsm_x4(addr, a0, a1, a2, a3);
            mma16816(sc, a0, a1, a2, a3, qb[kk][0], qb[kk][1]);
          }
        }
        const bool there = it * kTiles + x < nt;
        const int kbase = there ? list.key0(t0 + it * kTiles + x) + 16 * warp : 0;
        const bool none = !there || (kPaged && bad_tile[st * 2 + x]);
        const bool part = none || list.partial(kbase);
        masked |= part;
        float f0 = sl2, f1 = sl2, lv0 = 0.f, lv1 = 0.f;
        inv_vs[x][0] = inv_vs[x][1] = 1.f;
        if (kFp8) {
          const int i0 = x * kKeys + 16 * warp + g;
          f0 *= sc_st[i0];
          f1 *= sc_st[i0 + 8];
          // a zero row (scale 0) has zero codes: any positive scale serves
          const float v0 = fmaxf(sc_st[2 * kKeys + i0], 0x1p-60f);
          const float v1 = fmaxf(sc_st[2 * kKeys + i0 + 8], 0x1p-60f);
          lv0 = __log2f(v0);
          lv1 = __log2f(v1);
          inv_vs[x][0] = __fdividef(1.f, v0);
          inv_vs[x][1] = __fdividef(1.f, v1);
        }
        s[x][0] = fmaf(sc[0], f0, lv0);
        s[x][1] = fmaf(sc[1], f0, lv0);
        s[x][2] = fmaf(sc[2], f1, lv1);
        s[x][3] = fmaf(sc[3], f1, lv1);
        if (part) {
          const bool k0 = !none && list.sees(kbase + g), k1 = !none && list.sees(kbase + g + 8);
          if (!k0) {
            s[x][0] = s[x][1] = -INFINITY;
            inv_vs[x][0] = 1.f;
          }
          if (!k1) {
            s[x][2] = s[x][3] = -INFINITY;
            inv_vs[x][1] = 1.f;
          }
          const int q = kbase + 2 * t;
          keep[x][0] = none ? 0u : (list.sees(q) ? 0xFFFFu : 0u) | (list.sees(q + 1) ? 0xFFFF0000u : 0u);
          keep[x][1] = none ? 0u : (list.sees(q + 8) ? 0xFFFFu : 0u) | (list.sees(q + 9) ? 0xFFFF0000u : 0u);
        } else {
          keep[x][0] = keep[x][1] = 0xFFFFFFFFu;
        }
      }
      float mx0 = fmaxf(s[0][0], s[0][2]), mx1 = fmaxf(s[0][1], s[0][3]);
      if (kTiles == 2) {
        mx0 = fmaxf(mx0, fmaxf(s[kTiles - 1][0], s[kTiles - 1][2]));
        mx1 = fmaxf(mx1, fmaxf(s[kTiles - 1][1], s[kTiles - 1][3]));
      }
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
      }
      const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
      const float al0 = ex2(m0 - mn0), al1 = ex2(m1 - mn1);
      l0 *= al0;
      l1 *= al1;
      m0 = mn0;
      m1 = mn1;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        o[mt][0] *= al0;
        o[mt][1] *= al1;
        o[mt][2] *= al0;
        o[mt][3] *= al1;
      }
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        const float p0 = ex2(s[x][0] - mn0), p1 = ex2(s[x][1] - mn1);
        const float p2 = ex2(s[x][2] - mn0), p3 = ex2(s[x][3] - mn1);
        if (kFp8) {
          l0 += p0 * inv_vs[x][0] + p2 * inv_vs[x][1];
          l1 += p1 * inv_vs[x][0] + p3 * inv_vs[x][1];
        } else {
          l0 += p0 + p2;
          l1 += p1 + p3;
        }
        const uint32_t pb0 = movm_t(pack_half2(p0, p1));
        const uint32_t pb1 = movm_t(pack_half2(p2, p3));
        const uint32_t z0 = keep[x][0], z1 = keep[x][1];
        if (kFp8) {
          // A byte pair of the transposed load is (dim 2g, dim 2g+1) of keys
          // 2t and 2t+1: MMA rows g and g+8 stand for dims 2g and 2g+1.
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = 2 * i + a_chs;
            const uint32_t addr = vb + x * kTileBytes + a_row * 128 + ((c ^ (a_row & 7)) << 4);
            uint32_t r[4];
            ldsm_x4_t(addr, r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int q = 0; q < 4; ++q) r[q] = __byte_perm(r[q], 0u, 0x3120);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t a0 = f16x2_of_e4m3x2(r[2 * h]), a1 = f16x2_of_e4m3x2(r[2 * h] >> 16);
              uint32_t a2 = f16x2_of_e4m3x2(r[2 * h + 1]), a3 = f16x2_of_e4m3x2(r[2 * h + 1] >> 16);
              if (masked) {
                a0 &= z0;
                a1 &= z0;
                a2 &= z1;
                a3 &= z1;
              }
              mma16816(o[2 * i + h], a0, a1, a2, a3, pb0, pb1);
            }
          }
        } else {
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            const int c = 2 * mt + v_chs;
            const uint32_t addr =
                vb + (c >> 3) * (kTileBytes / 2) + v_row * 128 + (((c & 7) ^ (v_row & 7)) << 4);
            uint32_t a0, a1, a2, a3;
            ldsm_x4_t(addr, a0, a1, a2, a3);
            if (masked) {
              a0 &= z0;
              a1 &= z0;
              a2 &= z1;
              a3 &= z1;
            }
            mma16816(o[mt], a0, a1, a2, a3, pb0, pb1);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars[kStages + st]));
    }
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
  }
  __syncthreads();  // every stage consumed: the ring becomes the merge area
  // This split's result is valid unless it is empty or a wait gave up; an
  // invalid split contributes weight 0 to the merge.
  const bool valid = nt > 0 && !*abort_flag;

  RedSmem* red = reinterpret_cast<RedSmem*>(smem);
  FinSmem* fin = reinterpret_cast<FinSmem*>(smem + kFinOffset);
  if (valid && warp < 4) {
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      const int d0 = 16 * mt + (kFp8 ? 2 * g : g), d1 = d0 + (kFp8 ? 1 : 8);
      red->o[warp][d0][2 * t] = o[mt][0];
      red->o[warp][d0][2 * t + 1] = o[mt][1];
      red->o[warp][d1][2 * t] = o[mt][2];
      red->o[warp][d1][2 * t + 1] = o[mt][3];
    }
    if (g == 0) {
      red->m[warp][2 * t] = m0;
      red->m[warp][2 * t + 1] = m1;
      red->l[warp][2 * t] = l0;
      red->l[warp][2 * t + 1] = l1;
    }
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    const int d = threadIdx.x;
    for (int hd = 0; hd < G; ++hd) {
      float res = 0.f, lse = -INFINITY;
      if (valid) {
        float M = red->m[0][hd];
#pragma unroll
        for (int w = 1; w < 4; ++w) M = fmaxf(M, red->m[w][hd]);
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float sc = ex2(red->m[w][hd] - M);
          L += red->l[w][hd] * sc;
          O += red->o[w][d][hd] * sc;
        }
        if (L != 0.f) {  // L == 0: every key of the split was left out
          res = O / L;
          lse = M + __log2f(L);
        }
      }
      if (a.nks == 1) {
        if (valid || !pos_ok) a.out[(head0 + hd) * 128 + d] = __float2half_rn(res);
      } else if (kCluster) {
        fin->o[hd][d] = res;
        if (d == 0) fin->lse[hd] = lse;
      } else {
        a.part_o[((head0 + hd) * a.nks + split) * 128 + d] = res;
        if (d == 0) a.part_lse[(head0 + hd) * a.nks + split] = lse;
      }
    }
  }
  if (kCluster && a.nks > 1) {
    // Every CTA of the cluster reaches both barriers (no early exit above),
    // so the cluster cannot deadlock; the second keeps each CTA's shared
    // memory alive until the others have read it.
    cluster_sync_all();
    const uint32_t me = cluster_ctarank();
    if (threadIdx.x < 128) {
      const int d = threadIdx.x;
      for (int hd = (int)me; hd < G; hd += a.nks) {
        a.out[(head0 + hd) * 128 + d] = merge_splits(a.nks, [&](int s, bool want_lse) {
          return want_lse ? ld_dsmem_f32(&fin->lse[hd], (uint32_t)s)
                          : ld_dsmem_f32(&fin->o[hd][d], (uint32_t)s);
        });
      }
    }
    cluster_sync_all();
  }
}

// Workspace merge, one CTA per (sequence, query head), one thread per dim.
__global__ void __launch_bounds__(128) decode_window_merge_kernel(const DecodeWindowArgs a) {
  const int64_t row = blockIdx.x;
  const int d = threadIdx.x;
  const float* lse = a.part_lse + row * a.nks;
  const float* po = a.part_o + row * a.nks * 128 + d;
  a.out[row * 128 + d] = merge_splits(a.nks, [&](int s, bool want_lse) {
    return want_lse ? lse[s] : po[s * 128];
  });
}

template <bool kFp8, bool kPaged, bool kCluster>
cudaError_t set_attrs() {
  auto k = decode_window_kernel<kFp8, kPaged, kCluster>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kFp8 ? kSmemFp8 : kSmemF16);
  if (e == cudaSuccess && kCluster)
    e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

template <bool kFp8, bool kPaged, bool kCluster>
cudaError_t launch_split(const DecodeWindowArgs& a, const CUtensorMap& tm_k,
                         const CUtensorMap& tm_v, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.nks, a.hkv, a.batch);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kFp8 ? kSmemFp8 : kSmemF16;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  if (kCluster) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = a.nks;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, decode_window_kernel<kFp8, kPaged, kCluster>, tm_k, tm_v, a);
}

template <bool kFp8, bool kPaged>
cudaError_t launch_variant(const DecodeWindowArgs& a, const CUtensorMap& tm_k,
                           const CUtensorMap& tm_v, cudaStream_t s) {
  const bool cluster = a.nks > 1 && a.cluster;
  cudaError_t e = cluster ? launch_split<kFp8, kPaged, true>(a, tm_k, tm_v, s)
                          : launch_split<kFp8, kPaged, false>(a, tm_k, tm_v, s);
  if (e != cudaSuccess || a.nks == 1 || cluster) return e;
  decode_window_merge_kernel<<<(unsigned)((int64_t)a.batch * a.hq), 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t decode_window_set_attributes() {
  const cudaError_t es[] = {set_attrs<false, false, false>(), set_attrs<false, false, true>(),
                            set_attrs<false, true, false>(),  set_attrs<false, true, true>(),
                            set_attrs<true, true, false>(),   set_attrs<true, true, true>()};
  for (cudaError_t x : es)
    if (x != cudaSuccess) return x;
  return cudaSuccess;
}

cudaError_t launch_decode_window(const DecodeWindowArgs& a, const CUtensorMap& tm_k,
                                 const CUtensorMap& tm_v, cudaStream_t s) {
  if (a.k_scales) return launch_variant<true, true>(a, tm_k, tm_v, s);
  return a.page_table ? launch_variant<false, true>(a, tm_k, tm_v, s)
                      : launch_variant<false, false>(a, tm_k, tm_v, s);
}

}  // namespace grout
