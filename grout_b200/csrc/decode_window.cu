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
// HBM-bound; one CTA per split, KV head and sequence.  A producer warp fills a
// 96 KB TMA ring with 64-key tiles, three of f16 or six of 8-bit keys; a
// group of four consumer warps takes a tile, each warp 16 of its keys.  f16
// tiles have one group; 8-bit tiles, which take as long to consume and half as
// long to load, have two that take turns.  (A stage of the ring always belongs
// to the same group: a group that skipped phases of a stage's barrier could
// take an older phase of the same parity for its own.)  S^T = K Q^T and
// O^T += V^T P^T run on mma.sync m16n8k16 with the GQA group on the 8-wide N
// side, as in decode.cu.
// The warps merge through shared memory.  Up to 16 splits form a thread-block
// cluster: each CTA pushes its heads' results into the shared memory of the
// CTA that owns the head (no round trip, one barrier), which writes the row;
// more splits go through the caller's workspace and a merge kernel.
//
// Keys that are not seen get no weight and their V rows are zeroed before the
// product, so that whatever they hold (an unwritten page, a NaN) stays out.
//
// Measured on B200: f16, 64 sequences, window 4096 behind 64 sinks, 64/8 heads
// (1.09 GB): 155 us, 7.1 TB/s; 8-bit, 64 ragged sequences of up to 8192 keys,
// 32/8 heads (0.75 GB): 112 us, 6.6 TB/s (both in a graph; 160 and 126 us a call
// in a stream).  A 64-key tile of 8-bit keys takes a group about 0.8 us; two CTAs
// per SM, two groups each, just keep up with the memory.  One sequence is
// latency: 5.9 us for a window of 1024 (launch, position, first tile, two
// merges); 8 heads of 32768 8-bit keys (69 MB) 20 us in 32 splits, of which 9.3
// are there for 1024 keys in as many splits, 2.5 of them the merge launch (6.8 us
// in 8 splits, which a cluster merges).
//
// Range checks on the device as in decode.cu: a position >= max_seq records
// 0x200 and the row is zero; a page-table entry outside the pool that holds a
// visible key records 0x201 and its tile is left out of the softmax.
#include "fp8.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "split_merge.cuh"

namespace grout {
namespace {

constexpr int kKeys = 64;  // keys per tile
constexpr float kSlack = 8.0f;  // log2 units: weights stay below 2^8, well inside f16
constexpr int kRingBytes = 98304;
constexpr int kMaxStages = 6;
// Consumer warps; one more produces.
__host__ __device__ constexpr int consumers(bool fp8) { return fp8 ? 8 : 4; }
__host__ __device__ constexpr int threads(bool fp8) { return 32 * (consumers(fp8) + 1); }
constexpr int kCtlBytes = 256;     // full/empty barriers, abort flag, per-stage tile masks
// Split results pushed by the CTAs of a cluster: for each head that this CTA
// owns (head % splits == rank), [split] rows of 128 values, then [split] lse.
// At most ceil(8 / n) * n rows for n splits: 16.
constexpr int kRecvRows = 16;
constexpr int kRecvBytes = kRecvRows * (128 + 1) * 4;
constexpr int kOffCtl = kRingBytes;
constexpr int kOffStat = kOffCtl + kCtlBytes;  // m, then l * 2^(m - M), of each warp and head
constexpr int kStatBytes = 2 * 8 * 8 * 4;
constexpr int kOffRecv = kOffStat + kStatBytes;
constexpr int kOffScales = kOffRecv + kRecvBytes;  // 8-bit: [stage][K, V][64]
constexpr int kSmemF16 = kOffScales + 1024;
constexpr int kSmemFp8 = kSmemF16 + kMaxStages * 2 * kKeys * 4;

// Each warp's O^T, scaled to the common maximum; 132: conflict-free writes
// (lanes write 8 neighbouring dims of 4 head pairs) and 16-byte reads.
struct RedSmem {
  float o[8][8][132];  // [warp][head][dim]
};
static_assert(sizeof(RedSmem) <= kRingBytes, "the merge area must fit in the ring");

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_address(const float* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  return remote;
}
__device__ __forceinline__ void st_peer(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_peer4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}

__device__ __forceinline__ float fmax_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
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
    n = sink_tiles + (int)(((uint32_t)len + kKeys - 1) / kKeys) - first;  // (len up to 2^31 - 1)
  }
  __device__ __forceinline__ int key0(int i) const { return (i < sink_tiles ? i : i + skip) * kKeys; }
  __device__ __forceinline__ bool sees(int key) const {
    return key < kv_len && (key >= lo || key < sinks);
  }
  // whether tile i of the list may hold keys that are not seen: the sinks'
  // last tile, the window's first one, the last one
  __device__ __forceinline__ bool partial(int i) const {
    return i == sink_tiles - 1 || i == sink_tiles || i == n - 1;
  }
};

template <bool kFp8, bool kPaged, bool kCluster>
__global__ void __launch_bounds__(threads(kFp8), 2)
    decode_window_kernel(const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const DecodeWindowArgs a) {
  constexpr int kTileBytes = kKeys * 128 * (kFp8 ? 1 : 2);  // of K; as much of V follows
  constexpr int kStageBytes = 2 * kTileBytes;
  constexpr int kStages = kRingBytes / kStageBytes;
  constexpr int kWarps = consumers(kFp8);
  constexpr int kGroups = kWarps / 4;
  static_assert(kStages % kGroups == 0, "a stage belongs to one group");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffCtl);  // full[kStages], empty[kStages]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * kStages);
  volatile int* bad_tile = abort_flag + 1;  // [kStages]: a page outside the pool
  float* recv = reinterpret_cast<float*>(smem + kOffRecv);
  float* scales = reinterpret_cast<float*>(smem + kOffScales);

  if (kCluster) cluster_arrive();  // "this CTA runs": awaited before its peers' memory is written

  const int split = blockIdx.x;
  const int kh = blockIdx.y;
  const int b = blockIdx.z;
  const int G = a.hq / a.hkv;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const uint32_t pos = a.d_position[b];
  if (threadIdx.x == 32 * kWarps) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&bars[i]), 1);
      mbar_init(smem_u32(&bars[kStages + i]), 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  const bool pos_ok = pos < (uint32_t)a.max_seq;
  if (!pos_ok && split == 0 && kh == 0 && threadIdx.x == 0 && a.err)
    atomicCAS(a.err, 0, DEV_ERR_POSITION);
  const TileList list(pos_ok ? (int)pos + 1 : 0, a.window, a.sinks);
  const int tps = (list.n + a.nks - 1) / a.nks;
  const int t0 = min(split * tps, list.n);
  const int nt = min(tps, list.n - t0);
  const int64_t head0 = (int64_t)b * a.hq + (int64_t)kh * G;
  __syncthreads();

  // Consumer state lives at function scope so it survives the CTA barrier
  // that frees the ring for the cross-warp merge.
  const int g = lane >> 2;  // MMA row group: key (S^T) / dim (O^T) offset; head for Q
  const int t = lane & 3;   // MMA column pair: heads 2t, 2t+1
  float m0 = -1.0e30f, m1 = -1.0e30f, l0 = 0.f, l1 = 0.f;
  float o[8][4];
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    // The warp looks 32 tiles up at once (a lane each), so that the loop over
    // stages holds no division and no table load: issuing one stage must not
    // take longer than consuming it.
    int row_l = 0, outer_l = 0, bad_l = 0;  // of tile (it & ~31) + lane of the split
    int it = 0;
    for (; it < nt; ++it) {
      const int st = it % kStages;
      if ((it & 31) == 0) {
        bad_l = 0;
        outer_l = b;  // sequence (contiguous caches) or page (paged pool)
        if (it + lane < nt) {
          row_l = list.key0(t0 + it + lane);
          if (kPaged) {
            // a 64-key tile never straddles a page (page_size % 64 == 0)
            const int pg = row_l / a.page_size;
            outer_l = __ldg(a.page_table + (int64_t)b * a.table_stride + pg);
            row_l -= pg * a.page_size;
            if (outer_l < 0 || outer_l >= a.num_pages) {
              // load page 0 instead and leave the tile out of the softmax
              if (a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
              outer_l = 0;
              bad_l = 1;
            }
          }
        }
      }
      const int row = __shfl_sync(0xffffffffu, row_l, it & 31);
      const int outer = __shfl_sync(0xffffffffu, outer_l, it & 31);
      const int bad = __shfl_sync(0xffffffffu, bad_l, it & 31);
      if (it >= kStages && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars[kStages + st]),
                                                              (it / kStages - 1) & 1, a.err, 1, abort_flag)))
        break;
      const uint32_t full = smem_u32(&bars[st]);
      if (lane == 0) {
        bad_tile[st] = bad;
        mbar_arrive_expect_tx(full, kStageBytes + (kFp8 ? 2 * kKeys * 4 : 0));
      }
      __syncwarp();
      // lane 0 loads K, lane 1 V, and each its tile's 64 scales (256-byte
      // aligned: row % 64 == 0)
      if (lane < 2) {
        const CUtensorMap* map = lane == 0 ? &tm_k : &tm_v;
        const uint32_t dst = smem_u32(smem + st * kStageBytes + lane * kTileBytes);
        if (kFp8) {
          const int64_t off = ((int64_t)outer * a.hkv + kh) * a.page_size + row;
          bulk_load(smem_u32(scales + (2 * st + lane) * kKeys),
                    (lane == 0 ? a.k_scales : a.v_scales) + off, kKeys * 4, full);
          tma_load_4d(dst, map, full, 0, row, kh, outer);
        } else {
          tma_load_5d(dst, map, full, 0, row, 0, kh, outer);
        }
      }
    }
    // a wait gave up: let the copies in flight land before the CTA leaves
    if (*abort_flag)
      for (int i = max(0, it - kStages); i < it; ++i)
        for (int n = 0; n < (1 << 20); ++n)
          if (mbar_try_wait(smem_u32(&bars[i % kStages]), (i / kStages) & 1)) break;
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
    const int k16 = 16 * (warp & 3);  // this warp's keys of a tile
    const int a_row = k16 + (lane & 7) + ((lane >> 3) & 1) * 8;
    const int a_chs = lane >> 4;
    const int v_row = k16 + (lane & 7) + ((lane >> 4) & 1) * 8;
    const int v_chs = (lane >> 3) & 1;

    for (int it = warp >> 2; it < nt; it += kGroups) {
      const int st = it % kStages;
      if (!mbar_wait(smem_u32(&bars[st]), (it / kStages) & 1, a.err, 2, abort_flag)) break;
      const uint32_t kb = smem_u32(smem + st * kStageBytes);
      const uint32_t vb = kb + kTileBytes;

      // Every load of the tile first: each waited for where it is used would
      // put its latency into the chain (K, then V while the scores are made).
      float f0 = sl2, f1 = sl2, v0 = 1.f, v1 = 1.f;
      if (kFp8) {
        const float* sp = scales + 2 * st * kKeys + k16 + g;
        f0 *= sp[0];
        f1 *= sp[8];
        // A zero row (scale 0) has zero codes: any positive scale serves.  (Below
        // 2^-60 a row's values are under 2^-51, which no f16 output shows.)  A
        // NaN stays one, as in the read-back.
        v0 = fmax_nan(sp[kKeys], 0x1p-60f);
        v1 = fmax_nan(sp[kKeys + 8], 0x1p-60f);
      }
      constexpr int kFrag = kFp8 ? 4 : 8;
      uint32_t kf[kFrag][4], vf[kFrag][4];
#pragma unroll
      for (int i = 0; i < kFrag; ++i) {
        const int c = 2 * i + a_chs;
        const uint32_t addr = kb + (kFp8 ? 0 : (c >> 3) * (kTileBytes / 2)) + a_row * 128 + (((c & 7) ^ (a_row & 7)) << 4);
        ldsm_x4(addr, kf[i][0], kf[i][1], kf[i][2], kf[i][3]);
      }
#pragma unroll
      for (int i = 0; i < kFrag; ++i) {
        // f16: the transposed tile's keys on the MMA's k side; 8-bit: as K
        const int row = kFp8 ? a_row : v_row, c = 2 * i + (kFp8 ? a_chs : v_chs);
        const uint32_t addr = vb + (kFp8 ? 0 : (c >> 3) * (kTileBytes / 2)) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        ldsm_x4_t(addr, vf[i][0], vf[i][1], vf[i][2], vf[i][3]);
      }
      const bool none = kPaged && bad_tile[st];
      __syncwarp();  // the tile is in registers: its stage can be filled again
      if (lane == 0) mbar_arrive(smem_u32(&bars[kStages + st]));
      // Scores: [0],[1] key g (heads 2t, 2t+1); [2],[3] key g+8.  Two chains of
      // four products each.
      float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kFrag; ++i) {
        const uint32_t(&r)[4] = kf[i];
        if (kFp8) {
          mma16816(sc, f16x2_of_e4m3_lo(r[0]), f16x2_of_e4m3_lo(r[1]), f16x2_of_e4m3_hi(r[0]),
                   f16x2_of_e4m3_hi(r[1]), qb[2 * i][0], qb[2 * i][1]);
          mma16816(sd, f16x2_of_e4m3_lo(r[2]), f16x2_of_e4m3_lo(r[3]), f16x2_of_e4m3_hi(r[2]),
                   f16x2_of_e4m3_hi(r[3]), qb[2 * i + 1][0], qb[2 * i + 1][1]);
        } else {
          mma16816(i & 1 ? sd : sc, r[0], r[1], r[2], r[3], qb[i][0], qb[i][1]);
        }
      }
      const bool part = none || list.partial(t0 + it);
      float lv0 = 0.f, lv1 = 0.f, iv0 = 1.f, iv1 = 1.f;
      if (kFp8) {
        lv0 = __log2f(v0);
        lv1 = __log2f(v1);
        iv0 = __fdividef(1.f, v0);
        iv1 = __fdividef(1.f, v1);
      }
      float s0 = fmaf(sc[0] + sd[0], f0, lv0), s1 = fmaf(sc[1] + sd[1], f0, lv0);
      float s2 = fmaf(sc[2] + sd[2], f1, lv1), s3 = fmaf(sc[3] + sd[3], f1, lv1);
      uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;  // V halves: keys 2t, 2t+1 / 2t+8, 2t+9
      if (part) {
        const int kbase = list.key0(t0 + it) + k16;
        if (none || !list.sees(kbase + g)) s0 = s1 = -INFINITY, iv0 = 1.f;
        if (none || !list.sees(kbase + g + 8)) s2 = s3 = -INFINITY, iv1 = 1.f;
        const int q = kbase + 2 * t;
        keep0 = none ? 0u : (list.sees(q) ? 0xFFFFu : 0u) | (list.sees(q + 1) ? 0xFFFF0000u : 0u);
        keep1 = none ? 0u : (list.sees(q + 8) ? 0xFFFFu : 0u) | (list.sees(q + 9) ? 0xFFFF0000u : 0u);
      }
      // m is a reference, not the maximum: it moves (and O is rescaled) only
      // when a score passes it by more than kSlack, so the weights stay below
      // 2^kSlack and most tiles need one vote instead of the reduction.
      const float c0 = m0 + kSlack, c1 = m1 + kSlack;
      if (__any_sync(0xffffffffu, s0 > c0 || s1 > c1 || s2 > c0 || s3 > c1)) {
        float mx0 = fmaxf(s0, s2), mx1 = fmaxf(s1, s3);
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
      }
      const float p0 = ex2(s0 - m0), p1 = ex2(s1 - m1);
      const float p2 = ex2(s2 - m0), p3 = ex2(s3 - m1);
      l0 += kFp8 ? p0 * iv0 + p2 * iv1 : p0 + p2;
      l1 += kFp8 ? p1 * iv0 + p3 * iv1 : p1 + p3;
      // The weights are rounded to f16 here (2^-11 relative, 2^-25 of the largest
      // at least): the product takes both operands in V's type, and f32 ones
      // would want twice the matrix instructions.  l keeps the f32 values.
      const uint32_t pb0 = movm_t(pack_half2(p0, p1));
      const uint32_t pb1 = movm_t(pack_half2(p2, p3));
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        uint32_t a0, a1, a2, a3;
        if (kFp8) {
          // A byte pair of the transposed load is (dim 2g, dim 2g+1) of keys 2t
          // and 2t+1: MMA rows g and g+8 stand for dims 2g and 2g+1.
          const uint32_t u = __byte_perm(vf[mt >> 1][2 * (mt & 1)], 0u, 0x3120);
          const uint32_t w = __byte_perm(vf[mt >> 1][2 * (mt & 1) + 1], 0u, 0x3120);
          a0 = f16x2_of_e4m3_lo(u);
          a1 = f16x2_of_e4m3_hi(u);
          a2 = f16x2_of_e4m3_lo(w);
          a3 = f16x2_of_e4m3_hi(w);
        } else {
          const uint32_t(&r)[4] = vf[mt % kFrag];
          a0 = r[0], a1 = r[1], a2 = r[2], a3 = r[3];
        }
        if (part) {
          a0 &= keep0;
          a1 &= keep0;
          a2 &= keep1;
          a3 &= keep1;
        }
        mma16816(o[mt], a0, a1, a2, a3, pb0, pb1);
      }
    }
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
  }
  // ------------------------------------------------- merge of the warps
  // Every warp scales its O to the maximum over all warps itself, so that the
  // sum over warps is plain additions of 16-byte reads.
  float* stat_m = reinterpret_cast<float*>(smem + kOffStat);  // [warp][head]
  float* stat_l = stat_m + 64;
  if (warp < kWarps && g == 0) {
    stat_m[warp * 8 + 2 * t] = m0;
    stat_m[warp * 8 + 2 * t + 1] = m1;
  }
  __syncthreads();  // every stage consumed: the ring becomes the merge area
  // This split's result is valid unless it is empty or a wait gave up; an
  // invalid split contributes weight 0 to the merge.
  const bool valid = nt > 0 && !*abort_flag;
  RedSmem* red = reinterpret_cast<RedSmem*>(smem);
  if (warp < kWarps) {
    float M0 = m0, M1 = m1;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 m = *reinterpret_cast<const float2*>(stat_m + w * 8 + 2 * t);
      M0 = fmaxf(M0, m.x);
      M1 = fmaxf(M1, m.y);
    }
    const float f0 = ex2(m0 - M0), f1 = ex2(m1 - M1);
    if (g == 0) {
      stat_l[warp * 8 + 2 * t] = l0 * f0;
      stat_l[warp * 8 + 2 * t + 1] = l1 * f1;
    }
    float* o0 = red->o[warp][2 * t];
    float* o1 = red->o[warp][2 * t + 1];
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      if (kFp8) {
        *reinterpret_cast<float2*>(o0 + 16 * mt + 2 * g) = make_float2(o[mt][0] * f0, o[mt][2] * f0);
        *reinterpret_cast<float2*>(o1 + 16 * mt + 2 * g) = make_float2(o[mt][1] * f1, o[mt][3] * f1);
      } else {
        o0[16 * mt + g] = o[mt][0] * f0;
        o1[16 * mt + g] = o[mt][1] * f1;
        o0[16 * mt + g + 8] = o[mt][2] * f0;
        o1[16 * mt + g + 8] = o[mt][3] * f1;
      }
    }
  }
  if (kCluster) cluster_wait();  // every CTA of the cluster runs
  __syncthreads();
  for (int hd = warp; warp < kWarps && hd < G; hd += kWarps) {  // a warp takes a head, a lane four dims
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f, lse = -INFINITY, inv = 0.f;
    if (valid) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        L += stat_l[w * 8 + hd];
        M = fmaxf(M, stat_m[w * 8 + hd]);
        fma4(acc, 1.f, *reinterpret_cast<const float4*>(&red->o[w][hd][4 * lane]));
      }
      if (L != 0.f) {  // L == 0: every key of the split was left out
        inv = 1.f / L;
        lse = M + __log2f(L);
      }
    }
    if (a.nks == 1) {
      if (valid || !pos_ok) store_row4(a.out + (head0 + hd) * 128 + 4 * lane, acc, inv);
    } else if (kCluster) {
      const int row = hd / a.nks * a.nks + split;
      const uint32_t to = peer_address(recv, hd % a.nks);
      st_peer4(to + (row * 128 + 4 * lane) * 4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      if (lane == 0) st_peer(to + (kRecvRows * 128 + row) * 4, lse);
    } else {
      const int64_t row = (head0 + hd) * a.nks + split;
      reinterpret_cast<float4*>(a.part_o + row * 128)[lane] =
          make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (lane == 0) a.part_lse[row] = lse;
    }
  }
  if (kCluster) {
    // Every CTA of the cluster reaches both barriers (no early exit above);
    // after this one nobody touches a peer's memory.
    cluster_arrive();
    cluster_wait();
    for (int hd = (int)cluster_ctarank() + warp * a.nks; warp < kWarps && hd < G; hd += kWarps * a.nks) {
      const int row0 = hd / a.nks * a.nks;
      // w_s = 2^(lse_s - max) / sum, out = sum_s w_s * O_s, rounded to f16.
      // Splits without a visible key have lse = -inf and O = 0; if all have,
      // the row is 0.  A NaN lse passes into the row.
      const float lse = lane < a.nks ? recv[kRecvRows * 128 + row0 + lane] : -INFINITY;
      const float M = warp_max(lse);
      const float w = lse == -INFINITY ? 0.f : ex2(lse - M);
      const float W = warp_sum(w);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < a.nks; ++s)
        fma4(acc, __shfl_sync(0xffffffffu, w, s),
             reinterpret_cast<const float4*>(recv + (row0 + s) * 128)[lane]);
      store_row4(a.out + (head0 + hd) * 128 + 4 * lane, acc, W != 0.f ? 1.f / W : 0.f);
    }
  }
}

// Workspace merge, one CTA per (sequence, query head): every warp forms the
// weights, takes every fourth split, and the four sums meet in shared memory.
__global__ void __launch_bounds__(128) decode_window_merge_kernel(const DecodeWindowArgs a) {
  __shared__ float4 part[4][32];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* lse = a.part_lse + row * a.nks;
  const float4* po = reinterpret_cast<const float4*>(a.part_o + row * a.nks * 128) + lane;
  float M = -INFINITY, W = 0.f;
  for (int s = lane; s < a.nks; s += 32) M = fmaxf(M, lse[s]);
  M = warp_max(M);
  for (int s = lane; s < a.nks; s += 32) W += lse[s] == -INFINITY ? 0.f : ex2(lse[s] - M);
  W = warp_sum(W);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = warp; s < a.nks; s += 4) {
    const float w = lse[s] == -INFINITY ? 0.f : ex2(lse[s] - M);
    fma4(acc, w, po[(int64_t)s * 32]);
  }
  part[warp][lane] = acc;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < 4; ++w) fma4(acc, 1.f, part[w][lane]);
    store_row4(a.out + row * 128 + 4 * lane, acc, W != 0.f ? 1.f / W : 0.f);
  }
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
  cfg.blockDim = dim3(threads(kFp8), 1, 1);
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
