// Sliding-window causal GQA prefill with sinks on the 5th-generation tensor
// cores: row p of a sequence sees key n if n <= p and (n > p - window or
// n < sinks).  O = softmax(scale Q K^T + mask) V, f16 in, f32 accumulate, P
// rounded to f16 before the PV product, f16 out.  No counterpart in the
// reference (its prefill attends to every earlier key, src/kernels.rs:
// 2570-2725).
//
// The pipeline is prefill.cu's (persistent CTAs, 512 threads: two softmax
// warpgroups, one output warpgroup, a TMA warp, an MMA warp; S and P in TMEM,
// P feeds the PV MMA from there; one pass over the keys with a lazily moved
// reference maximum).  What a window changes:
//
// Rows.  A 128-row query tile holds floor(128 / G) tokens with all G query
// heads of one KV head (row = token * G + head).  All of a tile's rows so
// need nearly the same keys: a tile of 128 tokens of one head touches
// window + 127 keys, one of 16 tokens x 8 heads window + 15, and a chunk of
// a few tokens fills one tile with every head instead of one tile per head.
// An item is two such tiles of one (sequence, KV head), or one, when the
// sequence ends in the first.  If no sequence of a call is longer than a tile
// (kShort), both chains take the one tile, one the even and one the odd key
// tiles, and the output warps join the two.
//
// Splits.  Calls with few items and long windows cut each item's keys into
// nsplit runs of tiles, an item of its own each (kSplit): the output warps store
// normalised f32 rows and their log2-sum-exp, a second kernel merges them.  One
// sequence, 5 tokens, 64/8 heads: window 4096 39 -> 18 us (8 splits), 32005 keys
// 272 -> 39 us (16).
//
// Keys.  An item streams the 64-key blocks that hold a key one of its rows
// sees (the sinks' blocks, then from the first row's window on), two blocks
// to a 128-key tile whether they are neighbours or not.  TMA loads
// each block by itself (64-row boxes), from its page or its cache row.
//
// Unseen rows.  Rows that no row of the item sees may hold anything (freed
// pages, unwritten rows, NaN).  Their scores are replaced, but 0 * NaN in the
// PV product is a NaN, so blocks without a seen key are not read (TMA fills
// an out-of-range coordinate with zeros), and warp 14 clears the unseen
// rows of the at most three partial blocks of an item in shared memory before
// the MMA warp may use their V tile.
//
// Bound by the tensor cores and the chain S -> P -> PV -> next S of each of two
// query tiles: in long windows a 128-key tile of both takes 3600 cycles, 2048
// of them MMA; a chain's turn is 1300 waiting for S (PV and QK are 1024), 480
// for the maximum, 1290 for the exponentials, 110 for the hand-over and, spread
// over an item's tiles, about 440 for the change of items.  Measured on B200:
// 8192 tokens, window 1024, 4 sinks, 32/8 heads: 148 us, 0.87 PFLOP/s of visible
// keys (0.97 with the blocks' unseen keys); six chunks of up to 700 tokens,
// window 4096, 64/8 heads: 432 us, 1.04 PFLOP/s.  Both are bursts of 100 calls in
// a graph; sustained the GPU is at its power limit (about 1.6 GHz) and they take
// 171 and 493 us, so that fewer cycles in the softmax (masks in a pass of their
// own, P handed over in halves) did not shorten it.
// 64-key blocks with two S buffers per tile took 221 us: the MMA warp could not
// issue and wait for them as fast.
#include <algorithm>

#include "internal.h"
#include "prefill_common.cuh"
#include "ptx.cuh"
#include "split_merge.cuh"

namespace grout {
namespace {

constexpr int kBM = 128;       // query rows per tile (= TMEM lanes)
constexpr int kBlk = 64;       // keys per block, two blocks per KV tile
constexpr int kSlots = 4;      // K/V ring slots (even ring entries K, odd ones V)
constexpr int kThreads = 512;  // 4 warpgroups, one persistent CTA per SM
// Register split (setmaxnreg): launched at 128 per thread (512 x 128 =
// 65536); 2 x 128 x 152 + 2 x 128 x 104 = 65536.
constexpr int kRegsOther = 104;
constexpr int kRegsSoftmax = 152;
constexpr int kOffQ = 0;          // 2 query tiles
constexpr int kOffKV = 2 * kTile; // ring
constexpr int kOffBar = kOffKV + kSlots * kTile;
constexpr int kOffL = kOffBar + 512;  // row sums, row references [item parity][tile][row]
constexpr int kOffAbort = kOffBar + 448;
constexpr int kOffTmem = kOffBar + 452;
constexpr int kOffWalk = kOffL + 2 * 2 * 2 * 128 * 4;  // each warp's place in the item list
constexpr int kOffMask = kOffWalk + 16 * 32;       // softmax warps: what masks the tiles of their item
constexpr int kSmemBytes = kOffMask + 8 * 32 + 1024;

// barrier indices (phases run on across the work items of a CTA; those of
// tile 1 skip the items that have one tile)
constexpr int kBarQ = 0;                      // + tile: Q_t landed (TMA)
constexpr int kBarQfree = 2;                  // + tile: last QK_t of the item done (commit)
constexpr int kBarFull = 4;                   // + slot
constexpr int kBarEmpty = kBarFull + kSlots;  // + slot
constexpr int kBarS = kBarEmpty + kSlots;     // + tile (commit)
constexpr int kBarP = kBarS + 2;              // + tile (4 softmax warps)
constexpr int kBarOfull = kBarP + 2;          // + tile: O_t of the item final (commit)
constexpr int kBarOempty = kBarOfull + 2;     // + tile: O_t read out (4 output warps)
constexpr int kBarL = kBarOempty + 2;         // + tile: row sums written (4 softmax warps)
constexpr int kBarClr = kBarL + 2;            // + V slot (ring slot / 2): V tile with unseen rows cleared
constexpr int kBarDrain = kBarClr + 2;        // MMAs in flight when a wait gave up
constexpr int kNumBars = kBarDrain + 1;
static_assert(kNumBars * 8 <= 448, "barriers overlap the abort flag");

__device__ __forceinline__ int ring_slot(int i) { return i % kSlots; }
__device__ __forceinline__ uint32_t ring_parity(int i) { return (uint32_t)((i / kSlots) & 1); }

// Shared memory by 32-bit addresses: generic pointers would hold two registers
// each through the softmax loop, which has none to spare.
__device__ __forceinline__ int ld_shared(uint32_t addr) {
  int v;
  asm volatile("ld.volatile.shared.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int4 ld_shared4(uint32_t addr) {
  int4 v;
  asm volatile("ld.volatile.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared(uint32_t addr, int v) {
  asm volatile("st.volatile.shared.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_shared4(uint32_t addr, int x, int y, int z, int w) {
  asm volatile("st.volatile.shared.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y),
               "r"(z), "r"(w)
               : "memory");
}
// mbar_wait with the abort flag by its shared address.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int* err, int site,
                                         uint32_t abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 0) {
      if (ld_shared(abort_flag)) return false;
      if (globaltimer() - t0 > kWaitTimeoutNs) {
        st_shared(abort_flag, 1);
        if (err) atomicCAS(err, 0, DEV_ERR_TIMEOUT_BASE + site);
        return false;
      }
    }
  }
}

__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The lowest n of 32 bits (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t bits_below(int n) {
  return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1u;
}

struct Item {
  int b, kh, q0, S, P, q_start;
  int n0, n_kv;     // KV tiles of query tile 0, of the item (tile 1 takes all)
  int t0, last;     // (kSplit) KV tile 0 is tile t0 of the whole list; index of the list's last one
  int sp, nch;      // (kSplit) split, number of splits that have tiles
  bool two;         // the item has a second query tile
  bool alt;         // (kShort) it has not, but two KV tiles or more: chain t takes those of parity t
  // KV tiles of chain t
  __device__ __forceinline__ int count(int t) const {
    return alt ? (n_kv + 1 - t) >> 1 : (t == 0 ? n0 : (two ? n_kv : 0));
  }
  int nblk, sink_blk, skip;  // 64-key blocks; entry i is block i or, past the sinks, i + skip
  int wlo, vis_end; // keys some row sees: n < sinks, and wlo <= n < vis_end
  // first key of block entry i
  __device__ __forceinline__ int key0(int i) const { return (i < sink_blk ? i : i + skip) * kBlk; }
  // whether block entry i holds a key that no row of the item sees
  __device__ __forceinline__ bool partial(int i, int sinks) const {
    const int k = key0(i);
    return k + kBlk > vis_end || (k < wlo && k + kBlk > sinks);
  }
  // whether V tile j may have rows to clear: it holds the sinks' last block, the
  // window's first one or the list's last one
  __device__ __forceinline__ bool clears(int j) const {
    return j + t0 == (sink_blk - 1) >> 1 || j + t0 == sink_blk >> 1 || j == last;
  }
};

// Walks this CTA's items: entry r * grid + c of the list (r * grid + grid - 1
// - c in odd rounds, so that the longer items at the front even out), which
// numbers, sequence by sequence, token blocks in descending order, KV heads,
// splits fastest.  A sequence whose lengths or positions fit neither the query rows
// nor the cache has no items (device error 0x200).
template <bool kShort, bool kSplit>
struct Walk {
  int r = 0, b = -1, base = 0, cnt = 0;
  int S = 0, P = 0, pairs = 0, q_start = 0;

  // Items of sequence n (and its numbers).
  __device__ __forceinline__ void enter(const PrefillWindowArgs& a, int n) {
    cnt = 0;
    if (n >= a.batch) return;
    if (a.cu_q) {
      q_start = a.cu_q[n];
      S = a.cu_q[n + 1] - q_start;
    } else {
      q_start = 0;
      S = a.single_len;
    }
    P = a.pos0 ? a.pos0[n] : 0;
    const int ks = a.kv_start ? a.kv_start[n] : 0;
    if (S == 0) return;
    if (S < 0 || q_start < 0 || (int64_t)q_start + S > a.q_rows || P < 0 || ks < 0 ||
        (int64_t)ks + P + S > a.max_keys) {
      if (a.err) atomicCAS(a.err, 0, DEV_ERR_POSITION);
      return;
    }
    pairs = (S + 2 * a.tok - 1) / (2 * a.tok);
    cnt = pairs * a.hkv * (kSplit ? a.nsplit : 1);
  }

  // Called by whole warps: past the current sequence, each lane reads one of
  // the next 32 (one after the other would cost a memory latency each).
  __device__ __forceinline__ bool next(const PrefillWindowArgs& a, Item& it) {
    const int G = gridDim.x, c = blockIdx.x, lane = threadIdx.x & 31;
    for (;;) {  // (past the splits without tiles)
      const int k = r * G + ((r & 1) ? G - 1 - c : c);
      ++r;
      while (k >= base + cnt) {
        if (b >= a.batch - 1) return false;
        base += cnt;
        Walk w;
        w.enter(a, b + 1 + lane);
        int sum = w.cnt;  // of the lanes up to this one
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, sum, off);
          if (lane >= off) sum += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, k < base + sum);
        const int src = hit ? __ffs(hit) - 1 : 31;
        base += __shfl_sync(0xffffffffu, sum - w.cnt, src);
        cnt = __shfl_sync(0xffffffffu, w.cnt, src);
        S = __shfl_sync(0xffffffffu, w.S, src);
        P = __shfl_sync(0xffffffffu, w.P, src);
        pairs = __shfl_sync(0xffffffffu, w.pairs, src);
        q_start = __shfl_sync(0xffffffffu, w.q_start, src);
        b += 1 + src;
      }
      int local = k - base;
      it.sp = 0;
      if (kSplit) {
        it.sp = local % a.nsplit;
        local /= a.nsplit;
      }
      const int back = local / a.hkv;  // pairs behind this one
      const int pair = pairs - 1 - back;
      it.b = b;
      it.kh = local - back * a.hkv;
      it.S = S;
      it.P = P;
      it.q_start = q_start;
      it.q0 = pair * 2 * a.tok;
      it.two = S > it.q0 + a.tok;
      const int end0 = P + min(it.q0 + a.tok, S);
      it.vis_end = P + min(it.q0 + 2 * a.tok, S);
      it.wlo = max(0, P + it.q0 - a.window + 1);
      const int first = it.wlo / kBlk;
      it.sink_blk = min(first, (int)(((int64_t)a.sinks + kBlk - 1) / kBlk));
      it.skip = first - it.sink_blk;
      it.nblk = (it.vis_end + kBlk - 1) / kBlk - it.skip;
      it.n_kv = (it.nblk + 1) / 2;
      it.n0 = ((end0 + kBlk - 1) / kBlk - it.skip + 1) / 2;
      it.t0 = 0;
      it.last = it.n_kv - 1;
      it.nch = 1;
      if (kSplit) {
        // runs of tps tiles of query tile 0; the last run takes tile 1's further ones too
        const int tps = (it.n0 + a.nsplit - 1) / a.nsplit;
        it.nch = (it.n0 + tps - 1) / tps;
        if (it.sp >= it.nch) continue;
        it.t0 = it.sp * tps;
        const int end = min(it.n0, it.t0 + tps);
        it.n_kv = (end == it.n0 ? it.n_kv : end) - it.t0;
        it.n0 = end - it.t0;
        it.last -= it.t0;
      }
      it.alt = kShort && !it.two && it.n_kv > 1;
      return true;
    }
  }
};

// kShort: no sequence is longer than a query tile; its items have one tile, and
// both chains work on it (code that the other calls do not carry).
template <bool kPaged, bool kShort, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_window_kernel(const __grid_constant__ CUtensorMap tm_q,
                          const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v, const PrefillWindowArgs a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023) & ~1023u;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  auto bar = [&](int i) -> uint32_t { return smem_base + kOffBar + 8 * i; };
  auto wait = [&](int i, uint32_t parity, int site) -> bool {
    return bar_wait(bar(i), parity & 1u, a.err, site, smem_base + kOffAbort);
  };

  if (threadIdx.x < kNumBars) {  // a thread each: one after the other took 0.2 us of a short call
    const int i = threadIdx.x;
    // P, Oempty, L: one arrival per warp of a warpgroup
    const bool four = (i >= kBarP && i < kBarP + 2) || (i >= kBarOempty && i < kBarOempty + 2) ||
                      (i >= kBarL && i < kBarL + 2);
    // a V slot is empty once the MMA warp and warp 14 are through with it
    const bool v_empty = i == kBarEmpty + 1 || i == kBarEmpty + 3;
    mbar_init(bar(i), four ? 4 : (v_empty ? 2 : 1));
    if (i == 0) st_shared(smem_base + kOffAbort, 0);
    fence_mbar_init();
  }
  if (warp == 13) {
    tmem_alloc(smem_base + kOffTmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)ld_shared(smem_base + kOffTmem);

  // The next item of a whole warp.  Its place in the list waits in shared
  // memory between items: no role has eight registers to spare for it.
  const uint32_t place = smem_base + kOffWalk + warp * 32;
  if (lane == 0) {
    st_shared4(place, 0, -1, 0, 0);
    st_shared4(place + 16, 0, 0, 0, 0);
  }
  __syncwarp();
  auto next_item = [&](Item& x) -> bool {
    const int4 p0 = ld_shared4(place), p1 = ld_shared4(place + 16);
    Walk<kShort, kSplit> w;
    w.r = p0.x, w.b = p0.y, w.base = p0.z, w.cnt = p0.w;
    w.S = p1.x, w.P = p1.y, w.pairs = p1.z, w.q_start = p1.w;
    const bool has = w.next(a, x);
    __syncwarp();
    if (lane == 0) {
      st_shared4(place, w.r, w.b, w.base, w.cnt);
      st_shared4(place + 16, w.S, w.P, w.pairs, w.q_start);
    }
    __syncwarp();
    return has;
  };
  Item it = {};
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 12) {
      // ---------------------------------------------------------- producer
      // The whole warp: it looks 32 blocks up at once (a lane each), and lanes
      // 0..3 issue the four loads of a K or V tile together (64 rows x 64 dims
      // each: a block lies in one page).  One lane doing all of it took longer
      // for a tile than a chain of few rows needs.
      if (lane == 0) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
      }
      __syncwarp();
      auto wait_all = [&](int i, uint32_t parity, int site) -> bool {
        return __all_sync(0xffffffffu, wait(i, parity, site));
      };
      const int hh = lane & 1, half = lane >> 1;  // lanes 0..3: block of the tile, 64-dim half
      int ring = 0, nq0 = 0, nq1 = 0;
      Item nx = {};
      bool ok = true, has = next_item(nx);
      auto load_q = [&](int t, int& nq) -> bool {
        // a query buffer is refilled as soon as its last QK of the item before has run
        if (nq > 0 && !wait_all(kBarQfree + t, nq - 1, 11 + t)) return false;
        ++nq;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar(kBarQ + t), a.tok * a.group * 256);
          const uint32_t dst = smem_base + kOffQ + t * kTile;
          const int row = it.q_start + it.q0 + (it.two ? t * a.tok : 0), head = it.kh * a.group;
          tma_load_3d(dst, &tm_q, bar(kBarQ + t), 0, head, row);
          tma_load_3d(dst + kBox, &tm_q, bar(kBarQ + t), 64, head, row);
        }
        return true;
      };
      auto load_kv = [&](const CUtensorMap* map, int row, int outer) -> bool {
        const int slot = ring_slot(ring);
        if (ring >= kSlots && !wait_all(kBarEmpty + slot, ring_parity(ring) ^ 1u, 10)) return false;
        const uint32_t full = bar(kBarFull + slot);
        if (lane == 0) mbar_arrive_expect_tx(full, kTile);
        __syncwarp();
        if (lane < 4)
          tma_load_4d(smem_base + kOffKV + slot * kTile + half * kBox + hh * (kBox / 2), map, full, half * 64,
                      row, it.kh, outer);
        ++ring;
        return true;
      };
      while (ok && has) {
        it = nx;
        const int ks = a.kv_start ? a.kv_start[it.b] : 0;
        if (!(ok = load_q(0, nq0))) break;
        int row_l = 0, outer_l = 0;  // of entry 2 * (t0 + (j & ~15)) + lane
        for (int j = 0; ok && j < it.n_kv; ++j) {
          if ((j & 15) == 0) {
            const int e = 2 * (j + it.t0) + lane;
            // past the last block: an out-of-range coordinate, filled with zeros
            row_l = kPaged ? 0 : a.kv_rows;
            outer_l = kPaged ? a.num_pages : (a.kv_batched ? it.b : 0);
            if (e < it.nblk) {
              const int key = it.key0(e);
              if (kPaged) {
                const int pg = key / a.page_size;
                const int page = __ldg(a.page_table + (int64_t)it.b * a.table_stride + pg);
                row_l = key - pg * a.page_size;
                if (page >= 0 && page < a.num_pages) outer_l = page;
                else if (a.err) atomicCAS(a.err, 0, DEV_ERR_PAGE);
              } else {
                row_l = ks + key;
              }
            }
          }
          const int row = __shfl_sync(0xffffffffu, row_l, (2 * j + hh) & 31);
          const int outer = __shfl_sync(0xffffffffu, outer_l, (2 * j + hh) & 31);
          ok = load_kv(&tm_k, row, outer);
          // Q_0, K_0, Q_1, then the rest
          if (ok && j == 0 && it.count(1) > 0) ok = load_q(1, nq1);
          ok = ok && load_kv(&tm_v, row, outer);
          if (j == 0) has = next_item(nx);  // off the path between two items' loads
        }
      }
      // a wait gave up: let the loads in flight land before the CTA leaves
      if (ld_shared(smem_base + kOffAbort)) {
        for (int i = max(0, ring - kSlots); i < ring; ++i)
          for (int n = 0; n < (1 << 20); ++n)
            if (mbar_try_wait(bar(kBarFull + ring_slot(i)), ring_parity(i))) break;
        for (int n = 0; nq0 > 0 && n < (1 << 20); ++n)
          if (mbar_try_wait(bar(kBarQ + 0), (nq0 - 1) & 1)) break;
        for (int n = 0; nq1 > 0 && n < (1 << 20); ++n)
          if (mbar_try_wait(bar(kBarQ + 1), (nq1 - 1) & 1)) break;
      }
    } else if (warp == 13) {
      // ------------------------------------------------------------ MMA issue
      // The whole warp runs the issue loop (warp-uniform descriptors); one
      // elected lane issues every MMA and commit.  Per KV tile j of an item:
      // PV0(j), QK0(j+1), PV1(j), QK1(j+1); the first QKs of the next item
      // follow the last PVs of this one, and its first PV_t waits until the
      // output warps have read O_t of the item before out of TMEM.
      const bool leader = elect_one();
      constexpr uint32_t idesc_qk = idesc_f16_f32(kBM, 128, 0, 0);
      constexpr uint32_t idesc_pv = idesc_f16_f32(kBM, 128, 0, 1);
      const uint32_t base16 = smem_base >> 4;
      auto commit = [&](int i) {
        if (leader) tc_commit(bar(i));
      };
      auto qk = [&](int t, int slot) {
        const uint32_t qlo = base16 + (kOffQ + t * kTile) / 16 + kDescLboK;
        const uint32_t klo = base16 + (kOffKV + slot * kTile) / 16 + kDescLboK;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32) / 16;
          if (leader) mma_ss_lo(tmem + t * 128, qlo + off, klo + off, idesc_qk, kk > 0 ? 1u : 0u);
        }
      };
      auto pv = [&](int t, int slot, bool acc) {
        const uint32_t vlo = base16 + (kOffKV + slot * kTile) / 16 + kDescLboV;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          if (leader)
            mma_ts_lo(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, vlo + kk * (2048 / 16), idesc_pv,
                      (acc || kk > 0) ? 1u : 0u);
        }
      };
      int nst[2] = {0, 0};  // items started per tile (QK_t(0) issued)
      int npv[2] = {0, 0};  // items per tile whose first PV_t has been issued
      int pc[2] = {0, 0};   // P_t tiles taken
      int nclr[2] = {0, 0}; // cleared V tiles taken, per V slot
      auto start = [&](int t, const Item& x, int iring) -> bool {
        if (x.count(t) == 0) return true;
        if (t == 1 && x.alt) iring += 2;
        if (!wait(kBarQ + t, nst[t], 20 + t) || !wait(kBarFull + ring_slot(iring), ring_parity(iring), 22))
          return false;
        ++nst[t];
        tc_fence_after();
        qk(t, ring_slot(iring));
        commit(kBarS + t);
        if (t == 1 || !x.two) commit(kBarEmpty + ring_slot(iring));
        if (x.count(t) == 1) commit(kBarQfree + t);
        return true;
      };
      auto wait_v = [&](const Item& x, int j, int iv) -> bool {
        if (!wait(kBarFull + ring_slot(iv), ring_parity(iv), 23)) return false;
        if (x.clears(j)) {
          const int vs = ring_slot(iv) >> 1;
          if (!wait(kBarClr + vs, nclr[vs], 29)) return false;
          ++nclr[vs];
        }
        return true;
      };
      auto take_p = [&](int t, bool first) -> bool {
        if (!wait(kBarP + t, pc[t], 24 + t)) return false;
        ++pc[t];
        if (first) {
          if (npv[t] > 0 && !wait(kBarOempty + t, npv[t] - 1, 26 + t)) return false;
          ++npv[t];
        }
        tc_fence_after();
        return true;
      };
      int ring = 0;
      Item cur = {}, nx = {};
      bool has = next_item(cur);
      bool ok = !has || (start(0, cur, ring) && start(1, cur, ring));
      while (has && ok) {
        const bool hn = next_item(nx);
        const int n_kv = cur.n_kv, n0 = cur.n0;
        const int nring = ring + 2 * n_kv;  // K_0 of the next item
        // One query tile: KV tile j belongs to chain j & 1, whose next one is
        // j + 2.  Chain 0 starts the next item first: with two tiles chain 1's
        // QK gives the shared K tile back.
        auto alt_step = [&](int t, int j) -> bool {
          const int iv = ring + 2 * j + 1, ik = iv + 3;
          if (!wait_v(cur, j, iv) || !take_p(t, j < 2)) return false;
          pv(t, ring_slot(iv), j > 1);
          commit(kBarEmpty + ring_slot(iv));
          if (j + 2 < n_kv) {
            if (!wait(kBarFull + ring_slot(ik), ring_parity(ik), 22)) return false;
            tc_fence_after();
            qk(t, ring_slot(ik));
            commit(kBarS + t);
            commit(kBarEmpty + ring_slot(ik));
            if (j + 4 >= n_kv) commit(kBarQfree + t);
            return true;
          }
          commit(kBarOfull + t);
          return t == 1 || !hn || start(0, nx, nring);
        };
        for (int j = 0; kShort && cur.alt && ok && j < n_kv; j += 2)
          ok = alt_step(0, j) && (j + 1 == n_kv || alt_step(1, j + 1));
        if (kShort && cur.alt && ok && hn) ok = start(1, nx, nring);
        for (int j = 0; !(kShort && cur.alt) && ok && j < n_kv; ++j) {
          const int iv = ring + 2 * j + 1, ik = ring + 2 * j + 2;
          const bool next = j + 1 < n_kv;
          ok = wait_v(cur, j, iv);
          // K(j+1) only needs the slot K(j-1) released, so it is awaited
          // here, before P0(j), keeping the wait off the PV0 -> QK0 path.
          if (ok && next) ok = wait(kBarFull + ring_slot(ik), ring_parity(ik), 22);
          if (!ok) break;
          if (j < n0) {
            if (!(ok = take_p(0, j == 0))) break;
            pv(0, ring_slot(iv), j > 0);
            if (!cur.two) commit(kBarEmpty + ring_slot(iv));
            if (j == n0 - 1) commit(kBarOfull + 0);
          }
          if (j + 1 < n0) {
            qk(0, ring_slot(ik));
            commit(kBarS + 0);
            if (!cur.two) commit(kBarEmpty + ring_slot(ik));
            if (j + 1 == n0 - 1) commit(kBarQfree + 0);
          } else if (j + 1 == n0 && hn) {
            // tile 0 is done with this item: start the next one
            if (!(ok = start(0, nx, nring))) break;
          }
          if (cur.two) {
            if (!(ok = take_p(1, j == 0))) break;
            pv(1, ring_slot(iv), j > 0);
            commit(kBarEmpty + ring_slot(iv));
            if (!next) commit(kBarOfull + 1);
            if (next) {
              qk(1, ring_slot(ik));
              commit(kBarS + 1);
              commit(kBarEmpty + ring_slot(ik));
              if (j + 1 == n_kv - 1) commit(kBarQfree + 1);
            }
          }
          if (!next && hn && !(ok = start(1, nx, nring))) break;
        }
        if (!ok) break;
        ring = nring;
        cur = nx;
        has = hn;
      }
      if (!ok) {  // let the MMAs in flight finish before their memory is given back
        commit(kBarDrain);
        for (int n = 0; n < (1 << 20); ++n)
          if (mbar_try_wait(bar(kBarDrain), 0)) break;
      }
    } else if (warp == 14) {
      // ------------------------------------- clear the unseen rows of V tiles
      // A V tile is two boxes of 128 rows x 128 bytes; the swizzle moves bytes
      // within a row only, so whole rows are cleared in place.
      int ring = 0;
      bool ok = true;
      while (ok && next_item(it)) {
        for (int j = 0; j < it.n_kv; ++j, ring += 2) {
          const int iv = ring + 1;
          ok = wait(kBarFull + ring_slot(iv), ring_parity(iv), 50);
          if (!ok) break;
          const int e0 = 2 * (j + it.t0);
          for (int e = e0; e < min(e0 + 2, it.nblk); ++e) {
            if (!it.partial(e, a.sinks)) continue;  // (a second block past the last is TMA's zeros)
            const int key = it.key0(e);
            const int lo0 = max(0, a.sinks - key), hi0 = min(kBlk, it.wlo - key);  // before the window
            const int lo1 = max(0, it.vis_end - key);                             // past the last key
            const uint32_t v = smem_base + kOffKV + ring_slot(iv) * kTile + (e & 1) * (kBox / 2);
            for (int row = lane >> 3; row < kBlk; row += 4) {
              if ((row >= lo0 && row < hi0) || row >= lo1) {
                st_shared4(v + row * 128 + (lane & 7) * 16, 0, 0, 0, 0);
                st_shared4(v + kBox + row * 128 + (lane & 7) * 16, 0, 0, 0, 0);
              }
            }
          }
          const bool cleared = it.clears(j);
          if (cleared) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (cleared) mbar_arrive(bar(kBarClr + (ring_slot(iv) >> 1)));
            mbar_arrive(bar(kBarEmpty + ring_slot(iv)));
          }
        }
      }
    } else if (warp < 12) {
      // ------------------------------------------------------------ output
      // Warp 8 + q reads TMEM lanes 32q.. (query rows) of O_t once the MMA
      // warp reports it final, frees O_t for the next item, and writes the
      // normalised rows.
      const int quad = warp & 3;
      const int row = quad * 32 + lane;
      const int G = a.group;
      const int tok = row / G, head = row - tok * G;
      const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
      auto row_stat = [&](int which, int n, int t) -> float {  // 0: sum, 1: reference
        return __int_as_float(ld_shared(smem_base + kOffL + (((which * 2 + (n & 1)) * 2 + t) * 128 + row) * 4));
      };
      int n0 = 0, n1 = 0;  // items put out per chain
      bool ok = true;
      while (ok && next_item(it)) {
        const bool both = it.count(1) > 0;  // chain 1 has a part in the item
        // two tiles: each by itself; one tile: the two chains' sums joined
#pragma unroll 1
        for (int t = 0; t < (it.two ? 2 : 1); ++t) {
          const bool join = kShort && it.alt;
          if (t == 0 || join) ok = wait(kBarOfull + 0, n0, 40) && wait(kBarL + 0, n0, 42);
          if (ok && (t == 1 || join)) ok = wait(kBarOfull + 1, n1, 41) && wait(kBarL + 1, n1, 43);
          if (!ok) break;
          tc_fence_after();
          float w0, w1 = 0.f, l;
          if (join) {
            const float ma = row_stat(1, n0, 0), mb = row_stat(1, n1, 1);
            const float m = fmaxf(ma, mb);
            w0 = ma == -INFINITY ? 0.f : ex2(ma - m);
            w1 = mb == -INFINITY ? 0.f : ex2(mb - m);
            l = row_stat(0, n0, 0) * w0 + row_stat(0, n1, 1) * w1;
          } else {
            w0 = 1.f;
            l = row_stat(0, t ? n1 : n0, t);
          }
          const float inv = l != 0.f ? 1.0f / l : 0.f;
          w0 *= inv;
          w1 *= inv;
          const int row_q = it.q0 + t * a.tok + tok;
          const bool valid = tok < a.tok && row_q < it.S;
          float* prow = nullptr;  // (kSplit) this split's row
          if (kSplit && valid) {
            const int64_t at = ((int64_t)(it.q_start + row_q) * a.hq + it.kh * G + head) * a.nsplit;
            prow = a.part_o + (at + it.sp) * 128;
            const float m = join ? fmaxf(row_stat(1, n0, 0), row_stat(1, n1, 1)) : row_stat(1, t ? n1 : n0, t);
            a.part_lse[at + it.sp] = l != 0.f ? m + __log2f(l) : -INFINITY;
            for (int s = it.nch; it.sp == 0 && s < a.nsplit; ++s) a.part_lse[at + s] = -INFINITY;
          }
          __half* orow = a.out + (int64_t)(it.q_start + row_q) * a.q_row_stride +
                         (int64_t)(it.kh * G + head) * 128;
          const uint32_t tO = tmem + 256 + t * 128 + lane_off;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t r[32];
            tmem_ld32(tO + c * 32, r);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * w0);
            if (join) {
              uint32_t u[32];
              tmem_ld32(tO + 128 + c * 32, u);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i)
                r[i] = __float_as_uint(fmaf(__uint_as_float(u[i]), w1, __uint_as_float(r[i])));
            }
            if (c == 3) {  // all of O is in registers now: release it
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if (t == 0) mbar_arrive(bar(kBarOempty + 0));
                if (t == 1 || join) mbar_arrive(bar(kBarOempty + 1));
              }
            }
            if (kSplit) {
              float4* dst = reinterpret_cast<float4*>(prow + c * 32);
#pragma unroll
              for (int v = 0; v < 8; ++v)
                if (valid)
                  dst[v] = make_float4(__uint_as_float(r[4 * v]), __uint_as_float(r[4 * v + 1]),
                                       __uint_as_float(r[4 * v + 2]), __uint_as_float(r[4 * v + 3]));
            } else if (valid) {
              uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint4 u;
                u.x = pack_half2(__uint_as_float(r[8 * v + 0]), __uint_as_float(r[8 * v + 1]));
                u.y = pack_half2(__uint_as_float(r[8 * v + 2]), __uint_as_float(r[8 * v + 3]));
                u.z = pack_half2(__uint_as_float(r[8 * v + 4]), __uint_as_float(r[8 * v + 5]));
                u.w = pack_half2(__uint_as_float(r[8 * v + 6]), __uint_as_float(r[8 * v + 7]));
                dst[v] = u;
              }
            }
          }
        }
        ++n0;
        if (both) ++n1;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // --------------------------------------------------------------- softmax
    const int t = warp >> 2;            // query tile
    const int row = threadIdx.x & 127;  // TMEM lane == query row within the tile
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off;
    const uint32_t tO = tmem + 256 + t * 128 + lane_off;
    const float sl2 = a.scale_log2;
    // What masked tiles need waits in shared memory (two records: the next
    // item's is written while this one is worked on).  Tiles j_lo <= j < j_hi
    // hold only keys that every row of the tile sees.
    const int tok = row / a.group;
    uint32_t rec = 0, rec_next = smem_base + kOffMask + warp * 32;
    int n_next = 0, lo_next = 0, hi_next = 0, t0_next = 0;
    bool alt_next = false;
    auto next_tile = [&]() -> bool {
      Item x = {};
      do {
        if (!next_item(x)) return false;
      } while (x.count(t) == 0);
      const int first = x.P + x.q0 + (x.two ? t * a.tok : 0);  // position of the tile's first row
      if (lane == 0) st_shared4(rec_next, first, x.sink_blk, x.skip, x.vis_end);
      __syncwarp();
      n_next = x.count(t);
      t0_next = x.t0;
      alt_next = x.alt;
      // blocks from low_all on lie in every row's window, those before
      // first + 1 past no row's position
      const int low_all = max(0, first + a.tok - a.window);
      lo_next = max(0, (low_all + kBlk - 1) / kBlk - x.skip + 1) / 2;
      hi_next = max(0, (first + 1) / kBlk - x.skip) / 2;
      return true;
    };
    int sc = 0, nq = 0;
    bool ok = true;
    bool has = next_tile();
    while (ok && has) {
      const int n_t = n_next, j_lo = lo_next, j_hi = hi_next, t0 = t0_next;
      const bool alt = alt_next;
      rec = rec_next;
      rec_next ^= 16;
      float m_run = -INFINITY, l = 0.f;  // m_run: the max P is exponentiated against
      for (int i = 0; i < n_t; ++i) {
        const int j = t0 + (alt ? 2 * i + t : i);  // KV tile of the list
        if (i == n_t - 1) has = next_tile();  // while S is computed
        ok = wait(kBarS + t, sc, 30 + t);
        if (!ok) break;
        ++sc;
        tc_fence_after();
        // Two passes over S, a 64-key block at a time (rolled: code that is
        // unrolled over all 128 columns does not stay in the instruction
        // cache beside the other roles' code, and leaves no registers; 8192
        // tokens, window 1024: 188 -> 161 us).
        // Pass 1: the row maximum; masked scores go back to S.
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
        const bool masked = j < j_lo || j >= j_hi;
#pragma unroll 1
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t r[2][32];
          tmem_ld32(tS + hh * kBlk, r[0]);
          tmem_ld32(tS + hh * kBlk + 32, r[1]);
          tc_wait_ld();
          if (masked) {  // (a block past the last one starts past every row)
            const int4 m = ld_shared4(rec);
            const int pos = m.x + tok;  // this row's position
            const int e = 2 * j + hh;
            const int base = (e < m.y ? e : e + m.z) * kBlk;
            const int end = min(pos + 1, m.w) - base, low = pos - a.window + 1 - base, sk = a.sinks - base;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t keep = bits_below(end - 32 * w) & (~bits_below(low - 32 * w) | bits_below(sk - 32 * w));
              // a warp's rows are a few neighbouring tokens: most words are the same for all
              if (__all_sync(0xffffffffu, keep == 0xFFFFFFFFu)) continue;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!(keep & (1u << c))) r[w][c] = 0xFF800000u;  // -inf
              tmem_st32(tS + hh * kBlk + w * 32, r[w]);
            }
          }
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
              const auto f = [&](int i) { return __uint_as_float(r[w][c + i]); };
              mx0 = fmax3_nan(mx0, f(0), f(1));
              mx1 = fmax3_nan(mx1, f(2), f(3));
              mx2 = fmax3_nan(mx2, f(4), f(5));
              mx3 = fmax3_nan(mx3, f(6), f(7));
            }
        }
        if (masked) tc_wait_st();
        const float mx_s = fmax3_nan(fmax3_nan(mx0, mx1, mx2), mx3, mx3) * sl2;
        float alpha = 1.0f;
        float m_new = m_run;
        if (mx_s > m_run + kRescaleThreshold) {
          m_new = mx_s;
          alpha = ex2(m_run - m_new);
        }
        const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
        const uint64_t sl2x2 = f2pack(sl2, sl2);
        const uint64_t negm2 = f2pack(-m_use, -m_use);
        uint64_t rsum = f2pack(0.f, 0.f);
        // Pass 2: P.  Block hh's P lands on columns that its own S (hh = 0) or
        // block 0's S (hh = 1) no longer needs.
#pragma unroll 1
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t r[2][32];
          tmem_ld32(tS + hh * kBlk, r[0]);
          tmem_ld32(tS + hh * kBlk + 32, r[1]);
          tc_wait_ld();
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t x2 = ffma2(f2pack(__uint_as_float(r[w][2 * i]), __uint_as_float(r[w][2 * i + 1])), sl2x2, negm2);
              float p0, p1;
              if (poly_pair(i)) {
                ex2_poly2(x2, p0, p1);
              } else {
                float x0, x1;
                f2unpack(x2, x0, x1);
                p0 = ex2(x0);
                p1 = ex2(x1);
              }
              rsum = fadd2(rsum, f2pack(p0, p1));
              // f16 (2^-11 relative): both operands of the PV MMA have V's type, and
              // S leaves no TMEM columns for wider ones.  The row sum keeps f32.
              pk[i] = pack_half2(p0, p1);
            }
            asm volatile(
                "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, "
                "%10, %11, %12, %13, %14, %15, %16};" ::"r"(tS + hh * 32 + w * 16),
                "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]),
                "r"(pk[7]), "r"(pk[8]), "r"(pk[9]), "r"(pk[10]), "r"(pk[11]), "r"(pk[12]),
                "r"(pk[13]), "r"(pk[14]), "r"(pk[15])
                : "memory");
          }
        }
        float rs0, rs1;
        f2unpack(rsum, rs0, rs1);
        l = l * alpha + (rs0 + rs1);
        // a NaN or an infinite score of a visible key makes the row NaN (the
        // clamp of ex2_poly2 would lose it)
        if (!(mx_s < INFINITY)) l = NAN;
        // Rescale O_t only when some row of the warp moved its reference max
        // (PV_t(j-1) has completed: it was issued before the QK that produced
        // this S).
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarP + t));
        m_run = m_new;
      }
      if (!ok) break;
      // Row sums for the output warps.  The output warps must have taken
      // the previous item's sums (O_t of that item read out) first, so the
      // row-sum barrier never runs two phases ahead of its reader.
      if (nq > 0 && !(ok = wait(kBarOempty + t, nq - 1, 32 + t))) break;
      st_shared(smem_base + kOffL + (((nq & 1) * 2 + t) * 128 + row) * 4, __float_as_int(l));
      st_shared(smem_base + kOffL + (((2 + (nq & 1)) * 2 + t) * 128 + row) * 4, __float_as_int(m_run));
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kBarL + t));
      ++nq;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merge of the splits: a warp takes a (row, query head) of sequence blockIdx.y, a
// lane four dims.  w_s = 2^(lse_s - max) / sum, out = sum_s w_s * O_s, rounded
// once; splits without a visible key have lse = -inf; a NaN lse passes on.
__global__ void __launch_bounds__(128) prefill_window_merge_kernel(const PrefillWindowArgs a) {
  Walk<false, false> seq;
  seq.enter(a, blockIdx.y);
  if (seq.cnt == 0) return;  // no rows, or left out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)seq.S * a.hq;
  for (int64_t i = (int64_t)blockIdx.x * 4 + warp; i < rows; i += (int64_t)gridDim.x * 4) {
    const int64_t at = ((int64_t)seq.q_start * a.hq + i) * a.nsplit;
    const float lse = lane < a.nsplit ? a.part_lse[at + lane] : -INFINITY;
    const float M = warp_max(lse);
    const float w = lse == -INFINITY ? 0.f : ex2(lse - M);
    const float W = warp_sum(w);
    const float4* po = reinterpret_cast<const float4*>(a.part_o + at * 128) + lane;
    const unsigned some = __ballot_sync(0xffffffffu, lse != -INFINITY);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.nsplit; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      if (some >> s & 1) fma4(acc, ws, po[(int64_t)s * 32]);  // the others were not written
    }
    const int64_t row = i / a.hq;
    store_row4(a.out + (seq.q_start + row) * a.q_row_stride + (i - row * a.hq) * 128 + 4 * lane, acc,
               W != 0.f ? 1.f / W : 0.f);
  }
}

template <bool kPaged, bool kShort>
constexpr auto kernel_of(bool split) {
  return split ? prefill_window_kernel<kPaged, kShort, true> : prefill_window_kernel<kPaged, kShort, false>;
}

}  // namespace

cudaError_t prefill_window_set_attributes() {
  for (auto k : {kernel_of<false, false>(false), kernel_of<true, false>(false), kernel_of<false, true>(false),
                 kernel_of<true, true>(false), kernel_of<false, false>(true), kernel_of<true, false>(true),
                 kernel_of<false, true>(true), kernel_of<true, true>(true)}) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_prefill_window(const PrefillWindowArgs& a, int32_t max_q_len, int num_sms,
                                  const CUtensorMap& tm_q, const CUtensorMap& tm_k,
                                  const CUtensorMap& tm_v, cudaStream_t s) {
  const int64_t items =
      (int64_t)((max_q_len + 2 * (int64_t)a.tok - 1) / (2 * a.tok)) * a.hkv * a.batch * a.nsplit;
  if (items == 0) return cudaSuccess;
  const int grid = (int)(items < num_sms ? items : num_sms);
  // Drafts of 5 tokens x 4 heads, 32 sequences, window 1024: 50 us with one
  // chain a tile, 42 with two.  Carrying that code too, long prompts took 158
  // instead of 147 us (8192 tokens) and 293 instead of 249 us (window 64).
  const bool brief = max_q_len <= a.tok, split = a.nsplit > 1;
  auto k = a.page_table ? (brief ? kernel_of<true, true>(split) : kernel_of<true, false>(split))
                        : (brief ? kernel_of<false, true>(split) : kernel_of<false, false>(split));
  k<<<grid, kThreads, kSmemBytes, s>>>(tm_q, tm_k, tm_v, a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !split) return e;
  const int64_t blocks = std::min<int64_t>(((int64_t)max_q_len * a.hq + 3) / 4,
                                           std::max(1, 16 * num_sms / a.batch));
  prefill_window_merge_kernel<<<dim3((unsigned)blocks, (unsigned)a.batch), 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace grout
