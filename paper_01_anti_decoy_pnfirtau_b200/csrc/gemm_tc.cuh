// A persistent tcgen05 GEMM with a pluggable epilogue, the core of the gated
// feed-forward, streamed cross-entropy and 8-bit-checkpoint kernels:
//
//   acc[m, n] = sum_k A[m, k] B[n, k]     (bf16 or fp16 operands, fp32 in TMEM)
//
// Two CTAs of a cluster (one per SM) share a 256 x 256 output tile: each holds 128 rows
// of A and 128 rows of B in shared memory, and the even CTA issues the MMAs of both
// (cta_group::2, M = 256, N = 256, K = 16), so an operand byte brought into an SM feeds
// twice the products of a one-CTA tile. Each CTA has its 128 rows of the accumulator in
// its own TMEM, twice (2 x 256 columns). The pair walks work items; an item is one tile
// (or, for epilogues that carry state along a row, a strip of tiles), optionally one of
// several splits of K. Warp 0 loads 64-deep stages of A and B by TMA into a ring, one
// lane of the even CTA's warp 1 issues the MMAs, and 8 or 16 more run the epilogue of the
// other accumulator, so a tile's epilogue overlaps the next tile's MMAs. Either operand
// may be K-major (rows of K) or MN-major (K rows of M or N), so no caller transposes
// anything. Rows, columns and K past the end are zero-filled by TMA.
//
// Bound by the tensor core from K of about 1024 on, and by the power limit in long runs. Measured (B200,
// bf16, single calls): the gated product 16384 x 2048 x 2048 178 us (1.55 PFLOP/s), 16384 x 512 x 2048
// 55 us (1.25), cross entropy's forward 8192 x 50021 x 512 291 us (1.44), 16352 x 33278 x 256 240 us (1.16;
// whole calls: the rows' compaction and the join of the strips take 25 us of that).
#pragma once

#include <string.h>

#include <algorithm>
#include <atomic>

#include "flash.cuh"
#include "sm100_ptx.cuh"

namespace pnft {
namespace tc {

using namespace sm100;

constexpr int BM = 128;       // rows per CTA (TMEM lanes)
constexpr int PM = 2 * BM;    // rows per pair
constexpr int BN = 256, BK = 64;
constexpr int HALF_BYTES = BM * BK * 2;    // a CTA's A rows, or its half of B, of one stage
constexpr int STAGE_BYTES = 2 * HALF_BYTES;
constexpr int GROUP_BYTES = 64 * BK * 2;   // MN-major: 64 columns x 64 K rows
constexpr int STAGE_MAX = 225 * 1024;      // shared memory for the ring and the epilogue's buffers

// ------------------------------------------------------------------ dependent launches
// The kernels of one call follow each other on a stream. Each lets the next be launched at
// once and waits itself, before it touches memory, until the one before has completed: the
// launch, the barriers and the TMEM allocation of a kernel then pass while the one before
// still runs. Every thread of a kernel calls it. So what such a kernel reads may have been
// written while it was resident: its loads are ordinary ones (never the read-only path, which
// is for data that is constant as long as the kernel lives, and no restrict pointers to const,
// which let the compiler take that path or move a load above the wait).
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class K, class... A>
inline void launch_dependent(K* kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid, c.blockDim = dim3((unsigned)threads), c.dynamicSmemBytes = smem, c.stream = st;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &attr, c.numAttrs = 1;
  (void)cudaLaunchKernelEx(&c, kernel, args...);  // its error is the pending one that check_launch reads
}

// ------------------------------------------------------------------ PTX of the pair
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Address of the same shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Arrival on a barrier of either CTA that publishes no memory (TMEM reads are ordered by
// tcgen05.wait and tcgen05.fence), so it is relaxed: a release at cluster scope took a
// fifth of the epilogue's time.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Load into this CTA's shared memory, completing on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kSw128DescHi)
      : "memory");
}
// Arrive on `bar` in both CTAs once every MMA issued so far completes.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}

// Which tiles there are and in which order. Strips: an item is tiles_per_strip column tiles
// of one row tile and one split of K; items are taken group_m row tiles at a time, the row
// tile running fastest, so the pairs in flight share both operands in L2. Runs (`runs`): the
// tiles, row tile by row tile, are dealt to the pairs in equal contiguous runs, and an item
// is a run's part of one row tile: the pairs end together, and a pair finds its rows of A in L2 for many tiles.
// For a B that stays in L2 as a whole. strips = 0: strips as fit the number of row tiles (the
// rows that count, known on the device alone), see auto_strips.
struct Sched {
  int tiles_m;          // 256-row tiles (upper bound when live is given)
  int strips;           // items along N
  int tiles_n;          // column tiles
  int tiles_per_strip;  // column tiles per item
  int kb;               // 64-deep K blocks (upper bound when live_k)
  int splits;           // splits of K
  int whole;            // the first tiles, which are not split (strips of one tile)
  int chunk;            // K blocks that one accumulator takes before the epilogue collects it
  int group_m;
  int runs;
  int seg_kb;           // K blocks of the first pair of maps; the rest use the second
  const int32_t* live;  // device: rows that count (NULL: all)
  int live_m, live_k;   // the rows that count bound M / K
};

// First tile of pair p's run of `total` tiles over `pairs` pairs, and the pair of tile x.
__host__ __device__ inline int64_t run_begin(int64_t total, int p, int pairs) { return total * p / pairs; }
__host__ __device__ inline int run_owner(int64_t total, int64_t x, int pairs) {
  return (int)(((x + 1) * pairs + total - 1) / total) - 1;
}

// Strips per row tile: those of one to four equal rounds of items over the pairs, the one
// with the fewest tiles in a row, counting a third of a tile for an item's start and end (which
// decides between equal counts only: cross entropy's forward with no such share, a third and a
// whole tile, B200: 300 x 50021 x 512 47, 45, 47 us; 4096 x 131072 x 512 383 each).
__host__ __device__ inline int auto_strips(int tiles_m, int tiles_n, int pairs) {
  int best = 1;
  float least = 3e38f;
  for (int r = 0; r <= 4 && tiles_m > 0; ++r) {
    int strips = r * pairs / tiles_m;
    strips = strips < 1 ? 1 : strips > tiles_n ? tiles_n : strips;
    const int per = (tiles_n + strips - 1) / strips;
    strips = (tiles_n + per - 1) / per;
    const float cost = (float)((tiles_m * strips + pairs - 1) / pairs) * ((float)per + 0.333f);
    if (cost < least) least = cost, best = strips;
  }
  return best;
}

struct Args {
  CUtensorMap ta[2], tb[2];
  Sched s;
  uint32_t idesc;
  int32_t* status;
};

struct Item {
  int mt, nt0, ntn, split, kb0, kbn;
  int row0;  // first row of this CTA
  int slot;  // strip, or place of the run among those of its row tile
  int part;  // place among the split items behind whole tiles, or -1
};

// Row tile and strip of item r: group_m row tiles at a time, the row tile running fastest.
__host__ __device__ inline void item_order(int r, int tiles_m, int strips, int group_m, int* mt, int* strip) {
  const int per = group_m * strips, g = r / per;
  r -= g * per;
  const int gm = tiles_m - g * group_m < group_m ? tiles_m - g * group_m : group_m;
  *mt = g * group_m + r % gm;
  *strip = r / gm;
}

struct Walk {
  int tiles_m, kb, slots, pairs;
  int strips, per_strip, group_m;
  int64_t total;  // items, or tiles in runs
  __device__ Walk(const Sched& s, int launched) {
    tiles_m = s.tiles_m, kb = s.kb;
    if (s.live) {
      const int n = *s.live;
      if (s.live_m) tiles_m = (n + PM - 1) / PM;
      if (s.live_k) kb = (n + BK - 1) / BK;
    }
    strips = s.strips, per_strip = s.tiles_per_strip, group_m = s.group_m;
    if (strips == 0) {
      strips = auto_strips(tiles_m, s.tiles_n, launched);
      per_strip = (s.tiles_n + strips - 1) / strips;
      group_m = max(tiles_m, 1);
    }
    total = s.runs ? (int64_t)tiles_m * s.tiles_n : s.whole + (int64_t)(tiles_m * strips - s.whole) * s.splits;
    pairs = s.runs ? run_pairs(total, launched) : launched;
    slots = s.runs ? run_slots(tiles_m, pairs) : strips;
  }
  // Pairs that get a run: none is empty, also where fewer rows count than the launch was sized for.
  __host__ __device__ static int run_pairs(int64_t total, int launched) { return (int)(total < launched ? total : launched); }
  // Runs that a row tile may lie in.
  __host__ __device__ static int run_slots(int tiles_m, int pairs) {
    return tiles_m > 0 ? (pairs + tiles_m - 1) / tiles_m + 1 : 0;
  }
  // The item that starts at i of `end`.
  __device__ Item at(const Sched& s, int64_t i, int64_t end, int rank, int pair) const {
    Item it;
    if (s.runs) {
      it.split = 0, it.kb0 = 0, it.kbn = kb, it.part = -1;
      it.mt = (int)(i / s.tiles_n);
      const int64_t first = (int64_t)it.mt * s.tiles_n;
      it.nt0 = (int)(i - first);
      it.ntn = (int)min((int64_t)s.tiles_n, end - first) - it.nt0;
      it.slot = pair - run_owner(total, first, pairs);
    } else {
      const int per_split = tiles_m * strips - s.whole, j = (int)i - s.whole;
      const bool split = j >= 0;
      it.split = split ? j / per_split : 0;
      it.part = split && s.whole > 0 ? j : -1;
      item_order(split ? s.whole + j - it.split * per_split : (int)i, tiles_m, strips, group_m, &it.mt, &it.slot);
      it.nt0 = it.slot * per_strip;
      it.ntn = min(per_strip, s.tiles_n - it.nt0);
      // whole K blocks spread evenly over the splits
      const int splits = split ? s.splits : 1;
      it.kb0 = (int)((int64_t)kb * it.split / splits);
      it.kbn = (int)((int64_t)kb * (it.split + 1) / splits) - it.kb0;
    }
    it.row0 = it.mt * PM + rank * BM;
    return it;
  }
};

// The accumulators in the order in which they are filled: item by item, tile by tile,
// and within a tile one per `chunk` K blocks (at least one, empty where K is).
struct Steps {
  const Walk& walk;
  const Sched& s;
  int64_t i, end;
  int pair, rank, nt, kb;
  Item it;
  __device__ Steps(const Walk& w, const Sched& s_, int pair_, int rank_) : walk(w), s(s_), pair(pair_), rank(rank_) {
    const bool run = s.runs && pair < w.pairs;
    i = run ? run_begin(w.total, pair, w.pairs) : pair;
    end = run ? run_begin(w.total, pair + 1, w.pairs) : s.runs ? 0 : w.total;
    load();
  }
  __device__ void load() {
    if (i < end) it = walk.at(s, i, end, rank, pair), nt = it.nt0, kb = it.kb0;
  }
  __device__ bool valid() const { return i < end; }
  __device__ int kb_end() const { return min(kb + s.chunk, it.kb0 + it.kbn); }
  __device__ bool tile_first() const { return kb == it.kb0; }
  __device__ bool tile_last() const { return kb + s.chunk >= it.kb0 + it.kbn; }
  __device__ bool item_first() const { return nt == it.nt0 && tile_first(); }
  __device__ bool item_last() const { return nt == it.nt0 + it.ntn - 1 && tile_last(); }
  __device__ void next() {
    if (!tile_last()) {
      kb += s.chunk;
      return;
    }
    kb = it.kb0;
    if (++nt == it.nt0 + it.ntn) {
      i += s.runs ? it.ntn : walk.pairs;
      load();
    }
  }
};

// What an epilogue warp has: its group (ping-pong epilogues have two, which take the
// accumulators in turn), its TMEM lane quadrant, its slice of the columns (of 2 or 4), its
// boxes in shared memory and a barrier for loads into them.
struct EpiWarp {
  int quad, group, slice, lane;
  uint32_t smem, bar;
  __device__ int row() const { return 32 * quad + lane; }
};

// Epi: WARPS (8, or 16 where the arithmetic per element is what takes the time: a warp's
// chain of TMEM load, exponentials and stores has long latencies, and 16 warps of at most 96
// registers hide them twice as well), PING_PONG (the warps form two groups, one per
// accumulator: while one group is at its loads, the other keeps the arithmetic pipes busy,
// where all warps in step would use one after the other), BOXES of BOX_BYTES per warp;
// prepare(steps) and end(steps) for every accumulator, tile(steps, acc, release) between them for those of the warp's group
// (acc: its TMEM address with the warp's lanes; release() hands it back once its last
// column is in registers), done() at the end.
// DUAL_B: columns 0-127 of a tile come from tb[0] and 128-255 from tb[1], both at row
// 128 * nt.
template <class Epi>
constexpr int box_bytes() {
  return Epi::WARPS * Epi::BOXES * Epi::BOX_BYTES;
}
template <class Epi>
constexpr int stages() {
  return (STAGE_MAX - box_bytes<Epi>()) / STAGE_BYTES;
}
constexpr int SMEM = STAGE_MAX + 1024;

template <bool A_MN, bool B_MN, bool DUAL_B, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(32 * (2 + Epi::WARPS), 1)
    gemm_kernel(const __grid_constant__ Args p, const __grid_constant__ typename Epi::Params ep) {
  constexpr int EPI_WARPS = Epi::WARPS, STAGES = stages<Epi>();
  extern __shared__ __align__(1024) uint8_t raw[];
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  // full, empty, acc full x2, acc empty x2, done, warps
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 5 + EPI_WARPS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  launch_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t b0 = smem_u32(bars);
  auto full = [&](int s) { return b0 + 8u * s; };
  auto empty = [&](int s) { return b0 + 8u * (STAGES + s); };
  auto acc_full = [&](int s) { return b0 + 8u * (2 * STAGES + s); };
  auto acc_empty = [&](int s) { return b0 + 8u * (2 * STAGES + 2 + s); };
  const uint32_t done = b0 + 8u * (2 * STAGES + 4);
  auto warp_bar = [&](int w) { return b0 + 8u * (2 * STAGES + 5 + w); };
  const Abort ab{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 1);   // the even CTA's: its producer's arrival, and the bytes of both CTAs
      mbar_init(empty(s), 1);  // the MMAs that read the stage, told to both CTAs
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full(s), 1);
      mbar_init(acc_empty(s), Epi::PING_PONG ? EPI_WARPS : 2 * EPI_WARPS);  // the even CTA's: the epilogue warps of both
    }
    mbar_init(done, 1);
    for (int w = 0; w < EPI_WARPS; ++w) mbar_init(warp_bar(w), 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&tmem_slot), 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers are ready for this one's arrivals
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  wait_previous();
  const Walk walk(p.s, pairs);

  if (warp == 0) {
    // -------------------------------------------------------------- TMA producer
    if (lane == 0) {
      int st = 0, ph = 1, issued = 0;
      bool ok = true;
      for (Steps q(walk, p.s, pair, rank); ok && q.valid(); q.next()) {
        for (int kb = q.kb; kb < q.kb_end(); ++kb) {
          if (!mbar_wait(empty(st), ph, ab)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(full(st), 2 * STAGE_BYTES);
          const uint32_t bar = map_rank(full(st), 0);
          const int seg = kb >= p.s.seg_kb;
          const int k = (kb - (seg ? p.s.seg_kb : 0)) * BK;
          const uint32_t sa = ring + (uint32_t)st * STAGE_BYTES, sB = sa + HALF_BYTES;
          if (A_MN) {
#pragma unroll
            for (int g = 0; g < BM / 64; ++g) tma_load_pair(sa + g * GROUP_BYTES, &p.ta[seg], bar, q.it.row0 + 64 * g, k);
          } else {
            tma_load_pair(sa, &p.ta[seg], bar, k, q.it.row0);
          }
          if (B_MN) {
#pragma unroll
            for (int g = 0; g < BM / 64; ++g)
              tma_load_pair(sB + g * GROUP_BYTES, &p.tb[seg], bar, q.nt * BN + rank * (BN / 2) + 64 * g, k);
          } else if (DUAL_B) {
            tma_load_pair(sB, &p.tb[rank], bar, k, q.nt * (BN / 2));
          } else {
            tma_load_pair(sB, &p.tb[seg], bar, k, q.nt * BN + rank * (BN / 2));
          }
          ++issued;
          if (++st == STAGES) st = 0, ph ^= 1;
        }
      }
      // Never leave a copy in flight into shared memory: the even CTA's barriers count the
      // copies of both, and the odd CTA stays until the even one comes to the final barrier.
      if (rank == 0) {
        for (int n = 0; n < min(issued, STAGES); ++n) {
          const int last = issued - 1 - n;
          drain_wait(full(last % STAGES), (last / STAGES) & 1);
        }
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer (even CTA)
    if (rank == 0 && lane == 0) {
      int st = 0, ph = 0, t = 0;
      bool ok = true;
      for (Steps q(walk, p.s, pair, rank); ok && q.valid(); q.next(), ++t) {
        if (!mbar_wait(acc_empty(t & 1), ((t >> 1) & 1) ^ 1, ab)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(t & 1) * BN;
        for (int kb = q.kb; kb < q.kb_end(); ++kb) {
          if (!mbar_wait(full(st), ph, ab)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t slot = ring + (uint32_t)st * STAGE_BYTES;
          const uint32_t da = sw128_desc(slot, A_MN ? GROUP_BYTES : 0);
          const uint32_t db = sw128_desc(slot + HALF_BYTES, B_MN ? GROUP_BYTES : 0);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)  // 16 K: 32 bytes of a K-major row, 16 rows (2048 bytes) MN-major
            mma_pair(d, da + kk * (A_MN ? 128 : 2), db + kk * (B_MN ? 128 : 2), p.idesc, kb > q.kb || kk > 0);
          commit_pair(empty(st));
          if (++st == STAGES) st = 0, ph ^= 1;
        }
        if (ok) commit_pair(acc_full(t & 1));
      }
      commit_pair(done);
      drain_wait(done, 0);  // no MMA may still be writing TMEM, or reading either CTA's tiles, at teardown
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const int part = (warp - 2) >> 2;
    const EpiWarp w{warp & 3, Epi::PING_PONG ? part & 1 : 0, Epi::PING_PONG ? part >> 1 : part, lane,
                    ring + (uint32_t)(STAGES * STAGE_BYTES + (warp - 2) * Epi::BOXES * Epi::BOX_BYTES), warp_bar(warp - 2)};
    Epi epi(ep, w, ab);
    int t = 0;
    for (Steps q(walk, p.s, pair, rank); q.valid(); q.next(), ++t) {
      epi.prepare(q);
      if (Epi::PING_PONG && (t & 1) != w.group) {
        epi.end(q);
        continue;
      }
      if (!warp_wait(acc_full(t & 1), (t >> 1) & 1, ab)) break;
      tc_fence_after();
      const uint32_t release = map_rank(acc_empty(t & 1), 0);
      epi.tile(q, tmem + (uint32_t)(t & 1) * BN + ((uint32_t)(32 * w.quad) << 16), [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(release);
      });
      epi.end(q);
    }
    epi.done();
  }
  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still signal it or read its tiles
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN);
  }
}

// ------------------------------------------------------------------ rows of 32 values
// The element types an epilogue reads and writes (PNFT_DTYPE_*; uniform over a launch).
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t v, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ void store16(void* dst, float v, bool bf16) {
  if (bf16)
    *static_cast<__nv_bfloat16*>(dst) = __float2bfloat16_rn(v);
  else
    *static_cast<__half*>(dst) = __float2half_rn(v);
}
__device__ __forceinline__ float load16(const void* src, bool bf16) {
  return bf16 ? __bfloat162float(*static_cast<const __nv_bfloat16*>(src)) : __half2float(*static_cast<const __half*>(src));
}

// N consecutive values of one row to 16-bit storage; `n` of them exist, `vec`: the
// address is 16-byte aligned.
template <int N>
__device__ __forceinline__ void store_row16(uint16_t* dst, const float (&v)[N], int n, bool vec, bool bf16) {
  if (vec && n >= N) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      *reinterpret_cast<uint4*>(dst + i) = make_uint4(pack2(v[i], v[i + 1], bf16), pack2(v[i + 2], v[i + 3], bf16),
                                                      pack2(v[i + 4], v[i + 5], bf16), pack2(v[i + 6], v[i + 7], bf16));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) store16(dst + i, v[i], bf16);
  }
}
template <int N>
__device__ __forceinline__ void load_row16(const uint16_t* src, float (&v)[N], int n, bool vec, bool bf16) {
  if (vec && n >= N) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(src + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2(w[k], bf16);
        v[i + 2 * k] = f.x, v[i + 2 * k + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? load16(src + i, bf16) : 0.f;
  }
}
template <int N>
__device__ __forceinline__ void store_row32(float* dst, const float (&v)[N], int n, bool vec) {
  if (vec && n >= N) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) dst[i] = v[i];
  }
}

// 32 columns of an accumulator; `empty`: no K block contributed (it stands for 0).
__device__ __forceinline__ void acc_load32(uint32_t addr, bool empty, float (&v)[32]) {
  uint32_t r[32];
  tmem_load32(addr, r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = empty ? 0.f : __uint_as_float(r[i]);
}

// ------------------------------------------------------------------ boxes
// A box is 32 rows of RB = 128 (or 64) bytes in shared memory, swizzled (16-byte chunk c of
// row r at chunk c ^ (r & 7), or c ^ (r / 2 & 3)): a lane writes or reads its own row without bank conflicts, and
// TMA moves the box, clipped to the matrix. Boxes of a warp are used in turn; a box is free
// again once the store out of it has read it.
template <int N, int RB = 128>
struct Boxes {
  EpiWarp w;
  int at;
  __device__ explicit Boxes(const EpiWarp& w_) : w(w_), at(0) {}
  __device__ __forceinline__ uint32_t box(int i) const { return w.smem + (uint32_t)(i * 32 * RB); }
  __device__ __forceinline__ static uint32_t chunk_at(uint32_t b, int row, int chunk) {
    return b + (uint32_t)(RB * row) + 16u * (chunk ^ (RB == 128 ? row & 7 : (row >> 1) & 3));
  }
  // the next box, free to write (stores of the N - 1 others may be in flight)
  __device__ __forceinline__ uint32_t take() {
    if (w.lane == 0) bulk_wait_read<N - 1>();
    __syncwarp();
    const uint32_t b = box(at);
    at = at + 1 == N ? 0 : at + 1;
    return b;
  }
  // all N boxes, free to write
  __device__ __forceinline__ void take_all(uint32_t (&b)[N]) {
    if (w.lane == 0) bulk_wait_read<0>();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = box(i);
    at = 0;
  }
  __device__ __forceinline__ void put(uint32_t b, int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t u) const {
    const uint32_t a = chunk_at(b, w.lane, chunk);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(u) : "memory");
  }
  __device__ __forceinline__ uint4 get(uint32_t b, int chunk) const {
    const uint32_t a = chunk_at(b, w.lane, chunk);
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
  }
  // W columns as 16-bit values from column `c` of the box
  template <int W>
  __device__ __forceinline__ void put16(uint32_t b, int c, const float (&v)[W], bool bf16) const {
#pragma unroll
    for (int i = 0; i < W; i += 8)
      put(b, (c + i) / 8, pack2(v[i], v[i + 1], bf16), pack2(v[i + 2], v[i + 3], bf16), pack2(v[i + 4], v[i + 5], bf16),
          pack2(v[i + 6], v[i + 7], bf16));
  }
  template <int W>
  __device__ __forceinline__ void get16(uint32_t b, int c, float (&v)[W], bool bf16) const {
#pragma unroll
    for (int i = 0; i < W; i += 8) {
      const uint4 u = get(b, (c + i) / 8);
      const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2(q[k], bf16);
        v[i + 2 * k] = f.x, v[i + 2 * k + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void put32(uint32_t b, const float (&v)[32]) const {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      put(b, i / 4, __float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]));
  }
  // box -> matrix at column x, row y, slice z
  __device__ __forceinline__ void store(uint32_t b, const CUtensorMap* map, int x, int y, int z, bool add = false) const {
    fence_proxy_async_smem();
    __syncwarp();
    if (w.lane == 0) {
      if (add)
        tma_add_3d(map, b, x, y, z);
      else
        tma_store_3d(map, b, x, y, z);
      bulk_commit();
    }
  }
  // The same for rows that TMA cannot address (not 16-byte aligned): `rows` rows of `cols`
  // elements of SIZE bytes, whole warps along a row.
  template <int SIZE>
  __device__ __forceinline__ void store_plain(uint32_t b, void* dst, int64_t ld, int rows, int cols) const {
    __syncwarp();
    constexpr int PER = RB / SIZE;  // elements per row of a box
    for (int r = 0; r < min(rows, 32); ++r) {
#pragma unroll
      for (int k = 0; k < PER / 32; ++k) {
        const int c = 32 * k + w.lane, byte = c * SIZE;
        const uint32_t a = chunk_at(b, r, byte >> 4) + (byte & 15);
        if (c >= cols) continue;
        if (SIZE == 2) {
          uint16_t v;
          asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
          static_cast<uint16_t*>(dst)[r * ld + c] = v;
        } else {
          uint32_t v;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
          static_cast<uint32_t*>(dst)[r * ld + c] = v;
        }
      }
    }
    __syncwarp();
  }
  // Every store has been performed (before the CTA may leave).
  __device__ void finish() const {
    if (w.lane == 0) bulk_wait_all();
  }
};

// A matrix that an epilogue writes: by TMA where its rows are 16-byte aligned.
struct Out {
  CUtensorMap map;  // {columns, rows, slices}, boxes of 32 rows
  void* base;
  int64_t ld;
  int rows, cols;
  int tma;
};

// ------------------------------------------------------------------ plain epilogue
// C = alpha * acc as fp32, bf16 or fp16: the rows of two matrices one after the other
// (row_split, a multiple of 128, rows apart), or the fp32 partials of the splits (slices),
// or added to an fp32 C; of split tiles behind whole ones the fp32 partials, tile by tile. PROMOTE: an item's accumulators (chunks of K) are collected in
// fp32 registers: the tensor core's own sum over K loses about 2^-24 per 16 products,
// which an fp32 C would show.
template <bool PROMOTE>
struct StoreEpi {
  static constexpr int WARPS = 8, BOXES = 2, BOX_BYTES = 4096;
  static constexpr bool PING_PONG = false;
  struct Params {
    Out c[2];
    Out part;  // partials of the split tiles behind whole ones: a slice of 256 x 256 each
    int row_split;
    const float* alpha;  // device scalar (NULL: 1)
    int dtype;           // of C
    int add;             // C (fp32) += acc
  };
  const Params& p;
  EpiWarp w;
  Boxes<BOXES> boxes;
  float alpha;
  float sum[PROMOTE ? BN / 2 : 1];
  __device__ StoreEpi(const Params& p_, const EpiWarp& w_, const Abort&) : p(p_), w(w_), boxes(w) {
    alpha = p.alpha ? *p.alpha : 1.f;
#pragma unroll
    for (float& v : sum) v = 0.f;
  }
  __device__ void prepare(const Steps&) {}
  __device__ void end(const Steps&) {}
  __device__ void done() { boxes.finish(); }
  __device__ __forceinline__ void out32(const Steps& q, int c, float (&v)[32], uint32_t& box) {
    if (q.it.part >= 0) {
      const uint32_t b = boxes.take();
      boxes.put32(b, v);
      boxes.store(b, &p.part.map, c, q.it.row0 % PM + 32 * w.quad, q.it.part);
      return;
    }
    int row = q.it.row0 + 32 * w.quad;
    const int part = row >= p.row_split;
    if (part) row -= p.row_split;
    const Out& o = p.c[part];
    const int col = q.nt * BN + c, rows = o.rows - row;
    if (rows <= 0) return;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= alpha;
    if (PROMOTE || p.dtype == PNFT_DTYPE_F32) {
      if (o.cols - col <= 0) return;
      const uint32_t b = boxes.take();
      boxes.put32(b, v);
      if (o.tma)
        boxes.store(b, &o.map, col, row, q.it.split, p.add);
      else
        boxes.template store_plain<4>(b, static_cast<float*>(o.base) + (int64_t)row * o.ld + col, o.ld, rows, o.cols - col);
    } else {
      const int h = (c >> 5) & 1;  // a box takes 64 columns: two calls
      if (o.cols - (col - 32 * h) <= 0) return;
      if (h == 0) box = boxes.take();
      boxes.put16(box, 32 * h, v, p.dtype == PNFT_DTYPE_BF16);
      if (h == 0) return;
      if (o.tma)
        boxes.store(box, &o.map, col - 32, row, 0);
      else
        boxes.template store_plain<2>(box, static_cast<uint16_t*>(o.base) + (int64_t)row * o.ld + col - 32, o.ld, rows,
                                      o.cols - col + 32);
    }
  }
  template <class Release>
  __device__ __forceinline__ void tile(const Steps& q, uint32_t acc, Release release) {
    const int c0 = w.slice * (BN / 2);
    const bool empty = q.it.kbn == 0;
    uint32_t box = 0;
    if (PROMOTE) {
#pragma unroll
      for (int c = 0; c < BN / 2; c += 16) {  // 16 at a time: the sums take 128 registers
        uint32_t r[16];
        tmem_load16(acc + c0 + c, r);
        if (c + 16 == BN / 2) release();
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[c + i] += empty ? 0.f : __uint_as_float(r[i]);
      }
      if (!q.tile_last()) return;
#pragma unroll
      for (int c = 0; c < BN / 2; c += 32) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = sum[c + i], sum[c + i] = 0.f;
        out32(q, c0 + c, v, box);
      }
    } else {
#pragma unroll 1
      for (int c = 0; c < BN / 2; c += 32) {
        float v[32];
        acc_load32(acc + c0 + c, empty, v);
        if (c + 32 == BN / 2) release();
        out32(q, c0 + c, v, box);
      }
    }
  }
};

// ------------------------------------------------------------------ host side
int current_device();
int sm_count();  // of the current device
// Splits of K for an output of `tiles` tiles: about `rounds` work items per pair of SMs, at
// least 8 K blocks (512 of K) each, since shorter ones cost more in partial sums than
// they gain.
int plan_splits(int64_t tiles, int64_t kb, int rounds = 1);
// Pairs of SMs that a launch of `items` items takes.
inline int pairs_of(int64_t items) { return (int)std::min<int64_t>(items, sm_count() / 2); }
inline int64_t tiles_of(int64_t m, int64_t n) { return ((m + PM - 1) / PM) * ((n + BN - 1) / BN); }

// Sums the splits' fp32 partials [splits][rows_total][ldp] in split order (bitwise
// reproducible), times alpha, into C (two parts as StoreEpi) or onto an fp32 C.
struct SumArgs {
  void* c[2];
  int64_t ldc;
  int row_split, rows, cols;
  const float* alpha;
  int dtype, add, vec;
};
// The weight-gradient product behind pnft_weight_grad, its arguments checked.
int weight_grad(const char* what, const void* dy, int64_t lddy, const void* x, int64_t ldx, void* c0, void* c1, int64_t ldc,
                int64_t row_split, int64_t rows, int c_dtype, void* workspace, int64_t K, int64_t M, int64_t N, int dtype,
                int32_t* status, cudaStream_t st);
int sum_splits(const float* part, int64_t ldp, int64_t split_stride, int splits, const SumArgs& out, int rows_total,
               cudaStream_t st);

// How a product's tiles are dealt: in whole rounds over the pairs, and the rest of them (all,
// if there are fewer than pairs) in `splits` splits of K each, so that no round is half empty.
struct Plan {
  int splits;
  int whole;  // tiles that are not split
};
Plan plan_product(int64_t tiles, int64_t kb);
// Bytes of partial sums of an M x N product.
size_t product_workspace(int64_t M, int64_t N, int64_t kb);
// The same for the tiles from `s.whole` on, whose partials lie tile by tile.
int sum_tail(const float* part, const Sched& s, const SumArgs& out, cudaStream_t st);

inline bool rows16(const void* p, int64_t ld, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0;
}
inline int dtype_size(int dtype) { return dtype == PNFT_DTYPE_F32 ? 4 : 2; }

inline int make_out(Out* o, void* base, int dtype, int64_t cols, int64_t rows, int64_t ld, int64_t slices = 1,
                    int64_t slice_stride = 0, int row_bytes = 128) {
  memset(o, 0, sizeof(*o));
  if (!base) return PNFT_OK;  // no rows: nothing is written
  o->base = base, o->ld = ld, o->rows = (int)rows, o->cols = (int)cols;
  o->tma = rows16(base, ld, dtype_size(dtype)) && ld < ((int64_t)1 << 37);
  return o->tma ? tma_map_out(&o->map, base, dtype_size(dtype), cols, rows, ld, slices, slice_stride, 32, row_bytes) : PNFT_OK;
}

// K-major operand: `rows` rows of K elements; MN-major operand: K rows of `cols`
// elements. Both take the row stride in elements (a multiple of 8, 16-byte base).
inline int map_kmajor(CUtensorMap* m, const void* base, int64_t k, int64_t rows, int64_t ld) {
  return tma_map_rows(m, base, k, rows, ld, BM);
}
inline int map_mnmajor(CUtensorMap* m, const void* base, int64_t cols, int64_t k, int64_t ld) {
  return tma_map_rows(m, base, cols, k, ld, BK);
}

inline uint32_t idesc(int dtype, bool a_mn, bool b_mn) {
  return idesc_f16(PM, BN, dtype == PNFT_DTYPE_BF16 ? 1 : 0, a_mn, b_mn);
}

// Strips go eight row tiles at a time. Measured (B200, bf16) with 4, 8 and 16: gated forward 8192 x 2048 x 8192
// 358, 350, 346 us and its backward 842, 850, 858; cross entropy's backward 4096 x 128000 x 2048 4.81, 4.75, 4.61 ms.
inline Sched plain_sched(int64_t m, int64_t n, int64_t kb, int splits) {
  Sched s;
  memset(&s, 0, sizeof(s));
  s.tiles_m = (int)((m + PM - 1) / PM);
  s.tiles_n = s.strips = (int)((n + BN - 1) / BN);
  s.tiles_per_strip = 1;
  s.kb = s.seg_kb = s.chunk = (int)std::max<int64_t>(kb, 1);
  s.splits = splits;
  s.group_m = 8;
  return s;
}

// Runs where all of B (n rows of k elements) and the rows of A that the pairs are at (256 each) stay in
// L2 beside what streams through it. Measured (B200, bf16), runs against strips in us, by the sum of
// both. Gated product: 16384 x 512 x 2048 (21 MB) 55, 65; x 1024 x 4096 (50 MB) 181, 194; x 1536 x 4096
// (75 MB) 275, 271; x 2048 x 1024 (75 MB) 90, 93; x 2048 x 2048 (84 MB) 190, 177; x 2048 x 6000 (116 MB)
// 713, 535. Cross entropy's forward: 8192 x 50021 x 512 (60 MB) 291, 303; 8192 x 10000 x 2048 (75 MB)
// 252, 270; 8192 x 50021 x 1024 (119 MB) 633, 562.
inline void runs_if_resident(Sched* s, int64_t n, int64_t k) {
  const int64_t rows = (int64_t)PM * std::min(s->tiles_m, sm_count() / 2);
  s->runs = (n + rows) * k * 2 <= ((int64_t)76 << 20);
}

template <bool A_MN, bool B_MN, bool DUAL_B, class Epi>
int launch(const char* what, const Args& a, const typename Epi::Params& ep, cudaStream_t st) {
  const int64_t tiles = (int64_t)a.s.tiles_m * (a.s.runs || !a.s.strips ? a.s.tiles_n : a.s.strips);
  const int64_t items = a.s.whole + (tiles - a.s.whole) * a.s.splits;
  if (items <= 0) return PNFT_OK;
  if (items > (1 << 30)) return fail(PNFT_EUNSUPPORTED, "%s: too many tiles", what);
  auto* k = gemm_kernel<A_MN, B_MN, DUAL_B, Epi>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel has its shared memory
  const uint64_t bit = 1ull << (current_device() & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return check_launch(what, 0);
    ready.fetch_or(bit, std::memory_order_release);
  }
  launch_dependent(k, dim3((unsigned)(2 * pairs_of(items))), 32 * (2 + Epi::WARPS), SMEM, st, a, ep);
  return check_launch(what, 1);
}
// C = A B^T with the plain epilogue; K in chunks of 2048 for an fp32 C (see StoreEpi). Chunks of 1024, 2048, 4096
// and none (B200, weight gradient from 8 bits, 8192 rows into 4096 x 4096): 211, 203, 199, 193 us; the largest
// relative error over 65536 rows of positive numbers 2.2e-6, 4.3e-6, 1.0e-5, 3.0e-4.
constexpr int PROMOTE_KB = 32;
template <bool A_MN, bool B_MN>
int launch_store(const char* what, Args a, const StoreEpi<false>::Params& ep, cudaStream_t st) {
  if (ep.dtype == PNFT_DTYPE_F32 && a.s.kb > PROMOTE_KB * (a.s.whole ? 1 : a.s.splits)) {
    a.s.chunk = PROMOTE_KB;
    typename StoreEpi<true>::Params e;
    static_assert(sizeof(e) == sizeof(ep), "same parameters");
    memcpy(&e, &ep, sizeof(e));
    return launch<A_MN, B_MN, false, StoreEpi<true>>(what, a, e, st);
  }
  return launch<A_MN, B_MN, false, StoreEpi<false>>(what, a, ep, st);
}

// alpha A B^T (M x N, kb K blocks, the operands' maps in `a`) into C as planned: one matrix of M
// rows, or two (row_split). `work` has product_workspace's bytes; seg_kb: K blocks of the first
// pair of maps (0: all); live: device number of K that count.
template <bool A_MN, bool B_MN>
int product(const char* what, Args a, const SumArgs& c, float* work, int64_t M, int64_t N, int64_t kb, int64_t seg_kb,
            const int32_t* live, cudaStream_t st) {
  const Plan plan = plan_product(tiles_of(M, N), kb);
  a.s = plain_sched(M, N, kb, plan.splits);
  if (seg_kb) a.s.seg_kb = (int)seg_kb;
  a.s.whole = plan.whole;
  a.s.live = live;
  a.s.live_k = live != nullptr;
  typename StoreEpi<false>::Params out;
  memset(&out, 0, sizeof(out));
  const bool apart = plan.splits > 1 && !plan.whole;
  const int64_t ldp = (N + 3) / 4 * 4;
  int rc = PNFT_OK;
  if (apart) {
    out.row_split = 0x7fffffff;
    out.dtype = PNFT_DTYPE_F32;
    rc = make_out(&out.c[0], work, PNFT_DTYPE_F32, N, M, ldp, plan.splits, M * ldp);
  } else {
    out.row_split = c.row_split;
    out.dtype = c.dtype;
    out.alpha = c.alpha;
    rc = make_out(&out.c[0], c.c[0], c.dtype, N, c.rows, c.ldc);
    if (!rc && c.row_split < M) rc = make_out(&out.c[1], c.c[1], c.dtype, N, c.rows, c.ldc);
    const int64_t parts = (tiles_of(M, N) - plan.whole) * plan.splits;
    if (!rc && plan.whole) rc = make_out(&out.part, work, PNFT_DTYPE_F32, BN, PM, BN, parts, PM * BN);
  }
  if (!rc) rc = launch_store<A_MN, B_MN>(what, a, out, st);
  if (rc || plan.splits == 1) return rc;
  if (apart) return sum_splits(work, ldp, M * ldp, plan.splits, c, (int)M, st);
  return sum_tail(work, a.s, c, st);
}

// An operand that TMA can read: 16-byte base, row stride a multiple of 8 elements
// and inside the map's limit.
inline bool tma_rows_ok(const void* p, int64_t ld, int64_t cols) {
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld >= cols && ld < ((int64_t)1 << 38);
}
inline bool type16(int dtype) { return dtype == PNFT_DTYPE_BF16 || dtype == PNFT_DTYPE_F16; }

}  // namespace tc
}  // namespace pnft
