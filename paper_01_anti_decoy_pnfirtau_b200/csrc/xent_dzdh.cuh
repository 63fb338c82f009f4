// Backward of the streamed cross entropy for widths up to 256: the gradient of the logits
// and its product with the weights in one kernel, dz once to memory for dW and dh = dz W
// without reading it back.
//
// A pair of CTAs keeps its 256 rows of h in shared memory and goes through 256-word tiles
// of the vocabulary: MMA 1 computes the logits S = h W^T (256 columns of TMEM), the
// epilogue turns them into dz, 16 bits, written into shared memory as the K-major operand
// of MMA 2, dh += dz W (the other 256 columns), and from there by TMA to memory. A tile of
// W serves both products: rows x 64 columns, 128-byte swizzled, is K-major for the first
// and MN-major for the second. MMA 1 of tile j + 1 is issued before MMA 2 of tile j, also
// where tile j + 1 begins another row tile, so the tensor core has work while the epilogue
// of tile j runs: single buffers of S and dz suffice. The tiles of all rows are dealt to the pairs in
// equal runs; a run's part of a row tile leaves its share of dh in fp32, and a last kernel adds the
// shares in order. Bound by the MMAs and the store of dz: 16352 x 33278 x 256 (B200, bf16, four pieces)
// takes 465 us (1.2 PFLOP/s), 425 without that store; with three kernels instead (dz, dh, sum) a
// step's forward and backward take 1120 us, with this one 1075; at width 128 976 and 875.
#pragma once

#include "xent_math.cuh"

namespace pnft {
namespace xent {

using namespace tc;

struct DzDhArgs {
  CUtensorMap th, tw1, tw2, tdz, tpart;
  Sched s;
  const float *lse2, *rs;
  const int32_t *tgt, *live;
  int v0, V, D, Mp, bf16, stages, store_dz;
  uint32_t idesc1, idesc2;
  int32_t* status;
};

constexpr int DZDH_WARPS = 16;
constexpr int DZ_BYTES = 4 * HALF_BYTES;  // 128 rows x 256 words, 16 bits
// Stages of the ring beside kd blocks of h (464 us a step of the language model with 6, 480 with 5, 497 with 4).
__host__ __device__ constexpr int dzdh_stages(int kd) { return (STAGE_MAX - kd * HALF_BYTES - DZ_BYTES) / HALF_BYTES; }
constexpr int MAX_STAGES = dzdh_stages(1);

// NB: columns of dh per CTA's half of W in MMA 2 (64 for widths up to 128, else 128).
template <int NB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(32 * (2 + DZDH_WARPS), 1)
    xent_dzdh_kernel(const __grid_constant__ DzDhArgs p) {
  constexpr int N2 = 2 * NB, B2_BYTES = NB * 128;
  extern __shared__ __align__(1024) uint8_t raw[];
  const int stages = p.stages, kd = p.s.kb;
  const uint32_t sh = (smem_u32(raw) + 1023u) & ~1023u;  // h: kd blocks of 128 rows x 64
  const uint32_t sdz = sh + (uint32_t)kd * HALF_BYTES;   // dz: four blocks of 128 rows x 64
  const uint32_t ring = sdz + DZ_BYTES;
  // full, empty, S full / empty, dz full / empty, dh full / empty, h full / empty, done
  __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 9];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  launch_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t b0 = smem_u32(bars);
  auto full = [&](int s) { return b0 + 8u * s; };
  auto empty = [&](int s) { return b0 + 8u * (MAX_STAGES + s); };
  const uint32_t s_full = b0 + 16u * MAX_STAGES, s_empty = s_full + 8, dz_full = s_full + 16, dz_empty = s_full + 24,
                 dh_full = s_full + 32, dh_empty = s_full + 40, h_full = s_full + 48, h_empty = s_full + 56,
                 done = s_full + 64;
  const Abort ab{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_empty, 2 * DZDH_WARPS);  // the even CTA's: the epilogue warps of both
    mbar_init(dz_full, 2 * DZDH_WARPS);
    mbar_init(dz_empty, 1);
    mbar_init(dh_full, 1);
    mbar_init(dh_empty, 2 * DZDH_WARPS);
    mbar_init(h_full, 1);
    mbar_init(h_empty, 1);
    mbar_init(done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&tmem_slot), 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot), dh_acc = tmem + BN;
  wait_previous();
  const Walk walk(p.s, pairs);

  if (warp == 0) {
    // -------------------------------------------------------------- TMA producer
    if (lane == 0) {
      int st = 0, ph = 1, issued = 0, items = 0;
      auto slot = [&](uint32_t bytes) {  // the next stage of the ring, free and told what to expect
        if (!mbar_wait(empty(st), ph, ab)) return false;
        if (rank == 0) mbar_arrive_expect_tx(full(st), 2 * bytes);
        return true;
      };
      auto next = [&]() {
        ++issued;
        if (++st == stages) st = 0, ph ^= 1;
      };
      auto load1 = [&](int nt) {  // this CTA's 128 words, all columns
        for (int kb = 0; kb < kd; ++kb) {
          if (!slot(HALF_BYTES)) return false;
          tma_load_pair(ring + (uint32_t)st * HALF_BYTES, &p.tw1, map_rank(full(st), 0), kb * BK, nt * BN + rank * BM);
          next();
        }
        return true;
      };
      auto load2 = [&](int nt) {  // all 256 words, this CTA's columns
        for (int k = 0; k < BN / BK; ++k) {
          if (!slot(B2_BYTES)) return false;
          for (int g = 0; g < NB / 64; ++g)
            tma_load_pair(ring + (uint32_t)st * HALF_BYTES + (uint32_t)g * GROUP_BYTES, &p.tw2, map_rank(full(st), 0),
                          rank * NB + 64 * g, nt * BN + k * BK);
          next();
        }
        return true;
      };
      int before = -1;  // the tile whose words are still to be loaded for MMA 2
      bool ok = true;
      for (Steps q(walk, p.s, pair, rank); q.valid(); q.next()) {
        if (q.item_first()) {
          if (!(ok = mbar_wait(h_empty, (items & 1) ^ 1, ab))) break;
          if (rank == 0) mbar_arrive_expect_tx(h_full, (uint32_t)(2 * HALF_BYTES * kd));
          for (int kb = 0; kb < kd; ++kb)
            tma_load_pair(sh + (uint32_t)kb * HALF_BYTES, &p.th, map_rank(h_full, 0), kb * BK, q.it.row0);
          ++items;
        }
        if (!(ok = load1(q.nt) && (before < 0 || load2(before)))) break;
        before = q.nt;
      }
      if (ok && before >= 0) load2(before);
      if (rank == 0) {  // never leave a copy in flight (see gemm_kernel)
        if (items > 0) drain_wait(h_full, (items - 1) & 1);
        for (int n = 0; n < min(issued, stages); ++n) {
          const int last = issued - 1 - n;
          drain_wait(full(last % stages), (last / stages) & 1);
        }
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer (even CTA)
    if (rank == 0 && lane == 0) {
      int st = 0, ph = 0, items = 0, shares = 0, t1 = 0, t2 = 0;
      auto next = [&]() {
        commit_pair(empty(st));
        if (++st == stages) st = 0, ph ^= 1;
      };
      auto mma1 = [&]() {  // S = h W^T
        if (!mbar_wait(s_empty, (t1 & 1) ^ 1, ab)) return false;
        tc_fence_after();
        for (int kb = 0; kb < kd; ++kb) {
          if (!mbar_wait(full(st), ph, ab)) return false;
          tc_fence_after();
          const uint32_t da = sw128_desc(sh + (uint32_t)kb * HALF_BYTES, 0), db = sw128_desc(ring + (uint32_t)st * HALF_BYTES, 0);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) mma_pair(tmem, da + kk * 2, db + kk * 2, p.idesc1, kb > 0 || kk > 0);
          next();
        }
        commit_pair(s_full);
        ++t1;
        return true;
      };
      bool first = false, last = false;  // of its item: the tile whose MMA 2 is still to come
      auto mma2 = [&]() {  // dh (+)= dz W
        if (first && !mbar_wait(dh_empty, (shares++ & 1) ^ 1, ab)) return false;
        if (!mbar_wait(dz_full, t2 & 1, ab)) return false;
        tc_fence_after();
        for (int k = 0; k < BN / BK; ++k) {
          if (!mbar_wait(full(st), ph, ab)) return false;
          tc_fence_after();
          const uint32_t da = sw128_desc(sdz + (uint32_t)k * HALF_BYTES, 0),
                         db = sw128_desc(ring + (uint32_t)st * HALF_BYTES, GROUP_BYTES);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) mma_pair(dh_acc, da + kk * 2, db + kk * 128, p.idesc2, !first || k > 0 || kk > 0);
          next();
        }
        commit_pair(dz_empty);
        if (last) commit_pair(dh_full);
        ++t2;
        return true;
      };
      bool ok = true;
      for (Steps q(walk, p.s, pair, rank); q.valid(); q.next()) {
        if (q.item_first() && !(ok = mbar_wait(h_full, items++ & 1, ab))) break;
        if (!(ok = mma1())) break;
        if (q.item_last()) commit_pair(h_empty);
        if (t1 > 1 && !(ok = mma2())) break;
        first = q.item_first(), last = q.item_last();
      }
      if (ok && t1 > 0) mma2();
      commit_pair(done);
      drain_wait(done, 0);
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const EpiWarp w{warp & 3, 0, (warp - 2) >> 2, lane,
                    sdz + (uint32_t)((warp - 2) >> 2) * HALF_BYTES + (uint32_t)(warp & 3) * 4096u, 0u};
    Boxes<1> box(w);  // the warp's 32 rows x 64 words of dz: one box, and a quarter of an operand tile
    const uint32_t lanes = (uint32_t)(32 * w.quad) << 16;
    const uint32_t to_s = map_rank(s_empty, 0), to_dz = map_rank(dz_full, 0), to_dh = map_rank(dh_empty, 0);
    const int live = *p.live;
    float lse = 0.f, rs = 0.f;
    int tgt = -1, t = 0, shares = 0, share_of = -1;  // the row tile whose share of dh is still to be written
    bool ok = true;
    auto write_share = [&]() {
      if (!warp_wait(dh_full, shares & 1, ab)) return false;
      ++shares;
      tc_fence_after();
#pragma unroll 1
      for (int c = w.slice * (N2 / 4); c < min((w.slice + 1) * (N2 / 4), p.D); c += 32) {
        float v[32];
        acc_load32(dh_acc + lanes + c, false, v);
        const uint32_t s = box.take();
        box.put32(s, v);
        box.store(s, &p.tpart, c, rank * BM + 32 * w.quad, share_of + pair);
      }
      share_of = -1;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(to_dh);
      return true;
    };
    for (Steps q(walk, p.s, pair, rank); q.valid(); q.next(), ++t) {
      const int row = q.it.row0 + w.row();
      if (q.item_first()) {
        lse = row < live ? p.lse2[row] : 0.f;
        rs = row < live ? p.rs[row] : 0.f;
        tgt = row < live ? p.tgt[row] - p.v0 : -1;
      }
      if (!(ok = warp_wait(s_full, t & 1, ab))) break;
      tc_fence_after();
      uint32_t z[2][32];
      tmem_load32x2(tmem + lanes + w.slice * 64, z[0], tmem + lanes + w.slice * 64 + 32, z[1]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(to_s);
      const int col = q.nt * BN + w.slice * 64, n = row < live ? p.V - p.v0 - col : 0, tc = tgt - col;
      const f32x2 scale = pack(kLog2e, kLog2e), minus = pack(-lse, -lse), factor = pack(rs, rs);
      uint32_t d[2][16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x2 x = fma2(pack(__uint_as_float(z[h][2 * i]), __uint_as_float(z[h][2 * i + 1])), scale, minus);
          const float2 e = unpack(mul2(exp2_pair(x), factor));
          v[2 * i] = e.x, v[2 * i + 1] = e.y;
        }
        if ((unsigned)(tc - 32 * h) < 32u) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i == tc - 32 * h) v[i] -= rs;
        }
        if (n < 64) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * h + i >= n) v[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) d[h][i] = pack2(v[2 * i], v[2 * i + 1], p.bf16);
      }
      // free once MMA 2 of the tile before and the warp's own store out of it have read it
      if (!(ok = warp_wait(dz_empty, (t & 1) ^ 1, ab))) break;
      if (share_of >= 0 && !(ok = write_share())) break;  // through the same box, the item before being complete
      const uint32_t b = box.take();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; i += 4) box.put(b, 4 * h + i / 4, d[h][i], d[h][i + 1], d[h][i + 2], d[h][i + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        // Each CTA's tensor core reads its own shared memory: the proxy fence above has made the warp's
        // writes visible there, and the arrival on the even CTA's barrier comes after it. No other memory
        // is published by it.
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(to_dz) : "memory");
        if (p.store_dz && q.it.row0 < p.Mp) tma_store_3d(&p.tdz, b, col, q.it.row0 + 32 * w.quad, 0);
        bulk_commit();
      }
      if (q.item_last()) share_of = q.it.mt;
    }
    if (ok && share_of >= 0) write_share();
    box.finish();
  }
  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN);
  }
}

// Adds the runs' shares of dh in the order of the pairs: onto acc [compacted rows], or, for
// the last piece, times alpha into dh's rows (zeros where a row does not count).
struct JoinArgs {
  const float* part;  // [row tile + pair][256][ld]
  float* acc;
  int64_t ld;
  const int32_t *counts, *pos;
  const float* alpha;
  void* dh;
  int64_t lddh;
  int64_t M;
  int D, dtype, tiles_n, pairs, first, last, vec;
};
__global__ void __launch_bounds__(256) xent_join_kernel(JoinArgs p) {
  launch_next();
  wait_previous();
  const int lane = threadIdx.x & 31, tiles_m = (p.counts[0] + PM - 1) / PM;
  const int64_t total = (int64_t)tiles_m * p.tiles_n;
  const int pairs = Walk::run_pairs(total, p.pairs);
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < p.M; r += (int64_t)gridDim.x * 8) {
    const int at = p.pos[r];
    if (at < 0 && !p.last) continue;
    const float a = at >= 0 ? *p.alpha : 0.f;  // alpha may be infinite or NaN
    int k0 = 0, k1 = -1, mt = 0;
    if (at >= 0) {
      mt = at / PM;
      k0 = run_owner(total, (int64_t)mt * p.tiles_n, pairs), k1 = run_owner(total, (int64_t)(mt + 1) * p.tiles_n - 1, pairs);
    }
    for (int c = 4 * lane; c < p.D; c += 128) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at >= 0 && !p.first) v = *reinterpret_cast<const float4*>(p.acc + at * p.ld + c);
      for (int k = k0; k <= k1; ++k) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(p.part + ((int64_t)(mt + k) * PM + at % PM) * p.ld + c));
        v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
      }
      if (!p.last) {
        *reinterpret_cast<float4*>(p.acc + at * p.ld + c) = v;
        continue;
      }
      const float f[4] = {v.x * a, v.y * a, v.z * a, v.w * a};
      store_row4(p.dh, r * p.lddh + c, f, p.D - c, p.dtype, p.vec);
    }
  }
}

}  // namespace xent
}  // namespace pnft
