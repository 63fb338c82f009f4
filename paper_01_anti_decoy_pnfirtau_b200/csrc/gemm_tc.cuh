// A persistent tcgen05 GEMM with a pluggable epilogue, the core of the gated
// feed-forward, streamed cross-entropy and 8-bit-checkpoint kernels:
//
//   acc[m, n] = sum_k A[m, k] B[n, k]     (bf16 or fp16 operands, fp32 in TMEM)
//
// One CTA per SM walks work items; an item is a 128 x 256 output tile (or, for
// epilogues that carry state along a row, a strip of such tiles), optionally one
// of several splits of K. Warp 0 loads 64-deep stages of A and B by TMA into a
// ring, one lane of warp 1 issues the MMAs (M = 128, N = 256, K = 16) into one of
// two TMEM accumulators, warps 2-9 run the epilogue of the other, so the epilogue
// of a tile overlaps the next tile's MMAs. Either operand may be K-major (rows of
// K) or MN-major (K rows of M or N), so no caller transposes anything. Rows,
// columns and K past the end are zero-filled by TMA.
#pragma once

#include <string.h>

#include <algorithm>

#include "flash.cuh"
#include "sm100_ptx.cuh"

namespace pnft {
namespace tc {

using namespace sm100;

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int STAGES = 4;
constexpr int GROUP_BYTES = 64 * BK * 2;  // MN-major: 64 columns x 64 K rows
constexpr int SMEM = STAGES * STAGE_BYTES + 1024;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);

// Which tiles there are and in which order: items of one split are taken group_m
// row tiles at a time, the row tile running fastest, so the CTAs in flight share
// both operands in L2.
struct Sched {
  int tiles_m;          // row tiles (upper bound when live is given)
  int strips;           // items along N
  int tiles_n;          // column tiles
  int tiles_per_strip;  // column tiles per item
  int kb;               // 64-deep K blocks (upper bound when live_k)
  int splits;           // splits of K
  int group_m;
  int seg_kb;           // K blocks of the first pair of maps; the rest use the second
  const int32_t* live;  // device: rows that count (NULL: all)
  int live_m, live_k;   // the rows that count bound M / K
};

struct Args {
  CUtensorMap ta[2], tb[2];
  Sched s;
  uint32_t idesc;
  int32_t* status;
};

struct Item {
  int mt, nt0, ntn, split, kb0, kbn;
};

struct Walk {
  int tiles_m, kb, items;
  __device__ explicit Walk(const Sched& s) {
    tiles_m = s.tiles_m, kb = s.kb;
    if (s.live) {
      const int n = *s.live;
      if (s.live_m) tiles_m = (n + BM - 1) / BM;
      if (s.live_k) kb = (n + BK - 1) / BK;
    }
    items = tiles_m * s.strips * s.splits;
  }
  __device__ Item at(const Sched& s, int i) const {
    Item it;
    const int per_split = tiles_m * s.strips;
    it.split = i / per_split;
    int r = i - it.split * per_split;
    const int per = s.group_m * s.strips, g = r / per;
    r -= g * per;
    const int gm = min(s.group_m, tiles_m - g * s.group_m);
    it.mt = g * s.group_m + r % gm;
    const int strip = r / gm;
    it.nt0 = strip * s.tiles_per_strip;
    it.ntn = min(s.tiles_per_strip, s.tiles_n - it.nt0);
    // whole K blocks spread evenly over the splits
    it.kb0 = (int)((int64_t)kb * it.split / s.splits);
    it.kbn = (int)((int64_t)kb * (it.split + 1) / s.splits) - it.kb0;
    return it;
  }
};

// What an epilogue warp knows: its TMEM lane quadrant, its half of the columns.
struct EpiWarp {
  int quad, half, lane;
  __device__ int row() const { return 32 * quad + lane; }
  __device__ uint32_t lanes() const { return (uint32_t)(32 * quad) << 16; }
};

// Epi: item_begin(item), tile(item, nt, acc, zero, release), item_end(item).
// `acc` is the accumulator's TMEM address with the warp's lanes; `zero` says that
// no K block contributed (the accumulator is then undefined and stands for 0);
// release() hands the accumulator back once its last column is in registers.
// DUAL_B: columns 0-127 of a tile come from tb[0] and 128-255 from tb[1], both at
// row 128 * nt.
template <bool A_MN, bool B_MN, bool DUAL_B, class Epi>
__global__ void __launch_bounds__(THREADS, 1) gemm_kernel(const __grid_constant__ Args p,
                                                          const __grid_constant__ typename Epi::Params ep) {
  extern __shared__ __align__(1024) uint8_t raw[];
  const uint32_t sb = (smem_u32(raw) + 1023u) & ~1023u;
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 5];  // full, empty, acc full x2, acc empty x2, done
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t b0 = smem_u32(bars);
  auto full = [&](int s) { return b0 + 8u * s; };
  auto empty = [&](int s) { return b0 + 8u * (STAGES + s); };
  auto acc_full = [&](int s) { return b0 + 8u * (2 * STAGES + s); };
  auto acc_empty = [&](int s) { return b0 + 8u * (2 * STAGES + 2 + s); };
  const uint32_t done = b0 + 8u * (2 * STAGES + 4);
  const Abort ab{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full(s), 1);
      mbar_init(acc_empty(s), EPI_WARPS);
    }
    mbar_init(done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const Walk walk(p.s);

  if (warp == 0) {
    // -------------------------------------------------------------- TMA producer
    if (lane == 0) {
      int st = 0, ph = 1, issued = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < walk.items; i += gridDim.x) {
        const Item it = walk.at(p.s, i);
        for (int nt = it.nt0; ok && nt < it.nt0 + it.ntn; ++nt) {
          for (int kb = it.kb0; kb < it.kb0 + it.kbn; ++kb) {
            if (!mbar_wait(empty(st), ph, ab)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(full(st), STAGE_BYTES);
            const int seg = kb >= p.s.seg_kb;
            const int k = (kb - (seg ? p.s.seg_kb : 0)) * BK;
            const uint32_t sa = sb + (uint32_t)st * STAGE_BYTES, sB = sa + A_BYTES;
            if (A_MN) {
#pragma unroll
              for (int g = 0; g < BM / 64; ++g)
                tma_load_2d(sa + g * GROUP_BYTES, &p.ta[seg], full(st), it.mt * BM + 64 * g, k);
            } else {
              tma_load_2d(sa, &p.ta[seg], full(st), k, it.mt * BM);
            }
            if (B_MN) {
#pragma unroll
              for (int g = 0; g < BN / 64; ++g)
                tma_load_2d(sB + g * GROUP_BYTES, &p.tb[seg], full(st), nt * BN + 64 * g, k);
            } else if (DUAL_B) {
              tma_load_2d(sB, &p.tb[0], full(st), k, nt * (BN / 2));
              tma_load_2d(sB + B_BYTES / 2, &p.tb[1], full(st), k, nt * (BN / 2));
            } else {
              tma_load_2d(sB, &p.tb[seg], full(st), k, nt * BN);
              tma_load_2d(sB + B_BYTES / 2, &p.tb[seg], full(st), k, nt * BN + BN / 2);
            }
            ++issued;
            if (++st == STAGES) st = 0, ph ^= 1;
          }
        }
      }
      // never leave a copy in flight into this CTA's shared memory
      for (int n = 0; n < min(issued, STAGES); ++n) {
        const int last = issued - 1 - n;
        drain_wait(full(last % STAGES), (last / STAGES) & 1);
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      int st = 0, ph = 0, t = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < walk.items; i += gridDim.x) {
        const Item it = walk.at(p.s, i);
        for (int j = 0; ok && j < it.ntn; ++j, ++t) {
          if (!mbar_wait(acc_empty(t & 1), ((t >> 1) & 1) ^ 1, ab)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(t & 1) * BN;
          for (int kb = 0; kb < it.kbn; ++kb) {
            if (!mbar_wait(full(st), ph, ab)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = sb + (uint32_t)st * STAGE_BYTES;
            const uint32_t da = sw128_desc(sa, A_MN ? GROUP_BYTES : 0), db = sw128_desc(sa + A_BYTES, B_MN ? GROUP_BYTES : 0);
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)  // 16 K: 32 bytes of a K-major row, 16 rows (2048 bytes) MN-major
              mma_ss(d, da + kk * (A_MN ? 128 : 2), db + kk * (B_MN ? 128 : 2), p.idesc, (kb | kk) != 0);
            mma_commit(empty(st));
            if (++st == STAGES) st = 0, ph ^= 1;
          }
          if (ok) mma_commit(acc_full(t & 1));
        }
      }
      mma_commit(done);
      drain_wait(done, 0);  // no MMA may still be writing TMEM at teardown
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const EpiWarp w{warp & 3, (warp - 2) >> 2, lane};
    Epi epi(ep, w);
    int t = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < walk.items; i += gridDim.x) {
      const Item it = walk.at(p.s, i);
      epi.item_begin(it);
      for (int j = 0; j < it.ntn; ++j, ++t) {
        if (!warp_wait(acc_full(t & 1), (t >> 1) & 1, ab)) {
          ok = false;
          break;
        }
        tc_fence_after();
        epi.tile(it, it.nt0 + j, tmem + (uint32_t)(t & 1) * BN + w.lanes(), it.kbn == 0, [&]() {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty(t & 1));
        });
      }
      if (ok) epi.item_end(it);
    }
  }
  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * BN);
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

__device__ __forceinline__ void acc_load32(uint32_t addr, bool zero, float (&v)[32]) {
  uint32_t r[32];
  tmem_load32(addr, r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = zero ? 0.f : __uint_as_float(r[i]);
}

// ------------------------------------------------------------------ plain epilogue
// C = alpha * acc into rows of fp32 / bf16 / fp16 (rows row_split.. go to c[1]), or
// the fp32 partial of a split, or added to an fp32 C.
struct StoreEpi {
  struct Params {
    void* c[2];
    int64_t ldc;
    int row_split;         // rows of c[0]'s part in the product (a multiple of nothing: any)
    int rows, cols;        // rows of each part that exist, columns
    const float* alpha;    // device scalar (NULL: 1)
    int dtype;             // of C
    int accumulate;        // C (fp32) += acc
    int64_t split_stride;  // elements between the splits' partials (0: no splits)
    int vec;               // C's rows are 16-byte aligned
  };
  const Params& p;
  EpiWarp w;
  float alpha;
  __device__ StoreEpi(const Params& p_, const EpiWarp& w_) : p(p_), w(w_) { alpha = p.alpha ? *p.alpha : 1.f; }
  __device__ void item_begin(const Item&) {}
  __device__ void item_end(const Item&) {}
  template <class Release>
  __device__ void tile(const Item& it, int nt, uint32_t acc, bool zero, Release release) {
    int row = it.mt * BM + w.row();
    const int part = row >= p.row_split;
    if (part) row -= p.row_split;
    const bool live = row < p.rows;
    const int64_t at = (int64_t)it.split * p.split_stride + (int64_t)row * p.ldc;
#pragma unroll 1
    for (int c = w.half * (BN / 2); c < (w.half + 1) * (BN / 2); c += 32) {
      float v[32];
      acc_load32(acc + c, zero, v);
      if (c + 32 == (w.half + 1) * (BN / 2)) release();
      const int col = nt * BN + c, n = p.cols - col;
      if (!live || n <= 0) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha;
      if (p.dtype == PNFT_DTYPE_F32) {
        float* dst = static_cast<float*>(p.c[part]) + at + col;
        if (p.accumulate) {
          if (p.vec && n >= 32) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 f = *reinterpret_cast<const float4*>(dst + i);
              v[i] += f.x, v[i + 1] += f.y, v[i + 2] += f.z, v[i + 3] += f.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < n) v[i] += dst[i];
          }
        }
        store_row32<32>(dst, v, n, p.vec);
      } else {
        store_row16<32>(static_cast<uint16_t*>(p.c[part]) + at + col, v, n, p.vec, p.dtype == PNFT_DTYPE_BF16);
      }
    }
  }
};

// ------------------------------------------------------------------ host side
int sm_count();
// Splits of K for an output of `tiles` tiles: about one work item per SM, at least
// 8 K blocks (512 of K) each, since shorter ones cost more in partial sums than
// they gain.
int plan_splits(int tiles, int kb);
// Sums the splits' fp32 partials [splits][rows_total][ldp] in split order (bitwise
// reproducible), times alpha, into C (two parts as StoreEpi) or onto an fp32 C.
int sum_splits(const float* part, int64_t ldp, int64_t split_stride, int splits, const StoreEpi::Params& out,
               int rows_total, cudaStream_t st);

// K-major operand: `rows` rows of K elements; MN-major operand: K rows of `cols`
// elements. Both take the row stride in elements (a multiple of 8, 16-byte base).
inline int map_kmajor(CUtensorMap* m, const void* base, int64_t k, int64_t rows, int64_t ld) {
  return tma_map_rows(m, base, k, rows, ld, 128);
}
inline int map_mnmajor(CUtensorMap* m, const void* base, int64_t cols, int64_t k, int64_t ld) {
  return tma_map_rows(m, base, cols, k, ld, BK);
}

inline uint32_t idesc(int dtype, bool a_mn, bool b_mn) {
  return idesc_f16(BM, BN, dtype == PNFT_DTYPE_BF16 ? 1 : 0, a_mn, b_mn);
}

inline Sched plain_sched(int64_t m, int64_t n, int64_t kb, int splits) {
  Sched s;
  memset(&s, 0, sizeof(s));
  s.tiles_m = (int)((m + BM - 1) / BM);
  s.tiles_n = s.strips = (int)((n + BN - 1) / BN);
  s.tiles_per_strip = 1;
  s.kb = s.seg_kb = (int)kb;
  s.splits = splits;
  s.group_m = 16;
  return s;
}

template <bool A_MN, bool B_MN, bool DUAL_B, class Epi>
int launch(const char* what, const Args& a, const typename Epi::Params& ep, cudaStream_t st) {
  const int64_t items = (int64_t)a.s.tiles_m * a.s.strips * a.s.splits;
  if (items <= 0) return PNFT_OK;
  if (items > (1 << 30)) return fail(PNFT_EUNSUPPORTED, "%s: too many tiles", what);
  auto* k = gemm_kernel<A_MN, B_MN, DUAL_B, Epi>;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
    return check_launch(what, 0);
  k<<<(unsigned)std::min<int64_t>(items, sm_count()), THREADS, SMEM, st>>>(a, ep);
  return check_launch(what, 1);
}

inline bool rows16(const void* p, int64_t ld, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0;
}
// An operand that TMA can read: 16-byte base, row stride a multiple of 8 elements
// and inside the map's limit.
inline bool tma_rows_ok(const void* p, int64_t ld, int64_t cols) {
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld >= cols && ld < ((int64_t)1 << 38);
}
inline bool type16(int dtype) { return dtype == PNFT_DTYPE_BF16 || dtype == PNFT_DTYPE_F16; }

}  // namespace tc
}  // namespace pnft
