// Softmax cross entropy of a language-model head in pieces of the vocabulary, without
// keeping the logits, and its gradient:
//
//   z_iv = h_i . W_v,  loss_i = log sum_v exp(z_iv) - z_{i,t_i}
//   dz_iv = s_i (exp(z_iv - lse_i) - [v = t_i]),  dh = dz W,  dW = dz^T h
//
// Forward: one pass of the GEMM over strips of the vocabulary; the epilogue keeps each
// row's running maximum and sum in registers, so nothing of size rows x vocabulary
// exists. Backward: for one piece of the vocabulary at a time the logits are computed
// again from the kept logarithm of the sum, their gradient goes to a buffer of that
// piece, and two GEMMs turn it into a share of dh and the piece's rows of dW.
//
// Rows whose target is ignore_index cost nothing: the first kernel moves the rows that
// count to the front of a buffer (and their number to device memory), and every later
// kernel sizes its work by that number. So nothing in a masked row, NaN and infinities
// included, reaches a result.
#include "gemm_tc.cuh"
#include "skinny.cuh"
#include "xent_dzdh.cuh"

namespace pnft {
namespace {

using namespace tc;
using namespace xent;

// Device state of one call, in the caller's buffers (rows are compacted rows).
struct State {
  int32_t* counts;   // [0] rows that count, [1] blocks of the reduction that are done
  int32_t* pos;      // [M] compacted row of a row, or -1
  int32_t* idx;      // [Mp] row of a compacted row
  int32_t* tgt;      // [Mp] its target
  float* lse2;       // [Mp] log2 of the sum of exponentials
};

// ------------------------------------------------------------------ compaction
constexpr int CT = 256;
struct CompactArgs {
  const int64_t* t;
  int64_t ignore;
  const uint16_t* h;
  int64_t ldh;
  uint16_t* hc;
  int64_t ldc;
  State s;
  float* zt;        // [Mp] target logits (NaN where the target is no column)
  float* row_loss;  // [M] or NULL: ignored rows get 0
  int64_t M;
  int V, D, rows, vec;
  int64_t Mp;
  int32_t* status;
};

__device__ __forceinline__ int block_total(int v, int* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
  for (int k = 0; k < CT / 32; ++k) t += red[k];
  return t;
}

// Block b owns rows [b * rows, ...): it counts the rows that count before them (every
// block reads all earlier targets: at most 512 blocks, a few bytes per row), places its
// own in order and copies them.
__global__ void __launch_bounds__(CT) xent_compact_kernel(CompactArgs p) {
  __shared__ int red[CT / 32], place[CT];
  launch_next();
  wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows, r1 = std::min<int64_t>(p.M, r0 + p.rows);
  int n = 0;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < r0; r += CT) n += p.t[r] != p.ignore;
  int base = block_total(n, red);
  for (int64_t c0 = r0; c0 < r1; c0 += CT) {
    const int64_t r = c0 + threadIdx.x;
    const int64_t t = r < r1 ? p.t[r] : 0;
    const bool counts = r < r1 && t != p.ignore;
    const unsigned vote = __ballot_sync(0xffffffffu, counts);
    __syncthreads();
    if (lane == 0) red[warp] = __popc(vote);
    __syncthreads();
    int at = base, total = 0;
    for (int k = 0; k < CT / 32; ++k) {
      if (k < warp) at += red[k];
      total += red[k];
    }
    at += __popc(vote & ((1u << lane) - 1));
    place[threadIdx.x] = counts ? at : -1;
    if (r < r1) p.s.pos[r] = counts ? at : -1;
    if (counts) {
      p.s.idx[at] = (int)r;
      const bool good = t >= 0 && t < p.V;
      p.s.tgt[at] = good ? (int)t : -1;
      if (!good) {
        p.zt[at] = __int_as_float(0x7fc00000);
        report_status(p.status, PNFT_DEV_BAD_INDEX);
      }
    } else if (r < r1 && p.row_loss) {
      p.row_loss[r] = 0.f;
    }
    base += total;
    __syncthreads();
    // the rows themselves: 16 bytes at a time where both sides allow it, four in flight per thread
    const int rows = (int)std::min<int64_t>(CT, r1 - c0), vecs = p.vec ? p.D / 8 : 0, rest = p.D - 8 * vecs;
    const uint16_t* h = p.h + c0 * p.ldh;
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * vecs; i += CT) {
      const int k = i / vecs, v = i - k * vecs;
      if (place[k] >= 0)
        reinterpret_cast<uint4*>(p.hc + place[k] * p.ldc)[v] = __ldcs(reinterpret_cast<const uint4*>(h + k * p.ldh) + v);
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * rest; i += CT) {
      const int k = i / rest, v = 8 * vecs + i - k * rest;
      if (place[k] >= 0) p.hc[place[k] * p.ldc + v] = h[k * p.ldh + v];
    }
  }
  if (r1 == p.M) {  // the last block knows the number of rows; zeros up to the tile's end
    if (threadIdx.x == 0) p.s.counts[0] = base, p.s.counts[1] = 0;
    const int64_t end = std::min<int64_t>(p.Mp, ((int64_t)base + 127) / 128 * 128);
    for (int64_t r = base + warp; r < end; r += CT / 32)
      for (int i = lane; i < p.D; i += 32) p.hc[r * p.ldc + i] = 0;
  }
}

// ------------------------------------------------------------------ forward epilogue
// Per row, half of the columns and group of warps: running maximum (times log2 e) and sum of
// 2^(z log2 e - max), both fp32, over the group's tiles of an item. PROMOTE: a tile's
// accumulators (chunks of K) are collected in fp32 registers first: the tensor core's own sum
// over K truncates, which an fp32 loss shows (1.1e-6 of it at width 2048, 2.7e-6 at 4096). The
// registers for that leave room for 8 warps, enough where a tile has MMAs of more than 16 K blocks.
// At K = 256 a tile's exponentials take as long as its MMAs: for 16352 x 33278 x 256 this kernel
// takes 200 to 217 us with the clock (1.28 to 1.39 PFLOP/s), 190 with an epilogue of loads alone.
template <bool PROMOTE>
struct LseEpi {
  static constexpr int WARPS = PROMOTE ? 8 : 16, BOXES = 0, BOX_BYTES = 0;
  static constexpr bool PING_PONG = !PROMOTE;
  static constexpr int W = 64;
  struct Params {
    float *part_m, *part_s;  // [row tile][slot][group and half][256]
    float* zt;
    const int32_t* tgt;
    const int32_t* live;
    int V;
  };
  const Params& p;
  EpiWarp w;
  float m, s;
  int tgt, live;
  float sum[PROMOTE ? BN / 2 : 1];
  __device__ LseEpi(const Params& p_, const EpiWarp& w_, const Abort&) : p(p_), w(w_) {
    live = *p.live;
#pragma unroll
    for (float& v : sum) v = 0.f;
  }
  __device__ void prepare(const Steps& q) {
    if (!q.item_first()) return;
    m = kLow, s = 0.f;
    const int row = q.it.row0 + w.row();
    tgt = row < live ? p.tgt[row] : -1;
  }
  __device__ void done() {}
  __device__ void end(const Steps& q) {  // also of a group that had no tile of the item: maximum and sum of nothing
    const int row = q.it.row0 + w.row();
    if (!q.item_last() || row >= live) return;
    const int64_t at = (((int64_t)q.it.mt * q.walk.slots + q.it.slot) * 4 + 2 * w.group + w.slice) * PM + row % PM;
    p.part_m[at] = m;
    p.part_s[at] = s;
    if (PROMOTE) p.part_m[at + 2 * PM] = kLow, p.part_s[at + 2 * PM] = 0.f;  // there is no second group
  }
  // The logits z of columns col on.
  __device__ __forceinline__ void take(float (&z)[W], int row, int col) {
    const int n = p.V - col;
    if (n < W) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i >= n) z[i] = __int_as_float(0xff800000);  // -infinity
    }
    const int tc = tgt - col;
    if ((unsigned)tc < (unsigned)W) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v = i == tc ? z[i] : v;
      p.zt[row] = v;
    }
    float top[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) top[k] = max3(z[k], z[k + 4], z[k + 8]);
#pragma unroll
    for (int i = 12; i < W - 4; i += 8) {
#pragma unroll
      for (int k = 0; k < 4; ++k) top[k] = max3(top[k], z[i + k], z[i + k + 4]);
    }
    top[0] = max3(top[0], z[W - 4], z[W - 3]), top[1] = max3(top[1], z[W - 2], z[W - 1]);
    const float nm = fmaxf(m, kLog2e * max3(top[0], top[1], fmaxf(top[2], top[3])));
    const f32x2 scale = pack(kLog2e, kLog2e), minus = pack(-nm, -nm);
    f32x2 sums[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const f32x2 x = fma2(pack(z[2 * i], z[2 * i + 1]), scale, minus);
      sums[i & 3] = add2(sums[i & 3], exp2_pair(x));
    }
    const float2 t = unpack(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
    s = fmaf(s, ex2(m - nm), t.x + t.y);
    m = nm;
  }
  template <class Release>
  __device__ __forceinline__ void tile(const Steps& q, uint32_t acc, Release release) {
    const int row = q.it.row0 + w.row(), c0 = w.slice * (BN / 2);
    if constexpr (PROMOTE) {
#pragma unroll
      for (int c = 0; c < BN / 2; c += 16) {
        uint32_t r[16];
        tmem_load16(acc + c0 + c, r);
        if (c + 16 == BN / 2) release();
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[c + i] += __uint_as_float(r[i]);
      }
      if (!q.tile_last()) return;
#pragma unroll
      for (int c = 0; c < BN / 2; c += W) {
        float z[W];
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] = sum[c + i], sum[c + i] = 0.f;
        take(z, row, q.nt * BN + c0 + c);
      }
    } else {
#pragma unroll 1
      for (int c = c0; c < c0 + BN / 2; c += W) {
        uint32_t r[2][W / 2];
        tmem_load32x2(acc + c, r[0], acc + c + W / 2, r[1]);
        if (c + W == c0 + BN / 2) release();
        float z[W];
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] = __uint_as_float(r[i / (W / 2)][i % (W / 2)]);
        take(z, row, q.nt * BN + c);
      }
    }
  }
};

// Joins the strips' maxima and sums: lse2, the row's loss, and (last block) the loss of
// all rows, summed block by block in a fixed order in 64 bits.
struct ReduceArgs {
  const float *part_m, *part_s, *zt;
  State s;
  float* row_loss;  // [M], or NULL
  float* loss;      // scalar, or NULL
  double* block_sum;
  int runs, tiles_n, pairs, mean;
};
// A block takes ROWS rows, 256 / ROWS threads each: many threads per row when there are
// few rows, which then have many strips.
template <int ROWS>
__global__ void __launch_bounds__(256) xent_reduce_kernel(ReduceArgs p) {
  __shared__ double red[256];
  __shared__ float top[256], sum[256];
  __shared__ int last;
  constexpr int LANES = 256 / ROWS;
  launch_next();
  wait_previous();
  const int n = p.s.counts[0];
  const int r = threadIdx.x % ROWS, lane = threadIdx.x / ROWS;
  const int64_t i = (int64_t)blockIdx.x * ROWS + r;
  // the pairs of the row's tile: one per strip, or one per run that the tile lies in
  const int tiles_m = (n + PM - 1) / PM;
  const int64_t mt = i / PM, total = (int64_t)tiles_m * p.tiles_n;
  int slots = 1, parts = 4;
  if (i < n && !p.runs) {
    slots = auto_strips(tiles_m, p.tiles_n, p.pairs);
    parts = 4 * slots;
  }
  if (i < n && p.runs) {
    const int pairs = Walk::run_pairs(total, p.pairs);
    slots = Walk::run_slots(tiles_m, pairs);
    parts = 4 * (run_owner(total, (mt + 1) * p.tiles_n - 1, pairs) - run_owner(total, mt * p.tiles_n, pairs) + 1);
  }
  const float *pm = p.part_m + mt * slots * 4 * PM + i % PM, *ps = p.part_s + mt * slots * 4 * PM + i % PM;
  float m = kLow;
  if (i < n) {
#pragma unroll 4
    for (int k = lane; k < parts; k += LANES) m = fmaxf(m, pm[k * PM]);
  }
  top[threadIdx.x] = m;
  __syncthreads();
  for (int o = LANES / 2; o > 0; o >>= 1) {
    if (lane < o) top[threadIdx.x] = fmaxf(top[threadIdx.x], top[threadIdx.x + o * ROWS]);
    __syncthreads();
  }
  m = top[r];
  float s = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int k = lane; k < parts; k += LANES) s += ps[k * PM] * ex2(pm[k * PM] - m);
  }
  sum[threadIdx.x] = s;
  __syncthreads();
  for (int o = LANES / 2; o > 0; o >>= 1) {
    if (lane < o) sum[threadIdx.x] += sum[threadIdx.x + o * ROWS];
    __syncthreads();
  }
  double mine = 0.0;
  if (i < n && lane == 0) {
    s = sum[r];
    const float l = log2f(s);
    p.s.lse2[i] = m + l;
    const float loss = kLn2 * (fmaf(-p.zt[i], kLog2e, m) + l);
    if (p.row_loss) p.row_loss[p.s.idx[i]] = loss;
    mine = loss;
  }
  if (!p.loss) return;
  red[threadIdx.x] = mine;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.block_sum[blockIdx.x] = red[0];
    __threadfence();
    last = atomicAdd(&p.s.counts[1], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double t = 0.0;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 256) t += __ldcg(p.block_sum + b);
  __syncthreads();
  red[threadIdx.x] = t;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.loss = (float)(p.mean ? red[0] / (double)n : red[0]);
}

// ------------------------------------------------------------------ a few rows
// From 25 rows on the tiles win (B200, bf16, cold L2: 33278 x 256 weights 15 us here at one
// row, 20 at 24 and 28 to 35 in tiles; 50021 x 1024 36, 45 and 47 to 54).
constexpr int SKINNY_ROWS = PNFT_XENT_FEW_ROWS;
// Loss of few rows without a gradient: every warp takes 16 or 32 words of the vocabulary
// at a time and keeps each row's maximum and sum over them; a block joins its warps' and
// leaves one pair per row. Rows to ignore are computed with the others (a column of the
// product touches no other) and left out at the end.
struct SkinnyArgs {
  const uint16_t *h, *w;
  int64_t ldh, ldw;
  const int64_t* t;
  int64_t ignore;
  float *part_m, *part_s, *zt;  // [blocks][SKINNY_ROWS], [SKINNY_ROWS]
  float *row_loss, *loss;
  int M, D, V, blocks, mean;
  int32_t* status;
};
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  s = s * ex2(m - top) + s2 * ex2(m2 - top);
  m = top;
}
// Groups of 16 words per warp: two share the rows' fragments when there are many rows (B200, one group and
// two, us: 24 rows of 50021 x 1024 51, 45 and of 33278 x 256 18, 20; 16 rows 41, 43 and 16, 18; one row 37, 35
// and 14, 16).
constexpr int skinny_groups(int nt) { return nt <= 2 ? 1 : 2; }
template <int NT, bool VEC, bool BF16>
__global__ void __launch_bounds__(32 * skinny::WARPS, 2) xent_skinny_kernel(SkinnyArgs p) {
  __shared__ float sm[skinny::WARPS][8 * NT], ss[skinny::WARPS][8 * NT];
  launch_next();
  wait_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float m[NT][2], s[NT][2];
  int tgt[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = 8 * j + 2 * t + k;
      m[j][k] = kLow, s[j][k] = 0.f;
      const int64_t v = n < p.M ? p.t[n] : -1;
      tgt[j][k] = v >= 0 && v < p.V ? (int)v : -1;
    }
  constexpr int RG = skinny_groups(NT);
  for (int64_t v0 = (blockIdx.x * skinny::WARPS + warp) * (16 * RG); v0 < p.V; v0 += gridDim.x * skinny::WARPS * (16 * RG)) {
    float acc[RG][NT][4] = {};
    const uint16_t* w[2 * RG];
#pragma unroll
    for (int r = 0; r < 2 * RG; ++r) w[r] = p.w + min(v0 + g + 8 * r, (int64_t)p.V - 1) * p.ldw;
    skinny::dot<true, RG, NT, VEC, BF16>(w, p.h, p.ldh, p.M, p.D, 0, 1, acc);
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      const int r0 = (int)v0 + 16 * r + g, r1 = r0 + 8;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (r0 == tgt[j][k]) p.zt[8 * j + 2 * t + k] = acc[r][j][k];
          if (r1 == tgt[j][k]) p.zt[8 * j + 2 * t + k] = acc[r][j][k + 2];
          const float a = r0 < p.V ? acc[r][j][k] : -INFINITY, b = r1 < p.V ? acc[r][j][k + 2] : -INFINITY;
          const float top = max3(m[j][k], a * kLog2e, b * kLog2e);
          s[j][k] = s[j][k] * ex2(m[j][k] - top) + ex2(fmaf(a, kLog2e, -top)) + ex2(fmaf(b, kLog2e, -top));
          m[j][k] = top;
        }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
        join(m[j][k], s[j][k], __shfl_xor_sync(0xffffffffu, m[j][k], o), __shfl_xor_sync(0xffffffffu, s[j][k], o));
      if (g == 0) sm[warp][8 * j + 2 * t + k] = m[j][k], ss[warp][8 * j + 2 * t + k] = s[j][k];
    }
  __syncthreads();
  const int n = threadIdx.x;
  if (n >= p.M) return;
  float a = sm[0][n], b = ss[0][n];
  for (int k = 1; k < skinny::WARPS; ++k) join(a, b, sm[k][n], ss[k][n]);
  p.part_m[blockIdx.x * SKINNY_ROWS + n] = a;
  p.part_s[blockIdx.x * SKINNY_ROWS + n] = b;
}

// Joins the blocks' pairs, a warp per row, and sums the rows.
__global__ void __launch_bounds__(1024) xent_skinny_reduce_kernel(SkinnyArgs p) {
  __shared__ float losses[SKINNY_ROWS];
  __shared__ int counted[SKINNY_ROWS];
  launch_next();
  wait_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int n = warp; n < p.M; n += 32) {
    float m = kLow, s = 0.f;
#pragma unroll 8
    for (int b = lane; b < p.blocks; b += 32) join(m, s, p.part_m[b * SKINNY_ROWS + n], p.part_s[b * SKINNY_ROWS + n]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) join(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    if (lane == 0) {
      const int64_t t = p.t[n];
      float loss = 0.f;
      if (t != p.ignore) {
        const bool good = t >= 0 && t < p.V;
        loss = good ? kLn2 * (fmaf(-p.zt[n], kLog2e, m) + log2f(s)) : __int_as_float(0x7fc00000);
        if (!good) report_status(p.status, PNFT_DEV_BAD_INDEX);
      }
      losses[n] = loss, counted[n] = t != p.ignore;
      if (p.row_loss) p.row_loss[n] = loss;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && p.loss) {
    double sum = 0.0;
    int c = 0;
    for (int n = 0; n < p.M; ++n) sum += losses[n], c += counted[n];
    *p.loss = (float)(p.mean ? sum / (double)c : sum);
  }
}

// ------------------------------------------------------------------ backward
// The rows' factors: row i's gradient is multiplied by alpha * rs[i]. rs reaches from
// -top to top with top 1 for bf16; 2^14 for fp16, so that the small probabilities of a
// large vocabulary stay inside fp16's range whatever the loss's own factor is.
struct ScaleArgs {
  State s;
  const float* dloss;  // scalar, or [M] with stride `stride`
  int64_t stride;
  float *rs, *alpha;
  int per_row, mean;
  float top;
};
__global__ void __launch_bounds__(1024) xent_scale_kernel(ScaleArgs p) {
  __shared__ float red[32];
  launch_next();
  wait_previous();
  const int n = p.s.counts[0];
  if (!p.per_row) {
    for (int i = threadIdx.x; i < n; i += 1024) p.rs[i] = p.top;
    if (threadIdx.x == 0) *p.alpha = n == 0 ? 0.f : *p.dloss / (p.mean ? (float)n : 1.f) / p.top;
    return;
  }
  float m = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float v = fabsf(p.dloss[p.s.idx[i] * p.stride]);
    m = v < INFINITY ? fmaxf(m, v) : m;  // an infinite or NaN factor stays its own row's
  }
  m = group_max<32>(m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = group_max<32>(red[threadIdx.x & 31]);
  if (!(m > 0.f)) m = 1.f;  // all zero, or none finite
  for (int i = threadIdx.x; i < n; i += 1024) p.rs[i] = p.dloss[p.s.idx[i] * p.stride] / m * p.top;
  if (threadIdx.x == 0) *p.alpha = m / p.top;
}

// dz of one piece, 16 bits, zeros in rows past the last one that counts and in columns
// past the vocabulary (the two GEMMs run over whole 64-deep blocks of both).
struct DzEpi {
  static constexpr int WARPS = 16, BOXES = 1, BOX_BYTES = 4096;
  static constexpr bool PING_PONG = false;
  struct Params {
    Out dz;
    const float *lse2, *rs;
    const int32_t *tgt, *live;
    int v0, V, bf16;
  };
  const Params& p;
  EpiWarp w;
  Boxes<BOXES> boxes;
  float lse, rs;
  int tgt, live;
  __device__ DzEpi(const Params& p_, const EpiWarp& w_, const Abort&) : p(p_), w(w_), boxes(w) { live = *p.live; }
  __device__ void prepare(const Steps& q) {
    if (!q.item_first()) return;
    const int row = q.it.row0 + w.row();
    lse = row < live ? p.lse2[row] : 0.f;
    rs = row < live ? p.rs[row] : 0.f;
    tgt = row < live ? p.tgt[row] - p.v0 : -1;
  }
  __device__ void end(const Steps&) {}
  __device__ void done() { boxes.finish(); }
  template <class Release>
  __device__ __forceinline__ void tile(const Steps& q, uint32_t acc, Release release) {
    const int row = q.it.row0 + w.row();
    uint32_t b = 0;
#pragma unroll 1
    for (int c = w.slice * (BN / 4); c < (w.slice + 1) * (BN / 4); c += 32) {
      float z[32];
      acc_load32(acc + c, false, z);
      if (c + 32 == (w.slice + 1) * (BN / 4)) release();
      const int col = q.nt * BN + c, n = row < live ? p.V - p.v0 - col : 0, tc = tgt - col;
      const f32x2 scale = pack(kLog2e, kLog2e), minus = pack(-lse, -lse), factor = pack(rs, rs);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const f32x2 x = fma2(pack(z[2 * i], z[2 * i + 1]), scale, minus);
        const float2 v = unpack(mul2(exp2_pair(x), factor));
        z[2 * i] = v.x, z[2 * i + 1] = v.y;
      }
      if ((unsigned)tc < 32u) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i == tc) z[i] -= rs;
      }
      if (n < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i >= n) z[i] = 0.f;
      }
      const int h = (c >> 5) & 1;
      if (h == 0) b = boxes.take();
      boxes.put16(b, 32 * h, z, p.bf16);
      if (h == 1 && q.it.row0 < p.dz.rows) boxes.store(b, &p.dz.map, col - 32, q.it.row0 + 32 * w.quad, 0);
    }
  }
};

// dh[r] = alpha * acc[compacted row of r], 0 for rows that do not count.
__global__ void __launch_bounds__(256) xent_dh_kernel(const float* acc, int64_t lda, const int32_t* pos, const float* alpha,
                                                      void* dh, int64_t lddh, int dtype, int64_t M, int D, int vec) {
  launch_next();
  wait_previous();
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < M; r += (int64_t)gridDim.x * 8) {
    const int at = pos[r];
    const float a = at >= 0 ? *alpha : 0.f;  // alpha may be infinite or NaN
    for (int c0 = 4 * lane; c0 < D; c0 += 512) {  // four loads in flight before the first store
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = c0 + 128 * k;
        v[k] = at >= 0 && c < D ? *reinterpret_cast<const float4*>(acc + at * lda + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = c0 + 128 * k;
        const float f[4] = {v[k].x * a, v[k].y * a, v[k].z * a, v[k].w * a};
        if (c < D) store_row4(dh, r * lddh + c, f, D - c, dtype, vec);
      }
    }
  }
}

// ------------------------------------------------------------------ plans
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// What the backward needs: the rows that count (16-byte aligned, whole row tiles) and
// their state.
struct SavedLayout {
  int64_t ldc;
  size_t hc, counts, pos, idx, tgt, lse2, total;
};
SavedLayout saved_layout(int64_t M, int64_t D) {
  const int64_t Mp = up(std::max<int64_t>(M, 1), BM);
  SavedLayout l;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  l.ldc = up(D, 8);
  l.hc = take(2 * (size_t)Mp * l.ldc);
  l.counts = take(8);
  l.pos = take(4 * Mp);
  l.idx = take(4 * Mp);
  l.tgt = take(4 * Mp);
  l.lse2 = take(4 * Mp);
  l.total = at;
  return l;
}
State state_of(const SavedLayout& l, void* saved) {
  char* b = static_cast<char*>(saved);
  return State{reinterpret_cast<int32_t*>(b + l.counts), reinterpret_cast<int32_t*>(b + l.pos),
               reinterpret_cast<int32_t*>(b + l.idx), reinterpret_cast<int32_t*>(b + l.tgt),
               reinterpret_cast<float*>(b + l.lse2)};
}

struct FwdLayout {
  int runs, pairs, tiles_n;
  size_t zt, part_m, part_s, sums, total;
};
FwdLayout fwd_layout(int64_t M, int64_t V, int64_t D) {
  const int64_t Mp = up(M, BM), tiles_m = (M + PM - 1) / PM;
  FwdLayout l;
  Sched s = plain_sched(M, V, 1, 1);
  runs_if_resident(&s, V, D);
  l.runs = s.runs;
  l.tiles_n = (int)((V + BN - 1) / BN);
  l.pairs = pairs_of(tiles_m * l.tiles_n);
  // a row tile lies in at most pairs / row tiles + 2 runs, or has 4 pairs / row tiles strips (at least
  // one), for any number of rows that count
  const size_t parts = 4 * PM * (size_t)(l.runs ? l.pairs + 2 * tiles_m : 4 * l.pairs + tiles_m);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  l.zt = take(4 * Mp);
  l.part_m = take(4 * parts);
  l.part_s = take(4 * parts);
  l.sums = take(8 * std::max<int64_t>(64, (M + 7) / 8));
  l.total = at;
  return l;
}

// Columns per piece: its gradient buffer takes at most 288 MB (at least 1024 columns), and
// the pieces are alike. Measured (B200, 16352 x 33278 x 256, bf16, kernels of forward and
// backward): 64 MB, which the two products find in L2, 1433 us; 128 MB 1334; 192 MB 1223;
// 272 MB 1166: fewer launches and longer sums are worth more than L2.
int64_t piece_width(int64_t M, int64_t V) {
  const int64_t Mp = up(M, BM);
  const int64_t most = std::max<int64_t>(1024, ((int64_t)288 << 20) / (2 * Mp) / BN * BN);
  const int64_t pieces = (V + most - 1) / most;
  return up((V + pieces - 1) / pieces, BN);
}
// K blocks that the forward leaves to one accumulator. With 8, 16, 32 and all (B200): 8192 x 10000 x 2048 252, 240,
// 231, 231 us; relative error of losses over positive products of width 4096 3.2e-7, 8.2e-7, 2.2e-6, 7.3e-6.
constexpr int LSE_KB = 16;
constexpr int FUSED_WIDTH = 256;  // up to this width dz and dh come from one kernel
struct BwdLayout {
  int64_t P;
  int dh_splits;
  size_t rs, alpha, dz, acc, part, total;
};
// Shares of dh that the fused kernel leaves: one per row tile and run that meet.
int64_t dh_shares(int64_t M, int64_t P) {
  const int64_t tiles_m = (M + PM - 1) / PM;
  return tiles_m + pairs_of(tiles_m * (P / BN));
}
BwdLayout bwd_layout(int64_t M, int64_t V, int64_t D) {
  const int64_t Mp = up(M, BM), D4 = up(D, 4);
  BwdLayout l;
  l.P = piece_width(M, V);
  // few tiles: two rounds, which become one where half of the rows count (one, two and three rounds, B200: 512 x 50021
  // x 776 with half of the rows ignored 134, 126, 132 us, 300 x 20001 x 1024 93, 91, 95)
  l.dh_splits = plan_splits(tiles_of(M, D), l.P / BK, 4 * tiles_of(M, D) <= sm_count() / 2 ? 2 : 1);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  l.rs = take(4 * Mp);
  l.alpha = take(4);
  l.dz = take(2 * (size_t)Mp * l.P);
  l.acc = take(4 * (size_t)Mp * D4);
  const size_t a = D <= FUSED_WIDTH ? 4 * (size_t)dh_shares(M, l.P) * PM * D4 : l.dh_splits > 1 ? 4 * (size_t)l.dh_splits * Mp * D4 : 0;
  const size_t b = std::max(product_workspace(l.P, D, Mp / BK), product_workspace((V - 1) % l.P + 1, D, Mp / BK));
  l.part = take(std::max(a, b));  // the shares are joined before the splits of dW are written
  l.total = at;
  return l;
}

template <int NB>
int launch_dzdh(const DzDhArgs& f, int pairs, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel has its shared memory
  const uint64_t bit = 1ull << (current_device() & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(xent_dzdh_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
      return check_launch("stream_xent dz and dh", 0);
    ready.fetch_or(bit, std::memory_order_release);
  }
  launch_dependent(xent_dzdh_kernel<NB>, dim3((unsigned)(2 * pairs)), 32 * (2 + DZDH_WARPS), SMEM, st, f);
  return check_launch("stream_xent dz and dh", 1);
}

int xent_check(const char* what, int64_t M, int64_t D, int64_t V, int dtype) {
  if (M < 0 || D <= 0 || V <= 0 || M >= ((int64_t)1 << 31) - 256 || D > (1 << 24) || V >= ((int64_t)1 << 31) - 2 * BN)
    return fail(PNFT_EINVAL, "%s: bad shape M=%lld D=%lld V=%lld", what, (long long)M, (long long)D, (long long)V);
  if (!type16(dtype)) return fail(PNFT_EUNSUPPORTED, "%s: bfloat16 or float16 expected", what);
  return PNFT_OK;
}

}  // namespace
}  // namespace pnft

using namespace pnft;
using namespace pnft::tc;

extern "C" size_t pnft_stream_xent_saved_size(int64_t M, int64_t D) {
  return M <= 0 || D <= 0 ? 0 : saved_layout(M, D).total;
}

// Blocks of the kernel for a few rows: 16 words per warp, at most four blocks per SM.
static int skinny_blocks(int64_t V) {
  return (int)std::min<int64_t>((V + 16 * skinny::WARPS - 1) / (16 * skinny::WARPS), 4 * (int64_t)sm_count());
}

extern "C" size_t pnft_stream_xent_fwd_workspace_size(int64_t M, int64_t V, int64_t D, int save) {
  if (M <= 0 || V <= 0 || D <= 0) return 0;
  if (!save && M <= SKINNY_ROWS) return sizeof(float) * SKINNY_ROWS * (2 * (size_t)skinny_blocks(V) + 1);
  return fwd_layout(M, V, D).total + (save ? 0 : saved_layout(M, D).total);
}

extern "C" size_t pnft_stream_xent_bwd_workspace_size(int64_t M, int64_t V, int64_t D) {
  return M <= 0 || V <= 0 || D <= 0 ? 0 : bwd_layout(M, V, D).total;
}

extern "C" int pnft_stream_xent_fwd(const void* h, int64_t ldh, const void* w, int64_t ldw, const int64_t* targets,
                                    int64_t ignore_index, void* saved, float* row_loss, float* loss, int mean,
                                    void* workspace, size_t workspace_bytes, int64_t M, int64_t V, int64_t D, int dtype,
                                    int32_t* status, void* stream) {
  if (int rc = xent_check("stream_xent_fwd", M, D, V, dtype)) return rc;
  if (!row_loss && !loss) return fail(PNFT_EINVAL, "stream_xent_fwd: null output");
  if (M == 0) return fail(PNFT_EINVAL, "stream_xent_fwd: no rows");
  if (!h || !w || !targets) return fail(PNFT_EINVAL, "stream_xent_fwd: null pointer");
  if (ldh < D || ldw < D) return fail(PNFT_EINVAL, "stream_xent_fwd: row stride below the width");
  if (reinterpret_cast<uintptr_t>(saved) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(PNFT_EINVAL, "stream_xent_fwd: buffers must be 16-byte aligned");
  const size_t need = pnft_stream_xent_fwd_workspace_size(M, V, D, saved != nullptr);
  if (!workspace || workspace_bytes < need)
    return fail(PNFT_EINVAL, "stream_xent_fwd: workspace of %zu bytes < required %zu", workspace_bytes, need);
  char* ws = static_cast<char*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (!saved && M <= SKINNY_ROWS) {
    const int blocks = skinny_blocks(V);
    float* part = static_cast<float*>(workspace);
    const SkinnyArgs a{static_cast<const uint16_t*>(h), static_cast<const uint16_t*>(w), ldh, ldw, targets, ignore_index, part,
                       part + (size_t)blocks * SKINNY_ROWS, part + 2 * (size_t)blocks * SKINNY_ROWS, row_loss, loss,
                       (int)M, (int)D, (int)V, blocks, mean, status};
    const bool vec = D % 8 == 0 && rows16(h, ldh, 2) && rows16(w, ldw, 2);
    return skinny::dispatch<SKINNY_ROWS / 8>(M, vec, dtype == PNFT_DTYPE_BF16, [&](auto nt, auto v, auto b) {
      launch_dependent(xent_skinny_kernel<decltype(nt)::value, decltype(v)::value, decltype(b)::value>, dim3((unsigned)blocks),
                       32 * skinny::WARPS, 0, st, a);
      launch_dependent(xent_skinny_reduce_kernel, dim3(1), 1024, 0, st, a);
      return check_launch("stream_xent_fwd", 2);
    });
  }
  if (!tma_rows_ok(w, ldw, D))
    return fail(PNFT_EUNSUPPORTED, "stream_xent_fwd: weight rows must be 16-byte aligned (strides multiples of 8)");
  if (!device_is_sm100()) return fail(PNFT_EUNSUPPORTED, "stream_xent_fwd: needs an sm_100 device");
  const FwdLayout l = fwd_layout(M, V, D);
  const SavedLayout sl = saved_layout(M, D);
  if (!saved) saved = ws + l.total;
  const int64_t Mp = up(M, BM), ldc = sl.ldc;
  char* hc = static_cast<char*>(saved) + sl.hc;
  CompactArgs c;
  memset(&c, 0, sizeof(c));
  c.t = targets, c.ignore = ignore_index;
  c.h = static_cast<const uint16_t*>(h), c.ldh = ldh;
  c.hc = reinterpret_cast<uint16_t*>(hc), c.ldc = ldc;
  c.s = state_of(sl, saved);
  c.zt = reinterpret_cast<float*>(ws + l.zt);
  c.row_loss = row_loss;
  c.M = M, c.V = (int)V, c.D = (int)D, c.Mp = Mp;
  c.rows = (int)std::max<int64_t>(8, (M + 511) / 512);
  c.vec = rows16(h, ldh, 2);
  c.status = status;
  launch_dependent(xent_compact_kernel, dim3((unsigned)((M + c.rows - 1) / c.rows)), CT, 0, st, c);
  int rc = check_launch("stream_xent compaction", 1);
  if (rc) return rc;

  Args a;
  memset(&a, 0, sizeof(a));
  rc = map_kmajor(&a.ta[0], hc, D, Mp, ldc);
  if (!rc) rc = map_kmajor(&a.tb[0], w, D, V, ldw);
  if (rc) return rc;
  a.s = plain_sched(M, V, (D + BK - 1) / BK, 1);
  a.s.runs = l.runs;
  a.s.strips = 0;
  a.s.live = c.s.counts;
  a.s.live_m = 1;
  a.idesc = idesc(dtype, false, false);
  a.status = status;
  float *part_m = reinterpret_cast<float*>(ws + l.part_m), *part_s = reinterpret_cast<float*>(ws + l.part_s);
  auto run = [&](auto promote) {
    typename LseEpi<decltype(promote)::value>::Params ep{part_m, part_s, c.zt, c.s.tgt, c.s.counts, (int)V};
    return launch<false, false, false, LseEpi<decltype(promote)::value>>("stream_xent forward", a, ep, st);
  };
  const int chunks = (a.s.kb + LSE_KB - 1) / LSE_KB;
  a.s.chunk = (a.s.kb + chunks - 1) / chunks;
  rc = chunks > 1 ? run(std::true_type()) : run(std::false_type());
  if (rc) return rc;
  ReduceArgs r{part_m, part_s, c.zt, c.s, row_loss, loss, reinterpret_cast<double*>(ws + l.sums),
               l.runs, l.tiles_n, l.pairs, mean};
  if (M > 64)
    launch_dependent(xent_reduce_kernel<8>, dim3((unsigned)((M + 7) / 8)), 256, 0, st, r);
  else
    launch_dependent(xent_reduce_kernel<1>, dim3((unsigned)M), 256, 0, st, r);
  return check_launch("stream_xent reduction", 1);
}

extern "C" int pnft_stream_xent_bwd(const void* w, int64_t ldw, const void* saved, const float* dloss, int64_t dloss_stride,
                                    int per_row, int mean, void* dh, int64_t lddh, int dh_dtype, void* dw, int64_t lddw, int dw_dtype, void* workspace,
                                    size_t workspace_bytes, int64_t M, int64_t V, int64_t D, int dtype, int32_t* status,
                                    void* stream) {
  if (int rc = xent_check("stream_xent_bwd", M, D, V, dtype)) return rc;
  if (M == 0) return fail(PNFT_EINVAL, "stream_xent_bwd: no rows");
  if (!w || !saved || !dloss || (!dh && !dw)) return fail(PNFT_EINVAL, "stream_xent_bwd: null pointer");
  if (!tma_rows_ok(w, ldw, D) || reinterpret_cast<uintptr_t>(saved) % 16)
    return fail(PNFT_EUNSUPPORTED, "stream_xent_bwd: weight rows must be 16-byte aligned (strides multiples of 8)");
  if ((dh && lddh < D) || (dw && lddw < D)) return fail(PNFT_EINVAL, "stream_xent_bwd: row stride below the width");
  for (int t : {dh_dtype, dw_dtype})
    if (t < PNFT_DTYPE_F32 || t > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "stream_xent_bwd: unknown output type %d", t);
  const BwdLayout l = bwd_layout(M, V, D);
  if (!workspace || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(PNFT_EINVAL, "stream_xent_bwd: workspace of %zu bytes < required %zu (16-byte aligned)", workspace_bytes, l.total);
  if (!device_is_sm100()) return fail(PNFT_EUNSUPPORTED, "stream_xent_bwd: needs an sm_100 device");
  const int64_t Mp = up(M, BM), D4 = up(D, 4);
  char* ws = static_cast<char*>(workspace);
  cudaStream_t st = as_stream(stream);
  const SavedLayout sl = saved_layout(M, D);
  const State s = state_of(sl, const_cast<void*>(saved));
  const int64_t ldc = sl.ldc;
  const char* hc = static_cast<const char*>(saved) + sl.hc;
  float* rs = reinterpret_cast<float*>(ws + l.rs);
  float* alpha = reinterpret_cast<float*>(ws + l.alpha);
  uint16_t* dz = reinterpret_cast<uint16_t*>(ws + l.dz);
  float* acc = reinterpret_cast<float*>(ws + l.acc);
  float* part = reinterpret_cast<float*>(ws + l.part);
  const bool bf16 = dtype == PNFT_DTYPE_BF16;
  launch_dependent(xent_scale_kernel, dim3(1), 1024, 0, st,
                   ScaleArgs{s, dloss, dloss_stride, rs, alpha, per_row, mean, bf16 ? 1.f : 16384.f});
  int rc = check_launch("stream_xent scale", 1);
  for (int64_t v0 = 0; !rc && v0 < V; v0 += l.P) {
    const int64_t n = std::min(l.P, V - v0);
    const uint16_t* wp = static_cast<const uint16_t*>(w) + v0 * ldw;
    Args a;
    memset(&a, 0, sizeof(a));
    a.status = status;
    if (dh && D <= FUSED_WIDTH) {  // dz and dh of the piece
      const int tiles_n = (int)((n + BN - 1) / BN), kd = (int)((D + BK - 1) / BK), nb = D <= 128 ? 64 : 128;
      DzDhArgs f;
      memset(&f, 0, sizeof(f));
      f.s = plain_sched(M, n, kd, 1);
      f.s.runs = 1;
      f.s.live = s.counts;
      f.s.live_m = 1;
      const int pairs = pairs_of((int64_t)f.s.tiles_m * tiles_n);
      rc = tma_map_rows(&f.th, hc, D, Mp, ldc, BM);
      if (!rc) rc = tma_map_rows(&f.tw1, wp, D, n, ldw, BM);
      if (!rc) rc = tma_map_rows(&f.tw2, wp, D, n, ldw, BK);
      if (!rc) rc = tma_map_out(&f.tdz, dz, 2, l.P, Mp, l.P, 1, 0, 32);
      if (!rc) rc = tma_map_out(&f.tpart, part, 4, D, PM, D4, f.s.tiles_m + pairs, PM * D4, 32);
      if (rc) break;
      f.lse2 = s.lse2, f.rs = rs, f.tgt = s.tgt, f.live = s.counts;
      f.v0 = (int)v0, f.V = (int)V, f.D = (int)D, f.Mp = (int)Mp, f.bf16 = bf16, f.store_dz = dw != nullptr;
      f.stages = dzdh_stages(kd);
      f.idesc1 = idesc(dtype, false, false);
      f.idesc2 = idesc_f16(PM, 2 * nb, bf16 ? 1 : 0, 0, 1);
      f.status = status;
      rc = nb == 64 ? launch_dzdh<64>(f, pairs, st) : launch_dzdh<128>(f, pairs, st);
      if (rc) break;
      const JoinArgs j{part, acc, D4, s.counts, s.pos, alpha, dh, lddh, M, (int)D, dh_dtype, tiles_n, pairs, v0 == 0, v0 + l.P >= V,
                       rows16(dh, lddh, dtype_size(dh_dtype))};
      launch_dependent(xent_join_kernel, dim3((unsigned)std::min<int64_t>((M + 7) / 8, (int64_t)sm_count() * 16)), 256, 0, st, j);
      rc = check_launch("stream_xent dh rows", 1);
      if (rc) break;
    } else {
    // dz of the piece
    rc = map_kmajor(&a.ta[0], hc, D, Mp, ldc);
    if (!rc) rc = map_kmajor(&a.tb[0], wp, D, n, ldw);
    if (rc) break;
    a.s = plain_sched(M, n, (D + BK - 1) / BK, 1);
    runs_if_resident(&a.s, n, D);
    a.s.live = s.counts;
    a.s.live_m = 1;
    a.idesc = idesc(dtype, false, false);
    DzEpi::Params ep;
    memset(&ep, 0, sizeof(ep));
    rc = make_out(&ep.dz, dz, dtype, l.P, Mp, l.P);
    if (rc) break;
    ep.lse2 = s.lse2, ep.rs = rs, ep.tgt = s.tgt, ep.live = s.counts;
    ep.v0 = (int)v0, ep.V = (int)V, ep.bf16 = bf16;
    rc = launch<false, false, false, DzEpi>("stream_xent dz", a, ep, st);
    if (rc) break;
    if (dh) {  // dh (+)= dz W
      rc = map_kmajor(&a.ta[0], dz, n, Mp, l.P);
      if (!rc) rc = map_mnmajor(&a.tb[0], wp, D, n, ldw);
      if (rc) break;
      const int kb = (int)((n + BK - 1) / BK), splits = std::min(l.dh_splits, std::max(1, kb / 8));
      a.s = plain_sched(M, D, kb, splits);
      a.s.live = s.counts;
      a.s.live_m = 1;
      a.idesc = idesc(dtype, false, true);
      StoreEpi<false>::Params out;
      memset(&out, 0, sizeof(out));
      out.row_split = 0x7fffffff;
      out.dtype = PNFT_DTYPE_F32;
      if (splits > 1) {
        rc = make_out(&out.c[0], part, PNFT_DTYPE_F32, D, M, D4, splits, Mp * D4);
        if (!rc) rc = launch_store<false, true>("stream_xent dh", a, out, st);
        const SumArgs sum{{acc, nullptr}, D4, 0x7fffffff, (int)M, (int)D, nullptr, PNFT_DTYPE_F32, v0 > 0, 1};
        if (!rc) rc = sum_splits(part, D4, Mp * D4, splits, sum, (int)M, st);
      } else {
        rc = make_out(&out.c[0], acc, PNFT_DTYPE_F32, D, M, D4);
        out.add = v0 > 0;
        if (!rc) rc = launch_store<false, true>("stream_xent dh", a, out, st);
      }
      if (rc) break;
    }
    }
    if (dw) {  // the piece's rows of dW = dz^T h
      rc = map_mnmajor(&a.ta[0], dz, n, Mp, l.P);
      if (!rc) rc = map_mnmajor(&a.tb[0], hc, D, Mp, ldc);
      if (rc) break;
      a.idesc = idesc(dtype, true, true);
      const int size = dtype_size(dw_dtype);
      void* dst = static_cast<char*>(dw) + v0 * lddw * size;
      const SumArgs c{{dst, nullptr}, lddw, 0x7fffffff, (int)n, (int)D, alpha, dw_dtype, 0, rows16(dst, lddw, size)};
      rc = product<true, true>("stream_xent dW", a, c, part, n, D, Mp / BK, 0, s.counts, st);
    }
  }
  if (rc || !dh || D <= FUSED_WIDTH) return rc;
  launch_dependent(xent_dh_kernel, dim3((unsigned)std::min<int64_t>((M + 7) / 8, (int64_t)sm_count() * 16)), 256, 0, st,
                   (const float*)acc, D4, (const int32_t*)s.pos, (const float*)alpha, dh, lddh, dh_dtype, M, (int)D,
                   (int)rows16(dh, lddh, dtype_size(dh_dtype)));
  return check_launch("stream_xent dh rows", 1);
}
