// The gated feed-forward product of a decoder block and its backward pass:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u          (act: SiLU or erf GELU)
//   dg = dh * u * act'(g),  du = dh * act(g),  dx = dg Wg + du Wu
//
// (the weight gradients dg^T x, du^T x are pnft_weight_grad's). Both projections are
// one GEMM: a 256-column accumulator holds 128 columns of g and the same 128 of u, fed
// from the two weights' tiles with the x tile read once, so the epilogue has both
// values of an element in one thread and g, u never meet in memory unless a backward
// wants them.
//
// The backward has g, u again in one of two ways: computed from x by the same GEMM, whose
// epilogue then reads dh and writes dg, du; or kept by the forward with 24 bits each (the
// upper 16 bits of fp32 in two planes, the next 8 of both in a third: kept in 16 bits,
// their rounding would add as much error to the gradients as the operands' own).
// dg and du themselves are rounded to 16 bits, the operand type of the products that follow;
// with the results' own rounding that gives dx and dW 1.4 times the error of one rounding.
#include "gemm_tc.cuh"
#include "skinny.cuh"

namespace pnft {
namespace {

using namespace tc;

constexpr float kInvSqrt2Pi = 0.39894228040143268f, kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// act(g); deriv: also act'(g). The exponentials and the quotients are the fast ones
// (a few units of 2^-23; results below 2^-126 are 0): the results are rounded to 16 bits.
// GELU's normal distribution: for a = |g| and t = 1 / (1 + 0.3 a)
//   Phi(-a) = exp(-a^2 / 2) t Q(t),
// where t Q(t) stands for exp(a^2 / 2) erfc(a / sqrt 2) / 2, Q the polynomial of degree 7
// with the least relative error on 0 <= a <= 14 (1.5e-7; fitted by reweighted least
// squares). With fp32's rounding the relative error is 2^-20 up to a = 3 and 2^-17 where
// Phi(-a) ends, so the far negative side keeps its digits; Phi(a) = 1 - Phi(-a). It shares
// its exponential with the derivative (B200, 4095 x 1000 x 2731 with biases: the forward kernel
// 55 us and the backward one 57, 61 and 64 with erfcf).
template <bool DERIV, int ACT>
__device__ __forceinline__ float act_value(float g, float* deriv) {
  if (ACT == PNFT_ACT_SILU) {
    const float s = fast_rcp(1.f + fast_ex2(-kLog2e * g));
    if (DERIV) *deriv = s * (1.f + g * (1.f - s));
    return g * s;
  }
  const float a = fabsf(g), t = fast_rcp(fmaf(0.3f, a, 1.f)), e = fast_ex2(-0.5f * kLog2e * a * a);
  float q = 0.0356748118f;
  q = fmaf(q, t, -0.157203222f);
  q = fmaf(q, t, 0.206353707f);
  q = fmaf(q, t, -0.0536837867f);
  q = fmaf(q, t, 0.128561677f);
  q = fmaf(q, t, 0.0999134846f);
  q = fmaf(q, t, 0.120753956f);
  q = fmaf(q, t, 0.119629299f);
  const float tail = q * t * e, cdf = g < 0.f ? tail : 1.f - tail;
  if (DERIV) *deriv = cdf + g * (kInvSqrt2Pi * e);
  return g * cdf;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == PNFT_DTYPE_F32) return static_cast<const float*>(p)[i];
  return load16(static_cast<const uint16_t*>(p) + i, dtype == PNFT_DTYPE_BF16);
}

// W values of a bias vector from column `col` (a multiple of 16), `n` of them inside.
template <int W>
__device__ __forceinline__ void add_bias(float (&v)[W], const void* bias, int dtype, int col, int n) {
  if (n >= W && reinterpret_cast<uintptr_t>(bias) % 16 == 0) {
    if (dtype == PNFT_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(bias) + col + i);
        v[i] += f.x, v[i + 1] += f.y, v[i + 2] += f.z, v[i + 3] += f.w;
      }
    } else {
      float b[W];
      load_row16<W>(static_cast<const uint16_t*>(bias) + col, b, W, true, dtype == PNFT_DTYPE_BF16);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] += b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < n) v[i] += load_any(bias, col + i, dtype);
  }
}

// Sums of 16 values of every lane over the warp: lanes 2 k and 2 k + 1 return value k's, in
// an order that depends on the lanes alone.
__device__ __forceinline__ float column_sums(const float (&x)[16], int lane) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = x[i];
#pragma unroll
  for (int n = 8; n > 0; n /= 2) {  // a lane hands half of its values to the lane 2 n away
    const bool upper = lane & (2 * n);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + n], 2 * n);
      v[i] = (upper ? v[i + n] : v[i]) + other;
    }
  }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

// FWD: h. KEEP: h and the three planes of g, u. BWD: dg, du from dh and the recomputed g, u.
// A warp has 32 columns of g and of u of a tile, and takes them 16 at a time (96 registers).
enum { FWD, KEEP, BWD };
template <int MODE, int ACT>
struct GatedEpi {
  static constexpr bool PING_PONG = false;
  static constexpr int WARPS = 16, W = 32, ROW_BYTES = 2 * W;
  static constexpr int OUTS = MODE == KEEP ? 3 : 2;                                       // boxes for results
  static constexpr int BOXES = OUTS + (MODE == BWD), BOX_BYTES = 32 * ROW_BYTES;          // and one for dh
  struct Params {
    const void *bg, *bu;
    int b_dtype, bf16;
    Out h;            // FWD, KEEP: h; BWD: dg
    Out k;            // KEEP: the planes; BWD: du
    CUtensorMap dh;   // BWD
    float* sums;      // BWD: [32-row blocks][2][columns] sums of dg and du for the biases, or NULL
  };
  const Params& p;
  EpiWarp w;
  const Abort& ab;
  Boxes<OUTS, ROW_BYTES> boxes;
  int phase, issued;
  __device__ GatedEpi(const Params& p_, const EpiWarp& w_, const Abort& ab_)
      : p(p_), w(w_), ab(ab_), boxes(EpiWarp{w_.quad, w_.group, w_.slice, w_.lane, w_.smem + (MODE == BWD ? BOX_BYTES : 0), w_.bar}),
        phase(0), issued(0) {}
  __device__ int col0(const Steps& q) const { return q.nt * (BN / 2) + w.slice * W; }
  __device__ void end(const Steps&) {}
  __device__ void load_dh(const Steps& q) {
    if (w.lane == 0) {
      mbar_arrive_expect_tx(w.bar, BOX_BYTES);
      tma_load_3d(w.smem, &p.dh, w.bar, col0(q), q.it.row0 + 32 * w.quad, 0);
    }
    ++issued;
  }
  __device__ void prepare(const Steps& q) {
    if (MODE == BWD && issued == 0) load_dh(q);
  }
  __device__ void done() {
    if (MODE == BWD && issued > phase) drain_wait(w.bar, phase & 1);  // an abandoned tile's dh
    boxes.finish();
  }
  __device__ __forceinline__ void write(const Out& o, uint32_t b, int row, int col, int z) {
    if (o.tma)
      boxes.store(b, &o.map, col, row, z);
    else
      boxes.template store_plain<2>(b, static_cast<uint16_t*>(o.base) + (int64_t)row * o.ld + col, o.ld, o.rows - row,
                                    o.cols - col);
  }
  template <class Release>
  __device__ __forceinline__ void tile(const Steps& q, uint32_t acc, Release release) {
    const int row = q.it.row0 + 32 * w.quad, col = col0(q);
    const bool live = row < p.h.rows && col < p.h.cols, bf16 = p.bf16;
    if (MODE == BWD) {
      if (!warp_wait(w.bar, phase & 1, ab)) return;
      ++phase;
    }
    uint32_t b[OUTS];
    uint4 low[MODE == KEEP ? W / 8 : 1];
    if (live) {
      if (MODE == FWD)
        b[0] = boxes.take();
      else
        boxes.take_all(b);
    }
#pragma unroll
    for (int c = 0; c < W; c += 16) {
      float g[16], u[16];
      {
        uint32_t rg[16], ru[16];
        tmem_load16x2(acc + w.slice * W + c, rg, acc + BN / 2 + w.slice * W + c, ru);
        if (c + 16 == W) release();
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = __uint_as_float(rg[i]), u[i] = __uint_as_float(ru[i]);
      }
      const int n = p.h.cols - col - c;
      if (p.bg) add_bias<16>(g, p.bg, p.b_dtype, col + c, n);
      if (p.bu) add_bias<16>(u, p.bu, p.b_dtype, col + c, n);
      if (MODE == BWD) {
        float d[16];
        boxes.get16(w.smem, c, d, bf16);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float da;
          const float a = act_value<true, ACT>(g[i], &da);
          g[i] = d[i] * u[i] * da;
          u[i] = d[i] * a;
        }
        if (c + 16 == W) {  // dh's box has been read: the next tile's may come
          __syncwarp();
          Steps next = q;
          next.next();
          if (next.valid()) load_dh(next);
        }
        if (!live) continue;
        if (p.sums) {  // before the rounding to 16 bits
          const bool in = row + w.lane < p.h.rows;
          float s[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = in ? g[i] : 0.f;
          const float sg = column_sums(s, w.lane);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = in ? u[i] : 0.f;
          const float su = column_sums(s, w.lane);
          if (w.lane / 2 < n) {
            float* at = p.sums + (int64_t)(row / 32) * 2 * p.h.cols + col + c + w.lane / 2;
            at[w.lane & 1 ? p.h.cols : 0] = w.lane & 1 ? su : sg;
          }
        }
        boxes.put16(b[0], c, g, bf16);
        boxes.put16(b[OUTS - 1], c, u, bf16);
      } else {
        if (!live) continue;
        if (MODE == KEEP) {
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            uint32_t x[4], y[4], z[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t g0 = __float_as_uint(g[i + 2 * k]), g1 = __float_as_uint(g[i + 2 * k + 1]);
              const uint32_t u0 = __float_as_uint(u[i + 2 * k]), u1 = __float_as_uint(u[i + 2 * k + 1]);
              x[k] = __byte_perm(g0, g1, 0x7632);  // the upper halves of g
              y[k] = __byte_perm(u0, u1, 0x7632);  // and of u
              z[k] = __byte_perm(__byte_perm(g0, u0, 0x0051), __byte_perm(g1, u1, 0x0051), 0x5410);  // the bytes below
            }
            boxes.put(b[OUTS - 2], (c + i) / 8, x[0], x[1], x[2], x[3]);
            boxes.put(b[OUTS - 1], (c + i) / 8, y[0], y[1], y[2], y[3]);
            low[(c + i) / 8] = make_uint4(z[0], z[1], z[2], z[3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = act_value<false, ACT>(g[i], nullptr) * u[i];
        boxes.put16(b[0], c, g, bf16);
      }
    }
    if (!live) return;
    write(p.h, b[0], row, col, 0);
    if (MODE == BWD) write(p.k, b[OUTS - 1], row, col, 0);
    if (MODE == KEEP) {
      write(p.k, b[OUTS - 2], row, col, 0);
      write(p.k, b[OUTS - 1], row, col, 1);
      const uint32_t z = p.h.tma ? boxes.take() : b[0];  // h's box again, once its store has read it
#pragma unroll
      for (int i = 0; i < W / 8; ++i) boxes.put(z, i, low[i].x, low[i].y, low[i].z, low[i].w);
      boxes.store(z, &p.k.map, col, row, 2);
    }
  }
};

// ------------------------------------------------------------------ a few rows
// From 33 rows on the tiles win (B200, bf16, cold L2: 1024 x 4096 weights 9.3 us here at 32
// rows and 13.7 in tiles, 4096 x 16384 74 and 67; at one row 6.8 and 13.7, 51 and 67).
constexpr int SKINNY_ROWS = PNFT_GATED_FEW_ROWS;
// Forward for few rows: a block has 16 columns of h; each of its warps takes an
// eighth of K of the products of x with those rows of Wg and of Wu.
struct SkinnyArgs {
  const uint16_t *x, *wg, *wu;
  int64_t ldx, ldwg, ldwu;
  const void *bg, *bu;
  int b_dtype, act;
  uint16_t* h;
  int64_t ldh;
  int M, D, F;
};
template <int NT, bool VEC, bool BF16>
__global__ void __launch_bounds__(32 * skinny::WARPS, 2) gated_skinny_kernel(SkinnyArgs p) {
  launch_next();
  wait_previous();
  constexpr int N = 8 * NT;
  __shared__ float red[skinny::WARPS / 2][2][16][N + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int f0 = blockIdx.x * 16;
  // rows past F read the last one; their columns are not written
  const int64_t r0 = min(f0 + g, p.F - 1), r1 = min(f0 + g + 8, p.F - 1);
  const uint16_t* const w[4] = {p.wg + r0 * p.ldwg, p.wg + r1 * p.ldwg, p.wu + r0 * p.ldwu, p.wu + r1 * p.ldwu};
  float acc[2][NT][4] = {};
  skinny::dot<false, 2, NT, VEC, BF16>(w, p.x, p.ldx, p.M, p.D, warp, skinny::WARPS, acc);
  // the upper warps' parts are added to the lower ones', which keep shared memory small
  for (int half = 1; half >= 0; --half) {
    if ((warp >> 2) == half) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float& v = red[warp & 3][r][g + 8 * (k >> 1)][8 * j + 2 * t + (k & 1)];
            v = half ? acc[r][j][k] : v + acc[r][j][k];
          }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 16 * p.M; i += 32 * skinny::WARPS) {
    const int f = i & 15, n = i >> 4, col = f0 + f;
    if (col >= p.F) continue;
    float gv = (red[0][0][f][n] + red[1][0][f][n]) + (red[2][0][f][n] + red[3][0][f][n]);
    float uv = (red[0][1][f][n] + red[1][1][f][n]) + (red[2][1][f][n] + red[3][1][f][n]);
    if (p.bg) gv += load_any(p.bg, col, p.b_dtype);
    if (p.bu) uv += load_any(p.bu, col, p.b_dtype);
    const float a = p.act == PNFT_ACT_SILU ? act_value<false, PNFT_ACT_SILU>(gv, nullptr) : act_value<false, PNFT_ACT_GELU>(gv, nullptr);
    store16(p.h + n * p.ldh + col, a * uv, BF16);
  }
}

// ------------------------------------------------------------------ pointwise backward
// dg, du from dh and the kept g, u (their three planes), with the column sums of dg and du
// before their rounding for the biases' gradients. A block takes 8 columns per lane (256 in all) of a run of rows, a warp a row at a time. Bound by
// HBM: 12 bytes per element (B200, 8192 x 8192: 128 us, 6.3 TB/s); the loads of 32 warps per SM keep it busy (16 with two rows each
// reached 3.8 TB/s).
constexpr int PT = 256, PCOLS = 256, PBLOCKS = 4;  // blocks per SM
struct PointArgs {
  const uint16_t* dh;
  int64_t lddh;
  const uint16_t *g, *u, *low;
  int64_t ldp;
  uint16_t *dg, *du;
  int64_t ldd;
  float* part;  // [gridDim.y][2][F] (NULL: no sums)
  int M, F, bf16, rows, vec;
};

// 8 values of g and of u with 24 bits from their upper 16 and the third plane's bytes.
__device__ __forceinline__ void join24(const uint16_t* gp, const uint16_t* up, const uint16_t* lp, int n, float (&g)[8],
                                       float (&u)[8]) {
  uint32_t a[4], b[4], l[4];
  if (n >= 8) {
    const uint4 x = __ldcs(reinterpret_cast<const uint4*>(gp)), y = __ldcs(reinterpret_cast<const uint4*>(up)),
                z = __ldcs(reinterpret_cast<const uint4*>(lp));
    a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w, b[0] = y.x, b[1] = y.y, b[2] = y.z, b[3] = y.w;
    l[0] = z.x, l[1] = z.y, l[2] = z.z, l[3] = z.w;
  } else {
    auto pair = [&](const uint16_t* p, int k) {
      return (2 * k < n ? p[2 * k] : 0u) | (2 * k + 1 < n ? (uint32_t)p[2 * k + 1] << 16 : 0u);
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = pair(gp, k), b[k] = pair(up, k), l[k] = pair(lp, k);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // bytes 3, 2: the upper half; byte 1: the third plane's (g's, or u's above it); byte 0: cleared
    g[2 * k] = __uint_as_float(__byte_perm(a[k], l[k], 0x1040) & 0xffffff00u);
    g[2 * k + 1] = __uint_as_float(__byte_perm(a[k], l[k], 0x3260) & 0xffffff00u);
    u[2 * k] = __uint_as_float(__byte_perm(b[k], l[k], 0x1050) & 0xffffff00u);
    u[2 * k + 1] = __uint_as_float(__byte_perm(b[k], l[k], 0x3270) & 0xffffff00u);
  }
}

template <bool SUMS, int ACT>
__global__ void __launch_bounds__(PT, PBLOCKS) gated_point_kernel(PointArgs p) {
  launch_next();
  wait_previous();
  __shared__ float red[SUMS ? PT / 32 : 1][2][PCOLS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * PCOLS + 8 * lane, n = p.F - col;
  const bool bf16 = p.bf16;
  float sg[8] = {}, su[8] = {};
  const int64_t r0 = (int64_t)blockIdx.y * p.rows, r1 = std::min<int64_t>(p.M, r0 + p.rows);
  if (n > 0) {
#pragma unroll 1
    for (int64_t r = r0 + warp; r < r1; r += PT / 32) {
      float g[8], u[8];
      float d[8];
      join24(p.g + r * p.ldp + col, p.u + r * p.ldp + col, p.low + r * p.ldp + col, n, g, u);
      load_row16<8>(p.dh + r * p.lddh + col, d, n, p.vec, bf16);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float da;
        const float a = act_value<true, ACT>(g[k], &da);
        g[k] = d[k] * u[k] * da;
        u[k] = d[k] * a;
      }
      store_row16<8>(p.dg + r * p.ldd + col, g, n, true, bf16);
      store_row16<8>(p.du + r * p.ldd + col, u, n, true, bf16);
      if (SUMS) {
#pragma unroll
        for (int k = 0; k < 8; ++k) sg[k] += g[k], su[k] += u[k];
      }
    }
  }
  if (!SUMS) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[warp][0][8 * lane + k] = sg[k], red[warp][1][8 * lane + k] = su[k];
  __syncthreads();
  const int c = blockIdx.x * PCOLS + threadIdx.x;
  if (c >= p.F) return;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float t = 0.f;
    for (int k = 0; k < PT / 32; ++k) t += red[k][side][threadIdx.x];
    p.part[((int64_t)blockIdx.y * 2 + side) * p.F + c] = t;
  }
}

// Adds the blocks' column sums: 32 columns per block, eight threads each, in a fixed order.
__global__ void __launch_bounds__(256) gated_bias_sum_kernel(const float* part, int64_t blocks, int F, void* dbg,
                                                             void* dbu, int dtype) {
  __shared__ float red[8][32];
  launch_next();
  wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (i < 2 * F) {
#pragma unroll 8
    for (int64_t b = warp; b < blocks; b += 8) t += part[b * 2 * F + i];
  }
  red[warp][lane] = t;
  __syncthreads();
  if (warp > 0 || i >= 2 * F) return;
  for (int k = 1; k < 8; ++k) t += red[k][lane];
  void* dst = i < F ? dbg : dbu;
  const int c = i < F ? i : i - F;
  if (!dst) return;
  if (dtype == PNFT_DTYPE_F32)
    static_cast<float*>(dst)[c] = t;
  else
    store16(static_cast<uint16_t*>(dst) + c, t, dtype == PNFT_DTYPE_BF16);
}
int bias_sum(const float* part, int64_t blocks, int64_t F, void* dbg, void* dbu, int dtype, cudaStream_t st) {
  launch_dependent(gated_bias_sum_kernel, dim3((unsigned)((2 * F + 31) / 32)), 256, 0, st, part, blocks, (int)F, dbg, dbu, dtype);
  return check_launch("gated_bwd biases", 1);
}

// Rows per block of the pointwise kernel: one wave of PBLOCKS per SM.
int point_rows(int64_t M, int64_t F) {
  const int64_t cols = (F + PCOLS - 1) / PCOLS;
  const int64_t want = std::max<int64_t>(1, PBLOCKS * sm_count() / cols);
  const int64_t rows = std::max<int64_t>(16, (M + want - 1) / want);
  return (int)std::min<int64_t>(std::max<int64_t>(rows, (M + 65534) / 65535), 1 << 30);
}

int gated_check(const char* what, int64_t M, int64_t D, int64_t F, int act, int dtype) {
  if (M < 0 || D <= 0 || F <= 0 || M >= ((int64_t)1 << 31) - 256 || D > (1 << 24) || F > (1 << 24))
    return fail(PNFT_EINVAL, "%s: bad shape M=%lld D=%lld F=%lld", what, (long long)M, (long long)D, (long long)F);
  if (act != PNFT_ACT_SILU && act != PNFT_ACT_GELU) return fail(PNFT_EINVAL, "%s: unknown activation %d", what, act);
  if (!type16(dtype)) return fail(PNFT_EUNSUPPORTED, "%s: bfloat16 or float16 expected", what);
  return PNFT_OK;
}

template <int MODE, int ACT>
int gated_launch(const char* what, const Args& a, const void* bg, const void* bu, int b_dtype, int dtype, const Out& h,
                 const Out& k, const CUtensorMap* dh, float* sums, cudaStream_t st) {
  typename GatedEpi<MODE, ACT>::Params ep;
  memset(&ep, 0, sizeof(ep));
  ep.bg = bg, ep.bu = bu, ep.b_dtype = b_dtype, ep.bf16 = dtype == PNFT_DTYPE_BF16;
  ep.h = h, ep.k = k;
  if (dh) ep.dh = *dh;
  ep.sums = sums;
  return launch<false, false, true, GatedEpi<MODE, ACT>>(what, a, ep, st);
}

int gated_gemm(const char* what, int mode, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
               int64_t ldwu, const void* bg, const void* bu, int b_dtype, const Out& h, const Out& k, const CUtensorMap* dh,
               float* sums, int64_t M, int64_t D, int64_t F, int act, int dtype, int32_t* status, cudaStream_t st) {
  if (b_dtype < PNFT_DTYPE_F32 || b_dtype > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "%s: unknown bias type %d", what, b_dtype);
  Args a;
  memset(&a, 0, sizeof(a));
  int rc = map_kmajor(&a.ta[0], x, D, M, ldx);
  if (!rc) rc = map_kmajor(&a.tb[0], wg, D, F, ldwg);
  if (!rc) rc = map_kmajor(&a.tb[1], wu, D, F, ldwu);
  if (rc) return rc;
  a.s = plain_sched(M, 2 * ((F + BN / 2 - 1) / (BN / 2) * (BN / 2)), (D + BK - 1) / BK, 1);
  runs_if_resident(&a.s, 2 * F, D);
  a.idesc = idesc(dtype, false, false);
  a.status = status;
  auto go = [&](auto m, auto c) {
    return gated_launch<decltype(m)::value, decltype(c)::value>(what, a, bg, bu, b_dtype, dtype, h, k, dh, sums, st);
  };
  auto with_act = [&](auto m) {
    return act == PNFT_ACT_SILU ? go(m, std::integral_constant<int, PNFT_ACT_SILU>()) : go(m, std::integral_constant<int, PNFT_ACT_GELU>());
  };
  if (mode == FWD) return with_act(std::integral_constant<int, FWD>());
  if (mode == KEEP) return with_act(std::integral_constant<int, KEEP>());
  return with_act(std::integral_constant<int, BWD>());
}

int gated_operands(const char* what, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                   int64_t D) {
  if (!tma_rows_ok(x, ldx, D) || !tma_rows_ok(wg, ldwg, D) || !tma_rows_ok(wu, ldwu, D))
    return fail(PNFT_EUNSUPPORTED, "%s: x and weight rows must be 16-byte aligned (strides multiples of 8)", what);
  if (!device_is_sm100()) return fail(PNFT_EUNSUPPORTED, "%s: needs an sm_100 device", what);
  return PNFT_OK;
}

}  // namespace
}  // namespace pnft

using namespace pnft;
using namespace pnft::tc;

extern "C" int pnft_gated_fwd(const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                              const void* bg, const void* bu, int b_dtype, void* h, int64_t ldh, void* pre, int64_t ldp,
                              int64_t M, int64_t D, int64_t F, int act, int dtype, int32_t* status, void* stream) {
  if (int rc = gated_check("gated_fwd", M, D, F, act, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  if (!h) return fail(PNFT_EINVAL, "gated_fwd: null output");
  if (ldh < F || (pre && ldp < F)) return fail(PNFT_EINVAL, "gated_fwd: row strides below the width");
  if (pre && !rows16(pre, ldp, 2)) return fail(PNFT_EINVAL, "gated_fwd: the kept rows must be 16-byte aligned");
  if (b_dtype < PNFT_DTYPE_F32 || b_dtype > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "gated_fwd: unknown bias type %d", b_dtype);
  if (ldx < D || ldwg < D || ldwu < D) return fail(PNFT_EUNSUPPORTED, "gated_fwd: x and weight rows must not overlap (aligned strides of at least D)");
  if (M <= SKINNY_ROWS && !pre && x && wg && wu) {
    const SkinnyArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(wg), static_cast<const uint16_t*>(wu),
                       ldx, ldwg, ldwu, bg, bu, b_dtype, act, static_cast<uint16_t*>(h), ldh, (int)M, (int)D, (int)F};
    const bool vec = D % 8 == 0 && rows16(x, ldx, 2) && rows16(wg, ldwg, 2) && rows16(wu, ldwu, 2);
    return skinny::dispatch<SKINNY_ROWS / 8>(M, vec, dtype == PNFT_DTYPE_BF16, [&](auto nt, auto v, auto b) {
      launch_dependent(gated_skinny_kernel<decltype(nt)::value, decltype(v)::value, decltype(b)::value>,
                       dim3((unsigned)((F + 15) / 16)), 32 * skinny::WARPS, 0, as_stream(stream), a);
      return check_launch("gated_fwd", 1);
    });
  }
  if (int rc = gated_operands("gated_fwd", x, ldx, wg, ldwg, wu, ldwu, D)) return rc;
  Out o, k;
  int rc = make_out(&o, h, dtype, F, M, ldh, 1, 0, 64);
  if (!rc) rc = make_out(&k, pre, dtype, F, M, ldp, 3, M * ldp, 64);
  if (rc) return rc;
  return gated_gemm("gated_fwd", pre ? KEEP : FWD, x, ldx, wg, ldwg, wu, ldwu, bg, bu, b_dtype, o, k, nullptr, nullptr, M, D, F, act,
                    dtype, status, as_stream(stream));
}

namespace {

// Buffers of a backward call: dg, du side by side (each padded to whole row tiles of the
// weight-gradient product), dh with aligned rows where the caller's are not, the biases'
// partial sums, and the partial sums of the two products (one after the other).
struct BwdLayout {
  int64_t Fp;
  size_t d, dh, bias, part, total;
};
BwdLayout bwd_layout(int64_t M, int64_t D, int64_t F) {
  BwdLayout l;
  l.Fp = (F + BM - 1) / BM * BM;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  l.d = take(2 * (size_t)M * 2 * l.Fp);
  l.dh = take(F % 8 ? 2 * (size_t)M * l.Fp : 0);
  l.bias = take(sizeof(float) * 2 * (size_t)F * (size_t)std::max((M + point_rows(M, F) - 1) / point_rows(M, F), (M + 31) / 32));
  l.part = take(std::max(product_workspace(M, D, 2 * ((F + BK - 1) / BK)), pnft_weight_grad_workspace_size(M, 2 * l.Fp, D)));
  l.total = at;
  return l;
}

int point(const uint16_t* dh, int64_t lddh, const void* pre, int64_t ldp, uint16_t* dg, uint16_t* du, int64_t ldd, void* dbg,
          void* dbu, int b_dtype, float* part, int64_t M, int64_t F, int act, int dtype, cudaStream_t st) {
  const bool sums = dbg || dbu;
  PointArgs p;
  memset(&p, 0, sizeof(p));
  p.dh = dh, p.lddh = lddh, p.vec = rows16(dh, lddh, 2);
  p.g = static_cast<const uint16_t*>(pre), p.u = p.g + M * ldp, p.low = p.u + M * ldp, p.ldp = ldp;
  p.dg = dg, p.du = du, p.ldd = ldd;
  p.part = sums ? part : nullptr;
  p.M = (int)M, p.F = (int)F, p.bf16 = dtype == PNFT_DTYPE_BF16;
  p.rows = point_rows(M, F);
  const dim3 grid((unsigned)((F + PCOLS - 1) / PCOLS), (unsigned)((M + p.rows - 1) / p.rows));
  if (act == PNFT_ACT_SILU)
    launch_dependent(sums ? gated_point_kernel<true, PNFT_ACT_SILU> : gated_point_kernel<false, PNFT_ACT_SILU>, grid, PT, 0, st, p);
  else
    launch_dependent(sums ? gated_point_kernel<true, PNFT_ACT_GELU> : gated_point_kernel<false, PNFT_ACT_GELU>, grid, PT, 0, st, p);
  if (int rc = check_launch("gated_bwd pointwise", 1)) return rc;
  return sums ? bias_sum(p.part, grid.y, F, dbg, dbu, b_dtype, st) : PNFT_OK;
}

int gated_dx(const uint16_t* dg, const uint16_t* du, int64_t ldd, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
             void* dx, int64_t lddx, int dx_dtype, void* part, int64_t M, int64_t D, int64_t F, int dtype, int32_t* status,
             cudaStream_t st) {
  Args a;
  memset(&a, 0, sizeof(a));
  int rc = map_kmajor(&a.ta[0], dg, F, M, ldd);
  if (!rc) rc = map_kmajor(&a.ta[1], du, F, M, ldd);
  if (!rc) rc = map_mnmajor(&a.tb[0], wg, D, F, ldwg);
  if (!rc) rc = map_mnmajor(&a.tb[1], wu, D, F, ldwu);
  if (rc) return rc;
  const int kb = (int)((F + BK - 1) / BK);
  a.idesc = idesc(dtype, false, true);
  a.status = status;
  const SumArgs c{{dx, nullptr}, lddx, 0x7fffffff, (int)M, (int)D, nullptr, dx_dtype, 0, rows16(dx, lddx, dtype_size(dx_dtype))};
  return product<false, true>("gated_bwd dx", a, c, static_cast<float*>(part), M, D, 2 * kb, kb, nullptr, st);
}

}  // namespace

extern "C" size_t pnft_gated_bwd_workspace_size(int64_t M, int64_t D, int64_t F) {
  return M <= 0 || D <= 0 || F <= 0 ? 0 : bwd_layout(M, D, F).total;
}

extern "C" int pnft_gated_bwd(const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                              const void* bg, const void* bu, int b_dtype, const void* pre, int64_t ldp, const void* dh,
                              int64_t lddh, void* dx, int64_t lddx, int dx_dtype, void* dwg, void* dwu, int64_t lddw,
                              int dw_dtype, void* dbg, void* dbu, void* workspace, size_t workspace_bytes, int64_t M,
                              int64_t D, int64_t F, int act, int dtype, int32_t* status, void* stream) {
  if (int rc = gated_check("gated_bwd", M, D, F, act, dtype)) return rc;
  for (int t : {b_dtype, dx_dtype, dw_dtype})
    if (t < PNFT_DTYPE_F32 || t > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "gated_bwd: unknown type %d", t);
  if ((dx && lddx < D) || ((dwg || dwu) && lddw < D)) return fail(PNFT_EINVAL, "gated_bwd: row strides below the width");
  cudaStream_t st = as_stream(stream);
  if (M == 0) {
    for (void* d : {dwg, dwu})
      if (d && cudaMemset2DAsync(d, (size_t)lddw * dtype_size(dw_dtype), 0, (size_t)D * dtype_size(dw_dtype), (size_t)F, st) !=
                   cudaSuccess)
        return check_launch("gated_bwd memset", 0);
    for (void* d : {dbg, dbu})
      if (d && cudaMemsetAsync(d, 0, (size_t)F * dtype_size(b_dtype), st) != cudaSuccess) return check_launch("gated_bwd memset", 0);
    return PNFT_OK;
  }
  if (!dh) return fail(PNFT_EINVAL, "gated_bwd: null pointer");
  if (lddh < F || (pre && ldp < F)) return fail(PNFT_EINVAL, "gated_bwd: row strides below the width");
  if (pre && !rows16(pre, ldp, 2)) return fail(PNFT_EINVAL, "gated_bwd: the kept rows must be 16-byte aligned");
  const BwdLayout l = bwd_layout(M, D, F);
  if (!workspace || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(PNFT_EINVAL, "gated_bwd: workspace of %zu bytes < required %zu (16-byte aligned)", workspace_bytes, l.total);
  if (F % 8 == 0 && !pre && !rows16(dh, lddh, 2))
    return fail(PNFT_EUNSUPPORTED, "gated_bwd: dh rows must be 16-byte aligned (or F not a multiple of 8)");
  if (int rc = gated_operands("gated_bwd", x, ldx, wg, ldwg, wu, ldwu, D)) return rc;
  char* ws = static_cast<char*>(workspace);
  uint16_t* dg = reinterpret_cast<uint16_t*>(ws + l.d);
  uint16_t* du = dg + l.Fp;
  const int64_t ldd = 2 * l.Fp;
  float* bias = reinterpret_cast<float*>(ws + l.bias);
  int rc = PNFT_OK;
  if (pre) {
    rc = point(static_cast<const uint16_t*>(dh), lddh, pre, ldp, dg, du, ldd, dbg, dbu, b_dtype, bias, M, F, act, dtype, st);
  } else {
    const void* d = dh;
    int64_t ldh = lddh;
    if (!rows16(dh, lddh, 2)) {  // TMA reads dh: bring its rows to 16 bytes
      d = ws + l.dh, ldh = l.Fp;
      rc = pnft_copy_rows16(dh, lddh, ws + l.dh, l.Fp, M, F, stream);
    }
    Out g, u;
    CUtensorMap map;
    if (!rc) rc = make_out(&g, dg, dtype, F, M, ldd, 1, 0, 64);
    if (!rc) rc = make_out(&u, du, dtype, F, M, ldd, 1, 0, 64);
    if (!rc) rc = tma_map_out(&map, d, 2, F, M, ldh, 1, 0, 32, 64);
    if (!rc)
      rc = gated_gemm("gated_bwd", BWD, x, ldx, wg, ldwg, wu, ldwu, bg, bu, b_dtype, g, u, &map, dbg || dbu ? bias : nullptr, M, D, F, act,
                      dtype, status, st);
    if (!rc && (dbg || dbu))
      rc = bias_sum(bias, (M + 31) / 32, F, dbg, dbu, b_dtype, st);
  }
  if (!rc && dx) rc = gated_dx(dg, du, ldd, wg, ldwg, wu, ldwu, dx, lddx, dx_dtype, ws + l.part, M, D, F, dtype, status, st);
  if (!rc && (dwg || dwu))
    rc = weight_grad("gated_bwd dW", dg, ldd, x, ldx, dwg, dwu, lddw, l.Fp, F, dw_dtype, ws + l.part, M, 2 * l.Fp, D, dtype,
                     status, st);
  return rc;
}
