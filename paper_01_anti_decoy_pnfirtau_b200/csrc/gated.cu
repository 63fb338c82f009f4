// The gated feed-forward product of a decoder block and its backward pass:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u          (act: SiLU or erf GELU)
//   dg = dh * u * act'(g),  du = dh * act(g),  dx = dg Wg + du Wu
//
// (the weight gradients dg^T x, du^T x are pnft_weight_grad's). Both projections are
// one GEMM: a 128 x 256 accumulator holds 128 columns of g and the same 128 of u, fed
// from the two weights' tiles with the x tile read once, so the epilogue has both
// values of an element in one thread and g, u never meet in memory unless a backward
// wants them.
#include "gemm_tc.cuh"

namespace pnft {
namespace {

using namespace tc;

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;

// act(g); deriv: also act'(g). The exponentials and the quotient are the fast ones
// (a few units of 2^-23): the results are rounded to 16 bits. GELU's normal
// distribution goes through erfc, which keeps its relative accuracy for g << 0.
template <bool DERIV>
__device__ __forceinline__ float act_value(float g, int act, float* deriv) {
  if (act == PNFT_ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    if (DERIV) *deriv = s * (1.f + g * (1.f - s));
    return g * s;
  }
  const float cdf = 0.5f * erfcf(-kSqrtHalf * g);
  if (DERIV) *deriv = cdf + g * (kInvSqrt2Pi * __expf(-0.5f * g * g));
  return g * cdf;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == PNFT_DTYPE_F32) return static_cast<const float*>(p)[i];
  return load16(static_cast<const uint16_t*>(p) + i, dtype == PNFT_DTYPE_BF16);
}

// Forward (dh NULL): h, and g, u when asked for. Backward recomputation (dh given):
// dg, du of the recomputed g, u.
struct GatedEpi {
  struct Params {
    const void *bg, *bu;
    int b_dtype;
    uint16_t* h;
    int64_t ldh;
    uint16_t *g, *u;  // forward: the pre-activations to keep (may be NULL); backward: dg, du
    int64_t ldp;
    const uint16_t* dh;
    int64_t lddh;
    int M, F, act, bf16;
    int vec_h, vec_p, vec_dh;
  };
  const Params& p;
  EpiWarp w;
  __device__ GatedEpi(const Params& p_, const EpiWarp& w_) : p(p_), w(w_) {}
  __device__ void item_begin(const Item&) {}
  __device__ void item_end(const Item&) {}
  template <class Release>
  __device__ void tile(const Item& it, int nt, uint32_t acc, bool zero, Release release) {
    const int row = it.mt * BM + w.row();
    const bool live = row < p.M;
    const bool bf16 = p.bf16;
    constexpr int W = BN / 4;  // columns of g (and of u) of this warp's half
#pragma unroll 1
    for (int c = w.half * W; c < (w.half + 1) * W; c += 32) {
      uint32_t rg[32], ru[32];
      tmem_load32x2(acc + c, rg, acc + BN / 2 + c, ru);
      if (c + 32 == (w.half + 1) * W) release();
      const int col = nt * (BN / 2) + c, n = p.F - col;
      if (!live || n <= 0) continue;
      float g[32], u[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        g[i] = zero ? 0.f : __uint_as_float(rg[i]);
        u[i] = zero ? 0.f : __uint_as_float(ru[i]);
      }
      if (p.bg) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < n) g[i] += load_any(p.bg, col + i, p.b_dtype);
      }
      if (p.bu) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < n) u[i] += load_any(p.bu, col + i, p.b_dtype);
      }
      if (p.dh) {
        float d[32];
        load_row16<32>(p.dh + (int64_t)row * p.lddh + col, d, n, p.vec_dh, bf16);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float da;
          const float a = act_value<true>(g[i], p.act, &da);
          g[i] = d[i] * u[i] * da;
          u[i] = d[i] * a;
        }
      }
      if (p.g) {
        store_row16<32>(p.g + (int64_t)row * p.ldp + col, g, n, p.vec_p, bf16);
        store_row16<32>(p.u + (int64_t)row * p.ldp + col, u, n, p.vec_p, bf16);
      }
      if (p.h) {
#pragma unroll
        for (int i = 0; i < 32; ++i) g[i] = act_value<false>(g[i], p.act, nullptr) * u[i];
        store_row16<32>(p.h + (int64_t)row * p.ldh + col, g, n, p.vec_h, bf16);
      }
    }
  }
};

// ------------------------------------------------------------------ pointwise backward
// dg, du from dh and the kept g, u (16-bit rows), with the column sums of dg and du as
// stored for the biases' gradients; without dh only the sums of given dg, du. A block
// takes 8 columns per lane (256 in all) of a run of rows, a warp a row at a time.
constexpr int PT = 256, PCOLS = 256;
struct PointArgs {
  const uint16_t* dh;
  int64_t lddh;
  const uint16_t *g, *u;
  int64_t ldp;
  uint16_t *dg, *du;
  int64_t ldd;
  float* part;  // [gridDim.y][2][F] (NULL: no sums)
  int M, F, act, bf16, rows, vec;
};

template <bool POINT>
__global__ void __launch_bounds__(PT) gated_point_kernel(PointArgs p) {
  __shared__ float red[PT / 32][2][PCOLS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * PCOLS + 8 * lane, n = p.F - col;
  const bool bf16 = p.bf16;
  float sg[8], su[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) sg[k] = su[k] = 0.f;
  const int64_t r0 = (int64_t)blockIdx.y * p.rows, r1 = std::min<int64_t>(p.M, r0 + p.rows);
  if (n > 0) {
    for (int64_t r = r0 + warp; r < r1; r += PT / 32) {
      float g[8], u[8];
      load_row16<8>(p.g + r * p.ldp + col, g, n, p.vec, bf16);
      load_row16<8>(p.u + r * p.ldp + col, u, n, p.vec, bf16);
      if (POINT) {
        float d[8];
        load_row16<8>(p.dh + r * p.lddh + col, d, n, p.vec, bf16);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float da;
          const float a = act_value<true>(g[k], p.act, &da);
          g[k] = d[k] * u[k] * da;
          u[k] = d[k] * a;
        }
        store_row16<8>(p.dg + r * p.ldd + col, g, n, p.vec, bf16);
        store_row16<8>(p.du + r * p.ldd + col, u, n, p.vec, bf16);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sg[k] += g[k], su[k] += u[k];
    }
  }
  if (!p.part) return;
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

__global__ void __launch_bounds__(256) gated_bias_sum_kernel(const float* __restrict__ part, int blocks, int F, void* dbg,
                                                             void* dbu, int dtype) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * F) return;
  float t = 0.f;
  for (int b = 0; b < blocks; ++b) t += part[(int64_t)b * 2 * F + i];
  void* dst = i < F ? dbg : dbu;
  const int c = i < F ? i : i - F;
  if (!dst) return;
  if (dtype == PNFT_DTYPE_F32)
    static_cast<float*>(dst)[c] = t;
  else
    store16(static_cast<uint16_t*>(dst) + c, t, dtype == PNFT_DTYPE_BF16);
}

// Rows per block of the pointwise kernel: about four blocks per SM.
int point_rows(int64_t M, int64_t F) {
  const int64_t cols = (F + PCOLS - 1) / PCOLS;
  const int64_t want = std::max<int64_t>(1, 4 * sm_count() / cols);
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

int gated_gemm(const char* what, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
               int64_t M, int64_t D, int64_t F, int dtype, const GatedEpi::Params& ep, int32_t* status, cudaStream_t st) {
  if (!tma_rows_ok(x, ldx, D) || !tma_rows_ok(wg, ldwg, D) || !tma_rows_ok(wu, ldwu, D))
    return fail(PNFT_EUNSUPPORTED, "%s: x and weight rows must be 16-byte aligned (strides multiples of 8)", what);
  if (!device_is_sm100()) return fail(PNFT_EUNSUPPORTED, "%s: needs an sm_100 device", what);
  Args a;
  memset(&a, 0, sizeof(a));
  int rc = map_kmajor(&a.ta[0], x, D, M, ldx);
  if (!rc) rc = map_kmajor(&a.tb[0], wg, D, F, ldwg);
  if (!rc) rc = map_kmajor(&a.tb[1], wu, D, F, ldwu);
  if (rc) return rc;
  a.s = plain_sched(M, 2 * ((F + BN / 2 - 1) / (BN / 2) * (BN / 2)), (D + BK - 1) / BK, 1);
  a.idesc = idesc(dtype, false, false);
  a.status = status;
  return launch<false, false, true, GatedEpi>(what, a, ep, st);
}

}  // namespace
}  // namespace pnft

using namespace pnft;
using namespace pnft::tc;

extern "C" int pnft_gated_fwd(const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                              const void* bg, const void* bu, int b_dtype, void* h, int64_t ldh, void* g, void* u,
                              int64_t ldp, int64_t M, int64_t D, int64_t F, int act, int dtype, int32_t* status,
                              void* stream) {
  if (int rc = gated_check("gated_fwd", M, D, F, act, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  if (!h || (!g) != (!u)) return fail(PNFT_EINVAL, "gated_fwd: null output");
  if (ldh < F || (g && ldp < F)) return fail(PNFT_EINVAL, "gated_fwd: row strides below the width");
  GatedEpi::Params ep{bg, bu, b_dtype, static_cast<uint16_t*>(h), ldh, static_cast<uint16_t*>(g),
                      static_cast<uint16_t*>(u), ldp, nullptr, 0, (int)M, (int)F, act, dtype == PNFT_DTYPE_BF16,
                      rows16(h, ldh, 2), rows16(g, ldp, 2) && rows16(u, ldp, 2), 0};
  return gated_gemm("gated_fwd", x, ldx, wg, ldwg, wu, ldwu, M, D, F, dtype, ep, status, as_stream(stream));
}

extern "C" int pnft_gated_bwd_recompute(const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
                                        int64_t ldwu, const void* bg, const void* bu, int b_dtype, const void* dh,
                                        int64_t lddh, void* dg, void* du, int64_t ldd, int64_t M, int64_t D, int64_t F,
                                        int act, int dtype, int32_t* status, void* stream) {
  if (int rc = gated_check("gated_bwd_recompute", M, D, F, act, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  if (!dh || !dg || !du) return fail(PNFT_EINVAL, "gated_bwd_recompute: null pointer");
  if (lddh < F || ldd < F) return fail(PNFT_EINVAL, "gated_bwd_recompute: row strides below the width");
  GatedEpi::Params ep{bg, bu, b_dtype, nullptr, 0, static_cast<uint16_t*>(dg), static_cast<uint16_t*>(du), ldd,
                      static_cast<const uint16_t*>(dh), lddh, (int)M, (int)F, act, dtype == PNFT_DTYPE_BF16, 0,
                      rows16(dg, ldd, 2) && rows16(du, ldd, 2), rows16(dh, lddh, 2)};
  return gated_gemm("gated_bwd_recompute", x, ldx, wg, ldwg, wu, ldwu, M, D, F, dtype, ep, status, as_stream(stream));
}

extern "C" size_t pnft_gated_bias_workspace_size(int64_t M, int64_t F) {
  if (M <= 0 || F <= 0) return 0;
  const int64_t rows = point_rows(M, F);
  return sizeof(float) * 2 * (size_t)F * (size_t)((M + rows - 1) / rows);
}

extern "C" int pnft_gated_bwd_point(const void* dh, int64_t lddh, const void* g, const void* u, int64_t ldp, void* dg,
                                    void* du, int64_t ldd, void* dbg, void* dbu, int b_dtype, void* workspace,
                                    size_t workspace_bytes, int64_t M, int64_t F, int act, int dtype, void* stream) {
  if (int rc = gated_check("gated_bwd_point", M, 1, F, act, dtype)) return rc;
  const bool sums = dbg || dbu;
  cudaStream_t st = as_stream(stream);
  if (M == 0) {
    const size_t n = (size_t)F * (b_dtype == PNFT_DTYPE_F32 ? 4 : 2);
    if ((dbg && cudaMemsetAsync(dbg, 0, n, st) != cudaSuccess) || (dbu && cudaMemsetAsync(dbu, 0, n, st) != cudaSuccess))
      return check_launch("gated_bwd_point memset", 0);
    return PNFT_OK;
  }
  if (!g || !u || (dh && (!dg || !du)) || (!dh && !sums)) return fail(PNFT_EINVAL, "gated_bwd_point: null pointer");
  if (ldp < F || (dh && (lddh < F || ldd < F))) return fail(PNFT_EINVAL, "gated_bwd_point: row strides below the width");
  const size_t need = sums ? pnft_gated_bias_workspace_size(M, F) : 0;
  if (sums && (!workspace || workspace_bytes < need))
    return fail(PNFT_EINVAL, "gated_bwd_point: workspace of %zu bytes < required %zu", workspace_bytes, need);
  PointArgs p;
  memset(&p, 0, sizeof(p));
  p.dh = static_cast<const uint16_t*>(dh), p.lddh = lddh;
  p.g = static_cast<const uint16_t*>(g), p.u = static_cast<const uint16_t*>(u), p.ldp = ldp;
  p.dg = static_cast<uint16_t*>(dg), p.du = static_cast<uint16_t*>(du), p.ldd = ldd;
  p.part = sums ? static_cast<float*>(workspace) : nullptr;
  p.M = (int)M, p.F = (int)F, p.act = act, p.bf16 = dtype == PNFT_DTYPE_BF16;
  p.rows = point_rows(M, F);
  p.vec = rows16(g, ldp, 2) && rows16(u, ldp, 2) && (!dh || (rows16(dh, lddh, 2) && rows16(dg, ldd, 2) && rows16(du, ldd, 2)));
  const dim3 grid((unsigned)((F + PCOLS - 1) / PCOLS), (unsigned)((M + p.rows - 1) / p.rows));
  if (dh)
    gated_point_kernel<true><<<grid, PT, 0, st>>>(p);
  else
    gated_point_kernel<false><<<grid, PT, 0, st>>>(p);
  if (sums)
    gated_bias_sum_kernel<<<(unsigned)((2 * F + 255) / 256), 256, 0, st>>>(p.part, (int)grid.y, (int)F, dbg, dbu, b_dtype);
  return check_launch("gated_bwd_point", sums ? 2 : 1);
}

static int dx_splits(int64_t M, int64_t D, int64_t F) {
  return plan_splits((int)(((M + BM - 1) / BM) * ((D + BN - 1) / BN)), (int)(2 * ((F + BK - 1) / BK)));
}

extern "C" size_t pnft_gated_dx_workspace_size(int64_t M, int64_t D, int64_t F) {
  if (M <= 0 || D <= 0 || F <= 0) return 0;
  const int s = dx_splits(M, D, F);
  return s > 1 ? sizeof(float) * (size_t)s * (size_t)M * (size_t)((D + 3) / 4 * 4) : 0;
}

extern "C" int pnft_gated_dx(const void* dg, const void* du, int64_t ldd, const void* wg, int64_t ldwg, const void* wu,
                             int64_t ldwu, void* dx, int64_t lddx, int dx_dtype, void* workspace, size_t workspace_bytes,
                             int64_t M, int64_t D, int64_t F, int dtype, int32_t* status, void* stream) {
  if (int rc = gated_check("gated_dx", M, D, F, PNFT_ACT_SILU, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  if (!dx || lddx < D) return fail(PNFT_EINVAL, "gated_dx: null output or row stride below the width");
  if (dx_dtype < PNFT_DTYPE_F32 || dx_dtype > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "gated_dx: unknown output type %d", dx_dtype);
  if (!tma_rows_ok(dg, ldd, F) || !tma_rows_ok(du, ldd, F) || !tma_rows_ok(wg, ldwg, D) || !tma_rows_ok(wu, ldwu, D))
    return fail(PNFT_EUNSUPPORTED, "gated_dx: operand rows must be 16-byte aligned (strides multiples of 8)");
  if (!device_is_sm100()) return fail(PNFT_EUNSUPPORTED, "gated_dx: needs an sm_100 device");
  cudaStream_t st = as_stream(stream);
  Args a;
  memset(&a, 0, sizeof(a));
  int rc = map_kmajor(&a.ta[0], dg, F, M, ldd);
  if (!rc) rc = map_kmajor(&a.ta[1], du, F, M, ldd);
  if (!rc) rc = map_mnmajor(&a.tb[0], wg, D, F, ldwg);
  if (!rc) rc = map_mnmajor(&a.tb[1], wu, D, F, ldwu);
  if (rc) return rc;
  const int kb = (int)((F + BK - 1) / BK), splits = dx_splits(M, D, F);
  a.s = plain_sched(M, D, 2 * kb, splits);
  a.s.seg_kb = kb;
  a.idesc = idesc(dtype, false, true);
  a.status = status;
  const int osize = dx_dtype == PNFT_DTYPE_F32 ? 4 : 2;
  StoreEpi::Params out{{dx, nullptr}, lddx, 0x7fffffff, (int)M, (int)D, nullptr, dx_dtype, 0, 0, rows16(dx, lddx, osize)};
  if (splits == 1) return launch<false, true, false, StoreEpi>("gated_dx", a, out, st);
  const size_t need = pnft_gated_dx_workspace_size(M, D, F);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(PNFT_EINVAL, "gated_dx: workspace of %zu bytes < required %zu (16-byte aligned)", workspace_bytes, need);
  const int64_t ldp = (D + 3) / 4 * 4;
  StoreEpi::Params part{{workspace, nullptr}, ldp, 0x7fffffff, (int)M, (int)D, nullptr, PNFT_DTYPE_F32, 0, M * ldp, 1};
  rc = launch<false, true, false, StoreEpi>("gated_dx", a, part, st);
  if (rc) return rc;
  return sum_splits(static_cast<const float*>(workspace), ldp, M * ldp, splits, out, (int)M, st);
}
