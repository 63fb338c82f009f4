// Activations kept in 8 bits for the backward pass: per row and block of 128 columns
//
//   q = e4m3(x * 2^-e),   e the least exponent with max |x| <= 448 * 2^e
//
// The scale is a power of two, so multiplying by it rounds nothing and q * 2^e is a
// bf16 (and fp32) number again: what the backward reads differs from x by e4m3's
// rounding alone (at most 2^-4 relative, or half a step of 2^(e-9)). NaN and infinities
// become NaN and take no part in the maximum. Both kernels are bound by HBM.
#include "gemm_tc.cuh"

namespace pnft {
namespace {

constexpr int AT = 256;

// e's range: what is stored comes back finite and exact in the type that it came from
// (fp16: 2^-24 is its least step and 65504 its largest value; bf16 and fp32 share their
// exponents). In the largest exponent 256 * 2^e is past the type, so values end at 240.
__device__ __forceinline__ void exponent_range(int dtype, int* lo, int* hi) {
  *lo = dtype == PNFT_DTYPE_F16 ? -15 : -110;
  *hi = dtype == PNFT_DTYPE_F16 ? 8 : 120;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}

struct ActArgs {
  const void* x;
  int64_t ldx;
  uint8_t* q;
  int64_t ldq;
  int8_t* e;
  int64_t lde;
  int64_t M;
  int D, dtype, vec;
};

// Eight columns of a row as they are stored (16 or 32 bytes; zeros past the row's end).
template <bool F32>
struct Raw {
  uint32_t w[F32 ? 8 : 4];
  __device__ __forceinline__ void load(const void* x, int64_t at, int cnt, bool vec) {
    constexpr int SIZE = F32 ? 4 : 2;
    const char* src = static_cast<const char*>(x) + at * SIZE;
    if (vec && cnt >= 8) {
#pragma unroll
      for (int i = 0; i < SIZE / 2; ++i) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(src) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if (F32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[F32 ? k : 0] = k < cnt ? reinterpret_cast<const uint32_t*>(src)[k] : 0;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = (2 * k < cnt ? reinterpret_cast<const uint16_t*>(src)[2 * k] : 0u) |
               (2 * k + 1 < cnt ? (uint32_t) reinterpret_cast<const uint16_t*>(src)[2 * k + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ float2 pair(int k, bool bf16) const {
    if constexpr (F32) return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    return tc::unpack2(w[k], bf16);
  }
  // The largest magnitude's bits as fp32, NaN left out: magnitudes compare as integers, 16-bit
  // ones two at a time.
  __device__ __forceinline__ uint32_t top(bool bf16) const {
    if constexpr (F32) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(__uint_as_float(w[k])));
      return __float_as_uint(m);
    } else if (bf16) {
      __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
      for (int k = 1; k < 4; ++k) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[k])));
      return __float_as_uint(fmaxf(fmaxf(__low2float(m), __high2float(m)), 0.f));
    } else {
      __half2 m = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
      for (int k = 1; k < 4; ++k) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&w[k])));
      return __float_as_uint(fmaxf(fmaxf(__low2float(m), __high2float(m)), 0.f));
    }
  }
};

// A warp takes COLS columns of a row at a time, all of its loads in flight at once.
constexpr int COLS = 1024;

// Packing: eight lanes per block of 128 columns, each with two runs of eight columns 64 apart,
// so that a load of eight lanes is 128 bytes in a row and the exponent, its reduction and the
// votes are shared by 16 values (16384 x 1024 bf16 from
// cold L2: 12.7 us; 15.2 with 16 lanes and 8 values, bound by its instructions; reading 34 MB takes 5.1).
template <bool F32>
__global__ void __launch_bounds__(AT) act8_pack_kernel(ActArgs p) {
  tc::launch_next();
  tc::wait_previous();
  const int lane = threadIdx.x & 31, lane_col = 128 * (lane >> 3) + 8 * (lane & 7);
  const bool bf16 = p.dtype == PNFT_DTYPE_BF16;
  int lo, hi;
  exponent_range(p.dtype, &lo, &hi);
  for (int64_t row = (int64_t)blockIdx.x * (AT / 32) + (threadIdx.x >> 5); row < p.M; row += (int64_t)gridDim.x * (AT / 32)) {
    const int c0 = blockIdx.y * COLS;
    Raw<F32> v[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = c0 + 512 * (i / 2) + 64 * (i & 1) + lane_col;
      v[i / 2][i & 1].load(p.x, row * p.ldx + col, p.D - col, p.vec);
    }
    uint8_t* const q = p.q + row * p.ldq + c0 + lane_col;
    int8_t* const es = p.e + row * p.lde + c0 / 128 + (lane >> 3);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (c0 + 512 * j >= p.D) break;  // the same for the whole warp
      uint32_t top = max(v[j][0].top(bf16), v[j][1].top(bf16));  // not negative: ordered as integers
      const bool odd = top >= 0x7f800000u;
      if (__any_sync(0xffffffffu, odd)) {  // an infinity: the largest of the finite ones, value by value
        top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 f = v[j][k / 4].pair(k % 4, bf16);
          const uint32_t a = __float_as_uint(fabsf(f.x)), c = __float_as_uint(fabsf(f.y));
          top = max(top, max(a < 0x7f800000u ? a : 0u, c < 0x7f800000u ? c : 0u));
        }
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      // top = f * 2^k, 1 <= f < 2 (subnormals fall below the range anyway): 448 = 1.75 * 2^8
      int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffff) > 0x600000);
      e = max(lo, min(hi, top == 0 ? lo : e));
      const float scale = pow2(-e);
      uint32_t w[2][2];
      // Magnitudes are at most 448 after scaling, and NaN stays NaN in the conversion: only infinities
      // and the largest exponent (where values end at 240) need a look at each value.
      if (!__any_sync(0xffffffffu, odd || e == hi)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 f = v[j][k / 4].pair(k % 4, bf16);
          const uint32_t h = to_e4m3x2(f.x * scale, f.y * scale);
          uint32_t& to = w[k / 4][k % 4 / 2];
          to = k & 1 ? to | (h << 16) : h;
        }
      } else {
        const float end = e == hi ? 240.f : 448.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 f = v[j][k / 4].pair(k % 4, bf16);
          float a = f.x * scale, c = f.y * scale;
          a = fabsf(a) > end ? (fabsf(a) == INFINITY ? __int_as_float(0x7fc00000) : copysignf(end, a)) : a;
          c = fabsf(c) > end ? (fabsf(c) == INFINITY ? __int_as_float(0x7fc00000) : copysignf(end, c)) : c;
          const uint32_t h = to_e4m3x2(a, c);
          uint32_t& to = w[k / 4][k % 4 / 2];
          to = k & 1 ? to | (h << 16) : h;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = 512 * j + 64 * h, cnt = p.D - (c0 + at + lane_col);
        if (cnt >= 8) {
          *reinterpret_cast<uint2*>(q + at) = make_uint2(w[h][0], w[h][1]);
        } else {
          for (int k = 0; k < cnt; ++k) q[at + k] = (uint8_t)(w[h][k / 4] >> (8 * (k & 3)));
        }
      }
      if ((lane & 7) == 0 && c0 + 512 * j + lane_col < p.D) es[4 * j] = (int8_t)e;
    }
  }
}

// Unpacking: lanes and columns as in packing, so that an exponent is read for 16 values.
__global__ void __launch_bounds__(AT) act8_unpack_kernel(ActArgs p, void* y, int64_t ldy) {
  tc::launch_next();
  tc::wait_previous();
  const int lane = threadIdx.x & 31, lane_col = 128 * (lane >> 3) + 8 * (lane & 7);
  for (int64_t row = (int64_t)blockIdx.x * (AT / 32) + (threadIdx.x >> 5); row < p.M; row += (int64_t)gridDim.x * (AT / 32)) {
    const int c0 = blockIdx.y * COLS + lane_col;
    const uint8_t* const q = p.q + row * p.ldq + c0;
    const int8_t* const es = p.e + row * p.lde + c0 / 128;
    uint2 w[4];
    int e[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 512 * (i / 2) + 64 * (i & 1);
      if (c0 + at < p.D) w[i] = __ldcs(reinterpret_cast<const uint2*>(q + at));
      if (i % 2 == 0 && c0 + at < p.D) e[i / 2] = es[at / 128];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = c0 + 512 * (i / 2) + 64 * (i & 1), cnt = p.D - col;
      if (cnt <= 0) continue;
      const float scale = pow2(e[i / 2]);
      const uint32_t u[4] = {w[i].x, w[i].x >> 16, w[i].y, w[i].y >> 16};
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = from_e4m3x2(u[k] & 0xffffu);
        v[2 * k] = f.x * scale, v[2 * k + 1] = f.y * scale;
      }
      if (p.dtype == PNFT_DTYPE_F32)
        tc::store_row32<8>(static_cast<float*>(y) + row * ldy + col, v, cnt, p.vec);
      else
        tc::store_row16<8>(static_cast<uint16_t*>(y) + row * ldy + col, v, cnt, p.vec, p.dtype == PNFT_DTYPE_BF16);
    }
  }
}

dim3 act8_grid(int64_t M, int64_t D) {
  return dim3((unsigned)std::min<int64_t>((M + AT / 32 - 1) / (AT / 32), (int64_t)tc::sm_count() * 16), (unsigned)((D + COLS - 1) / COLS));
}

int act8_check(const char* what, const void* x, int64_t ldx, const void* q, int64_t ldq, const void* e, int64_t lde,
               int64_t M, int64_t D, int dtype) {
  if (M < 0 || D <= 0 || D > (1 << 24) || M >= ((int64_t)1 << 40))
    return fail(PNFT_EINVAL, "%s: bad shape M=%lld D=%lld", what, (long long)M, (long long)D);
  if (dtype < PNFT_DTYPE_F32 || dtype > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "%s: unknown dtype code %d", what, dtype);
  if (M == 0) return PNFT_OK;
  if (!x || !q || !e) return fail(PNFT_EINVAL, "%s: null pointer", what);
  if (ldx < D || ldq < (D + 7) / 8 * 8 || ldq % 8 || reinterpret_cast<uintptr_t>(q) % 8 || lde < (D + 127) / 128)
    return fail(PNFT_EINVAL, "%s: row strides (the 8-bit rows are 8-byte aligned, a whole number of 8 columns)", what);
  return PNFT_OK;
}

}  // namespace
}  // namespace pnft

using namespace pnft;

extern "C" int pnft_act8_pack(const void* x, int64_t ldx, void* q, int64_t ldq, int8_t* e, int64_t lde, int64_t M,
                              int64_t D, int dtype, void* stream) {
  if (int rc = act8_check("act8_pack", x, ldx, q, ldq, e, lde, M, D, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  ActArgs a{x, ldx, static_cast<uint8_t*>(q), ldq, e, lde, M, (int)D, dtype,
            tc::rows16(x, ldx, dtype == PNFT_DTYPE_F32 ? 4 : 2)};
  tc::launch_dependent(dtype == PNFT_DTYPE_F32 ? act8_pack_kernel<true> : act8_pack_kernel<false>, act8_grid(M, D), AT, 0,
                       as_stream(stream), a);
  return check_launch("act8_pack", 1);
}

extern "C" int pnft_act8_unpack(const void* q, int64_t ldq, const int8_t* e, int64_t lde, void* y, int64_t ldy, int64_t M,
                                int64_t D, int dtype, void* stream) {
  if (int rc = act8_check("act8_unpack", y, ldy, q, ldq, e, lde, M, D, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  ActArgs a{nullptr, 0, static_cast<uint8_t*>(const_cast<void*>(q)), ldq, const_cast<int8_t*>(e), lde, M, (int)D,
            dtype, tc::rows16(y, ldy, dtype == PNFT_DTYPE_F32 ? 4 : 2)};
  tc::launch_dependent(act8_unpack_kernel, act8_grid(M, D), AT, 0, as_stream(stream), a, y, ldy);
  return check_launch("act8_unpack", 1);
}

// Buffers of a weight gradient from 8 bits: the values as 16-bit rows, dy with aligned rows
// where the caller's are not, and the product's partial sums.
namespace {
struct GradLayout {
  int64_t ldx, ldy;
  size_t x, y, part, total;
};
GradLayout grad_layout(int64_t M, int64_t N, int64_t D) {
  GradLayout l;
  l.ldx = (D + 7) / 8 * 8, l.ldy = (N + 7) / 8 * 8;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  l.x = take(2 * (size_t)M * l.ldx);
  l.y = take(N % 8 ? 2 * (size_t)M * l.ldy : 0);
  l.part = take(pnft_weight_grad_workspace_size(M, N, D));
  l.total = at;
  return l;
}
}  // namespace

extern "C" size_t pnft_act8_weight_grad_workspace_size(int64_t M, int64_t N, int64_t D) {
  return M <= 0 || N <= 0 || D <= 0 ? 0 : grad_layout(M, N, D).total;
}

extern "C" int pnft_act8_weight_grad(const void* dy, int64_t lddy, const void* q, int64_t ldq, const int8_t* e, int64_t lde,
                                     void* dw, int64_t lddw, int dw_dtype, void* workspace, size_t workspace_bytes, int64_t M,
                                     int64_t N, int64_t D, int dtype, int32_t* status, void* stream) {
  if (!tc::type16(dtype)) return fail(PNFT_EUNSUPPORTED, "act8_weight_grad: bfloat16 or float16 gradient expected");
  if (M < 0 || N <= 0 || D <= 0 || lddy < N || lddw < D || !dw)
    return fail(PNFT_EINVAL, "act8_weight_grad: bad shape M=%lld N=%lld D=%lld", (long long)M, (long long)N, (long long)D);
  if (M == 0)
    return pnft_weight_grad(nullptr, 0, nullptr, 0, dw, nullptr, lddw, N, N, dw_dtype, nullptr, 0, 0, N, D, dtype, status, stream);
  if (!dy) return fail(PNFT_EINVAL, "act8_weight_grad: null pointer");
  const GradLayout l = grad_layout(M, N, D);
  if (!workspace || workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(PNFT_EINVAL, "act8_weight_grad: workspace of %zu bytes < required %zu (16-byte aligned)", workspace_bytes, l.total);
  if (N % 8 == 0 && !tc::rows16(dy, lddy, 2))
    return fail(PNFT_EUNSUPPORTED, "act8_weight_grad: dy rows must be 16-byte aligned (or N not a multiple of 8)");
  char* ws = static_cast<char*>(workspace);
  int rc = pnft_act8_unpack(q, ldq, e, lde, ws + l.x, l.ldx, M, D, dtype, stream);
  if (rc) return rc;
  if (!tc::rows16(dy, lddy, 2)) {
    rc = pnft_copy_rows16(dy, lddy, ws + l.y, l.ldy, M, N, stream);
    if (rc) return rc;
    dy = ws + l.y, lddy = l.ldy;
  }
  return pnft_weight_grad(dy, lddy, ws + l.x, l.ldx, dw, nullptr, lddw, N, N, dw_dtype, ws + l.part,
                          pnft_weight_grad_workspace_size(M, N, D), M, N, D, dtype, status, stream);
}
