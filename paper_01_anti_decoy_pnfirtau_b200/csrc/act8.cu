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
  int D, blocks, dtype, vec;
};

// Eight columns per lane, 16 lanes per block of 128.
__global__ void __launch_bounds__(AT) act8_pack_kernel(ActArgs p) {
  const int lane = threadIdx.x & 15;
  const int64_t n = p.M * p.blocks;
  int lo, hi;
  exponent_range(p.dtype, &lo, &hi);
  for (int64_t i = ((int64_t)blockIdx.x * AT + threadIdx.x) / 16; i < (n + 1) / 2 * 2; i += (int64_t)gridDim.x * AT / 16) {
    const int64_t row = i / p.blocks;
    const int b = (int)(i - row * p.blocks), col = b * 128 + 8 * lane;
    const int cnt = i < n ? p.D - col : 0;
    float v[8];
    if (p.dtype == PNFT_DTYPE_F32) {
      const float* src = static_cast<const float*>(p.x) + row * p.ldx + col;
      if (p.vec && cnt >= 8) {
        const float4 a = reinterpret_cast<const float4*>(src)[0], c = reinterpret_cast<const float4*>(src)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = c.x, v[5] = c.y, v[6] = c.z, v[7] = c.w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < cnt ? src[k] : 0.f;
      }
    } else {
      tc::load_row16<8>(static_cast<const uint16_t*>(p.x) + row * p.ldx + col, v, cnt, p.vec, p.dtype == PNFT_DTYPE_BF16);
    }
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (!(fabsf(v[k]) <= 3.402823466e38f)) v[k] = __int_as_float(0x7fc00000);
      top = fmaxf(top, fabsf(v[k]));  // fmaxf leaves NaN out
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // top = f * 2^k, 1 <= f < 2 (subnormals fall below the range anyway): 448 = 1.75 * 2^8
    const int bits = __float_as_int(top);
    int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
    e = max(lo, min(hi, top == 0.f ? lo : e));
    const float scale = pow2(-e), end = e == hi ? 240.f : 448.f;
    if (cnt <= 0) continue;
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a = v[2 * k] * scale, c = v[2 * k + 1] * scale;
      if (fabsf(a) > end) a = copysignf(end, a);  // leaves NaN alone
      if (fabsf(c) > end) c = copysignf(end, c);
      const uint32_t h = to_e4m3x2(a, c);
      w[k / 2] = k & 1 ? w[k / 2] | (h << 16) : h;
    }
    uint8_t* dst = p.q + row * p.ldq + col;
    if (cnt >= 8) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
      for (int k = 0; k < cnt; ++k) dst[k] = (uint8_t)(w[k / 4] >> (8 * (k & 3)));
    }
    if (lane == 0) p.e[row * p.lde + b] = (int8_t)e;
  }
}

__global__ void __launch_bounds__(AT) act8_unpack_kernel(ActArgs p, void* y, int64_t ldy) {
  const int vecs = (p.D + 7) / 8;
  const int64_t n = p.M * vecs;
  for (int64_t i = (int64_t)blockIdx.x * AT + threadIdx.x; i < n; i += (int64_t)gridDim.x * AT) {
    const int64_t row = i / vecs;
    const int col = (int)(i - row * vecs) * 8, cnt = p.D - col;
    const uint2 w = *reinterpret_cast<const uint2*>(p.q + row * p.ldq + col);
    const float scale = pow2(p.e[row * p.lde + col / 128]);
    const uint32_t u[4] = {w.x, w.x >> 16, w.y, w.y >> 16};
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
  ActArgs a{x, ldx, static_cast<uint8_t*>(q), ldq, e, lde, M, (int)D, (int)((D + 127) / 128), dtype,
            tc::rows16(x, ldx, dtype == PNFT_DTYPE_F32 ? 4 : 2)};
  const int64_t blocks = (M * a.blocks * 16 + AT - 1) / AT;
  act8_pack_kernel<<<(unsigned)std::min<int64_t>(blocks, (int64_t)tc::sm_count() * 32), AT, 0, as_stream(stream)>>>(a);
  return check_launch("act8_pack", 1);
}

extern "C" int pnft_act8_unpack(const void* q, int64_t ldq, const int8_t* e, int64_t lde, void* y, int64_t ldy, int64_t M,
                                int64_t D, int dtype, void* stream) {
  if (int rc = act8_check("act8_unpack", y, ldy, q, ldq, e, lde, M, D, dtype)) return rc;
  if (M == 0) return PNFT_OK;
  ActArgs a{nullptr, 0, static_cast<uint8_t*>(const_cast<void*>(q)), ldq, const_cast<int8_t*>(e), lde, M, (int)D,
            (int)((D + 127) / 128), dtype, tc::rows16(y, ldy, dtype == PNFT_DTYPE_F32 ? 4 : 2)};
  const int64_t blocks = (M * ((D + 7) / 8) + AT - 1) / AT;
  act8_unpack_kernel<<<(unsigned)std::min<int64_t>(blocks, (int64_t)tc::sm_count() * 32), AT, 0, as_stream(stream)>>>(a, y, ldy);
  return check_launch("act8_unpack", 1);
}
