// Arithmetic of the streamed cross entropy's kernels: base-2 exponentials, pairs of fp32,
// stores of four values.
#pragma once

#include "gemm_tc.cuh"

namespace pnft {
namespace xent {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e30f;  // running maximum before any logit: finite, so that low - low is 0

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Pairs of fp32 in one 64-bit register: two products or sums per instruction.
typedef uint64_t f32x2;
__device__ __forceinline__ f32x2 pack(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two values, both on the special-function unit. At K = 256 that unit (16 per clock
// and SM) is as busy as the tensor core, yet moving every third or second exponential to a
// polynomial on the FMA pipe made the forward's kernel slower (16352 x 33278 x 256: 217 us
// without, 227 and 237 with, at one clock): the instructions cost more clock than the unit does.
__device__ __forceinline__ f32x2 exp2_pair(f32x2 x) {
  const float2 v = unpack(x);
  return pack(ex2(v.x), ex2(v.y));
}

// Four values of a row from column offset `at`, `n` of them inside; vec: whole groups are aligned.
__device__ __forceinline__ void store_row4(void* dst, int64_t at, const float (&f)[4], int n, int dtype, bool vec) {
  const bool bf16 = dtype == PNFT_DTYPE_BF16;
  if (dtype == PNFT_DTYPE_F32) {
    float* d = static_cast<float*>(dst) + at;
    if (vec && n >= 4)
      *reinterpret_cast<float4*>(d) = make_float4(f[0], f[1], f[2], f[3]);
    else
      for (int k = 0; k < 4 && k < n; ++k) d[k] = f[k];
  } else {
    uint16_t* d = static_cast<uint16_t*>(dst) + at;
    if (vec && n >= 4)
      *reinterpret_cast<uint2*>(d) = make_uint2(tc::pack2(f[0], f[1], bf16), tc::pack2(f[2], f[3], bf16));
    else
      for (int k = 0; k < 4 && k < n; ++k) tc::store16(d + k, f[k], bf16);
  }
}

}  // namespace xent
}  // namespace pnft
