// Products of a weight matrix with a few rows (single tokens, small batches of answers):
//   acc[r, n] = sum_k W[r, k] x[n, k],   16 rows of W per warp, n < 8 NT <= 32
// Bound by reading W once. A 256-row tcgen05 tile would be almost empty and leave half of
// the SMs without a tile, so here every warp streams its own 16 rows straight from memory
// into the fragments of mma.sync (m16n8k16, W as the 16-row operand, the tokens as the 8
// columns): a lane's 16-byte load holds its four register words of two such steps, since
// the order of k within a dot product is free as long as both operands share it.
#pragma once

#include "gemm_tc.cuh"

namespace pnft {
namespace skinny {

constexpr int WARPS = 8;

template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements from column k of a row of D (zeros past its end). VEC: 16-byte aligned
// rows and D a multiple of 8. STREAM: read once (weights).
template <bool VEC, bool STREAM>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int D) {
  if constexpr (VEC) {
    if (k >= D) return make_uint4(0, 0, 0, 0);
    const uint4* p = reinterpret_cast<const uint4*>(row + k);
    return STREAM ? __ldcs(p) : *p;
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = k + 2 * i < D ? row[k + 2 * i] : 0, hi = k + 2 * i + 1 < D ? row[k + 2 * i + 1] : 0;
      w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The lane's part of a warp's product: RG groups of 16 rows (w[2 r]: the group's row
// lane / 4, w[2 r + 1]: 8 below), 32-wide steps first, first + stride, ... of K.
// acc[r][j]: rows (lane / 4, + 8) x tokens 8 j + 2 (lane & 3) + {0, 1}, in mma.sync's order.
// The groups share the tokens' fragments, which come from L1. FOLD: after 16 steps (512 of
// K) the sums go into a second set of accumulators: the tensor core's own sum over K
// truncates, which an fp32 result would show.
template <bool FOLD, int RG, int NT, bool VEC, bool BF16>
__device__ __forceinline__ void dot(const uint16_t* const (&w)[2 * RG], const uint16_t* x, int64_t ldx, int M, int D, int first,
                                    int stride, float (&acc)[RG][NT][4]) {
  // Steps in flight: four while their registers allow it. B200, four against two: one row of 50021 x 1024 37 and
  // 41 us; 32 rows of the gated 4096 x 16384 88 and 78.
  constexpr int U = RG * NT <= 2 ? 4 : 2;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int steps = (D + 31) / 32;
  float part[FOLD ? RG : 1][NT][4] = {};
  auto fold = [&]() {
#pragma unroll
    for (int r = 0; r < RG; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][j][k] += part[FOLD ? r : 0][j][k], part[FOLD ? r : 0][j][k] = 0.f;
  };
  int since = 0;
  for (int s = first; s < steps; s += U * stride) {
    if (FOLD && since >= 16) fold(), since = 0;
    since += U;
    uint4 a[U][2 * RG];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = s + i * stride < steps ? 32 * (s + i * stride) + 8 * t : D;  // past the last step: zeros
#pragma unroll
      for (int r = 0; r < 2 * RG; ++r) a[i][r] = load8<VEC, true>(w[r], k, D);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = s + i * stride < steps ? 32 * (s + i * stride) + 8 * t : D;
      uint4 v[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
        v[j] = 8 * j + g < M ? load8<VEC, false>(x + (8 * j + g) * ldx, k, D) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 &p = a[i][2 * r], &q = a[i][2 * r + 1];
          float(&sum)[4] = FOLD ? part[FOLD ? r : 0][j] : acc[r][j];
          mma<BF16>(sum, p.x, q.x, p.y, q.y, v[j].x, v[j].y);
          mma<BF16>(sum, p.z, q.z, p.w, q.w, v[j].z, v[j].w);
        }
    }
  }
  if (FOLD) fold();
}

// Calls f(NT, VEC, BF16 as integral constants) for M <= 8 MAX_NT rows.
template <int MAX_NT, class F>
int dispatch(int64_t M, bool vec, bool bf16, F f) {
  auto types = [&](auto nt) {
    if (vec) return bf16 ? f(nt, std::true_type(), std::true_type()) : f(nt, std::true_type(), std::false_type());
    return bf16 ? f(nt, std::false_type(), std::true_type()) : f(nt, std::false_type(), std::false_type());
  };
  if (M <= 8) return types(std::integral_constant<int, 1>());
  if (M <= 16) return types(std::integral_constant<int, 2>());
  if constexpr (MAX_NT > 3) {
    if (M > 24) return types(std::integral_constant<int, 4>());
  }
  return types(std::integral_constant<int, 3>());
}

}  // namespace skinny
}  // namespace pnft
