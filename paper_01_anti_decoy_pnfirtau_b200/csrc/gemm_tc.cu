// Host side and split sums of the tcgen05 GEMM core (gemm_tc.cuh), and the weight
// gradient dW = dY^T X built on it.
#include "gemm_tc.cuh"

namespace pnft {
namespace tc {

int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? dev : 0;
}

int sm_count() {
  static std::atomic<int> counts[64];
  const int dev = current_device();
  std::atomic<int>& c = counts[dev & 63];
  int n = c.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    c.store(n, std::memory_order_relaxed);
  }
  return n;
}

int plan_splits(int64_t tiles, int64_t kb, int rounds) {
  const int64_t want = std::max<int64_t>(1, rounds * (sm_count() / 2) / std::max<int64_t>(1, tiles));
  return (int)std::max<int64_t>(1, std::min(want, kb / 8));
}

// A round of whole tiles takes 0.42 us per K block; split tiles take a launch more and write and
// read their partials (0.09 us each, from L2). Measured (B200, weight gradient from 8 bits, fp32
// out), the last round split and whole: 8192 rows into 4096 x 4096 (34 of 256 tiles in the last
// round, split in 2) 218 and 228 us; 4096 into 5632 x 1000 (14 of 88, in 5) 53 and 65; 2048 into
// 2560 x 2560 (26 of 100, K too short: whole) 38. The three times are a fit to these shapes.
Plan plan_product(int64_t tiles, int64_t kb) {
  const int pairs = sm_count() / 2;
  if (tiles <= pairs) return Plan{plan_splits(tiles, kb), 0};
  const int rest = (int)(tiles % pairs);
  Plan best{1, 0};
  float least = rest ? 0.42f * (float)kb : 0.f;
  for (int n = 2; n <= 8 && kb / n >= 8; ++n) {
    const float cost = 0.42f * (float)kb * (float)((rest * n + pairs - 1) / pairs) / (float)n + 4.f + 0.09f * (float)(rest * n);
    if (cost < least) least = cost, best = Plan{n, (int)(tiles - rest)};
  }
  return best;
}

size_t product_workspace(int64_t M, int64_t N, int64_t kb) {
  if (M <= 0 || N <= 0 || kb <= 0) return 0;
  const int64_t tiles = tiles_of(M, N);
  const Plan p = plan_product(tiles, kb);
  if (p.splits == 1) return 0;
  if (p.whole) return sizeof(float) * (size_t)(PM * BN) * (size_t)(tiles - p.whole) * (size_t)p.splits;
  return sizeof(float) * (size_t)p.splits * (size_t)M * (size_t)((N + 3) / 4 * 4);
}

namespace {

// Where the split tiles behind whole ones lie (sum_splits_kernel<true>).
struct TailArgs {
  int tiles_m, tiles_n, group_m, whole;
};

// Four columns per thread; partial rows are 16-byte aligned (ldp a multiple of 4).
template <bool TAIL>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* part, int64_t ldp,
                                                         int64_t split_stride, int splits, SumArgs o,
                                                         int rows_total, TailArgs tail) {
  launch_next();
  wait_previous();
  const int n4 = TAIL ? BN / 4 : (o.cols + 3) / 4;
  const float alpha = o.alpha ? *o.alpha : 1.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows_total * n4; i += (int64_t)gridDim.x * 256) {
    int row = (int)(i / n4);
    int c = (int)(i - (int64_t)row * n4) * 4;
    const float* src = part + (int64_t)row * ldp + c;
    if (TAIL) {  // a row of a tile: its place in the matrix
      int mt, nt;
      item_order(tail.whole + row / PM, tail.tiles_m, tail.tiles_n, tail.group_m, &mt, &nt);
      row = mt * PM + row % PM, c += nt * BN;
      if (c >= o.cols) continue;
    }
    const int side = row >= o.row_split;
    if (side) row -= o.row_split;
    if (row >= o.rows || !(side ? o.c[1] : o.c[0])) continue;
    float4 a = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
    for (int s = 1; s < splits; ++s) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src + s * split_stride));
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
    float v[4] = {a.x * alpha, a.y * alpha, a.z * alpha, a.w * alpha};
    const int n = min(4, o.cols - c);
    const int64_t at = (int64_t)row * o.ldc + c;
    if (o.dtype == PNFT_DTYPE_F32) {
      float* dst = static_cast<float*>(side ? o.c[1] : o.c[0]) + at;
      for (int k = 0; k < n; ++k) dst[k] = o.add ? dst[k] + v[k] : v[k];
    } else {
      const bool bf16 = o.dtype == PNFT_DTYPE_BF16;
      uint16_t* dst = static_cast<uint16_t*>(side ? o.c[1] : o.c[0]) + at;
      if (n == 4 && o.vec) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16));
      } else {
        for (int k = 0; k < n; ++k) store16(dst + k, v[k], bf16);
      }
    }
  }
}

// dst[r] = src[r]: a warp per row, eight words in flight per lane.
template <typename W>
__global__ void __launch_bounds__(256) copy_rows_kernel(const char* src, int64_t ss, char* dst,
                                                        int64_t ds, int64_t rows, int64_t words) {
  launch_next();
  wait_previous();
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const W* from = reinterpret_cast<const W*>(src + r * ss);
    W* to = reinterpret_cast<W*>(dst + r * ds);
    for (int64_t i = lane; i < words; i += 256) {
      W v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + 32 * k < words) v[k] = from[i + 32 * k];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + 32 * k < words) to[i + 32 * k] = v[k];
    }
  }
}

// The same for 2-byte elements at any address into 4-byte aligned rows: a row that starts in the middle
// of a word is loaded by the aligned words behind its first element, and each word that is
// stored takes its lower half from the lane before (13.7 us for 4095 x 2731 from cold
// L2, 15.3 element by element).
__global__ void __launch_bounds__(256) copy_rows2_kernel(const uint16_t* src, int64_t ss, uint16_t* dst,
                                                         int64_t ds, int64_t rows, int64_t cols) {
  launch_next();
  wait_previous();
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const uint16_t* from = src + r * ss;
    uint16_t* to = dst + r * ds;
    const int odd = (reinterpret_cast<uintptr_t>(from) >> 1) & 1;
    for (int64_t c0 = 0; c0 < cols; c0 += 512) {
      uint32_t v[8], first[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t c = c0 + 64 * k + 2 * lane, at = c + odd;  // columns stored, column loaded from
        v[k] = at + 1 < cols ? *reinterpret_cast<const uint32_t*>(from + at) : at < cols ? from[at] : 0u;
        first[k] = odd && lane == 0 && c < cols ? from[c] : 0u;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t c = c0 + 64 * k + 2 * lane;
        if (odd) {
          const uint32_t before = __shfl_up_sync(0xffffffffu, v[k], 1) >> 16;
          v[k] = (lane == 0 ? first[k] : before) | (v[k] << 16);
        }
        if (c + 1 < cols)
          *reinterpret_cast<uint32_t*>(to + c) = v[k];
        else if (c < cols)
          to[c] = (uint16_t)v[k];
      }
    }
  }
}

}  // namespace

int sum_splits(const float* part, int64_t ldp, int64_t split_stride, int splits, const SumArgs& out,
               int rows_total, cudaStream_t st) {
  const int64_t items = (int64_t)rows_total * ((out.cols + 3) / 4);
  const int64_t blocks = std::min<int64_t>((items + 255) / 256, (int64_t)sm_count() * 8);
  launch_dependent(sum_splits_kernel<false>, dim3((unsigned)blocks), 256, 0, st, part, ldp, split_stride, splits, out, rows_total,
                   TailArgs{});
  return check_launch("split sum", 1);
}

int sum_tail(const float* part, const Sched& s, const SumArgs& out, cudaStream_t st) {
  const int rows = (s.tiles_m * s.tiles_n - s.whole) * PM;
  const int64_t blocks = std::min<int64_t>((int64_t)rows * (BN / 4) / 256, (int64_t)sm_count() * 8);
  launch_dependent(sum_splits_kernel<true>, dim3((unsigned)blocks), 256, 0, st, part, (int64_t)BN, (int64_t)rows * BN, s.splits, out,
                   rows, TailArgs{s.tiles_m, s.tiles_n, s.group_m, s.whole});
  return check_launch("split sum", 1);
}

}  // namespace tc
}  // namespace pnft

using namespace pnft;
using namespace pnft::tc;

namespace pnft {
namespace tc {

int weight_grad(const char* what, const void* dy, int64_t lddy, const void* x, int64_t ldx, void* c0, void* c1, int64_t ldc,
                int64_t row_split, int64_t rows, int c_dtype, void* workspace, int64_t K, int64_t M, int64_t N, int dtype,
                int32_t* status, cudaStream_t st) {
  Args a;
  memset(&a, 0, sizeof(a));
  int rc = map_mnmajor(&a.ta[0], dy, M, K, lddy);
  if (!rc) rc = map_mnmajor(&a.tb[0], x, N, K, ldx);
  if (rc) return rc;
  a.idesc = idesc(dtype, true, true);
  a.status = status;
  const SumArgs c{{c0, c1}, ldc, (int)row_split, (int)rows, (int)N, nullptr, c_dtype, 0,
                  rows16(c0, ldc, dtype_size(c_dtype)) && rows16(c1, ldc, dtype_size(c_dtype))};
  return product<true, true>(what, a, c, static_cast<float*>(workspace), M, N, (K + BK - 1) / BK, 0, nullptr, st);
}

}  // namespace tc
}  // namespace pnft

extern "C" size_t pnft_weight_grad_workspace_size(int64_t K, int64_t M, int64_t N) {
  return K <= 0 ? 0 : product_workspace(M, N, (K + BK - 1) / BK);
}

extern "C" int pnft_weight_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, void* c0, void* c1, int64_t ldc,
                                int64_t row_split, int64_t rows, int c_dtype, void* workspace, size_t workspace_bytes,
                                int64_t K, int64_t M, int64_t N, int dtype, int32_t* status, void* stream) {
  if (K < 0 || M <= 0 || N <= 0 || M > (1 << 24) || N > (1 << 24) || K >= ((int64_t)1 << 31) - BK)
    return fail(PNFT_EINVAL, "weight_grad: bad shape K=%lld M=%lld N=%lld", (long long)K, (long long)M, (long long)N);
  if (!type16(dtype)) return fail(PNFT_EUNSUPPORTED, "weight_grad: bfloat16 or float16 operands expected");
  if (c_dtype < PNFT_DTYPE_F32 || c_dtype > PNFT_DTYPE_F16) return fail(PNFT_EINVAL, "weight_grad: unknown output type %d", c_dtype);
  if (!c0 || (row_split < M && !c1)) return fail(PNFT_EINVAL, "weight_grad: null output");
  if (row_split >= M) row_split = 0x7fffffff, rows = std::min(rows, M);  // one output
  if (row_split < M && row_split % BM) return fail(PNFT_EINVAL, "weight_grad: row_split must be a multiple of %d", BM);
  if (rows <= 0 || row_split < rows || (row_split < M && row_split + rows > M) || ldc < N) return fail(PNFT_EINVAL, "weight_grad: bad output layout");
  const int osize = c_dtype == PNFT_DTYPE_F32 ? 4 : 2;
  cudaStream_t st = as_stream(stream);
  if (K == 0) {
    for (int part = 0; part < (row_split < M ? 2 : 1); ++part) {
      char* c = static_cast<char*>(part ? c1 : c0);
      const int64_t n = std::min<int64_t>(rows, part ? M - row_split : M);
      if (cudaMemset2DAsync(c, (size_t)(ldc * osize), 0, (size_t)(N * osize), (size_t)n, st) != cudaSuccess)
        return check_launch("weight_grad memset", 0);
    }
    return PNFT_OK;
  }
  if (!tma_rows_ok(dy, lddy, M) || !tma_rows_ok(x, ldx, N))
    return fail(PNFT_EUNSUPPORTED, "weight_grad: operand rows must be 16-byte aligned (strides multiples of 8)");
  if (!device_is_sm100()) return fail(PNFT_EUNSUPPORTED, "weight_grad: needs an sm_100 device");
  const size_t need = pnft_weight_grad_workspace_size(K, M, N);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(PNFT_EINVAL, "weight_grad: workspace of %zu bytes < required %zu (16-byte aligned)", workspace_bytes, need);
  return weight_grad("weight_grad", dy, lddy, x, ldx, c0, c1, ldc, row_split, rows, c_dtype, workspace, K, M, N, dtype,
                     status, st);
}

extern "C" int pnft_copy_rows16(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols,
                                void* stream) {
  if (rows < 0 || cols < 0 || lds < 0 || ldd < cols) return fail(PNFT_EINVAL, "copy_rows16: bad layout");
  if (rows == 0 || cols == 0) return PNFT_OK;
  if (!src || !dst) return fail(PNFT_EINVAL, "copy_rows16: null pointer");
  if (!rows16(dst, ldd, 2) && (rows > 1 || reinterpret_cast<uintptr_t>(dst) % 16))
    return fail(PNFT_EUNSUPPORTED, "copy_rows16: destination rows must be 16-byte aligned");
  const uintptr_t any = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | (uintptr_t)(lds * 2) |
                        (uintptr_t)(ldd * 2) | (uintptr_t)(cols * 2);
  const int64_t w = any % 16 == 0 ? 16 : any % 4 == 0 ? 4 : 2, words = cols * 2 / w;
  const unsigned grid = (unsigned)std::min<int64_t>((rows + 7) / 8, (int64_t)sm_count() * 8);
  const char* s = static_cast<const char*>(src);
  char* d = static_cast<char*>(dst);
  cudaStream_t st = as_stream(stream);
  if (w == 16)
    launch_dependent(copy_rows_kernel<uint4>, dim3(grid), 256, 0, st, s, lds * 2, d, ldd * 2, rows, words);
  else if (w == 4)
    launch_dependent(copy_rows_kernel<uint32_t>, dim3(grid), 256, 0, st, s, lds * 2, d, ldd * 2, rows, words);
  else
    launch_dependent(copy_rows2_kernel, dim3(grid), 256, 0, st, static_cast<const uint16_t*>(src), lds, static_cast<uint16_t*>(dst), ldd,
                     rows, cols);
  return check_launch("copy_rows16", 1);
}
