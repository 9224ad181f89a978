// block_gemm.cu — C = A * B^T for e4m3 operands with a power-of-two scale
// for each block of 128 values.
//
//   C[m,n] = sum_g 2^(sa[m,g] - 127) 2^(sb[n',g] - 127) sum_{k in g} a[m,k] b[n,k],
//   n' = n, or n / 128 where B has blocks of 128 x 128
#include "block128.cuh"
#include "cmb_host.h"

namespace cmb {
namespace {

constexpr int kTile = 64, kStep = 32;

__device__ __forceinline__ float e4m3_value(uint8_t q) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

__device__ __forceinline__ float e8m0_value(uint32_t s) {
  return s == 255u ? __uint_as_float(0x7FC00000u)
                   : __uint_as_float(s == 0u ? 0x00400000u : s << 23);
}

struct GemmArgs {
  const uint8_t *A, *sa, *B, *sb;
  size_t lda, ld_sa, ldb, ld_sb;
  void *C;
  size_t ldc;
  int c_type, block_rows_b, M, N, K;
};

// 64 x 64 outputs per CTA, operands restored to fp32 in shared memory.
__global__ void __launch_bounds__(256) k_gemm_plain(const GemmArgs g) {
  __shared__ float sA[kStep][kTile + 1], sB[kStep][kTile + 1];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < g.K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int r = i / kStep, k = k0 + i % kStep;
      const int m = m0 + r, n = n0 + r;
      sA[i % kStep][r] = m < g.M && k < g.K
                             ? e4m3_value(g.A[(size_t)m * g.lda + k]) *
                                   e8m0_value(g.sa[(size_t)m * g.ld_sa + k / b128::kBlock])
                             : 0.0f;
      sB[i % kStep][r] =
          n < g.N && k < g.K
              ? e4m3_value(g.B[(size_t)n * g.ldb + k]) *
                    e8m0_value(g.sb[(size_t)(n / g.block_rows_b) * g.ld_sb + k / b128::kBlock])
              : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(sA[k][ty * 4 + i], sB[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= g.M || n >= g.N) continue;
      if (g.c_type == CMB_BF16)
        static_cast<__nv_bfloat16 *>(g.C)[(size_t)m * g.ldc + n] = __float2bfloat16_rn(acc[i][j]);
      else
        static_cast<float *>(g.C)[(size_t)m * g.ldc + n] = acc[i][j];
    }
}

}  // namespace
}  // namespace cmb

using namespace cmb;

extern "C" int cmb_gemm_e4m3_block128(const uint8_t *A, size_t lda, const uint8_t *scale_a,
                                      size_t ld_scale_a, const uint8_t *B, size_t ldb,
                                      const uint8_t *scale_b, size_t ld_scale_b, int block_rows_b,
                                      void *C, size_t ldc, int c_type, int M, int N, int K,
                                      int *status, cmb_stream_t stream) {
  const char *fn = "cmb_gemm_e4m3_block128";
  if (c_type != CMB_BF16 && c_type != CMB_F32)
    return fail(CMB_ERR_INVALID_ARG, "%s: c_type %d is not CMB_BF16 or CMB_F32", fn, c_type);
  if (block_rows_b != 1 && block_rows_b != b128::kBlock)
    return fail(CMB_ERR_INVALID_ARG, "%s: block_rows_b %d not 1 or 128", fn, block_rows_b);
  if (M < 0 || N < 0 || K < 0)
    return fail(CMB_ERR_INVALID_ARG, "%s: M %d, N %d, K %d", fn, M, N, K);
  if (reinterpret_cast<uintptr_t>(status) % 4)
    return fail(CMB_ERR_INVALID_ARG, "%s: status is not aligned to its type", fn);
  if (M == 0 || N == 0) return CMB_OK;
  const size_t celem = c_type == CMB_BF16 ? 2 : 4;
  if (C == nullptr || reinterpret_cast<uintptr_t>(C) % celem)
    return fail(CMB_ERR_INVALID_ARG, "%s: C is null or not aligned to its type", fn);
  if (ldc < (size_t)N) return fail(CMB_ERR_INVALID_ARG, "%s: rows of C overlap (ldc %zu)", fn, ldc);
  if (K == 0) {
    CMB_CUDA_TRY(cudaMemset2DAsync(C, ldc * celem, 0, (size_t)N * celem, M, stream));
    return CMB_OK;
  }
  if (A == nullptr || B == nullptr || scale_a == nullptr || scale_b == nullptr)
    return fail(CMB_ERR_INVALID_ARG, "%s: null operand", fn);
  if (!b128::aligned_to(A, lda, 16) || !b128::aligned_to(B, ldb, 16))
    return fail(CMB_ERR_INVALID_ARG, "%s: A and B must be 16-byte aligned, lda and ldb multiples "
                "of 16", fn);
  const size_t groups = b128::groups_of(K);
  if (lda < (size_t)K || ldb < (size_t)K || ld_scale_a < groups || ld_scale_b < groups)
    return fail(CMB_ERR_INVALID_ARG, "%s: rows of an operand or its scales overlap", fn);
  if (current_cc() != 100)
    return fail(CMB_ERR_UNSUPPORTED, "%s: needs an sm_100 device (found cc %d)", fn, current_cc());
  const GemmArgs g = {A, scale_a, B, scale_b, lda, ld_scale_a, ldb, ld_scale_b, C, ldc, c_type,
                      block_rows_b, M, N, K};
  const dim3 grid((N + kTile - 1) / kTile, (M + kTile - 1) / kTile);
  if (grid.y > 65535u) return fail(CMB_ERR_INVALID_ARG, "%s: M %d is too large", fn, M);
  k_gemm_plain<<<grid, 256, 0, stream>>>(g);
  CMB_LAUNCH_CHECK();
  return CMB_OK;
}
