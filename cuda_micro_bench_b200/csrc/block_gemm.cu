// block_gemm.cu — C = A * B^T for e4m3 operands with a power-of-two scale
// for each block of 128 values, on the tensor core's own scaled MMA.
//
//   C[m,n] = sum_g 2^(sa[m,g] - 127) 2^(sb[n',g] - 127) sum_{k in g} a[m,k] b[n,k],
//   n' = n, or n / 128 where B has blocks of 128 x 128
//
// tcgen05.mma.kind::mxf8f6f4 multiplies each product of 32 values of K by
// two E8M0 scales, one for the row of each operand, inside the tensor core:
// a block of 128 is four such steps under one scale byte, so the sum stays in
// the fp32 accumulator in TMEM from the first group to the last and no
// partial product is scaled outside.
//
// The MMA's 128-row side is B (the weights) and its N side is A (the
// tokens): C^T = B * A^T.  A tile then takes as many tokens as there are, in
// steps of 16, with nothing padded to 128 of them, and a lane of the
// accumulator is a column of C, so a warp stores 32 neighbouring values of
// one row of C at any alignment.
//
// Scales travel apart from the values: a warp gathers the scale bytes of
// four K blocks (one 32-bit word for each row) into shared memory, tcgen05.cp
// takes them to TMEM, and the instruction descriptor of each MMA names the
// byte of the word its K block is.  Two buffers of words: the gather of four
// K blocks ahead waits for the MMAs of the last four but one.
#include <cuda.h>

#include "block128.cuh"
#include "cmb_host.h"
#include "tcgen05.cuh"

namespace cmb {

int make_tmap_2d(CUtensorMap *map, CUtensorMapDataType dtype, const void *base, uint64_t rows,
                 uint64_t cols, uint64_t pitch_bytes, uint32_t box_rows, uint32_t box_cols,
                 CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promo);

namespace {

using b128::kBlock;

// "w": B's rows (columns of C); "t": A's rows (rows of C).
struct Args {
  const uint8_t *scale_w, *scale_t;
  size_t ld_scale_w, ld_scale_t, ldc;
  void *C;
  int w_rows, t_rows, K, groups;
  int w_shift;               // 7 where B has blocks of 128 x 128, else 0
  bool w_words, t_words;     // scale rows can be read in aligned words
  bool bf16;                 // C's type
  int n;                     // token rows of an MMA
  int stages;
  int split;                 // CTAs that share a tile's K
  int *status;
};

constexpr int kMaxStages = 12;
constexpr int kWBytes = 128 * 128;      // a K block of 128 weight rows
constexpr int kScaleSlot = 512 + 1024;  // scale words of 128 weight rows and 256 token rows
constexpr int kScaleCol = 480;          // TMEM columns of the scales: 2 x 4 and 2 x 8
constexpr size_t kSmemMost = 227 * 1024 - 1024;  // less what is static

// The scale bytes of K blocks 4b .. 4b + 3 of a row, 0 where there is none.
__device__ __forceinline__ uint32_t scale_word(const uint8_t *scale, size_t ld, int row, int rows,
                                               int shift, int b, int groups, bool words) {
  if (row >= rows) return 0u;
  const uint8_t *p = scale + static_cast<size_t>(row >> shift) * ld + 4 * b;
  const int n = groups - 4 * b;
  if (words && n >= 4) return __ldg(reinterpret_cast<const uint32_t *>(p));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) w |= static_cast<uint32_t>(__ldg(p + i)) << (8 * i);
  return w;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void store_c(const Args &g, int t, int w, float v) {
  const size_t at = static_cast<size_t>(t) * g.ldc + w;
  if (g.bf16) static_cast<__nv_bfloat16 *>(g.C)[at] = __float2bfloat16_rn(v);
  else static_cast<float *>(g.C)[at] = v;
}

// One CTA for each part of the K of a tile of 128 weight rows x n token rows;
// the `split` CTAs of a tile are one cluster and add their parts, in order,
// through distributed shared memory.
//   warp 0 TMA loads, warp 1 MMAs, warp 2 scales, warps 4-7 accumulator
__global__ void __launch_bounds__(256, 1)
    k_gemm_split(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_t,
                 const Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ __align__(8) uint64_t sfull[2], sfree[2], done;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = kWBytes + g.n * 128;
  uint8_t *scales = ring + (size_t)g.stages * stage_bytes;
  const int part = blockIdx.x % g.split, tile = blockIdx.x / g.split;
  const int tiles_t = (g.t_rows + g.n - 1) / g.n;
  const int w0 = tile / tiles_t * 128, t0 = tile % tiles_t * g.n;
  const int kb0 = static_cast<int>(static_cast<long long>(g.groups) * part / g.split);
  const int kb1 = static_cast<int>(static_cast<long long>(g.groups) * (part + 1) / g.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      dev::mbar_init(dev::smem_addr(&full[s]), 1);
      dev::mbar_init(dev::smem_addr(&empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      dev::mbar_init(dev::smem_addr(&sfull[s]), 1);
      dev::mbar_init(dev::smem_addr(&sfree[s]), 1);
    }
    dev::mbar_init(dev::smem_addr(&done), 1);
    abort_flag = 0;
    dev::fence_mbar_init();
    dev::tma_prefetch_desc(&tm_w);
    dev::tma_prefetch_desc(&tm_t);
  }
  if (warp == 1) {
    tc::tmem_alloc<1>(dev::smem_addr(&tmem_holder), 512);
    tc::tmem_relinquish<1>();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_holder;
  // A wait that gives up reports and makes every role leave; false once one has.
  const auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (dev::mbar_wait_bounded(dev::smem_addr(bar), parity) &&
        *static_cast<volatile int *>(&abort_flag) == 0)
      return true;
    dev::report_status(g.status, CMB_ERR_TIMEOUT);
    atomicExch(&abort_flag, 1);
    return false;
  };

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, kb = kb0;
      uint32_t ph = 0;
      for (; kb < kb1; ++kb) {
        if (!wait(&empty[s], ph ^ 1)) break;
        uint8_t *w = ring + (size_t)s * stage_bytes;
        const uint32_t bar = dev::smem_addr(&full[s]);
        dev::mbar_arrive_expect_tx(bar, stage_bytes);
        dev::tma_load_2d(dev::smem_addr(w), &tm_w, kb * kBlock, w0, bar);
        dev::tma_load_2d(dev::smem_addr(w + kWBytes), &tm_t, kb * kBlock, t0, bar);
        if (++s == g.stages) s = 0, ph ^= 1;
      }
      // left early: the loads in flight land before the CTA ends
      if (kb < kb1)
        for (int i = 0; i < g.stages && kb - 1 - i >= kb0; ++i) {
          const int it = kb - 1 - i - kb0;
          dev::mbar_wait_bounded(dev::smem_addr(&full[it % g.stages]), (it / g.stages) & 1,
                                 100000000ull);
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int s = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int b = kb0 >> 2; b <= (kb1 - 1) >> 2 && ok; ++b, ++i) {
        const int slot = i & 1;
        if (!wait(&sfull[slot], (i >> 1) & 1)) break;
        tc::fence_after_sync();
        const uint32_t words = dev::smem_addr(scales + slot * kScaleSlot);
        const uint32_t sf_w = tmem + kScaleCol + 4 * slot, sf_t = tmem + kScaleCol + 8 + 8 * slot;
        tc::cp_scales<1>(sf_w, tc::rows16_desc(words));
        tc::cp_scales<1>(sf_t, tc::rows16_desc(words + 512));
        if (g.n > 128) tc::cp_scales<1>(sf_t + 4, tc::rows16_desc(words + 1024));
        for (int kb = max(kb0, 4 * b); kb < min(kb1, 4 * b + 4); ++kb) {
          if (!wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t w = dev::smem_addr(ring + (size_t)s * stage_bytes);
          const uint64_t dw = tc::sw128_kmajor_desc(w), dt = tc::sw128_kmajor_desc(w + kWBytes);
          const uint32_t idesc = tc::instr_desc_block_scaled(128, g.n, kb & 3);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::mma_block_scaled<1>(tmem, dw + 2 * k, dt + 2 * k, idesc, sf_w, sf_t,
                                    (kb != kb0 || k != 0) ? 1u : 0u);
          tc::commit<1>(dev::smem_addr(&empty[s]));
          if (++s == g.stages) s = 0, ph ^= 1;
        }
        tc::commit<1>(dev::smem_addr(&sfree[slot]));
      }
      tc::commit<1>(dev::smem_addr(&done));
      // every MMA issued above is complete once `done` flips
      if (!dev::mbar_wait_bounded(dev::smem_addr(&done), 0))
        dev::report_status(g.status, CMB_ERR_TIMEOUT);
    }
  } else if (warp == 2) {
    int i = 0;
    for (int b = kb0 >> 2; b <= (kb1 - 1) >> 2; ++b, ++i) {
      uint32_t w[4], t[2][4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        w[c] = scale_word(g.scale_w, g.ld_scale_w, w0 + 32 * c + lane, g.w_rows, g.w_shift, b,
                          g.groups, g.w_words);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 128 * j + 32 * c + lane;
          t[j][c] = r < g.n ? scale_word(g.scale_t, g.ld_scale_t, t0 + r, g.t_rows, 0, b, g.groups,
                                         g.t_words)
                            : 0u;
        }
      }
      const int slot = i & 1;
      if (!wait(&sfree[slot], ((i >> 1) & 1) ^ 1)) break;
      const uint32_t words = dev::smem_addr(scales + slot * kScaleSlot) + 16 * lane;
      st_shared_v4(words, w);
      st_shared_v4(words + 512, t[0]);
      if (g.n > 128) st_shared_v4(words + 1024, t[1]);
      dev::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(dev::smem_addr(&sfull[slot]));
    }
  } else if (warp >= 4) {
    const bool ok = wait(&done, 0);
    tc::fence_after_sync();
    const int row = (warp & 3) * 32 + lane;
    float *mine = reinterpret_cast<float *>(ring) + row;
    for (int c0 = 0; c0 < g.n && ok; c0 += 16) {
      uint32_t r[16];
      tc::ld_32x32b_x16(tmem + (static_cast<uint32_t>(row & 96) << 16) + c0, r);
      tc::wait_ld();
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        if (g.split > 1)
          mine[(c0 + c) * 128] = __uint_as_float(r[c]);
        else if (t0 + c0 + c < g.t_rows && w0 + row < g.w_rows)
          store_c(g, t0 + c0 + c, w0 + row, __uint_as_float(r[c]));
      }
    }
  }

  if (g.split > 1) {
    // Each CTA finishes 128 / split columns of the tile for every token.
    tc::cluster_sync();
    const int rows = 128 / g.split, first = part * rows;
    const int tokens = min(g.n, g.t_rows - t0);
    for (int i = threadIdx.x; i < rows * tokens; i += blockDim.x) {
      const int row = first + i % rows, t = i / rows;
      if (w0 + row >= g.w_rows) continue;
      const uint32_t at = dev::smem_addr(reinterpret_cast<float *>(ring) + t * 128 + row);
      float v = 0.0f;
      for (int p = 0; p < g.split; ++p) v += ld_cluster_f32(tc::map_to_cta(at, p));
      store_c(g, t0 + t, w0 + row, v);
    }
    tc::cluster_sync();  // nobody's shared memory goes while another reads it
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc<1>(tmem, 512);
  }
}

int launch_split(const uint8_t *A, size_t lda, const uint8_t *B, size_t ldb, Args g,
                 cudaStream_t stream) {
  // Even shares of the tokens, in steps of 16.
  const int tiles_t = (g.t_rows + 255) / 256;
  g.n = ((g.t_rows + tiles_t - 1) / tiles_t + 15) / 16 * 16;
  const long long tiles = static_cast<long long>((g.w_rows + 127) / 128) *
                          ((g.t_rows + g.n - 1) / g.n);
  g.split = 1;
  while (g.split < 8 && tiles * g.split * 2 <= current_sm_count() && g.groups >= g.split * 2)
    g.split *= 2;
  if (tiles * g.split > 0x7fffffffLL) return fail(CMB_ERR_INVALID_ARG, "gemm: too many tiles");
  const int stage_bytes = kWBytes + g.n * 128;
  g.stages = static_cast<int>((kSmemMost - 1024 - 2 * kScaleSlot) / stage_bytes);
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  const size_t smem = (size_t)g.stages * stage_bytes + 2 * kScaleSlot + 1024;
  CUtensorMap tw, tt;
  int rc = make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, g.w_rows, g.K, ldb, 128, kBlock,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = make_tmap_2d(&tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, g.t_rows, g.K, lda, g.n, kBlock,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  CMB_CUDA_TRY(cudaFuncSetAttribute(k_gemm_split, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(kSmemMost)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * g.split));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = g.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_gemm_split, tw, tt, g));
  return CMB_OK;
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
  if (block_rows_b != 1 && block_rows_b != kBlock)
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
  Args g = {};
  g.scale_w = scale_b;
  g.scale_t = scale_a;
  g.ld_scale_w = ld_scale_b;
  g.ld_scale_t = ld_scale_a;
  g.C = C;
  g.ldc = ldc;
  g.w_rows = N;
  g.t_rows = M;
  g.K = K;
  g.groups = static_cast<int>(groups);
  g.w_shift = block_rows_b == 1 ? 0 : 7;
  g.w_words = b128::aligned_to(scale_b, ld_scale_b, 4);
  g.t_words = b128::aligned_to(scale_a, ld_scale_a, 4);
  g.bf16 = c_type == CMB_BF16;
  g.status = status;
  return launch_split(A, lda, B, ldb, g, stream);
}
