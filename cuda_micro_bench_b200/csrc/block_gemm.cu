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
// steps of 16 or 32, with nothing padded to 128 of them, and a lane of the
// accumulator is a column of C, so a warp stores 32 neighbouring values of
// one row of C at any alignment.
//
// Scales travel apart from the values: a warp gathers the scale bytes of 16 K
// blocks of every row into shared memory, as words of four; for each four K
// blocks tcgen05.cp takes the words to TMEM, and the instruction descriptor of
// each MMA names the byte of the word its K block is.  Both places have two
// buffers.
//
// The tensor core adds to its fp32 accumulator by truncation, so a sum's error
// grows with K: 5.5e-7 of C (2-norm) at K = 2048, 2.7e-6 at 8192, against 3.6e-7
// for the same sums rounded to nearest.  For an fp32 C an accumulator takes at most
// 16 K blocks (kSumBlocks), for a bf16 C, which shows less, 256 (kSumBlocksBf16), and
// the parts are added in registers, rounded to nearest.
//
// Two kernels: k_gemm_pair for many tokens (tensor core and L2 delivery
// bound), k_gemm_split for few (bound by reading the weights once).
#include <cuda.h>

#include <cmath>
#include <mutex>

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
  bool w_vec, t_vec;         // scale rows can be read 16 bytes at a time
  bool bf16;                 // C's type
  int n;                     // token rows of an MMA
  int stages;
  int split;                 // CTAs that share a tile's K (k_gemm_split)
  int tmem_cols;             // TMEM columns to allocate (k_gemm_split)
  int sums;                  // accumulators in TMEM for a CTA's K (k_gemm_split)
  int *status;
};

constexpr int kMaxStages = 12;
constexpr int kWBytes = 128 * 128;      // a K block of 128 weight rows
constexpr int kScaleSlot = 512 + 1024;  // scale words of 128 weight rows and 256 token rows
constexpr int kSplitSlot = 512 + 512;   // the same with 128 token rows
constexpr int kScaleCol = 480;          // TMEM columns of the scales: 2 x 4 and 2 x 8
constexpr size_t kSmemMost = 227 * 1024 - 1024;  // less what is static
constexpr size_t kSmemHalf = 112 * 1024;         // two CTAs a SM
constexpr int kSplitThreads = 256;
// K blocks of an accumulator where C is fp32: as many as share a fetch of scales.
constexpr int kSumBlocks = 16;
// The same for a bf16 C.  32 of K are off by at most 4 u32 of the sum so far (2 for
// the addition and 2 for the products' alignment, both downwards; of positive terms
// that averages half the last), so 32768 of K by 2^-13 of C, 1/32 of the largest
// rounding to bf16.
constexpr int kSumBlocksBf16 = 256;

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// The scale bytes of K blocks 16 s .. 16 s + 15 of 4 U rows, each 32 behind the
// one before; rows behind the last give the last one's (the values there are
// zeros), K blocks behind the last anything, which no MMA reads.  32 lanes read
// 32 rows, so each load is 32 sectors: one for 16 K blocks, all in flight at
// once.  With a word for 4 K blocks and load the gather, not the tensor core,
// set the pace (1.0 us a K block of the 480-token tile).  Plain loads: the kernel
// may have started before the one that writes the scales ended, which loads
// through the read-only path do not allow for.
template <int U>
__device__ __forceinline__ void scale_pieces(uint4 (&v)[4 * U], const uint8_t *scale, size_t ld,
                                             int row, int rows, int shift, int s, int groups,
                                             bool vec) {
  const uint8_t *p[4 * U];
#pragma unroll
  for (int c = 0; c < 4 * U; ++c)
    p[c] = scale + static_cast<size_t>(min(row + 32 * c, rows - 1) >> shift) * ld + 16 * s;
  if (vec) {
#pragma unroll
    for (int c = 0; c < 4 * U; ++c) v[c] = *reinterpret_cast<const uint4 *>(p[c]);
  } else {
    const int last = groups - 1 - 16 * s;
#pragma unroll
    for (int c = 0; c < 4 * U; ++c) v[c] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int i = 0; i <= min(last, 15); ++i) {
      uint32_t byte[4 * U];
#pragma unroll
      for (int c = 0; c < 4 * U; ++c) byte[c] = p[c][i];
      const int word = i >> 2, at = 8 * (i & 3);
#pragma unroll
      for (int c = 0; c < 4 * U; ++c) {
        v[c].x |= word == 0 ? byte[c] << at : 0u;
        v[c].y |= word == 1 ? byte[c] << at : 0u;
        v[c].z |= word == 2 ? byte[c] << at : 0u;
        v[c].w |= word == 3 ? byte[c] << at : 0u;
      }
    }
  }
}

// Four words of each of U times 128 rows, for 4 times 4 K blocks, where the
// copies to TMEM look for them: lane r's four words are those of rows r, 32 +
// r, 64 + r and 96 + r.
template <int U>
__device__ __forceinline__ void put_pieces(uint32_t at, uint32_t slot_bytes,
                                           const uint4 (&v)[4 * U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint4 *q = v + 4 * u;
    st_shared_v4(at + 512 * u, q[0].x, q[1].x, q[2].x, q[3].x);
    st_shared_v4(at + 512 * u + slot_bytes, q[0].y, q[1].y, q[2].y, q[3].y);
    st_shared_v4(at + 512 * u + 2 * slot_bytes, q[0].z, q[1].z, q[2].z, q[3].z);
    st_shared_v4(at + 512 * u + 3 * slot_bytes, q[0].w, q[1].w, q[2].w, q[3].w);
  }
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The value of lane 0, which the compiler then knows to be the same in every
// lane: the roles' branches, and the operands that MMAs and loads take from
// uniform registers, stay out of the vector registers.
__device__ __forceinline__ int uniform(uint32_t v) {
  return static_cast<int>(__shfl_sync(0xffffffffu, v, 0));
}

// The rest of a wait whose phase was not complete at once: false after
// kWaitLimitNs, or once another role of the CTA has given up.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int *abort_flag,
                                       int *status) {
  const uint64_t deadline = dev::globaltimer() + dev::kWaitLimitNs;
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (__all_sync(0xffffffffu, dev::mbar_try_wait_cluster_acq(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0 || dev::globaltimer() > deadline)) break;
  }
  dev::report_status(status, CMB_ERR_TIMEOUT);
  *abort_flag = 1;
  return false;
}

// Waits of the whole warp.  Out of line from the second try on: with the whole
// bounded loop and a look at the abort flag in its path, a wait that is
// already over cost the issuing warp ~290 cycles, half a K block's MMAs.
struct Waiter {
  volatile int *abort_flag;
  int *status;
  __device__ __forceinline__ bool operator()(uint64_t *bar, uint32_t parity) const {
    const uint32_t b = dev::smem_addr(bar);
    return __all_sync(0xffffffffu, dev::mbar_try_wait(b, parity)) ||
           wait_long(b, parity, abort_flag, status);
  }
  // For a barrier that threads of the other CTA arrive on.
  __device__ __forceinline__ bool of_pair(uint64_t *bar, uint32_t parity) const {
    const uint32_t b = dev::smem_addr(bar);
    return __all_sync(0xffffffffu, dev::mbar_try_wait_cluster_acq(b, parity)) ||
           wait_long(b, parity, abort_flag, status);
  }
};

template <typename T>
__device__ __forceinline__ void store_as(T *p, float v) {
  *p = b128::from_float<T>(v);
}

// N accumulator columns, rows t .. t + N - 1 of C at column w, of which the
// first `rows` are there: 32 lanes write 32 neighbours of each row.
template <typename T, int N>
__device__ __forceinline__ void store_columns(const Args &g, int t, int w, int rows,
                                              const uint32_t *r) {
  T *p = static_cast<T *>(g.C) + static_cast<size_t>(t) * g.ldc + w;
  if (rows >= N) {
#pragma unroll
    for (int c = 0; c < N; ++c, p += g.ldc) store_as(p, __uint_as_float(r[c]));
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c, p += g.ldc)
      if (c < rows) store_as(p, __uint_as_float(r[c]));
  }
}

template <int N>
__device__ __forceinline__ void store_columns(const Args &g, int t, int w, const uint32_t *r) {
  if (w >= g.w_rows) return;
  if (g.bf16) store_columns<__nv_bfloat16, N>(g, t, w, g.t_rows - t, r);
  else store_columns<float, N>(g, t, w, g.t_rows - t, r);
}

__device__ __forceinline__ void store_c(const Args &g, int t, int w, float v) {
  const size_t at = static_cast<size_t>(t) * g.ldc + w;
  if (g.bf16) static_cast<__nv_bfloat16 *>(g.C)[at] = __float2bfloat16_rn(v);
  else static_cast<float *>(g.C)[at] = v;
}

// One CTA for each part of the K of a tile of 128 weight rows x n token rows;
// the `split` CTAs of a tile are one cluster and add their parts, in order,
// through distributed shared memory.
// Bound by reading the weights: 1 x 8192 x 8192 takes 13.8 us (67 MB, 10.2 us at
// the copy rate; 2-3 us of it are the launch and the pipe's start and end), 48 x
// 4096 x 8192 10.7 us (34 MB, 5.2 us).
// kParts: where TMEM does not hold an accumulator for each kSumBlocks (bf16 C:
// kSumBlocksBf16) K blocks, two of them take turns, one for each 16 K blocks whose
// scales come together, and warps 4-7 keep the sum, as in k_gemm_pair.  The sum's 128
// registers a thread leave room for one CTA a SM, as so many accumulators do.  The
// turns change with the batches of scales, outside the loop that issues MMAs: inside
// it they cost 7-17 % (128 x 18944 x 16384 91 us), here within 1 % of accumulators
// that grow with K (80).
//   warp 0 TMA loads, warp 1 MMAs, warp 2 scales, warps 4-7 accumulators
template <bool kParts>
__global__ void __launch_bounds__(kSplitThreads, kParts ? 1 : 2)
    k_gemm_split(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_t,
                 const Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ __align__(8) uint64_t sfull[2], sfree[2], bdone[2], done;
  __shared__ __align__(8) uint64_t tfull[2], tempty[2];  // kParts
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
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
      dev::mbar_init(dev::smem_addr(&bdone[s]), 1);
      if constexpr (kParts) {
        dev::mbar_init(dev::smem_addr(&tfull[s]), 1);
        dev::mbar_init(dev::smem_addr(&tempty[s]), 4);  // warps 4-7
      }
    }
    dev::mbar_init(dev::smem_addr(&done), 1);
    abort_flag = 0;
    dev::fence_mbar_init();
    dev::tma_prefetch_desc(&tm_w);
    dev::tma_prefetch_desc(&tm_t);
  }
  if (warp == 1) {
    tc::tmem_alloc<1>(dev::smem_addr(&tmem_holder), g.tmem_cols);
    tc::tmem_relinquish<1>();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = uniform(tmem_holder);
  const int each = (kb1 - kb0 + g.sums - 1) / g.sums;  // K blocks of an accumulator (!kParts)
  const Waiter wait{&abort_flag, g.status};
  dev::grid_dep_wait();
  dev::grid_dep_launch();

  // Warps 0 and 1 stay whole and elect a lane for each issue: their operands
  // are then warp-uniform, which the tensor core's and TMA's instructions need.
  if (warp == 0) {
    int s = 0, kb = kb0;
    uint32_t ph = 0;
    for (; kb < kb1; ++kb) {
      if (!wait(&empty[s], ph ^ 1)) break;
      uint8_t *w = ring + (size_t)s * stage_bytes;
      const uint32_t bar = dev::smem_addr(&full[s]);
      if (dev::elect_one()) {
        dev::mbar_arrive_expect_tx(bar, stage_bytes);
        dev::tma_load_2d(dev::smem_addr(w), &tm_w, kb * kBlock, w0, bar);
        dev::tma_load_2d(dev::smem_addr(w + kWBytes), &tm_t, kb * kBlock, t0, bar);
      }
      __syncwarp();
      if (++s == g.stages) s = 0, ph ^= 1;
    }
    // left early: the loads in flight land before the CTA ends
    if (kb < kb1)
      for (int i = 0; i < g.stages && kb - 1 - i >= kb0; ++i) {
        const int it = kb - 1 - i - kb0;
        dev::mbar_wait_bounded(dev::smem_addr(&full[it % g.stages]), (it / g.stages) & 1,
                               100000000ull);
      }
  } else if (warp == 1) {
    int s = 0, i = 0, sum = 0, left = each;
    uint32_t ph = 0;
    bool ok = true;
    for (int b = kb0 >> 2; b <= (kb1 - 1) >> 2 && ok; ++b, ++i) {
      const int slot = i & 1, piece = (b >> 2) - (kb0 >> 4), buf = piece & 1;
      if ((i == 0 || (b & 3) == 0) && !wait(&sfull[buf], (piece >> 1) & 1)) break;
      // the part before the last has been read from this part's accumulator
      if (kParts && (i == 0 || (b & 3) == 0) && !wait(&tempty[buf], ((piece >> 1) & 1) ^ 1)) break;
      // the MMAs of the batch before the last have read this slot's scales
      if (!wait(&bdone[slot], ((i >> 1) & 1) ^ 1)) break;
      tc::fence_after_sync();
      const uint32_t words = dev::smem_addr(scales + (4 * buf + (b & 3)) * kSplitSlot);
      const uint32_t sf_w = tmem + g.sums * g.n + 4 * slot, sf_t = sf_w + 8;
      if (dev::elect_one()) {
        tc::cp_scales<1>(sf_w, tc::rows16_desc(words));
        tc::cp_scales<1>(sf_t, tc::rows16_desc(words + 512));
      }
      __syncwarp();
      const int end = min(kb1, 4 * b + 4);
      for (int kb = max(kb0, 4 * b); kb < end; ++kb) {
        if (!wait(&full[s], ph)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        const uint32_t w = dev::smem_addr(ring + (size_t)s * stage_bytes);
        const uint64_t dw = tc::sw128_kmajor_desc(w), dt = tc::sw128_kmajor_desc(w + kWBytes);
        const uint32_t idesc = tc::instr_desc_block_scaled(128, g.n, kb & 3);
        const uint32_t d = kParts ? tmem + buf * g.n : tmem + sum * g.n;
        // of its accumulator
        const bool first = kParts ? kb == kb0 || (kb & 15) == 0 : left == each;
        if (dev::elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::mma_block_scaled<1>(d, dw + 2 * k, dt + 2 * k, idesc, sf_w, sf_t,
                                    (!first || k != 0) ? 1u : 0u);
          tc::commit<1>(dev::smem_addr(&empty[s]));
        }
        __syncwarp();
        if (++s == g.stages) s = 0, ph ^= 1;
        if (!kParts && --left == 0) left = each, ++sum;
      }
      if (dev::elect_one()) {
        tc::commit<1>(dev::smem_addr(&bdone[slot]));
        if ((b & 3) == 3) tc::commit<1>(dev::smem_addr(&sfree[buf]));
        if (kParts && ((b & 3) == 3 || end == kb1)) tc::commit<1>(dev::smem_addr(&tfull[buf]));
      }
      __syncwarp();
    }
    if (dev::elect_one()) tc::commit<1>(dev::smem_addr(&done));
    __syncwarp();
    // every MMA issued above is complete once `done` flips
    if (!dev::mbar_wait_bounded(dev::smem_addr(&done), 0))
      dev::report_status(g.status, CMB_ERR_TIMEOUT);
  } else if (warp == 2) {
    int i = 0;
    for (int b = kb0 >> 4; b <= (kb1 - 1) >> 4; ++b, ++i) {
      uint4 w[4], t[4];
      scale_pieces<1>(w, g.scale_w, g.ld_scale_w, w0 + lane, g.w_rows, g.w_shift, b, g.groups,
                      g.w_vec);
      scale_pieces<1>(t, g.scale_t, g.ld_scale_t, t0 + lane, g.t_rows, 0, b, g.groups, g.t_vec);
      const int buf = i & 1;
      if (!wait(&sfree[buf], ((i >> 1) & 1) ^ 1)) break;
      const uint32_t at = dev::smem_addr(scales + buf * 4 * kSplitSlot) + 16 * lane;
      put_pieces<1>(at, kSplitSlot, w);
      put_pieces<1>(at + 512, kSplitSlot, t);
      dev::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(dev::smem_addr(&sfull[buf]));
    }
  } else if (kParts && warp >= 4) {
    const int row = (warp & 3) * 32 + lane;
    uint32_t sum[8][16];  // n is at most 128
    bool ok = true;
    const int pieces = ((kb1 - 1) >> 4) - (kb0 >> 4) + 1;
    for (int j = 0; j < pieces; ++j) {
      const int a = j & 1;
      ok = wait(&tfull[a], (j >> 1) & 1);
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t at = tmem + (static_cast<uint32_t>(row & 96) << 16) + a * g.n;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (16 * c >= g.n) continue;
        if (j == 0) {
          tc::ld_32x32b_x16(at + 16 * c, sum[c]);
          tc::wait_ld();
        } else {
          uint32_t r[16];
          tc::ld_32x32b_x16(at + 16 * c, r);
          tc::wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sum[c][e] = __float_as_uint(__uint_as_float(sum[c][e]) + __uint_as_float(r[e]));
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(dev::smem_addr(&tempty[a]));
    }
    // every load has landed and every MMA has read it: the ring takes the sums
    float *mine = reinterpret_cast<float *>(ring) + row;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (16 * c >= g.n || !ok) continue;
      if (g.split > 1) {
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(16 * c + e) * 128] = __uint_as_float(sum[c][e]);
      } else {
        store_columns<16>(g, t0 + 16 * c, w0 + row, sum[c]);
      }
    }
  } else if (warp >= 4) {
    const bool ok = wait(&done, 0);
    tc::fence_after_sync();
    const int row = (warp & 3) * 32 + lane;
    float *mine = reinterpret_cast<float *>(ring) + row;
    for (int c0 = 0; c0 < g.n && ok; c0 += 16) {
      uint32_t r[16];
      const uint32_t at = tmem + (static_cast<uint32_t>(row & 96) << 16) + c0;
      tc::ld_32x32b_x16(at, r);
      tc::wait_ld();
      // (kb1 - kb0) / each of them have been written to, rounded up
      for (int u = 1; u * each < kb1 - kb0; ++u) {
        uint32_t more[16];
        tc::ld_32x32b_x16(at + u * g.n, more);
        tc::wait_ld();
#pragma unroll
        for (int c = 0; c < 16; ++c)
          r[c] = __float_as_uint(__uint_as_float(r[c]) + __uint_as_float(more[c]));
      }
      if (g.split > 1) {
#pragma unroll
        for (int c = 0; c < 16; ++c) mine[(c0 + c) * 128] = __uint_as_float(r[c]);
      } else {
        store_columns<16>(g, t0 + c0, w0 + row, r);
      }
    }
  }

  if (g.split > 1) {
    // Each CTA finishes 128 / split columns of the tile for every token, four
    // neighbours a thread, its parts' loads all in flight at once.
    tc::cluster_sync();
    const int quads = 32 / g.split;
    const int tokens = min(g.n, g.t_rows - t0);
    for (int i = threadIdx.x; i < quads * tokens; i += blockDim.x) {
      const int row = 4 * (part * quads + i % quads), t = i / quads;
      const uint32_t at = dev::smem_addr(reinterpret_cast<float *>(ring) + t * 128 + row);
      float4 v[8];
#pragma unroll
      for (int p = 0; p < 8; ++p)
        v[p] = p < g.split ? ld_cluster_f4(tc::map_to_cta(at, p)) : make_float4(0, 0, 0, 0);
      float4 sum = v[0];
#pragma unroll
      for (int p = 1; p < 8; ++p) {
        sum.x += v[p].x;
        sum.y += v[p].y;
        sum.z += v[p].z;
        sum.w += v[p].w;
      }
      const float out[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (w0 + row + c < g.w_rows) store_c(g, t0 + t, w0 + row + c, out[c]);
    }
    tc::cluster_sync();  // nobody's shared memory goes while another reads it
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc<1>(tmem, g.tmem_cols);
  }
}

// ------------------------------------------------ many tokens: CTA pairs

constexpr int kPairThreads = 384;

__device__ __forceinline__ void tile_at(int t, int tiles_w, int tiles_t, int &tw, int &tt) {
  // 8 rows of tiles advance together along the tokens, so the pairs at work
  // at one time share weights and tokens in L2.
  const int per_group = 8 * tiles_t, first = t / per_group * 8;
  const int high = min(tiles_w - first, 8), r = t % per_group;
  tw = first + r % high;
  tt = r / high;
}

// A cluster of two CTAs walks over tiles of 256 weight rows x n token rows (n
// a multiple of 32, up to 256): cta_group::2 MMAs issued by CTA 0, each CTA
// loading its 128 weight rows and half of the token rows.  Up to n = 224 TMEM
// holds two accumulators beside the scales, so a tile's MMAs run while the
// last one is stored.
// Bound by the tensor core and, in a long run, by its power: 8192 x 8192 x 8192
// takes 382-388 us alone (2.8-2.9 PFLOP/s, the pipe 91 % busy) and 440-470 us
// back to back, when the SM clock falls from 1.4 to 1.1-1.3 GHz.  L2 hands
// the SMs 4.9 GB meanwhile.  Wider tiles (256 x 448 in two parts of TMEM, 256 x
// 480) read less but store with no MMAs beside: 395 and 400 us.
// kPart > 0: each kPart K blocks of a tile go to the next of the accumulators, and the
// warps that read them keep the sum.  A bf16 C then has one at n = 256, which 256 K
// blocks (50 us) wait for no more than 1 us; an fp32 C stays at n <= 224.
//   warp 0 TMA loads, warp 1 MMAs, warp 2 scales, warps 4-11 accumulators
template <int kPart>
__global__ void __launch_bounds__(kPairThreads, 1)
    k_gemm_pair(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_t,
                const Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ __align__(8) uint64_t sfull[2], sfree[2], bdone[2], tfull[2], tempty[2], done;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  constexpr int kEach = kPart > 0 ? kPart : 1 << 30;     // K blocks of an accumulator
  const int n = g.n, bufs = 2 * n <= kScaleCol ? 2 : 1;  // accumulators
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = uniform(tc::cluster_ctarank());
  const int stage_bytes = kWBytes + n / 2 * 128;
  uint8_t *scales = ring + (size_t)g.stages * stage_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      dev::mbar_init(dev::smem_addr(&full[s]), 1);
      dev::mbar_init(dev::smem_addr(&empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      dev::mbar_init(dev::smem_addr(&sfull[s]), 2);  // both CTAs' words
      dev::mbar_init(dev::smem_addr(&sfree[s]), 1);
      dev::mbar_init(dev::smem_addr(&bdone[s]), 1);
      dev::mbar_init(dev::smem_addr(&tfull[s]), 1);
      dev::mbar_init(dev::smem_addr(&tempty[s]), 16);  // 8 warps of both CTAs
    }
    dev::mbar_init(dev::smem_addr(&done), 1);
    abort_flag = 0;
    dev::fence_mbar_init();
    dev::tma_prefetch_desc(&tm_w);
    dev::tma_prefetch_desc(&tm_t);
  }
  if (warp == 1) {
    tc::tmem_alloc<2>(dev::smem_addr(&tmem_holder), 512);
    tc::tmem_relinquish<2>();
  }
  tc::fence_before_sync();
  tc::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = uniform(tmem_holder);
  const int tiles_w = (g.w_rows + 255) / 256, tiles_t = (g.t_rows + n - 1) / n;
  const int tiles = tiles_w * tiles_t, first = blockIdx.x / 2, step = gridDim.x / 2;
  const Waiter wait{&abort_flag, g.status};
  dev::grid_dep_wait();
  dev::grid_dep_launch();

  // Warps 0 and 1 stay whole and elect a lane for each issue: their operands
  // are then warp-uniform, which the tensor core's and TMA's instructions need.
  if (warp == 0) {
    int s = 0, armed = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int tw, tt;
      tile_at(t, tiles_w, tiles_t, tw, tt);
      const int w_row = tw * 256 + rank * 128, t_row = tt * n + rank * (n / 2);
      for (int kb = 0; kb < g.groups; ++kb) {
        if (!wait(&empty[s], ph ^ 1)) {
          ok = false;
          break;
        }
        uint8_t *w = ring + (size_t)s * stage_bytes;
        // both CTAs' loads complete on CTA 0's barrier
        const uint32_t bar = tc::map_to_cta(dev::smem_addr(&full[s]), 0);
        if (dev::elect_one()) {
          if (rank == 0) dev::mbar_arrive_expect_tx(dev::smem_addr(&full[s]), 2 * stage_bytes);
          tc::tma_load_2d_pair(dev::smem_addr(w), &tm_w, kb * kBlock, w_row, bar);
          tc::tma_load_2d_pair(dev::smem_addr(w + kWBytes), &tm_t, kb * kBlock, t_row, bar);
        }
        __syncwarp();
        ++armed;
        if (++s == g.stages) s = 0, ph ^= 1;
      }
    }
    // left early: the loads in flight land before the pair ends
    if (!ok && rank == 0)
      for (int i = 0; i < g.stages && armed - 1 - i >= 0; ++i) {
        const int it = armed - 1 - i;
        dev::mbar_wait_bounded(dev::smem_addr(&full[it % g.stages]), (it / g.stages) & 1,
                               100000000ull);
      }
  } else if (warp == 1) {
    if (rank == 0) {
      int s = 0, j = 0;
      uint32_t ph = 0;
      unsigned i = 0, piece = 0;  // batches of four K blocks and of sixteen, over all tiles
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        int a = 0, from = 0;  // the accumulator and its first K block
        uint32_t d = 0;
        for (int b = 0; 4 * b < g.groups && ok; ++b, ++i) {
          if (4 * b % kEach == 0) {
            a = j % bufs, from = 4 * b, d = tmem + a * n;
            ok = wait.of_pair(&tempty[a], (static_cast<uint32_t>(j / bufs) & 1) ^ 1);
            if (!ok) break;
            ++j;
          }
          const int slot = i & 1, buf = piece & 1, kend = min(g.groups, 4 * b + 4);
          // the MMAs of the batch before the last have read this slot's scales
          if (((b & 3) == 0 && !wait.of_pair(&sfull[buf], (piece >> 1) & 1)) ||
              !wait(&bdone[slot], ((i >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t words = dev::smem_addr(scales + (4 * buf + (b & 3)) * kScaleSlot);
          const uint32_t sf_w = tmem + kScaleCol + 4 * slot, sf_t = tmem + kScaleCol + 8 + 8 * slot;
          if (dev::elect_one()) {
            tc::cp_scales<2>(sf_w, tc::rows16_desc(words));
            tc::cp_scales<2>(sf_t, tc::rows16_desc(words + 512));
            if (n > 128) tc::cp_scales<2>(sf_t + 4, tc::rows16_desc(words + 1024));
          }
          __syncwarp();
          for (int kb = 4 * b; kb < kend; ++kb) {
            if (!wait(&full[s], ph)) {
              ok = false;
              break;
            }
            tc::fence_after_sync();
            const uint32_t w = dev::smem_addr(ring + (size_t)s * stage_bytes);
            const uint64_t dw = tc::sw128_kmajor_desc(w), dt = tc::sw128_kmajor_desc(w + kWBytes);
            const uint32_t idesc = tc::instr_desc_block_scaled(256, n, kb & 3);
            if (dev::elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc::mma_block_scaled<2>(d, dw + 2 * k, dt + 2 * k, idesc, sf_w, sf_t,
                                        (kb != from || k != 0) ? 1u : 0u);
              tc::commit_pair(dev::smem_addr(&empty[s]));
            }
            __syncwarp();
            if (++s == g.stages) s = 0, ph ^= 1;
          }
          const bool last = (b & 3) == 3 || kend == g.groups;  // of its 16 K blocks
          if (dev::elect_one()) {
            tc::commit<2>(dev::smem_addr(&bdone[slot]));
            if (last) tc::commit_pair(dev::smem_addr(&sfree[buf]));
            if (kend == g.groups || kend % kEach == 0)
              tc::commit_pair(dev::smem_addr(&tfull[a]));
          }
          __syncwarp();
          if (last) ++piece;
        }
      }
      // every MMA issued above is complete once `done` flips
      if (dev::elect_one()) tc::commit<2>(dev::smem_addr(&done));
      __syncwarp();
      if (!dev::mbar_wait_bounded(dev::smem_addr(&done), 0))
        dev::report_status(g.status, CMB_ERR_TIMEOUT);
    }
  } else if (warp == 2) {
    unsigned i = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int tw, tt;
      tile_at(t, tiles_w, tiles_t, tw, tt);
      for (int b = 0; 16 * b < g.groups; ++b, ++i) {
        uint4 w[4], tv[8];
        scale_pieces<1>(w, g.scale_w, g.ld_scale_w, tw * 256 + rank * 128 + lane, g.w_rows,
                        g.w_shift, b, g.groups, g.w_vec);
        scale_pieces<2>(tv, g.scale_t, g.ld_scale_t, tt * n + lane, g.t_rows, 0, b, g.groups,
                        g.t_vec);
        const int buf = i & 1;
        ok = wait(&sfree[buf], ((i >> 1) & 1) ^ 1);
        if (!ok) break;
        const uint32_t at = dev::smem_addr(scales + buf * 4 * kScaleSlot) + 16 * lane;
        put_pieces<1>(at, kScaleSlot, w);
        put_pieces<2>(at + 512, kScaleSlot, tv);
        dev::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) dev::mbar_arrive_cluster(tc::map_to_cta(dev::smem_addr(&sfull[buf]), 0));
      }
    }
  } else if (warp >= 4) {
    const int q = warp & 3, h = (warp - 4) >> 2, chunks = n / 16;
    const auto hand_back = [&](int a) {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) dev::mbar_arrive_cluster(tc::map_to_cta(dev::smem_addr(&tempty[a]), 0));
    };
    int j = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int tw, tt;
      tile_at(t, tiles_w, tiles_t, tw, tt);
      const int w = tw * 256 + rank * 128 + q * 32 + lane;
      if constexpr (kPart == 0) {
        const int a = j % bufs;
        ok = wait(&tfull[a], static_cast<uint32_t>(j / bufs) & 1);
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t at = tmem + (static_cast<uint32_t>(q * 32) << 16) + a * n;
        for (int c = h; c < chunks; c += 2) {
          uint32_t r[16];
          tc::ld_32x32b_x16(at + 16 * c, r);
          tc::wait_ld();
          if (c + 2 >= chunks) hand_back(a);  // read to the end: hand it back, then store
          store_columns<16>(g, tt * n + 16 * c, w, r);
        }
        ++j;
      } else {
        // this warp's chunks of 16 columns: h, h + 2, ...
        constexpr int kChunks = kPart == kSumBlocks ? 7 : 8;
        uint32_t sum[kChunks][16];
        for (int from = 0; from < g.groups && ok; from += kPart, ++j) {
          const int a = j % bufs;
          ok = wait(&tfull[a], static_cast<uint32_t>(j / bufs) & 1);
          if (!ok) break;
          tc::fence_after_sync();
          const uint32_t at = tmem + (static_cast<uint32_t>(q * 32) << 16) + a * n + 16 * h;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if (h + 2 * c >= chunks) continue;
            if (from == 0) {
              tc::ld_32x32b_x16(at + 32 * c, sum[c]);
              tc::wait_ld();
            } else {
              uint32_t r[16];
              tc::ld_32x32b_x16(at + 32 * c, r);
              tc::wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                sum[c][e] = __float_as_uint(__uint_as_float(sum[c][e]) + __uint_as_float(r[e]));
            }
          }
          hand_back(a);
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (h + 2 * c < chunks) store_columns<16>(g, tt * n + 16 * (h + 2 * c), w, sum[c]);
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc<2>(tmem, 512);
  }
}

// ------------------------------------------------------------- launches

int launch_kernel(void (*kernel)(CUtensorMap, CUtensorMap, Args), const uint8_t *A, size_t lda,
                  const uint8_t *B, size_t ldb, Args g, int t_box, long long ctas, int cluster,
                  int threads, int slot_bytes, size_t smem_most, cudaStream_t stream) {
  const int stage_bytes = kWBytes + t_box * 128;
  g.stages = static_cast<int>((smem_most - 1024 - 8 * slot_bytes) / stage_bytes);
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  if (ctas > 0x7fffffffLL) return fail(CMB_ERR_INVALID_ARG, "gemm: too many tiles");
  CUtensorMap tw, tt;
  int rc = make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, B, g.w_rows, g.K, ldb, 128, kBlock,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = make_tmap_2d(&tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, A, g.t_rows, g.K, lda, t_box, kBlock,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  CMB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(kSmemMost)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)g.stages * stage_bytes + 8 * slot_bytes + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  // the prologue may run while the stream's last kernel ends
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tw, tt, g));
  return CMB_OK;
}

// Clusters of 1, 2, 4 and 8 CTAs of k_gemm_split that the device holds at one
// a SM (148, 74, 33 and 15 on a B200: clusters stay within a GPC).
struct ClusterRoom {
  int clusters[4];
};

ClusterRoom cluster_room() {
  constexpr int kMaxDevices = 64;
  static std::mutex mu;
  static ClusterRoom known[kMaxDevices];
  const int sms = current_sm_count();
  ClusterRoom room = {{sms, sms / 2, sms / 5, sms / 11}};  // where the query fails
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return room;
  std::lock_guard<std::mutex> lock(mu);
  if (known[device].clusters[0] != 0) return known[device];
  cudaFuncSetAttribute(k_gemm_split<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(kSmemMost));
  for (int i = 0; i < 4; ++i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << i);
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = kSmemMost;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << i;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, k_gemm_split<false>, &cfg) == cudaSuccess && n > 0)
      room.clusters[i] = n;
  }
  return known[device] = room;
}

// How a product is cut: `n` tokens a tile, the K of a tile over `split` CTAs
// (0: k_gemm_pair), and whether two CTAs share a SM.
struct Cut {
  int n, split;
  bool two;
};

long long tiles_of(const Args &g, int w, int n) {
  return static_cast<long long>((g.w_rows + w - 1) / w) * ((g.t_rows + n - 1) / n);
}

// The cut that takes least time by a model of both kernels in microseconds,
// fitted to 9000 timings (18 weight shapes from 128 x 8192 to 16384 x 2048,
// 1-8192 tokens, every cut): it picks one within 2 % of the fastest on
// average.  A K block takes a CTA ~0.27 us however few its tokens; a SM that
// two CTAs share, or a pair, is bound by the bytes that reach it (~0.13 us +
// 0.7 ns a token; 0.21 us + 0.5 ns; more where rows do not start on 128 bytes,
// `skewed`, and each 128 bytes of a row lie in two lines); all of it by
// reading the operands once (5.6 GB/ms).  What a cut adds: parts to sum (0.28 us
// a doubling + 20 ns a token), columns to store, which a short K does not
// hide, a wave that starts over.  Some of what it weighs (us): 1 x 8192 x 8192
// split 1/2/4: 19.5/14.3/13.7, pairs 20.4; 256 x 8192 x 8192 split 1 at n 128:
// 21.4, pairs 22.4; 1000 x 4600 x 2064 split 16.9, pairs at n 128/224/256:
// 17.3/20.3/13.3.
Cut choose_cut(const Args &g, bool skewed) {
  const ClusterRoom room = cluster_room();
  const double read = (static_cast<double>(g.w_rows) + g.t_rows) * g.K / 1e6;
  Cut best = {224, 0, false};
  double least = 1e30;
  // sums of several accumulators take two of them at once
  const bool sums = !g.bf16 && g.groups > kSumBlocks;
  for (int n = 32; n <= (sums ? 224 : 256); n += 32) {
    const long long waves = (tiles_of(g, 256, n) + current_sm_count() / 2 - 1) /
                            (current_sm_count() / 2);
    const double sum = g.groups * (0.205 + 0.0005 * n) * (skewed ? 1.26 : 1.0);
    const double store = g.bf16 ? 0.8 + 0.0075 * n : 0.52 + 0.0125 * n;
    const double us = 3.93 + fmax(waves * sum + (waves - 1) * fmax(0.0, store - 0.6 * sum),
                                  0.194 * read) +
                      0.007 * n + (2 * n > kScaleCol ? 3.0 * (waves - 1) : 0.0);
    if (us < least) least = us, best = {n, 0, false};
    if (n >= g.t_rows) break;
  }
  // even shares of the tokens in steps of 16, up to 128 a tile
  const int fewest = (g.t_rows + 127) / 128;
  int last = 0;
  for (int parts = fewest; parts < fewest + 8; ++parts) {
    // in 64 bits: parts is a 128th of up to 2^31
    const int n = static_cast<int>((static_cast<long long>(g.t_rows) + parts - 1) / parts + 15) /
                  16 * 16;
    if (n == last || (parts > 1 && n < 48)) continue;
    last = n;
    const long long tiles = tiles_of(g, 128, n);
    for (int i = 0; i < 4 && g.groups >= 1 << i; ++i) {
      const long long load = (tiles + room.clusters[i] - 1) / room.clusters[i];
      // k_gemm_split takes one tile a cluster: past two waves pairs, which
      // persist, are ahead, but for the single row of tiles of a wide layer
      if (load > 2 && (i > 0 || g.t_rows > n)) continue;
      const int blocks = (g.groups + (1 << i) - 1) >> i;
      double each = load * (0.134 + 0.0007 * n) * (skewed ? 1.7 : 1.0);
      if (load == 1) each = fmax(each, 0.266);
      const double us = 2.14 + fmax(blocks * each, 0.178 * read) + 0.0086 * n * load -
                        0.55 * (load - 1) + (i > 0 ? 0.28 * i + 0.02 * n * load : 0.0);
      // one CTA a SM where each has a place of its own and tiles are large:
      // twice the stages (128 x 8192 x 8192 by halves: 18.2 us against 21.1);
      // else two, and the next kernel's may start beside it (1 x 4096 x 4096
      // by quarters: 5.5 against 6.2)
      if (us < least) least = us, best = {n, 1 << i, load > 1 || n <= 48};
    }
  }
  return best;
}

int launch(const uint8_t *A, size_t lda, const uint8_t *B, size_t ldb, Args g,
           cudaStream_t stream) {
  Cut cut = choose_cut(g, lda % 128 != 0 || ldb % 128 != 0);
  g.n = cut.n;
  const int most = g.bf16 ? kSumBlocksBf16 : kSumBlocks;  // K blocks of an accumulator
  if (cut.split == 0) {
    const long long tiles = tiles_of(g, 256, g.n);
    if (tiles > 0x3fffffffLL) return fail(CMB_ERR_INVALID_ARG, "gemm: too many tiles");
    const int pairs = current_sm_count() / 2;
    const long long ctas = 2 * (tiles < pairs ? tiles : pairs);
    auto kernel = g.groups <= most ? k_gemm_pair<0>
                  : g.bf16         ? k_gemm_pair<kSumBlocksBf16>
                                   : k_gemm_pair<kSumBlocks>;
    return launch_kernel(kernel, A, lda, B, ldb, g, g.n / 2, ctas, 2, kPairThreads, kScaleSlot,
                         kSmemMost, stream);
  }
  g.split = cut.split;
  // an accumulator for each `most` of a CTA's K blocks: in half of TMEM or (one CTA a
  // SM) all of it, or two that take turns
  const int blocks = (g.groups + g.split - 1) / g.split;
  g.sums = (blocks + most - 1) / most;
  if (g.sums > (256 - 16) / g.n) cut.two = false;
  const bool parts = g.sums > (512 - 16) / g.n;
  if (parts) g.sums = 2;
  g.tmem_cols = 32;
  while (g.tmem_cols < g.sums * g.n + 16) g.tmem_cols *= 2;
  return launch_kernel(parts ? k_gemm_split<true> : k_gemm_split<false>, A, lda, B, ldb, g, g.n,
                       tiles_of(g, 128, g.n) * g.split, g.split, kSplitThreads, kSplitSlot,
                       cut.two ? kSmemHalf : kSmemMost, stream);
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
  // K: a tile's MMAs end well within the 2 s that a wait for them allows
  if (M < 0 || N < 0 || K < 0 || M > b128::kMostExtent || N > b128::kMostExtent || K > 1 << 28)
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
  g.w_vec = b128::aligned_to(scale_b, ld_scale_b, 16);
  g.t_vec = b128::aligned_to(scale_a, ld_scale_a, 16);
  g.bf16 = c_type == CMB_BF16;
  g.status = status;
  return launch(A, lda, B, ldb, g, stream);
}
