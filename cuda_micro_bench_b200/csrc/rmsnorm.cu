// rmsnorm.cu — root-mean-square norm with the residual's addition and a
// block-scaled e4m3 output, and its backward pass.
//
//   h = x + r, rstd = (mean h^2 + eps)^(-1/2), y = h rstd w, (q, s) = y in e4m3
//   g = dy w, dx = rstd (g - h rstd^2 mean(g h)) + dh, dw = sum_rows dy h rstd
//
// Memory bound.  h is rounded to the rows' type before the mean: the norm,
// its backward pass and every later reader then see the same h.  Sums and
// statistics are fp32, in a fixed order.
//
// A CTA works on a whole row.  Two ways to read rows (template kRing):
//   ring    rows that start and end on 16 bytes, several rows a CTA: a thread
//           keeps the next rows on their way into shared memory with bulk
//           copies, so loads never wait for a row's reduction.
//   direct  everything else, and calls with no more rows than CTAs, whose
//           latency is one load.
#include "block128.cuh"
#include "cmb_host.h"

namespace cmb {
namespace {

using b128::Raw8;

constexpr int kMaxParts = 1024;  // CTAs, each with a row of partial weight gradients
// Rows in the ring.  Two leave room for two CTAs of a wide row on a SM, which
// counts for more than depth: the backward pass of 8192 x 8192 bf16 takes 90 us
// with two, 108 with three or four (one CTA a SM); the norm 81, 80 and 102.
constexpr int kStages = 2;

// Sum over the CTA, the same value in every thread.  `part` holds one float
// for each warp; two calls in a row use different ones.
__device__ __forceinline__ float cta_sum(float v, float *part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) part[warp] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = lane < warps ? part[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows of up to three matrices on their way through shared memory: row i of
// a CTA (its rows are blockIdx.x, + gridDim.x, ...) in stage i % kStages.
struct Ring {
  const uint8_t *src[3];
  size_t pitch[3];
  int n;          // matrices
  uint32_t bytes;  // of a row of one of them
  uint8_t *mem;
  uint64_t *full;

  __device__ __forceinline__ void load(int i, int rows) const {
    const long long row = blockIdx.x + static_cast<long long>(i) * gridDim.x;
    if (row >= rows) return;
    const int s = i % kStages;
    const uint32_t bar = dev::smem_addr(full + s);
    dev::mbar_arrive_expect_tx(bar, bytes * n);
    for (int k = 0; k < n; ++k)
      dev::bulk_load(dev::smem_addr(mem + (size_t)(s * n + k) * bytes), src[k] + row * pitch[k],
                     bytes, bar);
  }
  __device__ __forceinline__ void start(int rows) const {
    if (threadIdx.x == 0) {
      for (int s = 0; s < kStages; ++s) dev::mbar_init(dev::smem_addr(full + s), 1);
      dev::fence_mbar_init();
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int s = 0; s < kStages; ++s) load(s, rows);
  }
  // Waits for row i; a bulk copy of this GPU's own memory ends, or the launch
  // has failed as a whole.
  __device__ __forceinline__ void wait(int i) const {
    dev::mbar_wait_bounded(dev::smem_addr(full + i % kStages), (i / kStages) & 1);
  }
  template <typename T>
  __device__ __forceinline__ const T *row(int i, int k) const {
    return reinterpret_cast<const T *>(mem + (size_t)(i % kStages * n + k) * bytes);
  }
};

struct NormArgs {
  const void *x, *residual, *weight;
  void *h, *y;
  uint8_t *q, *scale;
  float *rstd;
  size_t ld_x, ld_r, ld_h, ld_y, ld_q, ld_scale;
  float eps;
  int rows, cols;
  bool x_vec, r_vec, w_vec, h_vec, y_vec, q_vec;
};

// The e4m3 values and scales of 8 columns of a row; 16 neighbouring threads
// have a block of 128.
__device__ __forceinline__ void store_quantized(const NormArgs &a, int row, int col,
                                                const float (&y)[8]) {
  const int n = a.cols - col;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, b128::magnitude_bits(y[j]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool any = __any_sync(0xffffffffu, top >= b128::kInfBits);
  if (any) {  // the scale is that of the finite values
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, b128::finite_magnitude(y[j]));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    top = __float_as_uint(m);
  }
  const uint32_t byte = b128::scale_byte(__uint_as_float(top));
  const float inv = b128::scale_reciprocal(byte);
  if (n > 0) {
    b128::store_bytes(a.q + (size_t)row * a.ld_q + col,
                      any ? b128::e4m3x8<true>(y, inv) : b128::e4m3x8<false>(y, inv), n, a.q_vec);
    if ((threadIdx.x & 15) == 0)
      a.scale[(size_t)row * a.ld_scale + col / b128::kBlock] = static_cast<uint8_t>(byte);
  }
}

// A thread's chunks of the weights: kept in registers, or, where a row has
// more than two chunks a thread, read again for each row.
template <typename W, int NV>
struct Weight {
  const W *p;
  bool vec;
  Raw8<W> kept[NV <= 2 ? NV : 1];

  __device__ __forceinline__ Weight(const void *weight, bool aligned, int cols)
      : p(static_cast<const W *>(weight)), vec(aligned) {
    if constexpr (NV <= 2) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * blockDim.x + threadIdx.x) * 8;
        kept[i] = load(col, cols - col);
      }
    }
  }
  __device__ __forceinline__ Raw8<W> load(int col, int n) const {
    return n > 0 ? b128::load8_edge(p + col, n, vec) : Raw8<W>{};
  }
  __device__ __forceinline__ Raw8<W> chunk(int i, int col, int n) const {
    if constexpr (NV <= 2) return kept[i];
    else return load(col, n);
  }
};

// Thread t holds the chunks of 8 columns t, t + blockDim, ...: 16
// neighbouring threads hold a block of 128.
template <typename T, typename W, int NV, bool kRing>
__global__ void __launch_bounds__(1024, 1) k_rmsnorm(const NormArgs a) {
  __shared__ float part[2][32];
  __shared__ __align__(8) uint64_t full[kStages];
  extern __shared__ __align__(16) uint8_t rows_mem[];
  const T *x = static_cast<const T *>(a.x), *res = static_cast<const T *>(a.residual);
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  Ring ring;
  if constexpr (kRing) {
    ring = {{static_cast<const uint8_t *>(a.x), static_cast<const uint8_t *>(a.residual), nullptr},
            {a.ld_x * sizeof(T), a.ld_r * sizeof(T), 0},
            res != nullptr ? 2 : 1,
            static_cast<uint32_t>(a.cols * sizeof(T)),
            rows_mem,
            full};
    ring.start(a.rows);
  }
  const Weight<W, NV> weight(a.weight, a.w_vec, a.cols);
  int it = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, ++it) {
    Raw8<T> h[NV];  // as it is stored
    float sq = 0.0f;
    if constexpr (kRing) ring.wait(it);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      Raw8<T> raw{}, add{};
      if (n > 0) {
        if constexpr (kRing) {
          raw = b128::load8(ring.row<T>(it, 0) + col);
          if (res != nullptr) add = b128::load8(ring.row<T>(it, 1) + col);
        } else {
          raw = b128::load8_edge(x + (size_t)row * a.ld_x + col, n, a.x_vec);
          if (res != nullptr) add = b128::load8_edge(res + (size_t)row * a.ld_r + col, n, a.r_vec);
        }
        if (res != nullptr) {
          float v[8], u[8];
          b128::unpack(raw, v);
          b128::unpack(add, u);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += u[j];
          b128::pack(v, raw);
          b128::store8_edge(static_cast<T *>(a.h) + (size_t)row * a.ld_h + col, raw, n, a.h_vec);
        }
      }
      h[i] = raw;
      float v[8];
      b128::unpack(raw, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[j], v[j], sq);
    }
    sq = cta_sum(sq, part[it & 1]);
    if constexpr (kRing)
      if (threadIdx.x == 0) ring.load(it + kStages, a.rows);  // every thread has its chunks
    const float rstd = 1.0f / sqrtf(sq / static_cast<float>(a.cols) + a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      float y[8], wv[8];
      b128::unpack(h[i], y);
      b128::unpack(weight.chunk(i, col, n), wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = y[j] * rstd * wv[j];
        // behind the row's end: not 0 * inf, which would be NaN
        if (j >= n) y[j] = 0.0f;
      }
      if (a.y != nullptr && n > 0) {
        Raw8<T> out;
        b128::pack(y, out);
        b128::store8_edge(static_cast<T *>(a.y) + (size_t)row * a.ld_y + col, out, n, a.y_vec);
      }
      if (a.q != nullptr) store_quantized(a, row, col, y);
    }
  }
}

struct NormBackArgs {
  const void *dy, *h, *dh, *weight;
  const float *rstd;
  void *dx;
  float *parts;  // gridDim.x rows of cols partial weight gradients, or NULL
  size_t ld_dy, ld_h, ld_dh, ld_dx, ld_parts;
  int rows, cols;
  bool dy_vec, h_vec, dh_vec, w_vec, dx_vec;
};

// Both passes over a row read it from where it lies, the ring's shared memory
// or (direct) global memory, so a thread holds no more of it than a chunk; the
// weight gradient of its columns stays in registers from row to row.
template <typename T, typename W, int NV, bool kRing>
__global__ void __launch_bounds__(1024, 1) k_rmsnorm_back(const NormBackArgs a) {
  __shared__ float part[2][32];
  __shared__ __align__(8) uint64_t full[kStages];
  extern __shared__ __align__(16) uint8_t rows_mem[];
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  Ring ring;
  if constexpr (kRing) {
    ring = {{static_cast<const uint8_t *>(a.dy), static_cast<const uint8_t *>(a.h),
             static_cast<const uint8_t *>(a.dh)},
            {a.ld_dy * sizeof(T), a.ld_h * sizeof(T), a.ld_dh * sizeof(T)},
            a.dh != nullptr ? 3 : 2,
            static_cast<uint32_t>(a.cols * sizeof(T)),
            rows_mem,
            full};
    ring.start(a.rows);
  }
  const Weight<W, NV> weight(a.weight, a.w_vec, a.cols);
  float dw[NV][8] = {};
  int it = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, ++it) {
    const auto load = [&](int k, const void *p, size_t ld, int col, int n, bool vec) {
      if constexpr (kRing) return b128::load8(ring.row<T>(it, k) + col);
      else return b128::load8_edge(static_cast<const T *>(p) + (size_t)row * ld + col, n, vec);
    };
    const float rstd = a.rstd[row];
    float along = 0.0f;
    if constexpr (kRing) ring.wait(it);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      if (n <= 0) continue;
      float g[8], u[8], wv[8];
      b128::unpack(load(0, a.dy, a.ld_dy, col, n, a.dy_vec), g);
      b128::unpack(load(1, a.h, a.ld_h, col, n, a.h_vec), u);
      b128::unpack(weight.chunk(i, col, n), wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // behind the row's end: not 0 * inf, which would be NaN
        const float unit = j < n ? u[j] * rstd : 0.0f;
        dw[i][j] = fmaf(g[j], unit, dw[i][j]);
        along = fmaf(g[j] * wv[j], unit, along);
      }
    }
    const float mean = cta_sum(along, part[it & 1]) / static_cast<float>(a.cols);
    // every thread is past the last row: its place takes another
    if constexpr (kRing)
      if (threadIdx.x == 0 && it > 0) ring.load(it - 1 + kStages, a.rows);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      if (n <= 0) continue;
      float g[8], u[8], wv[8], past[8] = {};
      b128::unpack(load(0, a.dy, a.ld_dy, col, n, a.dy_vec), g);
      b128::unpack(load(1, a.h, a.ld_h, col, n, a.h_vec), u);
      if (a.dh != nullptr) b128::unpack(load(2, a.dh, a.ld_dh, col, n, a.dh_vec), past);
      b128::unpack(weight.chunk(i, col, n), wv);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        g[j] = fmaf(rstd, g[j] * wv[j] - u[j] * rstd * mean, past[j]);
      Raw8<T> out;
      b128::pack(g, out);
      b128::store8_edge(static_cast<T *>(a.dx) + (size_t)row * a.ld_dx + col, out, n, a.dx_vec);
    }
  }
  if (a.parts != nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8;
      Raw8<float> r;
      b128::pack(dw[i], r);
      // the workspace's rows are padded to whole chunks
      if (col < a.cols) b128::store8(a.parts + (size_t)blockIdx.x * a.ld_parts + col, r);
    }
  }
}

// dweight[c] = sum of the partial rows: 32 columns a CTA, 32 threads take
// every 32nd row each, in order, and their sums are added in a tree.
__global__ void __launch_bounds__(1024) k_sum_parts(const float *__restrict__ parts, size_t ld,
                                                    int n, int cols, float *__restrict__ out) {
  __shared__ float sums[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int r = threadIdx.y; r < n; r += 32) s += parts[(size_t)r * ld + c];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sums[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int at = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && at < cols) out[at] = s;
}

size_t parts_pitch(int cols) { return ((size_t)cols + 63) / 64 * 64; }

// Chunks of 8 columns a thread, and threads (at most 1024) that hold a row.
int chunks_for(int cols) { return cols <= 4096 ? 1 : cols <= 16384 ? 2 : 4; }

int threads_for(int cols, int nv) {
  const int chunks = (cols + 7) / 8;
  const int t = (chunks + nv - 1) / nv;
  return (t + 31) / 32 * 32;
}

template <typename A>
int launch_rows(void (*kernel)(A), const A &a, int grid, int threads, size_t smem,
                cudaStream_t stream) {
  if (smem > 48 * 1024)
    CMB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(smem)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return CMB_OK;
}

// How many CTAs walk over the rows: at most what fits on the device at once,
// with 64 registers a thread and `smem` bytes a CTA, in even shares (1000 x
// 4600 backward: 334 CTAs of 3 rows 14.9 us, 444 of 2 or 3 16.1 us).
int ctas_for(int rows, int threads, size_t smem) {
  int fit = 1024 / threads;
  const int by_smem = static_cast<int>(220 * 1024 / (smem + 1024));
  if (fit > by_smem) fit = by_smem;
  if (fit > 32) fit = 32;
  int most = current_sm_count() * (fit > 0 ? fit : 1);
  if (most > kMaxParts) most = kMaxParts;
  const int each = (rows + most - 1) / most;
  return (rows + each - 1) / each;
}

constexpr size_t kRingMost = 200 * 1024;

template <typename T, typename W, int NV>
int launch_norm(const NormArgs &a, cudaStream_t stream) {
  const int threads = threads_for(a.cols, NV), direct = ctas_for(a.rows, threads, 0);
  const size_t ring = (size_t)kStages * a.cols * sizeof(T) * (a.residual != nullptr ? 2 : 1);
  if (a.rows > direct && a.cols % 8 == 0 && a.x_vec && (a.residual == nullptr || a.r_vec) &&
      ring <= kRingMost)
    return launch_rows(k_rmsnorm<T, W, NV, true>, a, ctas_for(a.rows, threads, ring), threads,
                       ring, stream);
  return launch_rows(k_rmsnorm<T, W, NV, false>, a, direct, threads, 0, stream);
}

template <typename T, typename W>
int launch_norm(const NormArgs &a, cudaStream_t stream) {
  switch (chunks_for(a.cols)) {
    case 1: return launch_norm<T, W, 1>(a, stream);
    case 2: return launch_norm<T, W, 2>(a, stream);
    default: return launch_norm<T, W, 4>(a, stream);
  }
}

template <typename T, typename W, int NV>
int launch_back(NormBackArgs a, int *grid, cudaStream_t stream) {
  const int threads = threads_for(a.cols, NV), direct = ctas_for(a.rows, threads, 0);
  const size_t ring = (size_t)kStages * a.cols * sizeof(T) * (a.dh != nullptr ? 3 : 2);
  const bool use_ring = a.rows > direct && a.cols % 8 == 0 && a.dy_vec && a.h_vec &&
                        (a.dh == nullptr || a.dh_vec) && ring <= kRingMost;
  *grid = use_ring ? ctas_for(a.rows, threads, ring) : direct;
  if (use_ring) return launch_rows(k_rmsnorm_back<T, W, NV, true>, a, *grid, threads, ring, stream);
  return launch_rows(k_rmsnorm_back<T, W, NV, false>, a, *grid, threads, 0, stream);
}

template <typename T, typename W>
int launch_back(const NormBackArgs &a, int *grid, cudaStream_t stream) {
  switch (chunks_for(a.cols)) {
    case 1: return launch_back<T, W, 1>(a, grid, stream);
    case 2: return launch_back<T, W, 2>(a, grid, stream);
    default: return launch_back<T, W, 4>(a, grid, stream);
  }
}

// A matrix operand of a norm: its name, address, pitch and whether it has to
// be there.
struct Operand {
  const char *name;
  const void *p;
  size_t ld, elem;
};

int check_operands(const char *fn, const Operand *ops, int n, int cols) {
  for (int i = 0; i < n; ++i) {
    if (ops[i].p == nullptr) continue;
    if (reinterpret_cast<uintptr_t>(ops[i].p) % ops[i].elem)
      return fail(CMB_ERR_INVALID_ARG, "%s: %s is not aligned to its type", fn, ops[i].name);
    if (ops[i].ld < (size_t)cols)
      return fail(CMB_ERR_INVALID_ARG, "%s: rows of %s overlap (leading dimension %zu for %d)", fn,
                  ops[i].name, ops[i].ld, cols);
  }
  return CMB_OK;
}

int check_types(const char *fn, int type, int weight_type, int rows, int cols) {
  if ((type != CMB_BF16 && type != CMB_F32) || (weight_type != CMB_BF16 && weight_type != CMB_F32))
    return fail(CMB_ERR_INVALID_ARG, "%s: types %d, %d are not CMB_BF16 or CMB_F32", fn, type,
                weight_type);
  if (rows < 0 || cols <= 0 || cols > CMB_RMSNORM_MAX_COLS)
    return fail(CMB_ERR_INVALID_ARG, "%s: %d rows of %d columns (1-%d)", fn, rows, cols,
                CMB_RMSNORM_MAX_COLS);
  return CMB_OK;
}

}  // namespace
}  // namespace cmb

using namespace cmb;

extern "C" int cmb_rmsnorm_e4m3_block128(const void *x, size_t ld_x, const void *residual,
                                         size_t ld_residual, int type, const void *weight,
                                         int weight_type, float eps, int rows, int cols, void *h,
                                         size_t ld_h, void *y, size_t ld_y, uint8_t *q, size_t ld_q,
                                         uint8_t *scale, size_t ld_scale, float *rstd,
                                         cmb_stream_t stream) {
  const char *fn = "cmb_rmsnorm_e4m3_block128";
  int rc = check_types(fn, type, weight_type, rows, cols);
  if (rc) return rc;
  if (!(eps >= 0.0f)) return fail(CMB_ERR_INVALID_ARG, "%s: eps is negative or NaN", fn);
  if ((q == nullptr) != (scale == nullptr))
    return fail(CMB_ERR_INVALID_ARG, "%s: q and scale go together", fn);
  if ((residual == nullptr) != (h == nullptr))
    return fail(CMB_ERR_INVALID_ARG, "%s: residual and h go together", fn);
  if (q == nullptr && y == nullptr && h == nullptr && rstd == nullptr)
    return fail(CMB_ERR_INVALID_ARG, "%s: nothing to write", fn);
  if (rows == 0) return CMB_OK;
  if (x == nullptr || weight == nullptr)
    return fail(CMB_ERR_INVALID_ARG, "%s: null operand", fn);
  const size_t elem = type == CMB_BF16 ? 2 : 4, welem = weight_type == CMB_BF16 ? 2 : 4;
  const Operand ops[] = {{"x", x, ld_x, elem},           {"residual", residual, ld_residual, elem},
                         {"h", h, ld_h, elem},           {"y", y, ld_y, elem},
                         {"q", q, ld_q, 1},              {"weight", weight, (size_t)cols, welem},
                         {"rstd", rstd, (size_t)cols, 4}};
  rc = check_operands(fn, ops, 7, cols);
  if (rc) return rc;
  if (scale != nullptr && ld_scale < (size_t)b128::groups_of(cols))
    return fail(CMB_ERR_INVALID_ARG, "%s: rows of scale overlap", fn);
  if (current_cc() != 100)
    return fail(CMB_ERR_UNSUPPORTED, "%s: needs an sm_100 device (found cc %d)", fn, current_cc());

  NormArgs a = {x, residual, weight, h, y, q, scale, rstd, ld_x, ld_residual, ld_h, ld_y, ld_q,
                ld_scale, eps, rows, cols, false, false, false, false, false, false};
  a.x_vec = b128::aligned_to(x, ld_x * elem, 16);
  a.r_vec = b128::aligned_to(residual, ld_residual * elem, 16);
  a.w_vec = b128::aligned_to(weight, 0, 16);
  a.h_vec = b128::aligned_to(h, ld_h * elem, 16);
  a.y_vec = b128::aligned_to(y, ld_y * elem, 16);
  a.q_vec = b128::aligned_to(q, ld_q, 8);
  if (type == CMB_BF16)
    return weight_type == CMB_BF16 ? launch_norm<__nv_bfloat16, __nv_bfloat16>(a, stream)
                                   : launch_norm<__nv_bfloat16, float>(a, stream);
  return weight_type == CMB_BF16 ? launch_norm<float, __nv_bfloat16>(a, stream)
                                 : launch_norm<float, float>(a, stream);
}

extern "C" size_t cmb_rmsnorm_backward_workspace_bytes(int rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return sizeof(float) * parts_pitch(cols) * (size_t)(rows < kMaxParts ? rows : kMaxParts);
}

extern "C" int cmb_rmsnorm_backward(const void *dy, size_t ld_dy, const void *h, size_t ld_h,
                                    const void *dh, size_t ld_dh, int type, const void *weight,
                                    int weight_type, const float *rstd, int rows, int cols,
                                    void *dx, size_t ld_dx, float *dweight, void *workspace,
                                    size_t workspace_bytes, cmb_stream_t stream) {
  const char *fn = "cmb_rmsnorm_backward";
  int rc = check_types(fn, type, weight_type, rows, cols);
  if (rc) return rc;
  if (reinterpret_cast<uintptr_t>(dweight) % 4)
    return fail(CMB_ERR_INVALID_ARG, "%s: dweight is not aligned to its type", fn);
  if (rows == 0) {
    if (dweight != nullptr)
      CMB_CUDA_TRY(cudaMemsetAsync(dweight, 0, sizeof(float) * cols, stream));
    return CMB_OK;
  }
  if (dy == nullptr || h == nullptr || weight == nullptr || rstd == nullptr || dx == nullptr)
    return fail(CMB_ERR_INVALID_ARG, "%s: null operand", fn);
  const size_t elem = type == CMB_BF16 ? 2 : 4, welem = weight_type == CMB_BF16 ? 2 : 4;
  const Operand ops[] = {{"dy", dy, ld_dy, elem},
                         {"h", h, ld_h, elem},
                         {"dh", dh, ld_dh, elem},
                         {"dx", dx, ld_dx, elem},
                         {"weight", weight, (size_t)cols, welem},
                         {"rstd", rstd, (size_t)cols, 4}};
  rc = check_operands(fn, ops, 6, cols);
  if (rc) return rc;
  if (dweight != nullptr) {
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16)
      return fail(CMB_ERR_INVALID_ARG, "%s: workspace is null or not 16-byte aligned", fn);
    if (workspace_bytes < cmb_rmsnorm_backward_workspace_bytes(rows, cols))
      return fail(CMB_ERR_INVALID_ARG, "%s: workspace of %zu bytes, needs %zu", fn,
                  workspace_bytes, cmb_rmsnorm_backward_workspace_bytes(rows, cols));
  }
  if (current_cc() != 100)
    return fail(CMB_ERR_UNSUPPORTED, "%s: needs an sm_100 device (found cc %d)", fn, current_cc());

  NormBackArgs a = {dy, h, dh, weight, rstd, dx,
                    dweight != nullptr ? static_cast<float *>(workspace) : nullptr,
                    ld_dy, ld_h, ld_dh, ld_dx, parts_pitch(cols), rows, cols,
                    false, false, false, false, false};
  a.dy_vec = b128::aligned_to(dy, ld_dy * elem, 16);
  a.h_vec = b128::aligned_to(h, ld_h * elem, 16);
  a.dh_vec = b128::aligned_to(dh, ld_dh * elem, 16);
  a.w_vec = b128::aligned_to(weight, 0, 16);
  a.dx_vec = b128::aligned_to(dx, ld_dx * elem, 16);
  int grid = 0;
  if (type == CMB_BF16)
    rc = weight_type == CMB_BF16 ? launch_back<__nv_bfloat16, __nv_bfloat16>(a, &grid, stream)
                                 : launch_back<__nv_bfloat16, float>(a, &grid, stream);
  else
    rc = weight_type == CMB_BF16 ? launch_back<float, __nv_bfloat16>(a, &grid, stream)
                                 : launch_back<float, float>(a, &grid, stream);
  if (rc || dweight == nullptr) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((cols + 31) / 32);
  cfg.blockDim = dim3(32, 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_sum_parts, static_cast<const float *>(a.parts),
                                  a.ld_parts, grid, cols, dweight));
  return CMB_OK;
}
