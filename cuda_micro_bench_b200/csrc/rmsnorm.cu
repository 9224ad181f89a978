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
// A CTA of blockDim.x x blockDim.y threads works on blockDim.y rows at a time;
// thread x holds the chunks of 8 columns x, x + blockDim.x, ...: a warp stays
// within a row, and 16 neighbouring threads hold a block of 128.  Three ways to
// read and write rows (Way):
//   kRing  whole chunks that start on 16 bytes, several rows a CTA: a thread
//          keeps the next rows on their way into shared memory with bulk
//          copies, so loads never wait for a row's reduction.
//   kFew   the same with no more rows than the device has room for at once:
//          straight from global memory, since latency is one load.
//   kAny   every other width, pitch and alignment.
#include "block128.cuh"
#include "cmb_host.h"

namespace cmb {
namespace {

using b128::Bounds;
using b128::Raw8;

constexpr int kMaxParts = 1024;  // CTAs, each with a row of partial weight gradients
// Rows in the ring.  Two leave room for two CTAs of a wide row on a SM, which
// counts for more than depth: the backward pass of 8192 x 8192 bf16 took 90 us
// with two, 108 with three or four (one CTA a SM); the norm 81, 80 and 102.
constexpr int kStages = 2;

enum Way { kRing, kFew, kAny };

// Sum over the threads of a row, the same value in each.  `part` holds one
// float for each warp; two calls in a row use different ones.
__device__ __forceinline__ float row_sum(float v, float *part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  part += threadIdx.y * warps;
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? part[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kNever = 0x7FFFFFFF;

// A wait for turn `turn` that was not over at once.  Where it runs out, or one of the
// CTA has, the thread goes on with what the stage holds, and the CTA gives up its
// rows from that turn on once it is through them (Ring::failed).
static __device__ __noinline__ void wait_long(uint32_t bar, uint32_t parity, int turn,
                                              int *failed_at) {
  const uint64_t deadline = dev::globaltimer() + dev::kWaitLimitNs;
#pragma unroll 1
  while (!dev::mbar_try_wait(bar, parity)) {
    if (*const_cast<volatile int *>(failed_at) != kNever) return;
    if (dev::globaltimer() > deadline) {
      atomicMin(failed_at, turn);
      return;
    }
  }
}

// Rows of up to three matrices on their way through shared memory.  A CTA's
// turn i is over rows (blockIdx.x + i * gridDim.x) * blockDim.y and on, in stage
// i % kStages.
struct Ring {
  const uint8_t *src[3];
  size_t pitch[3];
  int n;           // matrices
  uint32_t bytes;  // of a row of one of them
  uint8_t *mem;
  uint64_t *full;
  int *failed_at;  // the first turn whose wait has run out, and the first not loaded for it

  __device__ __forceinline__ long long first_row(int i) const {
    return (blockIdx.x + static_cast<long long>(i) * gridDim.x) * blockDim.y;
  }
  // By one thread, whose own waits tell it that the turn's place is free.
  __device__ __forceinline__ void load(int i, int rows) const {
    const long long first = first_row(i);
    if (first >= rows) return;
    if (*const_cast<volatile int *>(failed_at) != kNever) {
      failed_at[1] = min(failed_at[1], i);
      return;
    }
    const int high = static_cast<int>(min(static_cast<long long>(blockDim.y), rows - first));
    const int s = i % kStages;
    const uint32_t bar = dev::smem_addr(full + s);
    dev::mbar_arrive_expect_tx(bar, bytes * n * high);
    for (int y = 0; y < high; ++y)
      for (int k = 0; k < n; ++k)
        dev::bulk_load(dev::smem_addr(at(s, y, k)), src[k] + (first + y) * pitch[k], bytes, bar);
  }
  __device__ __forceinline__ void start(int rows) const {
    if (threadIdx.x == 0 && threadIdx.y == 0) {
      for (int s = 0; s < kStages; ++s) dev::mbar_init(dev::smem_addr(full + s), 1);
      dev::fence_mbar_init();
      failed_at[0] = failed_at[1] = kNever;
    }
    __syncthreads();
    if (threadIdx.x == 0 && threadIdx.y == 0)
      for (int s = 0; s < kStages; ++s) load(s, rows);
  }
  __device__ __forceinline__ void wait(int i) const {
    const uint32_t bar = dev::smem_addr(full + i % kStages), parity = (i / kStages) & 1;
    if (!dev::mbar_try_wait(bar, parity)) wait_long(bar, parity, i, failed_at);
  }
  // All threads, when they are through their rows: whether a wait has run out.  The
  // copies that are still on their way then land (or their waits run out too), and
  // `row` is the first that the CTA gives up.
  __device__ __forceinline__ bool failed(int rows, int &row) const {
    __syncthreads();
    const int turn = failed_at[0];
    if (turn == kNever) return false;
    row = static_cast<int>(first_row(turn));
    if (threadIdx.x == 0 && threadIdx.y == 0) {
      int end = 0;
      while (end < failed_at[1] && first_row(end) < rows) ++end;
      for (int i = max(0, end - kStages); i < end; ++i)
        dev::mbar_wait_bounded(dev::smem_addr(full + i % kStages), (i / kStages) & 1, 100000000ull);
    }
    __syncthreads();
    return true;
  }
  __device__ __forceinline__ uint8_t *at(int s, int y, int k) const {
    return mem + static_cast<size_t>((s * static_cast<int>(blockDim.y) + y) * n + k) * bytes;
  }
  template <typename T>
  __device__ __forceinline__ const T *row(int i, int k) const {
    return reinterpret_cast<const T *>(at(i % kStages, threadIdx.y, k));
  }
};

// What the CTA's rows from `first` on read where a wait has run out: `word` over all
// of them, `bytes` (a multiple of 8, as the rows' starts are) each.
static __device__ __noinline__ void spoil_rows(void *p, size_t pitch, uint32_t bytes, uint32_t word,
                                               int first, int rows) {
  if (p == nullptr) return;
  for (; first < rows; first += gridDim.x * blockDim.y) {
    const int row = first + threadIdx.y;
    if (row >= rows) return;
    uint2 *to = reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p) + row * pitch);
    for (uint32_t i = threadIdx.x; i < bytes / 8; i += blockDim.x) to[i] = make_uint2(word, word);
  }
}
constexpr uint32_t kNanWord = 0x7FFF7FFFu;  // NaN as two bf16 and as a fp32

// 8 columns of a row, from the ring or from where the row lies.
template <typename T, int kWay>
__device__ __forceinline__ Raw8<T> load_chunk(const Ring &ring, int turn, int k, const void *p,
                                              size_t ld, int row, int col, int n,
                                              const Bounds &in) {
  if (n <= 0) return {};
  if constexpr (kWay == kRing) return b128::load8(ring.row<T>(turn, k) + col);
  const T *at = static_cast<const T *>(p) + static_cast<size_t>(row) * ld + col;
  if constexpr (kWay == kFew) return b128::load8(at);
  else return b128::load8_any(at, n, in);
}

// The whole warp (see b128::store8_any).
template <typename T, int kWay>
__device__ __forceinline__ void store_chunk(void *p, size_t ld, int row, int col, int n,
                                            const Raw8<T> &r) {
  T *at = static_cast<T *>(p) + static_cast<size_t>(row) * ld + col;
  if constexpr (kWay == kAny) {
    b128::store8_any(at, r, n);
  } else {
    if (n > 0) b128::store8(at, r);
  }
}

// A thread's chunks of the weights: kept in registers, or, where a row has
// more than two chunks a thread, read again for each row.
template <typename W, int NV>
struct Weight {
  const W *p;
  Bounds in;
  int cols;
  Raw8<W> kept[NV <= 2 ? NV : 1];

  __device__ __forceinline__ Weight(const void *weight, int cols)
      : p(static_cast<const W *>(weight)),
        in(Bounds::of(static_cast<const W *>(weight), 0, 1, cols)),
        cols(cols) {
    if constexpr (NV <= 2) {
#pragma unroll
      for (int i = 0; i < NV; ++i) kept[i] = load(i);
    }
  }
  __device__ __forceinline__ Raw8<W> load(int i) const {
    const int col = (i * blockDim.x + threadIdx.x) * 8;
    return b128::load8_any(p + col, cols - col, in);
  }
  __device__ __forceinline__ Raw8<W> chunk(int i) const {
    if constexpr (NV <= 2) return kept[i];
    else return load(i);
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
  bool q_vec;  // 8-byte stores of q
};

// The e4m3 values and scales of 8 columns of a row; the whole warp.
template <int kWay>
__device__ __forceinline__ void store_quantized(const NormArgs &a, int row, int col, int n,
                                                const float (&y)[8]) {
  float top = b128::max_magnitude(y[0], y[1]);
#pragma unroll
  for (int j = 2; j < 8; ++j) top = b128::max_magnitude(top, y[j]);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1)
    top = b128::max_magnitude(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool any = __any_sync(0xffffffffu, !(top <= b128::kMaxFinite));
  if (any) {  // the scale is that of the finite values
    top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, b128::finite_magnitude(y[j]));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const uint32_t byte = b128::scale_byte(top);
  const float inv = b128::scale_reciprocal(byte);
  uint2 q = b128::e4m3x8<false>(y, inv);
  if (any)
    q = b128::e4m3x8_any(make_float4(y[0], y[1], y[2], y[3]), make_float4(y[4], y[5], y[6], y[7]),
                         inv);
  if (n > 0) {
    uint8_t *to = a.q + static_cast<size_t>(row) * a.ld_q + col;
    if constexpr (kWay == kAny) b128::store_bytes(to, q, n, a.q_vec);
    else *reinterpret_cast<uint2 *>(to) = q;
    if ((threadIdx.x & 15) == 0)
      a.scale[static_cast<size_t>(row) * a.ld_scale + col / b128::kBlock] =
          static_cast<uint8_t>(byte);
  }
}

// 8192 x 8192 bf16 with a residual and e4m3 out: 75 us for 470 MB, 0.95 of the
// copy rate (fp32: 139 us, 0.96); with y and rstd too 113 us (0.82).  Without a
// residual (202 MB) 60 us: the instructions' issue bounds it then, 376 a warp for
// 512 values.
template <typename T, typename W, int NV, int kWay>
__global__ void __launch_bounds__(1024, 1) k_rmsnorm(const NormArgs a) {
  __shared__ float part[2][32];
  __shared__ __align__(8) uint64_t full[kStages];
  __shared__ int failed_at[2];
  extern __shared__ __align__(16) uint8_t rows_mem[];
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  Ring ring = {};
  if constexpr (kWay == kRing) {
    ring = {{static_cast<const uint8_t *>(a.x), static_cast<const uint8_t *>(a.residual), nullptr},
            {a.ld_x * sizeof(T), a.ld_r * sizeof(T), 0},
            a.residual != nullptr ? 2 : 1,
            static_cast<uint32_t>(a.cols * sizeof(T)),
            rows_mem,
            full,
            failed_at};
    ring.start(a.rows);
  }
  Bounds in_x{}, in_r{};
  if constexpr (kWay == kAny) {
    in_x = Bounds::of(static_cast<const T *>(a.x), a.ld_x, a.rows, a.cols);
    in_r = Bounds::of(static_cast<const T *>(a.residual), a.ld_r, a.rows, a.cols);
  }
  const Weight<W, NV> weight(a.weight, a.cols);
  int turn = 0;
  for (int first = blockIdx.x * blockDim.y; first < a.rows;
       first += gridDim.x * blockDim.y, ++turn) {
    const int row = first + threadIdx.y;
    const bool here = row < a.rows;  // the same in a warp
    Raw8<T> h[NV];                   // as it is stored
    float sq[8] = {};
    if constexpr (kWay == kRing) ring.wait(turn);
    if (here) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
        h[i] = load_chunk<T, kWay>(ring, turn, 0, a.x, a.ld_x, row, col, n, in_x);
        if (a.residual != nullptr) {
          float v[8];
          b128::add8(h[i],
                     load_chunk<T, kWay>(ring, turn, 1, a.residual, a.ld_r, row, col, n, in_r), v);
          h[i] = b128::packed<T>(v);
          store_chunk<T, kWay>(a.h, a.ld_h, row, col, n, h[i]);
        }
        b128::fma8(h[i], h[i], sq);
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
#pragma unroll
      for (int j = 0; j < o; ++j) sq[j] += sq[j + o];
    const float sum = row_sum(sq[0], part[turn & 1]);
    if constexpr (kWay == kRing)
      if (threadIdx.x == 0 && threadIdx.y == 0)
        ring.load(turn + kStages, a.rows);  // every thread has its chunks
    if (!here) continue;
    const float rstd = 1.0f / sqrtf(sum / static_cast<float>(a.cols) + a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      float y[8];
      b128::mul8(h[i], weight.chunk(i), y);
      // behind the row's end h is 0 and y too, or NaN where rstd is not finite,
      // which a block's scale passes over
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= rstd;
      if (a.y != nullptr) store_chunk<T, kWay>(a.y, a.ld_y, row, col, n, b128::packed<T>(y));
      if (a.q != nullptr) store_quantized<kWay>(a, row, col, n, y);
    }
  }
  if constexpr (kWay == kRing) {
    int row;
    if (ring.failed(a.rows, row)) {
      const uint32_t bytes = a.cols * sizeof(T);
      spoil_rows(a.h, a.ld_h * sizeof(T), bytes, kNanWord, row, a.rows);
      spoil_rows(a.y, a.ld_y * sizeof(T), bytes, kNanWord, row, a.rows);
      spoil_rows(a.q, a.ld_q, a.cols, 0x7F7F7F7Fu, row, a.rows);
      for (row += threadIdx.y; row < a.rows; row += gridDim.x * blockDim.y) {
        if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = __uint_as_float(kNanWord);
        if (a.q != nullptr)
          for (int g = threadIdx.x; g < b128::groups_of(a.cols); g += blockDim.x)
            a.scale[static_cast<size_t>(row) * a.ld_scale + g] = 255;
      }
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
};

// Both passes over a row read it from where it lies, the ring's shared memory
// or global memory, so a thread holds no more of it than a chunk; the weight
// gradient of its columns stays in registers from row to row.  8192 x 8192 bf16
// with dh: 88 us with the sum below for 537 MB, 0.93 of the copy rate; fp32 185 us
// (0.89), where a row's ring leaves one CTA a SM.
template <typename T, typename W, int NV, int kWay>
__global__ void __launch_bounds__(1024, 1) k_rmsnorm_back(const NormBackArgs a) {
  __shared__ float part[2][32];
  __shared__ __align__(8) uint64_t full[kStages];
  __shared__ int failed_at[2];
  extern __shared__ __align__(16) uint8_t rows_mem[];
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  Ring ring = {};
  if constexpr (kWay == kRing) {
    ring = {{static_cast<const uint8_t *>(a.dy), static_cast<const uint8_t *>(a.h),
             static_cast<const uint8_t *>(a.dh)},
            {a.ld_dy * sizeof(T), a.ld_h * sizeof(T), a.ld_dh * sizeof(T)},
            a.dh != nullptr ? 3 : 2,
            static_cast<uint32_t>(a.cols * sizeof(T)),
            rows_mem,
            full,
            failed_at};
    ring.start(a.rows);
  }
  Bounds in_dy{}, in_h{}, in_dh{};
  if constexpr (kWay == kAny) {
    in_dy = Bounds::of(static_cast<const T *>(a.dy), a.ld_dy, a.rows, a.cols);
    in_h = Bounds::of(static_cast<const T *>(a.h), a.ld_h, a.rows, a.cols);
    in_dh = Bounds::of(static_cast<const T *>(a.dh), a.ld_dh, a.rows, a.cols);
  }
  const Weight<W, NV> weight(a.weight, a.cols);
  float dw[NV][8] = {};
  int turn = 0;
  for (int first = blockIdx.x * blockDim.y; first < a.rows;
       first += gridDim.x * blockDim.y, ++turn) {
    const int row = first + threadIdx.y;
    const bool here = row < a.rows;  // the same in a warp
    const float rstd = here ? a.rstd[row] : 0.0f;
    float along = 0.0f;  // sum of g h
    if constexpr (kWay == kRing) ring.wait(turn);
    if (here) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
        if (n <= 0) continue;
        float p[8], w[8];  // dy h
        b128::mul8(load_chunk<T, kWay>(ring, turn, 0, a.dy, a.ld_dy, row, col, n, in_dy),
                   load_chunk<T, kWay>(ring, turn, 1, a.h, a.ld_h, row, col, n, in_h), p);
        b128::unpack(weight.chunk(i), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dw[i][j] = fmaf(p[j], rstd, dw[i][j]);
          along = fmaf(p[j], w[j], along);
        }
      }
    }
    const float sum = row_sum(along, part[turn & 1]);
    // every thread is past the last turn: its place takes another
    if constexpr (kWay == kRing)
      if (threadIdx.x == 0 && threadIdx.y == 0 && turn > 0) ring.load(turn - 1 + kStages, a.rows);
    if (!here) continue;
    // dx = rstd (g + h minus) + dh with minus = -rstd^2 mean(g h).  rstd mean(g h) is
    // of the size of g: rstd^2 alone is past fp32 for rows under 5e-20 (eps 0).
    const float minus = -rstd * (rstd * (sum / static_cast<float>(a.cols)));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      float g[8], u[8], past[8] = {};
      b128::mul8(load_chunk<T, kWay>(ring, turn, 0, a.dy, a.ld_dy, row, col, n, in_dy),
                 weight.chunk(i), g);
      b128::unpack(load_chunk<T, kWay>(ring, turn, 1, a.h, a.ld_h, row, col, n, in_h), u);
      if (a.dh != nullptr)
        b128::unpack(load_chunk<T, kWay>(ring, turn, 2, a.dh, a.ld_dh, row, col, n, in_dh), past);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = fmaf(rstd, fmaf(u[j], minus, g[j]), past[j]);
      store_chunk<T, kWay>(a.dx, a.ld_dx, row, col, n, b128::packed<T>(g));
    }
  }
  if constexpr (kWay == kRing) {
    int row;
    if (ring.failed(a.rows, row)) {
      spoil_rows(a.dx, a.ld_dx * sizeof(T), a.cols * sizeof(T), kNanWord, row, a.rows);
      if (a.parts != nullptr)  // and with them all of dweight
        spoil_rows(a.parts + static_cast<size_t>(blockIdx.x) * a.ld_parts, 0,
                   a.ld_parts * sizeof(float), kNanWord, 0, 1);
      return;
    }
  }
  if (a.parts == nullptr) return;
  // The CTA's rows of threads add theirs up, in order, where the ring was (or
  // in memory of their own), and the first writes the sum.
  float4 *sums = reinterpret_cast<float4 *>(rows_mem);
  for (int y = blockDim.y - 1; y >= 0; --y) {
    if (y != static_cast<int>(blockDim.y) - 1 || kWay == kRing) __syncthreads();
    if (static_cast<int>(threadIdx.y) != y) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int chunk = i * blockDim.x + threadIdx.x;
      float4 v[2] = {{dw[i][0], dw[i][1], dw[i][2], dw[i][3]},
                     {dw[i][4], dw[i][5], dw[i][6], dw[i][7]}};
      if (chunk * 8 >= a.cols) continue;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float4 *at = sums + 2 * chunk + k;
        if (y != static_cast<int>(blockDim.y) - 1) {
          const float4 o = *at;
          v[k] = make_float4(v[k].x + o.x, v[k].y + o.y, v[k].z + o.z, v[k].w + o.w);
        }
        // the workspace's rows are padded to whole chunks
        if (y == 0)
          reinterpret_cast<float4 *>(a.parts + static_cast<size_t>(blockIdx.x) * a.ld_parts)
              [2 * chunk + k] = v[k];
        else
          *at = v[k];
      }
    }
  }
}

// dweight[c] = sum of the partial rows: 32 columns a CTA, 32 threads take
// every 32nd row each, in order, and their sums are added in a tree.  Latency
// bound: 334 rows of 4600 columns add 4.7 us to the backward pass (6 MB, from L2);
// 16 or 8 columns a CTA, 16-byte loads, fewer threads with up to 16 loads each in
// flight: 4.0-9 us there, none ahead at 8192 columns.
__global__ void __launch_bounds__(1024) k_sum_parts(const float *parts, size_t ld, int n, int cols,
                                                    float *out) {
  __shared__ float sums[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int r = threadIdx.y; r < n; r += 32) s += parts[static_cast<size_t>(r) * ld + c];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sums[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int at = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && at < cols) out[at] = s;
}

size_t parts_pitch(int cols) { return (static_cast<size_t>(cols) + 63) / 64 * 64; }

// Chunks of 8 columns a thread.  Two up to a width of 16384: a row then takes
// half the threads, and twice the rows are under way on a SM.
int chunks_for(int cols) { return cols <= 1024 ? 1 : cols <= 16384 ? 2 : 4; }

// CTAs of x * y threads on y rows at a time.
struct Shape {
  int x, y, grid;
  size_t smem;
};

// `row_bytes`: of a row in the ring, 0 without one.
Shape shape_for(int rows, int cols, int nv, size_t row_bytes, bool sums) {
  Shape s;
  s.x = ((cols + 7) / 8 + nv - 1) / nv;
  s.x = (s.x + 31) / 32 * 32;
  // narrow rows: several at a time, as long as every SM has some
  s.y = 256 / s.x;
  while (s.y > 1 && rows < s.y * current_sm_count()) s.y /= 2;
  if (s.y < 1) s.y = 1;
  s.smem = kStages * row_bytes * s.y;
  if (sums && s.y > 1 && s.smem < parts_pitch(cols) * sizeof(float))
    s.smem = parts_pitch(cols) * sizeof(float);
  // what fits on the device at once, with 64 registers a thread, in even shares
  // (1000 x 4600 backward: 334 CTAs of 3 rows 14.9 us, 444 of 2 or 3 16.1 us)
  int fit = 1024 / (s.x * s.y);
  const int by_smem = static_cast<int>(220 * 1024 / (s.smem + 1024));
  if (fit > by_smem) fit = by_smem;
  int most = current_sm_count() * (fit > 0 ? fit : 1);
  if (most > kMaxParts) most = kMaxParts;
  const int turns = (rows + s.y - 1) / s.y, each = (turns + most - 1) / most;
  s.grid = (turns + each - 1) / each;
  return s;
}

constexpr size_t kRingMost = 200 * 1024;  // no launch takes more shared memory

template <typename A>
int launch_rows(void (*kernel)(A), const A &a, const Shape &s, cudaStream_t stream) {
  // One limit for every launch of the kernel: it is the function's, not the
  // call's, and another host thread may be between these two lines.
  CMB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(kRingMost)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.grid);
  cfg.blockDim = dim3(s.x, s.y);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return CMB_OK;
}

// `plain`: every row of every matrix starts on 16 bytes (of q on 8), and cols
// % 8 == 0.
template <typename T, typename W, int NV>
int launch_norm(const NormArgs &a, bool plain, cudaStream_t stream) {
  Shape s = shape_for(a.rows, a.cols, NV, 0, false);
  if (!plain) return launch_rows(k_rmsnorm<T, W, NV, kAny>, a, s, stream);
  const size_t row = a.cols * sizeof(T) * (a.residual != nullptr ? 2 : 1);
  if (a.rows <= s.grid * s.y || kStages * row * s.y > kRingMost)
    return launch_rows(k_rmsnorm<T, W, NV, kFew>, a, s, stream);
  s = shape_for(a.rows, a.cols, NV, row, false);
  return launch_rows(k_rmsnorm<T, W, NV, kRing>, a, s, stream);
}

template <typename T, typename W>
int launch_norm(const NormArgs &a, bool plain, cudaStream_t stream) {
  switch (chunks_for(a.cols)) {
    case 1: return launch_norm<T, W, 1>(a, plain, stream);
    case 2: return launch_norm<T, W, 2>(a, plain, stream);
    default: return launch_norm<T, W, 4>(a, plain, stream);
  }
}

template <typename T, typename W, int NV>
int launch_back(const NormBackArgs &a, bool plain, int *grid, cudaStream_t stream) {
  const bool sums = a.parts != nullptr;
  Shape s = shape_for(a.rows, a.cols, NV, 0, sums);
  const size_t row = a.cols * sizeof(T) * (a.dh != nullptr ? 3 : 2);
  const bool ring = plain && a.rows > s.grid * s.y && kStages * row * s.y <= kRingMost;
  if (ring) s = shape_for(a.rows, a.cols, NV, row, sums);
  *grid = s.grid;
  if (ring) return launch_rows(k_rmsnorm_back<T, W, NV, kRing>, a, s, stream);
  if (plain) return launch_rows(k_rmsnorm_back<T, W, NV, kFew>, a, s, stream);
  return launch_rows(k_rmsnorm_back<T, W, NV, kAny>, a, s, stream);
}

template <typename T, typename W>
int launch_back(const NormBackArgs &a, bool plain, int *grid, cudaStream_t stream) {
  switch (chunks_for(a.cols)) {
    case 1: return launch_back<T, W, 1>(a, plain, grid, stream);
    case 2: return launch_back<T, W, 2>(a, plain, grid, stream);
    default: return launch_back<T, W, 4>(a, plain, grid, stream);
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
  if (rows < 0 || rows > b128::kMostExtent || cols <= 0 || cols > CMB_RMSNORM_MAX_COLS)
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

  const NormArgs a = {x, residual, weight, h, y, q, scale, rstd, ld_x, ld_residual, ld_h, ld_y,
                      ld_q, ld_scale, eps, rows, cols, b128::aligned_to(q, ld_q, 8)};
  const auto on16 = [&](const void *p, size_t ld) {
    return p == nullptr || b128::aligned_to(p, ld * elem, 16);
  };
  const bool plain = cols % 8 == 0 && on16(x, ld_x) && on16(residual, ld_residual) &&
                     on16(h, ld_h) && on16(y, ld_y) && a.q_vec;
  if (type == CMB_BF16)
    return weight_type == CMB_BF16 ? launch_norm<__nv_bfloat16, __nv_bfloat16>(a, plain, stream)
                                   : launch_norm<__nv_bfloat16, float>(a, plain, stream);
  return weight_type == CMB_BF16 ? launch_norm<float, __nv_bfloat16>(a, plain, stream)
                                 : launch_norm<float, float>(a, plain, stream);
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

  const NormBackArgs a = {dy, h, dh, weight, rstd, dx,
                          dweight != nullptr ? static_cast<float *>(workspace) : nullptr,
                          ld_dy, ld_h, ld_dh, ld_dx, parts_pitch(cols), rows, cols};
  const auto on16 = [&](const void *p, size_t ld) {
    return p == nullptr || b128::aligned_to(p, ld * elem, 16);
  };
  const bool plain = cols % 8 == 0 && on16(dy, ld_dy) && on16(h, ld_h) && on16(dh, ld_dh) &&
                     on16(dx, ld_dx);
  int grid = 0;
  if (type == CMB_BF16)
    rc = weight_type == CMB_BF16
             ? launch_back<__nv_bfloat16, __nv_bfloat16>(a, plain, &grid, stream)
             : launch_back<__nv_bfloat16, float>(a, plain, &grid, stream);
  else
    rc = weight_type == CMB_BF16 ? launch_back<float, __nv_bfloat16>(a, plain, &grid, stream)
                                 : launch_back<float, float>(a, plain, &grid, stream);
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
