// rmsnorm.cu — root-mean-square norm with the residual's addition and a
// block-scaled e4m3 output, and its backward pass.
//
//   h = x + r, rstd = (mean h^2 + eps)^(-1/2), y = h rstd w, (q, s) = y in e4m3
//   g = dy w, dx = rstd (g - h rstd^2 mean(g h)) + dh, dw = sum_rows dy h rstd
//
// Memory bound.  h is rounded to the rows' type before the mean: the norm,
// its backward pass and every later reader then see the same h.  Sums and
// statistics are fp32, in a fixed order.
#include "block128.cuh"
#include "cmb_host.h"

namespace cmb {
namespace {

using b128::Raw8;

constexpr int kMaxParts = 1024;  // rows of partial weight gradients in the workspace

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

// One CTA walks over rows; thread t holds the chunks of 8 columns t, t +
// blockDim, ...: 16 neighbouring threads hold a block of 128.
template <typename T, typename W, int NV>
__global__ void __launch_bounds__(1024) k_rmsnorm(const NormArgs a) {
  __shared__ float part[2][32];
  const T *x = static_cast<const T *>(a.x), *res = static_cast<const T *>(a.residual);
  const W *w = static_cast<const W *>(a.weight);
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    float h[NV][8];
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      Raw8<T> raw{};
      if (n > 0) {
        raw = b128::load8_edge(x + (size_t)row * a.ld_x + col, n, a.x_vec);
        if (res != nullptr) {
          float v[8], u[8];
          b128::unpack(raw, v);
          b128::unpack(b128::load8_edge(res + (size_t)row * a.ld_r + col, n, a.r_vec), u);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += u[j];
          b128::pack(v, raw);
          b128::store8_edge(static_cast<T *>(a.h) + (size_t)row * a.ld_h + col, raw, n, a.h_vec);
        }
      }
      b128::unpack(raw, h[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(h[i][j], h[i][j], sq);
    }
    sq = cta_sum(sq, part[turn]);
    const float rstd = 1.0f / sqrtf(sq / static_cast<float>(a.cols) + a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      float wv[8], top = 0.0f;
      Raw8<W> wr{};
      if (n > 0) wr = b128::load8_edge(w + col, n, a.w_vec);
      b128::unpack(wr, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] = h[i][j] * rstd * wv[j];
        // behind the row's end: not 0 * inf, which would be NaN
        if (j >= n) h[i][j] = 0.0f;
        top = fmaxf(top, b128::finite_magnitude(h[i][j]));
      }
      if (a.y != nullptr && n > 0) {
        Raw8<T> out;
        b128::pack(h[i], out);
        b128::store8_edge(static_cast<T *>(a.y) + (size_t)row * a.ld_y + col, out, n, a.y_vec);
      }
      if (a.q != nullptr) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t byte = b128::scale_byte(top);
        if (n > 0) {
          b128::store_bytes(a.q + (size_t)row * a.ld_q + col,
                            b128::e4m3x8(h[i], b128::scale_reciprocal(byte)), n, a.q_vec);
          if ((threadIdx.x & 15) == 0)
            a.scale[(size_t)row * a.ld_scale + col / b128::kBlock] = static_cast<uint8_t>(byte);
        }
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
  bool dy_vec, h_vec, dh_vec, w_vec, dx_vec;
};

template <typename T, typename W, int NV>
__global__ void __launch_bounds__(1024) k_rmsnorm_back(const NormBackArgs a) {
  __shared__ float part[2][32];
  const T *dy = static_cast<const T *>(a.dy), *h = static_cast<const T *>(a.h);
  const T *dh = static_cast<const T *>(a.dh);
  const W *w = static_cast<const W *>(a.weight);
  float dw[NV][8] = {};
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const float rstd = a.rstd[row];
    float g[NV][8], u[NV][8];  // dy * w and h * rstd
    float along = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      Raw8<T> rd{}, rh{};
      Raw8<W> rw{};
      if (n > 0) {
        rd = b128::load8_edge(dy + (size_t)row * a.ld_dy + col, n, a.dy_vec);
        rh = b128::load8_edge(h + (size_t)row * a.ld_h + col, n, a.h_vec);
        rw = b128::load8_edge(w + col, n, a.w_vec);
      }
      float wv[8];
      b128::unpack(rd, g[i]);
      b128::unpack(rh, u[i]);
      b128::unpack(rw, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[i][j] = j < n ? u[i][j] * rstd : 0.0f;
        dw[i][j] = fmaf(g[i][j], u[i][j], dw[i][j]);
        g[i][j] *= wv[j];
        along = fmaf(g[i][j], u[i][j], along);
      }
    }
    const float mean = cta_sum(along, part[turn]) / static_cast<float>(a.cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * blockDim.x + threadIdx.x) * 8, n = a.cols - col;
      if (n <= 0) continue;
      float v[8], past[8] = {};
      if (dh != nullptr)
        b128::unpack(b128::load8_edge(dh + (size_t)row * a.ld_dh + col, n, a.dh_vec), past);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmaf(rstd, g[i][j] - u[i][j] * mean, past[j]);
      Raw8<T> out;
      b128::pack(v, out);
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

// dweight[c] = sum of the partial rows, in their order.
__global__ void k_sum_parts(const float *__restrict__ parts, size_t ld, int n, int cols,
                            float *__restrict__ out) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int r = 0; r < n; ++r) s += parts[(size_t)r * ld + c];
  out[c] = s;
}

int back_ctas(int rows) {
  const int most = current_sm_count() * 2;
  const int ctas = rows < most ? rows : most;
  return ctas < kMaxParts ? ctas : kMaxParts;
}

size_t parts_pitch(int cols) { return ((size_t)cols + 63) / 64 * 64; }

// Threads that hold `cols` in NV chunks of 8 each.
int threads_for(int cols, int nv) {
  const int chunks = (cols + 7) / 8;
  const int t = (chunks + nv - 1) / nv;
  return (t + 31) / 32 * 32;
}

int chunks_for(int cols) { return cols <= 8192 ? 1 : cols <= 16384 ? 2 : 4; }

template <typename T, typename W>
int launch_norm(const NormArgs &a, cudaStream_t stream) {
  const int nv = chunks_for(a.cols), threads = threads_for(a.cols, nv);
  const int most = current_sm_count() * (2048 / threads);
  const int grid = a.rows < most ? a.rows : most;
  if (nv == 1) k_rmsnorm<T, W, 1><<<grid, threads, 0, stream>>>(a);
  else if (nv == 2) k_rmsnorm<T, W, 2><<<grid, threads, 0, stream>>>(a);
  else k_rmsnorm<T, W, 4><<<grid, threads, 0, stream>>>(a);
  CMB_LAUNCH_CHECK();
  return CMB_OK;
}

template <typename T, typename W>
int launch_back(const NormBackArgs &a, int grid, cudaStream_t stream) {
  const int nv = chunks_for(a.cols), threads = threads_for(a.cols, nv);
  if (nv == 1) k_rmsnorm_back<T, W, 1><<<grid, threads, 0, stream>>>(a);
  else if (nv == 2) k_rmsnorm_back<T, W, 2><<<grid, threads, 0, stream>>>(a);
  else k_rmsnorm_back<T, W, 4><<<grid, threads, 0, stream>>>(a);
  CMB_LAUNCH_CHECK();
  return CMB_OK;
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
  const int grid = back_ctas(rows);
  if (type == CMB_BF16)
    rc = weight_type == CMB_BF16 ? launch_back<__nv_bfloat16, __nv_bfloat16>(a, grid, stream)
                                 : launch_back<__nv_bfloat16, float>(a, grid, stream);
  else
    rc = weight_type == CMB_BF16 ? launch_back<float, __nv_bfloat16>(a, grid, stream)
                                 : launch_back<float, float>(a, grid, stream);
  if (rc || dweight == nullptr) return rc;
  k_sum_parts<<<(cols + 127) / 128, 128, 0, stream>>>(a.parts, a.ld_parts, grid, cols, dweight);
  CMB_LAUNCH_CHECK();
  return CMB_OK;
}
