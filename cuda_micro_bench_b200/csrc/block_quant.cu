// block_quant.cu — quantisation to e4m3 with a power-of-two scale for each
// block of 128 (or 128 x 128) values, of a matrix and of its transpose in one
// read.
//
//   e = smallest integer with max|x| / 2^e <= 448,  q = e4m3(x * 2^-e)
//
// Memory bound: 2 or 4 bytes read and 1 or 2 written for each value.
#include "block128.cuh"
#include "cmb_host.h"

namespace cmb {
namespace {

using b128::kBlock;

struct QuantArgs {
  const void *src;
  size_t ld_src;
  int rows, cols, block_rows;
  uint8_t *dst, *scale, *dst_t, *scale_t;
  size_t ld_dst, ld_scale, ld_dst_t, ld_scale_t;
  bool src_vec, dst_vec, dst_t_vec;  // 16-byte loads, 8-byte stores
};

// One CTA per 128 x 128 tile: a whole block of every kind, so its maxima
// need nothing from outside.  8 warps stand 4 (columns) x 2 (rows); a thread
// holds 8 rows x 8 columns, a warp 64 rows x 32 columns, so each row a warp
// loads is 64 bytes (bf16) and each column it stores 64 bytes: whole 32-byte
// sectors both ways with no trip through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) k_quantize_tile(const QuantArgs a) {
  __shared__ float row_part[4][kBlock], col_part[2][kBlock], all_part[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wc = warp & 3, wr = warp >> 2;
  const int lc = lane & 3, lr = lane >> 2;
  const int col_in = wc * 32 + lc * 8, row_in = wr * 64 + lr * 8;
  const int col = blockIdx.x * kBlock + col_in;
  const int ncol = min(8, a.cols - col);
  const T *src = static_cast<const T *>(a.src);

  for (int tile_r = blockIdx.y; tile_r < b128::groups_of(a.rows); tile_r += gridDim.y) {
    const int row = tile_r * kBlock + row_in;
    b128::Raw8<T> raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      raw[i] = row + i < a.rows
                   ? b128::load8_edge(src + (size_t)(row + i) * a.ld_src + col, ncol, a.src_vec)
                   : b128::Raw8<T>{};
    float rmax[8], cmax[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cmax[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[8];
      b128::unpack(raw[i], v);
      rmax[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float m = b128::finite_magnitude(v[j]);
        rmax[i] = fmaxf(rmax[i], m);
        cmax[j] = fmaxf(cmax[j], m);
      }
    }
    if (a.block_rows == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // over the 4 lanes of a row, then the 4 warps
        rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], 1));
        rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], 2));
        if (lc == 0) row_part[wc][row_in + i] = rmax[i];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
          cmax[i] = fmaxf(cmax[i], __shfl_xor_sync(0xffffffffu, cmax[i], o));
        if (lr == 0) col_part[wr][col_in + i] = cmax[i];
      }
    } else {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, rmax[i]);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (lane == 0) all_part[warp] = m;
    }
    __syncthreads();
    uint32_t rbyte[8], cbyte[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (a.block_rows == 1) {
        const float r = fmaxf(fmaxf(row_part[0][row_in + i], row_part[1][row_in + i]),
                              fmaxf(row_part[2][row_in + i], row_part[3][row_in + i]));
        rbyte[i] = b128::scale_byte(r);
        cbyte[i] = b128::scale_byte(fmaxf(col_part[0][col_in + i], col_part[1][col_in + i]));
      } else {
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, all_part[k]);
        rbyte[i] = cbyte[i] = b128::scale_byte(m);
      }
    }
    if (a.dst != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (row + i >= a.rows) continue;
        float v[8];
        b128::unpack(raw[i], v);
        if (ncol > 0)
          b128::store_bytes(a.dst + (size_t)(row + i) * a.ld_dst + col,
                            b128::e4m3x8<true>(v, b128::scale_reciprocal(rbyte[i])), ncol, a.dst_vec);
        if (a.block_rows == 1 && col_in == 0)
          a.scale[(size_t)(row + i) * a.ld_scale + blockIdx.x] = static_cast<uint8_t>(rbyte[i]);
      }
      if (a.block_rows != 1 && threadIdx.x == 0)
        a.scale[(size_t)tile_r * a.ld_scale + blockIdx.x] = static_cast<uint8_t>(rbyte[0]);
    }
    if (a.dst_t != nullptr) {
      const int nrow = min(8, a.rows - row);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= ncol) continue;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float w[8];
          b128::unpack(raw[i], w);
          v[i] = w[j];
        }
        if (nrow > 0)
          b128::store_bytes(a.dst_t + (size_t)(col + j) * a.ld_dst_t + row,
                            b128::e4m3x8<true>(v, b128::scale_reciprocal(cbyte[j])), nrow, a.dst_t_vec);
        if (a.block_rows == 1 && row_in == 0)
          a.scale_t[(size_t)(col + j) * a.ld_scale_t + tile_r] = static_cast<uint8_t>(cbyte[j]);
      }
      if (a.block_rows != 1 && threadIdx.x == 0)
        a.scale_t[(size_t)blockIdx.x * a.ld_scale_t + tile_r] = static_cast<uint8_t>(cbyte[0]);
    }
    __syncthreads();  // the maxima are read before the next tile writes them
  }
}

}  // namespace
}  // namespace cmb

using namespace cmb;

extern "C" int cmb_quantize_e4m3_block128(const void *src, int src_type, int rows, int cols,
                                          size_t ld_src, int block_rows, uint8_t *dst,
                                          size_t ld_dst, uint8_t *scale, size_t ld_scale,
                                          uint8_t *dst_t, size_t ld_dst_t, uint8_t *scale_t,
                                          size_t ld_scale_t, cmb_stream_t stream) {
  const char *fn = "cmb_quantize_e4m3_block128";
  if (src_type != CMB_BF16 && src_type != CMB_F32)
    return fail(CMB_ERR_INVALID_ARG, "%s: src_type %d is not CMB_BF16 or CMB_F32", fn, src_type);
  if (block_rows != 1 && block_rows != kBlock)
    return fail(CMB_ERR_INVALID_ARG, "%s: block_rows %d not 1 or 128", fn, block_rows);
  if (rows < 0 || cols < 0)
    return fail(CMB_ERR_INVALID_ARG, "%s: %d x %d values", fn, rows, cols);
  if ((dst == nullptr) != (scale == nullptr) || (dst_t == nullptr) != (scale_t == nullptr))
    return fail(CMB_ERR_INVALID_ARG, "%s: values and scales go together", fn);
  if (dst == nullptr && dst_t == nullptr)
    return fail(CMB_ERR_INVALID_ARG, "%s: nothing to write", fn);
  if (rows == 0 || cols == 0) return CMB_OK;
  const size_t elem = src_type == CMB_BF16 ? 2 : 4;
  if (src == nullptr || reinterpret_cast<uintptr_t>(src) % elem)
    return fail(CMB_ERR_INVALID_ARG, "%s: src is null or not aligned to its type", fn);
  if (ld_src < (size_t)cols ||
      (dst != nullptr && (ld_dst < (size_t)cols || ld_scale < (size_t)b128::groups_of(cols))) ||
      (dst_t != nullptr && (ld_dst_t < (size_t)rows || ld_scale_t < (size_t)b128::groups_of(rows))))
    return fail(CMB_ERR_INVALID_ARG, "%s: rows overlap (a leading dimension is too small)", fn);
  if (current_cc() != 100)
    return fail(CMB_ERR_UNSUPPORTED, "%s: needs an sm_100 device (found cc %d)", fn, current_cc());

  QuantArgs a = {src, ld_src, rows, cols, block_rows, dst, scale, dst_t, scale_t,
                 ld_dst, ld_scale, ld_dst_t, ld_scale_t, false, false, false};
  a.src_vec = b128::aligned_to(src, ld_src * elem, 16);
  a.dst_vec = b128::aligned_to(dst, ld_dst, 8);
  a.dst_t_vec = b128::aligned_to(dst_t, ld_dst_t, 8);
  const int tiles_c = b128::groups_of(cols), tiles_r = b128::groups_of(rows);
  const dim3 grid(tiles_c, tiles_r < 65535 ? tiles_r : 65535);
  if (src_type == CMB_BF16)
    k_quantize_tile<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else
    k_quantize_tile<float><<<grid, 256, 0, stream>>>(a);
  CMB_LAUNCH_CHECK();
  return CMB_OK;
}
