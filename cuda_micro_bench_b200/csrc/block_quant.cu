// block_quant.cu — quantisation to e4m3 with a power-of-two scale for each
// block of 128 (or 128 x 128) values, of a matrix and of its transpose in one
// read.
//
//   e = smallest integer with max|x| / 2^e <= 448,  q = e4m3(x * 2^-e)
//
// Memory bound: 2 or 4 bytes read and 1 or 2 written for each value.  Maxima
// are taken on the values' bits, two bf16 an instruction; whether a block has
// anything that is not finite shows in its maximum, and only tiles that do
// take the path that looks at each value.
#include "block128.cuh"
#include "cmb_host.h"

namespace cmb {
namespace {

using b128::kBlock;
using b128::Raw8;

struct QuantArgs {
  const void *src;
  size_t ld_src;
  int rows, cols, block_rows;
  uint8_t *dst, *scale, *dst_t, *scale_t;
  size_t ld_dst, ld_scale, ld_dst_t, ld_scale_t;
  bool src_vec, dst_vec, dst_t_vec;  // 16-byte loads, 8-byte stores
};

// 8 values to e4m3, by the reciprocal of their scale.
template <bool kAny>
__device__ __forceinline__ uint2 row_bytes(const Raw8<__nv_bfloat16> &r, float inv) {
  const uint32_t s = __float_as_uint(inv);
  const float2 a = b128::mul_bf16x2(r.a.x, s, s), b = b128::mul_bf16x2(r.a.y, s, s),
               c = b128::mul_bf16x2(r.a.z, s, s), d = b128::mul_bf16x2(r.a.w, s, s);
  return make_uint2(b128::e4m3x4<kAny>(a.x, a.y, b.x, b.y),
                    b128::e4m3x4<kAny>(c.x, c.y, d.x, d.y));
}
template <bool kAny>
__device__ __forceinline__ uint2 row_bytes(const Raw8<float> &r, float inv) {
  float v[8];
  b128::unpack(r, v);
  return b128::e4m3x8<kAny>(v, inv);
}

// Few rows alone (blocks of 1 x 128, no transpose): 16 lanes a block, 8 values a
// lane, two blocks a thread in flight.  A token of 8192 bf16 takes 1.7 us, a
// launch's time.
template <typename T>
__global__ void __launch_bounds__(256) k_quantize_rows(const QuantArgs a) {
  constexpr int kUnroll = 2;
  const T *src = static_cast<const T *>(a.src);
  const int groups = b128::groups_of(a.cols);
  const int lane16 = threadIdx.x & 15;
  const long long half_warps = (long long)gridDim.x * (blockDim.x / 16);
  const long long total = (long long)a.rows * groups;
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  const b128::Bounds in = b128::Bounds::of(src, a.ld_src, a.rows, a.cols);
  // warp-uniform bound: both halves of a warp take part in the shuffles
  const long long me = (long long)blockIdx.x * (blockDim.x / 16) + threadIdx.x / 16;
  for (long long base = me & ~1LL; base < total; base += half_warps * kUnroll) {
    Raw8<T> raw[kUnroll];
    long long at[kUnroll];
    int row[kUnroll], group[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      at[u] = base + (me & 1) + u * half_warps;
      row[u] = static_cast<int>(at[u] / groups);
      group[u] = static_cast<int>(at[u] - (long long)row[u] * groups);
      const int col = group[u] * kBlock + lane16 * 8;
      raw[u] = {};
      if (at[u] < total && col < a.cols)
        raw[u] = b128::load8_any(src + (size_t)row[u] * a.ld_src + col, a.cols - col, in);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t top = b128::top_bits(raw[u]);
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const bool any = __any_sync(0xffffffffu, top >= b128::kInfBits);
      if (any) {
        float v[8], m = 0.0f;
        b128::unpack(raw[u], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, b128::finite_magnitude(v[j]));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        top = __float_as_uint(m);
      }
      const uint32_t byte = b128::scale_byte(__uint_as_float(top));
      const float inv = b128::scale_reciprocal(byte);
      const int col = group[u] * kBlock + lane16 * 8;
      if (at[u] < total && col < a.cols) {
        b128::store_bytes(a.dst + (size_t)row[u] * a.ld_dst + col,
                          any ? row_bytes<true>(raw[u], inv) : row_bytes<false>(raw[u], inv),
                          a.cols - col, a.dst_vec);
        if (lane16 == 0)
          a.scale[(size_t)row[u] * a.ld_scale + group[u]] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// What a thread of a tile holds: 8 rows x 8 columns.
template <typename T>
struct Piece {
  Raw8<T> raw[8];
  int row, col, nrow, ncol;  // in the matrix; how much of it is there (up to 8)
};

// Columns 2 k and 2 k + 1 of the piece, rows downwards, each by its own.
template <bool kAny>
__device__ __forceinline__ void column_bytes(const Raw8<__nv_bfloat16> (&raw)[8], int k, float inv0,
                                             float inv1, uint2 (&q)[2]) {
  float2 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 r = raw[i].a;
    v[i] = b128::mul_bf16x2(k == 0 ? r.x : k == 1 ? r.y : k == 2 ? r.z : r.w,
                            __float_as_uint(inv0), __float_as_uint(inv1));
  }
  q[0] = make_uint2(b128::e4m3x4<kAny>(v[0].x, v[1].x, v[2].x, v[3].x),
                    b128::e4m3x4<kAny>(v[4].x, v[5].x, v[6].x, v[7].x));
  q[1] = make_uint2(b128::e4m3x4<kAny>(v[0].y, v[1].y, v[2].y, v[3].y),
                    b128::e4m3x4<kAny>(v[4].y, v[5].y, v[6].y, v[7].y));
}
template <bool kAny>
__device__ __forceinline__ void column_bytes(const Raw8<float> (&raw)[8], int k, float inv0,
                                             float inv1, uint2 (&q)[2]) {
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 r = k < 2 ? raw[i].a : raw[i].b;
      const int at = 2 * (k & 1) + d;
      v[i] = __uint_as_float(at == 0 ? r.x : at == 1 ? r.y : at == 2 ? r.z : r.w);
    }
    q[d] = b128::e4m3x8<kAny>(v, d == 0 ? inv0 : inv1);
  }
}

// Writes both forms; row_inv and col_inv are the reciprocals of the scales of
// the piece's rows and columns.  kWhole: all of the tile is there, in aligned
// chunks, and finite.
template <bool kWhole, typename T>
__device__ __forceinline__ void store_piece(const QuantArgs &a, const Piece<T> &p,
                                            const float *row_inv, const float *col_inv) {
  if (a.dst != nullptr && (kWhole || p.ncol > 0)) {
    uint8_t *to = a.dst + (size_t)p.row * a.ld_dst + p.col;
#pragma unroll
    for (int i = 0; i < 8; ++i, to += a.ld_dst) {
      const uint2 q = row_bytes<!kWhole>(p.raw[i], row_inv[i]);
      if constexpr (kWhole) *reinterpret_cast<uint2 *>(to) = q;
      else if (i < p.nrow) b128::store_bytes(to, q, p.ncol, a.dst_vec);
    }
  }
  if (a.dst_t != nullptr && (kWhole || p.nrow > 0)) {
    uint8_t *to = a.dst_t + (size_t)p.col * a.ld_dst_t + p.row;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint2 q[2];
      column_bytes<!kWhole>(p.raw, k, col_inv[2 * k], col_inv[2 * k + 1], q);
#pragma unroll
      for (int d = 0; d < 2; ++d, to += a.ld_dst_t) {
        if constexpr (kWhole) *reinterpret_cast<uint2 *>(to) = q[d];
        else if (2 * k + d < p.ncol) b128::store_bytes(to, q[d], p.nrow, a.dst_t_vec);
      }
    }
  }
}

struct TileShared {
  uint32_t row_part[4][kBlock], col_part[2][kBlock];
  float row_inv[kBlock], col_inv[kBlock];
};

// Maxima of the tile's rows and columns (or of all of it), their scales and
// the reciprocals.  kFinite: over the bits of all values, and true if any is
// not finite, when nothing has been written; else over the finite ones.
template <bool kFinite, typename T>
__device__ __forceinline__ bool tile_scales(const QuantArgs &a, const Piece<T> &p, int tile_r,
                                            int row_in, int col_in, TileShared &sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wc = warp & 3, wr = warp >> 2, lc = lane & 3, lr = lane >> 2;
  uint32_t rmax[8], cmax[8];
  if constexpr (kFinite) {
    b128::tops(p.raw, rmax, cmax);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rmax[i] = cmax[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[8];
      b128::unpack(p.raw[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = __float_as_uint(b128::finite_magnitude(v[j]));
        rmax[i] = max(rmax[i], m);
        cmax[j] = max(cmax[j], m);
      }
    }
  }
  if (a.block_rows == kBlock) {  // one maximum: rows of the piece stand for all
#pragma unroll
    for (int i = 1; i < 8; ++i) rmax[0] = max(rmax[0], rmax[i]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      rmax[0] = max(rmax[0], __shfl_xor_sync(0xffffffffu, rmax[0], o));
    if (lane == 0) sh.row_part[wc][wr] = rmax[0];
  } else {
    if (a.dst != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // over the 4 lanes of a row, then the 4 warps
        rmax[i] = max(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], 1));
        rmax[i] = max(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], 2));
      }
      if (lc == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sh.row_part[wc][row_in + i] = rmax[i];
      }
    }
    if (a.dst_t != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
          cmax[i] = max(cmax[i], __shfl_xor_sync(0xffffffffu, cmax[i], o));
      if (lr == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sh.col_part[wr][col_in + i] = cmax[i];
      }
    }
  }
  __syncthreads();
  // thread t: row t of the tile, or column t - 128
  const int k = threadIdx.x & 127;
  const bool is_row = threadIdx.x < 128;
  uint32_t top = 0;
  if (a.block_rows == kBlock) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, sh.row_part[i & 3][i >> 2]);
  } else if (is_row && a.dst != nullptr) {
    top = max(max(sh.row_part[0][k], sh.row_part[1][k]),
              max(sh.row_part[2][k], sh.row_part[3][k]));
  } else if (!is_row && a.dst_t != nullptr) {
    top = max(sh.col_part[0][k], sh.col_part[1][k]);
  }
  const uint32_t byte = b128::scale_byte(__uint_as_float(top));
  (is_row ? sh.row_inv : sh.col_inv)[k] = b128::scale_reciprocal(byte);
  if (__syncthreads_or(top >= b128::kInfBits)) return true;
  const int tall = a.block_rows == 1 ? 1 : kBlock;  // rows that share a scale
  const int r = tile_r * kBlock + k, c = blockIdx.x * kBlock + k;
  if (is_row && a.dst != nullptr && r < a.rows && k % tall == 0)
    a.scale[(size_t)(r / tall) * a.ld_scale + blockIdx.x] = static_cast<uint8_t>(byte);
  if (!is_row && a.dst_t != nullptr && c < a.cols && k % tall == 0)
    a.scale_t[(size_t)(c / tall) * a.ld_scale_t + tile_r] = static_cast<uint8_t>(byte);
  return false;
}

// One CTA per 128 x 128 tile: a whole block of every kind, so its maxima
// need nothing from outside.  8 warps stand 4 (columns) x 2 (rows); a thread
// holds 8 rows x 8 columns, a warp 64 rows x 32 columns, so each row a warp
// loads is 64 bytes (bf16) and each column it stores 64 bytes: whole 32-byte
// sectors both ways with no trip through shared memory.  8192 x 8192 bf16 to both
// forms takes 49-53 us for 270 MB (41 us at the copy rate); what is left is a
// tile's chain of loads, maxima, two barriers and stores.  Two CTAs a SM that stay
// and hold the next tile in registers: 48 us there, 16 against 14 at 4096 x 4096.
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) k_quantize_tile(const QuantArgs a) {
  __shared__ TileShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col_in = (warp & 3) * 32 + (lane & 3) * 8, row_in = (warp >> 2) * 64 + (lane >> 2) * 8;
  const T *src = static_cast<const T *>(a.src);
  Piece<T> p;
  p.col = blockIdx.x * kBlock + col_in;
  p.ncol = min(8, a.cols - p.col);
  // a tile that is all there is stored without a look at its edges; where its
  // rows start is the loads' business
  const bool wide = (blockIdx.x + 1) * kBlock <= a.cols && (a.dst == nullptr || a.dst_vec) &&
                    (a.dst_t == nullptr || a.dst_t_vec);
  const b128::Bounds in = b128::Bounds::of(src, a.ld_src, a.rows, a.cols);
  dev::grid_dep_wait();
  dev::grid_dep_launch();

  for (int tile_r = blockIdx.y; tile_r < b128::groups_of(a.rows); tile_r += gridDim.y) {
    p.row = tile_r * kBlock + row_in;
    p.nrow = min(8, a.rows - p.row);
    const T *from = src + (size_t)p.row * a.ld_src + p.col;
    const bool whole = wide && (tile_r + 1) * kBlock <= a.rows;
    if (whole && a.src_vec) {
#pragma unroll
      for (int i = 0; i < 8; ++i, from += a.ld_src) p.raw[i] = b128::load8(from);
    } else if (a.src_vec) {
#pragma unroll
      for (int i = 0; i < 8; ++i, from += a.ld_src) {
        p.raw[i] = {};
        if (i < p.nrow) p.raw[i] = b128::load8_any(from, p.ncol, in);
      }
    } else {
      // four rows at a time on their way: one after the other, 6606 x 6634 bf16
      // both ways took 66 us instead of 53
#pragma unroll
      for (int half = 0; half < 8; half += 4) {
        b128::Fetch8<T> row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          row[i] = b128::Fetch8<T>(from + i * a.ld_src, half + i < p.nrow ? p.ncol : 0, in);
#pragma unroll
        for (int i = 0; i < 4; ++i, from += a.ld_src)
          p.raw[half + i] = row[i].get(from, half + i < p.nrow ? p.ncol : 0);
      }
    }
    const bool any = tile_scales<true>(a, p, tile_r, row_in, col_in, sh);
    if (any) tile_scales<false>(a, p, tile_r, row_in, col_in, sh);
    if (whole && !any) store_piece<true>(a, p, sh.row_inv + row_in, sh.col_inv + col_in);
    else store_piece<false>(a, p, sh.row_inv + row_in, sh.col_inv + col_in);
    __syncthreads();  // the reciprocals are read before the next tile writes them
  }
}

template <typename T>
int launch_quantize(const QuantArgs &a, cudaStream_t stream) {
  const int tiles_c = b128::groups_of(a.cols), tiles_r = b128::groups_of(a.rows);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Rows alone: by tiles too where there are enough for the SMs and rows start on 16
  // bytes (us by rows, by tiles; bf16: 8192 x 8192 54, 35; 512 x 8192 4.4, 3.7; 128 x
  // 8192 2.2, 2.3; 2000 x 5001 12.1, 12.5; fp32: 60, 52; 4.7, 3.8; 2.3, 2.7; 15, 19)
  const long long tiles = (long long)tiles_c * tiles_r;
  const bool many = 4 * tiles >= 3LL * current_sm_count() && a.src_vec && a.dst_vec;
  if (a.block_rows == 1 && a.dst_t == nullptr && !many) {
    const long long ctas = ((long long)a.rows * tiles_c + 31) / 32;  // 16 blocks a CTA, twice
    const long long most = (long long)current_sm_count() * 8;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas < most ? ctas : most));
    CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_quantize_rows<T>, a));
    return CMB_OK;
  }
  cfg.gridDim = dim3(tiles_c, tiles_r < 65535 ? tiles_r : 65535);
  CMB_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_quantize_tile<T>, a));
  return CMB_OK;
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
  if (rows < 0 || cols < 0 || rows > b128::kMostExtent || cols > b128::kMostExtent)
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
  return src_type == CMB_BF16 ? launch_quantize<__nv_bfloat16>(a, stream)
                              : launch_quantize<float>(a, stream);
}
