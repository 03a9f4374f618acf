// Microscaled 4-bit quantisation and its inverse (cvmm_mx_quantize,
// cvmm_mx_dequantize). The layout is described in mx.cuh.
#include "launch.h"
#include "mx.cuh"

namespace cvmm {
namespace mx {

// Strided source or destination [batch][rows][K], in elements.
struct View {
  int64_t batch, rows, K, sb, sr, sk;
};

// Quantises rows whose K is contiguous. 16 lanes take 128 values of one row (8
// each): four lanes share a block's scale, and the 16 write one 4-byte scale
// cell and 64 data bytes. Rows up to a multiple of 128 are visited, so that
// every padding scale is written (0).
__global__ void __launch_bounds__(256) quantize_k_kernel(const void* __restrict__ x, int dtype, View v, bool vec,
                                                         uint8_t* __restrict__ data, uint8_t* __restrict__ scale) {
  pdl_enter();
  const int64_t kp = pieces(v.K), rp = pieces(v.rows), rb = row_bytes(v.K);
  const int64_t items = v.batch * rp * 128 * kp;
  const int sub = threadIdx.x & 15;
  const int64_t stride = (int64_t)gridDim.x * (blockDim.x / 16);
  // Both halves of a warp run the same number of rounds (shuffles below).
  const int64_t rounds = (items + stride - 1) / stride;
  for (int64_t i = 0; i < rounds; ++i) {
    const int64_t it = blockIdx.x * (int64_t)(blockDim.x / 16) + (threadIdx.x >> 4) + i * stride;
    const bool live = it < items;
    const int64_t c = live ? it % kp : 0, br = live ? it / kp : 0;
    const int64_t b = br / (rp * 128), r = br % (rp * 128);
    const int64_t k0 = c * 128 + sub * 8;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    if (live && r < v.rows && k0 < v.K) {
      const int64_t at = b * v.sb + r * v.sr + k0;
      if (vec && k0 + 8 <= v.K) {
        load8(static_cast<const char*>(x) + at * dtype_bytes(dtype), dtype, f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k0 + j < v.K) f[j] = load_as_float(x, dtype, at + j);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, magnitude(f[j]));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const bool in = live && r < v.rows && c * 128 + (sub & 12) * 8 < v.K;  // this block exists
    const uint32_t byte = in ? scale_byte(m) : 0u;
    if (in) *reinterpret_cast<uint32_t*>(data + (b * v.rows + r) * rb + k0 / 2) = pack8(f, inverse_scale(byte));
    uint32_t cell = byte << (8 * ((sub >> 2) & 3));
    cell |= __shfl_xor_sync(0xffffffffu, cell, 4);
    cell |= __shfl_xor_sync(0xffffffffu, cell, 8);
    if (live && sub == 0)
      *reinterpret_cast<uint32_t*>(scale + b * scale_bytes(v.rows, v.K) + scale_cell(r, c, kp)) = cell;
  }
}

// Quantises rows that are contiguous along the rows (or strided both ways): a
// warp takes 32 rows x 128 values, a lane one row, so that a load of one k is
// contiguous over the lanes and a lane packs its own blocks.
__global__ void __launch_bounds__(256) quantize_r_kernel(const void* __restrict__ x, int dtype, View v,
                                                         uint8_t* __restrict__ data, uint8_t* __restrict__ scale) {
  pdl_enter();
  const int64_t kp = pieces(v.K), rp = pieces(v.rows), rb = row_bytes(v.K);
  const int64_t items = v.batch * rp * 4 * kp;
  const int lane = threadIdx.x & 31;
  const int64_t stride = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t it = blockIdx.x * (int64_t)(blockDim.x / 32) + (threadIdx.x >> 5); it < items; it += stride) {
    const int64_t q = it % (rp * 4), bc = it / (rp * 4);
    const int64_t c = bc % kp, b = bc / kp;
    const int64_t r = q * 32 + lane;
    uint32_t cell = 0;
    for (int blk = 0; blk < 4; ++blk) {
      const int64_t k0 = c * 128 + blk * 32;
      if (k0 >= v.K) break;
      float f[4][8];
      uint32_t m = 0;
      const int64_t at = b * v.sb + r * v.sr + k0 * v.sk;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        f[j >> 3][j & 7] = r < v.rows && k0 + j < v.K ? load_as_float(x, dtype, at + j * v.sk) : 0.f;
        m = max(m, magnitude(f[j >> 3][j & 7]));
      }
      if (r >= v.rows) continue;
      const uint32_t byte = scale_byte(m);
      const float inv = inverse_scale(byte);
      cell |= byte << (8 * blk);
      *reinterpret_cast<uint4*>(data + (b * v.rows + r) * rb + k0 / 2) =
          make_uint4(pack8(f[0], inv), pack8(f[1], inv), pack8(f[2], inv), pack8(f[3], inv));
    }
    *reinterpret_cast<uint32_t*>(scale + b * scale_bytes(v.rows, v.K) + scale_cell(r, c, kp)) = cell;
  }
}

// Values of 8 consecutive k of one row, K contiguous in the output.
__global__ void __launch_bounds__(256) dequantize_k_kernel(const uint8_t* __restrict__ data,
                                                           const uint8_t* __restrict__ scale, View v, bool vec,
                                                           void* __restrict__ out, int dtype) {
  pdl_enter();
  const int64_t kp = pieces(v.K), rb = row_bytes(v.K), per = (v.K + 7) / 8;
  const int64_t items = v.batch * v.rows * per;
  for (int64_t it = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; it < items;
       it += (int64_t)gridDim.x * blockDim.x) {
    const int64_t br = it / per, k0 = (it - br * per) * 8;
    const int64_t b = br / v.rows, r = br - b * v.rows;
    float f[8];
    unpack8(*reinterpret_cast<const uint32_t*>(data + br * rb + k0 / 2), f);
    const float s = scale_value(scale[b * scale_bytes(v.rows, v.K) + scale_cell(r, k0 >> 7, kp) + ((k0 >> 5) & 3)]);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s;
    const int64_t at = b * v.sb + r * v.sr + k0;
    if (vec && k0 + 8 <= v.K) {
      store8(static_cast<char*>(out) + at * dtype_bytes(dtype), dtype, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < v.K) store_from_float(out, dtype, at + j, f[j]);
    }
  }
}

// Values with the rows contiguous in the output: a lane takes one block of its row.
__global__ void __launch_bounds__(256) dequantize_r_kernel(const uint8_t* __restrict__ data,
                                                           const uint8_t* __restrict__ scale, View v,
                                                           void* __restrict__ out, int dtype) {
  pdl_enter();
  const int64_t kp = pieces(v.K), rb = row_bytes(v.K), blocks = rb / 16, rq = (v.rows + 31) / 32;
  const int64_t items = v.batch * rq * blocks;
  const int lane = threadIdx.x & 31;
  const int64_t stride = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t it = blockIdx.x * (int64_t)(blockDim.x / 32) + (threadIdx.x >> 5); it < items; it += stride) {
    const int64_t q = it % rq, bb = it / rq, blk = bb % blocks, b = bb / blocks;
    const int64_t r = q * 32 + lane;
    if (r >= v.rows) continue;
    const uint4 p = *reinterpret_cast<const uint4*>(data + (b * v.rows + r) * rb + blk * 16);
    const float s = scale_value(scale[b * scale_bytes(v.rows, v.K) + scale_cell(r, blk >> 2, kp) + (blk & 3)]);
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
    const int64_t at = b * v.sb + r * v.sr + blk * 32 * v.sk;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float f[8];
      unpack8(w[h], f);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (blk * 32 + h * 8 + j < v.K) store_from_float(out, dtype, at + (h * 8 + j) * v.sk, f[j] * s);
    }
  }
}

static int check_view(const View& v, const char* msg) {
  if (v.batch < 0 || v.rows < 0 || v.K < 0 || v.rows > (int64_t)INT32_MAX || v.K > (int64_t)INT32_MAX)
    return fail(CVMM_ERR_INVALID_ARG, msg);
  return CVMM_OK;
}

static int quantize(const void* x, int dtype, const View& v, uint8_t* data, uint8_t* scale, cudaStream_t stream) {
  const int64_t size = (int64_t)dtype_size(dtype);
  if (v.sk == 1) {
    const bool vec = al16(x) && v.sr * size % 16 == 0 && v.sb * size % 16 == 0;
    const int64_t items = v.batch * pieces(v.rows) * 128 * pieces(v.K);
    launch(quantize_k_kernel, grid_for(items, 16), 256, 0, stream, x, dtype, v, vec, data, scale);
  } else {
    const int64_t items = v.batch * pieces(v.rows) * 4 * pieces(v.K);
    launch(quantize_r_kernel, grid_for(items, 8), 256, 0, stream, x, dtype, v, data, scale);
  }
  return check_launch("cvmm_mx_quantize");
}

}  // namespace mx
}  // namespace cvmm

extern "C" {

int cvmm_mx_quantize(const void* x, int x_dtype, int64_t n_batch, int64_t rows, int64_t k_dim, int64_t stride_b,
                     int64_t stride_r, int64_t stride_k, uint8_t* data, uint8_t* scale, cvmm_stream_t stream) {
  using namespace cvmm;
  const mx::View v = {n_batch, rows, k_dim, stride_b, stride_r, stride_k};
  if (!is_float_dtype(x_dtype)) return fail(CVMM_ERR_UNSUPPORTED_DTYPE, "cvmm_mx_quantize: unsupported dtype");
  if (int rc = mx::check_view(v, "cvmm_mx_quantize: bad sizes")) return rc;
  if (n_batch == 0 || rows == 0 || k_dim == 0) return CVMM_OK;
  if (!x || !data || !scale) return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_quantize: null pointer");
  if (!al16(data) || !al16(scale)) return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_quantize: data and scale must be 16-byte aligned");
  return mx::quantize(x, x_dtype, v, data, scale, reinterpret_cast<cudaStream_t>(stream));
}

int cvmm_mx_dequantize(const uint8_t* data, const uint8_t* scale, int64_t n_batch, int64_t rows, int64_t k_dim,
                       int64_t stride_b, int64_t stride_r, int64_t stride_k, void* out, int out_dtype,
                       cvmm_stream_t stream) {
  using namespace cvmm;
  const mx::View v = {n_batch, rows, k_dim, stride_b, stride_r, stride_k};
  if (!is_float_dtype(out_dtype)) return fail(CVMM_ERR_UNSUPPORTED_DTYPE, "cvmm_mx_dequantize: unsupported dtype");
  if (int rc = mx::check_view(v, "cvmm_mx_dequantize: bad sizes")) return rc;
  if (n_batch == 0 || rows == 0 || k_dim == 0) return CVMM_OK;
  if (!out || !data || !scale) return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_dequantize: null pointer");
  if (!al16(data) || !al16(scale)) return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_dequantize: data and scale must be 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (stride_k == 1) {
    const int64_t size = (int64_t)dtype_size(out_dtype);
    const bool vec = al16(out) && stride_r * size % 16 == 0 && stride_b * size % 16 == 0;
    launch(mx::dequantize_k_kernel, grid_for(n_batch * rows * ((k_dim + 7) / 8), 256), 256, 0, s, data, scale, v, vec,
           out, out_dtype);
  } else {
    launch(mx::dequantize_r_kernel, grid_for(n_batch * ((rows + 31) / 32) * ((k_dim + 31) / 32), 8), 256, 0, s, data,
           scale, v, out, out_dtype);
  }
  return check_launch("cvmm_mx_dequantize");
}

}  // extern "C"
