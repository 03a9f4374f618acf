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

// Quantises rows whose K is contiguous. Rows up to a multiple of 128 are
// visited, so that every padding scale is written (0).
template <int DT>
__global__ void __launch_bounds__(256)
quantize_k_kernel(const void* __restrict__ x, View v, int vec, Divisor by_blocks, Divisor by_rows,
                  uint8_t* __restrict__ data, uint8_t* __restrict__ scale) {
  pdl_enter();
  const int64_t blocks = by_blocks.d, rows = by_rows.d, rb = row_bytes(v.K);  // blocks: 4 a piece; rows: 128 a piece
  auto at = [&](int64_t it) -> Block {
    const int64_t br = by_blocks.of(it), j = it - br * blocks;
    const int64_t b = by_rows.of(br), r = br - b * rows;
    return {b * v.sb + r * v.sr, data + (b * v.rows + r) * rb,
            reinterpret_cast<uint32_t*>(scale + b * rows * blocks + scale_cell(r, j >> 2, blocks >> 2)), j, r < v.rows};
  };
  quantize_blocks<DT>(x, v.K, vec, v.batch * rows * blocks, blockIdx.x * (int64_t)blockDim.x + threadIdx.x,
                      (int64_t)gridDim.x * blockDim.x, at);
}

// Quantises rows that are contiguous along the rows (or strided both ways). A
// block takes 32 rows x 256 values: in a warp of 32 values a lane is one row, so
// a load of one k is contiguous over the lanes and a lane packs its own block;
// the 128 bytes and 8 scales of every row then go out through shared memory in
// whole sectors.
__global__ void __launch_bounds__(256) quantize_r_kernel(const void* __restrict__ x, int dtype, View v,
                                                         uint8_t* __restrict__ data, uint8_t* __restrict__ scale) {
  pdl_enter();
  __shared__ uint4 packed[32][9];      // [row][32-value block], one block of padding against bank conflicts
  __shared__ __align__(8) uint8_t bytes[32][8];
  const int64_t kp = pieces(v.K), rp = pieces(v.rows), rb = row_bytes(v.K), kh = (kp + 1) / 2;
  const int64_t items = v.batch * kh * rp * 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t q = it % (rp * 4), bc = it / (rp * 4);
    const int64_t h = bc % kh, b = bc / kh;
    const int64_t r = q * 32 + lane, k0 = h * 256 + warp * 32;
    float f[4][8];
    uint32_t m = 0;
    const int64_t at = b * v.sb + r * v.sr + k0 * v.sk;
    if (r < v.rows && k0 + 32 <= v.K) {
      if (dtype == F32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j >> 3][j & 7] = static_cast<const float*>(x)[at + j * v.sk];
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          f[j >> 3][j & 7] = bits_to_float(static_cast<const uint16_t*>(x)[at + j * v.sk], dtype);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        f[j >> 3][j & 7] = r < v.rows && k0 + j < v.K ? load_as_float(x, dtype, at + j * v.sk) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) m = max(m, magnitude(f[j >> 3][j & 7]));
    const uint32_t byte = r < v.rows && k0 < v.K ? scale_byte(m) : 0u;
    const float inv = inverse_scale(byte);
    packed[lane][warp] = make_uint4(pack8(f[0], inv), pack8(f[1], inv), pack8(f[2], inv), pack8(f[3], inv));
    bytes[lane][warp] = (uint8_t)byte;
    __syncthreads();
    const int row = threadIdx.x >> 3, blk = threadIdx.x & 7;
    const int64_t ro = q * 32 + row;
    if (ro < v.rows && h * 128 + blk * 16 < rb)
      *reinterpret_cast<uint4*>(data + (b * v.rows + ro) * rb + h * 128 + blk * 16) = packed[row][blk];
    if (threadIdx.x < 64) {
      const int64_t rs = q * 32 + (threadIdx.x & 31), c = 2 * h + (threadIdx.x >> 5);
      if (c < kp)
        *reinterpret_cast<uint32_t*>(scale + b * scale_bytes(v.rows, v.K) + scale_cell(rs, c, kp)) =
            *reinterpret_cast<const uint32_t*>(&bytes[threadIdx.x & 31][4 * (threadIdx.x >> 5)]);
    }
    __syncthreads();
  }
}

// Values of one block of a row a lane, K contiguous in the output; kDeq blocks in flight.
constexpr int kDeq = 2;
__global__ void __launch_bounds__(256)
dequantize_k_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scale, View v, int vec,
                    Divisor by_blocks, Divisor by_rows, void* __restrict__ out, int dtype) {
  pdl_enter();
  const int64_t kp = pieces(v.K), rb = row_bytes(v.K), blocks = by_blocks.d;
  const int64_t items = v.batch * v.rows * blocks, stride = (int64_t)gridDim.x * blockDim.x;
  const int64_t batch_bytes = scale_bytes(v.rows, v.K);
  const int size = dtype_bytes(dtype);
  for (int64_t base = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; base < items; base += kDeq * stride) {
    uint4 packed[kDeq];
    uint32_t byte[kDeq];
    int64_t at[kDeq];
    int n[kDeq];
#pragma unroll
    for (int u = 0; u < kDeq; ++u) {
      const int64_t it = base + u * stride;
      if (it >= items) break;
      const int64_t br = by_blocks.of(it), j = it - br * blocks;
      const int64_t b = by_rows.of(br), r = br - b * v.rows;
      packed[u] = *reinterpret_cast<const uint4*>(data + br * rb + j * 16);
      byte[u] = scale[b * batch_bytes + scale_cell(r, j >> 2, kp) + (j & 3)];
      at[u] = b * v.sb + r * v.sr + j * 32;
      n[u] = (int)imin64(32, v.K - j * 32);
    }
#pragma unroll
    for (int u = 0; u < kDeq; ++u) {
      if (base + u * stride >= items) break;
      const float s = scale_value(byte[u]);
      const uint32_t w[4] = {packed[u].x, packed[u].y, packed[u].z, packed[u].w};
      char* to = static_cast<char*>(out) + at[u] * size;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 16 values
        float f[2][8];
        unpack8(w[2 * h], f[0]);
        unpack8(w[2 * h + 1], f[1]);
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j >> 3][j & 7] *= s;
        if (n[u] < 32) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (16 * h + j < n[u]) store_from_float(to, dtype, 16 * h + j, f[j >> 3][j & 7]);
        } else if (vec == 16) {
          store8(to + 16 * h * size, dtype, f[0]);
          store8(to + (16 * h + 8) * size, dtype, f[1]);
        } else if (dtype == F32) {
          st_v8(to + 64 * h, reinterpret_cast<const uint32_t*>(f[0]));
          st_v8(to + 64 * h + 32, reinterpret_cast<const uint32_t*>(f[1]));
        } else {
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = pack2(f[j >> 2][2 * (j & 3)], f[j >> 2][2 * (j & 3) + 1], dtype);
          st_v8(to + 32 * h, o);
        }
      }
    }
  }
}

// The same where the output has no 16-byte alignment: a warp takes four blocks,
// a lane one value of each (32768 x 2047 bf16: 329 us where a lane a block, value
// by value, took 459, both under a profiler; 285 without one).
__global__ void __launch_bounds__(256)
dequantize_any_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scale, View v, Divisor by_blocks,
                      Divisor by_rows, void* __restrict__ out, int dtype) {
  pdl_enter();
  const int64_t kp = pieces(v.K), rb = row_bytes(v.K), blocks = by_blocks.d;
  const int64_t items = v.batch * v.rows * blocks, batch_bytes = scale_bytes(v.rows, v.K);
  const int lane = threadIdx.x & 31;
  for (int64_t base = (blockIdx.x * 8ll + threadIdx.x / 32) * 4; base < items; base += gridDim.x * 32ll) {
    uint32_t packed[4], byte[4];
    int64_t at[4];
    bool in[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t it = imin64(base + u, items - 1);
      const int64_t br = by_blocks.of(it), j = it - br * blocks;
      const int64_t b = by_rows.of(br), r = br - b * v.rows;
      packed[u] = data[br * rb + j * 16 + lane / 2];
      byte[u] = scale[b * batch_bytes + scale_cell(r, j >> 2, kp) + (j & 3)];
      at[u] = b * v.sb + r * v.sr + j * 32 + lane;
      in[u] = base + u < items && j * 32 + lane < v.K;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = value_of_code(packed[u] >> (4 * (lane & 1)));
      if (in[u]) store_from_float(out, dtype, at[u], f * scale_value(byte[u]));
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
    const int vec = vector_bytes(x, v.sr * size, v.sb * size);
    const int64_t items = v.batch * pieces(v.rows) * 128 * pieces(v.K) * 4;
    const auto kernel = dtype == F32 ? quantize_k_kernel<F32> : dtype == BF16 ? quantize_k_kernel<BF16> : quantize_k_kernel<F16>;
    launch(kernel, grid_for(items, 256), 256, 0, stream, x, v, vec, Divisor(pieces(v.K) * 4),
           Divisor(pieces(v.rows) * 128), data, scale);
  } else {
    const int64_t items = v.batch * pieces(v.rows) * 4 * ((pieces(v.K) + 1) / 2);
    launch(quantize_r_kernel, (unsigned)std::min<int64_t>(items, 148 * 32), 256, 0, stream, x, dtype, v, data, scale);
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
    const int64_t blocks = (k_dim + 31) / 32;
    const int vec = mx::vector_bytes(out, stride_r * size, stride_b * size);
    if (vec)
      launch(mx::dequantize_k_kernel, grid_for(n_batch * rows * blocks, 256), 256, 0, s, data, scale, v, vec,
             mx::Divisor(blocks), mx::Divisor(rows), out, out_dtype);
    else
      launch(mx::dequantize_any_kernel, grid_for(n_batch * rows * blocks, 32), 256, 0, s, data, scale, v,
             mx::Divisor(blocks), mx::Divisor(rows), out, out_dtype);
  } else {
    launch(mx::dequantize_r_kernel, grid_for(n_batch * ((rows + 31) / 32) * ((k_dim + 31) / 32), 8), 256, 0, s, data,
           scale, v, out, out_dtype);
  }
  return check_launch("cvmm_mx_dequantize");
}

}  // extern "C"
