// Microscaled 4-bit values, shared by the quantisation and the product: 32
// consecutive values along K share one scale 2^(byte - 127) (byte 255: not a
// number), each value one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign in 4 bits,
// two to a byte, the lower index in the lower half.
//
// Layout of [batch][rows][K]:
//   data  [batch][rows][row_bytes], row_bytes = 16 ceil(K / 32); values past K are 0;
//   scale [batch][ceil(rows / 128)][ceil(K / 128)][32][4][4] bytes: row r, block
//         j at [r / 128][j / 4][r % 32][r % 128 / 32][j % 4]; padding bytes are 0.
// 512 consecutive scale bytes (128 rows x 128 values) are what one copy into
// tensor memory spreads over its lanes, so a tile's scales are whole pieces.
#pragma once

#include "common.cuh"

namespace cvmm {
namespace mx {

constexpr int kBlock = 32;
constexpr int kPiece = 512;  // scale bytes of 128 rows x 128 values

__host__ __device__ __forceinline__ int64_t row_bytes(int64_t K) { return (K + 31) / 32 * 16; }
__host__ __device__ __forceinline__ int64_t pieces(int64_t n) { return (n + 127) / 128; }
__host__ __device__ __forceinline__ int64_t scale_bytes(int64_t rows, int64_t K) {
  return pieces(rows) * pieces(K) * kPiece;
}
// Byte offset of the four scales of row r, values 128 c .. 128 c + 127.
__host__ __device__ __forceinline__ int64_t scale_cell(int64_t r, int64_t c, int64_t k_pieces) {
  return ((r >> 7) * k_pieces + c) * kPiece + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// Magnitude bits of the largest |v| of a block -> scale byte: the exponent of
// the largest power of two not above it, less the 2 that 4-bit values reach
// above theirs. Zero and the smallest numbers give byte 0 (2^-127); infinities
// and NaN, whose bits are above every finite number's, give 255.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// 2^-(byte - 127), exact and normal for every byte scale_byte gives; 0 for 255.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
  if (byte == 255u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
}

// Eight scaled values, rounded to the nearest 4-bit value (ties to even, held
// at 6), packed low to high. A block that is not finite is all zeros.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8], float inv) {
  if (inv == 0.f) return 0u;
  uint32_t out;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(out)
      : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
        "f"(v[6] * inv), "f"(v[7] * inv));
  return out;
}

// The eight values of four packed bytes.
__device__ __forceinline__ void unpack8(uint32_t p, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(p));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 x = *reinterpret_cast<const __half2*>(&h[i]);
    v[2 * i] = __low2float(x);
    v[2 * i + 1] = __high2float(x);
  }
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace mx
}  // namespace cvmm
