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

// The value of one code (sign, two exponent bits, one more bit).
__device__ __forceinline__ float value_of_code(uint32_t c) {
  const uint32_t m = c & 7u;
  const uint32_t bits = m >= 2u ? ((126u + (m >> 1)) << 23) | ((m & 1u) << 22) : m ? 0x3f000000u : 0u;
  return __uint_as_float(bits | (c & 8u) << 28);
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

// n / d by a multiplication for n < 2^31 (m = floor(2^(31 + l) / d) + 1 with
// l = ceil(log2 d) is at most d / 2^(31 + l) too large, and n times that stays
// below one); larger n divide.
struct Divisor {
  uint32_t d, m, l;
  Divisor() = default;
  __host__ explicit Divisor(int64_t by) : d((uint32_t)by), m(0), l(0) {
    while (((uint64_t)1 << l) < d) ++l;
    if (d > 1) m = (uint32_t)((((uint64_t)1 << (31 + l)) / d) + 1);
  }
  __device__ __forceinline__ int64_t of(int64_t n) const {
    if (d == 1) return n;
    if (n >> 31) return n / d;
    return __umulhi((uint32_t)n, m) >> (l - 1);
  }
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 32 consecutive values of one type as the words they are loaded in.
template <int DT>
constexpr int kWords = DT == F32 ? 32 : 16;

// 32-byte accesses (address a multiple of 32).
__device__ __forceinline__ void ld_v8(uint32_t* w, const void* p) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void st_v8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Loads values `at` .. at + 31 of x (those past n are 0). vec: bytes that the
// address is a multiple of (32, 16, else value by value).
template <int DT>
__device__ __forceinline__ void load_block(uint32_t (&w)[kWords<DT>], const void* x, int64_t at, int n, int vec) {
  constexpr int W = kWords<DT>;
  const char* from = static_cast<const char*>(x) + at * (DT == F32 ? 4 : 2);
  if (n >= 32 && vec == 32) {
#pragma unroll
    for (int i = 0; i < W; i += 8) ld_v8(w + i, from + 4 * i);
  } else if (n >= 32 && vec == 16) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(from + 4 * i);
      w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
    }
  } else if (DT == F32) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = i < n ? reinterpret_cast<const uint32_t*>(from)[i] : 0u;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
    for (int i = 0; i < W; ++i)
      w[i] = (2 * i < n ? h[2 * i] : 0u) | (uint32_t)(2 * i + 1 < n ? h[2 * i + 1] : 0u) << 16;
  }
}

// Magnitude bits (as a 32-bit float's) of the largest of 32 values: the bits of
// a type order its magnitudes, infinities and NaN above the rest.
template <int DT>
__device__ __forceinline__ uint32_t block_magnitude(const uint32_t (&w)[kWords<DT>]) {
  uint32_t m = 0;
  if (DT == F32) {
#pragma unroll
    for (int i = 0; i < kWords<DT>; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
#pragma unroll
  for (int i = 0; i < kWords<DT>; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  m = max(m & 0xffffu, m >> 16);
  return DT == BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((uint16_t)m)));
}

template <int DT>
__device__ __forceinline__ uint4 pack_block(const uint32_t (&w)[kWords<DT>], float inv) {
  uint32_t out[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (DT == F32) f[j] = __uint_as_float(w[8 * h + j]);
      else f[j] = bits_to_float((uint16_t)(j & 1 ? w[4 * h + j / 2] >> 16 : w[4 * h + j / 2] & 0xffffu), DT);
    }
    out[h] = pack8(f, inv);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// Quantises blocks of rows whose K is contiguous, a lane a block, so that a
// scale needs no other lane and a row's data go out 16 bytes a lane; four lanes
// put a 4-byte cell of scales together. at(i) gives block i; blocks of a cell
// are consecutive and start at a multiple of 4. `first` is blocks before this
// thread's, `stride` blocks of a round. Two blocks of 16-bit values in flight a
// lane instead of one took registers that were better spent on more warps (x of
// 16384 x 1024: 13.7 against 8.8 us).
struct Block {
  int64_t src;     // element offset of the row's first value
  uint8_t* data;   // the row's data bytes
  uint32_t* cell;  // where the four scales go
  int64_t j;       // which block of the row
  bool row;        // false: a padding row, scales 0 and no data
};

template <int DT, class At>
__device__ __forceinline__ void quantize_blocks(const void* __restrict__ x, int64_t K, int vec, int64_t items,
                                                int64_t first, int64_t stride, At at) {
  const int lane4 = threadIdx.x & 3;
  // Every lane of a warp runs the same number of rounds (shuffles below).
  const int64_t rounds = (items + stride - 1) / stride;
  for (int64_t i = 0; i < rounds; ++i) {
    const int64_t it = first + i * stride;
    const bool live = it < items;
    const Block q = at(live ? it : 0);
    const bool in = live && q.row && q.j * 32 < K;  // this block exists
    uint32_t w[kWords<DT>];
    load_block<DT>(w, x, q.src + q.j * 32, in ? (int)imin64(K - q.j * 32, 32) : 0, vec);
    const uint32_t byte = in ? scale_byte(block_magnitude<DT>(w)) : 0u;
    if (in) *reinterpret_cast<uint4*>(q.data + q.j * 16) = pack_block<DT>(w, inverse_scale(byte));
    uint32_t cell = byte << (8 * lane4);
    cell |= __shfl_xor_sync(0xffffffffu, cell, 1);
    cell |= __shfl_xor_sync(0xffffffffu, cell, 2);
    if (live && lane4 == 0) *q.cell = cell;
  }
}

// The largest of 32, 16 and 0 that an address, and steps of a and b bytes from it, are multiples of.
inline int vector_bytes(const void* p, int64_t a, int64_t b) {
  const uint64_t bits = (uint64_t)(uintptr_t)p | (uint64_t)a | (uint64_t)b;
  return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 0;
}

}  // namespace mx
}  // namespace cvmm
