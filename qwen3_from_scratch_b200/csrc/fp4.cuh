// Rows held in microscaled 4-bit floating point: the format, and rounding to it.
//
// A row of K values is cut into blocks of 32.  A block has one scale, a power of two 2^(b - 127) held as the byte b (255
// stands for NaN), and every value is held in four bits: a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, times the scale.
//   codes   [R, 16 ceil(K / 32)] bytes: value 2 i in the low half of byte i, value 2 i + 1 in the high half; zeros beyond K
//   scales  [ceil(R / 128), ceil(K / 128)] tiles of 512 bytes: row r, block j at 16 (r % 32) + 4 ((r % 128) / 32) + j % 4 of
//           tile (r / 128, j / 4), which is the order in which tcgen05.cp takes the scales of 128 rows into tensor memory;
//           the bytes of a row's blocks beyond K are zero, those of rows beyond R are never looked at
// Rounding a block: its scale is the smallest power of two X with max|x| <= 7 X, so a block's largest value lies in (3.5, 7]
// X and one above 6 X goes to 6 X, which is as near as a step of the scale above would bring it (in normal values this leaves an
// rms error of 11.2 %, the rule max|x| <= 6 X 11.5 %, X = 2^(floor(log2 max) - 2) 11.5 %).  Each x / X, exact because X is a
// power of two, goes to the nearest code, ties to the even one.  A block with a value that is not finite has the scale NaN.
#pragma once

#include "common.cuh"

namespace q3 {

constexpr int FP4_BLOCK = 32;        // values that share a scale
constexpr int FP4_TILE = 128;        // rows, and values of k, of a tile of scales
constexpr int FP4_TILE_BYTES = 512;  // 128 rows x 4 blocks

__host__ __device__ __forceinline__ int fp4_pitch(int k) { return (k + FP4_BLOCK - 1) / FP4_BLOCK * 16; }
__host__ __device__ __forceinline__ int fp4_tiles(int n) { return (n + FP4_TILE - 1) / FP4_TILE; }

// Where the four scale bytes of row r, blocks 4 c .. 4 c + 3 are; `across`: tiles per row of tiles.
__device__ __forceinline__ size_t fp4_scale_word(int r, int c, int across) {
  return ((size_t)(r / FP4_TILE) * across + c) * FP4_TILE_BYTES + (r % 32) * 16 + (r % FP4_TILE) / 32 * 4;
}

// The scale's byte from the largest |x| of a block, given by its bits (which are in the order of the numbers, with
// infinity and NaN above all).
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int b = (int)((top + 0x1fffffu) >> 23) - 2;  // one more where the significand is above 1.75, then 7 = 1.75 x 2^2
  return b < 0 ? 0u : (uint32_t)b;
}
// The larger of `top` and |v|, bits for bits; a NaN stays one.
__device__ __forceinline__ uint32_t fp4_top(uint32_t top, float v) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(v)), "f"(__uint_as_float(top)));
  return __float_as_uint(m);
}
// 1 / X.  b is at most 253, so this is a normal number; 255 gives 0, which leaves zeros (and NaN) for the codes.
__device__ __forceinline__ float fp4_inverse_scale(uint32_t b) { return b == 255u ? 0.f : __uint_as_float((254u - b) << 23); }

// Eight values, already divided by their scale, as codes: value i in bits 4 i .. 4 i + 3.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ uint32_t fp4_pack2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 a;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tmov.b32 %0, {a, a, a, a};\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
  return r & 255u;
}
// Eight values of a row in each of four neighbouring lanes, a block between them: their codes, and the block's scale.  Every
// lane of the warp takes part.
__device__ __forceinline__ uint32_t fp4_round8(const float (&v)[8], uint32_t* scale_byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fp4_top(top, v[i]);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t b = fp4_scale_byte(top);
  const float inv = fp4_inverse_scale(b);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = v[i] * inv;
  *scale_byte = b;
  return b == 255u ? 0u : fp4_pack8(s);
}
// The scales of the four blocks that sixteen neighbouring lanes hold, as a word (in every fourth lane's order).
__device__ __forceinline__ uint32_t fp4_scale_word_of_16(uint32_t byte) {
  uint32_t w = byte << (8 * ((threadIdx.x >> 2) & 3));
  w |= __shfl_xor_sync(0xffffffffu, w, 4);
  w |= __shfl_xor_sync(0xffffffffu, w, 8);
  return w;
}

}  // namespace q3
