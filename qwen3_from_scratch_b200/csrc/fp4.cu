// Rounding rows to microscaled 4-bit floating point (fp4.cuh), from memory and behind an RMSNorm.
//
// Both kernels pass over their data once; what bounds them is memory: 2 or 4 bytes in and 0.53 out per value (2 more where
// the rounded values are wanted as well), 8 to 10.5 per value of the norm, whose float32 stream is read and written.
#include "fp4.cuh"

namespace q3 {

template <typename T>
__device__ __forceinline__ void fp4_load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void fp4_load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void fp4_load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Columns col .. col + 7 of a row; zeros beyond K.  VEC: the row is on a 16-byte boundary.
template <typename T, bool VEC>
__device__ __forceinline__ void fp4_load_row8(const T* row, int col, int K, float (&v)[8]) {
  if (VEC && col + 8 <= K) {
    fp4_load8<T>(row + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < K ? to_float(row[col + i]) : 0.f;
  }
}

// ---------------------------------------------------------------- rows from memory
// The words (two bfloat16 or one float32 each) of values col .. col + 7 of a row; zeros beyond K.  VEC: the row is on a 16-byte
// boundary.  Other rows need be on no boundary but their type's: their words are read where they lie, those of a bfloat16 row that
// begins between two words as five, shifted by half a one.  Only the ends of rows, and the first value of all (`lo`: where the rows
// begin), are read one by one, so that nothing outside the rows is.
template <typename T, bool VEC>
__device__ __forceinline__ void fp4_load_words(const T* row, int col, int K, const T* lo, uint32_t (&w)[2 * sizeof(T)]) {
  constexpr int NW = 2 * sizeof(T);
  const T* const at = row + col;
  if (VEC && col + 8 <= K) {
#pragma unroll
    for (int q = 0; q < NW / 4; ++q) {
      const uint4 x = reinterpret_cast<const uint4*>(at)[q];
      w[4 * q] = x.x; w[4 * q + 1] = x.y; w[4 * q + 2] = x.z; w[4 * q + 3] = x.w;
    }
    return;
  }
  const bool between = ((uintptr_t)at & 3) != 0;  // uniform over the warp
  if (!VEC && col + 9 <= K && (!between || at > lo)) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(between ? at - 1 : at);
#pragma unroll
    for (int j = 0; j < NW; ++j) w[j] = __ldg(u + j);
    if (between) {
      const uint32_t last = __ldg(u + NW);
#pragma unroll
      for (int j = 0; j < NW; ++j) w[j] = __funnelshift_r(w[j], j + 1 < NW ? w[j + 1] : last, 16);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    if (sizeof(T) == 4) {
      w[j] = col + j < K ? *reinterpret_cast<const uint32_t*>(at + j) : 0u;
    } else {
      const uint32_t x = col + 2 * j < K ? *reinterpret_cast<const uint16_t*>(at + 2 * j) : 0u;
      w[j] = x | (col + 2 * j + 1 < K ? (uint32_t)*reinterpret_cast<const uint16_t*>(at + 2 * j + 1) << 16 : 0u);
    }
  }
}

// What eight codes of a block with this scale stand for, as bfloat16 (every such value is one, but for the 2^128 of a block that
// reaches beyond 1.75 x 2^127: infinity): the sizes by a table in two registers, whose bytes a permutation picks by three bits of each
// code, times the scale, with the sign.
__device__ __forceinline__ void fp4_values8(uint32_t codes, uint32_t scale_byte, uint32_t (&out)[4]) {
  const uint32_t unit = scale_byte == 0u ? 0x0040u : scale_byte == 255u ? 0x7fc0u : scale_byte << 7;  // bits of 2^(b - 127)
  const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&(const uint32_t&)(unit * 0x10001u));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c = codes >> (16 * h), pick = c & 0x7777u;
    // bfloat16 0, .5, 1, 1.5, 2, 3, 4, 6: high bytes 00 3f 3f 3f 40 40 40 40, low bytes 00 00 80 c0 00 40 80 c0
    const uint32_t high = __byte_perm(0x3f3f3f00u, 0x40404040u, pick), low = __byte_perm(0xc0800000u, 0xc0804000u, pick);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t v = __byte_perm(low, high, q == 0 ? 0x5140u : 0x7362u);
      const __nv_bfloat162 p = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), x);
      const uint32_t s = c >> (8 * q);
      out[2 * h + q] = *reinterpret_cast<const uint32_t*>(&p) | ((s & 0x8u) << 12) | ((s & 0x80u) << 24);
    }
  }
}
// Stores them at values col .. col + 7 of a row of K: by words, where the row begins between two of them of this lane's values and
// the last of the lane before.  The whole warp takes part.
__device__ __forceinline__ void fp4_store_values(__nv_bfloat16* row, int col, int K, const uint32_t (&w)[4]) {
  uint16_t* const to = reinterpret_cast<uint16_t*>(row + col);
  const bool between = ((uintptr_t)to & 3) != 0;  // uniform over the warp
  if (!between) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (col + 2 * j + 1 < K) reinterpret_cast<uint32_t*>(to)[j] = w[j];
      else if (col + 2 * j < K) to[2 * j] = (uint16_t)w[j];
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  uint32_t before = __shfl_up_sync(0xffffffffu, w[3], 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // values 2 j - 1 and 2 j of the lane
    const bool alone = j == 0 && lane == 0;
    if (col + 2 * j < K) {
      if (alone) to[0] = (uint16_t)w[0];
      else *reinterpret_cast<uint32_t*>(to + 2 * j - 1) = __funnelshift_r(before, w[j], 16);
    } else if (j > 0 && col + 2 * j - 1 < K) {
      to[2 * j - 1] = (uint16_t)(before >> 16);
    }
    before = w[j];
  }
  if ((lane == 31 || col + 8 >= K) && col + 7 < K) to[7] = (uint16_t)(w[3] >> 16);
}
__device__ __forceinline__ void fp4_store_values(float* row, int col, int K, const uint32_t (&w)[4]) {
  const bool whole = col + 8 <= K && ((uintptr_t)(row + col) & 15) == 0;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const float v[4] = {__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u), __uint_as_float(w[j + 1] << 16),
                        __uint_as_float(w[j + 1] & 0xffff0000u)};
    if (whole) {
      *reinterpret_cast<float4*>(row + col + 2 * j) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + 2 * j + i < K) row[col + 2 * j + i] = v[i];
    }
  }
}

// The codes of a lane's eight values, four neighbouring lanes holding a block, and the block's scale.
__device__ __forceinline__ uint32_t fp4_round_words(const uint32_t (&w)[8], uint32_t* scale_byte) {  // float32
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  return fp4_round8(v, scale_byte);
}
__device__ __forceinline__ uint32_t fp4_round_words(const uint32_t (&w)[4], uint32_t* scale_byte) {  // bfloat16, two to a word
  uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
  top = max(top & 0xffffu, top >> 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t b = fp4_scale_byte(top << 16);
  const float inv = fp4_inverse_scale(b);
  float s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[2 * i] = __uint_as_float(w[i] << 16) * inv;
    s[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * inv;
  }
  *scale_byte = b;
  return b == 255u ? 0u : fp4_pack8(s);
}

// A warp rounds 1,024 neighbouring values of a row, eight to a lane four times over, its loads all under way before the first is
// worked on; a block's eight warps take eight neighbouring rows.  FULL: all 1,024 are the row's, and nothing is off a 16-byte
// boundary, so nothing is asked for on the way (24,576 x 4,096 bfloat16 with values: 78 us, 5.8 TB/s; with the questions the loads
// went out one by one and it took 107; without values 50 us, 5.1 TB/s, and float32 70, 6.5).
constexpr int FP4_PIECE = 1024;
template <typename T, typename V, bool VEC, bool FULL>
__device__ __forceinline__ void fp4_quantise_piece(const T* row, const T* lo, uint8_t* codes, uint8_t* scales, V* values,
                                                   int r, int col0, int K) {
  const int lane = threadIdx.x & 31;
  uint32_t w[4][2 * sizeof(T)];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (FULL) {
      const uint4* at = reinterpret_cast<const uint4*>(row + col0 + i * 256);
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q) {
        const uint4 x = at[q];
        w[i][4 * q] = x.x; w[i][4 * q + 1] = x.y; w[i][4 * q + 2] = x.z; w[i][4 * q + 3] = x.w;
      }
    } else {
      fp4_load_words<T, VEC>(row, col0 + i * 256, K, lo, w[i]);
    }
  }
  const int pitch = fp4_pitch(K), across = fp4_tiles(K);
  uint8_t* const to = codes + (size_t)r * pitch;
  uint8_t* const scale_to = scales + fp4_scale_word(r, 0, across);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = col0 + i * 256;
    if (!FULL && col - lane * 8 >= across * FP4_TILE) break;  // uniform over the warp
    uint32_t byte;
    const uint32_t c = fp4_round_words(w[i], &byte);
    if (FULL || col < pitch * 2) *reinterpret_cast<uint32_t*>(to + col / 2) = c;
    const uint32_t word = fp4_scale_word_of_16(byte);
    if ((lane & 15) == 0 && (FULL || col / FP4_TILE < across))
      *reinterpret_cast<uint32_t*>(scale_to + col / FP4_TILE * FP4_TILE_BYTES) = word;
    if (values) {
      uint32_t v[4];
      fp4_values8(c, byte, v);
      if (FULL && sizeof(V) == 2)
        __stcs(reinterpret_cast<uint4*>(values + (size_t)r * K + col), make_uint4(v[0], v[1], v[2], v[3]));
      else
        fp4_store_values(values + (size_t)r * K, col, K, v);
    }
  }
}
template <typename T, bool VEC, typename V>
__global__ void __launch_bounds__(256, 4)
fp4_quantise_kernel(const T* __restrict__ x, long long x_pitch, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    V* __restrict__ values, int full, int R, int K) {
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), col0 = blockIdx.y * FP4_PIECE + (threadIdx.x & 31) * 8;
  if (r >= R) return;
  const T* row = x + r * x_pitch;
  if (VEC && full && (int)(blockIdx.y + 1) * FP4_PIECE <= K)  // uniform over the block
    fp4_quantise_piece<T, V, VEC, VEC>(row, x, codes, scales, values, r, col0, K);
  else
    fp4_quantise_piece<T, V, VEC, false>(row, x, codes, scales, values, r, col0, K);
}

template <typename T, typename V>
static int fp4_quantise_launch(const void* x, long long x_pitch, uint8_t* codes, uint8_t* scales, void* values, int R, int K,
                               cudaStream_t stream) {
  const dim3 grid((R - 1) / 8 + 1, (K - 1) / FP4_PIECE + 1);
  const bool vec = (uintptr_t)x % 16 == 0 && x_pitch * sizeof(T) % 16 == 0;
  const int full = (uintptr_t)values % 16 == 0 && (!values || (size_t)K * sizeof(V) % 16 == 0);
  if (vec)
    q3::launch(fp4_quantise_kernel<T, true, V>, grid, dim3(256), 0, stream, (const T*)x, x_pitch, codes, scales, (V*)values, full, R, K);
  else
    q3::launch(fp4_quantise_kernel<T, false, V>, grid, dim3(256), 0, stream, (const T*)x, x_pitch, codes, scales, (V*)values, full, R, K);
  return launch_status();
}

// ---------------------------------------------------------------- behind an RMSNorm
// One block per row: s = stream + delta goes to stream_out, s / sqrt(mean(s^2) + eps) * w is rounded.  A thread keeps its
// eight values of every `8 blockDim` of the row in registers between the sum and the rounding.  stream_out may be stream_in.
// What bounds it is memory, with the sum of each block in between (2,048 x 4,096, bfloat16 delta: 18 us for 88 MB, 4.9 TB/s, four
// blocks to an SM hiding each other's sums; blocks that go from row to row and ask for the next one ahead of the sum took 23, the
// registers for it leaving fewer of them), and for few rows the latency of its chain (1 x 4,096: 3.3 to 4 us between two launches).
// The weight is read behind the wait like the rest: ahead of it gained nothing that could be measured over the three launches
// of a feed-forward.
constexpr int FP4_NORM_MAX = 1024 * 8 * 4;
template <typename T, int G>
__global__ void __launch_bounds__(1024)
fp4_add_rmsnorm_kernel(const float* stream_in, const T* __restrict__ delta, const float* __restrict__ w, float* stream_out,
                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int H, float eps,
                       bool vec) {
  __shared__ float scratch[32];
  float wv[G][8];
  auto load_weight = [&](int g) {
    const int col = (g * blockDim.x + threadIdx.x) * 8;
    if (vec) fp4_load_row8<float, true>(w, col, H, wv[g]);
    else fp4_load_row8<float, false>(w, col, H, wv[g]);
  };
  pdl_wait();
  pdl_launch_dependents();
  constexpr bool AHEAD = G <= 2;  // where the registers suffice
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (AHEAD) load_weight(g);
  const size_t r = blockIdx.x;
  const float* in = stream_in + r * H;
  float v[G][8];
  float ss = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int col = (g * blockDim.x + threadIdx.x) * 8;
    if (vec) fp4_load_row8<float, true>(in, col, H, v[g]);
    else fp4_load_row8<float, false>(in, col, H, v[g]);
    if (delta) {
      float d[8];
      if (vec) fp4_load_row8<T, true>(delta + r * H, col, H, d);
      else fp4_load_row8<T, false>(delta + r * H, col, H, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g][i] += d[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[g][i], v[g][i], ss);
    if (vec && col + 8 <= H) {
      reinterpret_cast<float4*>(stream_out + r * H + col)[0] = make_float4(v[g][0], v[g][1], v[g][2], v[g][3]);
      reinterpret_cast<float4*>(stream_out + r * H + col)[1] = make_float4(v[g][4], v[g][5], v[g][6], v[g][7]);
    } else {
      for (int i = 0; i < 8; ++i)
        if (col + i < H) stream_out[r * H + col + i] = v[g][i];
    }
  }
  ss = block_sum(ss, scratch);
  const float rs = 1.0f / sqrtf(ss / (float)H + eps);
  const int pitch = fp4_pitch(H), across = fp4_tiles(H);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int col = (g * blockDim.x + threadIdx.x) * 8;
    if (!AHEAD) load_weight(g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[g][i] = v[g][i] * rs * wv[g][i];
    uint32_t byte;
    const uint32_t c = fp4_round8(v[g], &byte);
    if (col < pitch * 2) *reinterpret_cast<uint32_t*>(codes + r * pitch + col / 2) = c;
    const uint32_t word = fp4_scale_word_of_16(byte);
    if ((threadIdx.x & 15) == 0 && col / FP4_TILE < across)
      *reinterpret_cast<uint32_t*>(scales + fp4_scale_word((int)r, col / FP4_TILE, across)) = word;
  }
}

template <typename T>
static int fp4_add_rmsnorm_launch(const float* in, const void* delta, const float* w, float* out, uint8_t* codes, uint8_t* scales,
                                  int R, int H, float eps, cudaStream_t stream) {
  const bool vec = H % 8 == 0 && ((uintptr_t)in | (uintptr_t)delta | (uintptr_t)w | (uintptr_t)out) % 16 == 0;
  const int g = (H + 8 * 1024 - 1) / (8 * 1024);
  const int threads = ((H + 8 * g - 1) / (8 * g) + 31) / 32 * 32;
#define Q3_NORM(G)                                                                                                        \
  q3::launch(fp4_add_rmsnorm_kernel<T, G>, dim3(R), dim3(threads), 0, stream, in, (const T*)delta, w, out, codes, scales, H, \
             eps, vec)
  if (g == 1) Q3_NORM(1);
  else if (g == 2) Q3_NORM(2);
  else Q3_NORM(4);
#undef Q3_NORM
  note_stream_written();
  return launch_status();
}

}  // namespace q3

// Rows of x (R rows of K values, `x_pitch` values apart) to codes and scales; `values` (values_dtype, [R, K], or null): what
// the rows then stand for.
extern "C" int q3_fp4_quantise(const void* x, int dtype, long long x_pitch, void* codes, void* scales, void* values,
                               int values_dtype, int R, int K, cudaStream_t stream) {
  if (R <= 0) return 0;
  if (K <= 0 || K > 65535 * q3::FP4_PIECE) return Q3_ERR_SIZE;
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 16) return Q3_ERR_ALIGN;
  if ((dtype != Q3_F32 && dtype != Q3_BF16) || (values_dtype != Q3_F32 && values_dtype != Q3_BF16)) return Q3_ERR_DTYPE;
  using bf16 = __nv_bfloat16;
  uint8_t *c = (uint8_t*)codes, *s = (uint8_t*)scales;
  if (dtype == Q3_F32) {
    if (values_dtype == Q3_F32) return q3::fp4_quantise_launch<float, float>(x, x_pitch, c, s, values, R, K, stream);
    return q3::fp4_quantise_launch<float, bf16>(x, x_pitch, c, s, values, R, K, stream);
  }
  if (values_dtype == Q3_F32) return q3::fp4_quantise_launch<bf16, float>(x, x_pitch, c, s, values, R, K, stream);
  return q3::fp4_quantise_launch<bf16, bf16>(x, x_pitch, c, s, values, R, K, stream);
}

// stream_out = stream + delta (float32; delta may be null, stream_out may be the stream), and its RMSNorm times w as rows.
extern "C" int q3_fp4_add_rmsnorm(const float* in, const void* delta, int dtype, const float* w, float* out, void* codes,
                                  void* scales, int R, int H, float eps, cudaStream_t stream) {
  if (R <= 0) return 0;
  if (H <= 0 || H > q3::FP4_NORM_MAX) return Q3_ERR_SIZE;
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 16) return Q3_ERR_ALIGN;
  if (dtype == Q3_F32)
    return q3::fp4_add_rmsnorm_launch<float>(in, delta, w, out, (uint8_t*)codes, (uint8_t*)scales, R, H, eps, stream);
  if (dtype != Q3_BF16) return Q3_ERR_DTYPE;
  return q3::fp4_add_rmsnorm_launch<__nv_bfloat16>(in, delta, w, out, (uint8_t*)codes, (uint8_t*)scales, R, H, eps, stream);
}
