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

template <typename V>
__device__ __forceinline__ void fp4_store_values(V* row, int col, int K, uint32_t codes, uint32_t scale_byte, bool vec) {
  const float x = fp4_scale(scale_byte);
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = fp4_pair(codes >> (8 * i));
    v[2 * i] = p.x * x;
    v[2 * i + 1] = p.y * x;
  }
  if (vec && col + 8 <= K) {
    if (sizeof(V) == 2) {
      uint4 o;
      uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
      *reinterpret_cast<uint4*>(row + col) = o;
    } else {
      reinterpret_cast<float4*>(row + col)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(row + col)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < K) row[col + i] = from_float<V>(v[i]);
  }
}

// A warp rounds 256 neighbouring values of a row at a time, eight to a lane.
template <typename T, bool VEC, typename V>
__global__ void __launch_bounds__(256)
fp4_quantise_kernel(const T* __restrict__ x, long long x_pitch, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    V* __restrict__ values, bool values_vec, int K, int pieces, long long items) {
  pdl_wait();
  pdl_launch_dependents();
  const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item >= items) return;
  const int lane = threadIdx.x & 31;
  const long long r = item / pieces;
  const int col = (int)(item % pieces) * 256 + lane * 8;
  float v[8];
  fp4_load_row8<T, VEC>(x + r * x_pitch, col, K, v);
  uint32_t byte;
  const uint32_t c = fp4_round8(v, &byte);
  const int pitch = fp4_pitch(K), across = fp4_tiles(K);
  if (col < pitch * 2) *reinterpret_cast<uint32_t*>(codes + r * pitch + col / 2) = c;
  const uint32_t word = fp4_scale_word_of_16(byte);
  if ((lane & 15) == 0 && col / FP4_TILE < across)
    *reinterpret_cast<uint32_t*>(scales + fp4_scale_word((int)r, col / FP4_TILE, across)) = word;
  if (values) fp4_store_values(values + r * K, col, K, c, byte, values_vec);
}

template <typename T, typename V>
static int fp4_quantise_launch(const void* x, long long x_pitch, uint8_t* codes, uint8_t* scales, void* values, int R, int K,
                               cudaStream_t stream) {
  const int pieces = (K + 255) / 256;
  const long long items = (long long)R * pieces;
  const long long blocks = (items + 7) / 8;
  if (blocks > 0x7fffffffLL) return Q3_ERR_SIZE;
  const bool vec = (uintptr_t)x % 16 == 0 && x_pitch * sizeof(T) % 16 == 0;
  const bool values_vec = (uintptr_t)values % 16 == 0 && (long long)K * sizeof(V) % 16 == 0;
  if (vec)
    q3::launch(fp4_quantise_kernel<T, true, V>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x, x_pitch, codes, scales,
               (V*)values, values_vec, K, pieces, items);
  else
    q3::launch(fp4_quantise_kernel<T, false, V>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x, x_pitch, codes, scales,
               (V*)values, values_vec, K, pieces, items);
  note_stream_written();  // a product after it may take these rows as its w, which it reads ahead of its wait
  return launch_status();
}

// One block per row: s = stream + delta goes to stream_out, s / sqrt(mean(s^2) + eps) * w is rounded.  A thread keeps its
// eight values of every `8 blockDim` of the row in registers between the sum and the rounding.  stream_out may be stream_in.
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
  constexpr bool AHEAD = G <= 2;  // no kernel writes the weight: it is read ahead of the wait where the registers suffice
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (AHEAD) load_weight(g);
  pdl_wait();
  pdl_launch_dependents();
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
  note_stream_written();  // the stream, and rows that a product might take as its w
  return launch_status();
}

}  // namespace q3

// Rows of x (R rows of K values, `x_pitch` values apart) to codes and scales; `values` (values_dtype, [R, K], or null): what
// the rows then stand for.
extern "C" int q3_fp4_quantise(const void* x, int dtype, long long x_pitch, void* codes, void* scales, void* values,
                               int values_dtype, int R, int K, cudaStream_t stream) {
  if (R <= 0) return 0;
  if (K <= 0 || K > (1 << 30)) return Q3_ERR_SIZE;
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
