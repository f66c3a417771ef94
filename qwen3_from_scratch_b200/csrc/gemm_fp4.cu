// Products of matrices held in microscaled 4-bit floating point (fp4.cuh) on the fifth-generation tensor cores:
// y[T, N] = x[T, K] * w[N, K]^T, tcgen05.mma kind::mxf4 with a scale per 32 values of k on both sides, float32 accumulators
// in tensor memory.
//
// A block computes a tile of 128 rows of x by BN rows of w.  Three roles:
//   warp 0 (one thread)  brings the codes of 256 values of k at a time (128 bytes of each row) into shared memory by TMA
//                        with the 128-byte swizzle, and their scales by bulk copies of whole 512-byte tiles;
//   warp 1 (one thread)  copies each tile of scales into tensor memory (tcgen05.cp, which the instructions behind it in
//                        the same thread wait for) and issues four instructions of k = 64 per stage;
//   warps 2..5           read the accumulator, a thread per row of x, and store bfloat16 or float32; or, for a w whose rows
//                        alternate gate/up in blocks of eight, apply the gate and round each 32 results to the same format.
// The instruction reads a row's scales of k = 64 from two of the four bytes of a tensor-memory column; which two is in the
// instruction descriptor.
#include "fp4.cuh"
#include "tc_common.cuh"

namespace q3 {

constexpr int F4_BM = 128;
constexpr int F4_THREADS = 192;

struct F4Args {
  const uint8_t* x_scales;
  const uint8_t* w_scales;
  void* out;           // EPI 0, 1
  long long ldc;
  uint8_t* out_codes;  // EPI 2
  uint8_t* out_scales;
  int T, N, K, act;
};

// A stage holds 256 values of k: 128 bytes of codes from each row and two tiles of scales.

// Instruction descriptor of kind::mxf4: 4-bit operands, both K-major, power-of-two scales, M = 128, N = n; `id`: which bytes
// of the scales' columns (0: the first two, 2: the last two).
__host__ __device__ constexpr uint32_t f4_idesc(int n, int id, int m = 128) {
  return ((uint32_t)id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) |
         ((uint32_t)id << 29);
}
__device__ __forceinline__ void f4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
      : "memory");
}
// A tile of scales (32 x 16 bytes in shared memory, without swizzle) into four columns of tensor memory.
__device__ __forceinline__ uint64_t f4_scale_desc(const void* tile) {
  return (uint64_t)((s_addr(tile) & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
__device__ __forceinline__ void f4_copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void f4_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(s_addr(dst)), "l"(src), "r"(bytes), "r"(s_addr(bar))
               : "memory");
}

template <int BN>
struct F4Shape {
  static constexpr int A_BYTES = F4_BM * 128, B_BYTES = BN * 128;
  static constexpr int SA_BYTES = 2 * FP4_TILE_BYTES, SB_BYTES = (BN / FP4_TILE) * 2 * FP4_TILE_BYTES;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int BAR_BYTES = 256;
  static constexpr size_t SMEM_BYTES = (size_t)STAGES * STAGE_BYTES + BAR_BYTES;
  static constexpr uint32_t SCALE_COL = BN;  // behind the accumulator
  static constexpr uint32_t TMEM_COLS = 2 * BN;
};
static_assert(F4Shape<128>::STAGE_BYTES % 1024 == 0, "stages keep the swizzle's alignment");

template <int BN, int EPI>
__global__ void __launch_bounds__(F4_THREADS)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ F4Args p, int* status) {
  using S = F4Shape<BN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = smem_raw;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_raw + (size_t)S::STAGES * S::STAGE_BYTES);
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_full + 1);
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int across = fp4_tiles(p.K);          // tiles of scales along k
  const int k_stages = (across + 1) / 2;
  const int w_tiles = fp4_tiles(p.N);
  const int m0 = blockIdx.y * F4_BM, n0 = blockIdx.x * BN;
  const bool aligned = (s_addr(smem_raw) & 1023u) == 0;
  if (!aligned && threadIdx.x == 0) atomicOr(status, Q3_STATUS_TIMEOUT);

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_w);
    abort_flag = 0;
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_holder)),
                 "r"(S::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0 && aligned) {
      int it = 0;
      for (; it < k_stages; ++it) {
        const int s = it % S::STAGES, use = it / S::STAGES;
        if (use > 0 && !mbar_wait(&empty[s], (use & 1) ^ 1, &abort_flag)) {
          abort_flag = 1;
          atomicOr(status, Q3_STATUS_TIMEOUT);
          break;
        }
        const uint32_t sf = (uint32_t)min(2, across - 2 * it) * FP4_TILE_BYTES;  // the last stage may have one tile
        int w_here = 0;
        for (int j = 0; j < BN / FP4_TILE; ++j) w_here += n0 / FP4_TILE + j < w_tiles;
        unsigned char* a = tiles + (size_t)s * S::STAGE_BYTES;
        unsigned char *b = a + S::A_BYTES, *sa = b + S::B_BYTES, *sb = sa + S::SA_BYTES;
        mbar_expect_tx(&full[s], S::A_BYTES + S::B_BYTES + sf * (1 + w_here));
        tma_load_2d(b, &map_w, &full[s], it * 64, n0);
        for (int j = 0; j < w_here; ++j)
          f4_bulk_load(sb + j * S::SA_BYTES, p.w_scales + ((size_t)(n0 / FP4_TILE + j) * across + 2 * it) * FP4_TILE_BYTES, sf, &full[s]);
        f4_bulk_load(sa, p.x_scales + ((size_t)blockIdx.y * across + 2 * it) * FP4_TILE_BYTES, sf, &full[s]);
        if (it == tc_drop_copy) continue;  // tests of the give-up path only (see tc_common.cuh)
        tma_load_2d(a, &map_x, &full[s], it * 64, m0);
      }
      finish_copies(full, it, S::STAGES, tc_drop_copy, status);
    }
  } else if (warp == 1) {
    if (lane == 0 && aligned) {
      bool ok = true;
      for (int it = 0; it < k_stages; ++it) {
        const int s = it % S::STAGES, use = it / S::STAGES;
        if (!mbar_wait(&full[s], use & 1, &abort_flag)) {
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const unsigned char* a = tiles + (size_t)s * S::STAGE_BYTES;
        const unsigned char *b = a + S::A_BYTES, *sa = b + S::B_BYTES, *sb = sa + S::SA_BYTES;
        const uint64_t a_desc = umma_desc_sw128(a), b_desc = umma_desc_sw128(b);
        const int halves = min(2, across - 2 * it);
        for (int h = 0; h < halves; ++h) {
          const uint32_t ta = tmem + S::SCALE_COL + h * 4, tb = tmem + S::SCALE_COL + 8 + h * (BN / 32);
          f4_copy_scales(ta, f4_scale_desc(sa + h * FP4_TILE_BYTES));
          for (int j = 0; j < BN / FP4_TILE; ++j)
            f4_copy_scales(tb + 4 * j, f4_scale_desc(sb + j * S::SA_BYTES + h * FP4_TILE_BYTES));
          f4_mma(tmem, a_desc + 4 * h, b_desc + 4 * h, f4_idesc(BN, 0), ta, tb, (it | h) != 0);
          f4_mma(tmem, a_desc + 4 * h + 2, b_desc + 4 * h + 2, f4_idesc(BN, 2), ta, tb, 1);
        }
        umma_commit(&empty[s]);
      }
      if (ok) {
        umma_commit(acc_full);
      } else {
        abort_flag = 1;
        atomicOr(status, Q3_STATUS_TIMEOUT);
      }
    }
  } else if (aligned) {
    const int quarter = warp & 3, row = m0 + quarter * 32 + lane;
    const bool ready = mbar_wait(acc_full, 0, &abort_flag);
    if (!__all_sync(0xffffffffu, ready)) {
      if (lane == 0) {
        abort_flag = 1;
        atomicOr(status, Q3_STATUS_TIMEOUT);
      }
    } else {
      tcgen05_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
      if (EPI == 2) {
        const int inner = p.N / 2, blocks = (inner + FP4_BLOCK - 1) / FP4_BLOCK, out_across = fp4_tiles(inner);
        const int first = n0 / 64;
        // the last tile also clears the scales behind the last block, up to the end of their tile
        const int end = n0 + BN >= p.N ? out_across * 4 : first + BN / 64;
#pragma unroll 1
        for (int j = first; j < end; ++j) {
          uint32_t byte = 0, w[4] = {0, 0, 0, 0};
          if (j < blocks) {
            uint32_t v[2][32];
            tmem_ld_32(acc + (uint32_t)(j - first) * 64, v[0]);
            tmem_ld_32(acc + (uint32_t)(j - first) * 64 + 32, v[1]);
            tmem_wait_ld();
            float a[32];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int g = i / 8 * 16 + i % 8;
              a[i] = gated_f(__uint_as_float(v[g / 32][g % 32]), __uint_as_float(v[(g + 8) / 32][(g + 8) % 32]), p.act, 0.f);
              if (j * 32 + i >= inner) a[i] = 0.f;
              top = max(top, __float_as_uint(a[i]) & 0x7fffffffu);
            }
            byte = fp4_scale_byte(top);
            const float inv = fp4_inverse_scale(byte);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float s8[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) s8[i] = a[8 * q + i] * inv;
              w[q] = byte == 255u ? 0u : fp4_pack8(s8);
            }
          }
          if (row < p.T) {
            if (j < blocks) *reinterpret_cast<uint4*>(p.out_codes + (size_t)row * fp4_pitch(inner) + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            p.out_scales[fp4_scale_word(row, j / 4, out_across) + j % 4] = (uint8_t)byte;
          }
        }
      } else {
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += 32) {
          if (n0 + c0 >= p.N) break;
          uint32_t v[32];
          tmem_ld_32(acc + (uint32_t)c0, v);
          tmem_wait_ld();
          if (row < p.T) {
            using OutT = typename std::conditional<EPI == 0, __nv_bfloat16, float>::type;
            OutT* dst = (OutT*)p.out + (size_t)row * p.ldc + n0 + c0;
            if (n0 + c0 + 32 <= p.N && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
              for (int j = 0; j < 32 * (int)sizeof(OutT) / 16; ++j) {
                if (EPI == 0)
                  reinterpret_cast<uint4*>(dst)[j] = make_uint4(pack2(v[8 * j], v[8 * j + 1]), pack2(v[8 * j + 2], v[8 * j + 3]),
                                                               pack2(v[8 * j + 4], v[8 * j + 5]), pack2(v[8 * j + 6], v[8 * j + 7]));
                else
                  reinterpret_cast<uint4*>(dst)[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (n0 + c0 + j < p.N) dst[j] = from_float<OutT>(__uint_as_float(v[j]));
            }
          }
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
  }
}

template <int EPI>
static int gemm_fp4_launch(const void* x_codes, const void* w_codes, const F4Args& p, int* status, cudaStream_t stream) {
  constexpr int BN = 128;
  using S = F4Shape<BN>;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(gemm_fp4_kernel<BN, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const long long n_tiles = (p.N + BN - 1) / BN, m_tiles = (p.T + F4_BM - 1) / F4_BM;
  if (n_tiles > 0x7fffffffLL || m_tiles > 65535) return Q3_ERR_SIZE;
  // the maps take two bytes of codes as one bfloat16: only bytes move
  CUtensorMap map_x, map_w;
  const uint64_t cols = fp4_pitch(p.K) / 2;
  int code = make_map(&map_x, x_codes, (uint64_t)p.T, cols, F4_BM);
  if (code) return code;
  code = make_map(&map_w, w_codes, (uint64_t)p.N, cols, BN);
  if (code) return code;
  q3::launch(gemm_fp4_kernel<BN, EPI>, dim3((unsigned)n_tiles, (unsigned)m_tiles), dim3(F4_THREADS), S::SMEM_BYTES, stream, map_x,
             map_w, p, status);
  return launch_status();
}

static bool f4_sizes_ok(int T, int N, int K) { return N > 0 && K > 0 && T > 0 && K <= (1 << 30) && N <= (1 << 30); }
static bool f4_aligned(const void* a, const void* b, const void* c, const void* d) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0;
}

}  // namespace q3

// out[T, N] (row pitch ldc) = x w^T of rows held in four bits; out_f32: float32 results, else bfloat16.
extern "C" int q3_fp4_product(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out, int T,
                              int N, int K, long long ldc, int out_f32, int* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (!q3::f4_sizes_ok(T, N, K) || ldc < N) return Q3_ERR_SIZE;
  if (!q3::f4_aligned(x_codes, x_scales, w_codes, w_scales)) return Q3_ERR_ALIGN;
  q3::F4Args p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, out, ldc, nullptr, nullptr, T, N, K, 0};
  if (out_f32) return q3::gemm_fp4_launch<1>(x_codes, w_codes, p, status, stream);
  return q3::gemm_fp4_launch<0>(x_codes, w_codes, p, status, stream);
}

// act(gate) * up as rows held in four bits: w's N = 2 I rows alternate gate/up in blocks of eight, the output has T rows of I.
extern "C" int q3_fp4_gated_product(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales,
                                    void* out_codes, void* out_scales, int T, int N, int K, int act, int* status,
                                    cudaStream_t stream) {
  if (T <= 0) return 0;
  if (!q3::f4_sizes_ok(T, N, K) || N % 16 || (act != Q3_ACT_SILU && act != Q3_ACT_RELU && act != Q3_ACT_GELU_TANH)) return Q3_ERR_SIZE;
  if (!q3::f4_aligned(x_codes, x_scales, w_codes, w_scales) || !q3::f4_aligned(out_codes, out_scales, nullptr, nullptr)) return Q3_ERR_ALIGN;
  q3::F4Args p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, nullptr, 0, (uint8_t*)out_codes, (uint8_t*)out_scales, T, N, K, act};
  return q3::gemm_fp4_launch<2>(x_codes, w_codes, p, status, stream);
}

extern "C" int q3_fp4_add_rmsnorm(const float* in, const void* delta, int dtype, const float* w, float* out, void* codes,
                                  void* scales, int R, int H, float eps, cudaStream_t stream);

// A gated feed-forward behind its norm, in three launches: the norm's rows into h, the gated product into a, y = a w_down^T.
extern "C" int q3_fp4_feed_forward(const float* stream_in, const void* delta, const float* norm, float* stream_out, float eps,
                                   const void* gu_codes, const void* gu_scales, const void* down_codes, const void* down_scales,
                                   void* h_codes, void* h_scales, void* a_codes, void* a_scales, void* y, int dtype, int T,
                                   int H, int I, int act, int* status, cudaStream_t stream) {
  int code = q3_fp4_add_rmsnorm(stream_in, delta, dtype, norm, stream_out, h_codes, h_scales, T, H, eps, stream);
  if (code) return code;
  code = q3_fp4_gated_product(h_codes, h_scales, gu_codes, gu_scales, a_codes, a_scales, T, 2 * I, H, act, status, stream);
  if (code) return code;
  return q3_fp4_product(a_codes, a_scales, down_codes, down_scales, y, T, H, I, H, dtype == Q3_F32, status, stream);
}

// For the tests of the give-up path: see set_wait_test in tc_common.cuh.
extern "C" int q3_gemm_fp4_wait_test(unsigned limit, int drop) { return q3::set_wait_test(limit, drop); }
