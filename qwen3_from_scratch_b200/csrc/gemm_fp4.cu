// Products of matrices held in microscaled 4-bit floating point (fp4.cuh) on the fifth-generation tensor cores:
// y[T, N] = x[T, K] * w[N, K]^T, tcgen05.mma kind::mxf4 with a scale per 32 values of k on both sides, float32 accumulators
// in tensor memory.  The results are stored as bfloat16 or float32; or, for a w whose rows alternate gate/up in blocks of eight,
// the gate is applied and each 32 results are rounded to the same format, so that the [T, 2 I] product never goes to memory.
//
// Both kernels have the same three roles:
//   warp 0           brings the codes of 256 values of k at a time (128 bytes of each row) into shared memory by TMA with the
//                    128-byte swizzle, and their scales in whole 512-byte tiles;
//   warp 1           copies each tile of scales into tensor memory (tcgen05.cp, in order with the instructions of the same
//                    thread before and behind it) and issues instructions of k = 64, four for a stage's columns;
//   the other warps  the epilogue (of the few-tokens kernel all, when the two are done).
// An instruction reads a row's scales of k = 64 from two of the four bytes of a tensor-memory column; which two is in its
// descriptor.  Every wait on an mbarrier is bounded, as in gemm_tc.cu.
//
// gemm_fp4_few_kernel: small tiles; where they are fewer than the SMs, several blocks per tile share out the range of k.
// gemm_fp4_pair_kernel: tiles of 256 rows by pairs of CTAs, for many tokens.
#include "fp4.cuh"
#include "tc_common.cuh"

namespace q3 {

constexpr int F4_BM = 128;

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

// One lane of a converged warp, the same one every time.  The loader and the issuing role run their loops with the whole warp
// and pick the lane only around the instructions: what those are given (descriptors, addresses) is then the same in all lanes
// as the compiler sees it and stays in the uniform registers that the instructions want.  With the whole loop in one lane it is
// moved there anew for every instruction: a stage of two 128-column halves took 985 clocks to issue instead of 522.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// A wait of a whole warp: true if every lane saw the phase complete.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
__device__ __forceinline__ bool warp_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, abort_flag));
}

// a[i] = act(g[i]) * u[i].  SiLU and GELU's tanh form are g sigmoid(z) = g / (1 + 2^(-z log2 e)), as (1 + tanh(y)) / 2 = sigmoid(2 y).
// The fast power and reciprocal are off by a few times 2^-23, which moves a result across a boundary between two codes once in
// some 10^5 values; the exact ones, one value after another, took 1.2 us of a call's last 1.9 where a lane has four values to do.
// A loop for each gate, with nothing in it that the others need: where k is short, a gate is what bounds the call.
__device__ __forceinline__ float f4_over_one_and_power(float g, float e) {  // g / (1 + 2^e)
  float t, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + t));
  return g * r;
}
template <int N>
__device__ __forceinline__ void f4_gate(const float (&g)[N], const float (&u)[N], int act, float (&a)[N]) {
  constexpr float LOG2E = 1.4426950408889634f, Z = 1.5957691216057308f;  // 2 sqrt(2 / pi)
  if (act == Q3_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = u[i] * f4_over_one_and_power(g[i], -LOG2E * g[i]);
  } else if (act == Q3_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = u[i] * f4_over_one_and_power(g[i], g[i] * fmaf(-LOG2E * Z * 0.044715f * g[i], g[i], -LOG2E * Z));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float m;  // a NaN stays one
      asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(m) : "f"(g[i]));
      a[i] = m * u[i];
    }
  }
}

// 64 float32 columns as bfloat16, two to a word.
__device__ __forceinline__ void f4_pack(const uint32_t (&v0)[32], const uint32_t (&v1)[32], uint32_t (&w)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = pack2(v0[2 * i], v0[2 * i + 1]);
    w[16 + i] = pack2(v1[2 * i], v1[2 * i + 1]);
  }
}
// Where a warp of the epilogue puts the results of its 32 rows, 128 bytes of each (32 float32 or 64 bfloat16 columns) at a time, a
// row to a lane, by way of 4 KB of shared memory: there the lanes change places, so that eight of them store the 128 bytes of a row
// side by side.  Storing from the accumulator's own order, 16 bytes of 32 different rows at a time, took as long as the main loop
// (2,048 x 24,576 x 4,096: 90 us with it, 64 without any stores).  16-byte piece c of row r lies at r * 128 + ((c ^ (r % 8)) * 16),
// off the banks of its neighbours both ways.
//
// Memory takes whole sectors of 32 bytes far better than parts of them (8,000 x 16,001 x 64, float32: 101 us with 16,000 columns,
// 258 with a piece's first and last values stored one by one).  So where rows are off a sector's boundary, what leaves is the 128
// bytes up to the last boundary: each lane holds back the last bytes of its row and puts them in front of the next ones.
template <int EPI>
struct F4RowStore {
  using OutT = typename std::conditional<EPI == 0, __nv_bfloat16, float>::type;
  unsigned char* stage;
  unsigned char* first;  // the warp's first row, first column
  size_t pitch;          // bytes from a row to the next
  int rows, bytes;       // rows, and bytes of each, that are results
  int at;                // bytes of each row that have come
  bool whole;            // no row is off a sector's boundary, all columns are results (uniform over the warp)
  uint32_t held[8];      // the last 32 bytes that came

  __device__ __forceinline__ F4RowStore(const F4Args& p, unsigned char* stage_, int row0, int col, int cols)
      : stage(stage_), first((unsigned char*)p.out + ((size_t)row0 * p.ldc + col) * sizeof(OutT)), pitch((size_t)p.ldc * sizeof(OutT)),
        rows(min(32, p.T - row0)), bytes(min(cols, p.N - col) * (int)sizeof(OutT)), at(0),
        whole(col + cols <= p.N && (((uintptr_t)p.out | (size_t)p.ldc * sizeof(OutT)) & 31) == 0), held{} {}

  // The next 128 bytes of each row.
  __device__ __forceinline__ void push(const uint32_t (&w)[32], int lane) {
    if (at >= bytes) return;  // uniform over the warp
    if (whole) {
      put(w, lane, 8);
      const int c = lane & 7;
      unsigned char* to = first + (lane >> 3) * pitch + at + c * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i, to += 4 * pitch) {
        const int r = 4 * i + (lane >> 3);
        if (r < rows) *reinterpret_cast<uint4*>(to) = piece(r, c);
      }
    } else {
      uint32_t x[40];
#pragma unroll
      for (int j = 0; j < 40; ++j) x[j] = j < 8 ? held[j] : w[j - 8];
#pragma unroll
      for (int j = 0; j < 8; ++j) held[j] = w[24 + j];
      shift(x, lane);
      uint32_t y[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) y[j] = x[8 + j];
      put(y, lane, 8);
      leave(lane, true);
    }
    __syncwarp();
    at += 128;
  }
  // What is still held back.
  __device__ __forceinline__ void end(int lane) {
    if (whole || at == 0) return;  // uniform over the warp
    uint32_t x[16], y[32];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = j < 8 ? held[j] : 0u;
    shift(x, lane);
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = j < 8 ? x[8 + j] : 0u;
    put(y, lane, 2);
    leave(lane, false);
    __syncwarp();
  }

 private:
  __device__ __forceinline__ uint4 piece(int r, int c) const {
    return *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
  }
  __device__ __forceinline__ void put(const uint32_t (&y)[32], int lane, int pieces) {
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < pieces)
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) =
            make_uint4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
    __syncwarp();
  }
  // x, from its ninth word on, moves up by as many bytes as the lane's row is behind a sector's boundary.
  template <int N>
  __device__ __forceinline__ void shift(uint32_t (&x)[N], int lane) const {
    const uint32_t m = (uint32_t)(uintptr_t)(first + lane * pitch) & 31u;
#pragma unroll
    for (int j = N - 1; j >= 1; --j) x[j] = m & 4 ? x[j - 1] : x[j];
#pragma unroll
    for (int j = N - 1; j >= 3; --j) x[j] = m & 8 ? x[j - 2] : x[j];
#pragma unroll
    for (int j = N - 1; j >= 7; --j) x[j] = m & 16 ? x[j - 4] : x[j];
    if (EPI == 0) {
#pragma unroll
      for (int j = N - 1; j >= 8; --j) x[j] = m & 2 ? __funnelshift_r(x[j - 1], x[j], 16) : x[j];
    }
  }
  // Of the 128 bytes behind the boundary (`all`; else of the first sector): what is whole by sixteen bytes to a lane, of the row's
  // first and last sector what is the row's, a word to a lane.  Four rows' reads go out together: one by one they took longer than
  // the stores.
  __device__ __forceinline__ void leave(int lane, bool all) const {
    const int c = lane & 7, len = all ? 128 : 32;
    if (all) {
      unsigned char* row = first + (lane >> 3) * pitch;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = piece(16 * h + 4 * i + (lane >> 3), c);
#pragma unroll
        for (int i = 0; i < 4; ++i, row += 4 * pitch) {
          const int m = (int)((uintptr_t)row & 31), lo = m - at, hi = bytes + m - at;
          const bool ok = 16 * h + 4 * i + (lane >> 3) < rows && 32 * (c >> 1) >= lo && 32 * (c >> 1) + 32 <= hi;
          if (ok) *reinterpret_cast<uint4*>(row - m + at + c * 16) = q[i];
        }
      }
    }
    if (at == 0) part(lane, len, true);
    if (at + len > bytes) part(lane, len, false);
  }
  // The row's first sector (`low`), if a part of it is another's, or its last one, if it is another one and ends among these bytes.
  __device__ __forceinline__ void part(int lane, int len, bool low) const {
    const int c = lane & 7;
    unsigned char* row = first + (lane >> 3) * pitch;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t x[4];
      int from[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * h + 4 * i + (lane >> 3), m = (int)((uintptr_t)(row + i * 4 * pitch) & 31), hi = bytes + m - at;
        const bool ok = r < rows && (low ? m > 0 : hi > 0 && hi < len && (hi & 31) != 0 && (at > 0 || m == 0 || hi > 32));
        from[i] = ok ? (low ? 0 : hi & ~31) + c * 4 : -1;
        const int word = max(from[i], 0);
        x[i] = *reinterpret_cast<const uint32_t*>(stage + r * 128 + (((word >> 4) ^ (r & 7)) << 4) + (word & 15));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i, row += 4 * pitch) {
        const int m = (int)((uintptr_t)row & 31), lo = m - at, hi = bytes + m - at, w = from[i];
        unsigned char* const to = row - m + at + w;
        if (w >= 0 && lo <= w && hi >= w + 4) *reinterpret_cast<uint32_t*>(to) = x[i];
        if (EPI == 0) {
          if (w >= 0 && lo <= w && hi == w + 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)x[i];
          if (w >= 0 && lo == w + 2 && hi >= w + 4) *reinterpret_cast<uint16_t*>(to + 2) = (uint16_t)(x[i] >> 16);
        }
      }
    }
  }
};
// 64 columns, gate and up in blocks of eight: a block of 32 results, their codes and scale.
__device__ __forceinline__ void f4_gated_block(const uint32_t (&v0)[32], const uint32_t (&v1)[32], const F4Args& p, int row, int col) {
  const int inner = p.N / 2, blocks = (inner + FP4_BLOCK - 1) / FP4_BLOCK, out_across = fp4_tiles(inner), j = col / 64;
  float gate[32], up[32], a[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int c = i / 8 * 16 + i % 8;
    gate[i] = __uint_as_float(c < 32 ? v0[c % 32] : v1[c % 32]);
    up[i] = __uint_as_float(c < 32 ? v0[(c + 8) % 32] : v1[(c + 8) % 32]);
  }
  f4_gate<32>(gate, up, p.act, a);
  if (j * 32 + 32 > inner) {  // uniform over the warp
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (j * 32 + i >= inner) a[i] = 0.f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = fp4_top(top, a[i]);
  const uint32_t byte = fp4_scale_byte(top);
  const float inv = fp4_inverse_scale(byte);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float s8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s8[i] = a[8 * q + i] * inv;
    w[q] = byte == 255u ? 0u : fp4_pack8(s8);
  }
  *reinterpret_cast<uint4*>(p.out_codes + (size_t)row * fp4_pitch(inner) + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  uint8_t* word = p.out_scales + fp4_scale_word(row, j / 4, out_across);
  word[j % 4] = (uint8_t)byte;
  if (j + 1 == blocks)  // and the scales behind the last block, up to the end of their tile, are zero
    for (int i = j % 4 + 1; i < 4; ++i) word[i] = 0;
}

// ---------------------------------------------------------------- a few tokens: small tiles, k shared out
// A tile is up to 128 rows of x by 64, 128 or 192 rows of w, and `split` blocks of a cluster share out its range of k.  What
// bounds it is w's bytes where w is large (8 x 24,576 x 4,096: 12.1 to 12.5 us, 4.3 TB/s between the start of one call and of the next, some
// 5.7 while w streams) and the chain of latencies between two kernels where it is not (64 x 4,096 x 4,096: 5.9 us for 1.5 us of
// bytes: 1 from the kernel before to this one's start, 1 for x, 1 for the main loop, 2 for the sums and the results), so the sizes
// are chosen (f4_few_shape) to give each SM one block.
//
// The blocks of a cluster send each row of sums, by asynchronous stores that the receiver's mbarrier counts, to the block that
// finishes that row (rank r % split).  No block reads another's memory, so none has to stay for the others but one whose own wait
// for sums runs out: a barrier of the whole cluster behind the reading took 1.1 us.  The stores take some two clocks per 16 bytes; above 8,000 results of a tile a row
// goes as one bulk copy from shared memory instead, and the blocks stay for each other (by then with an arrival that waits for no
// stores): 128 x 4,096 x 12,288 11.8 us by stores and 10.2 by copies, 64 rows 9.2 and 8.5, but 64 x 4,096 x 4,096 in tiles of 64
// 6.1 and 6.4.
// Twelve warps, four for each 64 columns of a tile: with six in all 8 x 24,576 x 4,096 took 12.35 us instead of 12.1, with a gate and
// 64 rows 16.2 instead of 14.3.
constexpr int F4_FEW_THREADS = 384;
constexpr int F4_BAR_BYTES = 512;  // barriers and the address of the tensor memory, in both kernels
constexpr int F4_FEW_MAX_STAGES = 24;
constexpr int F4_FEW_MAX_SPLIT = 8;
constexpr int F4_FEW_COLS = 256;  // tensor memory: up to 192 columns of sums, two times 24 of scales
constexpr int F4_FEW_SCALE_COLS = 24;
constexpr int F4_BULK_FROM = 8000;  // results of a tile above which its sums travel by bulk copies

struct F4FewShape {
  int a_rows, bn, stages, split;  // rows of x in a tile (a multiple of 8, at most 128), rows of w in it, stages of the ring, blocks
  int depth;                      // stages that a block works through (the last one of a cluster may have fewer)
  int split_inverse;              // 65536 / split, rounded up: (r * split_inverse) >> 16 = r / split for r < 128
  int bulk;                       // rows of sums go to the blocks that finish them by bulk copies, else by stores (split > 1)
  int slots;                      // rows of sums that a block of the cluster receives from each (split > 1)
  __host__ __device__ int a_bytes() const { return a_rows * 128; }
  __host__ __device__ int b_bytes() const { return bn * 128; }
  __host__ __device__ int w_scale_tiles() const { return (bn + FP4_TILE - 1) / FP4_TILE; }
  __host__ __device__ int stage_bytes() const { return a_bytes() + b_bytes() + (1 + w_scale_tiles()) * 2 * FP4_TILE_BYTES; }
  // the last x tile is read as 128 rows
  __host__ __device__ int behind_bytes() const { return 128 * 128 > stage_bytes() ? 128 * 128 - stage_bytes() : 0; }
  __host__ __device__ int ring_bytes() const { return stages * stage_bytes() + behind_bytes(); }
  __host__ __device__ int received_bytes() const { return split > 1 ? split * slots * bn * 4 : 0; }
  __host__ __device__ size_t smem_bytes() const { return (size_t)ring_bytes() + received_bytes() + F4_BAR_BYTES; }
};

__device__ __forceinline__ uint32_t cluster_id() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
// Four values to `address` of the cluster's window; the mbarrier at `bar`, in the same block, counts their 16 bytes.
__device__ __forceinline__ void st_async_v4(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(address), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar)
               : "memory");
}

// One of four barriers (`which`, the same in a warp) for `threads` of the block.
__device__ __forceinline__ void named_barrier(int which, int threads) {
  if (which == 0) asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
  else if (which == 1) asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
  else if (which == 2) asm volatile("bar.sync 3, %0;" ::"r"(threads) : "memory");
  else asm volatile("bar.sync 4, %0;" ::"r"(threads) : "memory");
}
// `bytes` of this block's shared memory to `address` of the cluster's window; the mbarrier at `bar`, in the same block, counts them.
__device__ __forceinline__ void bulk_to_cluster(uint32_t address, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(address), "r"(s_addr(from)), "r"(bytes), "r"(bar)
               : "memory");
}

// Only the first a_rows rows of an x tile are brought in; the instruction reads 128, the rest being whatever follows in shared
// memory (every byte is two valid codes), into rows of the accumulator that are not looked at.
template <int EPI>
__global__ void __launch_bounds__(F4_FEW_THREADS)
gemm_fp4_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ F4Args p, const __grid_constant__ F4FewShape shape, const int early, int* status) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int stages = shape.stages, stage_bytes = shape.stage_bytes(), split = shape.split, bn = shape.bn;
  float* const received = reinterpret_cast<float*>(smem_raw + shape.ring_bytes());
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_raw + shape.ring_bytes() + shape.received_bytes());
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint64_t* sums_full = acc_full + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sums_full + 1);
  __shared__ int abort_flag, stay;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_rank() : 0, tile = split > 1 ? (int)cluster_id() : blockIdx.x;
  const int across = fp4_tiles(p.K), k_stages = (across + 1) / 2;
  const int k0 = rank * shape.depth, k_count = min(shape.depth, k_stages - k0);
  const int m0 = blockIdx.y * F4_BM, n0 = tile * bn, rows_here = min(F4_BM, p.T - m0);
  const int w_tile = n0 / FP4_TILE, w_here = min((n0 % FP4_TILE + bn + FP4_TILE - 1) / FP4_TILE, fp4_tiles(p.N) - w_tile);
  const bool aligned = (s_addr(smem_raw) & 1023u) == 0;
  if (!aligned && threadIdx.x == 0) atomicOr(status, Q3_STATUS_TIMEOUT);

  auto scale_bytes = [&](int it) { return (uint32_t)min(2, across - 2 * (k0 + it)) * FP4_TILE_BYTES; };  // the last stage may have one tile
  auto w_scales_at = [&](int it, int j) { return p.w_scales + ((size_t)(w_tile + j) * across + 2 * (k0 + it)) * FP4_TILE_BYTES; };
  auto load_w = [&](int it, int s) {
    unsigned char* b = smem_raw + (size_t)s * stage_bytes + shape.a_bytes();
    unsigned char* sb = b + shape.b_bytes() + 2 * FP4_TILE_BYTES;
    const uint32_t sf = scale_bytes(it);
    mbar_expect_tx(&full[s], shape.a_bytes() + shape.b_bytes() + (1 + w_here) * sf);
    tma_load_2d(b, &map_w, &full[s], (k0 + it) * 64, n0);
    for (int j = 0; j < w_here; ++j) f4_bulk_load(sb + j * 2 * FP4_TILE_BYTES, w_scales_at(it, j), sf, &full[s]);
  };
  auto load_x = [&](int it, int s) {
    unsigned char* a = smem_raw + (size_t)s * stage_bytes;
    f4_bulk_load(a + shape.a_bytes() + shape.b_bytes(), p.x_scales + ((size_t)blockIdx.y * across + 2 * (k0 + it)) * FP4_TILE_BYTES,
                 scale_bytes(it), &full[s]);
    if (it != tc_drop_copy)  // tests of the give-up path only (see tc_common.cuh)
      tma_load_2d(a, &map_x, &full[s], (k0 + it) * 64, m0);
  };
  if (threadIdx.x == 0) {
    abort_flag = 0;
    stay = 0;  // set by a block of the cluster whose wait for its sums runs out (sums by bulk copies)
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(sums_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // the rows that this block finishes, from every block of the cluster
    if (split > 1) mbar_expect_tx(sums_full, (uint32_t)(split * (((rows_here - rank + split - 1) * shape.split_inverse) >> 16) * bn * 4));
  }
  __syncthreads();
  if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for before anything is sent

  if (warp == 0) {
    // Where w is known not to come from the kernel before, its part of the ring's first round goes out ahead of the wait.
    const int ahead = early ? min(stages, k_count) : 0;
    if (aligned && elect_one()) {
      tma_prefetch_map(&map_x);
      for (int it = 0; it < ahead; ++it) load_w(it, it);
    }
    __syncwarp();
    pdl_wait();  // x comes from the kernel before this one
    if (aligned) {
      if (elect_one())
        for (int it = 0; it < ahead; ++it) load_x(it, it);
      __syncwarp();
      int it = ahead, s = ahead == stages ? 0 : ahead;
      for (uint32_t parity = 1; it < k_count; ++it) {
        if (it >= stages && !warp_wait(&empty[s], parity ^ 1, &abort_flag)) {
          if (lane == 0) {
            abort_flag = 1;
            atomicOr(status, Q3_STATUS_TIMEOUT);
          }
          break;
        }
        if (elect_one()) {
          load_w(it, s);
          load_x(it, s);
        }
        __syncwarp();
        if (++s == stages) {
          s = 0;
          if (it >= stages) parity ^= 1;
        }
      }
      if (lane == 0) finish_copies(full, it, stages, tc_drop_copy, status);
      __syncwarp();
    }
  } else if (warp == 1) {
    pdl_wait();
    pdl_launch_dependents();
    // Tensor memory is taken only after the wait: a block that holds some while it waits for the kernel before it could keep
    // that kernel's own blocks from ever getting theirs.
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_holder)), "r"(F4_FEW_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    const uint32_t tmem = *(volatile uint32_t*)tmem_holder;
    if (aligned) {
      bool ok = true;
      const uint32_t low = f4_idesc(bn, 0), high = f4_idesc(bn, 2);
      uint32_t parity = 0;
      for (int it = 0, s = 0; it < k_count; ++it) {
        if (!warp_wait(&full[s], parity, &abort_flag)) {
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const unsigned char* a = smem_raw + (size_t)s * stage_bytes;
        const unsigned char *b = a + shape.a_bytes(), *sa = b + shape.b_bytes(), *sb = sa + 2 * FP4_TILE_BYTES;
        const uint64_t a_desc = umma_desc_sw128(a), b_desc = umma_desc_sw128(b), sa_desc = f4_scale_desc(sa), sb_desc = f4_scale_desc(sb);
        // the scales of this stage beside those of the last one, which its instructions may still read; a column per 32 rows
        const uint32_t ta = tmem + bn + (it & 1) * F4_FEW_SCALE_COLS, tb = ta + 8, tb_here = tb + (n0 % FP4_TILE) / 32;
        const bool both = across - 2 * (k0 + it) > 1;
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (h == 0 || both) {
              f4_copy_scales(ta + 4 * h, sa_desc + h * (FP4_TILE_BYTES >> 4));
              f4_copy_scales(tb + 8 * h, sb_desc + h * (FP4_TILE_BYTES >> 4));
              if (w_here > 1) f4_copy_scales(tb + 8 * h + 4, sb_desc + (2 + h) * (FP4_TILE_BYTES >> 4));
              f4_mma(tmem, a_desc + 4 * h, b_desc + 4 * h, low, ta + 4 * h, tb_here + 8 * h, (it | h) != 0);
              f4_mma(tmem, a_desc + 4 * h + 2, b_desc + 4 * h + 2, high, ta + 4 * h, tb_here + 8 * h, 1);
            }
          umma_commit(&empty[s]);
          if (it + 1 == k_count) umma_commit(acc_full);
        }
        __syncwarp();
        if (++s == stages) {
          s = 0;
          parity ^= 1;
        }
      }
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicOr(status, Q3_STATUS_TIMEOUT);
      }
      __syncwarp();
    }
  } else {
    pdl_wait();
  }
  // A gate's rows are finished either by sixteen lanes to 64 columns (below) or, where they are more than a few, by a lane to a row
  // straight from the accumulator (24,576 x 4,096, us: 8 rows 13.1 and 13.9, 16 rows 13.7 and 13.9, 24 rows 14.1 and 13.7, 64 rows
  // 17.5 and 14.3, 128 rows 23.3 and 15.6).
  const bool by_rows = EPI == 2 && split == 1 && rows_here > 16;
  // Every thread gets here, whatever was given up, so the cluster's barrier needs no bound.
  if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  float* const sums = split > 1 ? received : reinterpret_cast<float*>(smem_raw);  // alone: over the ring, which nothing reads by then
  const bool by_bulk = shape.bulk != 0;
  // Four warps for each 64 columns of the accumulator, the first of them the last ones: by then they are done with their own work.
  const int c0 = (F4_FEW_THREADS / 128 - 1 - (warp >> 2)) * 64;
  if (c0 < bn && aligned) {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const bool summed = warp_wait(acc_full, 0, &abort_flag);
    if (!summed) {
      if (lane == 0) {
        abort_flag = 1;
        atomicOr(status, Q3_STATUS_TIMEOUT);
      }
      __syncwarp();
    } else if (quarter * 32 < rows_here) {
      tcgen05_fence_after();
      const uint32_t acc = *(volatile uint32_t*)tmem_holder + ((uint32_t)(quarter * 32) << 16) + c0;
      uint32_t v[2][32];
      tmem_ld_32(acc, v[0]);
      tmem_ld_32(acc + 32, v[1]);
      tmem_wait_ld();
      if (row >= rows_here) {
      } else if (EPI == 2 && by_rows) {
        if (n0 + c0 < p.N) f4_gated_block(v[0], v[1], p, m0 + row, n0 + c0);
      } else if (split > 1 && !by_bulk) {
        const int slot = (row * shape.split_inverse) >> 16, owner = row - slot * split;  // row / split, row % split
        const uint32_t to = cluster_addr(s_addr(received + (rank * shape.slots + slot) * bn), owner);
        const uint32_t bar = cluster_addr(s_addr(sums_full), owner);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          st_async_v4(to + (c0 + 4 * j) * 4, v[j / 8][4 * (j % 8)], v[j / 8][4 * (j % 8) + 1], v[j / 8][4 * (j % 8) + 2],
                      v[j / 8][4 * (j % 8) + 3], bar);
      } else {  // rows bn + 4 values apart, off each other's banks
#pragma unroll
        for (int j = 0; j < 16; ++j)
          *reinterpret_cast<uint4*>(reinterpret_cast<float*>(smem_raw) + row * (bn + 4) + c0 + 4 * j) =
              make_uint4(v[j / 8][4 * (j % 8)], v[j / 8][4 * (j % 8) + 1], v[j / 8][4 * (j % 8) + 2], v[j / 8][4 * (j % 8) + 3]);
      }
      __syncwarp();
    }
    if (by_bulk && quarter * 32 < rows_here) {
      fence_async_proxy();  // the copies read what these stores left
      named_barrier(quarter, bn / 2);  // of the warps of these 32 rows, all of which get here
      if (summed && c0 == 0 && row < rows_here) {
        const int slot = (row * shape.split_inverse) >> 16, owner = row - slot * split;
        bulk_to_cluster(cluster_addr(s_addr(received + (rank * shape.slots + slot) * bn), owner),
                        reinterpret_cast<float*>(smem_raw) + row * (bn + 4), bn * 4, cluster_addr(s_addr(sums_full), owner));
      }
      __syncwarp();
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    const uint32_t tmem = *(volatile uint32_t*)tmem_holder;
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F4_FEW_COLS) : "memory");
  }
  // A block that gave up does not cut this wait short: the others' sums may still be on their way into its memory.  What other blocks
  // wrote is acquired at the cluster's scope.
  int never = 0;
  const bool here = split == 1 || warp_wait_cluster(sums_full, 0, &never);
  if (!here && lane == 0) atomicOr(status, Q3_STATUS_TIMEOUT);
  __syncwarp();
  if (by_bulk) {
    // What was sent by bulk copies is read from here until it is there: a block stays until all of its cluster have their sums, or,
    // where one's wait ran out, until that one says so and the copies have had another such wait (below).
    if (here) {
      asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    } else {
      if (lane < split) st_cluster_u32(cluster_addr(s_addr(&stay), lane), 1u);  // none of them leaves before this warp arrives
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
  } else if (!here) {
    // Another block may be late by several waits of its own and send its sums only now.  So this warp stays until every thread of the
    // cluster has sent all that it will (one that has returned holds the barrier up no longer, so the others wait for nobody), and
    // then for what is still on its way.
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    warp_wait_cluster(sums_full, 0, &never);
  }

  // Sixteen lanes finish 64 columns of a row, four to a lane.  The blocks' sums are added in the order of their ranges of k.
  const int inner = p.N / 2, out_across = fp4_tiles(inner), blocks = (inner + FP4_BLOCK - 1) / FP4_BLOCK;
  const int groups = bn / 64, my_rows = ((rows_here - rank + split - 1) * shape.split_inverse) >> 16;
  const int items = by_rows || !here ? 0 : my_rows * groups, l = lane & 15;
  for (int i0 = warp * 2; i0 < items; i0 += 2 * (F4_FEW_THREADS / 32)) {
    const int item = min(i0 + (lane >> 4), items - 1);  // lanes without an item of their own do the last one again
    const int slot = groups == 1 ? item : groups == 2 ? item >> 1 : item / 3, g = item - slot * groups;
    const float* mine = sums + slot * (split > 1 ? bn : bn + 4) + g * 64 + l * 4;
    float4 v = *reinterpret_cast<const float4*>(mine);
    for (int q = 1; q < split; ++q) {
      const float4 u = *reinterpret_cast<const float4*>(mine + (size_t)q * shape.slots * bn);
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
    const int row = m0 + (split > 1 ? slot * split + rank : slot), col = n0 + g * 64 + l * 4;
    if (EPI == 2) {
      // Of four lanes two hold eight gate columns and two their up columns; each takes two of the eight results, the other
      // operand from the lane two further.  Sixteen lanes have a block of 32.
      const bool second = l & 2;
      const float o0 = __shfl_xor_sync(0xffffffffu, second ? v.x : v.z, 2), o1 = __shfl_xor_sync(0xffffffffu, second ? v.y : v.w, 2);
      const float gate[2] = {second ? o0 : v.x, second ? o1 : v.y}, up[2] = {second ? v.z : o0, second ? v.w : o1};
      const int block = n0 / 64 + g, place = (l >> 2) * 4 + (l & 1) * 2 + (second ? 1 : 0);  // of the lane's two among the block's
      float a[2];
      f4_gate<2>(gate, up, p.act, a);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (block * 32 + place * 2 + i >= inner) a[i] = 0.f;
      const uint32_t half = lane < 16 ? 0xffffu : 0xffff0000u;
      const uint32_t top = __reduce_max_sync(half, fp4_top(fp4_top(0u, a[0]), a[1]));
      const uint32_t byte = fp4_scale_byte(top);
      const float inv = fp4_inverse_scale(byte);
      uint32_t c = byte == 255u ? 0u : fp4_pack2(a[0] * inv, a[1] * inv) << (8 * (place & 3));
      c |= __shfl_xor_sync(0xffffffffu, c, 1);
      c |= __shfl_xor_sync(0xffffffffu, c, 2);
      if (block < blocks) {
        if ((l & 3) == 0) *reinterpret_cast<uint32_t*>(p.out_codes + (size_t)row * fp4_pitch(inner) + block * 16 + l) = c;
        if (l == 0) {
          uint8_t* word = p.out_scales + fp4_scale_word(row, block / 4, out_across);
          word[block % 4] = (uint8_t)byte;
          if (block + 1 == blocks)  // and the scales behind the last block, up to the end of their tile, are zero
            for (int j = block % 4 + 1; j < 4; ++j) word[j] = 0;
        }
      }
    } else if (EPI == 0) {
      __nv_bfloat16* dst = (__nv_bfloat16*)p.out + (size_t)row * p.ldc + col;
      if (col + 4 <= p.N && ((uintptr_t)dst & 7) == 0) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(__float_as_uint(v.x), __float_as_uint(v.y)),
                                                    pack2(__float_as_uint(v.z), __float_as_uint(v.w)));
      } else {
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < p.N) dst[i] = __float2bfloat16_rn(f[i]);
      }
    } else {
      float* dst = (float*)p.out + (size_t)row * p.ldc + col;
      if (col + 4 <= p.N && ((uintptr_t)dst & 15) == 0) {
        *reinterpret_cast<float4*>(dst) = v;
      } else {
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < p.N) dst[i] = f[i];
      }
    }
  }
  if (by_bulk) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (*(volatile int*)&stay) {  // the same in every thread of the cluster: written before the barrier or not at all
      warp_wait_cluster(sums_full, 0, &never);
      asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
  }
}

// ---------------------------------------------------------------- many tokens: tiles of 256 x 192, 256 or 384 by pairs of CTAs
// The CTA of rank r holds rows 128 r .. of the x tile and half of the w tile's rows, rows 128 r .. of the accumulator, its own rows'
// scales and all of the w tile's scales; the roles are those of gemm_tc_pair_kernel (gemm_tc.cu).
//
// What bounds the main loop is what an SM takes in, 64 bytes a clock: a stage of 192, 256 or 384 columns is 31, 35 or 44 KB and
// takes the tensor cores 384, 512 or 768 clocks; measured 490, 522 and 800.  Against that, tensor memory has room for two
// accumulators only of 192 columns beside the scales, the epilogue of one tile running under the main loop of the next; with one
// accumulator the tensor cores stand still until the epilogue's warps have it in their registers, which takes 450 clocks, and some
// 1,000 with the ways there and back (of 384 columns, two instructions of 192, as bfloat16: with a gate or float32 results, which
// the registers do not hold, such a tile took 92 us against 79 for 2,048 x 24,576 x 4,096 and is not built).  For long calls the
// device holds its 1 kW by its clock, at about 1.6 GHz: 2,048 x 24,576 x 4,096 one after another 86 us, 73 with pauses.
template <int BN, int EPI>
struct F4Pair {
  static constexpr int ACCS = BN == 192 ? 2 : 1;
  static constexpr int MMA_N = BN == 384 ? 192 : BN, PARTS = BN / MMA_N;  // columns of an instruction, instructions for a tile's columns
  static constexpr int STORE_BYTES = EPI == 2 ? 0 : 8 * 4096;  // where each of the epilogue's warps turns its rows around
  static constexpr int STAGES = (BN == 192 ? 7 : BN == 256 ? 6 : 5) - (EPI == 2 ? 0 : 1);
  static constexpr int W_TILES = BN == 384 ? 3 : 2;  // tiles of scales that a w tile may touch
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / 2 * 128, SA_BYTES = 2 * FP4_TILE_BYTES, SB_BYTES = W_TILES * 2 * FP4_TILE_BYTES;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
  static constexpr size_t SMEM_BYTES = (size_t)STAGES * STAGE_BYTES + STORE_BYTES + F4_BAR_BYTES;
  static constexpr uint32_t SCALE_COL = ACCS * BN, SCALE_COLS = 8 + 8 * W_TILES, COLS = 512;  // two sets of scales
  static_assert(SCALE_COL + 2 * SCALE_COLS <= COLS && (BN != 384 || EPI == 0), "");
};
constexpr int F4_PAIR_EPI_WARPS = 8;
constexpr int F4_PAIR_THREADS = 64 + 32 * F4_PAIR_EPI_WARPS;
constexpr int F4_PAIR_GROUP = 8;  // tiles of x that are walked through for one tile of w before the next one

__device__ __forceinline__ void f4_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
      : "memory");
}
// Each CTA of the pair copies from its own shared memory, at this place, into its own tensor memory.
__device__ __forceinline__ void f4_copy_scales_pair(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// An arrival on a barrier of the pair that orders nothing by itself: what goes before it (a warp's reads of tensor memory) and behind
// the wait for it (instructions that write there) is ordered by the tcgen05 fences on either side.  One that releases at the
// cluster's scope waits for the warp's stores to memory: 1,050 to 3,600 clocks of every tile, 81 us instead of 74 for 2,048 x 24,576
// x 4,096 in tiles of 256 columns.
__device__ __forceinline__ void f4_arrive_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Tile number `i` of a walk over m_tiles x n_tiles in which GROUP tiles of x stay in the second-level cache.
__device__ __forceinline__ void f4_tile(int i, int m_tiles, int n_tiles, int* m, int* n) {
  const int per = F4_PAIR_GROUP * n_tiles, g = i / per, first = g * F4_PAIR_GROUP;
  const int high = min(F4_PAIR_GROUP, m_tiles - first), j = i - g * per;
  *m = first + j % high;
  *n = j / high;
}

template <int EPI, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F4_PAIR_THREADS)
gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws,
                     const __grid_constant__ F4Args p, int* status) {
  using S = F4Pair<BN, EPI>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_raw + (size_t)S::STAGES * S::STAGE_BYTES + S::STORE_BYTES);  // used in rank 0
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;
  uint64_t* acc_empty = acc_full + S::ACCS;  // used in rank 0
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + S::ACCS);
  __shared__ int abort_flag;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int across = fp4_tiles(p.K), k_stages = (across + 1) / 2;
  const int m_tiles = (p.T + 255) / 256, n_tiles = (p.N + BN - 1) / BN;
  const bool aligned = (s_addr(smem_raw) & 1023u) == 0;  // the same in both CTAs
  const int num_tiles = aligned ? m_tiles * n_tiles : 0;
  if (!aligned && threadIdx.x == 0) atomicOr(status, Q3_STATUS_TIMEOUT);
  auto give_up = [&]() {  // one thread
    abort_flag = 1;
    st_cluster_u32(cluster_addr(s_addr(&abort_flag), rank ^ 1u), 1u);
    atomicOr(status, Q3_STATUS_TIMEOUT);
  };

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_xs);
    tma_prefetch_map(&map_ws);
    abort_flag = 0;
    *tmem_holder = 0;
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < S::ACCS; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * F4_PAIR_EPI_WARPS);  // the epilogue warps of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  cluster_sync_all();
  pdl_wait();  // x comes from the kernel before this one
  pdl_launch_dependents();
  if (warp == 1) {  // only after the wait, as above; the same warp of both CTAs asks, for the pair
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_holder)), "r"(S::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    uint32_t it = 0;
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += pairs) {
      int m, n;
      f4_tile(tile, m_tiles, n_tiles, &m, &n);
      for (int kt = 0; kt < k_stages; ++kt, ++it) {
        const int s = it % S::STAGES;
        const uint32_t use = it / S::STAGES;
        if (use > 0 && !warp_wait(&empty[s], (use & 1) ^ 1, &abort_flag)) {
          if (lane == 0) give_up();
          ok = false;
          break;
        }
        unsigned char* a = smem_raw + (size_t)s * S::STAGE_BYTES;
        unsigned char *b = a + S::A_BYTES, *sa = b + S::B_BYTES, *sb = sa + S::SA_BYTES;
        const uint32_t bar = cluster_addr(s_addr(&full[s]), 0);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&full[s], 2 * S::STAGE_BYTES);
#pragma unroll
          for (int q = 0; q < S::PARTS; ++q)  // of the rows of an instruction the first half is rank 0's
            tma_load_2d_pair(b + q * (S::MMA_N / 2 * 128), &map_w, bar, kt * 64, n * BN + q * S::MMA_N + (int)rank * (S::MMA_N / 2));
          tma_load_2d_pair(sb, &map_ws, bar, kt * 256, n * BN / FP4_TILE);
          tma_load_2d_pair(sa, &map_xs, bar, kt * 256, m * 2 + (int)rank);
          if ((int)it != tc_drop_copy || rank != 0)  // tests of the give-up path only (see tc_common.cuh)
            tma_load_2d_pair(a, &map_x, bar, kt * 64, m * 256 + (int)rank * 128);
        }
        __syncwarp();
      }
    }
    if (rank == 0 && lane == 0) finish_copies(full, it, S::STAGES, tc_drop_copy, status);  // its barriers count both CTAs' copies
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t it = 0, t = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += pairs, ++t) {
        int m, n;
        f4_tile(tile, m_tiles, n_tiles, &m, &n);
        const uint32_t buf = t % S::ACCS, acc = tmem + buf * BN, shift = n * BN % FP4_TILE / 32;  // of its scales: a column per 32 rows
        if (t >= S::ACCS && !warp_wait_cluster(&acc_empty[buf], ((t / S::ACCS) & 1) ^ 1, &abort_flag)) {
          ok = false;
          break;
        }
        tcgen05_fence_after();
        for (int kt = 0; kt < k_stages; ++kt, ++it) {
          const int s = it % S::STAGES;
          if (!warp_wait_cluster(&full[s], (it / S::STAGES) & 1, &abort_flag)) {
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const unsigned char* a = smem_raw + (size_t)s * S::STAGE_BYTES;
          const unsigned char *b = a + S::A_BYTES, *sa = b + S::B_BYTES, *sb = sa + S::SA_BYTES;
          const uint64_t a_desc = umma_desc_sw128(a), b_desc = umma_desc_sw128(b), sa_desc = f4_scale_desc(sa), sb_desc = f4_scale_desc(sb);
          // the scales of this stage beside those of the last one, which its instructions may still read
          const uint32_t ta = tmem + S::SCALE_COL + (it & 1) * S::SCALE_COLS, tb = ta + 8;
          const bool both = across - 2 * kt > 1;
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (h == 0 || both) {
                f4_copy_scales_pair(ta + 4 * h, sa_desc + h * (FP4_TILE_BYTES >> 4));
#pragma unroll
                for (int j = 0; j < S::W_TILES; ++j)
                  f4_copy_scales_pair(tb + 4 * (S::W_TILES * h + j), sb_desc + j * (S::SA_BYTES >> 4) + h * (FP4_TILE_BYTES >> 4));
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int q = 0; q < S::PARTS; ++q)
                    f4_mma_pair(acc + q * S::MMA_N, a_desc + 4 * h + 2 * e, b_desc + q * (S::MMA_N / 2 * 128 >> 4) + 4 * h + 2 * e,
                                f4_idesc(S::MMA_N, 2 * e, 256), ta + 4 * h, tb + shift + 4 * S::W_TILES * h + q * (S::MMA_N / 32),
                                (kt | h | e) != 0);
              }
            umma_commit_pair(&empty[s]);
            if (kt + 1 == k_stages) umma_commit_pair(&acc_full[buf]);
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) give_up();
    }
  } else {
    // two warps for each quarter of the rows, for the first and the other columns
    constexpr int FIRST = BN == 384 ? 192 : 128;
    const int quarter = warp & 3, half = (warp - 2) >> 2, pieces = (half ? BN - FIRST : FIRST) / 64;
    unsigned char* const store = smem_raw + (size_t)S::STAGES * S::STAGE_BYTES + (warp - 2) * 4096;  // EPI 0, 1
    uint32_t t = 0;
    for (int tile = pair; tile < num_tiles; tile += pairs, ++t) {
      int m, n;
      f4_tile(tile, m_tiles, n_tiles, &m, &n);
      const uint32_t buf = t % S::ACCS;
      if (!warp_wait(&acc_full[buf], (t / S::ACCS) & 1, &abort_flag)) {
        if (lane == 0) give_up();
        __syncwarp();
        break;
      }
      tcgen05_fence_after();
      const int row0 = m * 256 + (int)rank * 128 + quarter * 32, n0 = n * BN + half * FIRST;
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + buf * BN + (uint32_t)half * FIRST;
      auto release = [&]() {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) f4_arrive_relaxed(cluster_addr(s_addr(&acc_empty[buf]), 0));
        __syncwarp();
      };
      F4RowStore<EPI> to(p, store, row0, n0, 64 * pieces);
      const bool any = row0 < p.T && n0 < p.N;  // uniform over the warp, as all that follows
      if (BN != 384) {
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (c < 2 * pieces) tmem_ld_32(acc + 32 * c, v[c]);
        tmem_wait_ld();
        release();
        uint32_t w[2][32];
        if (EPI == 0 && BN == 256) {  // here and not later, or the registers do not suffice for what follows
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            f4_pack(v[2 * c], v[2 * c + 1], w[c]);
#pragma unroll
            for (int j = 0; j < 32; ++j) asm volatile("" : "+r"(w[c][j]));
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (any && c < pieces) {  // 64 columns: what leaves
            if (EPI == 2) {
              if (row0 + lane < p.T && n0 + 64 * c < p.N) f4_gated_block(v[2 * c], v[2 * c + 1], p, row0 + lane, n0 + 64 * c);
            } else if (EPI == 0) {
              if (BN != 256) f4_pack(v[2 * c], v[2 * c + 1], w[c]);
              to.push(w[c], lane);
            } else {
              to.push(v[2 * c], lane);
              to.push(v[2 * c + 1], lane);
            }
          }
      } else {  // bfloat16 results only: a tile of 384 columns fits in the registers as such
        uint32_t v[2][2][32], w[3][32];
        tmem_ld_32(acc, v[0][0]);
        tmem_ld_32(acc + 32, v[0][1]);
#pragma unroll
        for (int c = 0; c < 3; ++c) {  // the next 64 columns on their way while these are packed
          tmem_wait_ld();
          if (c < 2) {
            tmem_ld_32(acc + 64 * (c + 1), v[(c + 1) & 1][0]);
            tmem_ld_32(acc + 64 * (c + 1) + 32, v[(c + 1) & 1][1]);
          } else {
            release();
          }
          f4_pack(v[c & 1][0], v[c & 1][1], w[c]);
        }
#pragma unroll
        for (int c = 0; c < 3; ++c)
          if (any) to.push(w[c], lane);
      }
      if (EPI != 2 && any) to.end(lane);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
}

// ---------------------------------------------------------------- launches
// A launch with blocks in clusters of `cluster` along x.
template <typename... KArgs, typename... Args>
static int f4_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled() && g_launch_early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  g_plain_launch_stream.store((uintptr_t)stream, std::memory_order_relaxed);
  return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// The scales [tiles, across * 512 bytes] as boxes of 1,024 bytes x `rows` rows of tiles; beyond their end: zeros.
static int f4_scale_map(CUtensorMap* map, const void* ptr, uint64_t tiles, uint64_t across, uint32_t rows) {
  PFN_cuTensorMapEncodeTiled enc = tensor_map_encoder();
  if (!enc) return Q3_ERR_DRIVER;
  const cuuint64_t dims[2] = {across * (FP4_TILE_BYTES / 4), tiles};
  const cuuint64_t strides[1] = {across * FP4_TILE_BYTES};
  const cuuint32_t box[2] = {2 * FP4_TILE_BYTES / 4, rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : Q3_ERR_DRIVER;
}

template <typename Kernel>
static cudaError_t f4_few_configure(Kernel kernel) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024);
  // a kernel that asks for less keeps its SM from taking a block of one that asks for more beside its own
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

template <int EPI>
static int gemm_fp4_few_launch(const CUtensorMap& map_x, const CUtensorMap& map_w, const F4Args& p, const F4FewShape& shape, int early,
                               int* status, cudaStream_t stream) {
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = f4_few_configure(gemm_fp4_few_kernel<EPI>);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const long long blocks = (long long)((p.N + shape.bn - 1) / shape.bn) * shape.split, m_tiles = (p.T + F4_BM - 1) / F4_BM;
  if (blocks > 0x7fffffffLL || m_tiles > 65535) return Q3_ERR_SIZE;
  const int code = f4_launch(gemm_fp4_few_kernel<EPI>, dim3((unsigned)blocks, (unsigned)m_tiles), F4_FEW_THREADS, shape.smem_bytes(),
                             shape.split, stream, map_x, map_w, p, shape, early, status);
  const int last = launch_status();
  return code ? code : last;
}

// How many clusters of 1 to 8 blocks, one to an SM, the device runs at a time: 148, 74, 45, 33, 26, 22, 15 and 15 on 148 SMs, as a
// cluster's SMs are of one group.  (1 x 5,120 x 25,600 with its 27 tiles of 192 rows shared out among 5 blocks each: 21.5 us, the
// last cluster alone in a second round; as 40 tiles of 128 among 3: 14.5.)
static const int* f4_few_slots() {
  static int slots[64][F4_FEW_MAX_SPLIT + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  for (int split = F4_FEW_MAX_SPLIT; slots[dev][1] == 0; --split) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split * sm_count());
    cfg.blockDim = dim3(F4_FEW_THREADS);
    cfg.dynamicSmemBytes = 160 * 1024;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (f4_few_configure(gemm_fp4_few_kernel<0>) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, gemm_fp4_few_kernel<0>, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sm_count() / split;
    }
    slots[dev][split] = n > 0 ? n : 1;
  }
  return slots[dev];
}

// The few-tokens kernel's tiles.  Blocks run one to an SM in rounds; a round takes its stages times what issuing one takes (clocks,
// measured on one SM: 386, 415 and 470 for 64, 128 and 192 rows of w), and sharing out k costs the sending and adding of sums.
static F4FewShape f4_few_shape(int T, int N, int K, double* clocks) {
  F4FewShape best{};
  double best_cost = 0, best_rounds = 0;
  const int k_stages = (fp4_tiles(K) + 1) / 2, rows = T < F4_BM ? T : F4_BM, *const slots = f4_few_slots();
  for (int bn = 64; bn <= 192; bn += 64) {
    const long long tiles = (long long)((N + bn - 1) / bn) * ((T + F4_BM - 1) / F4_BM);
    const int results = rows * bn, sums = results > F4_BULK_FROM && results <= 128 * 160 ? 3000 + results / 5 : 600 + results / 2;
    for (int split = 1; split <= F4_FEW_MAX_SPLIT && split <= k_stages; ++split) {
      const int depth = (k_stages + split - 1) / split;
      if ((split - 1) * depth >= k_stages) continue;  // no block without a stage
      const double rounds = (double)((tiles + slots[split] - 1) / slots[split]);
      const double cost = rounds * (depth * (bn == 64 ? 386 : bn == 128 ? 415 : 470) + (split > 1 ? sums : 0));
      if (best.bn == 0 || cost < best_cost) {
        best_cost = cost;
        best_rounds = rounds;
        best.bn = bn;
        best.split = split;
        best.depth = depth;
      }
    }
  }
  best.a_rows = (rows + 7) / 8 * 8;
  best.slots = (rows + best.split - 1) / best.split;
  best.split_inverse = (65536 + best.split - 1) / best.split;
  const int alone = best.split > 1 ? 0 : rows * (best.bn + 4) * 4;  // the sums' place over the ring
  // Up to eight stages a block keeps to half of an SM's shared memory, so that a block of the next kernel fits beside it and starts
  // while this one ends (1 x 4,096 x 12,288, eight stages: 6.2 us in 112 KB, 7.2 in 224); where it works through more and has an
  // SM for itself, a deeper ring does more for it (8 x 24,576 x 4,096, sixteen stages: 14.1 us in 112 KB, 12.4 in 160).  All of it
  // where that leaves under three stages, or no place for the sums.
  for (int room = best.depth > 8 && best_rounds <= 1 ? 160 * 1024 : 112 * 1024;; room = 224 * 1024) {
    best.stages = (room - best.behind_bytes() - best.received_bytes() - F4_BAR_BYTES) / best.stage_bytes();
    if (best.stages > best.depth) best.stages = best.depth;
    if (best.stages > F4_FEW_MAX_STAGES) best.stages = F4_FEW_MAX_STAGES;
    if (best.stages < 1) best.stages = 1;
    if (room > 160 * 1024 || ((best.stages >= 3 || best.stages == best.depth) && best.ring_bytes() >= alone)) break;
  }
  while (best.ring_bytes() < alone) ++best.stages;
  best.bulk = best.split > 1 && rows * best.bn > F4_BULK_FROM && rows * (best.bn + 4) * 4 <= best.ring_bytes();
  // Rounds of blocks that take more than half of an SM's shared memory do not overlap (128 rows of 192 columns: some 8,000 clocks from
  // one's start to its first stage and from its last one to its end).
  const double apart = best.smem_bytes() > 113 * 1024 ? (best_rounds - 1) * (3000 + rows * best.bn / 5) : 0;
  // What it takes, for the choice between the kernels: with many rows a stage takes as long as its bytes do, some 40 a clock.
  const int issue = best.bn == 64 ? 386 : best.bn == 128 ? 415 : 470, bytes = best.stage_bytes() / 40;
  *clocks = best_cost + best_rounds * best.depth * (bytes > issue ? bytes - issue : 0) + apart;
  return best;
}

// How many pairs of CTAs the device runs at a time (a cluster's two CTAs need SMs of one group).
static int f4_pair_slots() {
  static int slots[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  if (slots[dev] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * sm_count());
    cfg.blockDim = dim3(F4_PAIR_THREADS);
    cfg.dynamicSmemBytes = F4Pair<256, 0>::SMEM_BYTES;
    int n = 0;
    if (cudaFuncSetAttribute(gemm_fp4_pair_kernel<0, 256>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F4Pair<256, 0>::SMEM_BYTES) !=
            cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, gemm_fp4_pair_kernel<0, 256>, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sm_count() / 2;
    }
    slots[dev] = n < sm_count() / 2 ? n : sm_count() / 2;
  }
  return slots[dev];
}

// Clocks of the pair kernel's rounds: its stages, and what a tile takes beside them.  Measured with 192, 256 and 384 columns, us:
// 79, 77, 73 at 2,048 x 24,576 x 4,096, 43, 40, 53 at 2,048 x 4,096 x 12,288, 350, 341, 364 at 8,192 x 5,120 x 25,600, 16.4, 20,
// 28 at 256 x 4,096 x 12,288 (a stage 420, 560 and 715 clocks, and 1,700, 1,200 and 3,700 a tile, fit these and ten more).  Where k is
// short a tile takes as long as its results do to leave: 53, 50 and 49 us at 8,000 x 16,000 x 64, in float32 105 and 101; and with
// rows off a sector's boundary (16,001 columns) 122, 105 and 98, in float32 177 and 147.
static double f4_pair_cost(int T, int N, int K, int bn, int epi, bool whole) {
  const long long tiles = (long long)((N + bn - 1) / bn) * ((T + 255) / 256), slots = f4_pair_slots();
  const int k_stages = (fp4_tiles(K) + 1) / 2;
  const double stage = bn == 192 ? 420 : bn == 256 ? 560 : 715, hold = bn == 192 ? 1700 : bn == 256 ? 1200 : 3700;
  double leave = bn == 192 ? 4500 : 6000;  // a gate
  if (epi == 0) leave = whole ? (bn == 192 ? 2200 : bn == 256 ? 2700 : 3900) : (bn == 192 ? 5000 : bn == 256 ? 5600 : 7700);
  if (epi == 1) leave = whole ? (bn == 192 ? 4300 : 5400) : (bn == 192 ? 7200 : 7900);
  const double tile = k_stages * stage + hold;
  return (double)((tiles + slots - 1) / slots) * (tile > leave ? tile : leave);
}

template <int EPI, int BN>
static int gemm_fp4_pair_launch(const void* x_codes, const void* w_codes, const F4Args& p, int* status, cudaStream_t stream) {
  using S = F4Pair<BN, EPI>;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(gemm_fp4_pair_kernel<EPI, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  // the maps of codes take two bytes as one bfloat16: only bytes move
  CUtensorMap map_x, map_w, map_xs, map_ws;
  const uint64_t cols = fp4_pitch(p.K) / 2, across = fp4_tiles(p.K);
  int code = cached_map(&map_x, x_codes, (uint64_t)p.T, cols, 128);
  if (!code) code = cached_map(&map_w, w_codes, (uint64_t)p.N, cols, S::MMA_N / 2);
  if (!code) code = f4_scale_map(&map_xs, p.x_scales, fp4_tiles(p.T), across, 1);
  if (!code) code = f4_scale_map(&map_ws, p.w_scales, fp4_tiles(p.N), across, S::W_TILES);
  if (code) return code;
  const long long tiles = (long long)((p.N + BN - 1) / BN) * ((p.T + 255) / 256);
  if (tiles > 0x3fffffffLL) return Q3_ERR_SIZE;
  const long long slots = f4_pair_slots();
  code = f4_launch(gemm_fp4_pair_kernel<EPI, BN>, dim3((unsigned)(2 * (tiles < slots ? tiles : slots))), F4_PAIR_THREADS, S::SMEM_BYTES,
                   1, stream, map_x, map_w, map_xs, map_ws, p, status);
  const int last = launch_status();
  return code ? code : last;
}

// early: w was not written by the kernel that runs before this one.  form: 0 by the clocks that the forms take, 1 the kernel for a few
// tokens, 192, 256 or (bfloat16 results) 384 columns by pairs of CTAs.
template <int EPI>
static int gemm_fp4(const void* x_codes, const void* w_codes, const F4Args& p, int form, int early, int* status, cudaStream_t stream) {
  double few = 0;
  const F4FewShape shape = f4_few_shape(p.T, p.N, p.K, &few);
  if (form == 0 && p.T > 64) {
    // Pairs of CTAs where their rounds, and some 3,500 clocks that their start and end take longer (5,500 with a gate), are fewer
    // clocks.  Measured, few / pairs, us: 72 rows 28.0 / 30.2 at 51,200 x 5,120; 96 rows 14.6 / 15.5 at 24,576 x 4,096, 32.4 / 31.2
    // at 51,200 x 5,120, 11.4 / 15.4 at 4,096 x 12,288; 128 rows 22.3 / 28.8 at 5,120 x 25,600; 200 rows 24.5 / 16.7 at 24,576 x
    // 4,096, 18.6 / 16.1 at 4,096 x 12,288; 400 rows 4.9 / 5.7 at 1,024 x 1,024, 9.8 / 9.1 at 4,096 x 4,096, 20.9 / 17.6 at 4,096 x
    // 12,288; with a gate 128 rows 15.3 / 17.0 at 24,576 x 4,096, 400 rows 9.8 / 10.6 at 4,096 x 4,096 and 42.7 / 25.1 at 24,576 x 4,096.
    const bool whole = EPI == 2 || (((uintptr_t)p.out | (size_t)p.ldc * (EPI == 0 ? 2 : 4)) & 31) == 0;
    // The kernel for a few tokens has its tiles of rows along the grid's second dimension, of which there are at most 65,535.
    double clocks = p.T > 65535LL * F4_BM ? 1e300 : few - (EPI == 2 ? 5500 : 3500);
    for (int bn : {192, 256, 384}) {
      if (bn == 384 && EPI != 0) break;
      const double c = f4_pair_cost(p.T, p.N, p.K, bn, EPI, whole);
      if (c < clocks) {
        clocks = c;
        form = bn;
      }
    }
  }
  if (form == 192) return gemm_fp4_pair_launch<EPI, 192>(x_codes, w_codes, p, status, stream);
  if (form == 256) return gemm_fp4_pair_launch<EPI, 256>(x_codes, w_codes, p, status, stream);
  if (form == 384) return EPI == 0 ? gemm_fp4_pair_launch<EPI, EPI == 0 ? 384 : 256>(x_codes, w_codes, p, status, stream) : Q3_ERR_SIZE;
  if (form != 0 && form != 1) return Q3_ERR_SIZE;
  // the maps take two bytes of codes as one bfloat16: only bytes move
  CUtensorMap map_x, map_w;
  const uint64_t cols = fp4_pitch(p.K) / 2;
  int code = cached_map(&map_x, x_codes, (uint64_t)p.T, cols, shape.a_rows);
  if (code) return code;
  code = cached_map(&map_w, w_codes, (uint64_t)p.N, cols, shape.bn);
  if (code) return code;
  return gemm_fp4_few_launch<EPI>(map_x, map_w, p, shape, early, status, stream);
}

static bool f4_sizes_ok(int T, int N, int K) { return N > 0 && K > 0 && T > 0 && K <= (1 << 30) && N <= (1 << 30); }
static bool f4_aligned(const void* a, const void* b, const void* c, const void* d) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0;
}

// What is asked of a call before anything of it, or of the calls that belong with it, is launched.
static int fp4_product_check(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, int T, int N, int K,
                             long long ldc) {
  if (!f4_sizes_ok(T, N, K) || ldc < N) return Q3_ERR_SIZE;
  return f4_aligned(x_codes, x_scales, w_codes, w_scales) ? 0 : Q3_ERR_ALIGN;
}
static int fp4_gated_check(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, const void* out_codes,
                           const void* out_scales, int T, int N, int K, int act) {
  if (!f4_sizes_ok(T, N, K) || N % 16 || (act != Q3_ACT_SILU && act != Q3_ACT_RELU && act != Q3_ACT_GELU_TANH)) return Q3_ERR_SIZE;
  return f4_aligned(x_codes, x_scales, w_codes, w_scales) && f4_aligned(out_codes, out_scales, nullptr, nullptr) ? 0 : Q3_ERR_ALIGN;
}

static int fp4_product(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out, int T, int N,
                       int K, long long ldc, int out_f32, int form, int early, int* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (const int code = fp4_product_check(x_codes, x_scales, w_codes, w_scales, T, N, K, ldc)) return code;
  const F4Args p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, out, ldc, nullptr, nullptr, T, N, K, 0};
  if (out_f32) return gemm_fp4<1>(x_codes, w_codes, p, form, early, status, stream);
  return gemm_fp4<0>(x_codes, w_codes, p, form, early, status, stream);
}

static int fp4_gated_product(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out_codes,
                             void* out_scales, int T, int N, int K, int act, int form, int early, int* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (const int code = fp4_gated_check(x_codes, x_scales, w_codes, w_scales, out_codes, out_scales, T, N, K, act)) return code;
  const F4Args p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, nullptr, 0, (uint8_t*)out_codes, (uint8_t*)out_scales, T, N, K, act};
  return gemm_fp4<2>(x_codes, w_codes, p, form, early, status, stream);
}

}  // namespace q3

extern "C" int q3_fp4_add_rmsnorm(const float* in, const void* delta, int dtype, const float* w, float* out, void* codes,
                                  void* scales, int R, int H, float eps, cudaStream_t stream);

// out[T, N] (row pitch ldc) = x w^T of rows held in four bits; out_f32: float32 results, else bfloat16.  form: see gemm_fp4.
extern "C" int q3_fp4_product(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out, int T,
                              int N, int K, long long ldc, int out_f32, int form, int* status, cudaStream_t stream) {
  return q3::fp4_product(x_codes, x_scales, w_codes, w_scales, out, T, N, K, ldc, out_f32, form, 0, status, stream);
}

// act(gate) * up as rows held in four bits: w's N = 2 I rows alternate gate/up in blocks of eight, the output has T rows of I.
extern "C" int q3_fp4_gated_product(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales,
                                    void* out_codes, void* out_scales, int T, int N, int K, int act, int form, int* status,
                                    cudaStream_t stream) {
  return q3::fp4_gated_product(x_codes, x_scales, w_codes, w_scales, out_codes, out_scales, T, N, K, act, form, 0, status, stream);
}

// A gated feed-forward behind its norm, in three launches: the norm's rows into h, the gated product into a, y = a w_down^T.  What
// runs before each product is the launch above it here, which writes neither product's w, so both may read theirs ahead of it; all
// that ran before this call is over when the norm's kernel lets the next one start.  (Before a product called by itself anything
// may have run, the kernel that writes its w included; there reading ahead gains nothing that could be measured.)  All three are
// checked before the first is launched: the norm may update the stream in place, and a call that refuses leaves it as it was.
extern "C" int q3_fp4_feed_forward(const float* stream_in, const void* delta, const float* norm, float* stream_out, float eps,
                                   const void* gu_codes, const void* gu_scales, const void* down_codes, const void* down_scales,
                                   void* h_codes, void* h_scales, void* a_codes, void* a_scales, void* y, int dtype, int T,
                                   int H, int I, int act, int* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (I <= 0 || I > (1 << 29)) return Q3_ERR_SIZE;
  int code = q3::fp4_gated_check(h_codes, h_scales, gu_codes, gu_scales, a_codes, a_scales, T, 2 * I, H, act);
  if (!code) code = q3::fp4_product_check(a_codes, a_scales, down_codes, down_scales, T, H, I, H);
  if (code) return code;
  code = q3_fp4_add_rmsnorm(stream_in, delta, dtype, norm, stream_out, h_codes, h_scales, T, H, eps, stream);
  if (code) return code;
  code = q3::fp4_gated_product(h_codes, h_scales, gu_codes, gu_scales, a_codes, a_scales, T, 2 * I, H, act, 0, 1, status, stream);
  if (code) return code;
  return q3::fp4_product(a_codes, a_scales, down_codes, down_scales, y, T, H, I, H, dtype == Q3_F32, 0, 1, status, stream);
}

// For the tests of the give-up path: see set_wait_test in tc_common.cuh.
extern "C" int q3_gemm_fp4_wait_test(unsigned limit, int drop) { return q3::set_wait_test(limit, drop); }
