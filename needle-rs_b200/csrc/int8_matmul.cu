// int8_matmul.cu — product of 8-bit integers with a scale for each token and
// each output channel, and the rounding of rows to 8 bits:
//   y[m][n] = (sum_k q[m][k] w[n][k]) * (sq[m] * sw[n]) + bias[n]
//
// The sums are exact: tcgen05.mma kind::i8 accumulates in 32-bit integers, so
// neither the split of K over CTAs nor its order changes a bit.
//
// Orientation.  The output channels take the 128 rows of the MMA (the lanes
// of TMEM) and BT tokens its columns: y^T = W q^T.  Both operands are stored
// with K contiguous, so either order feeds the tensor cores; this one pads
// few tokens to 16 columns instead of 128 rows, and in the epilogue a warp's
// lanes hold consecutive channels of one token, so it stores whole
// contiguous pieces of y without staging.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "ops.h"
#include "quant8.cuh"
#include "rowio.cuh"
#include "tc_common.cuh"
#include "tma_encode.h"

namespace ndl {
namespace {

using namespace tc;

// ── rounding to 8 bits ──────────────────────────────────────────────────────

template <typename T>
__device__ __forceinline__ uint32_t abs_bits(T v) {
  return __float_as_uint((float)v) & 0x7fffffffu;
}

// Largest |x| of a thread's vectors of 8, as the bits of an f32.  16-bit types
// compare as pairs of 16-bit integers: their bits without the sign order as the
// values do, infinities and NaN on top.
template <typename T>
struct TopOf {
  uint32_t top = 0;
  __device__ __forceinline__ void see(const uint4 *raw) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(raw);
#pragma unroll
    for (int j = 0; j < 2 * (int)sizeof(T); ++j)
      top = sizeof(T) == 4 ? max(top, w[j] & 0x7fffffffu) : __vmaxu2(top, w[j] & 0x7fff7fffu);
  }
  __device__ __forceinline__ uint32_t bits() const {
    if constexpr (sizeof(T) == 4) {
      return top;
    } else {
      const uint16_t h = (uint16_t)max(top & 0xffffu, top >> 16);
      return __float_as_uint((float)*reinterpret_cast<const T *>(&h));
    }
  }
};

// Rows on 16-byte boundaries: read once, 8 elements a load, and kept in
// registers between the maximum and the rounding.
template <typename T, int CH>
__global__ void __launch_bounds__(CH == 4 ? 1024 : 512)
    quantize_rows_kernel(const T *x, int64_t M, int K, int64_t ldx, int8_t *q, int Kp, float *scales) {
  __shared__ uint32_t sm[32];
  constexpr int V = sizeof(T) / 2;  // 16-byte pieces of 8 elements
  pdl_trigger();
  const int threads = blockDim.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= M) return;  // blockDim.y > 1 only when a warp owns a row: no barrier is skipped
  x += row * ldx;
  q += row * Kp;
  uint4 raw[CH][V];
  TopOf<T> top;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * threads + threadIdx.x) * 8;
    if (i < K) {
#pragma unroll
      for (int p = 0; p < V; ++p) raw[c][p] = reinterpret_cast<const uint4 *>(x + i)[p];
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if ((c * threads + (int)threadIdx.x) * 8 < K) top.see(raw[c]);
  const RowScale rs = int8_row_scale(row_max_bits(top.bits(), threads >> 5, sm));
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * threads + threadIdx.x) * 8;
    if (i < K) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)reinterpret_cast<const T *>(raw[c])[j];
      *reinterpret_cast<uint2 *>(q + i) = make_uint2(int8_pack4(v, rs.inv), int8_pack4(v + 4, rs.inv));
    } else if (i < Kp) {
      *reinterpret_cast<uint2 *>(q + i) = make_uint2(0, 0);
    }
  }
  if (threadIdx.x == 0) scales[row] = rs.scale;
}

// Rows at any alignment: a thread's columns are `threads` apart, so that a warp
// reads neighbours, and stay in registers; the values leave through shared memory
// in whole words.
template <typename T, int CH>
__global__ void __launch_bounds__(1024)
    quantize_any_kernel(const T *x, int64_t M, int K, int64_t ldx, int8_t *q, int Kp, float *scales) {
  extern __shared__ __align__(16) int8_t line[];  // [rows of the block][Kp]
  __shared__ uint32_t sm[32];
  pdl_trigger();
  const int threads = blockDim.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= M) return;  // blockDim.y > 1 only when a warp owns a row: no barrier is skipped
  x += row * ldx;
  T v[CH];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c * threads + (int)threadIdx.x < K) v[c] = x[c * threads + threadIdx.x];
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c * threads + (int)threadIdx.x < K) top = max(top, abs_bits(v[c]));
  const RowScale rs = int8_row_scale(row_max_bits(top, threads >> 5, sm));
  int8_t *mine = line + threadIdx.y * Kp;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * threads + threadIdx.x;
    if (i < K) mine[i] = int8_round((float)v[c], rs.inv);
  }
  if (threadIdx.x < Kp - K) mine[K + threadIdx.x] = 0;
  if (threads > 32)
    __syncthreads();
  else
    __syncwarp();
  uint32_t *out = reinterpret_cast<uint32_t *>(q + row * Kp);
  for (int i = threadIdx.x; i < Kp / 4; i += threads) out[i] = reinterpret_cast<const uint32_t *>(mine)[i];
  if (threadIdx.x == 0) scales[row] = rs.scale;
}

// Any length: a block a row, in two passes.
template <typename T>
__global__ void quantize_long_kernel(const T *x, int64_t K, int64_t ldx, int8_t *q, int64_t Kp, float *scales) {
  __shared__ uint32_t sm[32];
  pdl_trigger();
  const int64_t row = blockIdx.x;
  x += row * ldx;
  q += row * Kp;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x; i < K; i += blockDim.x) top = max(top, abs_bits(x[i]));
  const RowScale rs = int8_row_scale(row_max_bits(top, blockDim.x >> 5, sm));
  for (int64_t i = threadIdx.x; i < Kp; i += blockDim.x)
    q[i] = i < K ? int8_round((float)x[i], rs.inv) : (int8_t)0;
  if (threadIdx.x == 0) scales[row] = rs.scale;
}

template <typename T>
cudaError_t quantize_rows(const T *x, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scales, cudaStream_t st) {
  const int64_t Kp = int8_row_bytes(K);
  if (K > 32768) {
    quantize_long_kernel<T><<<(unsigned)M, 1024, 0, st>>>(x, K, ldx, q, Kp, scales);
    return cudaGetLastError();
  }
  if (K % 8 || ldx % 8 || ((uintptr_t)x & 15)) {
    // 16 columns a thread, 32 above 16,384
    const int each = K <= 16384 ? 16 : 32, threads = (int)((K + each - 1) / each + 31) / 32 * 32, rows = threads == 32 ? 8 : 1;
    const unsigned grid = (unsigned)((M + rows - 1) / rows);
    if (each == 16)
      quantize_any_kernel<T, 16><<<grid, dim3(threads, rows), rows * Kp, st>>>(x, M, (int)K, ldx, q, (int)Kp, scales);
    else
      quantize_any_kernel<T, 32><<<grid, dim3(threads, rows), rows * Kp, st>>>(x, M, (int)K, ldx, q, (int)Kp, scales);
    return cudaGetLastError();
  }
  // A row's reductions and two divisions are the same work for every thread: 32
  // elements a thread from 512 on (8192 x 4096 bf16: 28.6 us with 8 a thread, 21.0 with 16,
  // 18.6 with 32; 16384 x 4096 f32: 51 us, the copy rate.  Persistent blocks that
  // fetch rows ahead took 19.1 and 87 us.)
  const int CH = K <= 256 ? 1 : K <= 512 ? 2 : 4;
  const int threads = (int)((Kp + 8 * CH - 1) / (8 * CH) + 31) / 32 * 32, rows = threads == 32 ? 8 : 1;
  const unsigned grid = (unsigned)((M + rows - 1) / rows);
  const dim3 block(threads, rows);
  if (CH == 1)
    quantize_rows_kernel<T, 1><<<grid, block, 0, st>>>(x, M, (int)K, ldx, q, (int)Kp, scales);
  else if (CH == 2)
    quantize_rows_kernel<T, 2><<<grid, block, 0, st>>>(x, M, (int)K, ldx, q, (int)Kp, scales);
  else
    quantize_rows_kernel<T, 4><<<grid, block, 0, st>>>(x, M, (int)K, ldx, q, (int)Kp, scales);
  return cudaGetLastError();
}

// w[K][N] -> data[N][Kp]: a block owns 32 columns; 32 x 32 tiles are turned
// in shared memory so that both sides move whole rows.
template <typename T>
__global__ void quantize_cols_kernel(const T *w, int64_t K, int64_t N, int8_t *data, int64_t Kp, float *scales) {
  __shared__ uint32_t tops[8][32];
  __shared__ int8_t tile[32][33];
  const int tx = threadIdx.x, ty = threadIdx.y;
  const int64_t n = (int64_t)blockIdx.x * 32 + tx;
  uint32_t top = 0;
  if (n < N)
    for (int64_t k = ty; k < K; k += 8) top = max(top, abs_bits(w[k * N + n]));
  tops[ty][tx] = top;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, tops[j][tx]);
  const RowScale rs = int8_row_scale(top);
  if (ty == 0 && n < N) scales[n] = rs.scale;
  for (int64_t k0 = 0; k0 < Kp; k0 += 32) {
    for (int j = ty; j < 32; j += 8) {
      const int64_t k = k0 + j;
      tile[j][tx] = n < N && k < K ? int8_round((float)w[k * N + n], rs.inv) : (int8_t)0;
    }
    __syncthreads();
    for (int j = ty; j < 32; j += 8) {
      const int64_t row = (int64_t)blockIdx.x * 32 + j, k = k0 + tx;
      if (row < N && k < Kp) data[row * Kp + k] = tile[tx][j];
    }
    __syncthreads();
  }
}

// ── the product ─────────────────────────────────────────────────────────────

constexpr int BN = 128, BK = 128;  // output channels of a tile, bytes of K in a stage

// tcgen05.mma kind::i8: signed 8-bit operands, both K-major, 32-bit sums; 32
// bytes of K an instruction.
__host__ __device__ constexpr uint32_t i8_idesc(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// The same over a CTA pair: rows of A and of B split between the CTAs' shared
// memory at the same offsets, rows of D between their TMEM.
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// 16 columns of this warp's TMEM lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// y = sum * scale + bias, rounded once to the type.
template <typename TY>
__device__ __forceinline__ void finish(TY *y, int acc, float s, float bias) {
  *y = from_f32<TY>(fmaf(__int2float_rn(acc), s, bias));
}

// Scales of the NC tokens from m0 on: lane l holds tokens l, l + 32, ...
template <int NC>
__device__ __forceinline__ void token_scales(const float *scales, int m0, int M, int lane, float *sq) {
#pragma unroll
  for (int q = 0; q < (NC + 31) / 32; ++q) {
    const int m = m0 + 32 * q + lane;
    sq[q] = 32 * q + lane < NC && m < M ? scales[m] : 0.0f;
  }
}

// Results of NC tokens from m0 on and this lane's channel n, from NC columns of its
// TMEM lane.
template <int NC, typename TY>
__device__ __forceinline__ void store_tokens(const Int8Args &a, uint32_t taddr, int m0, int n, float sw, float bias,
                                             const float *sq) {
  const int left = a.M - m0;
  const bool in = n < a.N;
  TY *y = (TY *)a.y + (int64_t)m0 * a.ldy + n;
#pragma unroll
  for (int c = 0; c < NC; c += 16) {
    if (c >= left) break;
    __syncwarp();  // channels past the last stored nothing; TMEM is read by whole warps
    int v[16];
    tmem_ld16(taddr + c, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float s = __shfl_sync(0xffffffffu, sq[c >> 5], (c & 31) + j) * sw;
      if (in && c + j < left) finish(y, v[j], s, bias);
      y += a.ldy;
    }
  }
}

// Stages of operand tiles in flight: as many as fit 196 KB.  The fused form holds
// only weights in its ring, and the tokens of all of its K beside it.
template <int BT, bool FUSED>
constexpr int kStages = FUSED ? 7 : BT <= 64 ? 8 : BT == 128 ? 6 : 4;
template <int BT, bool FUSED>
constexpr int kStageBytes = (BN + (FUSED ? 0 : BT)) * BK;
constexpr int kFusedBlocks = 32;  // blocks of K of the most values that a kernel rounds itself
template <int BT, bool FUSED>
constexpr size_t kSmem = (size_t)kStages<BT, FUSED> * kStageBytes<BT, FUSED> + (FUSED ? kFusedBlocks * 16 * BK : 0) + 1024 + 512;

// 8 elements of a row from k on, as f32, zero past K.
__device__ __forceinline__ void load8(const Int8Args &a, int64_t row, int k, float *v) {
  const int64_t at = row * a.ldx + k;
  if (a.x_vec && k + 8 <= a.K) {
    if (a.x_dtype == DT_F32)
      load<8>((const float *)a.x + at, v);
    else if (a.x_dtype == DT_F16)
      load<8>((const __half *)a.x + at, v);
    else
      load<8>((const __nv_bfloat16 *)a.x + at, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = 0.0f;
    if (k + j < a.K)
      v[j] = a.x_dtype == DT_F32   ? ((const float *)a.x)[at + j]
             : a.x_dtype == DT_F16 ? (float)((const __half *)a.x)[at + j]
                                   : (float)((const __nv_bfloat16 *)a.x)[at + j];
  }
}

// Warp 0 loads (TMA, a ring of stages), warp 1 allocates TMEM and issues the
// MMAs, warps 4.. turn sums into results from one of two accumulators while
// the other fills.  Persistent over the tiles when `split` is 1.  With split =
// S > 1 a cluster of S CTAs shares one tile, each summing 1/S of K; the
// partial tiles meet in distributed shared memory, CTA r finishing the r-th
// part of the tokens: the grid then has a cluster for each tile.
//
// Small products are a chain of latencies, so nothing waits that need not: the
// thread that initialises the barriers requests the first weight tiles at once,
// before TMEM is allocated and before the kernel that rounds the tokens is done
// (programmatic dependent launch), and scales and biases are fetched before the sums.
//
// FUSED (up to 16 tokens): no such kernel.  Every CTA finds the rows' maxima
// itself and rounds its part of K into the MMA's operand layout while its
// weights arrive: the values are few enough to be read by every CTA, and a
// launch costs more (1 x 512 x 2048: 6.1 us, rounded by a launch before it 8.2).
//
// Bound by latency and then by the weights' bytes: 64 x 4096 x 4096 takes 10.3 us with the
// rounding of its tokens (13.3 with weights requested after TMEM and scales after the
// sums, 17.7 without the split by estimate), its 16.8 MB alone 2.6 at the copy rate.
template <int BT, typename TY, bool FUSED>
__global__ void __launch_bounds__(384, 1)
    int8_tc_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mq, Int8Args a, int lg,
                   int *err) {
  constexpr int STAGES = kStages<BT, FUSED>, BYTES = kStageBytes<BT, FUSED>, W_BYTES = BN * BK;
  constexpr uint32_t IDESC = i8_idesc(BN, BT);
  constexpr int COLS = 2 * BT;  // TMEM columns: two accumulators
  constexpr int HALF = BT / 2 < 16 ? 16 : BT / 2;  // tokens of an epilogue warpgroup (16: the second has none)
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *tokens = smem + STAGES * BYTES;  // FUSED: [block of K][16 rows][128 bytes]
  uint64_t *full = (uint64_t *)(tokens + (FUSED ? kFusedBlocks * 16 * BK : 0)), *empty = full + STAGES;
  uint64_t *tfull = empty + STAGES, *tempty = tfull + 2;
  uint64_t *done = tempty + 2;  // of MMAs in flight, after a wait that ran out
  uint32_t *tmem_slot = (uint32_t *)(done + 1), *tops = tmem_slot + 2;  // tops: [12 warps]
  float *scales = (float *)(tops + 12);                                   // FUSED: [16]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = 1 << lg, rank = lg ? (int)cluster_ctarank() : 0;
  const int num_n = (a.N + BN - 1) / BN, num_t = (a.M + BT - 1) / BT;
  const int tiles = num_n * num_t;
  const int first = (int)blockIdx.x >> lg, step = (int)gridDim.x >> lg;
  const int nkb = (a.K + BK - 1) / BK;
  const int kb0 = (nkb * rank) >> lg, kb1 = (nkb * (rank + 1)) >> lg;
  const int burst = min(STAGES, kb1 - kb0);

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mw) : "memory");
    if (!FUSED) asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    for (int i = 0; i < burst; ++i) {
      mbar_expect_tx(&full[i], BYTES);
      tma_load_2d(smem + i * BYTES, &mw, &full[i], (kb0 + i) * BK, (first % num_n) * BN);
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  __syncwarp();
  if (FUSED) {
    // the rows' maxima: a row by as many warps as there are for each
    const int wpr = max(1, 12 / a.M), groups = 12 / wpr, group = warp / wpr;
    for (int r0 = 0; r0 < a.M; r0 += groups) {
      const int r = r0 + group;
      uint32_t top = 0;
      if (group < groups && r < a.M)
        for (int k = (warp % wpr * 32 + lane) * 8; k < a.K; k += wpr * 256) {
          float v[8];
          load8(a, r, k, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) tops[warp] = top;
      __syncthreads();
      if (threadIdx.x < groups && r0 + (int)threadIdx.x < a.M) {
        uint32_t t = 0;
        for (int i = 0; i < wpr; ++i) t = max(t, tops[threadIdx.x * wpr + i]);
        const RowScale rs = int8_row_scale(t);
        scales[r0 + threadIdx.x] = rs.scale;
        scales[16 + r0 + threadIdx.x] = rs.inv;
      }
      __syncthreads();
    }
    // this CTA's part of K in the swizzled layout; the rows past M hold anything,
    // which reaches no token that is stored
    const int blocks = kb1 - kb0;
    for (int i = threadIdx.x; i < a.M * blocks * (BK / 8); i += blockDim.x) {  // 8 values: chunk c % 16 of a row's block
      const int c = i % (BK / 8), r = i / (BK / 8) % a.M, block = i / (BK / 8) / a.M;
      float v[8];
      load8(a, r, (kb0 + block) * BK + c * 8, v);
      const float inv = scales[16 + r];
      *reinterpret_cast<uint2 *>(tokens + block * 16 * BK + r * BK + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8) =
          make_uint2(int8_pack4(v, inv), int8_pack4(v + 4, inv));
    }
    fence_async_smem();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t *)tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      if (!FUSED) {
        pdl_wait();  // the tokens
        for (int i = 0; i < burst; ++i)
          tma_load_2d(smem + i * BYTES + W_BYTES, &mq, &full[i], (kb0 + i) * BK, (first / num_n) * BT);
      }
      int s = burst == STAGES ? 0 : burst, issued = burst;  // issued: up to STAGES
      uint32_t ph = burst == STAGES ? 1 : 0;
      int kb = kb0 + burst;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step, kb = kb0) {
        const int n0 = t % num_n * BN, m0 = t / num_n * BT;
        for (; kb < kb1; ++kb) {
          if (!(ok = mbar_wait(&empty[s], ph ^ 1, err))) break;
          mbar_expect_tx(&full[s], BYTES);
          tma_load_2d(smem + s * BYTES, &mw, &full[s], kb * BK, n0);
          if (!FUSED) tma_load_2d(smem + s * BYTES + W_BYTES, &mq, &full[s], kb * BK, m0);
          issued = min(issued + 1, STAGES);
          if (++s == STAGES) s = 0, ph ^= 1;
        }
      }
      // no copy may be in flight when the CTA leaves
      for (int i = 0; i < issued; ++i) {
        if (s-- == 0) s = STAGES - 1, ph ^= 1;
        mbar_drain(&full[s], ph);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    int s = 0, i = 0;
    uint32_t ph = 0;
    bool ok = true;
    // descriptors: a common high word, the address / 16 in the low one (a block
    // of 16 tokens is 16 * BK / 16 = BK units)
    const uint64_t hi = umma_desc(smem) & 0xFFFFFFFF00000000ull;
    const uint32_t w16 = (smem_u32(smem) >> 4) | (1u << 16), t16 = (smem_u32(tokens) >> 4) | (1u << 16);
    for (int t = first; t < tiles && ok; t += step, ++i) {
      const int buf = i & 1;
      if (i >= 2 && !(ok = warp_wait(&tempty[buf], ((i >> 1) & 1) ^ 1, err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem + (uint32_t)(buf * BT);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = warp_wait(&full[s], ph, err))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t dw = w16 + (uint32_t)(s * (BYTES >> 4)), dq = FUSED ? t16 + (uint32_t)((kb - kb0) * BK) : dw + (W_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          mma_i8(d, hi | (dw + 2 * k), hi | (dq + 2 * k), IDESC, (kb > kb0 || k) ? 1u : 0u);  // 32 bytes: 2 units
        umma_commit_e(&empty[s]);
        if (++s == STAGES) s = 0, ph ^= 1;
      }
      if (ok) umma_commit_e(&tfull[buf]);
    }
    if (!ok) {
      umma_commit_e(done);
      mbar_drain(done, 0);
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;  // TMEM lanes, tokens
    if (!FUSED) pdl_wait();                                // the tokens' scales
    int i = 0;
    for (int t = first; t < tiles; t += step, ++i) {
      const int buf = i & 1;
      const int n = t % num_n * BN + quarter * 32 + lane, m0 = t / num_n * BT + half * HALF;
      const bool in = n < a.N;
      const float sw = in ? a.w_scales[n] : 0.0f, bias = in && a.bias ? a.bias[n] : 0.0f;
      float sq[(HALF + 31) / 32];
      token_scales<HALF>(FUSED ? scales : a.q_scales, m0, a.M, lane, sq);
      if (!warp_wait(&tfull[buf], (uint32_t)((i >> 1) & 1), err)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BT + half * HALF);
      if (half * HALF >= BT) {
      } else if (split == 1) {
        store_tokens<HALF, TY>(a, base, m0, n, sw, bias, sq);
      } else {  // over the operand ring, which is drained: every MMA that read it has completed
#pragma unroll
        for (int c = 0; c < HALF; c += 16) {
          int v[16];
          tmem_ld16(base + c, v);
          int *part = reinterpret_cast<int *>(smem) + (half * HALF + c) * BN + quarter * 32 + lane;
#pragma unroll
          for (int j = 0; j < 16; ++j) part[j * BN] = v[j];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (split > 1) {
    // this CTA's tokens of the tile: 4 channels a thread, all CTAs' parts at once
    const int n0 = (first % num_n) * BN, m0 = (first / num_n) * BT;
    const int c0 = (BT * rank) >> lg, units = (BT >> lg) * (BN / 4);
    const uint32_t mine = smem_u32(smem);
    const int in = (int)threadIdx.x % (BN / 4) * 4, n = n0 + in;  // the same channels in every turn
    float sw[4], bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sw[j] = n + j < a.N ? a.w_scales[n + j] : 0.0f;
      bias[j] = n + j < a.N && a.bias ? a.bias[n + j] : 0.0f;
    }
    __syncwarp();
    cluster_sync();
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      const int c = c0 + u / (BN / 4), m = m0 + c;
      if (m >= a.M) break;  // the later units are of later tokens
      const float sq = FUSED ? scales[m] : a.q_scales[m];
      int4 part[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < split) {
          uint32_t at;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + 4u * (uint32_t)(c * BN + in)), "r"(r));
          asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(part[r].x), "=r"(part[r].y), "=r"(part[r].z), "=r"(part[r].w)
                       : "r"(at)
                       : "memory");
        }
      int4 acc = part[0];
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < split) acc.x += part[r].x, acc.y += part[r].y, acc.z += part[r].z, acc.w += part[r].w;
      const int sums[4] = {acc.x, acc.y, acc.z, acc.w};
      TY *y = (TY *)a.y + (int64_t)m * a.ldy + n;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) finish(y + j, sums[j], sq * sw[j], bias[j]);
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while another reads its part
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
  }
}

// Many tokens: a cluster of two CTAs computes 256 channels x 256 tokens with
// tcgen05.mma.cta_group::2 M256 N256.  Each CTA loads its own 128 channels and
// its own 128 tokens (32 KB a stage of 128 bytes of K); the leader's MMAs read both
// CTAs' tiles and leave each its 128 channels' sums of all 256 tokens.  A stage is
// 512 clocks of MMA and 512 of L2 intake at 64 bytes a clock; one CTA alone
// takes in 768 for 128 channels x 256 tokens.  8192 x 4096 x 4096: 87 us, 3.15 POP/s, 0.93
// of twice the measured bf16 rate, the tensor pipe busy 88% of the time that SMs run; with the
// rounding of the tokens 128 us where one CTA's tiles took 138.
// Synchronisation: both CTAs' loads complete on the leader's `full`; an
// MMA's completion is signalled to both CTAs' `empty` and `tfull`; both CTAs' epilogue
// warps arrive on the leader's `tempty`.  After a wait that ran out the leader waits for
// the copies that either CTA has in flight: `asked` tells it how far both came.
constexpr int kPairStages = 6, kPairBytes = 2 * BN * BK;
constexpr size_t kPairSmem = (size_t)kPairStages * kPairBytes + 1024 + 256;

template <typename TY>
__global__ void __launch_bounds__(384, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mq, Int8Args a, int *err) {
  constexpr int STAGES = kPairStages, W_BYTES = BN * BK, BT = 256, HALF = 128;
  constexpr uint32_t IDESC = i8_idesc(2 * BN, BT);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t *full = (uint64_t *)(smem + STAGES * kPairBytes), *empty = full + STAGES;
  uint64_t *tfull = empty + STAGES, *tempty = tfull + 2;
  uint64_t *done = tempty + 2;  // of MMAs in flight, after a wait that ran out
  uint32_t *tmem_slot = (uint32_t *)(done + 1);
  uint32_t *asked = tmem_slot + 2;  // of each CTA: stages requested * 2, and 1 if a wait of its loader ran out

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank(), pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  const int num_n = (a.N + 2 * BN - 1) / (2 * BN), num_t = (a.M + BT - 1) / BT, tiles = num_n * num_t;
  const int nkb = (a.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mw) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2 * BT));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before either is signalled
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t *)tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();  // the tokens
      int s = 0;
      uint32_t ph = 0, requested = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int n0 = t % num_n * 2 * BN + rank * BN, m0 = t / num_n * BT + rank * BN;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!(ok = mbar_wait(&empty[s], ph ^ 1, err))) break;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * kPairBytes);  // both CTAs' bytes
          const uint32_t fb = pair_leader_addr(&full[s]);
          tma_load_2d_pair(smem + s * kPairBytes, &mw, fb, kb * BK, n0);
          tma_load_2d_pair(smem + s * kPairBytes + W_BYTES, &mq, fb, kb * BK, m0);
          ++requested;
          if (++s == STAGES) s = 0, ph ^= 1;
        }
      }
      // every requested stage has been multiplied before the CTA leaves
      for (int i = 0; i < STAGES && ok; ++i) {
        ok = mbar_wait(&empty[s], ph ^ 1, err);
        if (++s == STAGES) s = 0, ph ^= 1;
      }
      for (uint32_t r = 0; r < 2; ++r) store_cluster(&asked[rank], r, requested << 1 | (ok ? 0u : 1u));
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    int s = 0, i = 0;
    uint32_t ph = 0;
    bool ok = true;
    const uint64_t hi = umma_desc(smem) & 0xFFFFFFFF00000000ull;
    const uint32_t w16 = (smem_u32(smem) >> 4) | (1u << 16);
    for (int t = pair; t < tiles && ok; t += pairs, ++i) {
      const int buf = i & 1;
      if (i >= 2 && !(ok = warp_wait(&tempty[buf], ((i >> 1) & 1) ^ 1, err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem + (uint32_t)(buf * BT);
      for (int kb = 0; kb < nkb; ++kb) {
        if (!(ok = warp_wait(&full[s], ph, err))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t dw = w16 + (uint32_t)(s * (kPairBytes >> 4)), dq = dw + (W_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k) mma_i8_pair(d, hi | (dw + 2 * k), hi | (dq + 2 * k), IDESC, (kb | k) ? 1u : 0u);
        umma_commit_pair_e(&empty[s]);
        if (++s == STAGES) s = 0, ph ^= 1;
      }
      if (ok) umma_commit_pair_e(&tfull[buf]);
    }
    if (!ok) {
      umma_commit_pair_e(done);
      mbar_drain(done, 0);
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    pdl_wait();  // the tokens' scales
    int i = 0;
    for (int t = pair; t < tiles; t += pairs, ++i) {
      const int buf = i & 1;
      const int n = t % num_n * 2 * BN + rank * BN + quarter * 32 + lane, m0 = t / num_n * BT + half * HALF;
      const float sw = n < a.N ? a.w_scales[n] : 0.0f, bias = n < a.N && a.bias ? a.bias[n] : 0.0f;
      float sq[HALF / 32];
      token_scales<HALF>(a.q_scales, m0, a.M, lane, sq);
      if (!warp_wait(&tfull[buf], (uint32_t)((i >> 1) & 1), err)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      store_tokens<HALF, TY>(a, tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BT + half * HALF), m0, n, sw, bias,
                             sq);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(&tempty[buf], 0);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // no arrive or MMA reaches a CTA that has left
  if ((asked[0] | asked[1]) & 1u) {  // the same in both CTAs
    if (rank == 0 && threadIdx.x == 0) {
      // The stages from `both` on were requested by one CTA alone.  Where that is the
      // leader, `full` was told to expect the other's bytes too: it copies once more in its place.
      const uint32_t n0 = asked[0] >> 1, n1 = asked[1] >> 1, most = max(n0, n1), both = min(n0, n1);
      for (uint32_t k = most > STAGES ? most - STAGES : 0; k < most; ++k) {
        const int s = (int)(k % STAGES);
        if (k >= both && n1 > n0) mbar_expect_tx(&full[s], kPairBytes);
        if (k >= both && n0 > n1) {
          const uint32_t fb = pair_leader_addr(&full[s]);
          tma_load_2d_pair(smem + s * kPairBytes, &mw, fb, 0, 0);
          tma_load_2d_pair(smem + s * kPairBytes + W_BYTES, &mq, fb, 0, 0);
        }
        mbar_drain(&full[s], k / STAGES & 1);
      }
    }
    __syncthreads();
    cluster_sync();  // no copy is in flight when a CTA leaves
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BT));
  }
}

cudaError_t row_map(CUtensorMap *map, const int8_t *p, int64_t rows, int K, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows}, strides[1] = {(uint64_t)int8_row_bytes(K)};
  const uint32_t box[2] = {BK, (uint32_t)box_rows};
  return tma_map_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p, dims, strides, box);
}

template <int BT, typename TY, bool FUSED>
cudaError_t launch_tc(const Int8Args &a, int lg, int sms, bool pdl, int *err, cudaStream_t st) {
  static thread_local int ready = -1;  // device whose kernel attributes are set
  auto *kernel = int8_tc_kernel<BT, TY, FUSED>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && ready != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem<BT, FUSED>);
    if (e == cudaSuccess) ready = dev;
  }
  CUtensorMap mq = *a.w_map;
  if (e == cudaSuccess && !FUSED) e = row_map(&mq, a.q, a.M, a.K, BT);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)((a.N + BN - 1) / BN) * ((a.M + BT - 1) / BT);
  cudaLaunchConfig_t cfg = {};
  const int split = 1 << lg;
  cfg.gridDim = dim3((unsigned)(split > 1 ? tiles * split : std::min<int64_t>(tiles, sms)));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = kSmem<BT, FUSED>;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  if (split > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs++].val.clusterDim = {(unsigned)split, 1, 1};
  }
  if (pdl) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  return cudaLaunchKernelEx(&cfg, kernel, *a.w_map, mq, a, lg, err);
}

template <typename TY>
cudaError_t launch_pair(const Int8Args &a, int sms, bool pdl, int *err, cudaStream_t st) {
  static thread_local int ready = -1;
  auto *kernel = int8_pair_kernel<TY>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && ready != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem);
    if (e == cudaSuccess) ready = dev;
  }
  CUtensorMap mq;
  if (e == cudaSuccess) e = row_map(&mq, a.q, a.M, a.K, BN);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)((a.N + 2 * BN - 1) / (2 * BN)) * ((a.M + 255) / 256);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, sms / 2)));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {2, 1, 1};
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, *a.w_map, mq, a, err);
}

// Clusters of 2^lg CTAs that run at once on the current device: fewer than its SMs
// would hold, since a cluster stays within one of their groups (15 of 8 CTAs on 148 SMs; a
// sixteenth waits for a second round: 64 x 2048 x 2048 14.5 us, split by four instead 8.6).
cudaError_t clusters_at_once(int dev, int sms, int *fit) {
  static thread_local int last_dev = -1, last[4];
  if (last_dev != dev) {
    auto *kernel = int8_tc_kernel<16, float, false>;  // as the others, a CTA an SM
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem<16, false>);
    for (int lg = 0; lg < 4 && e == cudaSuccess; ++lg) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(sms >> lg << lg));
      cfg.blockDim = dim3(384);
      cfg.dynamicSmemBytes = kSmem<16, false>;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim = {1u << lg, 1, 1};
      cfg.attrs = at;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&last[lg], kernel, &cfg);
    }
    if (e != cudaSuccess) return e;
    last_dev = dev;
  }
  for (int lg = 0; lg < 4; ++lg) fit[lg] = last[lg];
  return cudaSuccess;
}

// Tokens of a tile and CTAs that share one: the least estimated time, in
// clocks of an SM that takes in about 64 bytes each from L2, which is what
// binds: the waves of tiles, each the bytes of its stages and a start and end of
// about 2,000 clocks, and as much again for the CTAs of a cluster to meet.
// A CTA pair's tile of 256 channels x 256 tokens (bt 512) takes in 512 clocks a
// stage instead of the 768 of one CTA's 128 x 256.
struct Shape {
  int bt, lg;  // tokens (512: a pair's tile), log2 of the CTAs
};
Shape choose_shape(int M, int N, int K, int sms, const int *fit) {
  const int num_n = (N + BN - 1) / BN, nkb = (K + BK - 1) / BK;
  Shape best{16, 0};
  int64_t least = INT64_MAX;
  for (int b = 256; b >= 16; b /= 2) {
    const int64_t tiles = (int64_t)num_n * ((M + b - 1) / b);
    for (int lg = 0; lg <= (b <= 128 ? 3 : 0); ++lg) {
      const int s = 1 << lg;
      if (lg && (s > nkb || tiles > fit[lg])) break;
      const int64_t waves = (tiles * s + sms - 1) / sms;
      const int64_t cost = waves * ((BN + b) * 2 * ((nkb + s - 1) / s)) + 2000 + (s > 1 ? 1000 + b * 16 / s : 0) + b * 8;
      if (cost < least) least = cost, best = Shape{b, lg};
    }
  }
  const int64_t pair_tiles = (int64_t)((N + 2 * BN - 1) / (2 * BN)) * ((M + 255) / 256);
  const int64_t cost = (pair_tiles + sms / 2 - 1) / (sms / 2) * (2 * BN * 2 * nkb) + 4000 + 256 * 8;
  if (cost < least) best = Shape{512, 0};
  return best;
}

// Whether a product of unrounded tokens takes the fused kernel: one tile of up to 16
// tokens, 4,096 values in all (fused and with a launch to round them, us, bf16: 8 x 512 x 512
// 6.3 and 8.0, 1 x 4096 x 4096 8.6 and 9.0, 16 x 512 x 512 8.3 and 8.0, 4 x 2048 x 2048 14.0
// and 12.2, 16 x 2048 x 2048 22.6 and 12.4: every CTA reads all of them).
bool fuses(const Shape &sh, int M, int K) { return sh.bt == 16 && M <= 16 && (int64_t)M * K <= kFusedBlocks * BK; }

template <typename TY>
cudaError_t product(const Int8Args &a, bool pdl, int *err, cudaStream_t st) {
  int dev = 0, sms = 0, fit[4];
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = clusters_at_once(dev, sms, fit);
  if (e != cudaSuccess) return e;
  const Shape sh = choose_shape(a.M, a.N, a.K, sms, fit);
  switch (sh.bt) {
    case 16:
      return a.x ? launch_tc<16, TY, true>(a, sh.lg, sms, false, err, st)
                 : launch_tc<16, TY, false>(a, sh.lg, sms, pdl, err, st);
    case 32: return launch_tc<32, TY, false>(a, sh.lg, sms, pdl, err, st);
    case 64: return launch_tc<64, TY, false>(a, sh.lg, sms, pdl, err, st);
    case 128: return launch_tc<128, TY, false>(a, sh.lg, sms, pdl, err, st);
    case 512: return launch_pair<TY>(a, sms, pdl, err, st);
    default: return launch_tc<256, TY, false>(a, sh.lg, sms, pdl, err, st);
  }
}

}  // namespace

cudaError_t int8_quantize_rows(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scales,
                               cudaStream_t st) {
  if (dtype == DT_F32) return quantize_rows((const float *)x, M, K, ldx, q, scales, st);
  if (dtype == DT_F16) return quantize_rows((const __half *)x, M, K, ldx, q, scales, st);
  return quantize_rows((const __nv_bfloat16 *)x, M, K, ldx, q, scales, st);
}

cudaError_t int8_quantize_cols(const void *w, int dtype, int64_t K, int64_t N, int8_t *data, float *scales,
                               cudaStream_t st) {
  const int64_t Kp = int8_row_bytes(K);
  const unsigned grid = (unsigned)((N + 31) / 32);
  const dim3 block(32, 8);
  if (dtype == DT_F32)
    quantize_cols_kernel<<<grid, block, 0, st>>>((const float *)w, K, N, data, Kp, scales);
  else if (dtype == DT_F16)
    quantize_cols_kernel<<<grid, block, 0, st>>>((const __half *)w, K, N, data, Kp, scales);
  else
    quantize_cols_kernel<<<grid, block, 0, st>>>((const __nv_bfloat16 *)w, K, N, data, Kp, scales);
  return cudaGetLastError();
}

cudaError_t int8_weight_map(CUtensorMap *map, const int8_t *w, int64_t N, int K) { return row_map(map, w, N, K, BN); }

bool int8_matmul_fuses(int M, int N, int K) {
  int dev = 0, sms = 0, fit[4];
  return cudaGetDevice(&dev) == cudaSuccess &&
         cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
         clusters_at_once(dev, sms, fit) == cudaSuccess && fuses(choose_shape(M, N, K, sms, fit), M, K);
}

cudaError_t int8_matmul(const Int8Args &a, bool pdl, int *err, cudaStream_t st) {
  if (a.y_dtype == DT_F32) return product<float>(a, pdl, err, st);
  if (a.y_dtype == DT_F16) return product<__half>(a, pdl, err, st);
  return product<__nv_bfloat16>(a, pdl, err, st);
}

}  // namespace ndl
