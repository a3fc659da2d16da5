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

// Rows on 16-byte boundaries: read once, 8 elements a load, and kept in
// registers between the maximum and the rounding.
template <typename T, int CH>
__global__ void __launch_bounds__(CH <= 2 ? 256 : 1024)
    quantize_rows_kernel(const T *x, int64_t M, int K, int64_t ldx, int8_t *q, int Kp, float *scales) {
  __shared__ uint32_t sm[32];
  pdl_trigger();
  const int T_ = blockDim.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= M) return;  // blockDim.y > 1 only when a warp owns a row: no barrier is skipped
  x += row * ldx;
  q += row * Kp;
  float v[CH][8];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * T_ + threadIdx.x) * 8;
    if (i < K) {
      load<8>(x + i, v[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[c][j]));
    }
  }
  const RowScale rs = int8_row_scale(row_max_bits(top, T_ >> 5, sm));
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * T_ + threadIdx.x) * 8;
    if (i < K)
      *reinterpret_cast<uint2 *>(q + i) = make_uint2(int8_pack4(v[c], rs.inv), int8_pack4(v[c] + 4, rs.inv));
    else if (i < Kp)
      *reinterpret_cast<uint2 *>(q + i) = make_uint2(0, 0);
  }
  if (threadIdx.x == 0) scales[row] = rs.scale;
}

// Any alignment and length: a block a row, in two passes.
template <typename T>
__global__ void quantize_any_kernel(const T *x, int64_t K, int64_t ldx, int8_t *q, int64_t Kp, float *scales) {
  __shared__ uint32_t sm[32];
  pdl_trigger();
  const int64_t row = blockIdx.x;
  x += row * ldx;
  q += row * Kp;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x; i < K; i += blockDim.x) top = max(top, abs_bits(x[i]));
  const RowScale rs = int8_row_scale(row_max_bits(top, blockDim.x >> 5, sm));
  for (int64_t i = threadIdx.x; i < Kp; i += blockDim.x)
    q[i] = i < K ? (int8_t)int8_round((float)x[i], rs.inv) : (int8_t)0;
  if (threadIdx.x == 0) scales[row] = rs.scale;
}

template <typename T>
cudaError_t quantize_rows(const T *x, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scales, cudaStream_t st) {
  const int64_t Kp = int8_row_bytes(K);
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && ((uintptr_t)x & 15) == 0 && K <= 32768;
  if (!vec) {
    quantize_any_kernel<T><<<(unsigned)M, 256, 0, st>>>(x, K, ldx, q, Kp, scales);
    return cudaGetLastError();
  }
  const int CH = K <= 256 ? 1 : K <= 4096 ? 2 : 4;
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
      tile[j][tx] = n < N && k < K ? (int8_t)int8_round((float)w[k * N + n], rs.inv) : (int8_t)0;
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

template <typename TY>
__device__ __forceinline__ void finish(const Int8Args &a, TY *y, int acc, float s, float bias) {
  *y = from_f32<TY>(fmaf(__int2float_rn(acc), s, bias));
}

// Stages of operand tiles in flight: as many as fit 196 KB.
template <int BT>
constexpr int kStages = BT <= 64 ? 8 : BT == 128 ? 6 : 4;
template <int BT>
constexpr int kStageBytes = (BN + BT) * BK;
template <int BT>
constexpr size_t kSmem = (size_t)kStages<BT> * kStageBytes<BT> + 1024 + 256;

// Warp 0 loads (TMA, a ring of stages), warp 1 allocates TMEM and issues the
// MMAs, warps 4.. turn sums into results from one of two accumulators while
// the other fills.  Persistent over the tiles when `split` is 1.  With split =
// S > 1 a cluster of S CTAs shares one tile, each summing 1/S of K; the
// partial tiles meet in distributed shared memory, CTA r finishing the r-th
// part of the tokens: the grid then has a cluster for each tile.
//
// Under programmatic dependent launch (behind the kernel that rounds the
// tokens) the set-up and the first weight tiles do not wait for it.
template <int BT, typename TY>
__global__ void __launch_bounds__(384, 1)
    int8_tc_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mq, Int8Args a, int split,
                   int *err) {
  constexpr int STAGES = kStages<BT>, BYTES = kStageBytes<BT>, W_BYTES = BN * BK;
  constexpr uint32_t IDESC = i8_idesc(BN, BT);
  constexpr int COLS = 2 * BT;  // TMEM columns: two accumulators
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t *full = (uint64_t *)(smem + STAGES * BYTES), *empty = full + STAGES;
  uint64_t *tfull = empty + STAGES, *tempty = tfull + 2;
  uint32_t *tmem_slot = (uint32_t *)(tempty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int num_n = (a.N + BN - 1) / BN, num_t = (a.M + BT - 1) / BT;
  const int64_t tiles = (int64_t)num_n * num_t;
  const int first = blockIdx.x / split, step = gridDim.x / split;
  const int nkb = (a.K + BK - 1) / BK;
  const int kb0 = (int)((int64_t)nkb * rank / split), kb1 = (int)((int64_t)nkb * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t *)tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int64_t issued = 0;  // stages requested so far
      bool ok = true, waited = false;
      for (int64_t t = first; t < tiles && ok; t += step) {
        const int n0 = (int)(t % num_n) * BN, m0 = (int)(t / num_n) * BT;
        for (int kb = kb0; kb < kb1;) {
          // the weight tiles of as many stages as are free at the start; then one stage at a time
          const int burst = waited ? 1 : min(STAGES, kb1 - kb);
          for (int i = 0; i < burst && ok; ++i) {
            const int s = (int)((issued + i) % STAGES);
            ok = mbar_wait(&empty[s], (uint32_t)(((issued + i) / STAGES) & 1) ^ 1, err);
            if (!ok) break;
            mbar_expect_tx(&full[s], BYTES);
            tma_load_2d(smem + s * BYTES, &mw, &full[s], (kb + i) * BK, n0);
          }
          if (!ok) break;
          if (!waited) pdl_wait();  // the tokens
          waited = true;
          for (int i = 0; i < burst; ++i) {
            const int s = (int)((issued + i) % STAGES);
            tma_load_2d(smem + s * BYTES + W_BYTES, &mq, &full[s], (kb + i) * BK, m0);
          }
          kb += burst;
          issued += burst;
        }
      }
      // no copy may be in flight when the CTA leaves
      for (int64_t i = max((int64_t)0, issued - STAGES); i < issued; ++i)
        mbar_drain(&full[i % STAGES], (uint32_t)((i / STAGES) & 1));
    }
    __syncwarp();
  } else if (warp == 1) {
    int64_t used = 0;
    int i = 0;
    bool ok = true;
    for (int64_t t = first; t < tiles && ok; t += step, ++i) {
      const int buf = i & 1;
      if (!(ok = warp_wait(&tempty[buf], ((i >> 1) & 1) ^ 1, err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem + (uint32_t)(buf * BT);
      for (int kb = kb0; kb < kb1; ++kb, ++used) {
        const int s = (int)(used % STAGES);
        if (!(ok = warp_wait(&full[s], (uint32_t)((used / STAGES) & 1), err))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t dw = umma_desc(smem + s * BYTES), dq = umma_desc(smem + s * BYTES + W_BYTES);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          mma_i8(d, dw + 2 * k, dq + 2 * k, IDESC, (kb > kb0 || k) ? 1u : 0u);  // 32 bytes: 2 in descriptor units
        umma_commit_e(&empty[s]);
      }
      if (ok) umma_commit_e(&tfull[buf]);
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;  // TMEM lanes, columns
    constexpr int HALF = BT / 2 < 16 ? 16 : BT / 2;        // 16 columns leave the second warpgroup idle
    pdl_wait();                                            // the tokens' scales
    int i = 0;
    for (int64_t t = first; t < tiles; t += step, ++i) {
      const int buf = i & 1;
      const int n = (int)(t % num_n) * BN + quarter * 32 + lane, m0 = (int)(t / num_n) * BT;
      const bool in = n < a.N;
      const float sw = in ? a.w_scales[n] : 0.0f, bias = in && a.bias ? a.bias[n] : 0.0f;
      if (!warp_wait(&tfull[buf], (uint32_t)((i >> 1) & 1), err)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BT);
      for (int c = half * HALF; c < min((half + 1) * HALF, BT); c += 16) {
        int v[16];
        tmem_ld16(base + c, v);
        if (split == 1) {
          const int m = m0 + c;
          if (m >= a.M) break;
          const float sq = lane < 16 && m + lane < a.M ? a.q_scales[m + lane] : 0.0f;
          TY *y = (TY *)a.y + (int64_t)m * a.ldy + n;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float s = __shfl_sync(0xffffffffu, sq, j) * sw;
            if (in && m + j < a.M) finish(a, y + j * a.ldy, v[j], s, bias);
          }
        } else {  // over the operand ring, which is drained: every MMA that read it has completed
          int *part = reinterpret_cast<int *>(smem);
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c + j) * BN + quarter * 32 + lane] = v[j];
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
    cluster_sync();
    const int n0 = (first % num_n) * BN, m0 = (first / num_n) * BT;
    const int c0 = BT * rank / split, c1 = BT * (rank + 1) / split;
    const uint32_t mine = smem_u32(smem);
    for (int u = c0 * BN + threadIdx.x; u < c1 * BN; u += blockDim.x) {
      const int c = u / BN, n = n0 + u % BN, m = m0 + c;
      int acc = 0;
      for (int r = 0; r < split; ++r) {
        uint32_t at;
        int v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + 4u * (uint32_t)u), "r"(r));
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
        acc += v;
      }
      if (n < a.N && m < a.M)
        finish(a, (TY *)a.y + (int64_t)m * a.ldy + n, acc, a.q_scales[m] * a.w_scales[n], a.bias ? a.bias[n] : 0.0f);
    }
    cluster_sync();  // no CTA leaves while another reads its part
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
  }
}

cudaError_t row_map(CUtensorMap *map, const int8_t *p, int64_t rows, int K, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows}, strides[1] = {(uint64_t)int8_row_bytes(K)};
  const uint32_t box[2] = {BK, (uint32_t)box_rows};
  return tma_map_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p, dims, strides, box);
}

template <int BT, typename TY>
cudaError_t launch_tc(const Int8Args &a, int split, int sms, bool pdl, int *err, cudaStream_t st) {
  static thread_local int ready = -1;  // device whose kernel attributes are set
  auto *kernel = int8_tc_kernel<BT, TY>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && ready != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem<BT>);
    if (e == cudaSuccess) ready = dev;
  }
  CUtensorMap mq;
  if (e == cudaSuccess) e = row_map(&mq, a.q, a.M, a.K, BT);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)((a.N + BN - 1) / BN) * ((a.M + BT - 1) / BT);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(split > 1 ? tiles * split : std::min<int64_t>(tiles, sms)));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = kSmem<BT>;
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
  return cudaLaunchKernelEx(&cfg, kernel, *a.w_map, mq, a, split, err);
}

template <typename TY>
cudaError_t product(const Int8Args &a, bool pdl, int *err, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  const int num_n = (a.N + BN - 1) / BN, nkb = (a.K + BK - 1) / BK;
  // Tokens of a tile and CTAs that share one: the least estimated time, in
  // clocks of an SM that takes in about 64 bytes each from L2, which is what
  // binds: the waves of tiles, each the bytes of its stages and a start and end of
  // about 2,000 clocks, and as much again for the CTAs of a cluster to meet.
  int bt = 16, split = 1;
  int64_t best = INT64_MAX;
  for (int b = 256; b >= 16; b /= 2) {
    const int64_t tiles = (int64_t)num_n * ((a.M + b - 1) / b);
    for (int s = 1; s <= (b <= 128 ? 8 : 1) && s <= nkb && (s == 1 || tiles * s <= sms); s *= 2) {
      const int64_t waves = (tiles * s + sms - 1) / sms;
      const int64_t cost = waves * ((BN + b) * 2 * ((nkb + s - 1) / s)) + 2000 + (s > 1 ? 1000 + b * 16 / s : 0) + b * 8;
      if (cost < best) best = cost, bt = b, split = s;
    }
  }
  switch (bt) {
    case 16: return launch_tc<16, TY>(a, split, sms, pdl, err, st);
    case 32: return launch_tc<32, TY>(a, split, sms, pdl, err, st);
    case 64: return launch_tc<64, TY>(a, split, sms, pdl, err, st);
    case 128: return launch_tc<128, TY>(a, split, sms, pdl, err, st);
    default: return launch_tc<256, TY>(a, split, sms, pdl, err, st);
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

cudaError_t int8_matmul(const Int8Args &a, bool pdl, int *err, cudaStream_t st) {
  if (a.y_dtype == DT_F32) return product<float>(a, pdl, err, st);
  if (a.y_dtype == DT_F16) return product<__half>(a, pdl, err, st);
  return product<__nv_bfloat16>(a, pdl, err, st);
}

}  // namespace ndl
