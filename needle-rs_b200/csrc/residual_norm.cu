// residual_norm.cu — the norms before and after a block, its gate and the
// residual in one pass.
//
//   r = a x + g post(y)      post(y) = (1 + s_post) y / sqrt(mean(y^2) + 1e-6)
//   h = (1 + s_pre) r / sqrt(mean(r^2) + 1e-6)
// and, for an 8-bit h, its row scale max|h| / 127 and rounded values.
//
// Bound by HBM: x and y (and a token gate) are read once and r and h written once.
// A row stays in the registers of its threads from the loads to the last
// store: 8 elements (16 bytes of a 16-bit type) a load where every row is
// aligned for that, single elements otherwise.  Each of the two or three
// statistics is one reduction over the row's threads, in f32.  Up to 512
// elements a warp owns a row and reduces with shuffles alone; above, a block
// does.
//
// Many rows up to 8,192 elements are streamed by persistent blocks where that is
// faster (residual_norm_stream_kernel, and residual_norm_any_kernel off 16-byte
// boundaries); the others take residual_norm_kernel, a block or warp for each row.
#include <algorithm>

#include "common.cuh"
#include "ops.h"
#include "quant8.cuh"
#include "residual_norm.cuh"
#include "rowio.cuh"

namespace ndl {
namespace {

constexpr int kWarpRows = 8;  // rows of a block whose warps own a row each

// Sum over the threads of a row; `warps` of them when the block owns the row,
// else one.  sm: a word for each warp.
__device__ __forceinline__ float row_sum(float v, int warps, float *sm) {
  v = warp_sum(v);
  if (warps == 1) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sm[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? sm[lane] : 0.0f);
}

// Threads of a block: up to 256 with 8 or 16 elements each in whole vectors
// (rows up to 4,096 elements), up to 1,024 else.
template <int VEC, int CH>
constexpr int kMaxThreads = VEC == 8 && CH <= 2 ? 256 : 1024;

template <typename TX, typename TY, int VEC, int CH>
__global__ void __launch_bounds__(kMaxThreads<VEC, CH>) residual_norm_kernel(ResidualNormArgs a) {
  __shared__ float sm[3][32];
  const int T = blockDim.x, warps = T >> 5, d = a.d;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.M) return;  // blockDim.y > 1 only when a warp owns a row: no barrier is skipped
  const TX *x = (const TX *)a.x + row * a.ldx;
  // a row here and there is a chain of latencies: x is on its way while y is reduced
  float r[CH][VEC];
  alignas(16) TX xraw[CH][VEC];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * T + threadIdx.x) * VEC;
    if (i >= d) continue;
    if constexpr (VEC == 1) {
      xraw[c][0] = x[i];
    } else {
#pragma unroll
      for (int p = 0; p < VEC * (int)sizeof(TX) / 16; ++p)
        reinterpret_cast<uint4 *>(xraw[c])[p] = reinterpret_cast<const uint4 *>(x + i)[p];
    }
  }
  if (a.y) {
    const TY *y = (const TY *)a.y + row * a.ldy;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * T + threadIdx.x) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[c][j] = 0.0f;
      if (i < d) load<VEC>(y + i, r[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss += r[c][j] * r[c][j];
    float g = 1.0f;
    if (a.gate_kind == 1) {
      g = *(const float *)a.gate;
      if (a.sigmoid) g = logistic(g);
    }
    if (a.post) g *= 1.0f / sqrtf(row_sum(ss, warps, sm[0]) / (float)d + kEps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * T + threadIdx.x) * VEC;
      if (i >= d) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[c][j] *= g;
      if (a.post) {
        float s[VEC];
        load<VEC>(a.post + i, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) r[c][j] *= 1.0f + s[j];
      }
      if (a.gate_kind >= 2) {
        float gv[VEC];
        if (a.gate_kind == 2)
          load<VEC>((const float *)a.gate + i, gv);
        else
          load<VEC>((const TY *)a.gate + row * a.ldg + i, gv);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          r[c][j] *= !a.sigmoid ? gv[j] : a.gate_kind == 3 && sizeof(TY) == 2 ? logistic16(gv[j]) : logistic(gv[j]);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[c][j] = fmaf(a.scale, (float)xraw[c][j], r[c][j]);
      if (a.r) store<VEC>((TX *)a.r + row * a.ldr + i, r[c]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        r[c][j] = (c * T + (int)threadIdx.x) * VEC < d ? a.scale * (float)xraw[c][j] : 0.0f;
  }
  if (!a.h) return;
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < VEC; ++j) ss += r[c][j] * r[c][j];
  const float inv = 1.0f / sqrtf(row_sum(ss, warps, sm[1]) / (float)d + kEps);
  uint32_t top = 0;  // largest |h| as bits: infinities and NaN order above every number
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * T + threadIdx.x) * VEC;
    if (i < d) {
      float s[VEC];
      load<VEC>(a.pre + i, s);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        r[c][j] = ((1.0f + s[j]) * r[c][j]) * inv;
        top = max(top, __float_as_uint(r[c][j]) & 0x7fffffffu);
      }
      if (a.h_dtype != DT_I8) store<VEC>((TY *)a.h + row * a.ldh + i, r[c]);
    }
  }
  if (a.h_dtype != DT_I8) return;
  top = row_max_bits(top, warps, reinterpret_cast<uint32_t *>(sm[2]));
  const RowScale rs = int8_row_scale(top);
  int8_t *h = (int8_t *)a.h + row * a.ldh;
  const int dp = (d + 15) / 16 * 16;  // the row's bytes past d are zero
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * T + threadIdx.x) * VEC;
    if (i < d) {
      if constexpr (VEC == 8) {
        *reinterpret_cast<uint2 *>(h + i) = make_uint2(int8_pack4(r[c], rs.inv), int8_pack4(r[c] + 4, rs.inv));
      } else {
        h[i] = int8_round(r[c][0], rs.inv);
      }
    }
  }
  for (int i = d + (int)threadIdx.x; i < dp; i += T) h[i] = 0;
  if (threadIdx.x == 0) a.h_scales[row] = rs.scale;
}

// f32 vectors are two pieces of 16 bytes: through L1, so that the second finds the
// 32-byte sector there that the first has fetched.
template <typename T>
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  if constexpr (sizeof(T) == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// 8 elements as four packed pairs, from pieces of 16 bytes `stride` apart, and
// to consecutive memory.
template <typename T>
__device__ __forceinline__ void take8(const uint8_t *p, int stride, uint64_t *v) {
  if constexpr (sizeof(T) == 4) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(p), b = *reinterpret_cast<const ulonglong2 *>(p + stride);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    v[0] = pair_f32<T>(w.x), v[1] = pair_f32<T>(w.y), v[2] = pair_f32<T>(w.z), v[3] = pair_f32<T>(w.w);
  }
}
template <typename T>
__device__ __forceinline__ void put8(T *p, const uint64_t *v) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<ulonglong2 *>(p)[0] = make_ulonglong2(v[0], v[1]);
    reinterpret_cast<ulonglong2 *>(p)[1] = make_ulonglong2(v[2], v[3]);
  } else {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pair_bits<T>(v[0]), pair_bits<T>(v[1]), pair_bits<T>(v[2]), pair_bits<T>(v[3]));
  }
}

// Persistent blocks over many rows.  A thread owns CH vectors of 8 columns of
// every row of its block (or warp): their factors ((1 + s_post) g and
// 1 + s_pre, f32) stay in registers, since reading 12 bytes of them an element from L1
// took longer than the row itself, and the next row is in flight as cp.async
// copies into slots of shared memory that only this thread reads, so no barrier
// is needed for them and no register holds data in flight.  (Two rows ahead took 2
// to 6% longer than one.)
//
// The instructions of a row, not its bytes, bound the first forms (42 a lane and
// column; 65,536 x 2,048 bf16 took 236 us a block for each row, 280 with one
// row ahead in registers, 209 with the copies), hence packed pairs of f32
// throughout, the reciprocal square root of CUDA instead of an exact root and
// quotient (its 2 ulp are part of the row factor's few), and what is known before the
// first row as a template: MODE 0 no y, 1 y, 2 y and a token gate; FULL: every
// thread has all its vectors.  172 us now, 6.2 TB/s; calls one behind the other whose
// outputs rotate over four buffers take 185 (5.8 TB/s), as they do for any writer.
template <typename TX, typename TY, int MODE, bool FULL, int CH>
__global__ void __launch_bounds__(512) residual_norm_stream_kernel(ResidualNormArgs a) {
  constexpr int S = kStreamStages, PX = sizeof(TX) / 2, PY = sizeof(TY) / 2;  // 16-byte pieces of 8 elements
  constexpr int PER = PX + MODE * PY, PIECES = CH * PER;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float sm[2][3][16];  // of even and odd rows: a row's writes follow a barrier of the row between
  const int T = blockDim.x, warps = T >> 5, d = a.d, threads = T * blockDim.y;
  if (warps > 1) {
    for (int i = threadIdx.x; i < 96; i += T) (&sm[0][0][0])[i] = 0.0f;
    __syncthreads();
  }
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.M) return;  // blockDim.y > 1 only when a warp owns a row: no barrier is skipped
  const int tid = threadIdx.y * T + threadIdx.x, piece = threads * 16;
  const uint8_t *mine = ring + tid * 16;  // piece p of stage s at (s * PIECES + p) * piece
  const uint32_t mine_u = (uint32_t)__cvta_generic_to_shared(mine);
  const int i0 = threadIdx.x * 8;
  bool in[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) in[c] = FULL || c * T * 8 + i0 < d;
  // this thread's first vector of the next row to fetch; the second lies T * 8 further
  const TX *fx = (const TX *)a.x + row * a.ldx + i0;
  const TY *fy = MODE >= 1 ? (const TY *)a.y + row * a.ldy + i0 : nullptr;
  const TY *fg = MODE == 2 ? (const TY *)a.gate + row * a.ldg + i0 : nullptr;
  int64_t next = row;
  auto fetch = [&](int s) {
    if (next < a.M) {
      const uint32_t dst = mine_u + s * PIECES * piece;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (!in[c]) continue;
#pragma unroll
        for (int p = 0; p < PX; ++p) copy16<TX>(dst + (c * PER + p) * piece, (const uint8_t *)(fx + c * T * 8) + 16 * p);
#pragma unroll
        for (int p = 0; p < PY && MODE >= 1; ++p)
          copy16<TY>(dst + (c * PER + PX + p) * piece, (const uint8_t *)(fy + c * T * 8) + 16 * p);
#pragma unroll
        for (int p = 0; p < PY && MODE == 2; ++p)
          copy16<TY>(dst + (c * PER + PX + PY + p) * piece, (const uint8_t *)(fg + c * T * 8) + 16 * p);
      }
      next += step;
      fx += step * a.ldx;
      if (MODE >= 1) fy += step * a.ldy;
      if (MODE == 2) fg += step * a.ldg;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);

  uint64_t fp[CH][4], fh[CH][4];
  float g = 1.0f;  // scalar gate
  if (a.gate_kind == 1) {
    g = *(const float *)a.gate;
    if (a.sigmoid) g = logistic(g);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float p[8], h[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = g, h[j] = 1.0f;
    if (in[c]) {
      const int i = c * T * 8 + i0;
      if (a.post) {
        load<8>(a.post + i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] *= 1.0f + v[j];
      }
      if (a.gate_kind == 2) {
        load<8>((const float *)a.gate + i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] *= a.sigmoid ? logistic(v[j]) : v[j];
      }
      if (a.h) {
        load<8>(a.pre + i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) fp[c][j] = f2pack(p[2 * j], p[2 * j + 1]), fh[c][j] = f2pack(h[2 * j], h[2 * j + 1]);
  }
  const uint64_t zero = f2pack(0.0f, 0.0f), sc = f2pack(a.scale, a.scale);
  const float over_d = 1.0f / (float)d;
  TX *pr = a.r ? (TX *)a.r + row * a.ldr + i0 : nullptr;
  TY *ph = (TY *)a.h + (a.h_dtype == DT_I8 ? 0 : row * a.ldh + i0);

  int s = 0;
  for (int parity = 0; row < a.M; row += step, parity ^= 1) {
    fetch(s == 0 ? S - 1 : s - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    const uint8_t *at = mine + s * PIECES * piece;
    if (++s == S) s = 0;
    uint64_t r[CH][4], ss = zero;
    if (MODE >= 1) {
      float inv = 1.0f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[c][j] = zero;
        if (in[c]) take8<TY>(at + (c * PER + PX) * piece, piece, r[c]);
      }
      if (a.post) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) ss = ffma2(r[c][j], r[c][j], ss);
        inv = rsqrtf(fmaf(stream_sum(ss, warps, sm[parity][0]), over_d, kEps));
      }
      const uint64_t inv2 = f2pack(inv, inv);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) r[c][j] = fmul2(fmul2(r[c][j], inv2), fp[c][j]);
      if (MODE == 2) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (!in[c]) continue;
          uint64_t gv[4];
          take8<TY>(at + (c * PER + PX + PY) * piece, piece, gv);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (a.sigmoid) {
              float u, v;
              f2unpack(gv[j], u, v);
              gv[j] = f2pack(sizeof(TY) == 2 ? logistic16(u) : logistic(u), sizeof(TY) == 2 ? logistic16(v) : logistic(v));
            }
            r[c][j] = fmul2(r[c][j], gv[j]);
          }
        }
      }
    }
    ss = zero;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      uint64_t xv[4] = {zero, zero, zero, zero};
      if (in[c]) take8<TX>(at + c * PER * piece, piece, xv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[c][j] = MODE >= 1 ? ffma2(xv[j], sc, r[c][j]) : fmul2(xv[j], sc);
        ss = ffma2(r[c][j], r[c][j], ss);
      }
      if (MODE >= 1 && pr && in[c]) put8<TX>(pr + c * T * 8, r[c]);
    }
    if (MODE >= 1 && pr) pr += step * a.ldr;
    if (!a.h) continue;
    const float inv = rsqrtf(fmaf(stream_sum(ss, warps, sm[parity][1]), over_d, kEps));
    const uint64_t inv2 = f2pack(inv, inv);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) r[c][j] = fmul2(fmul2(r[c][j], inv2), fh[c][j]);
    if (a.h_dtype != DT_I8) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (in[c]) put8<TY>(ph + c * T * 8, r[c]);
      ph += step * a.ldh;
      continue;
    }
    uint32_t top = 0;  // largest |h| as bits: infinities and NaN order above every number
    float v[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f2unpack(r[c][j], v[c][2 * j], v[c][2 * j + 1]);
        top = max(top, max(__float_as_uint(v[c][2 * j]) & 0x7fffffffu, __float_as_uint(v[c][2 * j + 1]) & 0x7fffffffu));
      }
    const RowScale rs = int8_row_scale(row_max_bits(top, warps, reinterpret_cast<uint32_t *>(sm[parity][2])));
    int8_t *h = (int8_t *)a.h + row * a.ldh;
    const int dp = (d + 15) / 16 * 16;  // the row's bytes past d are zero
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * T * 8 + i0;
      if (in[c])
        *reinterpret_cast<uint2 *>(h + i) = make_uint2(int8_pack4(v[c], rs.inv), int8_pack4(v[c] + 4, rs.inv));
      else if (i < dp)
        *reinterpret_cast<uint2 *>(h + i) = make_uint2(0, 0);
    }
    if (threadIdx.x == 0) a.h_scales[row] = rs.scale;
  }
}

template <typename TX, typename TY, int VEC, int CH>
cudaError_t launch_rows(const ResidualNormArgs &a, cudaStream_t st) {
  const int need = (a.d + VEC * CH - 1) / (VEC * CH);
  const int T = (need + 31) / 32 * 32;
  const int rows = T == 32 ? kWarpRows : 1;
  const int64_t grid = (a.M + rows - 1) / rows;
  residual_norm_kernel<TX, TY, VEC, CH><<<dim3((unsigned)grid), dim3(T, rows), 0, st>>>(a);
  return cudaGetLastError();
}

// Rows of whole vectors up to 8,192 elements on as many blocks as fit the
// device at once; from two rows a block on (*done).
template <typename TX, typename TY, int MODE, bool FULL, int CH>
cudaError_t launch_stream(const ResidualNormArgs &a, int T, bool *done, cudaStream_t st) {
  constexpr size_t pieces = CH * (sizeof(TX) / 2 + MODE * sizeof(TY) / 2);
  const int rows = T == 32 ? 4 : 1;
  const size_t smem = kStreamStages * pieces * 16 * T * rows;
  auto *kernel = residual_norm_stream_kernel<TX, TY, MODE, FULL, CH>;
  static thread_local int last_dev = -1, last_threads = 0, fit = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (last_dev != dev || last_threads != T)) {
    int sms = 0, each = 0;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, T * rows, smem);
    if (e == cudaSuccess) last_dev = dev, last_threads = T, fit = sms * each;
  }
  *done = e != cudaSuccess || (fit > 0 && a.M >= 2 * (int64_t)fit * rows);
  if (e != cudaSuccess || !*done) return e;
  kernel<<<dim3((unsigned)fit), dim3(T, rows), smem, st>>>(a);
  return cudaGetLastError();
}
template <typename TX, typename TY, int MODE, int CH>
cudaError_t stream_vectors(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  const int T = ((a.d + 8 * CH - 1) / (8 * CH) + 31) / 32 * 32;
  return a.d == 8 * CH * T ? launch_stream<TX, TY, MODE, true, CH>(a, T, done, st)
                           : launch_stream<TX, TY, MODE, false, CH>(a, T, done, st);
}
// One vector of 8 a thread, two above 4,096 elements: more warps with fewer
// columns each cover each other's reductions better (65,536 x 2,048 bf16 into one
// buffer: 169 us with one, 190 with two).
template <typename TX, typename TY, int MODE>
cudaError_t stream_mode(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  return a.d <= 4096 ? stream_vectors<TX, TY, MODE, 1>(a, done, st) : stream_vectors<TX, TY, MODE, 2>(a, done, st);
}
// An f32 x has twice the bytes for the same instructions, and a block for each row
// then keeps up (32,768 x 2,048 with a bf16 y: 131 us, streamed 147; 16-bit x
// 65,536 x 2,048: 231, streamed 169), unless a token gate adds to them
// (4,096 x 4,096: 49, streamed 43).
template <typename TX, typename TY>
cudaError_t stream_rows(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  if (a.gate_kind == 3) return stream_mode<TX, TY, 2>(a, done, st);
  if constexpr (sizeof(TX) == 2) return a.y ? stream_mode<TX, TY, 1>(a, done, st) : stream_mode<TX, TY, 0>(a, done, st);
  *done = false;
  return cudaSuccess;
}

template <typename TX, typename TY>
cudaError_t dispatch(const ResidualNormArgs &a, cudaStream_t st) {
  auto al = [](const void *p) { return ((uintptr_t)p & 15) == 0; };
  // a scalar gate is read as one f32, wherever it lies
  const bool vec = a.d % 8 == 0 && al(a.x) && al(a.y) && (a.gate_kind < 2 || al(a.gate)) && al(a.r) && al(a.h) && al(a.post) &&
                   al(a.pre) && a.ldx % 8 == 0 && (!a.y || a.ldy % 8 == 0) && (!a.r || a.ldr % 8 == 0) &&
                   (!a.h || a.ldh % 8 == 0) && (a.gate_kind != 3 || a.ldg % 8 == 0);
  if (vec) {
    bool done = false;
    if (a.d <= 8192) {
      const cudaError_t e = stream_rows<TX, TY>(a, &done, st);
      if (done) return e;
    }
    if (a.d <= 256) return launch_rows<TX, TY, 8, 1>(a, st);
    if (a.d <= 4096) return launch_rows<TX, TY, 8, 2>(a, st);
    return launch_rows<TX, TY, 8, 4>(a, st);
  }
  if (a.d <= 8192) {
    bool done = false;
    const cudaError_t e = residual_norm_any(a, &done, st);
    if (done) return e;
  }
  if (a.d <= 8192) return launch_rows<TX, TY, 1, 8>(a, st);
  if (a.d <= 16384) return launch_rows<TX, TY, 1, 16>(a, st);
  return launch_rows<TX, TY, 1, 32>(a, st);
}

}  // namespace

cudaError_t residual_norm(const ResidualNormArgs &a, cudaStream_t st) {
  if (a.x_dtype == DT_F32) {
    if (a.y_dtype == DT_F32) return dispatch<float, float>(a, st);
    if (a.y_dtype == DT_F16) return dispatch<float, __half>(a, st);
    return dispatch<float, __nv_bfloat16>(a, st);
  }
  if (a.x_dtype == DT_F16) return dispatch<__half, __half>(a, st);
  return dispatch<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace ndl
