// residual_norm_any.cu — the residual norm of many rows that do not all start on
// 16-byte boundaries (residual_norm.cu has the formulas).
#include <algorithm>

#include "common.cuh"
#include "ops.h"
#include "quant8.cuh"
#include "residual_norm.cuh"
#include "rowio.cuh"

namespace ndl {
namespace {

constexpr int kAnyPairs = 8;  // pairs of columns a thread, up to
constexpr size_t kAnySmem = 226 * 1024;

// The pairs of columns t, t + T, ... of a row that starts `off` bytes into a
// 16-byte aligned buffer, read and written as words: lanes that hold neighbouring
// pairs touch neighbouring words.  Pairs from the
// `nc`-th on lie past the row: they are zero and not written.
template <typename E, int T, int P>
__device__ __forceinline__ void pairs_in(const uint8_t *buf, int off, int t, int nc, uint64_t *v) {
  const uint32_t *w = reinterpret_cast<const uint32_t *>(buf) + (off >> 2) + t * (int)(sizeof(E) / 2);
  const int sh = (off & 2) << 3;
#pragma unroll
  for (int c = 0; c < P; ++c) {
    uint32_t a = 0, b = 0;
    if (c < nc) {
      a = w[c * T * (int)(sizeof(E) / 2)];
      b = w[c * T * (int)(sizeof(E) / 2) + 1];
    }
    if constexpr (sizeof(E) == 4)
      v[c] = f2pack(__uint_as_float(a), __uint_as_float(b));
    else
      v[c] = pair_f32<E>(__funnelshift_r(a, b, sh));
  }
}
template <typename E, int T, int P>
__device__ __forceinline__ void pairs_out(uint8_t *buf, int off, int t, int nc, const uint64_t *v) {
  uint32_t *w = reinterpret_cast<uint32_t *>(buf) + (off >> 2) + t * (int)(sizeof(E) / 2);
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int c = 0; c < P; ++c) {
      float a, b;
      f2unpack(v[c], a, b);
      if (c < nc) {
        w[2 * c * T] = __float_as_uint(a);
        w[2 * c * T + 1] = __float_as_uint(b);
      }
    }
  } else if (off & 2) {
    uint16_t *h = reinterpret_cast<uint16_t *>(w) + 1;
#pragma unroll
    for (int c = 0; c < P; ++c) {
      const uint32_t bits = pair_bits<E>(v[c]);
      if (c < nc) {
        h[2 * c * T] = (uint16_t)bits;
        h[2 * c * T + 1] = (uint16_t)(bits >> 16);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < P; ++c)
      if (c < nc) w[c * T] = pair_bits<E>(v[c]);
  }
}

// Many rows off 16-byte boundaries (odd d).  As the streaming kernel, but a row
// crosses between global and shared memory in whole 16-byte pieces (row_in,
// row_out), and there a thread takes every T-th pair of columns, wherever the row
// starts; T is a template, so that a pair's place is a constant.  Element by element in
// global memory 14,785 x 6,738 bf16 took 847 us, element by element in shared memory 431
// (92 instructions an element and warp), by pairs with T a variable 320.
template <typename TX, typename TY, bool TOKEN, bool EACH, int T, int P>
__global__ void __launch_bounds__(T < 128 ? 128 : T, 1024 / (T < 128 ? 128 : T)) residual_norm_any_kernel(ResidualNormArgs a, int bx, int by) {
  constexpr int S = kStreamStages, warps = T / 32;
  // a row group's shared memory: S stages of x, y and gate rows, then r and h
  extern __shared__ __align__(16) uint8_t buf[];
  __shared__ __align__(16) float sm[3][16];
  const int t = threadIdx.x, d = a.d;
  const bool have_y = TOKEN || a.y != nullptr;
  // the logistic function of a channel gate: EACH row's work, or found once a block and kept behind the rows
  const bool logi = !TOKEN && a.gate_kind == 2 && a.sigmoid, keep = !EACH && logi;
  const int stage = bx + (TOKEN ? 2 : 1) * by;
  float *gates = reinterpret_cast<float *>(buf + (size_t)blockDim.y * (S * stage + bx + by));
  if (keep)
    for (int i = threadIdx.y * T + t; i < d; i += T * blockDim.y) gates[i] = logistic(((const float *)a.gate)[i]);
  if (warps > 1)
    for (int i = t; i < 48; i += T) (&sm[0][0])[i] = 0.0f;
  if (warps > 1 || keep) __syncthreads();
  auto sync = [&] {
    if (warps > 1)
      __syncthreads();
    else
      __syncwarp();
  };
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.M) return;  // blockDim.y > 1 only when a warp owns a row: no barrier is skipped
  uint8_t *in = buf + (size_t)threadIdx.y * (S * stage + bx + by), *out_r = in + S * stage, *out_h = out_r + bx;
  auto fetch = [&](int64_t at, int s) {
    if (at < a.M) {
      row_in(in + s * stage, (const TX *)a.x + at * a.ldx, d * (int)sizeof(TX), t, T);
      if (have_y) row_in(in + s * stage + bx, (const TY *)a.y + at * a.ldy, d * (int)sizeof(TY), t, T);
      if (TOKEN) row_in(in + s * stage + bx + by, (const TY *)a.gate + at * a.ldg, d * (int)sizeof(TY), t, T);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(row + s * step, s);
  float g = 1.0f;  // scalar gate
  if (a.gate_kind == 1) {
    g = *(const float *)a.gate;
    if (a.sigmoid) g = logistic(g);
  }
  // pairs of this thread; a row's column behind the last (odd d) is kept zero in
  // shared memory, so that no pair is a special case; factors of a pair's columns are read
  // from L1 every row (registers for them would halve the blocks on an SM)
  const int nc = ((d + 1) / 2 - t + T - 1) / T;
  const int odd = (d & 1) && (d >> 1) % T == t ? (d >> 1) / T : -1;  // the pair that holds that column
  auto times = [&](uint64_t *r, const float *p, float one) {  // r *= one + p; EACH: logistic(p) for the gate
#pragma unroll
    for (int c = 0; c < P; ++c) {
      float u = 0.0f, v = 0.0f;
      if (c < nc) u = p[2 * (c * T + t)], v = p[min(2 * (c * T + t) + 1, d - 1)];
      u = EACH && one == 0.0f ? logistic(u) : one + u;
      v = EACH && one == 0.0f ? logistic(v) : one + v;
      r[c] = fmul2(r[c], f2pack(u, v));
    }
  };
  const float *channel = a.gate_kind != 2 ? nullptr : keep ? gates : (const float *)a.gate;
  const uint64_t zero = f2pack(0.0f, 0.0f), sc = f2pack(a.scale, a.scale);
  const float over_d = 1.0f / (float)d;
  // bytes from the last 16-byte boundary to row `at` of p
  auto offset = [](const void *p, int64_t at, int64_t ld, int size) {
    return (int)(((uint32_t)(uintptr_t)p + (uint32_t)at * (uint32_t)ld * (uint32_t)size) & 15u);
  };
  int s = 0;
  for (; row < a.M; row += step) {
    fetch(row + (S - 1) * step, s == 0 ? S - 1 : s - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    uint8_t *at = in + s * stage;
    if (++s == S) s = 0;
    const int ox = offset(a.x, row, a.ldx, sizeof(TX)), oy = offset(a.y, row, a.ldy, sizeof(TY)),
              og = offset(a.gate, row, a.ldg, sizeof(TY));
    if ((d & 1) && t == 0) {
      *reinterpret_cast<TX *>(at + ox + d * sizeof(TX)) = from_f32<TX>(0.0f);
      if (have_y) *reinterpret_cast<TY *>(at + bx + oy + d * sizeof(TY)) = from_f32<TY>(0.0f);
      if (TOKEN) *reinterpret_cast<TY *>(at + bx + by + og + d * sizeof(TY)) = from_f32<TY>(0.0f);
    }
    sync();  // the whole row has arrived, and the last one has left out_r and out_h
    uint64_t r[P], v[P], ss = zero;
#pragma unroll
    for (int c = 0; c < P; ++c) r[c] = zero;
    if (have_y) {
      float inv = g;
      pairs_in<TY, T, P>(at + bx, oy, t, nc, r);
      if (a.post) {
#pragma unroll
        for (int c = 0; c < P; ++c) ss = ffma2(r[c], r[c], ss);
        inv *= rsqrtf(fmaf(stream_sum(ss, warps, sm[0]), over_d, kEps));
      }
#pragma unroll
      for (int c = 0; c < P; ++c) r[c] = fmul2(r[c], f2pack(inv, inv));
      if (a.post) times(r, a.post, 1.0f);
      if (!TOKEN && channel) times(r, channel, 0.0f);
      if (TOKEN) {
        pairs_in<TY, T, P>(at + bx + by, og, t, nc, v);
#pragma unroll
        for (int c = 0; c < P; ++c) {
          if (a.sigmoid) {
            float x0, x1;
            f2unpack(v[c], x0, x1);
            v[c] = f2pack(sizeof(TY) == 2 ? logistic16(x0) : logistic(x0), sizeof(TY) == 2 ? logistic16(x1) : logistic(x1));
          }
          r[c] = fmul2(r[c], v[c]);
        }
      }
      if (odd >= 0) {  // the last column's factor, which that column was multiplied by, may be infinite
#pragma unroll
        for (int c = 0; c < P; ++c) {
          float x0, x1;
          f2unpack(r[c], x0, x1);
          if (c == odd) r[c] = f2pack(x0, 0.0f);
        }
      }
    }
    ss = zero;
    pairs_in<TX, T, P>(at, ox, t, nc, v);
#pragma unroll
    for (int c = 0; c < P; ++c) {
      r[c] = ffma2(v[c], sc, r[c]);
      ss = ffma2(r[c], r[c], ss);
    }
    if (a.r) pairs_out<TX, T, P>(out_r, offset(a.r, row, a.ldr, sizeof(TX)), t, nc, r);
    if (a.h) {
      const float inv = rsqrtf(fmaf(stream_sum(ss, warps, sm[1]), over_d, kEps));
#pragma unroll
      for (int c = 0; c < P; ++c) r[c] = fmul2(r[c], f2pack(inv, inv));
      times(r, a.pre, 1.0f);
      if (a.h_dtype == DT_I8) {
        uint32_t top = 0;  // largest |h| as bits: infinities and NaN order above every number
#pragma unroll
        for (int c = 0; c < P; ++c) {
          float x0, x1;
          f2unpack(r[c], x0, x1);
          top = max(top, max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu));
        }
        const RowScale rs = int8_row_scale(row_max_bits(top, warps, reinterpret_cast<uint32_t *>(sm[2])));
        const int dp = (d + 15) / 16 * 16;  // rows of 8-bit values start on 16-byte boundaries
#pragma unroll
        for (int c = 0; c < P; ++c) {
          float x0, x1;
          f2unpack(r[c], x0, x1);
          if (c < nc)
            reinterpret_cast<char2 *>(out_h)[c * T + t] = make_char2(int8_round(x0, rs.inv), int8_round(x1, rs.inv));
        }
        if (t < dp - d) out_h[d + t] = 0;
        if (t == 0) a.h_scales[row] = rs.scale;
      } else {
        pairs_out<TY, T, P>(out_h, offset(a.h, row, a.ldh, sizeof(TY)), t, nc, r);
      }
    }
    sync();
    if (a.r) row_out((TX *)a.r + row * a.ldr, out_r, d * (int)sizeof(TX), t, T);
    if (a.h && a.h_dtype == DT_I8)
      row_out((int8_t *)a.h + row * a.ldh, out_h, (d + 15) / 16 * 16, t, T);
    else if (a.h)
      row_out((TY *)a.h + row * a.ldh, out_h, d * (int)sizeof(TY), t, T);
  }
}

// The same for rows at any alignment; from one row a block on.
template <typename TX, typename TY, bool TOKEN, int T, int P = kAnyPairs>
cudaError_t launch_any(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  const int rows = T == 32 ? 4 : 1;  // blocks of several rows only where no barrier spans them
  // bytes of a row and its offset, to the next 16-byte boundary
  const int bx = (a.d * (int)sizeof(TX) + 31) / 16 * 16, by = (a.d * (int)sizeof(TY) + 31) / 16 * 16;
  const size_t smem = (size_t)rows * (kStreamStages * (bx + (TOKEN ? 2 : 1) * by) + bx + by);
  const size_t kept_smem = smem + 4 * (size_t)a.d;
  auto *kernel = residual_norm_any_kernel<TX, TY, TOKEN, false, T, P>;
  // the form that finds a channel gate's logistic function for each row: where one block would be left of two
  constexpr bool kEach = !TOKEN && T == 512;
  auto *each_row = residual_norm_any_kernel<TX, TY, TOKEN, kEach, T, P>;
  static thread_local int last_dev = -1, last_d = 0, fit = 0, fit_kept = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (last_dev != dev || last_d != a.d)) {
    int sms = 0, each = 0, kept = 0;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAnySmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(each_row, cudaFuncAttributeMaxDynamicSharedMemorySize, kAnySmem);
    if (e == cudaSuccess && smem <= kAnySmem)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, T * rows, smem);
    if (e == cudaSuccess && kept_smem <= kAnySmem)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&kept, kernel, T * rows, kept_smem);
    if (e == cudaSuccess) last_dev = dev, last_d = a.d, fit = sms * each, fit_kept = sms * kept;
  }
  // 9,001 x 2,050, f32 and bf16, a sigmoid channel gate: 94 us kept, 119 for each row; 9,001 x 8,190
  // bf16, where one block would be left of two: 333 and 283
  const bool logi = a.gate_kind == 2 && a.sigmoid, keep = logi && !(kEach && fit_kept < fit);
  const int blocks = keep ? fit_kept : fit;
  *done = e != cudaSuccess || (blocks > 0 && a.M >= (int64_t)blocks * rows);
  if (e != cudaSuccess || !*done) return e;
  (logi && !keep ? each_row : kernel)<<<dim3((unsigned)blocks), dim3(T, rows), keep ? kept_smem : smem, st>>>(a, bx, by);
  return cudaGetLastError();
}

// The fewest threads, a power of two, whose pairs cover a row; for less than a
// warp's 512 columns fewer pairs a thread, 2 or 4 (60,000 rows, with 8 in brackets:
// 63 f32 and f16 43 us (70), 117 f16 with a token gate 50 (72), 201 bf16 52 (62), 255 f32 62 (69)).
template <typename TX, typename TY, bool TOKEN>
cudaError_t launch_threads(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  const int need = (a.d + 2 * kAnyPairs - 1) / (2 * kAnyPairs);
  if (need <= 8) return launch_any<TX, TY, TOKEN, 32, 2>(a, done, st);
  if (need <= 16) return launch_any<TX, TY, TOKEN, 32, 4>(a, done, st);
  if (need <= 32) return launch_any<TX, TY, TOKEN, 32>(a, done, st);
  if (need <= 64) return launch_any<TX, TY, TOKEN, 64>(a, done, st);
  if (need <= 128) return launch_any<TX, TY, TOKEN, 128>(a, done, st);
  if (need <= 256) return launch_any<TX, TY, TOKEN, 256>(a, done, st);
  return launch_any<TX, TY, TOKEN, 512>(a, done, st);
}
template <typename TX, typename TY>
cudaError_t launch_types(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  return a.gate_kind == 3 ? launch_threads<TX, TY, true>(a, done, st) : launch_threads<TX, TY, false>(a, done, st);
}

}  // namespace

cudaError_t residual_norm_any(const ResidualNormArgs &a, bool *done, cudaStream_t st) {
  if (a.x_dtype == DT_F32) {
    if (a.y_dtype == DT_F32) return launch_types<float, float>(a, done, st);
    if (a.y_dtype == DT_F16) return launch_types<float, __half>(a, done, st);
    return launch_types<float, __nv_bfloat16>(a, done, st);
  }
  if (a.x_dtype == DT_F16) return launch_types<__half, __half>(a, done, st);
  return launch_types<__nv_bfloat16, __nv_bfloat16>(a, done, st);
}

}  // namespace ndl
