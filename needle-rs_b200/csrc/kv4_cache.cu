// kv4_cache.cu — keys and values to 4 bits as a cache takes them, and back.
//
// A head of a token in groups of 32 dimensions (the last may be shorter):
//   minimum = f16(min x), scale = f16((max x - min x) / 15)
//   code = rint((x - minimum) * (1 / scale)), within 0 to 15
//   value = minimum + scale * code
// every other operation rounded to f32, so that any program that follows the
// formula gets the same codes.  The codes are of the rounded scale and
// minimum: what their rounding to f16 moves is within the codes' rounding.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kv4.cuh"
#include "ops.h"
#include "rowio.cuh"

namespace ndl {
namespace {

using namespace kv4;

// The request and the token of row `row` of a call (n = 0: none).
struct Row {
  int seq, pos;
  bool there;
};
__device__ __forceinline__ Row row_at(const Kv4Rows &b, const Kv4Shape &s, int64_t row, int *bad) {
  int lo = 0, hi = b.n_seq;  // the last request that starts at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.row_start[mid] <= row) lo = mid; else hi = mid;
  }
  const Seq q = sequence(b, s, lo, true, bad);
  const bool there = row >= q.row0 && row < q.row0 + q.n;
  return Row{lo, there ? q.len - q.n + (int)(row - q.row0) : 0, there};
}

template <typename T>
__global__ void append_kernel(Kv4Call c, Kv4Shape s, Kv4Rows b, int *bad) {
  check_all(b, s, true, bad);
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = unit / s.KVH;
  const int kvh = (int)(unit % s.KVH), lane = threadIdx.x & 31, ng = s.ng;
  if (row >= b.rows) return;
  const Row at = row_at(b, s, row, bad);
  if (!at.there) return;
  uint8_t *tile = tile_at(c.pages, b, s, at.seq, at.pos / kTokens, kvh, bad);
  if (!tile) return;
  const T *k = (const T *)c.k + row * c.k_row + (int64_t)kvh * c.k_head;
  const T *v = (const T *)c.v + row * c.v_row + (int64_t)kvh * c.v_head;
  const int t = at.pos % kTokens;
  bool ok = true;
  for (int d = lane; d < s.D; d += 32) ok = ok && fabsf((float)k[d]) <= kLargest && fabsf((float)v[d]) <= kLargest;
  ok = __all_sync(0xffffffffu, ok);
  for (int u = 0; u < 2 * ng; ++u) {
    const int g = u >> 1, d = g * 32 + lane;
    const bool is_v = u & 1, in = d < s.D;
    const float x = in ? (float)(is_v ? v : k)[d] : 0.0f;
    const float lo = -warp_max(in ? -x : -INFINITY), hi = warp_max(in ? x : -INFINITY);
    __half scale = __float2half_rn(__fdiv_rn(hi - lo, 15.0f)), least = __float2half_rn(lo);
    if (!ok) scale = least = __ushort_as_half(is_v ? 0 : 0x7fff);
    const float sc = __half2float(scale), inv = sc > 0.0f ? __fdiv_rn(1.0f, sc) : 0.0f;
    const float q = rintf(__fmul_rn(__fsub_rn(x, __half2float(least)), inv));
    const uint32_t code = ok && in ? (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f) : 0u;
    if (is_v) {
      uint32_t w = code << (4 * (lane & 3));
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      if ((lane & 3) == 0) *(uint16_t *)(tile + v_half(ng, t, g, lane >> 2)) = (uint16_t)w;
      if (lane < 2) *(__half *)(tile + v_param(ng, t, g, lane)) = lane ? least : scale;
    } else {
      uint32_t w = code << (4 * (((lane & 7) >> 1) + 4 * (lane & 1)));
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      if ((lane & 7) == 0) *(uint32_t *)(tile + k_word(t, g, lane >> 3)) = w;
      if (lane < 2) *(__half *)(tile + k_param(ng, t, g, lane)) = lane ? least : scale;
    }
  }
}

template <typename T>
__global__ void read_kernel(Kv4Call c, Kv4Shape s, Kv4Rows b, int *bad) {
  check_all(b, s, true, bad);
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = unit / s.KVH;
  const int kvh = (int)(unit % s.KVH), lane = threadIdx.x & 31, ng = s.ng;
  if (row >= b.rows) return;
  const Row at = row_at(b, s, row, bad);
  if (!at.there) return;
  const uint8_t *tile = tile_at(c.pages, b, s, at.seq, at.pos / kTokens, kvh, bad);
  if (!tile) return;
  T *k = (T *)c.k_out + row * c.k_row + (int64_t)kvh * c.k_head, *v = (T *)c.v_out + row * c.v_row + (int64_t)kvh * c.v_head;
  const int t = at.pos % kTokens;
  for (int d = lane; d < s.D; d += 32) {
    const int g = d >> 5, i = d & 31;
    const float2 kp = make_float2(__half2float(*(const __half *)(tile + k_param(ng, t, g, 0))),
                                  __half2float(*(const __half *)(tile + k_param(ng, t, g, 1))));
    if (c.k_out) {
      const uint32_t w = *(const uint32_t *)(tile + k_word(t, g, i >> 3));
      k[d] = from_f32<T>(fmaf(kp.x, (float)((w >> (4 * (((i & 7) >> 1) + 4 * (i & 1)))) & 15u), kp.y));
    }
    if (c.v_out) {
      const uint32_t w = *(const uint16_t *)(tile + v_half(ng, t, g, i >> 2));
      const float sc = __half2float(*(const __half *)(tile + v_param(ng, t, g, 0)));
      const float least = __half2float(*(const __half *)(tile + v_param(ng, t, g, 1)));
      // a key of NaN marks a token that did not fit
      v[d] = from_f32<T>(isnan(kp.x) ? kp.x : fmaf(sc, (float)((w >> (4 * (i & 3))) & 15u), least));
    }
  }
}

}  // namespace

cudaError_t kv4_append(const Kv4Shape &s, const Kv4Rows &b, const Kv4Call &c, int *bad, cudaStream_t st) {
  if (b.rows == 0) return cudaSuccess;
  const unsigned grid = (unsigned)((b.rows * s.KVH + 7) / 8);
  if (s.dtype == DT_F16) append_kernel<__half><<<grid, 256, 0, st>>>(c, s, b, bad);
  else append_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(c, s, b, bad);
  return cudaGetLastError();
}

cudaError_t kv4_read(const Kv4Shape &s, const Kv4Rows &b, const Kv4Call &c, int *bad, cudaStream_t st) {
  if (b.rows == 0) return cudaSuccess;
  const unsigned grid = (unsigned)((b.rows * s.KVH + 7) / 8);
  if (s.dtype == DT_F16) read_kernel<__half><<<grid, 256, 0, st>>>(c, s, b, bad);
  else read_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(c, s, b, bad);
  return cudaGetLastError();
}

}  // namespace ndl
