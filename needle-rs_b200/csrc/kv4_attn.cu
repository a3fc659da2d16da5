// kv4_attn.cu — attention of query rows to a cache of keys and values in 4
// bits.
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

// A warp for each row and head, a key after another.
template <typename T>
__global__ void attn_kernel(Kv4AttnCall c, Kv4Shape s, Kv4Rows b, int *bad) {
  check_all(b, s, c.causal, bad);
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = unit / s.H;
  const int h = (int)(unit % s.H), lane = threadIdx.x & 31, ng = s.ng, kvh = h / (s.H / s.KVH);
  if (row >= b.rows) return;
  int lo = 0, hi = b.n_seq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.row_start[mid] <= row) lo = mid; else hi = mid;
  }
  const Seq sq = sequence(b, s, lo, c.causal, bad);
  if (row < sq.row0 || row >= sq.row0 + sq.n) return;
  const int keys = c.causal ? sq.len - sq.n + (int)(row - sq.row0) + 1 : sq.len;
  float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
  for (int g = 0; g < 4; ++g) {
    const int d = g * 32 + lane;
    q[g] = d < s.D ? (float)((const T *)c.q)[row * c.q_row + (int64_t)h * c.q_head + d] : 0.0f;
  }
  for (int j = 0; j < keys; ++j) {
    const int t = j % kTokens;
    const uint8_t *tile = tile_at((uint8_t *)c.pages, b, s, lo, j / kTokens, kvh, bad);
    if (!tile) break;
    float x = 0.0f, v[4];
    for (int g = 0; g < ng; ++g) {
      const float2 kp = __half22float2(*(const __half2 *)(tile + k_param(ng, t, g)));
      const uint32_t w = *(const uint32_t *)(tile + k_word(t, g, lane >> 3));
      x += q[g] * fmaf(kp.x, (float)((w >> (4 * (((lane & 7) >> 1) + 4 * (lane & 1)))) & 15u), kp.y);
      const uint32_t u = *(const uint16_t *)(tile + v_half(ng, t, g, lane >> 2));
      v[g] = fmaf(__half2float(*(const __half *)(tile + v_param(ng, t, g, 0))), (float)((u >> (4 * (lane & 3))) & 15u),
                  __half2float(*(const __half *)(tile + v_param(ng, t, g, 1))));
    }
    x = warp_sum(x) * c.scale;
    const float top = fmaxf(m, x), f = m == -INFINITY ? 0.0f : expf(m - top), p = expf(x - top);
    l = l * f + p;
    for (int g = 0; g < ng; ++g) o[g] = o[g] * f + p * v[g];
    m = top;
  }
  for (int g = 0; g < ng; ++g)
    if (g * 32 + lane < s.D)
      ((T *)c.out)[row * c.o_row + (int64_t)h * c.o_head + g * 32 + lane] = from_f32<T>(keys ? o[g] / l : 0.0f);
  if (lane == 0 && c.lse) c.lse[row * s.H + h] = keys ? m + logf(l) : -INFINITY;
}

}  // namespace

cudaError_t kv4_attn(const Kv4Shape &s, const Kv4Rows &b, const Kv4AttnCall &c, const Kv4Work &w, cudaStream_t st) {
  if (b.rows == 0) return cudaSuccess;
  const unsigned grid = (unsigned)((b.rows * s.H + 7) / 8);
  if (s.dtype == DT_F16) attn_kernel<__half><<<grid, 256, 0, st>>>(c, s, b, w.bad);
  else attn_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(c, s, b, w.bad);
  return cudaGetLastError();
}

}  // namespace ndl
