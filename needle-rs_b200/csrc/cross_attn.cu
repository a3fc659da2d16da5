// cross_attn.cu — attention of ragged query rows to encoder states of other
// lengths:
//   s_j = scale * q . k_j     out = sum_j e^(s_j) v_j / sum_j e^(s_j)
// over a request's keys, masked ones left out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "ops.h"

namespace ndl {
namespace {

constexpr int kRows = 8;

// A warp for each packed row: 32 keys at a time, a lane for each key's score,
// then a lane for each 4 dimensions of the sum.
template <typename T>
__global__ void cross_attn_rows_kernel(XAttnWork w, XAttnCall c) {
  const XAttnItem it = w.items[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = w.s.H / w.s.KVH, D = w.s.D;
  if (warp >= it.rows) return;
  const int r = it.r0 + warp, h = it.kvh * G + r % G;
  const int64_t qrow = it.q0 + r / G;
  const T *q = (const T *)c.q + qrow * c.q_row + (int64_t)h * c.q_head;
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < it.klen; j0 += 32) {
    const int64_t key = it.k0 + j0 + lane;
    const bool seen = j0 + lane < it.klen && (!c.mask || c.mask[key]);
    float s = -INFINITY;
    if (seen) {
      const T *k = (const T *)c.k + key * c.k_row + (int64_t)it.kvh * c.k_head;
      s = 0.0f;
      for (int i = 0; i < D; ++i) s += (float)q[i] * (float)k[i];
      s *= c.scale;
    }
    const float mn = fmaxf(m, warp_max(s));
    if (mn == -INFINITY) continue;
    const float p = s == -INFINITY ? 0.0f : expf(s - mn), f = expf(m - mn);
    l = l * f + warp_sum(p);
    for (int i = 0; i < 4; ++i) o[i] *= f;
    m = mn;
    const unsigned live = __ballot_sync(0xffffffffu, seen);
    for (int j = 0; j < 32; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      if (!((live >> j) & 1)) continue;
      const T *v = (const T *)c.v + (it.k0 + j0 + j) * c.v_row + (int64_t)it.kvh * c.v_head;
      for (int i = 0; i < 4; ++i)
        if (4 * lane + i < D) o[i] += pj * (float)v[4 * lane + i];
    }
  }
  T *out = (T *)c.out + qrow * c.o_row + (int64_t)h * c.o_head;
  for (int i = 0; i < 4; ++i)
    if (4 * lane + i < D) out[4 * lane + i] = (T)(l > 0.0f ? o[i] / l : (l == 0.0f ? 0.0f : l));
  if (c.lse && lane == 0) c.lse[qrow * w.s.H + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

std::vector<XAttnItem> cross_attn_split(const XAttnShape &s, const uint64_t *q_start, const uint64_t *q_len,
                                        const uint64_t *k_start, const uint64_t *k_len, size_t n_seq, int sms) {
  std::vector<XAttnItem> items;
  for (size_t i = 0; i < n_seq; ++i) {
    const int64_t rows = (int64_t)q_len[i] * (s.H / s.KVH);
    for (int g = 0; g < s.KVH; ++g)
      for (int64_t r0 = 0; r0 < rows; r0 += kRows)
        items.push_back(XAttnItem{(int64_t)q_start[i], (int64_t)k_start[i], (int)k_len[i], (int)r0,
                                  (int)std::min<int64_t>(kRows, rows - r0), g, 0, 1, 0, 0});
  }
  return items;
}

cudaError_t cross_attn(const XAttnWork &w, const XAttnCall &c, int *err, cudaStream_t st) {
  if (w.n_items == 0) return cudaSuccess;
  if (w.s.dtype == DT_F16)
    cross_attn_rows_kernel<__half><<<w.n_items, 32 * kRows, 0, st>>>(w, c);
  else
    cross_attn_rows_kernel<__nv_bfloat16><<<w.n_items, 32 * kRows, 0, st>>>(w, c);
  return cudaGetLastError();
}

}  // namespace ndl
