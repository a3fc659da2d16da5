// verify.cu — drafted tokens checked against the target's logits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ops.h"

namespace ndl {
namespace {

constexpr int kThreads = 256;

// Whether entry v of a row may be taken: its mask bit, and a logit above minus infinity.
__device__ __forceinline__ bool allowed(const uint64_t *mask, int v) { return !mask || ((mask[v >> 6] >> (v & 63)) & 1); }

template <typename F>
__device__ double block_reduce(double x, F f) {
  __shared__ double sm[kThreads];
  __syncthreads();
  sm[threadIdx.x] = x;
  __syncthreads();
  for (int n = kThreads / 2; n > 0; n >>= 1) {
    if (threadIdx.x < n) sm[threadIdx.x] = f(sm[threadIdx.x], sm[threadIdx.x + n]);
    __syncthreads();
  }
  return sm[0];
}

// A block for each request, one row after another.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyCall c, VerifyShape s, int *bad) {
  const int i = blockIdx.x, a = c.start[i], n = c.start[i + 1] - a, tid = threadIdx.x;
  uint32_t *out = c.out_ids + (int64_t)i * c.ld_out;
  float *logp = c.logprobs ? c.logprobs + (int64_t)i * c.ld_out : nullptr;
  for (int64_t j = tid; j < c.ld_out; j += kThreads) {
    out[j] = 0xffffffffu;
    if (logp) logp[j] = 0.0f;
  }
  if (a < 0 || n < 0 || a + n > c.n_drafts || n + 1 > c.ld_out) {
    if (tid == 0) *bad = 1, c.out_len[i] = 0;
    return;
  }
  __syncthreads();
  const float temp = c.temperature ? c.temperature[i] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  const double T1 = greedy ? 1.0 : (double)temp;
  const double inf = 1.0 / 0.0;
  int len = n + 1;
  for (int j = 0; j <= n; ++j) {
    const T *l = (const T *)c.logits + (int64_t)(a + i + j) * c.ldl;
    const uint64_t *mask = c.mask ? c.mask + (int64_t)(a + i + j) * c.ld_mask : nullptr;
    auto score = [&](int v) { return allowed(mask, v) && (float)l[v] != -INFINITY ? (double)(float)l[v] / T1 : -inf; };
    double top = -inf;
    bool broken = false;
    for (int v = tid; v < s.V; v += kThreads) {
      const double z = score(v);
      broken = broken || isnan(z) || z == inf;
      top = fmax(top, z);
    }
    broken = __syncthreads_or(broken);
    top = block_reduce(top, [](double x, double y) { return fmax(x, y); });
    if (broken || top == -inf) {
      len = j;
      break;
    }
    const bool last = c.flags & 1;
    double best = last ? -1.0 : (double)s.V, W = 0.0;
    for (int v = tid; v < s.V; v += kThreads) {
      const double z = score(v);
      if (z == top) best = last ? fmax(best, (double)v) : fmin(best, (double)v);
      if (z > -inf) W += exp(z - top);
    }
    best = last ? block_reduce(best, [](double x, double y) { return fmax(x, y); })
                : block_reduce(best, [](double x, double y) { return fmin(x, y); });
    W = block_reduce(W, [](double x, double y) { return x + y; });
    const uint32_t d = j < n ? c.ids[a + j] : 0xffffffffu;
    const bool known = j < n && d < (uint32_t)s.V;
    const double pd = known && score(d) > -inf ? exp(score(d) - top) / W : 0.0;
    const float *q = c.probs && j < n ? c.probs + (int64_t)(a + j) * c.ldp : nullptr;
    bool take = false;
    if (j < n) take = greedy ? (double)d == best : (double)c.accept_u[a + j] * (q && known ? (double)q[d] : 1.0) < pd;
    uint32_t token = d;
    if (!take) {
      token = (uint32_t)best;
      if (!greedy) {
        // chunks of the vocabulary, a thread each, then the thread's own
        const int per = (s.V + kThreads - 1) / kThreads, v0 = tid * per, v1 = min(v0 + per, s.V);
        __shared__ double sums[kThreads];
        __shared__ int found;
        bool rest = j < n;
        auto weight = [&](int v) {
          const double z = score(v), p = z > -inf ? exp(z - top) / W : 0.0;
          if (!rest) return p;
          return q ? fmax(p - (double)q[v], 0.0) : (uint32_t)v == d ? 0.0 : p;
        };
        double sum = 0.0, total = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
          sum = 0.0;
          for (int v = v0; v < v1; ++v) sum += weight(v);
          __syncthreads();
          sums[tid] = sum;
          if (tid == 0) found = -1;
          __syncthreads();
          total = 0.0;
          for (int u = 0; u < kThreads; ++u) total += sums[u];
          if (total > 0.0 || !rest) break;
          rest = false;
        }
        double before = 0.0;
        for (int u = 0; u < tid; ++u) before += sums[u];
        const double want = (double)c.final_u[i] * total;
        if (sum > 0.0 && before <= want) {
          double at = before;
          int pick = -1;
          for (int v = v0; v < v1 && pick < 0; ++v) {
            const double x = weight(v);
            at += x;
            if (x > 0.0 && at > want) pick = v;
          }
          if (pick >= 0) atomicMin((unsigned *)&found, (unsigned)pick);
        }
        __syncthreads();
        if (found < 0) {  // rounding: the last entry of any weight
          __syncthreads();
          if (tid == 0) found = -1;
          __syncthreads();
          int lastv = -1;
          for (int v = v0; v < v1; ++v)
            if (weight(v) > 0.0) lastv = v;
          atomicMax(&found, lastv);
          __syncthreads();
        }
        token = (uint32_t)found;
        __syncthreads();
      }
      len = j + 1;
    }
    if (tid == 0) {
      out[j] = token;
      if (logp) logp[j] = (float)(score(token) - top - log(W));
    }
    if (!take) break;
  }
  if (tid == 0) c.out_len[i] = len;
}

}  // namespace

cudaError_t verify_drafts(const VerifyShape &s, const VerifyCall &c, const VerifyWork &w, cudaStream_t st) {
  switch (s.dtype) {
    case DT_F32: verify_kernel<float><<<c.n_seq, kThreads, 0, st>>>(c, s, w.bad); break;
    case DT_F16: verify_kernel<__half><<<c.n_seq, kThreads, 0, st>>>(c, s, w.bad); break;
    default: verify_kernel<__nv_bfloat16><<<c.n_seq, kThreads, 0, st>>>(c, s, w.bad);
  }
  return cudaGetLastError();
}

}  // namespace ndl
