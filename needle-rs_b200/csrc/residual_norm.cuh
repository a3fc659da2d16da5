// residual_norm.cuh — pieces shared by the residual norm's kernels.
#pragma once
#include "common.cuh"
#include "ops.h"
#include "rowio.cuh"

namespace ndl {

constexpr float kEps = 1e-6f;
constexpr int kStreamStages = 2;  // rows in shared memory: the current one and the next

__device__ __forceinline__ float logistic(float v) { return 1.0f / (1.0f + expf(-v)); }

// The same for a token gate read from 16 bits, by the approximate instructions (a few
// ulp and one more for each unit of |v|, below half a step of the gate's own type up to
// |v| = 90); gates of f32 take the form above.
__device__ __forceinline__ float logistic16(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(1.0f + e));
  return e;
}

// Two elements of a 32-bit word as packed f32.
template <typename T>
__device__ __forceinline__ uint64_t pair_f32(uint32_t w);
template <>
__device__ __forceinline__ uint64_t pair_f32<__nv_bfloat16>(uint32_t w) {
  return f2pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint64_t pair_f32<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  return f2pack(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t pair_bits(uint64_t v);
template <>
__device__ __forceinline__ uint32_t pair_bits<__nv_bfloat16>(uint64_t v) {
  float a, b;
  f2unpack(v, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pair_bits<__half>(uint64_t v) {
  float a, b;
  f2unpack(v, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Sum over a row's threads: its warp, or all `warps` of the block through sm
// (16-byte aligned, zero past the warps).
__device__ __forceinline__ float stream_sum(uint64_t v, int warps, float *sm) {
  float a, b;
  f2unpack(v, a, b);
  a = warp_sum(a + b);
  if (warps == 1) return a;
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = a;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < warps; i += 4) {
    const float4 f = *reinterpret_cast<const float4 *>(sm + i);
    t += (f.x + f.y) + (f.z + f.w);
  }
  return t;
}

// Many rows off 16-byte boundaries (residual_norm_any.cu), up to 8,192 elements;
// *done says whether there were enough.
cudaError_t residual_norm_any(const ResidualNormArgs &a, bool *done, cudaStream_t st);

}  // namespace ndl
