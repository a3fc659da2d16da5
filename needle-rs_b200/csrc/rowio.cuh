// rowio.cuh — rows of f32, f16 or bf16 elements moved in whole vectors and
// converted to and from f32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ndl {

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// VEC consecutive elements as f32 (16-byte accesses for VEC = 8).
template <int VEC, typename T>
__device__ __forceinline__ void load(const T *p, float *v) {
  if constexpr (VEC == 1) {
    v[0] = (float)*p;
  } else {
    constexpr int N = VEC * (int)sizeof(T) / 16;
    uint4 raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (float)e[i];
  }
}
template <int VEC, typename T>
__device__ __forceinline__ void store(T *p, const float *v) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(v[0]);
  } else {
    constexpr int N = VEC * (int)sizeof(T) / 16;
    alignas(16) T e[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(e)[i];
  }
}

// Rows at any byte offset, moved in 16-byte pieces.  A row of n bytes at p lies in
// shared memory from buf + (p & 15) on, so that its whole 16-byte pieces are
// aligned on both sides; the bytes before the first and behind the last whole
// piece (under 32) move as elements of E, one a thread of the last 32.  `t` of `T`
// threads each take a share.
template <typename E>
__device__ __forceinline__ void row_in(uint8_t *buf, const E *p, int n, int t, int T) {
  const int o = (int)((uintptr_t)p & 15), head = min((16 - o) & 15, n), whole = (n - head) & ~15;
  const uint8_t *g = (const uint8_t *)p + head + 16 * t;
  uint32_t s = (uint32_t)__cvta_generic_to_shared(buf) + o + head + 16 * t;
  for (int i = 16 * t; i < whole; i += 16 * T, g += 16 * T, s += 16 * T)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(g) : "memory");
  const int e = (t - T + 32) * (int)sizeof(E);
  if (e >= 0 && e < n - whole) {
    const int at = e < head ? e : e + whole;
    *reinterpret_cast<E *>(buf + o + at) = *reinterpret_cast<const E *>((const uint8_t *)p + at);
  }
}
template <typename E>
__device__ __forceinline__ void row_out(E *p, const uint8_t *buf, int n, int t, int T) {
  const int o = (int)((uintptr_t)p & 15), head = min((16 - o) & 15, n), whole = (n - head) & ~15;
  uint8_t *g = (uint8_t *)p + head + 16 * t;
  const uint8_t *s = buf + o + head + 16 * t;
  for (int i = 16 * t; i < whole; i += 16 * T, g += 16 * T, s += 16 * T)
    *reinterpret_cast<uint4 *>(g) = *reinterpret_cast<const uint4 *>(s);
  const int e = (t - T + 32) * (int)sizeof(E);
  if (e >= 0 && e < n - whole) {
    const int at = e < head ? e : e + whole;
    *reinterpret_cast<E *>((uint8_t *)p + at) = *reinterpret_cast<const E *>(buf + o + at);
  }
}

// Largest of `top` over the threads of a row: `warps` warps of the block, or
// the warp alone (warps = 1); sm: a word for each warp.
__device__ __forceinline__ uint32_t row_max_bits(uint32_t top, int warps, uint32_t *sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (warps == 1) return top;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sm[warp] = top;
  __syncthreads();
  top = lane < warps ? sm[lane] : 0u;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  return top;
}

}  // namespace ndl
