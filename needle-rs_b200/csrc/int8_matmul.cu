// int8_matmul.cu — product of 8-bit integers with a scale for each token and
// each output channel:
//   y[m][n] = (sum_k q[m][k] w[n][k]) * (sq[m] * sw[n]) + bias[n]
// The sum is exact in 32-bit integers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "ops.h"
#include "quant8.cuh"

namespace ndl {
namespace {

template <typename T>
__device__ __forceinline__ uint32_t abs_bits(T v) {
  return __float_as_uint((float)v) & 0x7fffffffu;
}

// One block a row: two passes over it (the second hits L1/L2).
template <typename T>
__global__ void quantize_rows_kernel(const T *x, int64_t K, int64_t ldx, int8_t *q, int64_t Kp, float *scales) {
  __shared__ uint32_t sm[32];
  const int64_t row = blockIdx.x;
  x += row * ldx;
  q += row * Kp;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x; i < K; i += blockDim.x) top = max(top, abs_bits(x[i]));
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = top;
  __syncthreads();
  top = (threadIdx.x & 31) < (blockDim.x >> 5) ? sm[threadIdx.x & 31] : 0u;
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const RowScale rs = int8_row_scale(top);
  for (int64_t i = threadIdx.x; i < Kp; i += blockDim.x)
    q[i] = i < K ? (int8_t)int8_round((float)x[i], rs.inv) : (int8_t)0;
  if (threadIdx.x == 0) scales[row] = rs.scale;
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

__device__ __forceinline__ void store_y(const Int8Args &a, int64_t m, int n, float v) {
  const int64_t i = m * a.ldy + n;
  if (a.y_dtype == DT_F32)
    ((float *)a.y)[i] = v;
  else if (a.y_dtype == DT_F16)
    ((__half *)a.y)[i] = __float2half_rn(v);
  else
    ((__nv_bfloat16 *)a.y)[i] = __float2bfloat16_rn(v);
}

// A thread for each output, four products an instruction.
__global__ void int8_dot_kernel(Int8Args a) {
  const int n = blockIdx.x * 32 + threadIdx.x;
  const int64_t m = (int64_t)blockIdx.y * 8 + threadIdx.y;
  if (n >= a.N || m >= a.M) return;
  const int64_t Kp = int8_row_bytes(a.K);
  const int8_t *q = a.q + m * Kp, *w = a.w + n * Kp;
  int acc = 0;
  for (int k = 0; k < a.K / 4 * 4; k += 4) acc = __dp4a(*(const int *)(q + k), *(const int *)(w + k), acc);
  for (int k = a.K / 4 * 4; k < a.K; ++k) acc += (int)q[k] * (int)w[k];
  const float v = __int2float_rn(acc) * (a.q_scales[m] * a.w_scales[n]);
  store_y(a, m, n, a.bias ? v + a.bias[n] : v);
}

}  // namespace

cudaError_t int8_quantize_rows(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scales,
                               cudaStream_t st) {
  const int64_t Kp = int8_row_bytes(K);
  const unsigned grid = (unsigned)M;
  if (dtype == DT_F32)
    quantize_rows_kernel<<<grid, 256, 0, st>>>((const float *)x, K, ldx, q, Kp, scales);
  else if (dtype == DT_F16)
    quantize_rows_kernel<<<grid, 256, 0, st>>>((const __half *)x, K, ldx, q, Kp, scales);
  else
    quantize_rows_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16 *)x, K, ldx, q, Kp, scales);
  return cudaGetLastError();
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

cudaError_t int8_matmul(const Int8Args &a, int *err, cudaStream_t st) {
  const int64_t step = 65535 * 8;  // rows a grid can hold
  for (int64_t m0 = 0; m0 < a.M; m0 += step) {
    Int8Args b = a;
    b.M = (int)std::min<int64_t>(step, a.M - m0);
    b.q += m0 * int8_row_bytes(a.K);
    b.q_scales += m0;
    b.y = (char *)a.y + m0 * a.ldy * (int64_t)dtype_size(a.y_dtype);
    int8_dot_kernel<<<dim3((a.N + 31) / 32, (b.M + 7) / 8), dim3(32, 8), 0, st>>>(b);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace ndl
