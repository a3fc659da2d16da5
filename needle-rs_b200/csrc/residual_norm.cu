// residual_norm.cu — the norms before and after a block, its gate and the
// residual in one pass.
//
//   r = a x + g post(y)      post(y) = (1 + s_post) y / sqrt(mean(y^2) + 1e-6)
//   h = (1 + s_pre) r / sqrt(mean(r^2) + 1e-6)
// and, for an 8-bit h, its row scale max|h| / 127 and rounded values.
//
// A row stays in the registers of its threads from the loads to the last
// store: 8 elements (16 bytes of a 16-bit type) a load where every row is
// aligned for that, single elements otherwise.  Each of the two or three
// statistics is one reduction over the row's threads, in f32.  Up to 1,024
// elements a warp owns a row and reduces with shuffles alone; above, a block
// does.
#include <algorithm>

#include "common.cuh"
#include "ops.h"
#include "quant8.cuh"
#include "rowio.cuh"

namespace ndl {
namespace {

constexpr float kEps = 1e-6f;
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
  float r[CH][VEC];
  if (a.y) {
    const TY *y = (const TY *)a.y + row * a.ldy;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * T + threadIdx.x) * VEC;
      if (i < d) {
        load<VEC>(y + i, r[c]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) r[c][j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss += r[c][j] * r[c][j];
    }
    float inv = 1.0f;
    if (a.post) inv = 1.0f / sqrtf(row_sum(ss, warps, sm[0]) / (float)d + kEps);
    float g = 1.0f;
    if (a.gate_kind == 1) {
      g = *(const float *)a.gate;
      if (a.sigmoid) g = 1.0f / (1.0f + expf(-g));
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * T + threadIdx.x) * VEC;
      if (i < d) {
        float xv[VEC];
        load<VEC>(x + i, xv);
        if (a.post) {
          float s[VEC];
          load<VEC>(a.post + i, s);
#pragma unroll
          for (int j = 0; j < VEC; ++j) r[c][j] = ((1.0f + s[j]) * r[c][j]) * inv;
        }
        if (a.gate_kind >= 2) {
          float gv[VEC];
          if (a.gate_kind == 2)
            load<VEC>((const float *)a.gate + i, gv);
          else
            load<VEC>((const TY *)a.gate + row * a.ldg + i, gv);
#pragma unroll
          for (int j = 0; j < VEC; ++j) r[c][j] *= a.sigmoid ? 1.0f / (1.0f + expf(-gv[j])) : gv[j];
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) r[c][j] *= g;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) r[c][j] += a.scale * xv[j];
        if (a.r) store<VEC>((TX *)a.r + row * a.ldr + i, r[c]);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * T + threadIdx.x) * VEC;
      if (i < d) load<VEC>(x + i, r[c]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[c][j] = i < d ? a.scale * r[c][j] : 0.0f;
    }
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
        h[i] = (int8_t)int8_round(r[c][0], rs.inv);
      }
    }
  }
  for (int i = d + (int)threadIdx.x; i < dp; i += T) h[i] = 0;
  if (threadIdx.x == 0) a.h_scales[row] = rs.scale;
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

template <typename TX, typename TY>
cudaError_t dispatch(const ResidualNormArgs &a, cudaStream_t st) {
  auto al = [](const void *p) { return ((uintptr_t)p & 15) == 0; };
  const bool vec = a.d % 8 == 0 && al(a.x) && al(a.y) && al(a.gate) && al(a.r) && al(a.h) && al(a.post) && al(a.pre) &&
                   a.ldx % 8 == 0 && (!a.y || a.ldy % 8 == 0) && (!a.r || a.ldr % 8 == 0) && a.ldh % 8 == 0 &&
                   (a.gate_kind != 3 || a.ldg % 8 == 0);
  if (vec) {
    if (a.d <= 256) return launch_rows<TX, TY, 8, 1>(a, st);
    if (a.d <= 4096) return launch_rows<TX, TY, 8, 2>(a, st);
    return launch_rows<TX, TY, 8, 4>(a, st);
  }
  if (a.d <= 8192) return launch_rows<TX, TY, 1, 8>(a, st);
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
