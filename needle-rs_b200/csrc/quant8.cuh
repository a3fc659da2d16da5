// quant8.cuh — rounding of a row to 8 bits, shared by the kernels that write
// quantised rows.
//
// top = max|x|, scale = top / 127, value = rint(x * (127 / top)): every
// operation is rounded to f32, so each kernel (and any caller that follows
// the formula) gets the same values bit for bit.
#pragma once
#include <stdint.h>

namespace ndl {

struct RowScale {
  float scale, inv;
};

// top: the row's largest |x| as the bits of an f32 (infinities and NaN compare
// above every finite value).
__device__ __forceinline__ RowScale int8_row_scale(uint32_t top) {
  RowScale r;
  if (top >= 0x7f800000u) {  // an infinity or NaN: zeros with scale NaN
    r.scale = __uint_as_float(0x7fc00000u);
    r.inv = 0.0f;
  } else {
    const float t = __uint_as_float(top);
    // below 127 * 2^-126 the scale would be subnormal: the row counts as zero
    const bool some = t >= 127.0f * 1.17549435e-38f;
    r.scale = some ? __fdiv_rn(t, 127.0f) : 0.0f;
    r.inv = some ? __fdiv_rn(127.0f, t) : 0.0f;
  }
  return r;
}

// |x * inv| is at most 127 (1 + 2^-23), which rounds to 127: no clamp.  A row
// with an infinity or NaN has inv = 0 and becomes zeros: infinity * 0 is NaN,
// which __float2int_rn turns into 0.
__device__ __forceinline__ int int8_round(float x, float inv) { return __float2int_rn(__fmul_rn(x, inv)); }

__device__ __forceinline__ uint32_t int8_pack4(const float *x, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= ((uint32_t)int8_round(x[j], inv) & 0xffu) << (8 * j);
  return w;
}

}  // namespace ndl
