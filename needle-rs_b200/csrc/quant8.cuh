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
// with inv = 0 (all zero, or with an infinity or NaN) becomes zeros.  Adding
// 1.5 * 2^23 to a product rounds it to an integer, half to even, and leaves that
// integer's low bits in the sum's: one addition instead of a conversion.
__device__ __forceinline__ uint32_t int8_low(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}
__device__ __forceinline__ int8_t int8_round(float x, float inv) {
  return inv == 0.0f ? (int8_t)0 : (int8_t)(int8_low(x, inv) & 0xffu);
}
__device__ __forceinline__ uint32_t int8_pack4(const float *x, float inv) {
  const uint32_t a = __byte_perm(int8_low(x[0], inv), int8_low(x[1], inv), 0x0040);
  const uint32_t b = __byte_perm(int8_low(x[2], inv), int8_low(x[3], inv), 0x0040);
  return inv == 0.0f ? 0u : __byte_perm(a, b, 0x5410);
}

}  // namespace ndl
