// 8-bit operands with a scale for every 128 consecutive channels of a row:
//   x_i = code_i * 2^e,  code_i = e4m3(x_i * 2^-e) rounded to nearest even,
// e the smallest integer with max |x_i| <= 448 * 2^e over the block's finite
// values, from -127 to 127, and 0 for a block of zeros; values that are not
// finite become NaN, e4m3's only other. The scale is held as e + 127 in a byte
// (e8m0). With a power of two the division is exact, a code's relative error
// (2^-4 at most) is what any other scale would leave, and the matrix
// instructions apply it by themselves.
#pragma once

#include "common.h"

namespace dfs {
namespace {

constexpr int kScaleBlock = 128;

// e + 127 of a block whose largest finite magnitude is `top`. Its bits give it:
// top = 1.m * 2^p <= 1.75 * 2^8 * 2^e. fp32 subnormals have p = -127 here: they
// end at -127 as they should.
__device__ __forceinline__ uint32_t block_scale(float top) {
  const uint32_t u = __float_as_uint(top), p = u >> 23, m = u & 0x7fffffu;
  const int e = static_cast<int>(p) - 8 + (m > 0x600000u ? 1 : 0);
  return u == 0 ? 127u : static_cast<uint32_t>(e < 0 ? 0 : e);
}

// 2^-e of a scale byte (up to 254: top is finite, so e <= 120).
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// |v| where it is finite, else 0.
__device__ __forceinline__ float finite_magnitude(float v) {
  const float a = __builtin_fabsf(v);
  return a < __builtin_inff() ? a : 0.f;
}

// Eight codes of v * inverse. The product of an infinity is one, and of e4m3's
// conversion only NaN is sure to be NaN: infinities are made that first.
__device__ __forceinline__ uint2 to_codes8(const float* v, float inverse) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = v[i] * inverse;
    y[i] = __builtin_fabsf(t) < __builtin_inff() ? t : __builtin_nanf("");
  }
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true)));
}
// Largest over aligned groups of eight or sixteen lanes, in each of them
// (values not negative).
__device__ __forceinline__ float max8(float v) {
  v = dpp_max<0xB1>(v);  // quad_perm [1, 0, 3, 2]
  v = dpp_max<0x4E>(v);  // quad_perm [2, 3, 0, 1]
  return dpp_max<0x141>(v);  // row_half_mirror
}
__device__ __forceinline__ float max16(float v) { return dpp_max<0x140>(max8(v)); }  // row_mirror

}  // namespace

// Enqueues the quantisation of `rows` rows of k 16-bit values (row strides in
// elements) into codes (row stride ldv bytes, zeros from k up to `fill`) and
// scale bytes (block stride lds, the rows of a block one behind the other).
void launch_quantize(const uint16_t* x, int64_t rows, int64_t k, int64_t ldx, bool f16, uint8_t* values, int64_t ldv,
                     int64_t fill, uint8_t* scales, int64_t lds, hipStream_t stream);

}  // namespace dfs
