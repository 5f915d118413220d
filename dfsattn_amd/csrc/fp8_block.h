// 8-bit operands with a scale for every 128 consecutive channels of a row:
//   x_i = code_i * 2^e,  code_i = e4m3(x_i * 2^-e) rounded to nearest even,
// e the smallest integer with max |x_i| <= 448 * 2^e over the block's finite
// values, from -127 to 127, and 0 for a block of zeros; values that are not
// finite become NaN, e4m3's only other. The scale is held as e + 127 in a byte
// (e8m0). A code is off by 2^-4 of its value at most, or, for values below 2^-6 *
// 2^e, whose codes are subnormal, by 2^-10 * 2^e: what lies below that beside one
// large channel becomes zero. With a power of two the division is exact, the error
// of normal codes is what any other scale would leave, and the matrix
// instructions apply it by themselves.
#pragma once

#include "common.h"

namespace dfs {

constexpr int kScaleBlock = 128;

// Rows of k codes at any address and stride, laid out in rows of `wide` on 16-byte
// boundaries, zeros behind the k.
struct PadCodes {
  const uint8_t* src;
  int64_t ld, rows;
  int k, wide;
  uint8_t* dst;
};

namespace {

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
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true)));
}
// Largest over aligned groups of 8 or 16 lanes, in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  static_assert(LANES == 8 || LANES == 16, "half a row of lanes or a whole one");
  v = dpp_max<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v = dpp_max<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v = dpp_max<0x141>(v);  // row_half_mirror
  return LANES == 16 ? dpp_max<0x140>(v) : v;  // row_mirror
}

// The largest magnitude of eight 16-bit values, as its bits: both types order
// as integers.
__device__ __forceinline__ uint32_t top_bits8(const uint4& v) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  auto mag = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7fff7fffu); };
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(v.x), mag(v.y)),
                                            __builtin_elementwise_max(mag(v.z), mag(v.w)));
  return max(static_cast<uint32_t>(m.x), static_cast<uint32_t>(m.y));
}

// Eight codes of finite 16-bit values under a scale byte of 1 at least.
template <bool F16>
__device__ __forceinline__ uint2 to_codes8_scaled(const uint4& v, uint32_t scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const float s = __uint_as_float(scale << 23);
  auto pair = [&](uint32_t lo, uint32_t hi) {
    s16x2 r = {0, 0};
    if constexpr (F16) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, lo), s, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, hi), s, true);
    } else {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, lo), s, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, hi), s, true);
    }
    return __builtin_bit_cast(uint32_t, r);
  };
  return make_uint2(pair(v.x, v.y), pair(v.z, v.w));
}

// A block of 128 values held by LANES neighbouring lanes, eight in each of the
// N vectors of a lane (zeros where the row has ended): its scale byte and codes.
// Magnitudes are compared as integers and the conversion takes pairs of 16-bit
// values with the scale, one instruction each for two values. Blocks with values
// that are not finite, and those with the smallest scale, whose float is no
// normal number, go the long way.
template <bool F16, int LANES, int N>
__device__ __forceinline__ uint32_t encode(const uint4 (&v)[N], uint2 (&codes)[N]) {
  static_assert(LANES * N == 16, "a block has 128 values");
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) top = max(top, top_bits8(v[k]));
  top = group_max<LANES>(top);
  uint32_t scale = block_scale(F16 ? f16_bits_to_f32(top) : bf16_bits_to_f32(top));
  if (top < (F16 ? 0x7c00u : 0x7f80u) && scale > 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) codes[k] = to_codes8_scaled<F16>(v[k], scale);
    return scale;
  }
  float f[N][8], most = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[k][i] = F16 ? f16_bits_to_f32(u16_at(v[k], i)) : bf16_bits_to_f32(u16_at(v[k], i));
      most = fmaxf(most, finite_magnitude(f[k][i]));
    }
  scale = block_scale(__uint_as_float(group_max<LANES>(__float_as_uint(most))));
#pragma unroll
  for (int k = 0; k < N; ++k) codes[k] = to_codes8(f[k], inverse_scale(scale));
  return scale;
}

// By a workgroup of 256, number `group` of `groups`: sixteen codes a thread.
__device__ __forceinline__ void pad_codes(const PadCodes& p, int64_t group, int64_t groups) {
  const int chunks = p.wide / 16;
  for (int64_t id = group * 256 + threadIdx.x; id < p.rows * chunks; id += groups * 256) {
    const int64_t r = id / chunks;
    const int c = static_cast<int>(id - r * chunks) * 16;
    const uint8_t* const s = p.src + r * p.ld;
    uint4 v;
    if (c + 16 <= p.k) {
      __builtin_memcpy(&v, s + c, 16);
    } else {
      uint8_t t[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = s[min(c + i, p.k - 1)];
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = c + i < p.k ? t[i] : 0;
      __builtin_memcpy(&v, t, 16);
    }
    *reinterpret_cast<uint4*>(p.dst + r * p.wide + c) = v;
  }
}
inline unsigned pad_groups(const PadCodes& p) {
  const int64_t groups = (p.rows * (p.wide / 16) + 255) / 256;
  return static_cast<unsigned>(groups < (1 << 20) ? groups : 1 << 20);
}

}  // namespace

// Enqueues the quantisation of `rows` rows of k 16-bit values (row strides in
// elements) into codes (row stride ldv bytes, zeros from k up to `fill`) and
// scale bytes (block stride lds, the rows of a block one behind the other), and in
// the same launch of the codes of `also`, where there are any.
void launch_quantize(const uint16_t* x, int64_t rows, int64_t k, int64_t ldx, bool f16, uint8_t* values, int64_t ldv,
                     int64_t fill, uint8_t* scales, int64_t lds, hipStream_t stream, const PadCodes* also = nullptr);

}  // namespace dfs
