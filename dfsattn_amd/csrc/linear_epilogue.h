// What the matrix products of 16-bit and of 8-bit operands share: the epilogue
//   out[m][n] = round(residual[m][n] + gate[n] * act(sum + bias[n]))
// in fp32 with one rounding, and the order in which workgroups take tiles.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace dfs {
namespace {

constexpr uint32_t kOutside = 0x80000000u;  // byte offset past every buffer's records

enum Activation { kActNone = 0, kActGeluTanh = 1, kActGelu = 2, kActSilu = 3, kActGeluTanhShort = 4, kActGeluShort = 5 };

struct Epilogue {
  int M, N;
  int64_t ldr, ldo;
  const void* bias;  // [N] or NULL
  int bias_dtype;
  int act;
  const float* gate;         // [N] or NULL
  const uint16_t* residual;  // [M][N], row stride ldr, or NULL; may be out
  uint16_t* out;
};

typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <bool F16>
struct Half;
template <>
struct Half<false> {
  typedef bf16x8 vec;
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint32_t bits) { return bf16_bits_to_f32(bits); }
  static __device__ __forceinline__ uint32_t from_f32(float v) { return f32_to_bf16_bits(v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {  // one v_cvt_pk, a in the low half
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, pair));
  }
};
template <>
struct Half<true> {
  typedef f16x8 vec;
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint32_t bits) { return f16_bits_to_f32(bits); }
  static __device__ __forceinline__ uint32_t from_f32(float v) { return f32_to_f16_bits(v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, pair));
  }
};

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  // sigmoid(t) = 1 / (1 + e^-t); 0.5 (1 + tanh u) = sigmoid(2 u). e^-t may
  // overflow to infinity: its reciprocal is 0 then.
  if constexpr (ACT == kActGeluTanh) {
    const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
    return z * __builtin_amdgcn_rcpf(1.f + exp2_fast(-1.4426950408889634f * u));
  } else if constexpr (ACT == kActGeluTanhShort) {
    // The tanh form with its exponent as z (c0 + c1 z^2), two steps fewer:
    // c0 = -2 sqrt(2 / pi) log2(e), c1 = 0.044715 c0.
    return z * __builtin_amdgcn_rcpf(1.f + exp2_fast(z * __builtin_fmaf(-0.10294324f, z * z, -2.3022082f)));
  } else if constexpr (ACT == kActGeluShort) {
    // erfc(a / sqrt(2)) = t 2^(p(t) - a^2 / ln 4), t = 1 / (1 + a / sqrt(8)),
    // for a = |z|, with p fitted to erfc on a up to 17 (relative 8e-7; with the
    // exponent's roundings 2^-18.4 for z above -8, 2^-16.9 below, where bf16's
    // rounding is 2^-8 and f16's 2^-11). z erfc(-z / sqrt(2)) / 2 is z or 0 less
    // a / 2 times that; past a of 14 it is 0, and the factor stays finite.
    const float a = __builtin_fabsf(z), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35355339f, a, 1.f));
    float p = -0.27580905f;
    p = __builtin_fmaf(p, t, 1.1047108f);
    p = __builtin_fmaf(p, t, -1.4792635f);
    p = __builtin_fmaf(p, t, 0.5366208f);
    p = __builtin_fmaf(p, t, -0.07368178f);
    p = __builtin_fmaf(p, t, 0.5731423f);
    p = __builtin_fmaf(p, t, 1.4399331f);
    p = __builtin_fmaf(p, t, -1.8256538f);
    const float e = t * exp2_fast(__builtin_fmaf(-0.72134752f * z, z, p));
    return __builtin_fmaf(-0.5f * fminf(a, 64.f), e, fmaxf(z, 0.f));
  } else if constexpr (ACT == kActGelu) {
    return 0.5f * z * erfcf(-0.70710678118654752f * z);
  } else if constexpr (ACT == kActSilu) {
    return z * __builtin_amdgcn_rcpf(1.f + exp2_fast(-1.4426950408889634f * z));
  } else {
    return z;
  }
}

// f(integral_constant<ACT>) with the call's activation.
template <typename F>
__host__ __device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case kActGeluTanh: return f(std::integral_constant<int, kActGeluTanh>{});
    case kActGelu: return f(std::integral_constant<int, kActGelu>{});
    case kActSilu: return f(std::integral_constant<int, kActSilu>{});
    default: return f(std::integral_constant<int, kActNone>{});
  }
}

__device__ __forceinline__ float bias_at(const Epilogue& p, int n) {
  if (!p.bias) return 0.f;
  if (p.bias_dtype == DFS_DTYPE_F32) return static_cast<const float*>(p.bias)[n];
  const uint32_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.bias_dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// Bias and gate of eight consecutive outputs n.. (any values past N).
__device__ __forceinline__ void load_columns8(const Epilogue& p, int n, float* bias, float* gate) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = min(n + i, p.N - 1);
    bias[i] = bias_at(p, c);
    gate[i] = p.gate ? p.gate[c] : 1.f;
  }
}

// Eight consecutive outputs n.. of row m from their sums, all of them inside
// the matrix; 16-byte accesses at any 2-byte address.
template <bool F16, int ACT>
__device__ __forceinline__ void finish8_wide(const Epilogue& p, int m, int n, const float* z, const float* bias,
                                             const float* gate) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = activate<ACT>(z[i] + bias[i]);
  if (p.gate) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= gate[i];
  }
  if (p.residual) {
    uint4 rv;
    __builtin_memcpy(&rv, p.residual + m * p.ldr + n, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] += Half<F16>::to_f32(u16_at(rv, i));
  }
  const uint4 packed = make_uint4(Half<F16>::pack(y[0], y[1]), Half<F16>::pack(y[2], y[3]),
                                  Half<F16>::pack(y[4], y[5]), Half<F16>::pack(y[6], y[7]));
  __builtin_memcpy(p.out + m * p.ldo + n, &packed, 16);
}

// The same at the matrix's edge.
template <bool F16, int ACT>
__device__ __forceinline__ void finish8_edge(const Epilogue& p, int m, int n, const float* z, const float* bias,
                                             const float* gate) {
  if (m >= p.M) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float y = activate<ACT>(z[i] + bias[i]) * gate[i];
    if (n + i < p.N) {
      if (p.residual) y += Half<F16>::to_f32(p.residual[m * p.ldr + n + i]);
      p.out[m * p.ldo + n + i] = static_cast<uint16_t>(Half<F16>::from_f32(y));
    }
  }
}

template <bool F16, int ACT>
__device__ __forceinline__ void finish8(const Epilogue& p, int m, int n, const float* z, const float* bias,
                                        const float* gate) {
  if (m >= p.M || n >= p.N) return;
  if (n + 8 <= p.N)
    finish8_wide<F16, ACT>(p, m, n, z, bias, gate);
  else
    finish8_edge<F16, ACT>(p, m, n, z, bias, gate);
}

// Tiles of 32 NI WN outputs by 32 MI WM rows and the places of their 16-byte
// chunks in LDS: chunk c of a row r of eight at c ^ swz(r).
template <int NI, int MI, int WN, int WM, bool F16>
struct Tile {
  static constexpr int BN = 32 * NI * WN, BM = 32 * MI * WM;
  static constexpr int kShift = NI == 1 ? 2 : NI == 2 ? 3 : 4;
  typedef typename Half<F16>::vec vec;
  static __device__ __forceinline__ int swz_w(int n) { return ((n >> 1) & 1) | ((n >> kShift) & 3) << 1; }
  static __device__ __forceinline__ int swz_x(int m) { return (m >> 1) & 7; }
};

// Tile of a workgroup: XCD i takes the i-th eighth of the tile list, which
// walks bands of 4 tile rows, so the 32 tiles an XCD has in flight share 4
// slices of x and 8 of w in its L2 (75,600 x 13,824 x 5,120: 7.92 ms, bands of
// 8 8.11, of 16 8.69, of 2 7.99).
__device__ __forceinline__ void tile_of(int id, int mt, int nt, int& tm, int& tn) {
  const int total = mt * nt, x = id & 7, i = id >> 3;
  const int lin = x * (total >> 3) + min(x, total & 7) + i;
  const int band = lin / (4 * nt), rows = min(4, mt - band * 4), at = lin - band * 4 * nt;
  tn = at / rows;
  tm = band * 4 + at - tn * rows;
}

}  // namespace
}  // namespace dfs
