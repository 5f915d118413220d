// Matrix products of 8-bit operands (linear_fp8.hip): arguments and matrix
// instructions.
#pragma once

#include "fp8_block.h"
#include "lds_copy.h"
#include "linear_epilogue.h"

namespace dfs {

struct Fp8Params : Epilogue {
  const uint8_t *x, *w;    // codes [M][K], [N][K], row strides ldx, ldw
  const uint8_t *xs, *ws;  // scale bytes [kb][M], [kb][N], block strides ldxs, ldws
  int64_t ldx, ldw, ldxs, ldws;
  int K, kb;
  // The channels of a tile are cut into `splits` parts of `depth` (a multiple of
  // 256); a part's sums go to part [split][M][ceil(N / 8) * 8] in fp32. Of the
  // 256 x 256 tiles the first `whole` are not cut, the others' sums go to part
  // [split][tile][256][256].
  int splits, depth, whole;
  float* part;
  // 256 x 256 tiles: the result as codes and scales [ceil(N / 128)][M], or NULL.
  uint8_t *out8, *out8_scales;
  int64_t ldo8, ldos;
};

// The 256 x 256 tiles of a product (and the join of those in parts), for each
// type of result: they are compiled apart.
void run_fp8_large_bf16(const Fp8Params& p, int64_t rest, hipStream_t stream);
void run_fp8_large_f16(const Fp8Params& p, int64_t rest, hipStream_t stream);

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 chunk_at(const uint8_t* p) { return *reinterpret_cast<const i32x4*>(p); }
__device__ __forceinline__ i32x8 join(i32x4 lo, i32x4 hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// sa, sb: the scales of the lane's rows.
__device__ __forceinline__ f32x16 mfma32(i32x8 a, i32x8 b, f32x16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, static_cast<int>(sa), 0,
                                                         static_cast<int>(sb));
}
__device__ __forceinline__ f32x4 mfma16(i32x8 a, i32x8 b, f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, static_cast<int>(sa), 0,
                                                          static_cast<int>(sb));
}

// with_activation with GELU in its short forms: these products take half the
// time, so their epilogues count for twice as much.
template <typename F>
__host__ __device__ __forceinline__ void with_fp8_activation(int act, F&& f) {
  if (act == kActGeluTanh) return f(std::integral_constant<int, kActGeluTanhShort>{});
  if (act == kActGelu) return f(std::integral_constant<int, kActGeluShort>{});
  with_activation(act, f);
}

}  // namespace
}  // namespace dfs
