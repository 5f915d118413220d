// What stands between two branches of a transformer block, in one pass:
//   r = round(a x + g P(y))            P: none, RMS or layer norm with its weight
//   h = round((N(r) w + b) (1 + s) + t)  N: RMS or layer norm of r as it is stored
// x, y, r, h bf16 or f16 rows of C channels; gate g, scale s and shift t fp32,
// one vector for so many consecutive rows; weights and biases one vector. h
// leaves as it is or as 8-bit operand (fp8_block.h). Statistics are fp32 over
// the values held in registers: mean first, then the mean of squares about it.
// Products and sums are rounded one by one, in the order written, so with no
// P and a = 1 the results are those of gated_residual and adaln_modulate.
#pragma once

#include "fp8_block.h"

namespace dfs {

constexpr int kMaxChunks = 16;  // at most 16 x 512 channels per row

struct Vector {  // [C] fp32 values for `rows` consecutive rows each, or NULL
  const float* at;
  int64_t stride;
  uint32_t rows;
};
struct Weight {  // [C] values of a type, or NULL
  const void* at;
  int dtype;
};
struct NormParams {
  const uint16_t *x, *y;  // y NULL: r is x and is not written
  uint16_t *out, *h;
  uint8_t *h8, *h8_scales;
  int64_t ldx, ldy, ldo, ldh, lds;
  int rows, C;
  int post, norm;  // DFS_NORM_*
  float residual_scale, eps, post_eps;
  Vector gate, scale, shift;
  Weight post_weight, post_bias, weight, bias;
};

// The call, its arguments checked, for each type: they are compiled apart.
void run_residual_norm_bf16(const NormParams& p, hipStream_t stream);
void run_residual_norm_f16(const NormParams& p, hipStream_t stream);

namespace {

template <bool F16>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  return F16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
}
template <bool F16>
__device__ __forceinline__ uint32_t from_f32(float v) {
  return F16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v);
}

template <int CTRL>
__device__ __forceinline__ float dpp_plus(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// Sum over the wave, the same bits in every lane (every step adds a value and
// its mirror).
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_plus<0xB1>(v);
  v = dpp_plus<0x4E>(v);
  v = dpp_plus<0x141>(v);
  v = dpp_plus<0x140>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Eight values from channel e on, any address. STREAM: nontemporal accesses, for
// rows beyond the last-level cache.
template <bool STREAM>
__device__ __forceinline__ uint4 load8_u16(const uint16_t* row, int e) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  const u32x4u* const q = reinterpret_cast<const u32x4u*>(row + e);
  const u32x4u t = STREAM ? __builtin_nontemporal_load(q) : *q;
  return make_uint4(t.x, t.y, t.z, t.w);
}
template <bool STREAM>
__device__ __forceinline__ void store8_u16(uint16_t* row, int e, const uint4& v) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  const u32x4u t = {v.x, v.y, v.z, v.w};
  u32x4u* const q = reinterpret_cast<u32x4u*>(row + e);
  if constexpr (STREAM)
    __builtin_nontemporal_store(t, q);
  else
    *q = t;
}
__device__ __forceinline__ void load8_f32(const float* p, int e, float* v) { __builtin_memcpy(v, p + e, 32); }
__device__ __forceinline__ void load8_weight(const Weight& w, int e, float* v) {
  if (w.dtype == DFS_DTYPE_F32) return load8_f32(static_cast<const float*>(w.at), e, v);
  uint4 t;
  __builtin_memcpy(&t, static_cast<const uint16_t*>(w.at) + e, 16);
  if (w.dtype == DFS_DTYPE_BF16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_bits_to_f32(u16_at(t, i));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f16_bits_to_f32(u16_at(t, i));
  }
}

// Mean (0 for RMS) and 1 / sqrt(mean square about it + eps) of a row of C
// channels, eight of v[j] a lane and chunk, zeros behind its end.
template <int NCH, bool F16>
__device__ __forceinline__ void statistics(const uint4 (&v)[NCH], int lane, int C, bool layer, float eps, float& mean,
                                           float& rstd) {
  mean = 0.f;
  if (layer) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += to_f32<F16>(u16_at(v[j], i));
    mean = wave_sum(sum) / static_cast<float>(C);
  }
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    if (j * 512 + lane * 8 < C) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = to_f32<F16>(u16_at(v[j], i)) - mean;
        sq += d * d;
      }
    }
  }
  rstd = 1.0f / sqrtf(wave_sum(sq) / static_cast<float>(C) + eps);
}

// What the steps take for eight channels: vectors that are there, as the flags of
// the call say.
struct Before {
  float gate[8], weight[8], bias[8];
};
struct After {
  float weight[8], bias[8], scale[8], shift[8];
};

// Steps of eight values each, so that a vector that is not there costs one branch.
__device__ __forceinline__ void times8(float* f, const float* w) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = f[i] * w[i];
}
__device__ __forceinline__ void plus8(float* f, const float* b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = f[i] + b[i];
}
template <bool F16>
__device__ __forceinline__ uint4 packed8(const float* f) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = from_f32<F16>(f[i]);
  return make_uint4(r[0] | r[1] << 16, r[2] | r[3] << 16, r[4] | r[5] << 16, r[6] | r[7] << 16);
}

// Eight values of r from x and y; mean, rstd: of y's norm, where there is one.
template <bool F16>
__device__ __forceinline__ uint4 residual8(const NormParams& p, const uint4& x, const uint4& y, const Before& s, bool post,
                                           float mean, float rstd) {
#pragma clang fp contract(off)
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<F16>(u16_at(y, i));
  if (post) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (f[i] - mean) * rstd;
    if (p.post_weight.at) times8(f, s.weight);
    if (p.post_bias.at) plus8(f, s.bias);
  }
  if (p.gate.at) times8(f, s.gate);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<F16>(u16_at(x, i)) * p.residual_scale + f[i];
  return packed8<F16>(f);
}

// Eight values of h from r.
template <bool F16>
__device__ __forceinline__ uint4 norm8(const NormParams& p, const uint4& v, const After& s, float mean, float rstd) {
#pragma clang fp contract(off)
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (to_f32<F16>(u16_at(v, i)) - mean) * rstd;
  if (p.weight.at) times8(y, s.weight);
  if (p.bias.at) plus8(y, s.bias);
  if (p.scale.at) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * (1.0f + s.scale[i]);
  }
  if (p.shift.at) plus8(y, s.shift);
  return packed8<F16>(y);
}

__device__ __forceinline__ const float* vector_of(const Vector& v, int row) {
  return v.at ? v.at + static_cast<uint32_t>(row) / v.rows * v.stride : nullptr;
}

// One wave per row (16-byte chunks, 512 channels per wave step, the row held in
// registers), as in the layer norm kernel of dit_fused.hip; rows of whole chunks.
// Bound by memory: 75,600 x 5,120 with gate, scale and shift 540 us, 5.75 TB/s. A
// vector that is not there costs a branch for eight values: default vectors in
// its place took 607 to 701 us, two rows a wave were slower too. STREAM, for rows
// beyond a quarter of the last-level cache (in and out together): 4,680 x 5,120
// with a post norm and quantised 62.5 us cached and 44.7 streaming among other
// work, the same rows again and again 43 and 38.6; smaller ones stay for what reads
// them next.
template <int NCH, bool F16, bool POST, bool STREAM>
__global__ void __launch_bounds__(256) residual_norm_kernel(NormParams p) {
  const int lane = threadIdx.x & 63, C = p.C;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (row >= p.rows) return;
  uint4 v[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 512 + lane * 8;
    v[j] = make_uint4(0, 0, 0, 0);
    if (e < C) v[j] = load8_u16<STREAM>(p.x + row * p.ldx, e);
  }
  const float* const gate = vector_of(p.gate, row);
  if (p.y) {
    uint4 y[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 512 + lane * 8;
      y[j] = make_uint4(0, 0, 0, 0);
      if (e < C) y[j] = load8_u16<STREAM>(p.y + row * p.ldy, e);
    }
    float mean = 0.f, rstd = 0.f;
    if constexpr (POST) statistics<NCH, F16>(y, lane, C, p.post == DFS_NORM_LAYER, p.post_eps, mean, rstd);
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 512 + lane * 8;
      if (e >= C) continue;
      Before s;
      if (gate) load8_f32(gate, e, s.gate);
      if (POST && p.post_weight.at) load8_weight(p.post_weight, e, s.weight);
      if (POST && p.post_bias.at) load8_weight(p.post_bias, e, s.bias);
      v[j] = residual8<F16>(p, v[j], y[j], s, POST, mean, rstd);
      store8_u16<STREAM>(p.out + row * p.ldo, e, v[j]);
    }
  }
  float mean, rstd;
  statistics<NCH, F16>(v, lane, C, p.norm == DFS_NORM_LAYER, p.eps, mean, rstd);
  const float *const scale = vector_of(p.scale, row), *const shift = vector_of(p.shift, row);
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 512 + lane * 8;
    After s;
    if (e < C) {
      if (p.weight.at) load8_weight(p.weight, e, s.weight);
      if (p.bias.at) load8_weight(p.bias, e, s.bias);
      if (scale) load8_f32(scale, e, s.scale);
      if (shift) load8_f32(shift, e, s.shift);
    }
    const uint4 h = norm8<F16>(p, v[j], s, mean, rstd);
    if (p.h8) {  // a scale's 128 channels are sixteen lanes'
      const uint4 values[1] = {e < C ? h : make_uint4(0, 0, 0, 0)};
      uint2 codes[1];
      const uint32_t byte = encode<F16, 16, 1>(values, codes);
      if (e < C) {
        __builtin_memcpy(p.h8 + row * p.ldh + e, &codes[0], 8);
        if ((lane & 15) == 0) p.h8_scales[(e >> 7) * p.lds + row] = static_cast<uint8_t>(byte);
      }
    } else if (e < C) {
      store8_u16<STREAM>(p.h + row * p.ldh, e, h);
    }
  }
}

// Rows that end inside a chunk: a workgroup a row, chunk t + 256 k for thread t,
// with the row's last chunk taken value by value. Its sums meet in LDS, up to four
// times a row behind a barrier each, which is what bounds it: 75,600 x 5,119 with
// gate, scale and shift 1,112 us where 5,120 takes 551, 75,600 x 333 (42 threads at
// work) 219 where 336 takes 55; 4,680 x 5,119 59 and 45.
__device__ __forceinline__ uint4 part8_u16(const uint16_t* row, int e, int C) {
  if (e + 8 <= C) return load8_u16<false>(row, e);
  uint16_t t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = row[min(e + i, C - 1)];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = e + i < C ? t[i] : 0;
  uint4 v;
  __builtin_memcpy(&v, t, 16);
  return v;
}
__device__ __forceinline__ void part8_f32(const float* p, int e, int C, float* v) {
  if (e + 8 <= C) return load8_f32(p, e, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[min(e + i, C - 1)];
}
__device__ __forceinline__ void part8_weight(const Weight& w, int e, int C, float* v) {
  if (e + 8 <= C) return load8_weight(w, e, v);
  if (w.dtype == DFS_DTYPE_F32) return part8_f32(static_cast<const float*>(w.at), e, C, v);
  const uint4 t = part8_u16(static_cast<const uint16_t*>(w.at), e, C);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = w.dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(u16_at(t, i)) : f16_bits_to_f32(u16_at(t, i));
}
// The first n of eight values, zeros behind them.
__device__ __forceinline__ uint4 first_of(const uint4& v, int n) {
  auto keep = [&](uint32_t w, int i) { return n >= 2 * i + 2 ? w : n == 2 * i + 1 ? w & 0xffffu : 0u; };
  return make_uint4(keep(v.x, 0), keep(v.y, 1), keep(v.z, 2), keep(v.w, 3));
}
template <typename T, typename V>
__device__ __forceinline__ void part8_store(T* row, int e, int C, const V& v) {  // eight values of T
  if (e + 8 <= C) {
    __builtin_memcpy(row + e, &v, sizeof(V));
  } else {
    T t[8];
    __builtin_memcpy(t, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < C) row[e + i] = t[i];
  }
}

template <int NCH, bool F16>
__global__ void __launch_bounds__(256) residual_norm_part_kernel(NormParams p) {
  __shared__ float sums[4][4];  // of each of four reductions and waves
  const int t = threadIdx.x, C = p.C, row = blockIdx.x;
  auto block_sum = [&](float v, int n) {
    v = wave_sum(v);
    if ((t & 63) == 0) sums[n][t >> 6] = v;
    __syncthreads();
    return (sums[n][0] + sums[n][1]) + (sums[n][2] + sums[n][3]);
  };
  auto statistics_of = [&](const uint4 (&v)[NCH], bool layer, float eps, int n, float& mean, float& rstd) {
    mean = 0.f;
    if (layer) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += to_f32<F16>(u16_at(v[j], i));
      mean = block_sum(sum, n) / static_cast<float>(C);
    }
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = to_f32<F16>(u16_at(v[j], i)) - mean;
        sq += j * 2048 + t * 8 + i < C ? d * d : 0.f;
      }
    rstd = 1.0f / sqrtf(block_sum(sq, n + 1) / static_cast<float>(C) + eps);
  };
  uint4 v[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 2048 + t * 8;
    v[j] = make_uint4(0, 0, 0, 0);
    if (e < C) v[j] = part8_u16(p.x + row * p.ldx, e, C);
  }
  if (p.y) {
    uint4 y[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 2048 + t * 8;
      y[j] = make_uint4(0, 0, 0, 0);
      if (e < C) y[j] = part8_u16(p.y + row * p.ldy, e, C);
    }
    const bool post = p.post != DFS_NORM_NONE;
    float mean = 0.f, rstd = 0.f;
    if (post) statistics_of(y, p.post == DFS_NORM_LAYER, p.post_eps, 0, mean, rstd);
    const float* const gate = vector_of(p.gate, row);
    // In the place of x or y: every thread has read its part of both rows before.
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 2048 + t * 8;
      if (e >= C) continue;
      Before s;
      if (gate) part8_f32(gate, e, C, s.gate);
      if (p.post_weight.at) part8_weight(p.post_weight, e, C, s.weight);
      if (p.post_bias.at) part8_weight(p.post_bias, e, C, s.bias);
      v[j] = first_of(residual8<F16>(p, v[j], y[j], s, post, mean, rstd), C - e);
      part8_store(p.out + row * p.ldo, e, C, v[j]);
    }
  }
  float mean, rstd;
  statistics_of(v, p.norm == DFS_NORM_LAYER, p.eps, 2, mean, rstd);
  const float *const scale = vector_of(p.scale, row), *const shift = vector_of(p.shift, row);
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 2048 + t * 8;
    uint4 h = make_uint4(0, 0, 0, 0);
    if (e < C) {
      After s;
      if (p.weight.at) part8_weight(p.weight, e, C, s.weight);
      if (p.bias.at) part8_weight(p.bias, e, C, s.bias);
      if (scale) part8_f32(scale, e, C, s.scale);
      if (shift) part8_f32(shift, e, C, s.shift);
      h = first_of(norm8<F16>(p, v[j], s, mean, rstd), C - e);
    }
    if (p.h8) {
      const uint4 values[1] = {h};
      uint2 codes[1];
      const uint32_t byte = encode<F16, 16, 1>(values, codes);
      if (e < C) {
        part8_store(p.h8 + row * p.ldh, e, C, codes[0]);
        if ((t & 15) == 0) p.h8_scales[(e >> 7) * p.lds + row] = static_cast<uint8_t>(byte);
      }
    } else if (e < C) {
      part8_store(p.h + row * p.ldh, e, C, h);
    }
  }
}

template <bool F16, int NCH>
void launch(const NormParams& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.rows + 3) / 4));
  const bool stream = int64_t(2) * p.rows * p.C * (p.y ? 4 : 2) > kLastLevelCache / 4;
  if (p.post != DFS_NORM_NONE)
    stream ? residual_norm_kernel<NCH, F16, true, true><<<grid, 256, 0, s>>>(p)
           : residual_norm_kernel<NCH, F16, true, false><<<grid, 256, 0, s>>>(p);
  else
    stream ? residual_norm_kernel<NCH, F16, false, true><<<grid, 256, 0, s>>>(p)
           : residual_norm_kernel<NCH, F16, false, false><<<grid, 256, 0, s>>>(p);
}
template <bool F16, int NCH>
void launch_part(const NormParams& p, hipStream_t s) {
  residual_norm_part_kernel<NCH, F16><<<dim3(static_cast<unsigned>(p.rows)), 256, 0, s>>>(p);
}
template <bool F16>
void run(const NormParams& p, hipStream_t st) {
  if (p.C % 8 == 0) {
    switch ((p.C + 1023) / 1024) {  // smallest even count of chunks of 512 channels that covers the row
      case 1: launch<F16, 2>(p, st); break;
      case 2: launch<F16, 4>(p, st); break;
      case 3: launch<F16, 6>(p, st); break;
      case 4: launch<F16, 8>(p, st); break;
      case 5: launch<F16, 10>(p, st); break;
      case 6: launch<F16, 12>(p, st); break;
      case 7: launch<F16, 14>(p, st); break;
      default: launch<F16, 16>(p, st); break;
    }
  } else if (p.C <= 2048) {
    launch_part<F16, 1>(p, st);
  } else if (p.C <= 4096) {
    launch_part<F16, 2>(p, st);
  } else {
    launch_part<F16, 4>(p, st);
  }
}

}  // namespace
}  // namespace dfs
