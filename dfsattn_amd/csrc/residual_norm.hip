// What stands between two branches of a transformer block, in one pass:
//   r = round(a x + g P(y))            P: none, RMS or layer norm with its weight
//   h = round((N(r) w + b) (1 + s) + t)  N: RMS or layer norm of r as it is stored
// x, y, r, h bf16 or f16 rows of C channels; gate g, scale s and shift t fp32,
// one vector for so many consecutive rows; weights and biases one vector. h
// leaves as it is or as 8-bit operand (fp8_block.h). Statistics are fp32 over
// the values held in registers: mean first, then the mean of squares about it.
// Products and sums are rounded one by one, in the order written, so with no
// P and a = 1 the results are those of gated_residual and adaln_modulate.
#include "fp8_block.h"
#include "lds_copy.h"

namespace dfs {
namespace {

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

// Eight values from channel e on, any address; EDGE: rows may end inside them.
// Values behind the row's end are zeros (16 bits) or any (fp32).
template <bool EDGE>
__device__ __forceinline__ uint4 load8_u16(const uint16_t* row, int e, int C) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (!EDGE || e + 8 <= C) {
    typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    const u32x4u t = __builtin_nontemporal_load(reinterpret_cast<const u32x4u*>(row + e));
    v = make_uint4(t.x, t.y, t.z, t.w);
  } else {
    uint16_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = row[min(e + i, C - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = e + i < C ? t[i] : 0;
    __builtin_memcpy(&v, t, 16);
  }
  return v;
}
template <bool EDGE>
__device__ __forceinline__ void load8_f32(const float* p, int e, int C, float* v) {
  if (!EDGE || e + 8 <= C) {
    __builtin_memcpy(v, p + e, 32);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[min(e + i, C - 1)];
  }
}
template <bool EDGE>
__device__ __forceinline__ void load8_weight(const Weight& w, int e, int C, float* v) {
  if (w.dtype == DFS_DTYPE_F32) return load8_f32<EDGE>(static_cast<const float*>(w.at), e, C, v);
  const uint16_t* const p = static_cast<const uint16_t*>(w.at);
  uint4 t;
  if (!EDGE || e + 8 <= C)
    __builtin_memcpy(&t, p + e, 16);
  else
    t = load8_u16<true>(p, e, C);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = w.dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(u16_at(t, i)) : f16_bits_to_f32(u16_at(t, i));
}
template <bool EDGE>
__device__ __forceinline__ void store8_u16(uint16_t* row, int e, int C, const uint4& v) {
  if (!EDGE || e + 8 <= C) {
    typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    const u32x4u t = {v.x, v.y, v.z, v.w};
    __builtin_nontemporal_store(t, reinterpret_cast<u32x4u*>(row + e));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < C) row[e + i] = static_cast<uint16_t>(u16_at(v, i));
  }
}
template <bool EDGE>
__device__ __forceinline__ void store8_u8(uint8_t* row, int e, int C, const uint2& v) {
  if (!EDGE || e + 8 <= C) {
    __builtin_memcpy(row + e, &v, 8);
  } else {
    uint8_t b[8];
    __builtin_memcpy(b, &v, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < C) row[e + i] = b[i];
  }
}

// Mean (0 for RMS) and 1 / sqrt(mean square about it + eps) of a row of C
// channels, eight of v[j] a lane and chunk, zeros behind its end.
template <int NCH, bool F16, bool EDGE>
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
        if (!EDGE || j * 512 + lane * 8 + i < C) sq += d * d;
      }
    }
  }
  rstd = 1.0f / sqrtf(wave_sum(sq) / static_cast<float>(C) + eps);
}

// One wave per RPW rows (16-byte chunks, 512 channels per wave step, the rows
// held in registers), as in the layer norm kernel of dit_fused.hip.
template <int NCH, bool F16, bool POST, bool EDGE, int RPW>
__global__ void __launch_bounds__(256) residual_norm_kernel(NormParams p) {
  const int lane = threadIdx.x & 63, C = p.C;
  const int row0 = __builtin_amdgcn_readfirstlane((blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW);
  if (row0 >= p.rows) return;
  uint4 v[RPW][NCH];
#pragma unroll
  for (int q = 0; q < RPW; ++q) {
    const int row = min(row0 + q, p.rows - 1);  // a missing second row repeats the last
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 512 + lane * 8;
      v[q][j] = make_uint4(0, 0, 0, 0);
      if (e < C) v[q][j] = load8_u16<EDGE>(p.x + row * p.ldx, e, C);
    }
  }
  const float* const gate = p.gate.at ? p.gate.at + row0 / p.gate.rows * p.gate.stride : nullptr;
  if (p.y) {
    uint4 y[RPW][NCH];
#pragma unroll
    for (int q = 0; q < RPW; ++q) {
      const int row = min(row0 + q, p.rows - 1);
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int e = j * 512 + lane * 8;
        y[q][j] = make_uint4(0, 0, 0, 0);
        if (e < C) y[q][j] = load8_u16<EDGE>(p.y + row * p.ldy, e, C);
      }
    }
    float mean[RPW], rstd[RPW];
    if constexpr (POST) {
#pragma unroll
      for (int q = 0; q < RPW; ++q)
        statistics<NCH, F16, EDGE>(y[q], lane, C, p.post == DFS_NORM_LAYER, p.post_eps, mean[q], rstd[q]);
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 512 + lane * 8;
      if (e >= C) continue;
      float g[8], w[8], b[8];
      if (gate) load8_f32<EDGE>(gate, e, C, g);
      if (POST && p.post_weight.at) load8_weight<EDGE>(p.post_weight, e, C, w);
      if (POST && p.post_bias.at) load8_weight<EDGE>(p.post_bias, e, C, b);
#pragma unroll
      for (int q = 0; q < RPW; ++q) {
        uint32_t packed[4];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          uint32_t r[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma clang fp contract(off)
            float f = to_f32<F16>(u16_at(y[q][j], i + t));
            if constexpr (POST) {
              f = (f - mean[q]) * rstd[q];
              if (p.post_weight.at) f = f * w[i + t];
              if (p.post_bias.at) f = f + b[i + t];
            }
            if (gate) f = f * g[i + t];
            r[t] = from_f32<F16>(to_f32<F16>(u16_at(v[q][j], i + t)) * p.residual_scale + f);
            if (EDGE && e + i + t >= C) r[t] = 0;
          }
          packed[i / 2] = r[0] | r[1] << 16;
        }
        v[q][j] = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        if (row0 + q < p.rows) store8_u16<EDGE>(p.out + (row0 + q) * p.ldo, e, C, v[q][j]);
      }
    }
  }
  float mean[RPW], rstd[RPW];
#pragma unroll
  for (int q = 0; q < RPW; ++q)
    statistics<NCH, F16, EDGE>(v[q], lane, C, p.norm == DFS_NORM_LAYER, p.eps, mean[q], rstd[q]);
  const float* const scale = p.scale.at ? p.scale.at + row0 / p.scale.rows * p.scale.stride : nullptr;
  const float* const shift = p.shift.at ? p.shift.at + row0 / p.shift.rows * p.shift.stride : nullptr;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 512 + lane * 8;
    float w[8], b[8], sc[8], sh[8];
    if (e < C) {
      if (p.weight.at) load8_weight<EDGE>(p.weight, e, C, w);
      if (p.bias.at) load8_weight<EDGE>(p.bias, e, C, b);
      if (scale) load8_f32<EDGE>(scale, e, C, sc);
      if (shift) load8_f32<EDGE>(shift, e, C, sh);
    }
#pragma unroll
    for (int q = 0; q < RPW; ++q) {
      uint32_t packed[4];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint32_t r[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma clang fp contract(off)
          float y = (to_f32<F16>(u16_at(v[q][j], i + t)) - mean[q]) * rstd[q];
          if (p.weight.at) y = y * w[i + t];
          if (p.bias.at) y = y + b[i + t];
          if (scale) y = y * (1.0f + sc[i + t]);
          if (shift) y = y + sh[i + t];
          r[t] = from_f32<F16>(y);
          if (EDGE && e + i + t >= C) r[t] = 0;
        }
        packed[i / 2] = r[0] | r[1] << 16;
      }
      const uint4 out = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      const int row = row0 + q;
      if (p.h8) {  // a scale's 128 channels are sixteen lanes'
        const uint4 values[1] = {e < C ? out : make_uint4(0, 0, 0, 0)};
        uint2 codes[1];
        const uint32_t byte = encode<F16, 16, 1>(values, codes);
        if (e < C && row < p.rows) {
          store8_u8<EDGE>(p.h8 + row * p.ldh, e, C, codes[0]);
          if ((lane & 15) == 0) p.h8_scales[(e >> 7) * p.lds + row] = static_cast<uint8_t>(byte);
        }
      } else if (e < C && row < p.rows) {
        store8_u16<EDGE>(p.h + row * p.ldh, e, C, out);
      }
    }
  }
}

template <int NCH, bool POST, bool EDGE, int RPW>
void launch_as(const NormParams& p, bool f16, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.rows + 4 * RPW - 1) / (4 * RPW)));
  if (f16)
    residual_norm_kernel<NCH, true, POST, EDGE, RPW><<<grid, 256, 0, s>>>(p);
  else
    residual_norm_kernel<NCH, false, POST, EDGE, RPW><<<grid, 256, 0, s>>>(p);
}

template <int NCH, bool EDGE>
void launch(const NormParams& p, bool f16, hipStream_t s) {
  if (p.post != DFS_NORM_NONE)
    launch_as<NCH, true, EDGE, 1>(p, f16, s);
  else
    launch_as<NCH, false, EDGE, 1>(p, f16, s);
}

}  // namespace
}  // namespace dfs

extern "C" int dfs_residual_norm(const dfs_residual_norm_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "residual_norm";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  const int64_t rows = a->rows, C = a->channels;
  DFS_REQUIRE(a->x && (a->y == nullptr) == (a->out == nullptr) && (a->h != nullptr) != (a->h8 != nullptr) &&
                  (a->h8 == nullptr) == (a->h8_scales == nullptr),
              "%s: x and h, or h8 with its scales, must be non-NULL, and y and out go together", name);
  DFS_REQUIRE(rows > 0 && rows < (int64_t(1) << 26) && C > 0 && C <= 512 * kMaxChunks,
              "%s: rows=%lld channels=%lld must be positive, below 2^26 and up to %d", name, (long long)rows,
              (long long)C, 512 * kMaxChunks);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(a->norm == DFS_NORM_RMS || a->norm == DFS_NORM_LAYER, "%s: norm code %lld is not supported", name,
              (long long)a->norm);
  DFS_REQUIRE(a->post_norm >= DFS_NORM_NONE && a->post_norm <= DFS_NORM_LAYER, "%s: norm code %lld is not supported",
              name, (long long)a->post_norm);
  DFS_REQUIRE(a->y || (!a->gate && a->post_norm == DFS_NORM_NONE), "%s: a gate or norm of y without it", name);
  DFS_REQUIRE(a->post_norm != DFS_NORM_NONE || (!a->post_weight && !a->post_bias), "%s: a weight without its norm", name);
  DFS_REQUIRE(a->eps >= 0. && a->post_eps >= 0., "%s: eps must not be negative", name);
  DFS_REQUIRE(a->x_stride >= 0 && a->y_stride >= 0 && (!a->out || a->out_stride >= C) && a->h_stride >= C &&
                  (!a->h8 || a->h8_scales_stride >= rows),
              "%s: strides must not be negative, the results' rows must not overlap", name);
  auto addr = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  DFS_REQUIRE((addr(a->x) | addr(a->y) | addr(a->out) | addr(a->h)) % 2 == 0, "%s: operands must be aligned to their elements",
              name);
  NormParams p{};
  const struct {
    const float* at;
    int64_t rows, stride;
    Vector* to;
  } vectors[3] = {{a->gate, a->gate_rows, a->gate_stride, &p.gate},
                  {a->scale, a->scale_rows, a->scale_stride, &p.scale},
                  {a->shift, a->shift_rows, a->shift_stride, &p.shift}};
  for (const auto& v : vectors) {
    if (!v.at) continue;
    DFS_REQUIRE(addr(v.at) % 4 == 0 && v.rows > 0 && rows % v.rows == 0 && v.stride >= 0,
                "%s: a vector for %lld of %lld rows each, stride %lld", name, (long long)v.rows, (long long)rows,
                (long long)v.stride);
    *v.to = Vector{v.at, v.stride, static_cast<uint32_t>(v.rows)};
  }
  const struct {
    const void* at;
    int64_t dtype;
    Weight* to;
  } weights[4] = {{a->post_weight, a->post_weight_dtype, &p.post_weight},
                  {a->post_bias, a->post_bias_dtype, &p.post_bias},
                  {a->weight, a->weight_dtype, &p.weight},
                  {a->bias, a->bias_dtype, &p.bias}};
  for (const auto& w : weights) {
    if (!w.at) continue;
    DFS_REQUIRE(w.dtype >= DFS_DTYPE_BF16 && w.dtype <= DFS_DTYPE_F32 && addr(w.at) % (w.dtype == DFS_DTYPE_F32 ? 4 : 2) == 0,
                "%s: weight dtype code %lld, or its alignment, is not supported", name, (long long)w.dtype);
    *w.to = Weight{w.at, static_cast<int>(w.dtype)};
  }
  p.x = static_cast<const uint16_t*>(a->x);
  p.y = static_cast<const uint16_t*>(a->y);
  p.out = static_cast<uint16_t*>(a->out);
  p.h = static_cast<uint16_t*>(a->h);
  p.h8 = static_cast<uint8_t*>(a->h8);
  p.h8_scales = static_cast<uint8_t*>(a->h8_scales);
  p.ldx = a->x_stride;
  p.ldy = a->y_stride;
  p.ldo = a->out_stride;
  p.ldh = a->h_stride;
  p.lds = a->h8_scales_stride;
  p.rows = static_cast<int>(rows);
  p.C = static_cast<int>(C);
  p.post = static_cast<int>(a->post_norm);
  p.norm = static_cast<int>(a->norm);
  p.residual_scale = static_cast<float>(a->residual_scale);
  p.eps = static_cast<float>(a->eps);
  p.post_eps = static_cast<float>(a->post_eps);
  const bool f16 = a->dtype == DFS_DTYPE_F16;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (C % 8 == 0) {
    switch ((C + 1023) / 1024) {  // smallest even count of chunks of 512 channels that covers the row
      case 1: launch<2, false>(p, f16, st); break;
      case 2: launch<4, false>(p, f16, st); break;
      case 3: launch<6, false>(p, f16, st); break;
      case 4: launch<8, false>(p, f16, st); break;
      case 5: launch<10, false>(p, f16, st); break;
      case 6: launch<12, false>(p, f16, st); break;
      case 7: launch<14, false>(p, f16, st); break;
      default: launch<16, false>(p, f16, st); break;
    }
  } else if (C <= 1024) {
    launch<2, true>(p, f16, st);
  } else if (C <= 2048) {
    launch<4, true>(p, f16, st);
  } else if (C <= 4096) {
    launch<8, true>(p, f16, st);
  } else {
    launch<16, true>(p, f16, st);
  }
  return check_launch(name);
}
