// RMS norm of the heads of q and k and their rotation by positions of several
// axes (time, height, width):
//   y = x / sqrt(mean(x^2) + eps) * weight  over a head's D channels or over
//       all heads' (by the weight's length), fp32
//   (y0, y1) -> (y0 c - y1 s, y1 c + y0 s) for every pair of channels, with
//       (c, s) of the angle pos[a] * f; pair i of the n channels of axis a has
//       f = speed_a theta_a^(-2i/n)
// rounded once. Pairs are neighbours (2p, 2p + 1) or halves (p, p + D/2); the
// axes' channels follow each other over the pairs, those behind them are not
// rotated. No table: a token's D/2 angles are made by the wave that needs them
// and serve all its heads. f and the angle are 64 bits, in turns, so that the
// whole turns of a far position leave nothing behind: what is left of one goes
// to fp32's sine and cosine.
#include <cfloat>

#include "common.h"
#include "lds_copy.h"

namespace dfs {
namespace {

constexpr int kMaxChunks = 16, kMaxAxes = 4;

struct RopeParams {
  const uint16_t* x[2];  // q, k: [B][T][H][D]
  uint16_t* out[2];
  int64_t x_sb[2], x_st[2], x_sh[2], o_sb[2], o_st[2], o_sh[2];
  int heads[2];
  const void* weight[2];  // NULL: no norm
  int w_dtype[2], w_all[2];
  float eps;
  int B, T, D, log2l;  // a head has 2^log2l lanes, D / 8 of them at work
  int axes, pairs[kMaxAxes];           // pairs of channels of each axis
  double slope[kMaxAxes], turn[kMaxAxes];  // f / 2 pi = turn * 2^(slope * i)
  uint32_t size[kMaxAxes];             // of the grid's axes behind the first
  const int32_t* start;                // [B] or NULL
  const int32_t* positions;            // [B or 1][T][axes] or NULL
  int64_t p_sb, p_st;
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
// Sum over aligned groups of `lanes` lanes, the same bits in each of them.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  if (lanes >= 2) v = dpp_plus<0xB1>(v);
  if (lanes >= 4) v = dpp_plus<0x4E>(v);
  if (lanes >= 8) v = dpp_plus<0x141>(v);
  if (lanes >= 16) v = dpp_plus<0x140>(v);
  if (lanes >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if (lanes >= 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return v;
}

typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
template <bool STREAM>
__device__ __forceinline__ uint2 load_half(const uint16_t* p) {
  const u32x2_t* const q = reinterpret_cast<const u32x2_t*>(p);
  const u32x2_t t = STREAM ? __builtin_nontemporal_load(q) : *q;
  return make_uint2(t.x, t.y);
}
template <bool STREAM>
__device__ __forceinline__ void store_half(uint16_t* p, const uint2& v) {
  const u32x2_t t = {v.x, v.y};
  u32x2_t* const q = reinterpret_cast<u32x2_t*>(p);
  if constexpr (STREAM)
    __builtin_nontemporal_store(t, q);
  else
    *q = t;
}

// Four weights from element e on, a multiple of 4, in fp32.
__device__ __forceinline__ void load_weight4(const void* w, int dtype, int e, float* out) {
  if (dtype == DFS_DTYPE_F32) {
    __builtin_memcpy(out, static_cast<const float*>(w) + e, 16);
    return;
  }
  uint16_t t[4];
  __builtin_memcpy(t, static_cast<const uint16_t*>(w) + e, 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(t[i]) : f16_bits_to_f32(t[i]);
}

// One wave per token and tensor (grid y). Lane l of a head's has its pairs
// 4 l .. 4 l + 3: eight neighbouring channels, or four of either half. Values
// i and pair(i): HALVES 4 + i, else 2 i and 2 i + 1.
// Bound by memory: 75,600 x 40 heads of 128, q and k with their norms, 590 us, 5.25
// TB/s; weights loaded value by value instead of four at once took 988. STREAM:
// for tensors beyond a quarter of the last-level cache, as in residual_norm.h.
template <int NCH, bool F16, bool HALVES, bool STREAM>
__global__ void __launch_bounds__(256) axial_rope_kernel(RopeParams p) {
  __shared__ __attribute__((aligned(16))) float table[4][2][256];  // cosines, sines of a wave's token
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = blockIdx.y;
  const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + w);
  if (row >= static_cast<unsigned>(p.B) * static_cast<unsigned>(p.T)) return;  // whole waves; no barrier follows
  const int b = static_cast<int>(row / static_cast<unsigned>(p.T)), t = static_cast<int>(row) - b * p.T;
  const int lanes = 1 << p.log2l, l = lane & (lanes - 1), at_once = 64 >> p.log2l, H = p.heads[n], D = p.D;
  const bool working = l * 8 < D;
  const int c0 = HALVES ? l * 4 : l * 8, c1 = HALVES ? D / 2 + l * 4 : l * 8 + 4;  // first channels of the four and four
  const uint16_t* const src = p.x[n] + b * p.x_sb[n] + t * p.x_st[n];
  uint4 v[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int h = j * at_once + (lane >> p.log2l);
    v[j] = make_uint4(0, 0, 0, 0);
    if (working && h < H) {
      if constexpr (HALVES) {
        const uint2 lo = load_half<STREAM>(src + h * p.x_sh[n] + c0), hi = load_half<STREAM>(src + h * p.x_sh[n] + c1);
        v[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      } else {
        v[j] = load_chunk<STREAM>(reinterpret_cast<const uint4*>(src + h * p.x_sh[n] + c0));
      }
    }
  }
  // The token's angles, a pair a lane.
  uint32_t place[kMaxAxes] = {};
  if (!p.positions) {
    uint32_t at = static_cast<uint32_t>(t) + (p.start ? static_cast<uint32_t>(p.start[b]) : 0u);
#pragma unroll
    for (int a = kMaxAxes - 1; a > 0; --a) {
      if (a >= p.axes) continue;
      place[a] = at % p.size[a];
      at /= p.size[a];
    }
    place[0] = at;
  }
  for (int q = lane; q < D / 2; q += 64) {
    int a = 0, i = q;
    double turn = 0., slope = 0.;
    uint32_t whole = 0;
#pragma unroll
    for (int k = 0; k < kMaxAxes; ++k) {
      if (k >= p.axes) break;
      if (i >= 0 && i < p.pairs[k]) {
        a = k;
        turn = p.turn[k] * exp2(p.slope[k] * i);
        whole = place[k];
        i = -1;
      }
      i -= i >= 0 ? p.pairs[k] : 0;
    }
    double angle = whole;
    if (p.positions) angle = p.positions[b * p.p_sb + t * p.p_st + a];
    angle *= turn;
    const float part = static_cast<float>(angle - rint(angle));  // in turns, at most a half
    float s, c;
    sincospif(2.f * part, &s, &c);
    table[w][0][q] = c;
    table[w][1][q] = s;
  }
  wait_lgkm_0();  // this wave's own table
  float cs[4] = {}, sn[4] = {};
  if (working) {
    const float4 c = *reinterpret_cast<const float4*>(&table[w][0][l * 4]);
    const float4 s = *reinterpret_cast<const float4*>(&table[w][1][l * 4]);
    cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
    sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
  }
  const void* const weight = p.weight[n];
  const bool w_all = p.w_all[n] != 0;
  const int w_dtype = p.w_dtype[n];
  float rstd[NCH], all = 0.f;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = to_f32<F16>(u16_at(v[j], i));
      ss += f * f;
    }
    rstd[j] = ss;
    all += ss;
  }
  float wt[8] = {};
  if (weight) {
    if (w_all) {
      const float r = 1.f / sqrtf(group_sum(all, 64) / static_cast<float>(H * D) + p.eps);
#pragma unroll
      for (int j = 0; j < NCH; ++j) rstd[j] = r;
    } else {
      if (working) {
        load_weight4(weight, w_dtype, c0, wt);
        load_weight4(weight, w_dtype, c1, wt + 4);
      }
#pragma unroll
      for (int j = 0; j < NCH; ++j) rstd[j] = 1.f / sqrtf(group_sum(rstd[j], lanes) / static_cast<float>(D) + p.eps);
    }
  }
  uint16_t* const dst = p.out[n] + b * p.o_sb[n] + t * p.o_st[n];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int h = j * at_once + (lane >> p.log2l);
    if (!working || h >= H) continue;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_f32<F16>(u16_at(v[j], i));
    if (weight) {
      if (w_all) {
        load_weight4(weight, w_dtype, h * D + c0, wt);
        load_weight4(weight, w_dtype, h * D + c1, wt + 4);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * rstd[j] * wt[i];
    }
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int i0 = HALVES ? i : 2 * i, i1 = HALVES ? 4 + i : 2 * i + 1;
      r[i0] = from_f32<F16>(y[i0] * cs[i] - y[i1] * sn[i]);
      r[i1] = from_f32<F16>(y[i1] * cs[i] + y[i0] * sn[i]);
    }
    const uint4 o = make_uint4(r[0] | r[1] << 16, r[2] | r[3] << 16, r[4] | r[5] << 16, r[6] | r[7] << 16);
    if constexpr (HALVES) {
      store_half<STREAM>(dst + h * p.o_sh[n] + c0, make_uint2(o.x, o.y));
      store_half<STREAM>(dst + h * p.o_sh[n] + c1, make_uint2(o.z, o.w));
    } else {
      store_chunk<STREAM>(reinterpret_cast<uint4*>(dst + h * p.o_sh[n] + c0), o);
    }
  }
}

template <int NCH, bool STREAM>
void launch_as(const RopeParams& p, bool f16, bool halves, dim3 grid, hipStream_t st) {
  if (halves)
    f16 ? axial_rope_kernel<NCH, true, true, STREAM><<<grid, 256, 0, st>>>(p)
        : axial_rope_kernel<NCH, false, true, STREAM><<<grid, 256, 0, st>>>(p);
  else
    f16 ? axial_rope_kernel<NCH, true, false, STREAM><<<grid, 256, 0, st>>>(p)
        : axial_rope_kernel<NCH, false, false, STREAM><<<grid, 256, 0, st>>>(p);
}
template <int NCH>
void launch(const RopeParams& p, bool f16, bool halves, dim3 grid, hipStream_t st) {
  const int64_t bytes = int64_t(4) * p.B * p.T * (p.heads[0] + p.heads[1]) * p.D;
  bytes > kLastLevelCache / 4 ? launch_as<NCH, true>(p, f16, halves, grid, st) : launch_as<NCH, false>(p, f16, halves, grid, st);
}

}  // namespace
}  // namespace dfs

extern "C" int dfs_axial_rope(const dfs_axial_rope_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "axial_rope";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  DFS_REQUIRE(a->q && a->q_out && (a->k == nullptr) == (a->k_out == nullptr), "%s: NULL operand", name);
  DFS_REQUIRE(a->batch > 0 && a->tokens > 0 && a->q_heads > 0 && (!a->k || a->kv_heads > 0),
              "%s: batch, tokens and heads must be positive", name);
  constexpr int64_t kMax = int64_t(1) << 30;
  DFS_REQUIRE(a->batch < kMax && a->tokens < kMax && a->batch * a->tokens < (1 << 26) - 4, "%s: too many tokens", name);
  DFS_REQUIRE(a->head_dim >= 8 && a->head_dim <= 512 && a->head_dim % 8 == 0,
              "%s: head_dim %lld must be a multiple of 8 up to 512", name, (long long)a->head_dim);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(a->axes >= 1 && a->axes <= kMaxAxes, "%s: 1 to %d axes", name, kMaxAxes);
  DFS_REQUIRE(a->eps >= 0. && a->eps <= FLT_MAX, "%s: eps must not be negative and in fp32's range", name);
  RopeParams p{};
  while ((int64_t(8) << p.log2l) < a->head_dim) ++p.log2l;
  const int64_t heads = a->k && a->kv_heads > a->q_heads ? a->kv_heads : a->q_heads;
  const int64_t chunks = (heads + (64 >> p.log2l) - 1) / (64 >> p.log2l);
  DFS_REQUIRE(chunks <= kMaxChunks, "%s: %lld heads of %lld channels (supported: %d)", name, (long long)heads,
              (long long)a->head_dim, kMaxChunks * (64 >> p.log2l));
  int64_t left = a->head_dim / 2;
  for (int i = 0; i < a->axes; ++i) {
    DFS_REQUIRE(a->pairs[i] >= 0 && a->pairs[i] <= left, "%s: the axes have more pairs of channels than a head", name);
    left -= a->pairs[i];
    p.pairs[i] = static_cast<int>(a->pairs[i]);
    p.turn[i] = a->turn[i];
    p.slope[i] = a->slope[i];
    DFS_REQUIRE(a->positions || i == 0 || (a->size[i] > 0 && a->size[i] < kMax), "%s: axis %d of the grid has size %lld",
                name, i, (long long)a->size[i]);
    p.size[i] = static_cast<uint32_t>(a->positions || i == 0 ? 1 : a->size[i]);
  }
  p.axes = static_cast<int>(a->axes);
  const void* xs[2] = {a->q, a->k};
  void* os[2] = {a->q_out, a->k_out};
  const int64_t xst[6] = {a->q_batch_stride, a->q_token_stride, a->q_head_stride, a->k_batch_stride, a->k_token_stride, a->k_head_stride};
  const int64_t ost[6] = {a->q_out_batch_stride, a->q_out_token_stride, a->q_out_head_stride,
                          a->k_out_batch_stride, a->k_out_token_stride, a->k_out_head_stride};
  const void* weights[2] = {a->q_weight, a->k_weight};
  const int64_t wd[2] = {a->q_weight_dtype, a->k_weight_dtype}, all[2] = {a->q_norm_all, a->k_norm_all};
  for (int i = 0; i < (a->k ? 2 : 1); ++i) {
    DFS_REQUIRE((reinterpret_cast<uintptr_t>(xs[i]) | reinterpret_cast<uintptr_t>(os[i])) % 16 == 0,
                "%s: operands must be 16-byte aligned", name);
    for (int j = 0; j < 3; ++j)
      DFS_REQUIRE(xst[3 * i + j] >= 0 && xst[3 * i + j] % 8 == 0 && ost[3 * i + j] >= 0 && ost[3 * i + j] % 8 == 0,
                  "%s: strides must be non-negative multiples of 8 elements", name);
    p.x[i] = static_cast<const uint16_t*>(xs[i]);
    p.out[i] = static_cast<uint16_t*>(os[i]);
    p.x_sb[i] = xst[3 * i]; p.x_st[i] = xst[3 * i + 1]; p.x_sh[i] = xst[3 * i + 2];
    p.o_sb[i] = ost[3 * i]; p.o_st[i] = ost[3 * i + 1]; p.o_sh[i] = ost[3 * i + 2];
    p.heads[i] = static_cast<int>(i == 0 ? a->q_heads : a->kv_heads);
    if (!weights[i]) continue;
    DFS_REQUIRE(wd[i] >= DFS_DTYPE_BF16 && wd[i] <= DFS_DTYPE_F32 &&
                    reinterpret_cast<uintptr_t>(weights[i]) % (wd[i] == DFS_DTYPE_F32 ? 4 : 2) == 0,
                "%s: weight dtype code %lld, or its alignment, is not supported", name, (long long)wd[i]);
    p.weight[i] = weights[i];
    p.w_dtype[i] = static_cast<int>(wd[i]);
    p.w_all[i] = all[i] != 0;
  }
  p.eps = static_cast<float>(a->eps);
  p.B = static_cast<int>(a->batch);
  p.T = static_cast<int>(a->tokens);
  p.D = static_cast<int>(a->head_dim);
  p.start = a->start;
  p.positions = a->positions;
  p.p_sb = a->positions_batch_stride;
  p.p_st = a->positions_token_stride;
  const dim3 grid(static_cast<unsigned>((a->batch * a->tokens + 3) / 4), a->k ? 2 : 1);
  const bool f16 = a->dtype == DFS_DTYPE_F16, halves = a->halves != 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (chunks <= 1) launch<1>(p, f16, halves, grid, st);
  else if (chunks <= 2) launch<2>(p, f16, halves, grid, st);
  else if (chunks <= 4) launch<4>(p, f16, halves, grid, st);
  else if (chunks <= 6) launch<6>(p, f16, halves, grid, st);
  else if (chunks <= 8) launch<8>(p, f16, halves, grid, st);
  else if (chunks <= 10) launch<10>(p, f16, halves, grid, st);
  else if (chunks <= 12) launch<12>(p, f16, halves, grid, st);
  else launch<16>(p, f16, halves, grid, st);
  return check_launch(name);
}
