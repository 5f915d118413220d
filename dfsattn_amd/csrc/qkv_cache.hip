// The way of new tokens into attention over a cache: RMS norm and rotation of
// the heads of q and k, with k and v appended to their sequence's cache.
//   y = x / sqrt(mean(x^2) + eps) * weight  over a head's D channels or over
//       all heads' (by the weight's length), fp32
//   (y[2i], y[2i+1]) -> (y[2i] c - y[2i+1] s, y[2i+1] c + y[2i] s) with (c, s)
//       the table's row of the token's position, fp32
// rounded once to the storage type. Token t of sequence b stands at position
// lens[b] + t; its k and v go to that slot of the cache, or, in a rolling
// cache of S slots, to pos < sinks ? pos : sinks + (pos - sinks) mod (S - sinks).
#include "common.h"

namespace dfs {
namespace {

constexpr int kMaxChunks = 16;  // at most 16 x 512 channels per row

struct CacheParams {
  const uint16_t* x[3];  // q, k, v: [B][T][H][D]
  uint16_t* out[3];      // q_out, k_cache, v_cache
  int64_t x_sb[3], x_st[3], x_sh[3];
  int64_t o_sb[3], o_st[3], o_sh[3];  // o_st: rows of q_out, slots of the caches
  int heads[3];
  const void* weight[3];  // NULL: no norm
  int w_dtype[3];
  int w_all[3];  // 1: norm over all heads' channels
  float eps;
  const float *cos_t, *sin_t;  // [table_rows][D / 2] or NULL
  int64_t table_rows;
  const int32_t *lens, *new_lens;
  int B, T, log2d, S, sinks, rolling;  // heads of 2^log2d channels
};

template <bool F16>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  return F16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
}
template <bool F16>
__device__ __forceinline__ uint32_t from_f32(float v) {
  return F16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v);
}

// Eight weights from element e on, in fp32.
__device__ __forceinline__ void load_weight8(const void* w, int dtype, int e, float* out) {
  if (dtype == DFS_DTYPE_F32) {
    const float* f = static_cast<const float*>(w) + e;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = f[i];
    return;
  }
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + e);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    out[i] = dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(u16_at(v, i)) : f16_bits_to_f32(u16_at(v, i));
}

template <int CTRL>
__device__ __forceinline__ float dpp_plus(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// Sum over aligned groups of `lanes` lanes (2 to 64), the same bits in each of
// them: register moves, every step adds a value and its mirror.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  v = dpp_plus<0xB1>(v);                   // quad_perm [1, 0, 3, 2]
  if (lanes >= 4) v = dpp_plus<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  if (lanes >= 8) v = dpp_plus<0x141>(v);  // row_half_mirror
  if (lanes >= 16) v = dpp_plus<0x140>(v);  // row_mirror
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

// One wave per token and tensor (grid y): the row of H * D channels in
// registers (16 bytes a lane and step of 512 channels; D divides 512, so a
// lane's channels lie at the same place of every head and one slice of the
// table row serves them all). Everything that does not hang on the sequence's
// length is loaded while that is on its way. Bound by memory: 3,600 tokens x 40
// heads in 41 us (223 MB, 5.4 TB/s), 65 with sums through LDS, 64-bit divisions
// and the loads behind the length; 32 single tokens 6.9 us (11.6), latency.
template <int NCH, bool F16>
__global__ void __launch_bounds__(256) qkv_cache_kernel(CacheParams p) {
  const int lane = threadIdx.x & 63, n = blockIdx.y;
  const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (row >= static_cast<unsigned>(p.B) * static_cast<unsigned>(p.T)) return;
  const int b = static_cast<int>(row / static_cast<unsigned>(p.T)), t = static_cast<int>(row) - b * p.T;
  const int len = p.lens[b], live = p.new_lens ? p.new_lens[b] : p.T;
  const int C = p.heads[n] << p.log2d;
  const int d = lane * 8 & ((1 << p.log2d) - 1);
  const uint16_t* const src = p.x[n] + b * p.x_sb[n] + t * p.x_st[n] + d;
  const int64_t x_sh = p.x_sh[n], o_sh = p.o_sh[n];
  uint4 v[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 512 + lane * 8;
    v[j] = make_uint4(0, 0, 0, 0);
    if (e < C) v[j] = *reinterpret_cast<const uint4*>(src + (e >> p.log2d) * x_sh);
  }
  const int64_t pos = static_cast<int64_t>(len) + t;
  int64_t dst_row = t;
  if (n > 0) {
    dst_row = pos;
    if (p.rolling && pos >= p.sinks)
      dst_row = p.sinks + static_cast<uint32_t>(pos - p.sinks) % static_cast<uint32_t>(p.S - p.sinks);
    if (t >= live || pos < 0 || dst_row >= p.S) return;  // a token without a slot is not kept
  }
  uint16_t* const dst = p.out[n] + b * p.o_sb[n] + dst_row * p.o_st[n] + d;
  if (n == 2 || t >= live) {  // v as it is; q rows behind the sequence are zero
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int e = j * 512 + lane * 8;
      if (e < C) *reinterpret_cast<uint4*>(dst + (e >> p.log2d) * o_sh) = n == 2 ? v[j] : make_uint4(0, 0, 0, 0);
    }
    return;
  }
  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
  if (p.cos_t) {
    const bool inside = pos >= 0 && pos < p.table_rows;
    const int64_t at = inside ? (pos << p.log2d >> 1) + (d >> 1) : 0;
    const float4 c = *reinterpret_cast<const float4*>(p.cos_t + at), s = *reinterpret_cast<const float4*>(p.sin_t + at);
    cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
    sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
    if (!inside) cs[0] = cs[1] = cs[2] = cs[3] = NAN;  // a position without a table row is not passed over silently
  }
  const void* const weight = p.weight[n];
  const bool w_all = p.w_all[n] != 0;
  const int w_dtype = p.w_dtype[n];
  float rstd[NCH];
  float all = 0.f;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = to_f32<F16>(u16_at(v[j], i));  // zeros past the row's end
      ss += f * f;
    }
    rstd[j] = ss;
    all += ss;
  }
  float w[8];
  if (weight) {
    if (w_all) {
      const float r = 1.f / sqrtf(group_sum(all, 64) / static_cast<float>(C) + p.eps);
#pragma unroll
      for (int j = 0; j < NCH; ++j) rstd[j] = r;
    } else {
      load_weight8(weight, w_dtype, d, w);
      const float inv = 1.f / static_cast<float>(1 << p.log2d);
#pragma unroll
      for (int j = 0; j < NCH; ++j) rstd[j] = 1.f / sqrtf(group_sum(rstd[j], 1 << p.log2d >> 3) * inv + p.eps);
    }
  }
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int e = j * 512 + lane * 8;
    if (e >= C) continue;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_f32<F16>(u16_at(v[j], i));
    if (weight) {
      if (w_all) load_weight8(weight, w_dtype, e, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * rstd[j] * w[i];
    }
    uint32_t packed[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float re = y[2 * i] * cs[i] - y[2 * i + 1] * sn[i], im = y[2 * i + 1] * cs[i] + y[2 * i] * sn[i];
      packed[i] = from_f32<F16>(re) | from_f32<F16>(im) << 16;
    }
    *reinterpret_cast<uint4*>(dst + (e >> p.log2d) * o_sh) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
  }
}

template <int NCH>
void launch_cache(const CacheParams& p, bool f16, dim3 grid, hipStream_t st) {
  if (f16)
    qkv_cache_kernel<NCH, true><<<grid, 256, 0, st>>>(p);
  else
    qkv_cache_kernel<NCH, false><<<grid, 256, 0, st>>>(p);
}

}  // namespace
}  // namespace dfs

extern "C" int dfs_qkv_cache(const dfs_cache_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "qkv_cache";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  DFS_REQUIRE(a->q && a->k && a->v && a->q_out && a->k_cache && a->v_cache && a->lens, "%s: NULL operand", name);
  DFS_REQUIRE(a->batch > 0 && a->tokens > 0 && a->q_heads > 0 && a->kv_heads > 0 && a->slots > 0,
              "%s: batch, tokens, heads and slots must be positive", name);
  DFS_REQUIRE(a->head_dim >= 16 && a->head_dim <= 512 && (a->head_dim & (a->head_dim - 1)) == 0,
              "%s: head_dim %lld must be a power of two from 16 to 512", name, (long long)a->head_dim);
  const int64_t widest = (a->q_heads > a->kv_heads ? a->q_heads : a->kv_heads) * a->head_dim;
  DFS_REQUIRE(a->q_heads <= 4096 && a->kv_heads <= 4096 && widest <= 512 * kMaxChunks,
              "%s: heads*head_dim = %lld exceeds %d", name, (long long)widest, 512 * kMaxChunks);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  constexpr int64_t kMax = int64_t(1) << 30;
  DFS_REQUIRE(a->batch < kMax && a->tokens < kMax && a->slots < kMax && a->batch * a->tokens < (1 << 26) - 4,
              "%s: sizes too large", name);
  DFS_REQUIRE(a->sinks >= 0, "%s: sinks must not be negative", name);
  DFS_REQUIRE(!a->rolling || a->tokens <= a->slots - a->sinks,
              "%s: %lld new tokens do not fit the %lld rolling slots", name, (long long)a->tokens,
              (long long)(a->slots - a->sinks));
  DFS_REQUIRE((a->cos_table == nullptr) == (a->sin_table == nullptr), "%s: pass both cos and sin tables or neither",
              name);
  DFS_REQUIRE(a->cos_table == nullptr ||
                  (a->table_rows > 0 && (reinterpret_cast<uintptr_t>(a->cos_table) |
                                         reinterpret_cast<uintptr_t>(a->sin_table)) % 16 == 0),
              "%s: tables must have rows and be 16-byte aligned", name);
  DFS_REQUIRE(a->eps >= 0., "%s: eps must be non-negative", name);
  const void* xs[3] = {a->q, a->k, a->v};
  void* os[3] = {a->q_out, a->k_cache, a->v_cache};
  const int64_t xst[9] = {a->q_batch_stride, a->q_token_stride, a->q_head_stride, a->k_batch_stride, a->k_token_stride,
                          a->k_head_stride,  a->v_batch_stride, a->v_token_stride, a->v_head_stride};
  const int64_t ost[9] = {a->q_out_batch_stride,   a->q_out_token_stride,  a->q_out_head_stride,
                          a->k_cache_batch_stride, a->k_cache_slot_stride, a->k_cache_head_stride,
                          a->v_cache_batch_stride, a->v_cache_slot_stride, a->v_cache_head_stride};
  CacheParams p{};
  for (int i = 0; i < 3; ++i) {
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
  }
  const void* weights[2] = {a->q_weight, a->k_weight};
  const int64_t wd[2] = {a->q_weight_dtype, a->k_weight_dtype}, all[2] = {a->q_norm_all, a->k_norm_all};
  for (int i = 0; i < 2; ++i) {
    if (!weights[i]) continue;
    DFS_REQUIRE(wd[i] == DFS_DTYPE_BF16 || wd[i] == DFS_DTYPE_F16 || wd[i] == DFS_DTYPE_F32,
                "%s: weight dtype code %lld is not supported", name, (long long)wd[i]);
    DFS_REQUIRE(reinterpret_cast<uintptr_t>(weights[i]) % 16 == 0, "%s: weights must be 16-byte aligned", name);
    p.weight[i] = weights[i];
    p.w_dtype[i] = static_cast<int>(wd[i]);
    p.w_all[i] = all[i] != 0;
  }
  p.eps = static_cast<float>(a->eps);
  p.cos_t = a->cos_table;
  p.sin_t = a->sin_table;
  p.table_rows = a->table_rows;
  p.lens = a->lens;
  p.new_lens = a->new_lens;
  p.B = static_cast<int>(a->batch);
  p.T = static_cast<int>(a->tokens);
  while ((int64_t(1) << p.log2d) < a->head_dim) ++p.log2d;
  p.S = static_cast<int>(a->slots);
  p.sinks = static_cast<int>(a->sinks < kMax ? a->sinks : kMax);
  p.rolling = a->rolling != 0;
  const dim3 grid(static_cast<unsigned>((a->batch * a->tokens + 3) / 4), 3);
  const bool f16 = a->dtype == DFS_DTYPE_F16;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch ((widest + 1023) / 1024) {  // chunks of 512 channels, rounded up to an even count
    case 1: launch_cache<2>(p, f16, grid, st); break;
    case 2: launch_cache<4>(p, f16, grid, st); break;
    case 3: launch_cache<6>(p, f16, grid, st); break;
    case 4: launch_cache<8>(p, f16, grid, st); break;
    case 5: launch_cache<10>(p, f16, grid, st); break;
    case 6: launch_cache<12>(p, f16, grid, st); break;
    case 7: launch_cache<14>(p, f16, grid, st); break;
    default: launch_cache<16>(p, f16, grid, st); break;
  }
  return check_launch(name);
}
