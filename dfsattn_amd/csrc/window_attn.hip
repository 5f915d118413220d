// Softmax attention with a sliding window and sinks (the first tokens, which
// stay visible). A sequence of nq queries and nk keys: query i stands at
// position p = nk - nq + i and sees key j where
//   0 <= j < nk,  j <= p + right,  (j >= p - left or j < sinks),
// out_i = sum_j softmax_j(scale q_i k_j) v_j over the keys it sees (0 where it
// sees none), lse_i the log of the softmax's denominator (-inf there).
// Key j lies in slot j of the sequence's rows, or, in a rolling cache of S
// slots, in slot j < sinks ? j : sinks + (j - sinks) mod (S - sinks).
#include "common.h"

namespace dfs {
namespace {

constexpr int kNoLimit = 1 << 30;

struct WindowParams {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  float* lse;  // [B][Hq][Lq] or NULL
  const int32_t *q_lens, *kv_lens;  // [B] or NULL
  int64_t q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, v_sb, v_sh, v_sl, o_sb, o_sh, o_sl;
  int B, Hq, Hkv, Lq, S;
  int left, right, sinks;  // kNoLimit for no limit
  int rolling;
  float scale_log2;
};

template <bool F16>
__device__ __forceinline__ float half_to_f32(uint32_t bits) {
  return F16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
}

__device__ __forceinline__ int slot_of(const WindowParams& p, int64_t pos) {
  if (!p.rolling || pos < p.sinks) return static_cast<int>(pos);
  return p.sinks + static_cast<int>((pos - p.sinks) % (p.S - p.sinks));
}

// One wave a query: its D channels over the lanes, the keys one at a time with
// the running maximum and sum.
template <int D, bool F16>
__global__ void __launch_bounds__(256) window_simple_kernel(WindowParams p) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(p.B) * p.Hq * p.Lq) return;
  const int i = static_cast<int>(row % p.Lq), h = static_cast<int>(row / p.Lq % p.Hq);
  const int b = static_cast<int>(row / p.Lq / p.Hq), g = h / (p.Hq / p.Hkv);
  const int nq = p.q_lens ? min(max(p.q_lens[b], 0), p.Lq) : p.Lq;
  int nk = p.kv_lens ? max(p.kv_lens[b], 0) : p.S;
  if (!p.rolling) nk = min(nk, p.S);
  const uint16_t* q = p.q + b * p.q_sb + h * p.q_sh + i * p.q_sl;
  const uint16_t* k = p.k + b * p.k_sb + g * p.k_sh;
  const uint16_t* v = p.v + b * p.v_sb + g * p.v_sh;
  float qv[E], o[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) qv[e] = half_to_f32<F16>(q[lane * E + e]) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  const int64_t pos = static_cast<int64_t>(nk) - nq + i;
  const int64_t hi = i < nq ? min(static_cast<int64_t>(nk), pos + p.right + 1) : 0;
  const int64_t lo = max(int64_t(0), pos - p.left);
  for (int64_t j = 0; j < hi; ++j) {
    if (j >= p.sinks && j < lo) j = lo;
    if (j >= hi) break;
    const int64_t slot = slot_of(p, j);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += qv[e] * half_to_f32<F16>(k[slot * p.k_sl + lane * E + e]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - ref), w = exp2f(s - ref);
    l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + w * half_to_f32<F16>(v[slot * p.v_sl + lane * E + e]);
    m = mn;
  }
  uint16_t* out = p.out + b * p.o_sb + h * p.o_sh + i * p.o_sl;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = l > 0.f ? o[e] / l : (l == 0.f ? 0.f : l);
    out[lane * E + e] = static_cast<uint16_t>(F16 ? f32_to_f16_bits(y) : f32_to_bf16_bits(y));
  }
  if (p.lse && lane == 0)
    p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

}  // namespace
}  // namespace dfs

extern "C" int64_t dfs_window_attention_workspace_size(const dfs_window_args* a) { return a ? 0 : -1; }

extern "C" int dfs_window_attention(const dfs_window_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "window_attention";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  DFS_REQUIRE(a->q && a->k && a->v && a->out, "%s: q, k, v and out must be non-NULL", name);
  DFS_REQUIRE(a->batch > 0 && a->q_heads > 0 && a->kv_heads > 0 && a->q_rows > 0 && a->slots > 0,
              "%s: batch, heads, q_rows and slots must be positive", name);
  DFS_REQUIRE(a->q_heads % a->kv_heads == 0, "%s: q_heads=%lld is not a multiple of kv_heads=%lld", name,
              (long long)a->q_heads, (long long)a->kv_heads);
  DFS_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "%s: head_dim=%lld (supported: 64, 128)", name,
              (long long)a->head_dim);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(a->q_rows < kNoLimit && a->slots < kNoLimit && a->batch < 65536 && a->q_heads < 65536,
              "%s: sizes too large", name);
  DFS_REQUIRE(a->left >= -1 && a->right >= -1 && a->sinks >= 0, "%s: left and right must be -1 or more, sinks 0 or more",
              name);
  DFS_REQUIRE(a->scale > 0. && a->scale < 1e30, "%s: scale must be positive and finite", name);
  const int64_t strides[12] = {a->q_batch_stride, a->q_head_stride, a->q_row_stride, a->k_batch_stride,
                               a->k_head_stride,  a->k_row_stride,  a->v_batch_stride, a->v_head_stride,
                               a->v_row_stride,   a->out_batch_stride, a->out_head_stride, a->out_row_stride};
  for (int64_t s : strides)
    DFS_REQUIRE(s >= 0 && s % 8 == 0, "%s: strides must be non-negative multiples of 8 elements", name);
  const uintptr_t any = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                        reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->out);
  DFS_REQUIRE(any % 16 == 0, "%s: q, k, v and out must be 16-byte aligned", name);
  if (a->rolling) {
    DFS_REQUIRE(a->kv_lens != nullptr, "%s: a rolling cache needs kv_lens", name);
    DFS_REQUIRE(a->left >= 0 && a->slots - a->sinks >= a->left + a->q_rows,
                "%s: a rolling cache needs sinks + left + q_rows = %lld slots, got %lld", name,
                (long long)(a->sinks + a->left + a->q_rows), (long long)a->slots);
  }
  auto limit = [](int64_t n) { return static_cast<int>(n < 0 || n > kNoLimit ? kNoLimit : n); };
  WindowParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  p.q_lens = a->q_lens;
  p.kv_lens = a->kv_lens;
  p.q_sb = a->q_batch_stride; p.q_sh = a->q_head_stride; p.q_sl = a->q_row_stride;
  p.k_sb = a->k_batch_stride; p.k_sh = a->k_head_stride; p.k_sl = a->k_row_stride;
  p.v_sb = a->v_batch_stride; p.v_sh = a->v_head_stride; p.v_sl = a->v_row_stride;
  p.o_sb = a->out_batch_stride; p.o_sh = a->out_head_stride; p.o_sl = a->out_row_stride;
  p.B = static_cast<int>(a->batch);
  p.Hq = static_cast<int>(a->q_heads);
  p.Hkv = static_cast<int>(a->kv_heads);
  p.Lq = static_cast<int>(a->q_rows);
  p.S = static_cast<int>(a->slots);
  p.left = limit(a->left);
  p.right = limit(a->right);
  p.sinks = limit(a->sinks);
  p.rolling = a->rolling != 0;
  p.scale_log2 = static_cast<float>(a->scale * 1.4426950408889634);
  const int64_t blocks = (a->batch * a->q_heads * a->q_rows + 3) / 4;
  DFS_REQUIRE(blocks < (int64_t(1) << 31), "%s: too many rows", name);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool f16 = a->dtype == DFS_DTYPE_F16;
  if (a->head_dim == 128)
    f16 ? window_simple_kernel<128, true><<<grid, 256, 0, st>>>(p) : window_simple_kernel<128, false><<<grid, 256, 0, st>>>(p);
  else
    f16 ? window_simple_kernel<64, true><<<grid, 256, 0, st>>>(p) : window_simple_kernel<64, false><<<grid, 256, 0, st>>>(p);
  return check_launch(name);
}
