// Matrix product with its epilogue, out = residual + gate * act(x W^T + bias):
// the projections and the feed-forward products of a transformer block.
//   z[m][n] = sum_k x[m][k] w[n][k] + bias[n]     (x, w bf16 or f16, sums fp32)
//   out[m][n] = round(residual[m][n] + gate[n] * act(z[m][n]))
// act: none, GELU (erf or tanh form) or SiLU; everything behind the sum runs in
// fp32 and is rounded once.
//
// The products run as W X^T: the rows of a 32x32x16 MFMA's result are outputs n
// and its columns rows m of x, so a lane holds one row of out. Its register
// groups cover 4 consecutive n; the A operand's rows are dealt to the tiles so
// that the groups of a wave's tiles join into 8 or 16 consecutive n and leave
// as 16-byte stores (TileRows).
#include "common.h"
#include "lds_copy.h"

namespace dfs {
namespace {

enum Activation { kActNone = 0, kActGeluTanh = 1, kActGelu = 2, kActSilu = 3 };

struct LinearParams {
  const uint16_t* x;  // [M][K], row stride ldx
  const uint16_t* w;  // [N][K], row stride ldw
  int64_t ldx, ldw, ldr, ldo;
  int M, N, K;
  const void* bias;  // [N] or NULL
  int bias_dtype;
  int act;
  const float* gate;         // [N] or NULL
  const uint16_t* residual;  // [M][N], row stride ldr, or NULL; may be out
  uint16_t* out;
  int wide;  // rows of out and residual allow 16-byte accesses at multiples of 8
};

template <bool F16>
struct Half;
template <>
struct Half<false> {
  typedef bf16x8 vec;
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint32_t bits) { return bf16_bits_to_f32(bits); }
  static __device__ __forceinline__ uint32_t from_f32(float v) { return f32_to_bf16_bits(v); }
};
template <>
struct Half<true> {
  typedef f16x8 vec;
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_f32(uint32_t bits) { return f16_bits_to_f32(bits); }
  static __device__ __forceinline__ uint32_t from_f32(float v) { return f32_to_f16_bits(v); }
};

__device__ __forceinline__ float activate(float z, int act) {
  // sigmoid(t) = 1 / (1 + e^-t); 0.5 (1 + tanh u) = sigmoid(2 u). e^-t may
  // overflow to infinity: the quotient is 0 then.
  switch (act) {
    case kActGeluTanh: {
      const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      return z / (1.f + exp2_fast(-1.4426950408889634f * u));
    }
    case kActGelu:
      return 0.5f * z * erfcf(-0.70710678118654752f * z);
    case kActSilu:
      return z / (1.f + exp2_fast(-1.4426950408889634f * z));
    default:
      return z;
  }
}

__device__ __forceinline__ float bias_at(const LinearParams& p, int n) {
  if (!p.bias) return 0.f;
  if (p.bias_dtype == DFS_DTYPE_F32) return static_cast<const float*>(p.bias)[n];
  const uint32_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.bias_dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// Eight consecutive outputs n.. of row m from their sums.
template <bool F16>
__device__ __forceinline__ void finish8(const LinearParams& p, int m, int n, const float* z) {
  if (m >= p.M || n >= p.N) return;
  const uint16_t* r = p.residual ? p.residual + m * p.ldr + n : nullptr;
  uint16_t* o = p.out + m * p.ldo + n;
  if (p.wide && n + 8 <= p.N) {
    uint4 rv = make_uint4(0, 0, 0, 0);
    if (r) rv = *reinterpret_cast<const uint4*>(r);
    uint32_t packed[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float y = activate(z[i] + bias_at(p, n + i), p.act);
      if (p.gate) y *= p.gate[n + i];
      if (r) y += Half<F16>::to_f32(u16_at(rv, i));
      const uint32_t h = Half<F16>::from_f32(y);
      packed[i / 2] = i & 1 ? packed[i / 2] | h << 16 : h;
    }
    *reinterpret_cast<uint4*>(o) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (n + i >= p.N) break;
    float y = activate(z[i] + bias_at(p, n + i), p.act);
    if (p.gate) y *= p.gate[n + i];
    if (r) y += Half<F16>::to_f32(r[i]);
    o[i] = static_cast<uint16_t>(Half<F16>::from_f32(y));
  }
}

// Eight elements k..k+7 of a row of K that may start at any 2-byte address;
// zeros past the row's end.
__device__ __forceinline__ uint4 load_row8(const uint16_t* row, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 8 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < K) {
    uint16_t t[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) t[i] = row[k + i];
    __builtin_memcpy(&v, t, 16);
  }
  return v;
}

// 64 x 64 outputs a workgroup, four waves of 32 x 32, 64 channels a step, any
// strides and sizes: rows are loaded into registers and stored to LDS from
// there.
template <bool F16>
__global__ void __launch_bounds__(256) linear_any_kernel(LinearParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t ws[64 * 64];
  __shared__ __attribute__((aligned(16))) uint16_t xs[64 * 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l32 = lane & 31, hl = lane >> 5;
  const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
  f32x16 acc = f32x16{};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    uint4 a[2], b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = j * 32 + (tid >> 3), k = k0 + (tid & 7) * 8;
      a[j] = load_row8(p.w + min(n0 + r, p.N - 1) * p.ldw, k, p.K);
      b[j] = load_row8(p.x + min(m0 + r, p.M - 1) * p.ldx, k, p.K);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = j * 32 + (tid >> 3), c = (tid & 7) ^ (r & 7);
      *reinterpret_cast<uint4*>(ws + (r * 8 + c) * 8) = a[j];
      *reinterpret_cast<uint4*>(xs + (r * 8 + c) * 8) = b[j];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint4 fa = lds_chunk<8>(ws, (w & 1) * 32 + l32, 2 * s + hl);
      const uint4 fb = lds_chunk<8>(xs, (w >> 1) * 32 + l32, 2 * s + hl);
      acc = Half<F16>::mfma(__builtin_bit_cast(typename Half<F16>::vec, fa),
                            __builtin_bit_cast(typename Half<F16>::vec, fb), acc);
    }
  }
  // The lane halves hold alternate groups of four n: joined into eight by an
  // exchange, half 0 keeps the even eights.
  const int m = m0 + (w >> 1) * 32 + l32;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float z[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[g * 8 + i]),
                                                      __float_as_uint(acc[g * 8 + 4 + i]), false, false);
      z[i] = __uint_as_float(t[0]);
      z[4 + i] = __uint_as_float(t[1]);
    }
    finish8<F16>(p, m, n0 + (w & 1) * 32 + g * 16 + hl * 8, z);
  }
}

}  // namespace
}  // namespace dfs

extern "C" int64_t dfs_linear_workspace_size(int64_t rows, int64_t n, int64_t k) {
  using namespace dfs;
  if (rows <= 0 || n <= 0 || k <= 0) {
    set_error("linear: rows=%lld n=%lld k=%lld must be positive", (long long)rows, (long long)n, (long long)k);
    return -1;
  }
  return 0;
}

extern "C" int dfs_linear(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int64_t rows, int64_t n,
                          int64_t k, int dtype, const void* bias, int bias_dtype, int activation, const float* gate,
                          const void* residual, int64_t r_stride, void* out, int64_t o_stride, void* workspace,
                          int64_t workspace_bytes, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "linear";
  DFS_REQUIRE(x && w && out, "%s: x, w and out must be non-NULL", name);
  DFS_REQUIRE(rows > 0 && n > 0 && k > 0, "%s: rows=%lld n=%lld k=%lld must be positive", name, (long long)rows,
              (long long)n, (long long)k);
  constexpr int64_t kMax = int64_t(1) << 30;
  DFS_REQUIRE(rows < kMax && n < kMax && k < kMax, "%s: rows, n and k must be below 2^30", name);
  DFS_REQUIRE(dtype == DFS_DTYPE_BF16 || dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(x_stride >= 0 && w_stride >= 0 && o_stride >= n && (!residual || r_stride >= 0),
              "%s: strides must be non-negative, and out's rows must not overlap", name);
  DFS_REQUIRE(bias == nullptr || bias_dtype == DFS_DTYPE_BF16 || bias_dtype == DFS_DTYPE_F16 ||
                  bias_dtype == DFS_DTYPE_F32,
              "%s: bias dtype code %d is not supported", name, bias_dtype);
  DFS_REQUIRE(activation >= kActNone && activation <= kActSilu, "%s: activation code %d is not supported", name,
              activation);
  auto addr = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  DFS_REQUIRE(addr(x) % 2 == 0 && addr(w) % 2 == 0 && addr(out) % 2 == 0 && addr(residual) % 2 == 0 &&
                  addr(gate) % 4 == 0 && addr(bias) % (bias_dtype == DFS_DTYPE_F32 ? 4 : 2) == 0,
              "%s: operands must be aligned to their elements", name);
  const int64_t need = dfs_linear_workspace_size(rows, n, k);
  DFS_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "%s: workspace of %lld bytes needed",
              name, (long long)need);
  LinearParams p{};
  p.x = static_cast<const uint16_t*>(x);
  p.w = static_cast<const uint16_t*>(w);
  p.ldx = x_stride;
  p.ldw = w_stride;
  p.ldr = r_stride;
  p.ldo = o_stride;
  p.M = static_cast<int>(rows);
  p.N = static_cast<int>(n);
  p.K = static_cast<int>(k);
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.act = activation;
  p.gate = gate;
  p.residual = static_cast<const uint16_t*>(residual);
  p.out = static_cast<uint16_t*>(out);
  p.wide = o_stride % 8 == 0 && addr(out) % 16 == 0 && (!residual || (r_stride % 8 == 0 && addr(residual) % 16 == 0));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t mt = (rows + 63) / 64, nt = (n + 63) / 64;
  DFS_REQUIRE(mt < 65536, "%s: too many rows", name);
  const dim3 grid(static_cast<unsigned>(nt), static_cast<unsigned>(mt));
  if (dtype == DFS_DTYPE_F16)
    linear_any_kernel<true><<<grid, 256, 0, st>>>(p);
  else
    linear_any_kernel<false><<<grid, 256, 0, st>>>(p);
  return check_launch(name);
}
