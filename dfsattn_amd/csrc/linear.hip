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
// as 16-byte stores.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "lds_copy.h"

namespace dfs {
namespace {

constexpr uint32_t kOutside = 0x80000000u;  // byte offset past every buffer's records

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
  // The channels of a tile are cut into `splits` parts of `depth` (a multiple
  // of 128); a part's sums go to part [split][M][ceil(N / 8) * 8] in fp32. Of the
  // 256 x 256 tiles the first `whole` are not cut, the others' sums go to part
  // [split][tile][256][256].
  int splits, depth, whole;
  float* part;
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

__device__ __forceinline__ float bias_at(const LinearParams& p, int n) {
  if (!p.bias) return 0.f;
  if (p.bias_dtype == DFS_DTYPE_F32) return static_cast<const float*>(p.bias)[n];
  const uint32_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.bias_dtype == DFS_DTYPE_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// Bias and gate of eight consecutive outputs n.. (any values past N).
__device__ __forceinline__ void load_columns8(const LinearParams& p, int n, float* bias, float* gate) {
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
__device__ __forceinline__ void finish8_wide(const LinearParams& p, int m, int n, const float* z, const float* bias,
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
__device__ __forceinline__ void finish8_edge(const LinearParams& p, int m, int n, const float* z, const float* bias,
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
__device__ __forceinline__ void finish8(const LinearParams& p, int m, int n, const float* z, const float* bias,
                                        const float* gate) {
  if (m >= p.M || n >= p.N) return;
  if (n + 8 <= p.N)
    finish8_wide<F16, ACT>(p, m, n, z, bias, gate);
  else
    finish8_edge<F16, ACT>(p, m, n, z, bias, gate);
}

// Elements k..k+7 of a row of K, zeros past its end: one by one, but all on
// their way at once.
__device__ __forceinline__ uint4 load_edge8(const uint16_t* row, int k, int K) {
  uint16_t t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = row[min(k + i, K - 1)];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = k + i < K ? t[i] : 0;
  uint4 v;
  __builtin_memcpy(&v, t, 16);
  return v;
}

// The same from a row that may start at any 2-byte address.
__device__ __forceinline__ uint4 load_row8(const uint16_t* row, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 8 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < K) {
    v = load_edge8(row, k, K);
  }
  return v;
}

// 64 x 64 outputs a workgroup, four waves of 32 x 32, 64 channels a step, any
// strides and sizes: rows are loaded into registers, four steps ahead, and
// stored to one of two LDS buffers from there, one barrier a step. The channels
// behind the last whole step go first, so that the steps' loads have no edge.
// 333 x 1,017 x 709, one of many in a graph: 8.8 us, 10.4 with bias, SiLU and
// residual (11.4 by trace); loads a step ahead, with two barriers, 11.9 for 8.8.
template <bool F16>
__global__ void __launch_bounds__(256) linear_any_kernel(LinearParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t ws[2][64 * 64];
  __shared__ __attribute__((aligned(16))) uint16_t xs[2][64 * 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l32 = lane & 31, hl = lane >> 5;
  const unsigned nt = (p.N + 63) / 64;
  const int m0 = static_cast<int>(blockIdx.x / nt) * 64, n0 = static_cast<int>(blockIdx.x % nt) * 64;
  const int steps = p.K >> 6, c8 = (tid & 7) * 8;
  const uint16_t *wrow[2], *xrow[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = j * 32 + (tid >> 3);
    wrow[j] = p.w + min(n0 + r, p.N - 1) * p.ldw + c8;
    xrow[j] = p.x + min(m0 + r, p.M - 1) * p.ldx + c8;
  }
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef u32x4 Chunks[4];  // two of w, two of x
  auto load = [&](int t, Chunks& c) {  // past the last step: that again, unread
    const int k = min(t, steps - 1) * 64;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4 a, b;
      __builtin_memcpy(&a, wrow[j] + k, 16);
      __builtin_memcpy(&b, xrow[j] + k, 16);
      c[j] = a;
      c[2 + j] = b;
    }
  };
  f32x16 acc = f32x16{};
  auto step = [&](const Chunks& ch, int buf) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = j * 32 + (tid >> 3), c = (tid & 7) ^ (r >> 1 & 7);
      *reinterpret_cast<u32x4*>(ws[buf] + (r * 8 + c) * 8) = ch[j];
      *reinterpret_cast<u32x4*>(xs[buf] + (r * 8 + c) * 8) = ch[2 + j];
    }
    block_barrier();  // stored by all; the other buffer has been read by all
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int wr = (w & 1) * 32 + l32, xr = (w >> 1) * 32 + l32, c = 2 * s + hl;
      const uint4 fa = *reinterpret_cast<const uint4*>(ws[buf] + (wr * 8 + (c ^ (wr >> 1 & 7))) * 8);
      const uint4 fb = *reinterpret_cast<const uint4*>(xs[buf] + (xr * 8 + (c ^ (xr >> 1 & 7))) * 8);
      acc = Half<F16>::mfma(__builtin_bit_cast(typename Half<F16>::vec, fa),
                            __builtin_bit_cast(typename Half<F16>::vec, fb), acc);
    }
  };
  Chunks c0, c1, c2, c3;
  if (steps > 0) {
    load(0, c0);
    load(1, c1);
    load(2, c2);
    load(3, c3);
  }
  if (p.K & 63) {
    Chunks tail;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      tail[j] = __builtin_bit_cast(u32x4, load_edge8(wrow[j] - c8, steps * 64 + c8, p.K));
      tail[2 + j] = __builtin_bit_cast(u32x4, load_edge8(xrow[j] - c8, steps * 64 + c8, p.K));
    }
    step(tail, 1);
  }
  int t = 0;
  for (; t + 4 <= steps; t += 4) {
    step(c0, 0);
    load(t + 4, c0);
    step(c1, 1);
    load(t + 5, c1);
    step(c2, 0);
    load(t + 6, c2);
    step(c3, 1);
    load(t + 7, c3);
  }
  if (t < steps) step(c0, 0);
  if (t + 1 < steps) step(c1, 1);
  if (t + 2 < steps) step(c2, 0);
  // The lane halves hold alternate groups of four n: joined into eight by an
  // exchange, half 0 keeps the even eights.
  const int m = m0 + (w >> 1) * 32 + l32;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float z[8], bias[8], gate[8];
    const int n = n0 + (w & 1) * 32 + g * 16 + hl * 8;
    load_columns8(p, n, bias, gate);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[g * 8 + i]),
                                                      __float_as_uint(acc[g * 8 + 4 + i]), false, false);
      z[i] = __uint_as_float(t[0]);
      z[4 + i] = __uint_as_float(t[1]);
    }
    with_activation(p.act, [&](auto act) { finish8<F16, decltype(act)::value>(p, m, n, z, bias, gate); });
  }
}

// Sums of a workgroup's 16 outputs n0.. for up to 16 rows, one set a wave in LDS
// ([wave][lane][4]: output 4 g + r of row m lies in register r of lane
// 16 g + m), joined in the waves' order and finished.
template <bool F16>
__device__ __forceinline__ void finish16(const LinearParams& p, int n0, const float* sums, int waves) {
  const int e = threadIdx.x, n16 = e & 15, m = e >> 4, n = n0 + n16;
  if (e >= 256 || m >= p.M || n >= p.N) return;
  float z = 0.f;
  for (int v = 0; v < waves; ++v) z += sums[v * 256 + ((n16 >> 2) * 16 + m) * 4 + (n16 & 3)];
  z += bias_at(p, n);
  with_activation(p.act, [&](auto act) { z = activate<decltype(act)::value>(z); });
  if (p.gate) z *= p.gate[n];
  if (p.residual) z += Half<F16>::to_f32(p.residual[m * p.ldr + n]);
  p.out[m * p.ldo + n] = static_cast<uint16_t>(Half<F16>::from_f32(z));
}

// At most 16 rows of x: what counts is reading w once. A workgroup owns 16
// outputs, and its waves deal the channels among themselves in blocks of 128. A
// wave's blocks of w pass through three LDS buffers of its own that the loads
// fill directly, 256 bytes of a row at a time; x comes from L2 as it is needed.
// No barrier before the waves' sums meet. One row by 30,720 x 5,120: 54.4 us
// (5.8 TB/s) with streaming loads, taken where w is beyond the last-level cache,
// 58.2 with ordinary ones; with w read into registers in the products' layout,
// 64 bytes of a row at a time, 61 to 69. Four rows by 5,120 x 13,824: 23.7 and
// 37.1 (streaming 46).
template <int WAVES, bool F16, bool STREAM>
__global__ void __launch_bounds__(64 * WAVES) linear_few_kernel(LinearParams p) {
  typedef typename Half<F16>::vec vec;
  constexpr int kBlock = 16 * 128;  // elements of w in a wave's buffer
  __shared__ __attribute__((aligned(16))) uint16_t s0[WAVES * kBlock], s1[WAVES * kBlock], s2[WAVES * kBlock];
  __shared__ __attribute__((aligned(16))) float sums[WAVES * 256];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, c4 = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const auto rs = make_rsrc(p.w + n0 * p.ldw, kOutside);
  // Load j: rows 4 j .. 4 j + 3, chunk c of row r at c ^ r (16 chunks a row).
  uint32_t wv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 4 * j + c4;
    wv[j] = static_cast<uint32_t>(min(n0 + r, p.N - 1) - n0) * static_cast<uint32_t>(p.ldw * 2) + (r16 ^ r) * 16;
  }
  const uint16_t* const xr = p.x + min(r16, p.M - 1) * p.ldx;
  const int blocks = (p.K + 127) >> 7;
  auto load = [&](int b, uint16_t* buf) {  // past the last block: zeros, without a memory access
    const int left = p.K - b * 128;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = (r16 ^ (4 * j + c4)) * 8 < left;
      load_lds16<STREAM>(rs, buf + w * kBlock + j * 512, in ? wv[j] + b * 256 : kOutside, 0);
    }
  };
  f32x4 acc = f32x4{};
  auto step = [&](int b, const uint16_t* buf, uint16_t* next) {
    uint4 x[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = b * 128 + s * 32 + c4 * 8;
      x[s] = make_uint4(0, 0, 0, 0);
      if (r16 < p.M && k < p.K) x[s] = *reinterpret_cast<const uint4*>(xr + k);
    }
    wait_lgkm_0();  // the reads of `next`, a step ago, are done (zeros come at once)
    load(b + 2 * WAVES, next);
    const uint16_t* const row = buf + w * kBlock + r16 * 128;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint4 a = *reinterpret_cast<const uint4*>(row + ((s * 4 + c4) ^ r16) * 8);
      acc = Half<F16>::mfma16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, x[s]), acc);
    }
  };
  load(w, s0);
  load(w + WAVES, s1);
  for (int b = w; b < blocks; b += 3 * WAVES) {
    step(b, s0, s2);
    step(b + WAVES, s1, s0);
    step(b + 2 * WAVES, s2, s1);
  }
  wait_vmcnt_0();
  *reinterpret_cast<f32x4*>(sums + (w * 64 + lane) * 4) = acc;
  __syncthreads();
  finish16<F16>(p, n0, sums, WAVES);
}

// Tiles of BN = 32 NI WN outputs by BM = 32 MI WM rows, a workgroup of WN x WM
// = 4 waves with NI x MI products of 32 x 32 each, 64 channels a step through
// NS LDS buffers that the loads fill directly. For operands on 16-byte rows.
// Few workgroups wait for memory unless several steps are on their way (64 x 64
// alone on a CU: 0.5 us a step with two buffers, 0.26 with four); many hide it
// from each other and want the room.
//
// A step's 128-byte rows hold eight 16-byte chunks; chunk c of row r lies at
// c ^ f(r) with f such that any 16 rows that one quarter of a wave reads
// together fall on all 64 banks. Row i of the A operand of tile ni is output
// (i >> 2) * 4 NI + ni * 4 + (i & 3), so a lane ends with 4 NI consecutive
// outputs.
//
// Order of a step: the fragments of a quarter (16 channels) are read while the
// quarter before is multiplied; before the last quarter's products, the next
// step's data is waited for and, behind the barrier, the loads of the step NS on
// go into the buffer just read. So there is one barrier a step, the products of
// a quarter are there on both sides of it, and a load has NS - 1 steps to land.
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

template <int NI, int MI, int WN, int WM, int NS, bool F16>
__global__ void __launch_bounds__(256, 2) linear_tile_kernel(LinearParams p) {
  typedef Tile<NI, MI, WN, WM, F16> T;
  typedef typename T::vec vec;
  constexpr int JW = T::BN / 32, JX = T::BM / 32;  // loads of 1 KB a wave and step
  // Of buffers 2 and 3, those past NS are empty.
  constexpr int N2 = NS > 2 ? 64 : 1, N3 = NS > 3 ? 64 : 1;
  __shared__ __attribute__((aligned(16))) uint16_t w0[T::BN * 64], w1[T::BN * 64], w2[T::BN * N2], w3[T::BN * N3];
  __shared__ __attribute__((aligned(16))) uint16_t x0[T::BM * 64], x1[T::BM * 64], x2[T::BM * N2], x3[T::BM * N3];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int mt = (p.M + T::BM - 1) / T::BM, nt = (p.N + T::BN - 1) / T::BN;
  const int split = p.splits > 1 ? blockIdx.x / (mt * nt) : 0, from = split * p.depth;
  int tm, tn;
  tile_of(blockIdx.x - split * mt * nt, mt, nt, tm, tn);
  const int n0 = tn * T::BN, m0 = tm * T::BM;
  const int K = p.splits > 1 ? min(p.K - from, p.depth) : p.K;
  const auto wrs = make_rsrc(p.w + static_cast<int64_t>(n0) * p.ldw + from, kOutside);
  const auto xrs = make_rsrc(p.x + static_cast<int64_t>(m0) * p.ldx + from, kOutside);
  // Byte offsets of this lane's chunks in step 0; rows past the matrix repeat
  // its last one.
  uint32_t wv[JW], xv[JX];
  const int r8 = w * 8 + (lane >> 3), c8 = lane & 7;
#pragma unroll
  for (int j = 0; j < JW; ++j) {
    const int r = j * 32 + r8;
    wv[j] = static_cast<uint32_t>(min(n0 + r, p.N - 1) - n0) * static_cast<uint32_t>(p.ldw * 2) +
            (c8 ^ T::swz_w(r)) * 16;
  }
#pragma unroll
  for (int j = 0; j < JX; ++j) {
    const int r = j * 32 + r8;
    xv[j] = static_cast<uint32_t>(min(m0 + r, p.M - 1) - m0) * static_cast<uint32_t>(p.ldx * 2) +
            (c8 ^ T::swz_x(r)) * 16;
  }
  const int steps = (K + 64 * NS - 1) / (64 * NS) * NS;  // the last may be all zeros
  auto issue = [&](int t, uint16_t* wb, uint16_t* xb) {
    const int left = K - t * 64;
    if (left < 64) {  // the last steps: chunks past K come as zeros
#pragma unroll
      for (int j = 0; j < JX; ++j)
        if ((c8 ^ T::swz_x(j * 32 + r8)) * 8 >= left) xv[j] = kOutside;
#pragma unroll
      for (int j = 0; j < JW; ++j)
        if ((c8 ^ T::swz_w(j * 32 + r8)) * 8 >= left) wv[j] = kOutside;
    }
#pragma unroll
    for (int j = 0; j < JX; ++j)
      load_lds16(xrs, xb + (j * 4 + w) * 512, xv[j], t * 128);
#pragma unroll
    for (int j = 0; j < JW; ++j)
      load_lds16(wrs, wb + (j * 4 + w) * 512, wv[j], t * 128);
  };
  // Fragment addresses (elements): row part, then the chunk of quarter s.
  const int wn = w % WN, wm = w / WN;
  const int arow = (wn * 32 * NI + (l32 >> 2) * 4 * NI + (l32 & 3)) * 64;
  const int brow = (wm * 32 * MI + l32) * 64;
  const int fa = T::swz_w((l32 >> 2) * 4 * NI + (l32 & 3)), fb = T::swz_x(l32);
  f32x16 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j) acc[i][j] = f32x16{};
  auto fetch = [&](const uint16_t* wb, const uint16_t* xb, int s, uint4* a, uint4* b) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      a[i] = *reinterpret_cast<const uint4*>(wb + arow + i * 256 + ((2 * s + hl) ^ fa) * 8);
#pragma unroll
    for (int j = 0; j < MI; ++j)
      b[j] = *reinterpret_cast<const uint4*>(xb + brow + j * 2048 + ((2 * s + hl) ^ fb) * 8);
  };
  auto multiply = [&](const uint4* a, const uint4* b) {
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i)
        acc[i][j] = Half<F16>::mfma(__builtin_bit_cast(vec, a[i]), __builtin_bit_cast(vec, b[j]), acc[i][j]);
  };
  constexpr int kMfma = 0x008, kDsRead = 0x100, kVmem = 0x020;
  constexpr int PER = NI * MI / (NI + MI) > 0 ? NI * MI / (NI + MI) : 1;
  auto pin = [&](bool loads) {
#pragma unroll
    for (int i = 0; i < NI + MI; ++i) {
      __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
      if (loads) __builtin_amdgcn_sched_group_barrier(kVmem, (JW + JX) / (NI + MI), 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, PER, 0);
    }
  };
  uint4 a0[NI], b0[MI], a1[NI], b1[MI];
  auto step = [&](int t, uint16_t* wc, uint16_t* xc, const uint16_t* wnext, const uint16_t* xnext) {
    fetch(wc, xc, 1, a1, b1);
    multiply(a0, b0);
    pin(false);
    __builtin_amdgcn_sched_barrier(0);
    fetch(wc, xc, 2, a0, b0);
    multiply(a1, b1);
    pin(false);
    __builtin_amdgcn_sched_barrier(0);
    fetch(wc, xc, 3, a1, b1);
    multiply(a0, b0);
    pin(false);
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<(NS - 2) * (JW + JX)>();
    block_barrier();
    issue(t + NS, wc, xc);  // past the last step: zeros, without a memory access
    fetch(wnext, xnext, 0, a0, b0);  // past the last step: read and not used
    multiply(a1, b1);
    pin(true);
    __builtin_amdgcn_sched_barrier(0);
  };
  issue(0, w0, x0);
  issue(1, w1, x1);
  if constexpr (NS > 2) issue(2, w2, x2);
  if constexpr (NS > 3) issue(3, w3, x3);
  wait_vmcnt<(NS - 1) * (JW + JX)>();
  block_barrier();
  fetch(w0, x0, 0, a0, b0);
  for (int t = 0; t < steps; t += NS) {
    step(t, w0, x0, w1, x1);
    if constexpr (NS == 2) step(t + 1, w1, x1, w0, x0);
    if constexpr (NS == 3) {
      step(t + 1, w1, x1, w2, x2);
      step(t + 2, w2, x2, w0, x0);
    }
    if constexpr (NS == 4) {
      step(t + 1, w1, x1, w2, x2);
      step(t + 2, w2, x2, w3, x3);
      step(t + 3, w3, x3, w0, x0);
    }
  }
  wait_vmcnt_0();  // the trailing loads have landed before the workgroup's LDS is released
  const int nb = n0 + wn * 32 * NI + hl * 4 * NI, mb = m0 + wm * 32 * MI + l32;
  if (p.splits > 1) {  // four outputs a register group, n = nb + ...; 16-byte stores
    const int64_t ld = (p.N + 7) & ~7;
    float* const part = p.part + static_cast<int64_t>(split) * p.M * ld;
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int n = nb + g * 8 * NI + i * 4, m = mb + j * 32;
          const f32x16& z = acc[i][j];
          if (m < p.M && n < ld)
            *reinterpret_cast<float4*>(part + m * ld + n) = make_float4(z[g * 4], z[g * 4 + 1], z[g * 4 + 2], z[g * 4 + 3]);
        }
    return;
  }
  with_activation(p.act, [&](auto act) {
    if constexpr (NI == 1) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float bias[8], gate[8];
        const int n = n0 + wn * 32 + g * 16 + hl * 8;
        load_columns8(p, n, bias, gate);
#pragma unroll
        for (int j = 0; j < MI; ++j) {
          float z[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[0][j][g * 8 + i]),
                                                            __float_as_uint(acc[0][j][g * 8 + 4 + i]), false, false);
            z[i] = __uint_as_float(u[0]);
            z[4 + i] = __uint_as_float(u[1]);
          }
          finish8<F16, decltype(act)::value>(p, mb + j * 32, n, z, bias, gate);
        }
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int q = 0; q < NI / 2; ++q) {
          float bias[8], gate[8];
          const int n = nb + g * 8 * NI + q * 8;
          load_columns8(p, n, bias, gate);
#pragma unroll
          for (int j = 0; j < MI; ++j) {
            float z[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = acc[2 * q + (i >> 2)][j][g * 4 + (i & 3)];
            finish8<F16, decltype(act)::value>(p, mb + j * 32, n, z, bias, gate);
          }
        }
    }
  });
}

// 256 x 256 outputs a workgroup, four waves of 128 x 128, 64 channels a step.
// Each operand's slice of a step is two halves of 128 rows (64 of each wave
// row's 128), and a step is four phases of one quadrant each, 16 products:
//   (A0, B0) (A1, B0) (A1, B1) (A0, B1)
// A phase reads one half into registers for the next (A1, B1, then the next
// step's B0 and A0: the registers just left), and loads a half read in the pair
// of phases before, two steps on. So all pairs are alike: two halves read, two
// loaded three pairs before they are read, one barrier that says both that the
// halves to be read have landed and that those to be loaded were read by all.
//
// 75,600 x 13,824 x 5,120 with GELU: 7.97 to 8.2 ms by the card, 1.3 PFLOP/s (the
// library's product alone 7.1, 1.50); 75,600 x 5,120 x 13,824: 7.56 to 7.7 ms, 1.4
// PFLOP/s (6.9 to 7.0, 1.53), 7.86 to 8.0 with bias, gate and residual; 16,384 x
// 16,384 x 5,120: 1.90 to 1.97 ms, 1.4 PFLOP/s (1.77 to 1.80, 1.54). The matrix
// cores are busy 79% of the cycles and the clock falls to 1.55 GHz: power is the
// bound, and a barrier a phase costs 0.5%. A barrier a step of 64 channels with
// its loads behind it took 10.6 ms, the phases with a branch for the last step's
// edge 9.0; outputs stored from the products' layout, 16 bytes of a row at a
// time, cost 40 us a tile instead of 3.
template <bool F16, int ACT>
__global__ void __launch_bounds__(256, 1) linear_big_kernel(LinearParams p) {
  typedef typename Half<F16>::vec vec;
  typedef Tile<2, 2, 2, 2, F16> T;  // swizzles of a half
  __shared__ __attribute__((aligned(16))) uint16_t a00[128 * 64], a01[128 * 64], a10[128 * 64], a11[128 * 64];
  __shared__ __attribute__((aligned(16))) uint16_t b00[128 * 64], b01[128 * 64], b10[128 * 64], b11[128 * 64];
  __shared__ __attribute__((aligned(16))) float stage[4 * 2048];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int mt = (p.M + 255) / 256, nt = (p.N + 255) / 256, cut = mt * nt - p.whole;
  const bool in_parts = static_cast<int>(blockIdx.x) >= p.whole;
  const int split = in_parts ? (static_cast<int>(blockIdx.x) - p.whole) / cut : 0, from = split * p.depth;
  const int K = in_parts ? min(p.K - from, p.depth) : p.K, id = blockIdx.x - split * cut;
  int tm, tn;
  tile_of(id, mt, nt, tm, tn);
  const int n0 = tn * 256, m0 = tm * 256;
  const auto wrs = make_rsrc(p.w + static_cast<int64_t>(n0) * p.ldw + from, kOutside);
  const auto xrs = make_rsrc(p.x + static_cast<int64_t>(m0) * p.ldx + from, kOutside);
  // Byte offsets of this lane's chunks in step 0, [half][load]; rows past the
  // matrix repeat its last one. Row q of wave row r's 64 in half h is output
  // r * 128 + (q >> 3) * 16 + h * 8 + (q & 7), so that a lane ends with 16
  // consecutive outputs, or row r * 128 + h * 64 + q of x.
  uint32_t wv[2][4], xv[2][4];
  const int r8 = w * 8 + (lane >> 3), c8 = lane & 7;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = j * 32 + r8, q = r & 63, base = (r >> 6) * 128;
      const int n = min(n0 + base + (q >> 3) * 16 + h * 8 + (q & 7), p.N - 1) - n0;
      const int m = min(m0 + base + h * 64 + q, p.M - 1) - m0;
      wv[h][j] = static_cast<uint32_t>(n) * static_cast<uint32_t>(p.ldw * 2) + (c8 ^ T::swz_w(q)) * 16;
      xv[h][j] = static_cast<uint32_t>(m) * static_cast<uint32_t>(p.ldx * 2) + (c8 ^ T::swz_x(q)) * 16;
    }
  const int steps = (K + 127) >> 7 << 1;  // an even number: the last may be all zeros
  // The last steps' chunks past K (tail) come as zeros, without a memory access.
  auto load_w = [&](auto tail, int t, int h, uint16_t* buf) {
    const int left = K - t * 64;
    if (tail.value && left < 64) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((c8 ^ T::swz_w((j * 32 + r8) & 63)) * 8 >= left) wv[h][j] = kOutside;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) load_lds16(wrs, buf + (j * 4 + w) * 512, wv[h][j], t * 128);
  };
  auto load_x = [&](auto tail, int t, int h, uint16_t* buf) {
    const int left = K - t * 64;
    if (tail.value && left < 64) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((c8 ^ T::swz_x((j * 32 + r8) & 63)) * 8 >= left) xv[h][j] = kOutside;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) load_lds16(xrs, buf + (j * 4 + w) * 512, xv[h][j], t * 128);
  };
  const int wn = w & 1, wm = w >> 1;
  const int arow = (wn * 64 + (l32 >> 2) * 8 + (l32 & 3)) * 64, brow = (wm * 64 + l32) * 64;
  const int fa = T::swz_w((l32 >> 2) * 8 + (l32 & 3)), fb = T::swz_x(l32);
  f32x16 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x16{};
  typedef uint4 Frag[8];  // [quarter][tile]
  auto read_w = [&](const uint16_t* buf, Frag& f) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        f[2 * s + i] = *reinterpret_cast<const uint4*>(buf + arow + i * 256 + ((2 * s + hl) ^ fa) * 8);
  };
  auto read_x = [&](const uint16_t* buf, Frag& f) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        f[2 * s + i] = *reinterpret_cast<const uint4*>(buf + brow + i * 2048 + ((2 * s + hl) ^ fb) * 8);
  };
  auto quadrant = [&](const Frag& a, const Frag& b, int ha, int hb) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          acc[2 * ha + i][2 * hb + j] = Half<F16>::mfma(__builtin_bit_cast(vec, a[2 * s + i]),
                                                        __builtin_bit_cast(vec, b[2 * s + j]),
                                                        acc[2 * ha + i][2 * hb + j]);
    constexpr int kMfma = 0x008, kDsRead = 0x100, kVmem = 0x020;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kVmem, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto landed = [&] {  // the halves loaded three pairs of phases ago; two pairs' loads are behind them
    wait_vmcnt<16>();
    block_barrier();
  };
  Frag fa0, fa1, fb0, fb1;
  // One step with its A0 in c0, the other A registers c1; ends with the next
  // step's A0 in c1. *c: this step's buffers, *n: the next step's.
  constexpr std::true_type may_end{};
  constexpr std::false_type whole{};
  auto step = [&](auto tail, int t, Frag& c0, Frag& c1, uint16_t* a0c, uint16_t* a1c, uint16_t* b0c, uint16_t* b1c, uint16_t* a0n,
                  uint16_t* b0n) {
    landed();
    read_w(a1c, c1);
    load_x(tail, t + 2, 0, b0c);
    quadrant(c0, fb0, 0, 0);
    read_x(b1c, fb1);
    load_w(tail, t + 2, 0, a0c);
    quadrant(c1, fb0, 1, 0);
    landed();
    read_x(b0n, fb0);
    load_w(tail, t + 2, 1, a1c);
    quadrant(c1, fb1, 1, 1);
    read_w(a0n, c1);
    load_x(tail, t + 2, 1, b1c);
    quadrant(c0, fb1, 0, 1);
  };
  load_x(may_end, 0, 0, b00);
  load_w(may_end, 0, 0, a00);
  load_w(may_end, 0, 1, a10);
  load_x(may_end, 0, 1, b10);
  load_x(may_end, 1, 0, b01);
  load_w(may_end, 1, 0, a01);
  load_w(may_end, 1, 1, a11);
  load_x(may_end, 1, 1, b11);
  wait_vmcnt<24>();
  block_barrier();
  read_x(b00, fb0);
  read_w(a00, fa0);
  int t = 0;
  for (; (t + 4) * 64 <= K; t += 2) {  // nothing past K is loaded
    step(whole, t, fa0, fa1, a00, a10, b00, b10, a01, b01);
    step(whole, t + 1, fa1, fa0, a01, a11, b01, b11, a00, b00);
  }
#pragma unroll 1
  for (; t < steps; t += 2) {
    step(may_end, t, fa0, fa1, a00, a10, b00, b10, a01, b01);
    step(may_end, t + 1, fa1, fa0, a01, a11, b01, b11, a00, b00);
  }
  wait_vmcnt_0();  // the trailing loads have landed before the workgroup's LDS is released
  // A lane's 16 outputs of a row lie 64 rows apart from its neighbour's, so the
  // sums go through LDS, 32 rows x 64 outputs at a time, in the wave's own part
  // of it: whole rows of 128 bytes leave (and come, for the residual).
  float* const st = stage + w * 2048;
  const bool inside = m0 + 256 <= p.M && n0 + 256 <= p.N;
  float* const part = p.part + static_cast<int64_t>(split * cut + id - p.whole) * 65536;  // of a tile in parts
#pragma unroll
  for (int gp = 0; gp < 2; ++gp) {
    const int n = n0 + wn * 128 + gp * 64 + (lane & 7) * 8, c = (lane & 7) * 2;
    float bias[8], gate[8];
    load_columns8(p, n, bias, gate);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // outputs g * 32 + hl * 16 + 4 i .. + 3 of row l32
          const f32x16& z = acc[i][j];
          *reinterpret_cast<float4*>(st + l32 * 64 + ((g * 8 + hl * 4 + i) ^ (l32 & 15)) * 4) =
              make_float4(z[gp * 8 + g * 4], z[gp * 8 + g * 4 + 1], z[gp * 8 + g * 4 + 2], z[gp * 8 + g * 4 + 3]);
        }
      auto row = [&](int i, float* z) {
        const int r = i * 8 + (lane >> 3);
        const float4 lo = *reinterpret_cast<const float4*>(st + r * 64 + (c ^ (r & 15)) * 4);
        const float4 hi = *reinterpret_cast<const float4*>(st + r * 64 + ((c + 1) ^ (r & 15)) * 4);
        z[0] = lo.x; z[1] = lo.y; z[2] = lo.z; z[3] = lo.w;
        z[4] = hi.x; z[5] = hi.y; z[6] = hi.z; z[7] = hi.w;
        return m0 + wm * 128 + j * 32 + r;
      };
      if (in_parts) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float z[8];
          float* const at = part + (row(i, z) - m0) * 256 + n - n0;
          *reinterpret_cast<float4*>(at) = make_float4(z[0], z[1], z[2], z[3]);
          *reinterpret_cast<float4*>(at + 4) = make_float4(z[4], z[5], z[6], z[7]);
        }
      } else if (inside) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float z[8];
          const int m = row(i, z);
          finish8_wide<F16, ACT>(p, m, n, z, bias, gate);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          float z[8];
          const int m = row(i, z);
          finish8_edge<F16, ACT>(p, m, n, z, bias, gate);
        }
      }
    }
  }
}

// Joins the parts of a cut product, in their order, and finishes: a thread has
// eight outputs.
template <bool F16>
__global__ void __launch_bounds__(256) linear_join_kernel(LinearParams p) {
  const int chunks = (p.N + 7) / 8;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int m = static_cast<int>(id / chunks), n = static_cast<int>(id - static_cast<int64_t>(m) * chunks) * 8;
  if (m >= p.M) return;
  const int64_t ld = chunks * 8;
  const float* src = p.part + m * ld + n;
  float z[8] = {};
  for (int i = 0; i < p.splits; ++i, src += p.M * ld) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    z[0] += a.x; z[1] += a.y; z[2] += a.z; z[3] += a.w;
    z[4] += b.x; z[5] += b.y; z[6] += b.z; z[7] += b.w;
  }
  float bias[8], gate[8];
  load_columns8(p, n, bias, gate);
  with_activation(p.act, [&](auto act) { finish8<F16, decltype(act)::value>(p, m, n, z, bias, gate); });
}

// The same for the 256 x 256 tiles in parts, 32 workgroups a tile.
template <bool F16>
__global__ void __launch_bounds__(256) linear_join_big_kernel(LinearParams p) {
  const int mt = (p.M + 255) / 256, nt = (p.N + 255) / 256, cut = mt * nt - p.whole;
  const int tile = blockIdx.x >> 5, row = (blockIdx.x & 31) * 8 + (threadIdx.x >> 5), col = (threadIdx.x & 31) * 8;
  int tm, tn;
  tile_of(p.whole + tile, mt, nt, tm, tn);
  const int m = tm * 256 + row, n = tn * 256 + col;
  if (m >= p.M || n >= p.N) return;
  float z[8] = {};
  for (int i = 0; i < p.splits; ++i) {
    const float* const src = p.part + static_cast<int64_t>(i * cut + tile) * 65536 + row * 256 + col;
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    z[0] += a.x; z[1] += a.y; z[2] += a.z; z[3] += a.w;
    z[4] += b.x; z[5] += b.y; z[6] += b.z; z[7] += b.w;
  }
  float bias[8], gate[8];
  load_columns8(p, n, bias, gate);
  with_activation(p.act, [&](auto act) { finish8<F16, decltype(act)::value>(p, m, n, z, bias, gate); });
}

template <int NI, int MI, int WN, int WM, int NS>
void launch_tile(const LinearParams& p, bool f16, hipStream_t st) {
  const int64_t mt = (p.M + 32 * MI * WM - 1) / (32 * MI * WM), nt = (p.N + 32 * NI * WN - 1) / (32 * NI * WN);
  const dim3 grid(static_cast<unsigned>(mt * nt * p.splits));
  if (f16)
    linear_tile_kernel<NI, MI, WN, WM, NS, true><<<grid, 256, 0, st>>>(p);
  else
    linear_tile_kernel<NI, MI, WN, WM, NS, false><<<grid, 256, 0, st>>>(p);
  if (p.splits > 1) {
    const int64_t threads = static_cast<int64_t>(p.M) * ((p.N + 7) / 8);
    const dim3 join(static_cast<unsigned>((threads + 255) / 256));
    if (f16)
      linear_join_kernel<true><<<join, 256, 0, st>>>(p);
    else
      linear_join_kernel<false><<<join, 256, 0, st>>>(p);
  }
}

// Whether the few-row form reads w past the last-level cache, and whether it
// takes more waves a workgroup, where there are few of them.
bool few_stream(int64_t n, int64_t k) { return n * k * 2 > kLastLevelCache; }
bool few_wide(int64_t n, int64_t k) { return !few_stream(n, k) && (n + 15) / 16 < 256; }

template <bool F16>
void launch_few(const LinearParams& p, hipStream_t st) {
  const int groups = (p.N + 15) / 16;
  if (few_stream(p.N, p.K))
    linear_few_kernel<4, F16, true><<<groups, 256, 0, st>>>(p);
  else if (few_wide(p.N, p.K))
    linear_few_kernel<8, F16, false><<<groups, 512, 0, st>>>(p);
  else
    linear_few_kernel<4, F16, false><<<groups, 256, 0, st>>>(p);
}

// The rows of x, then those of w, K elements each at any stride, into rows of
// `wide` >= K elements on 16-byte boundaries, zeros behind the K: eight elements
// a thread, a row a grid row.
__global__ void __launch_bounds__(256) pad_rows_kernel(LinearParams p, int wide, uint16_t* dst) {
  const int k = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (k >= wide) return;
  for (int r = blockIdx.y; r < p.M + p.N; r += gridDim.y) {
    const uint16_t* const src = r < p.M ? p.x + r * p.ldx : p.w + (r - p.M) * p.ldw;
    *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(r) * wide + k) = load_row8(src, k, p.K);
  }
}

// How a product is cut: its form and, for the tiles, the parts of the channels.
enum Form {
  kFew = DFS_LINEAR_FEW,
  kTileAny = DFS_LINEAR_ANY,
  kTile64 = DFS_LINEAR_64,
  kTile64x128 = DFS_LINEAR_64X128,
  kTile128Deep = DFS_LINEAR_128_DEEP,
  kTile128 = DFS_LINEAR_128,
  kTile256 = DFS_LINEAR_256
};
struct Cut {
  Form form;
  int splits, depth;
  bool pad;       // operands are laid out on 16-byte rows first
  int64_t whole;  // 256 x 256 tiles that are not cut
};
int64_t big_tiles(int64_t rows, int64_t n) { return (rows + 255) / 256 * ((n + 255) / 256); }
Cut cut_of(int64_t rows, int64_t n, int64_t k, bool chunks) {
  // Rows on no 16-byte boundary: small products of few steps as they are, the
  // others laid out anew (us in a graph, as they are and anew: 333 by 1,017 x 709 8.9 and
  // 11.3, 100 by 5,119 x 1,001 11.7 and 15.9; 333 by 1,017 x 1,501 13.6 and 14.9,
  // 100 by 1,001 x 2,001 16.6 and 13.6, 64 by 640 x 6,001 35.8 and 18.8).
  if (!chunks && k <= 1024 && rows * n * k < (int64_t(1) << 30)) return Cut{kTileAny, 1, 0, false, 0};
  if (rows <= 8) return Cut{kFew, 1, 0, !chunks, 0};
  // The tiles and parts with the least time by what each took on an idle CU and
  // beside others, a step of 64 channels of a workgroup in us, and by writing
  // and joining the parts' sums at 3 TB/s behind 5 us. Where several fit on a
  // CU, those that get one more than others run it half hidden. Measured, us,
  // in the order below: 128 rows by 5,120 x 5,120 20.8, 28.5, 38.7, 58, 93; 256
  // rows 34.9, 29.4, 39.8, 57, 84; 512 by 5,120 x 4,096 44.9, 38.8, 35.4, 44.6,
  // 70; 1,000 by 5,120 x 5,120 96, 87, 83, 70, 98; 1,560 144, 129, 130, 132, 89;
  // 64 rows in four parts of 64 x 64 17.3, in one 20.8.
  const struct {
    Form form;
    int m, n, most;  // most: parts
    bool single;     // one workgroup a CU
    double alone, beside;
  } kinds[5] = {{kTile64, 64, 64, 8, false, 0.26, 0.25},
                {kTile64x128, 128, 64, 4, false, 0.36, 0.375},
                {kTile128Deep, 128, 128, 2, true, 0.55, 0.55},
                {kTile128, 128, 128, 4, false, 0.72, 0.57},
                {kTile256, 256, 256, 1, true, 1.15, 1.4}};
  Cut best{kTile64, 1, 0, !chunks, 0};
  double least = 1e30;
  for (const auto& f : kinds)
    for (int s = 1; s <= f.most; s *= 2) {
      const int64_t depth = ((k + s - 1) / s + 127) / 128 * 128, parts = (k + depth - 1) / depth;
      if (s > 1 && (depth < 256 || parts < 2)) break;
      const int64_t groups = ((rows + f.m - 1) / f.m) * ((n + f.n - 1) / f.n) * parts;
      const double full = static_cast<double>((groups + 255) / 256), part = static_cast<double>(groups) / 256.0;
      const double each = f.single ? full : 0.5 * (full + part);
      double us = static_cast<double>((depth + 63) / 64) * std::max(f.alone, f.beside * (f.single && full < 2 ? 0 : each));
      if (parts > 1) us += 5.0 + 8e-6 / 3.0 * static_cast<double>(parts * rows * n);
      if (us < least) {
        least = us;
        best.form = f.form;
        best.splits = static_cast<int>(parts);
        best.depth = static_cast<int>(depth);
      }
    }
  // The 256 x 256 tiles behind the last full round of 256 in parts, which
  // together fill it (us, whole and in parts: 3,600 by 5,120 x 5,120 204 and 170,
  // 4,200 by 4,200 x 3,000 164 and 121, 4,680 by 5,120 x 5,120 212 and 206,
  // 75,600 by 5,120 x 13,824 7,680 and 7,565).
  const int64_t tiles = big_tiles(rows, n), whole = tiles / 256 * 256, rest = tiles - whole, steps = (k + 63) / 64;
  best.whole = best.form == kTile256 ? tiles : 0;
  for (int64_t s = 2; rest > 0 && rest * s <= 256; ++s) {
    const int64_t depth = ((k + s - 1) / s + 127) / 128 * 128, parts = (k + depth - 1) / depth;
    if (depth < 512) break;
    const double us = 1.4 * static_cast<double>(steps * (whole / 256) + depth / 64) + 10.0 +
                      8e-6 / 3.0 * static_cast<double>(parts * rest * 65536);
    if (parts == s && us < least) {
      least = us;
      best = Cut{kTile256, static_cast<int>(parts), static_cast<int>(depth), best.pad, whole};
    }
  }
  return best;
}

int64_t padded(int64_t k) { return (k + 7) / 8 * 8; }
int64_t part_bytes(const Cut& c, int64_t rows, int64_t n) {
  if (c.splits <= 1) return 0;
  return c.form == kTile256 ? c.splits * (big_tiles(rows, n) - c.whole) * 65536 * 4 : c.splits * rows * padded(n) * 4;
}
int64_t workspace_bytes_of(const Cut& c, int64_t rows, int64_t n, int64_t k) {
  return part_bytes(c, rows, n) + (c.pad ? (rows + n) * padded(k) * 2 : 0);
}

}  // namespace
}  // namespace dfs

extern "C" int64_t dfs_linear_workspace_size(int64_t rows, int64_t n, int64_t k, int aligned) {
  using namespace dfs;
  if (rows <= 0 || n <= 0 || k <= 0) {
    set_error("linear: rows=%lld n=%lld k=%lld must be positive", (long long)rows, (long long)n, (long long)k);
    return -1;
  }
  return workspace_bytes_of(cut_of(rows, n, k, aligned != 0), rows, n, k);
}

extern "C" int dfs_linear_form(int64_t rows, int64_t n, int64_t k, int aligned) {
  using namespace dfs;
  if (rows <= 0 || n <= 0 || k <= 0) {
    set_error("linear: rows=%lld n=%lld k=%lld must be positive", (long long)rows, (long long)n, (long long)k);
    return -1;
  }
  const Cut c = cut_of(rows, n, k, aligned != 0);
  int form = c.form;
  if (c.splits > 1) form |= DFS_FORM_PARTS;
  if (c.pad) form |= DFS_LINEAR_LAID_OUT;
  if (c.form == kFew && few_stream(n, padded(k))) form |= DFS_FORM_STREAM;
  if (c.form == kFew && few_wide(n, padded(k))) form |= DFS_LINEAR_WIDE;
  return form;
}

extern "C" int dfs_linear(const dfs_linear_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "linear";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  const void *x = a->x, *w = a->w, *bias = a->bias, *residual = a->residual;
  const int64_t rows = a->rows, n = a->n, k = a->k, x_stride = a->x_stride, w_stride = a->w_stride;
  DFS_REQUIRE(x && w && a->out, "%s: x, w and out must be non-NULL", name);
  DFS_REQUIRE(rows > 0 && n > 0 && k > 0, "%s: rows=%lld n=%lld k=%lld must be positive", name, (long long)rows,
              (long long)n, (long long)k);
  constexpr int64_t kMax = int64_t(1) << 30;
  DFS_REQUIRE(rows < kMax && n < kMax && k < (1 << 21), "%s: rows and n must be below 2^30, k below 2^21", name);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(x_stride >= 0 && w_stride >= 0 && a->out_stride >= n && (!residual || a->residual_stride >= 0),
              "%s: strides must be non-negative, and out's rows must not overlap", name);
  DFS_REQUIRE(bias == nullptr || a->bias_dtype == DFS_DTYPE_BF16 || a->bias_dtype == DFS_DTYPE_F16 ||
                  a->bias_dtype == DFS_DTYPE_F32,
              "%s: bias dtype code %lld is not supported", name, (long long)a->bias_dtype);
  DFS_REQUIRE(a->activation >= kActNone && a->activation <= kActSilu, "%s: activation code %lld is not supported",
              name, (long long)a->activation);
  auto addr = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  DFS_REQUIRE(addr(x) % 2 == 0 && addr(w) % 2 == 0 && addr(a->out) % 2 == 0 && addr(residual) % 2 == 0 &&
                  addr(a->gate) % 4 == 0 && addr(bias) % (a->bias_dtype == DFS_DTYPE_F32 ? 4 : 2) == 0,
              "%s: operands must be aligned to their elements", name);
  const bool chunks = k % 8 == 0 && x_stride % 8 == 0 && w_stride % 8 == 0 && addr(x) % 16 == 0 && addr(w) % 16 == 0 &&
                      x_stride < (1 << 21) && w_stride < (1 << 21);
  const Cut cut = cut_of(rows, n, k, chunks);
  const int64_t need = workspace_bytes_of(cut, rows, n, k);
  DFS_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need && addr(a->workspace) % 16 == 0),
              "%s: a 16-byte aligned workspace of %lld bytes is needed", name, (long long)need);
  // A launch holds fewer than 2^32 threads.
  DFS_REQUIRE(((rows + 63) / 64) * ((n + 63) / 64) * cut.splits < (1 << 24) && (cut.form != kFew || n < (1 << 27)),
              "%s: too many outputs", name);
  LinearParams p{};
  p.x = static_cast<const uint16_t*>(x);
  p.w = static_cast<const uint16_t*>(w);
  p.ldx = x_stride;
  p.ldw = w_stride;
  p.ldr = a->residual_stride;
  p.ldo = a->out_stride;
  p.M = static_cast<int>(rows);
  p.N = static_cast<int>(n);
  p.K = static_cast<int>(k);
  p.bias = bias;
  p.bias_dtype = static_cast<int>(a->bias_dtype);
  p.act = static_cast<int>(a->activation);
  p.gate = a->gate;
  p.residual = static_cast<const uint16_t*>(residual);
  p.out = static_cast<uint16_t*>(a->out);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  p.splits = cut.splits;
  p.depth = cut.depth;
  p.whole = static_cast<int>(cut.whole);
  p.part = static_cast<float*>(a->workspace);
  const bool f16 = a->dtype == DFS_DTYPE_F16;
  if (cut.pad) {
    uint16_t* const wide = reinterpret_cast<uint16_t*>(static_cast<char*>(a->workspace) + part_bytes(cut, rows, n));
    const int64_t kp = padded(k);
    const dim3 grid(static_cast<unsigned>((kp + 2047) / 2048), static_cast<unsigned>(std::min<int64_t>(rows + n, 65535)));
    pad_rows_kernel<<<grid, 256, 0, st>>>(p, static_cast<int>(kp), wide);
    p.x = wide;
    p.w = wide + rows * kp;
    p.ldx = p.ldw = kp;
    p.K = static_cast<int>(kp);
  }
  switch (cut.form) {
    case kFew:
      f16 ? launch_few<true>(p, st) : launch_few<false>(p, st);
      break;
    case kTileAny: {
      const unsigned grid = static_cast<unsigned>(((n + 63) / 64) * ((rows + 63) / 64));
      f16 ? linear_any_kernel<true><<<grid, 256, 0, st>>>(p) : linear_any_kernel<false><<<grid, 256, 0, st>>>(p);
      break;
    }
    case kTile64:
      launch_tile<1, 1, 2, 2, 4>(p, f16, st);
      break;
    case kTile64x128:
      launch_tile<1, 2, 2, 2, 3>(p, f16, st);
      break;
    case kTile128Deep:
      launch_tile<2, 2, 2, 2, 3>(p, f16, st);
      break;
    case kTile128:
      launch_tile<2, 2, 2, 2, 2>(p, f16, st);
      break;
    case kTile256: {
      const int64_t rest = big_tiles(rows, n) - cut.whole;
      const dim3 grid(static_cast<unsigned>(cut.whole + rest * cut.splits));
      with_activation(p.act, [&](auto act) {
        if (f16)
          linear_big_kernel<true, decltype(act)::value><<<grid, 256, 0, st>>>(p);
        else
          linear_big_kernel<false, decltype(act)::value><<<grid, 256, 0, st>>>(p);
      });
      if (rest > 0) {
        const dim3 join(static_cast<unsigned>(rest * 32));
        f16 ? linear_join_big_kernel<true><<<join, 256, 0, st>>>(p) : linear_join_big_kernel<false><<<join, 256, 0, st>>>(p);
      }
      break;
    }
  }
  return check_launch(name);
}
