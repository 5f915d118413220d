// Matrix product of 8-bit operands with a scale for every 128 channels of a row
// (fp8_block.h) and the epilogue of linear_epilogue.h:
//   z[m][n] = sum_b 2^(ex[m][b] + ew[n][b]) sum_{k in b} x[m][k] w[n][k] + bias[n]
// The scaled matrix instructions take 32 channels a lane and the power of two of
// the lane's row for them, so a block's scales cost no arithmetic: a product of
// K = 64 or 128 is one instruction. It adds the products of eight consecutive
// channels after cutting each, towards zero, to a multiple of 2^-13 of the
// largest one's power of two (all 8-bit forms do), and the eights' sums in fp32,
// as the sums stay from the first channel to the last. The cut is taken for the
// rate: codes multiplied as 16-bit values would lose nothing at half of it. It
// leaves a sum of 5,120 channels off by 3.5e-5 of its size where fp32 steps leave
// 1e-7; rounded to bf16 that is 1.670e-3 for both, to f16 2.11e-4 for 2.07e-4.
// Which channels a lane holds is free as long as both operands agree: a lane
// takes whole 16-byte chunks, as the 16-bit products do, and the layouts in LDS,
// the dealing of rows to tiles and the epilogue are theirs, 128 codes in the place
// of 64 values.
#include <algorithm>

#include "linear_fp8.h"

namespace dfs {
namespace {

// Sums of a workgroup's 16 outputs n0.. for up to 16 rows, one set a wave in LDS
// ([wave][lane][4]: output 4 g + r of row m lies in register r of lane
// 16 g + m), joined in the waves' order and finished.
template <bool F16>
__device__ __forceinline__ void finish16(const Epilogue& p, int n0, const float* sums, int waves) {
  const int e = threadIdx.x, n16 = e & 15, m = e >> 4, n = n0 + n16;
  if (e >= 256 || m >= p.M || n >= p.N) return;
  float z = 0.f;
  for (int v = 0; v < waves; ++v) z += sums[v * 256 + ((n16 >> 2) * 16 + m) * 4 + (n16 & 3)];
  z += bias_at(p, n);
  with_fp8_activation(p.act, [&](auto act) { z = activate<decltype(act)::value>(z); });
  if (p.gate) z *= p.gate[n];
  if (p.residual) z += Half<F16>::to_f32(p.residual[m * p.ldr + n]);
  p.out[m * p.ldo + n] = static_cast<uint16_t>(Half<F16>::from_f32(z));
}

// At most 16 rows of x, the columns of one matrix instruction: what counts is
// reading w once. A workgroup owns 16 outputs, and its waves deal the channels
// among themselves in blocks of 256. A wave's blocks of w pass through three LDS
// buffers of its own that the loads fill directly, 256 bytes of a row at a time; x
// and the scales come from L2 as they are needed. No barrier before the waves'
// sums meet. Bound by memory: 1 row by 30,720 x 5,120 25.4 us, 6.2 TB/s. Rows
// quantised here, by each workgroup for itself, instead of before took 39.3 us
// for 28.0 with the launch before it.
template <int WAVES, bool F16, bool STREAM>
__global__ void __launch_bounds__(64 * WAVES) fp8_few_kernel(Fp8Params p) {
  constexpr int kBytes = 16 * 256;  // of a wave's buffer
  __shared__ __attribute__((aligned(16))) uint8_t s0[WAVES * kBytes], s1[WAVES * kBytes], s2[WAVES * kBytes];
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
    wv[j] = static_cast<uint32_t>(min(n0 + r, p.N - 1) - n0) * static_cast<uint32_t>(p.ldw) + (r16 ^ r) * 16;
  }
  const uint8_t* const xr = p.x + min(r16, p.M - 1) * p.ldx;
  const uint8_t* const xsr = p.xs + min(r16, p.M - 1);
  const uint8_t* const wsr = p.ws + min(n0 + r16, p.N - 1);
  const int blocks = (p.K + 255) >> 8;
  auto load = [&](int b, uint8_t* buf) {  // past the last block: zeros, without a memory access
    const int left = p.K - b * 256;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = (r16 ^ (4 * j + c4)) * 16 < left;
      load_lds16<STREAM>(rs, buf + w * kBytes + j * 1024, in ? wv[j] + b * 256 : kOutside, 0);
    }
  };
  f32x4 acc = f32x4{};
  auto step = [&](int b, const uint8_t* buf, uint8_t* next) {
    i32x4 x[4];
    uint32_t sx[2], sw[2];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = b * 256 + s * 64 + c4 * 16;
      x[s] = i32x4{};
      if (r16 < p.M && k < p.K) x[s] = chunk_at(xr + k);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = min(2 * b + s, p.kb - 1);
      sx[s] = xsr[at * p.ldxs];
      sw[s] = wsr[at * p.ldws];
    }
    wait_lgkm_0();  // the reads of `next`, a step ago, are done (zeros come at once)
    load(b + 2 * WAVES, next);
    const uint8_t* const row = buf + w * kBytes + r16 * 256;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const i32x4 lo = chunk_at(row + ((s * 8 + c4) ^ r16) * 16), hi = chunk_at(row + ((s * 8 + c4 + 4) ^ r16) * 16);
      acc = mfma16(join(lo, hi), join(x[2 * s], x[2 * s + 1]), acc, sw[s], sx[s]);
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
// = 4 waves with NI x MI products of 32 x 32 each, 128 channels (a scale's
// block) a step through NS LDS buffers that the loads fill directly. Layouts
// and order are those of the 16-bit products' tiles: a row of a step is eight
// 16-byte chunks, chunk c of row r at c ^ f(r), and a lane ends with 4 NI
// consecutive outputs. A step has two halves of 64 channels, each one matrix
// instruction a tile: the fragments of a half are read while the half before is
// multiplied; before the second half's products the next step's data is waited
// for and, behind the barrier, the loads of the step NS on go into the buffer
// just read. A step's scales, a byte for each of the lane's rows, lie row by row
// in memory and come with its data. Bound by a step's latency where there are few
// tiles: 512 rows by 5,120 x 4,096 24.0 us in 160 tiles of 128 x 128, 32 steps of
// 0.65 us behind another; five or six buffers gained nothing (23.8, 25.8).
template <int NI, int MI, int WN, int WM, int NS, bool F16>
__global__ void __launch_bounds__(256, 2) fp8_tile_kernel(Fp8Params p) {
  typedef Tile<NI, MI, WN, WM, F16> T;
  constexpr int JW = T::BN / 32, JX = T::BM / 32;  // loads of 1 KB a wave and step
  constexpr int DATA = JW + JX, SCALES = NI + MI;  // loads of a wave and step
  // Of buffers 2 and 3, those past NS are empty.
  constexpr int N2 = NS > 2 ? 128 : 1, N3 = NS > 3 ? 128 : 1;
  __shared__ __attribute__((aligned(16))) uint8_t w0[T::BN * 128], w1[T::BN * 128], w2[T::BN * N2], w3[T::BN * N3];
  __shared__ __attribute__((aligned(16))) uint8_t x0[T::BM * 128], x1[T::BM * 128], x2[T::BM * N2], x3[T::BM * N3];
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
    wv[j] = static_cast<uint32_t>(min(n0 + r, p.N - 1) - n0) * static_cast<uint32_t>(p.ldw) + (c8 ^ T::swz_w(r)) * 16;
  }
#pragma unroll
  for (int j = 0; j < JX; ++j) {
    const int r = j * 32 + r8;
    xv[j] = static_cast<uint32_t>(min(m0 + r, p.M - 1) - m0) * static_cast<uint32_t>(p.ldx) + (c8 ^ T::swz_x(r)) * 16;
  }
  const int steps = (K + 128 * NS - 1) / (128 * NS) * NS;  // the last may be all zeros
  // The scales of this lane's rows.
  const int wn = w % WN, wm = w / WN;
  const int nrow = wn * 32 * NI + (l32 >> 2) * 4 * NI + (l32 & 3), mrow = wm * 32 * MI + l32;
  const uint8_t *wsr[NI], *xsr[MI];
#pragma unroll
  for (int i = 0; i < NI; ++i) wsr[i] = p.ws + min(n0 + nrow + i * 4, p.N - 1);
#pragma unroll
  for (int j = 0; j < MI; ++j) xsr[j] = p.xs + min(m0 + mrow + j * 32, p.M - 1);
  struct Scales {
    uint32_t w[NI], x[MI];
  };
  auto load_scales = [&](int t, Scales& s) {
    const int b = min((from >> 7) + t, p.kb - 1);
#pragma unroll
    for (int i = 0; i < NI; ++i) s.w[i] = wsr[i][b * p.ldws];
#pragma unroll
    for (int j = 0; j < MI; ++j) s.x[j] = xsr[j][b * p.ldxs];
  };
  auto issue = [&](int t, uint8_t* wb, uint8_t* xb) {
    const int left = K - t * 128;
    if (left < 128) {  // the last steps: chunks past K come as zeros
#pragma unroll
      for (int j = 0; j < JX; ++j)
        if ((c8 ^ T::swz_x(j * 32 + r8)) * 16 >= left) xv[j] = kOutside;
#pragma unroll
      for (int j = 0; j < JW; ++j)
        if ((c8 ^ T::swz_w(j * 32 + r8)) * 16 >= left) wv[j] = kOutside;
    }
#pragma unroll
    for (int j = 0; j < JX; ++j) load_lds16(xrs, xb + (j * 4 + w) * 1024, xv[j], t * 128);
#pragma unroll
    for (int j = 0; j < JW; ++j) load_lds16(wrs, wb + (j * 4 + w) * 1024, wv[j], t * 128);
  };
  const int fa = T::swz_w((l32 >> 2) * 4 * NI + (l32 & 3)), fb = T::swz_x(l32);
  f32x16 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j) acc[i][j] = f32x16{};
  auto fetch = [&](const uint8_t* wb, const uint8_t* xb, int u, i32x8* a, i32x8* b) {
    const int ca = (4 * u + hl) ^ fa, cb = (4 * u + hl) ^ fb;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint8_t* const row = wb + (nrow + i * 4) * 128;
      a[i] = join(chunk_at(row + ca * 16), chunk_at(row + (ca ^ 2) * 16));
    }
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const uint8_t* const row = xb + (mrow + j * 32) * 128;
      b[j] = join(chunk_at(row + cb * 16), chunk_at(row + (cb ^ 2) * 16));
    }
  };
  auto multiply = [&](const i32x8* a, const i32x8* b, const Scales& s) {
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][j] = mfma32(a[i], b[j], acc[i][j], s.w[i], s.x[j]);
  };
  // Loads keep their order over a fence (neither moves over it), within a stretch
  // between two they may not: so a step's data and the scales of another lie in
  // stretches of their own, taking turns from the beginning on, and a wait can
  // count what is behind the data it needs: DATA and SCALES instructions a step, to
  // which the built code is held by tests/test_waits_host.py.
  auto fence = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  i32x8 a0[NI], b0[MI], a1[NI], b1[MI];
  auto step = [&](int t, uint8_t* wc, uint8_t* xc, const Scales& s, Scales& before, const uint8_t* wnext,
                  const uint8_t* xnext) {
    load_scales(t + NS - 1, before);
    fetch(wc, xc, 1, a1, b1);
    multiply(a0, b0, s);
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<(NS - 2) * DATA + (NS - 1) * SCALES>();
    block_barrier();
    issue(t + NS, wc, xc);           // past the last step: zeros, without a memory access
    fetch(wnext, xnext, 0, a0, b0);  // past the last step: read and not used
    multiply(a1, b1, s);
    fence();
  };
  Scales s0, s1, s2, s3;
  issue(0, w0, x0);
  fence();
  load_scales(0, s0);
  fence();
  issue(1, w1, x1);
  fence();
  if constexpr (NS > 2) {
    load_scales(1, s1);
    fence();
    issue(2, w2, x2);
    fence();
  }
  if constexpr (NS > 3) {
    load_scales(2, s2);
    fence();
    issue(3, w3, x3);
    fence();
  }
  wait_vmcnt<(NS - 1) * (DATA + SCALES)>();
  block_barrier();
  fetch(w0, x0, 0, a0, b0);
  for (int t = 0; t < steps; t += NS) {
    if constexpr (NS == 2) {
      step(t, w0, x0, s0, s1, w1, x1);
      step(t + 1, w1, x1, s1, s0, w0, x0);
    }
    if constexpr (NS == 3) {
      step(t, w0, x0, s0, s2, w1, x1);
      step(t + 1, w1, x1, s1, s0, w2, x2);
      step(t + 2, w2, x2, s2, s1, w0, x0);
    }
    if constexpr (NS == 4) {
      step(t, w0, x0, s0, s3, w1, x1);
      step(t + 1, w1, x1, s1, s0, w2, x2);
      step(t + 2, w2, x2, s2, s1, w3, x3);
      step(t + 3, w3, x3, s3, s2, w0, x0);
    }
  }
  wait_vmcnt_0();  // the trailing loads have landed before the workgroup's LDS is released
  const int nb = n0 + wn * 32 * NI + hl * 4 * NI, mb = m0 + mrow;
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
  with_fp8_activation(p.act, [&](auto act) {
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

// Joins the parts of a cut product, in their order, and finishes: a thread has
// eight outputs.
template <bool F16>
__global__ void __launch_bounds__(256) fp8_join_kernel(Fp8Params p) {
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
  with_fp8_activation(p.act, [&](auto act) { finish8<F16, decltype(act)::value>(p, m, n, z, bias, gate); });
}

// Scale bytes [blocks][rows] at any stride into ones of stride `wide`, a multiple
// of 4, zeros behind the rows.
__global__ void __launch_bounds__(256) pad_scales_kernel(const uint8_t* src, int64_t ld, int rows, int wide, uint8_t* dst) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < wide) dst[static_cast<int64_t>(blockIdx.y) * wide + r] = r < rows ? src[blockIdx.y * ld + r] : 0;
}

__global__ void __launch_bounds__(256) pad_codes_kernel(PadCodes p) { pad_codes(p, blockIdx.x, gridDim.x); }

template <int NI, int MI, int WN, int WM, int NS>
void launch_tile(const Fp8Params& p, bool f16, hipStream_t st) {
  const int64_t mt = (p.M + 32 * MI * WM - 1) / (32 * MI * WM), nt = (p.N + 32 * NI * WN - 1) / (32 * NI * WN);
  const dim3 grid(static_cast<unsigned>(mt * nt * p.splits));
  if (f16)
    fp8_tile_kernel<NI, MI, WN, WM, NS, true><<<grid, 256, 0, st>>>(p);
  else
    fp8_tile_kernel<NI, MI, WN, WM, NS, false><<<grid, 256, 0, st>>>(p);
  if (p.splits > 1) {
    const int64_t threads = static_cast<int64_t>(p.M) * ((p.N + 7) / 8);
    const dim3 join(static_cast<unsigned>((threads + 255) / 256));
    f16 ? fp8_join_kernel<true><<<join, 256, 0, st>>>(p) : fp8_join_kernel<false><<<join, 256, 0, st>>>(p);
  }
}

// Whether the few-row form reads w past the last-level cache, and whether it
// takes more waves a workgroup, where there are few of them.
bool few_stream(int64_t n, int64_t k) { return n * k > kLastLevelCache; }
bool few_wide(int64_t n, int64_t k) { return !few_stream(n, k) && (n + 15) / 16 < 256; }

template <bool F16>
void launch_few(const Fp8Params& p, hipStream_t st) {
  const int groups = (p.N + 15) / 16;
  if (few_stream(p.N, p.K))
    fp8_few_kernel<4, F16, true><<<groups, 256, 0, st>>>(p);
  else if (few_wide(p.N, p.K))
    fp8_few_kernel<8, F16, false><<<groups, 512, 0, st>>>(p);
  else
    fp8_few_kernel<4, F16, false><<<groups, 256, 0, st>>>(p);
}

// How a product is cut: its form and, for the tiles, the parts of the channels.
enum Form {
  kFew = DFS_LINEAR_FEW,
  kTile64 = DFS_LINEAR_64,
  kTile64x128 = DFS_LINEAR_64X128,
  kTile128Deep = DFS_LINEAR_128_DEEP,
  kTile128 = DFS_LINEAR_128,
  kTile256 = DFS_LINEAR_256
};
struct Cut {
  Form form;
  int splits, depth;
  int64_t whole;  // 256 x 256 tiles that are not cut
};
int64_t big_tiles(int64_t rows, int64_t n) { return (rows + 255) / 256 * ((n + 255) / 256); }
Cut cut_of(int64_t rows, int64_t n, int64_t k) {
  // Few rows: their form reads x from L2 for each 16 outputs, the tiles for each
  // 64, so it is for four rows (a quarter of w's bytes), more only by so many
  // outputs. Measured, us for 1, 4, 8 and 16 rows, and for the tiles: 5,120 x
  // 5,120 5.6, 6.4, 7.1, 8.8 and 11.3; 8,192 x 5,120 9.1, 9.4, 9.8, 10.8 and 12.5;
  // 10,240 x 5,120 11.2, 11.8, 12.4, 14.4 and 13.3; 20,480 x 13,824 47.9, 47.0,
  // 50.6, 63.0 and 51.9; 30,720 x 5,120 25.4, 26.5, 28.0, 32.7 and 25.5; 131,072 x
  // 5,120 109.3 for one row, 126.2 in tiles. Few channels by many outputs are the
  // exception that the rule leaves: 30,720 x 1,024 9.4 for one row, 7.3 in tiles.
  if (rows <= 4 || (rows <= 16 && rows * n <= (1 << 17))) return Cut{kFew, 1, 0, 0};
  // The tiles and parts with the least time by what each takes on an idle CU and
  // beside others, a step of 128 channels of a workgroup in us, and by writing
  // and joining the parts' sums at 3 TB/s behind 5 us. Where several fit on a
  // CU, those that get one more than others run it half hidden. Measured, us, in
  // the order below: 128 rows by 5,120 x 5,120 14.5, 20.5, 27.8, 28.1; 256 rows
  // 22.1, 21.4, 28.6, 33.3, 47.6; 512 by 5,120 x 4,096 26.2, 25.5, 24.0, 25.9,
  // 40.0; 1,000 by 5,120 x 5,120 55.5, 47.9, 55.4, 42.8, 58.1; 1,560 79, 76, 86,
  // 75, 50.5; 4,096 by 4,096 x 4,096 128, 102, 98, 79, 55; 64 rows by 5,120 x 5,120
  // in two parts of 64 x 64 12.3, in one 13.4, in four 14.7.
  const struct {
    Form form;
    int m, n, most;  // most: parts
    bool single;     // one workgroup a CU
    double alone, beside;
  } kinds[5] = {{kTile64, 64, 64, 8, false, 0.29, 0.26},
                {kTile64x128, 128, 64, 4, false, 0.44, 0.40},
                {kTile128Deep, 128, 128, 2, true, 0.63, 0.65},
                {kTile128, 128, 128, 4, false, 0.68, 0.61},
                {kTile256, 256, 256, 1, true, 1.2, 1.6}};
  Cut best{kTile64, 1, 0, 0};
  double least = 1e30;
  for (const auto& f : kinds)
    for (int s = 1; s <= f.most; s *= 2) {
      const int64_t depth = ((k + s - 1) / s + 255) / 256 * 256, parts = (k + depth - 1) / depth;
      if (s > 1 && parts < 2) break;
      const int64_t groups = ((rows + f.m - 1) / f.m) * ((n + f.n - 1) / f.n) * parts;
      const double full = static_cast<double>((groups + 255) / 256), part = static_cast<double>(groups) / 256.0;
      const double each = f.single ? full : 0.5 * (full + part);
      double us = static_cast<double>((depth + 127) / 128) * std::max(f.alone, f.beside * (f.single && full < 2 ? 0 : each));
      if (parts > 1) us += 5.0 + 8e-6 / 3.0 * static_cast<double>(parts * rows * n);
      if (us < least) {
        least = us;
        best = Cut{f.form, static_cast<int>(parts), static_cast<int>(depth), 0};
      }
    }
  // The 256 x 256 tiles behind the last full round of 256 in parts, which
  // together fill it.
  const int64_t tiles = big_tiles(rows, n), whole = tiles / 256 * 256, rest = tiles - whole, steps = (k + 127) / 128;
  best.whole = best.form == kTile256 ? tiles : 0;
  for (int64_t s = 2; rest > 0 && rest * s <= 256; ++s) {
    const int64_t depth = ((k + s - 1) / s + 255) / 256 * 256, parts = (k + depth - 1) / depth;
    if (depth < 1024) break;
    const double us = 1.6 * static_cast<double>(steps * (whole / 256)) + 1.3 * static_cast<double>(depth / 128) + 10.0 +
                      8e-6 / 3.0 * static_cast<double>(parts * rest * 65536);
    if (parts == s && us < least) {
      least = us;
      best = Cut{kTile256, static_cast<int>(parts), static_cast<int>(depth), whole};
    }
  }
  return best;
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }
int64_t part_bytes(const Cut& c, int64_t rows, int64_t n) {
  if (c.splits <= 1) return 0;
  return c.form == kTile256 ? c.splits * (big_tiles(rows, n) - c.whole) * 65536 * 4
                            : c.splits * rows * ((n + 7) / 8 * 8) * 4;
}
// The workspace: the parts' sums, x's codes (where x comes in 16 bits, or its
// codes off 16-byte rows) and scales (where x comes in 16 bits, or for the
// 256 x 256 tiles, which read four scales at once, off 4-byte boundaries), w's
// the same, and the rounded result where it is left as codes but the form does
// not make them. Each begins on 16 bytes.
struct Workspace {
  int64_t part, x, xs, w, ws, y, total;  // offsets
};
Workspace workspace_of(const Cut& c, int64_t rows, int64_t n, int64_t k, int flags) {
  const int64_t kb = (k + kScaleBlock - 1) / kScaleBlock;
  const bool codes = flags & DFS_FP8_X_CODES, big = c.form == kTile256;
  Workspace s{};
  s.x = s.part + part_bytes(c, rows, n);
  s.xs = s.x + (codes && (flags & DFS_FP8_X_ALIGNED) ? 0 : rows * up16(k));
  s.w = s.xs + (!codes || (big && !(flags & DFS_FP8_XS_ALIGNED)) ? up16(up4(rows) * kb) : 0);
  s.ws = s.w + (flags & DFS_FP8_W_ALIGNED ? 0 : n * up16(k));
  s.y = s.ws + (big && !(flags & DFS_FP8_WS_ALIGNED) ? up16(up4(n) * kb) : 0);
  s.total = s.y + (flags & DFS_FP8_OUT_CODES && !big ? up16(rows * n * 2) : 0);
  return s;
}

bool sizes_fit(int64_t rows, int64_t n, int64_t k) {
  constexpr int64_t kMax = int64_t(1) << 30;
  if (rows > 0 && n > 0 && k > 0 && rows < kMax && n < kMax && k < (1 << 21)) return true;
  set_error("linear_fp8: rows=%lld n=%lld k=%lld must be positive, below 2^30, 2^30 and 2^21", (long long)rows,
            (long long)n, (long long)k);
  return false;
}

}  // namespace
}  // namespace dfs

extern "C" int64_t dfs_linear_fp8_workspace_size(int64_t rows, int64_t n, int64_t k, int flags) {
  using namespace dfs;
  if (!sizes_fit(rows, n, k)) return -1;
  return workspace_of(cut_of(rows, n, k), rows, n, k, flags).total;
}

extern "C" int dfs_linear_fp8_form(int64_t rows, int64_t n, int64_t k) {
  using namespace dfs;
  if (!sizes_fit(rows, n, k)) return -1;
  const Cut c = cut_of(rows, n, k);
  int form = c.form;
  if (c.splits > 1) form |= DFS_FORM_PARTS;
  if (c.form == kFew && few_stream(n, k)) form |= DFS_FORM_STREAM;
  if (c.form == kFew && few_wide(n, k)) form |= DFS_LINEAR_WIDE;
  return form;
}

extern "C" int dfs_linear_fp8(const dfs_linear_fp8_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "linear_fp8";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  const bool codes = a->x_dtype == DFS_DTYPE_E4M3, out8 = a->out8 != nullptr;
  DFS_REQUIRE(a->x && a->w && a->w_scales && (a->out != nullptr) != out8 && out8 == (a->out8_scales != nullptr),
              "%s: x, w, w_scales and out, or out8 with its scales, must be non-NULL", name);
  const int64_t rows = a->rows, n = a->n, k = a->k;
  if (!sizes_fit(rows, n, k)) return 1;
  const int64_t kb = (k + kScaleBlock - 1) / kScaleBlock, nb = (n + kScaleBlock - 1) / kScaleBlock;
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(codes || a->x_dtype == a->dtype, "%s: x must be e4m3 or of the result's dtype", name);
  DFS_REQUIRE(codes == (a->x_scales != nullptr), "%s: x_scales go with codes", name);
  DFS_REQUIRE(a->x_stride >= 0 && a->w_stride >= 0 && (!codes || a->x_scales_stride >= 0) && a->w_scales_stride >= 0 &&
                  (!a->residual || a->residual_stride >= 0),
              "%s: strides must not be negative", name);
  DFS_REQUIRE(out8 ? a->out8_stride >= n && a->out8_scales_stride >= rows : a->out_stride >= n,
              "%s: out's rows must not overlap", name);
  DFS_REQUIRE(a->bias == nullptr || a->bias_dtype == DFS_DTYPE_BF16 || a->bias_dtype == DFS_DTYPE_F16 ||
                  a->bias_dtype == DFS_DTYPE_F32,
              "%s: bias dtype code %lld is not supported", name, (long long)a->bias_dtype);
  DFS_REQUIRE(a->activation >= kActNone && a->activation <= kActSilu, "%s: activation code %lld is not supported",
              name, (long long)a->activation);
  auto addr = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  DFS_REQUIRE((codes || addr(a->x) % 2 == 0) && addr(a->out) % 2 == 0 && addr(a->residual) % 2 == 0 &&
                  addr(a->gate) % 4 == 0 && addr(a->bias) % (a->bias_dtype == DFS_DTYPE_F32 ? 4 : 2) == 0,
              "%s: operands must be aligned to their elements", name);
  auto in_place = [&](const void* q, int64_t stride) {
    return addr(q) % 16 == 0 && k % 16 == 0 && stride % 16 == 0 && stride < (1 << 22);
  };
  int flags = (codes ? DFS_FP8_X_CODES : 0) | (out8 ? DFS_FP8_OUT_CODES : 0);
  if (codes && in_place(a->x, a->x_stride)) flags |= DFS_FP8_X_ALIGNED;
  if (in_place(a->w, a->w_stride)) flags |= DFS_FP8_W_ALIGNED;
  auto in_fours = [&](const void* q, int64_t count, int64_t stride) {
    return addr(q) % 4 == 0 && count % 4 == 0 && stride % 4 == 0;
  };
  if (codes && in_fours(a->x_scales, rows, a->x_scales_stride)) flags |= DFS_FP8_XS_ALIGNED;
  if (in_fours(a->w_scales, n, a->w_scales_stride)) flags |= DFS_FP8_WS_ALIGNED;
  const Cut cut = cut_of(rows, n, k);
  const Workspace at = workspace_of(cut, rows, n, k, flags);
  DFS_REQUIRE(at.total == 0 || (a->workspace != nullptr && a->workspace_bytes >= at.total && addr(a->workspace) % 16 == 0),
              "%s: a 16-byte aligned workspace of %lld bytes is needed", name, (long long)at.total);
  // A launch holds fewer than 2^32 threads: 2^24 - 1 workgroups of x's quantisation
  // (with that of w's rows laid out beside it) and of the result's.
  const PadCodes w_codes{static_cast<const uint8_t*>(a->w), a->w_stride, n, static_cast<int>(k), static_cast<int>(up16(k)),
                         static_cast<uint8_t*>(a->workspace) + at.w};
  const bool pad_w = !(flags & DFS_FP8_W_ALIGNED);
  const int64_t x_groups = codes ? 0 : (rows * kb + 15) / 16 + (pad_w ? pad_groups(w_codes) : 0);
  DFS_REQUIRE(((rows + 63) / 64) * ((n + 63) / 64) * cut.splits < (1 << 24) && kb < 65536 && (cut.form != kFew || n < (1 << 27)) &&
                  rows * kb < (1 << 28) && x_groups < (1 << 24) && (!out8 || rows * nb <= (1 << 28) - 16),
              "%s: too many outputs, or rows by channels", name);
  char* const ws = static_cast<char*>(a->workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = a->dtype == DFS_DTYPE_F16;
  Fp8Params p{};
  p.M = static_cast<int>(rows);
  p.N = static_cast<int>(n);
  p.kb = static_cast<int>(kb);
  p.x = static_cast<const uint8_t*>(a->x);
  p.xs = static_cast<const uint8_t*>(a->x_scales);
  p.ldx = a->x_stride;
  p.ldxs = a->x_scales_stride;
  p.w = static_cast<const uint8_t*>(a->w);
  p.ws = static_cast<const uint8_t*>(a->w_scales);
  p.ldw = a->w_stride;
  p.ldws = a->w_scales_stride;
  const int64_t wide = up16(k);
  if (!codes) {  // w's codes in the same launch
    uint8_t *const xq = reinterpret_cast<uint8_t*>(ws + at.x), *const xsq = reinterpret_cast<uint8_t*>(ws + at.xs);
    p.ldx = wide;
    p.ldxs = up4(rows);
    launch_quantize(static_cast<const uint16_t*>(a->x), rows, k, a->x_stride, f16, xq, wide, wide, xsq, p.ldxs, st,
                    pad_w ? &w_codes : nullptr);
    p.x = xq;
    p.xs = xsq;
  } else if (!(flags & DFS_FP8_X_ALIGNED)) {
    const PadCodes x_codes{p.x, p.ldx, rows, w_codes.k, w_codes.wide, reinterpret_cast<uint8_t*>(ws + at.x)};
    pad_codes_kernel<<<pad_groups(x_codes), 256, 0, st>>>(x_codes);
    p.x = x_codes.dst;
    p.ldx = wide;
  }
  if (pad_w) {
    if (codes) pad_codes_kernel<<<pad_groups(w_codes), 256, 0, st>>>(w_codes);
    p.w = w_codes.dst;
    p.ldw = wide;
  }
  auto fours = [&](const uint8_t* src, int64_t ld, int64_t count, int64_t offset) {
    uint8_t* const dst = reinterpret_cast<uint8_t*>(ws + offset);
    const dim3 grid(static_cast<unsigned>((up4(count) + 255) / 256), static_cast<unsigned>(kb));
    pad_scales_kernel<<<grid, 256, 0, st>>>(src, ld, static_cast<int>(count), static_cast<int>(up4(count)), dst);
    return dst;
  };
  const bool big = cut.form == kTile256;
  if (big && codes && !(flags & DFS_FP8_XS_ALIGNED)) {
    p.xs = fours(p.xs, p.ldxs, rows, at.xs);
    p.ldxs = up4(rows);
  }
  if (big && !(flags & DFS_FP8_WS_ALIGNED)) {
    p.ws = fours(p.ws, p.ldws, n, at.ws);
    p.ldws = up4(n);
  }
  p.K = static_cast<int>(wide);  // zeros behind the k
  p.bias = a->bias;
  p.bias_dtype = static_cast<int>(a->bias_dtype);
  p.act = static_cast<int>(a->activation);
  p.gate = a->gate;
  p.residual = static_cast<const uint16_t*>(a->residual);
  p.ldr = a->residual_stride;
  p.out = out8 ? reinterpret_cast<uint16_t*>(ws + at.y) : static_cast<uint16_t*>(a->out);
  p.ldo = out8 ? n : a->out_stride;
  p.splits = cut.splits;
  p.depth = cut.depth;
  p.whole = static_cast<int>(cut.whole);
  p.part = reinterpret_cast<float*>(ws + at.part);
  if (big && out8) {
    p.out8 = static_cast<uint8_t*>(a->out8);
    p.out8_scales = static_cast<uint8_t*>(a->out8_scales);
    p.ldo8 = a->out8_stride;
    p.ldos = a->out8_scales_stride;
  }
  switch (cut.form) {
    case kFew:
      f16 ? launch_few<true>(p, st) : launch_few<false>(p, st);
      break;
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
      f16 ? run_fp8_large_f16(p, rest, st) : run_fp8_large_bf16(p, rest, st);
      break;
    }
  }
  if (out8 && !big)
    launch_quantize(p.out, rows, n, n, f16, static_cast<uint8_t*>(a->out8), a->out8_stride, n,
                    static_cast<uint8_t*>(a->out8_scales), a->out8_scales_stride, st);
  return check_launch(name);
}
