// The largest tiles of the products of 8-bit operands.
#pragma once

#include <type_traits>

#include "linear_fp8.h"

namespace dfs {
namespace {

// Eight outputs n.. of row m, finished and rounded, as they are stored; zeros
// past the matrix (INSIDE: there are none).
template <bool F16, int ACT, bool INSIDE>
__device__ __forceinline__ uint4 finished8(const Epilogue& p, int m, int n, const float* z, const float* bias,
                                           const float* gate) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = activate<ACT>(z[i] + bias[i]);
  if (p.gate) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= gate[i];
  }
  if (p.residual) {
    if (INSIDE || (m < p.M && n + 8 <= p.N)) {
      uint4 rv;
      __builtin_memcpy(&rv, p.residual + m * p.ldr + n, 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += Half<F16>::to_f32(u16_at(rv, i));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (m < p.M && n + i < p.N) y[i] += Half<F16>::to_f32(p.residual[m * p.ldr + n + i]);
    }
  }
  if constexpr (!INSIDE) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (m >= p.M || n + i >= p.N) y[i] = 0.f;
  }
  return make_uint4(Half<F16>::pack(y[0], y[1]), Half<F16>::pack(y[2], y[3]), Half<F16>::pack(y[4], y[5]),
                    Half<F16>::pack(y[6], y[7]));
}
// Codes of eight outputs n.. of row m.
template <bool INSIDE>
__device__ __forceinline__ void store_codes8(const Fp8Params& p, int m, int n, const uint2& codes) {
  if (!INSIDE && (m >= p.M || n >= p.N)) return;
  uint8_t* const dst = p.out8 + m * p.ldo8 + n;
  if (INSIDE || n + 8 <= p.N) {
    __builtin_memcpy(dst, &codes, 8);
  } else {
    uint8_t b[8];
    __builtin_memcpy(b, &codes, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < p.N) dst[i] = b[i];
  }
}

// 256 x 256 outputs a workgroup, four waves of 128 x 128, 128 channels a step, in
// the order of the 16-bit products' large tiles: each operand's slice of a step
// is two halves of 128 rows, a step is four phases of one quadrant each, eight
// products of K = 64:
//   (A0, B0) (A1, B0) (A1, B1) (A0, B1)
// A phase reads one half into registers for the next (A1, B1, then the next
// step's B0 and A0: the registers just left), and loads a half read in the pair
// of phases before, two steps on; one barrier a pair says both that the halves to
// be read have landed and that those to be loaded were read by all.
//
// Row l of the 32 of tile 2 h + i of a wave (half h) is its row 4 l + 2 h + i of
// 128, of x as of w: so the scales of a lane's four rows are four neighbouring
// bytes, one load a step and operand, of which the matrix instruction picks its
// tile's, and a lane ends with 16 consecutive outputs, tile by tile.
//
// 75,600 rows by 5,120 x 13,824 with bias, gate and residual 4.1 ms (2.6 PFLOP/s,
// matrix cores busy 71% of the cycles at 1.63 GHz, no LDS bank conflicts): bound
// by power, as the 16-bit products are; 128 x 128 tiles took 6.5. By 13,824 x 5,120
// with bias 4.05, with GELU's tanh form 4.26 and its erf form 4.66 (an epilogue
// runs alone, since a workgroup fills a CU), with the first and the result
// quantised 4.29; a pass of its own for that took 1.1 more.
template <bool F16, int ACT>
__global__ void __launch_bounds__(256, 1) fp8_big_kernel(Fp8Params p) {
  __shared__ __attribute__((aligned(16))) uint8_t a00[128 * 128], a01[128 * 128], a10[128 * 128], a11[128 * 128];
  __shared__ __attribute__((aligned(16))) uint8_t b00[128 * 128], b01[128 * 128], b10[128 * 128], b11[128 * 128];
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
  // Rows past the matrix lie past the buffers' records and come as zeros. The
  // whole offset is the lane's: the check against the records subtracts a scalar
  // part from them, which could be more than they are.
  auto slice = [&](const uint8_t* base, int64_t ld, int at, int rows) {
    const int64_t records = (min(rows - at, 256) - 1) * ld + p.K - from;
    return make_rsrc(base + at * ld + from, static_cast<uint32_t>(records));
  };
  const auto wrs = slice(p.w, p.ldw, n0, p.N), xrs = slice(p.x, p.ldx, m0, p.M);
  // This lane's chunk of step 0 in load j of half h is row r8 * 4 + 2 h + (j & 1)
  // of wave row j >> 1: the lane's own part of its byte offset is r8 * 4 rows.
  const int r8 = w * 8 + (lane >> 3), c8 = (lane & 7) ^ (r8 >> 1 & 7);
  uint32_t wv = static_cast<uint32_t>(r8 * 4) * static_cast<uint32_t>(p.ldw) + c8 * 16;
  uint32_t xv = static_cast<uint32_t>(r8 * 4) * static_cast<uint32_t>(p.ldx) + c8 * 16;
  const int ldw = static_cast<int>(p.ldw), ldx = static_cast<int>(p.ldx);
  const int steps = (K + 255) >> 8 << 1;  // an even number: the last may be all zeros
  // The last steps' chunks past K (tail) come as zeros, without a memory access.
  auto load = [&](auto tail, __amdgpu_buffer_rsrc_t rs, uint32_t v, int ld, int t, int h, uint8_t* buf) {
    if (tail.value && c8 * 16 >= K - t * 128) v = kOutside;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      load_lds16(rs, buf + (j * 4 + w) * 1024, v + (t * 128 + ((j >> 1) * 128 + 2 * h + (j & 1)) * ld), 0);
  };
  auto load_w = [&](auto tail, int t, int h, uint8_t* buf) { load(tail, wrs, wv, ldw, t, h, buf); };
  auto load_x = [&](auto tail, int t, int h, uint8_t* buf) { load(tail, xrs, xv, ldx, t, h, buf); };
  const int wn = w & 1, wm = w >> 1;
  // Scales of this lane's rows, four a load (rows past the matrix: the last four).
  const uint32_t wsv = min(n0 + wn * 128 + l32 * 4, (p.N - 1) & ~3), xsv = min(m0 + wm * 128 + l32 * 4, (p.M - 1) & ~3);
  auto load_scales = [&](int t, uint32_t& sw, uint32_t& sx) {
    const int b = min((from >> 7) + t, p.kb - 1);
    sw = *reinterpret_cast<const uint32_t*>(p.ws + b * p.ldws + wsv);
    sx = *reinterpret_cast<const uint32_t*>(p.xs + b * p.ldxs + xsv);
  };
  const int arow = (wn * 64 + l32) * 128, brow = (wm * 64 + l32) * 128, f = l32 >> 1 & 7;
  f32x16 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x16{};
  typedef i32x8 Frag[4];  // [64 channels][tile]
  auto read = [&](const uint8_t* row, Frag& v) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = (4 * u + hl) ^ f;
        v[2 * u + i] = join(chunk_at(row + i * 4096 + c * 16), chunk_at(row + i * 4096 + (c ^ 2) * 16));
      }
  };
  // One quadrant: halves HA of w and HB of x.
  auto quadrant = [&](auto ha, auto hb, const Frag& a, const Frag& b, uint32_t sw, uint32_t sx) {
    constexpr int HA = decltype(ha)::value, HB = decltype(hb)::value;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 &c00 = acc[2 * HA][2 * HB], &c10 = acc[2 * HA + 1][2 * HB];
      f32x16 &c01 = acc[2 * HA][2 * HB + 1], &c11 = acc[2 * HA + 1][2 * HB + 1];
      const i32x8 &a0 = a[2 * u], &a1 = a[2 * u + 1], &b0 = b[2 * u], &b1 = b[2 * u + 1];
      const int s = static_cast<int>(sw), x = static_cast<int>(sx);
      c00 = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a0, b0, c00, 0, 0, 2 * HA, s, 2 * HB, x);
      c10 = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a1, b0, c10, 0, 0, 2 * HA + 1, s, 2 * HB, x);
      c01 = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a0, b1, c01, 0, 0, 2 * HA, s, 2 * HB + 1, x);
      c11 = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a1, b1, c11, 0, 0, 2 * HA + 1, s, 2 * HB + 1, x);
    }
    constexpr int kMfma = 0x008, kDsRead = 0x100, kVmem = 0x020;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kVmem, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto landed = [&] {  // the halves loaded three pairs of phases ago; two pairs' loads, and scales, are behind them
    wait_vmcnt<16>();
    block_barrier();
  };
  Frag fa0, fa1, fb0, fb1;
  uint32_t sw0, sx0, sw1, sx1;
  // One step with its A0 in c0, the other A registers c1; ends with the next
  // step's A0 in c1. *c: this step's buffers, *n: the next step's.
  constexpr std::true_type may_end{};
  constexpr std::false_type whole{};
  constexpr std::integral_constant<int, 0> h0{};
  constexpr std::integral_constant<int, 1> h1{};
  auto step = [&](auto tail, int t, Frag& c0, Frag& c1, uint32_t& sw, uint32_t& sx, uint8_t* a0c, uint8_t* a1c,
                  uint8_t* b0c, uint8_t* b1c, uint8_t* a0n, uint8_t* b0n) {
    landed();
    read(a1c + arow, c1);
    load_x(tail, t + 2, 0, b0c);
    quadrant(h0, h0, c0, fb0, sw, sx);
    read(b1c + brow, fb1);
    load_w(tail, t + 2, 0, a0c);
    quadrant(h1, h0, c1, fb0, sw, sx);
    landed();
    read(b0n + brow, fb0);
    load_w(tail, t + 2, 1, a1c);
    quadrant(h1, h1, c1, fb1, sw, sx);
    read(a0n + arow, c1);
    load_x(tail, t + 2, 1, b1c);
    quadrant(h0, h1, c0, fb1, sw, sx);
    load_scales(t + 2, sw, sx);
  };
  load_scales(0, sw0, sx0);
  load_scales(1, sw1, sx1);
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
  read(b00 + brow, fb0);
  read(a00 + arow, fa0);
  int t = 0;
  for (; (t + 4) * 128 <= K; t += 2) {  // nothing past K is loaded
    step(whole, t, fa0, fa1, sw0, sx0, a00, a10, b00, b10, a01, b01);
    step(whole, t + 1, fa1, fa0, sw1, sx1, a01, a11, b01, b11, a00, b00);
  }
#pragma unroll 1
  for (; t < steps; t += 2) {
    step(may_end, t, fa0, fa1, sw0, sx0, a00, a10, b00, b10, a01, b01);
    step(may_end, t + 1, fa1, fa0, sw1, sx1, a01, a11, b01, b11, a00, b00);
  }
  wait_vmcnt_0();  // the trailing loads have landed before the workgroup's LDS is released
  // The sums stay in the accumulation registers to here: otherwise the compiler
  // moves some of them between the files in every step.
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) asm volatile("" : "+a"(acc[i][j]));
  // The sums go through LDS, 32 rows x 64 outputs at a time, in the wave's own
  // part of it: whole rows of 128 bytes leave (and come, for the residual). Row r
  // of tile j is 4 r + j of the wave's 128.
  float* const st = stage + w * 2048;
  const bool inside = m0 + 256 <= p.M && n0 + 256 <= p.N;
  float* const part = p.part + static_cast<int64_t>(split * cut + id - p.whole) * 65536;  // of a tile in parts
  const int nw = n0 + wn * 128 + (lane & 7) * 8, mw = m0 + wm * 128 + (lane >> 3) * 4;
  float bias[2][8], gate[2][8];
#pragma unroll
  for (int gp = 0; gp < 2; ++gp) load_columns8(p, nw + gp * 64, bias[gp], gate[gp]);
  auto to_stage = [&](auto tile, auto half) {  // outputs gp * 64 .. + 63 of tile j's rows
    constexpr int j = decltype(tile)::value, gp = decltype(half)::value;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // outputs g * 32 + hl * 16 + 4 e .. + 3 of row l32
        constexpr int kFirst = gp * 8;
        const int r = kFirst + g * 4 + e;
        *reinterpret_cast<float4*>(st + l32 * 64 + ((g * 8 + hl * 4 + e) ^ (l32 & 15)) * 4) =
            make_float4(acc[0][j][r], acc[1][j][r], acc[2][j][r], acc[3][j][r]);
      }
  };
  auto from_stage = [&](int i, float* z) {  // outputs (lane & 7) * 8 .. + 7 of row i * 8 + (lane >> 3)
    const int r = i * 8 + (lane >> 3), c = (lane & 7) * 2;
    const float4 lo = *reinterpret_cast<const float4*>(st + r * 64 + (c ^ (r & 15)) * 4);
    const float4 hi = *reinterpret_cast<const float4*>(st + r * 64 + ((c + 1) ^ (r & 15)) * 4);
    z[0] = lo.x; z[1] = lo.y; z[2] = lo.z; z[3] = lo.w;
    z[4] = hi.x; z[5] = hi.y; z[6] = hi.z; z[7] = hi.w;
  };
  constexpr std::integral_constant<int, 2> h2{};
  constexpr std::integral_constant<int, 3> h3{};
  auto each_tile = [&](auto&& f) {
    f(h0);
    f(h1);
    f(h2);
    f(h3);
  };
  auto each_half = [&](auto&& f) {
    f(h0);
    f(h1);
  };
  if (in_parts) {
    each_tile([&](auto j) {
      each_half([&](auto gp) {
        to_stage(j, gp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float z[8];
          from_stage(i, z);
          float* const at = part + (mw + i * 32 + decltype(j)::value - m0) * 256 + nw + decltype(gp)::value * 64 - n0;
          *reinterpret_cast<float4*>(at) = make_float4(z[0], z[1], z[2], z[3]);
          *reinterpret_cast<float4*>(at + 4) = make_float4(z[4], z[5], z[6], z[7]);
        }
      });
    });
  } else if (p.out8) {  // a scale's 128 outputs are the wave's: eight lanes, twice
    auto quantized = [&](auto in) {
      constexpr bool INSIDE = decltype(in)::value;
      each_tile([&](auto j) {
        uint4 y[4][2];
        each_half([&](auto gp) {
          constexpr int GP = decltype(gp)::value;
          to_stage(j, gp);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float z[8];
            from_stage(i, z);
            y[i][GP] = finished8<F16, ACT, INSIDE>(p, mw + i * 32 + decltype(j)::value, nw + GP * 64, z, bias[GP], gate[GP]);
          }
        });
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = mw + i * 32 + decltype(j)::value;
          uint2 codes[2];
          const uint32_t scale = encode<F16, 8, 2>(y[i], codes);
          store_codes8<INSIDE>(p, m, nw, codes[0]);
          store_codes8<INSIDE>(p, m, nw + 64, codes[1]);
          if ((lane & 7) == 0 && (INSIDE || (m < p.M && nw < p.N)))
            p.out8_scales[(nw >> 7) * p.ldos + m] = static_cast<uint8_t>(scale);
        }
      });
    };
    if (inside)
      quantized(std::true_type{});
    else
      quantized(std::false_type{});
  } else {
    each_tile([&](auto j) {
      each_half([&](auto gp) {
        constexpr int GP = decltype(gp)::value;
        to_stage(j, gp);
        if (inside) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float z[8];
            from_stage(i, z);
            finish8_wide<F16, ACT>(p, mw + i * 32 + decltype(j)::value, nw + GP * 64, z, bias[GP], gate[GP]);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            float z[8];
            from_stage(i, z);
            finish8_edge<F16, ACT>(p, mw + i * 32 + decltype(j)::value, nw + GP * 64, z, bias[GP], gate[GP]);
          }
        }
      });
    });
  }
}

// Joins the parts of the tiles behind the last full round, in their order, and
// finishes: 32 workgroups a tile, eight outputs a thread.
template <bool F16>
__global__ void __launch_bounds__(256) fp8_join_big_kernel(Fp8Params p) {
  const int mt = (p.M + 255) / 256, nt = (p.N + 255) / 256, cut = mt * nt - p.whole;
  const int tile = blockIdx.x >> 5, row = (blockIdx.x & 31) * 8 + (threadIdx.x >> 5), col = (threadIdx.x & 31) * 8;
  int tm, tn;
  tile_of(p.whole + tile, mt, nt, tm, tn);
  const int m = tm * 256 + row, n = tn * 256 + col;
  float z[8] = {};
  for (int i = 0; i < p.splits; ++i) {
    const float* const src = p.part + static_cast<int64_t>(i * cut + tile) * 65536 + row * 256 + col;
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    z[0] += a.x; z[1] += a.y; z[2] += a.z; z[3] += a.w;
    z[4] += b.x; z[5] += b.y; z[6] += b.z; z[7] += b.w;
  }
  float bias[8], gate[8];
  load_columns8(p, n, bias, gate);
  with_fp8_activation(p.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (!p.out8) return finish8<F16, ACT>(p, m, n, z, bias, gate);
    const uint4 y[1] = {finished8<F16, ACT, false>(p, m, n, z, bias, gate)};  // a scale's outputs are sixteen lanes'
    uint2 codes[1];
    const uint32_t scale = encode<F16, 16, 1>(y, codes);
    store_codes8<false>(p, m, n, codes[0]);
    if ((threadIdx.x & 15) == 0 && m < p.M && n < p.N) p.out8_scales[(n >> 7) * p.ldos + m] = static_cast<uint8_t>(scale);
  });
}

template <bool F16>
void run_fp8_large(const Fp8Params& p, int64_t rest, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.whole + rest * p.splits));
  with_fp8_activation(p.act, [&](auto act) { fp8_big_kernel<F16, decltype(act)::value><<<grid, 256, 0, st>>>(p); });
  if (rest > 0) fp8_join_big_kernel<F16><<<dim3(static_cast<unsigned>(rest * 32)), 256, 0, st>>>(p);
}

}  // namespace
}  // namespace dfs
