// Softmax attention with a sliding window and sinks (the first tokens, which
// stay visible). A sequence of nq queries and nk keys: query i stands at
// position p = nk - nq + i and sees key j where
//   0 <= j < nk,  j <= p + right,  (j >= p - left or j < sinks),
// out_i = sum_j softmax_j(scale q_i k_j) v_j over the keys it sees (0 where it
// sees none), lse_i the log of the softmax's denominator (-inf there).
// Key j lies in slot j of the sequence's rows, or, in a rolling cache of S
// slots, in slot j < sinks ? j : sinks + (j - sinks) mod (S - sinks).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "lds_copy.h"

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
  // How the call is cut (plan).
  int group;   // query heads of a key head
  int few;     // window_few_kernel
  int stream;  // its keys and values are beyond the last-level cache
  int blocks;  // of 128 rows of a (sequence, key head)
  int chunks, whole, split, parts;
  int short_last;  // the heads' last blocks, of few rows, come behind all others
  // Of the parts: O [row][D], (m, l) [row][2] and, where lse is wanted, the sum
  // for it [row].
  float *part_o, *part_ml, *part_e;
};

__device__ __forceinline__ int slot_of(const WindowParams& p, int pos) {
  if (pos < p.sinks) return pos;
  return p.sinks + static_cast<int>(static_cast<uint32_t>(pos - p.sinks) % static_cast<uint32_t>(p.S - p.sinks));
}

template <bool F16>
struct Half;
template <>
struct Half<false> {
  typedef bf16x8 vec;
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // acc + x.lo + x.hi in fp32.
  static __device__ __forceinline__ float sum2(pair x, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(x, (pair){(__bf16)1.0f, (__bf16)1.0f}, acc, false);
  }
};
template <>
struct Half<true> {
  typedef f16x8 vec;
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum2(pair x, float acc) {
    return __builtin_amdgcn_fdot2(x, (pair){(_Float16)1.0f, (_Float16)1.0f}, acc, false);
  }
};
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Two values rounded to the storage type, the first in the low half.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, typename Half<F16>::pair));
}

// This lane's value with the other lane half's (lane ^ 32).
__device__ __forceinline__ float xhalf_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xhalf_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Queries and keys of sequence b.
struct Seq {
  int nq;
  int64_t nk;
};
__device__ __forceinline__ Seq seq_of(const WindowParams& p, int b) {
  Seq s;
  s.nq = p.q_lens ? min(max(p.q_lens[b], 0), p.Lq) : p.Lq;
  s.nk = p.kv_lens ? max(p.kv_lens[b], 0) : p.S;
  s.nk = min(s.nk, static_cast<int64_t>(p.rolling ? 0x7fffff00 : p.S));  // tile ends stay within 32 bits
  return s;
}
// Last key and first key behind the sinks that query i sees.
__device__ __forceinline__ int last_key(const WindowParams& p, const Seq& s, int i) {
  return static_cast<int>(max(min(s.nk - s.nq + i + p.right, s.nk - 1), int64_t(-1)));
}
__device__ __forceinline__ int first_key(const WindowParams& p, const Seq& s, int i) {
  return static_cast<int>(max(s.nk - s.nq + i - p.left, int64_t(0)));
}

// The key tiles of T keys that queries q0..q1 see: `sink` tiles from 0 on,
// then those from `low` on, `n` in all.
struct Tiles {
  int sink, low, n;
  __device__ __forceinline__ int at(int i) const { return i < sink ? i : low + i - sink; }
};
template <int T>
__device__ __forceinline__ Tiles tiles_of(const WindowParams& p, const Seq& s, int q0, int q1) {
  Tiles t{0, 0, 0};
  if (q1 < q0) return t;
  const int hi = last_key(p, s, q1) + 1, lo = first_key(p, s, q0);
  t.low = lo / T;
  t.sink = min((min(p.sinks, hi) + T - 1) / T, t.low);
  t.n = t.sink + max((hi + T - 1) / T - t.low, 0);
  return t;
}

// Copies of a key tile into LDS by NW waves, rows of D channels straight from
// the sequence's slab: load j of wave w fills 1 KB. Rows past the sequence come
// as zeros.
template <int D, int T, int NW>
struct KeyTile {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, LOADS = T * D * 2 / (NW * 1024);
  bool value;
  int row0;      // this lane's row in load 0
  uint32_t col;  // byte of its chunk within that row
  __device__ __forceinline__ KeyTile(int w, int lane, bool value_) : value(value_) {
    row0 = w * RPI + lane / CPR;
    const int c = lane % CPR;
    col = (value ? c ^ swz_v(row0) : c ^ swz_k(row0)) * 16;
  }
  // ... and in load j, whose rows lie j * NW * RPI further.
  __device__ __forceinline__ uint32_t col_of(int j) const {
    return col ^ (value ? swz_v(j * NW * RPI) : swz_k(j * NW * RPI)) * 16;
  }
  // Chunk c of row r lies at c ^ swz(r): 16 keys read one chunk each, or 4 keys
  // four chunks each (the transposing reads of V), without a bank conflict.
  static __device__ __forceinline__ int swz_k(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ int swz_v(int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }

  template <bool ROLL, bool STREAM = false>
  __device__ __forceinline__ void issue(const WindowParams& p, const uint16_t* slab, int64_t stride, int64_t nk,
                                        int tile, uint16_t* lds, int w) const {
    const int first = tile * T;
    const uint32_t bytes = static_cast<uint32_t>(stride * 2);
    if (!ROLL) {
      const int rows = static_cast<int>(max(min(nk - first, static_cast<int64_t>(T)), int64_t(0)));
      const auto rs = make_rsrc(slab + first * stride, rows ? (rows - 1) * bytes + D * 2 : 0);
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        load_lds16<STREAM>(rs, lds + (j * NW + w) * 512, (row0 + j * NW * RPI) * bytes + col_of(j), 0);
      return;
    }
    const auto rs = make_rsrc(slab, (p.S - 1) * bytes + D * 2);
    const int s0 = slot_of(p, first);
    uint32_t off[LOADS];
    if (first + T <= nk && s0 + T <= p.S) {  // one stretch of slots
#pragma unroll
      for (int j = 0; j < LOADS; ++j) off[j] = (s0 + row0 + j * NW * RPI) * bytes + col_of(j);
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int r = row0 + j * NW * RPI;
        const int slot = s0 + r < p.S ? s0 + r : slot_of(p, s0 + r);
        off[j] = first + r < nk ? slot * bytes + col_of(j) : 0xfffffff0u;
      }
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_lds16<STREAM>(rs, lds + (j * NW + w) * 512, off[j], 0);
  }
};

// S^T of T keys (LDS rows) and the wave's 32 queries, 32 keys a product; the
// products of different keys alternate, so that none waits for the one before.
template <int D, bool F16, int T>
__device__ __forceinline__ void scores(const uint16_t* keys, const typename Half<F16>::vec* q, int l32, int hl,
                                       f32x16* s) {
  typedef KeyTile<D, T, 1> KT;
#pragma unroll
  for (int k = 0; k < T / 32; ++k) s[k] = f32x16{};
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int k = 0; k < T / 32; ++k) {
      const uint4 a =
          *reinterpret_cast<const uint4*>(keys + (k * 32 + l32) * D + ((2 * i + hl) ^ KT::swz_k(l32)) * 8);
      s[k] = Half<F16>::mfma(__builtin_bit_cast(typename Half<F16>::vec, a), q[i], s[k]);
    }
}

// V^T operand of 16 keys (LDS rows k0..) and channels dc * 32..: two
// transposing reads, which give a lane 4 keys of one channel each, in the order
// in which its scores hold them (k0 + hl * 4 + 0..3, then 8 further).
template <int D, bool F16, int T>
__device__ __forceinline__ typename Half<F16>::vec values16(const uint16_t* vals, int k0, int dc, int lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int i = lane & 15, key = (lane >> 5) * 4 + (i >> 2);
  const int chunk = dc * 4 + ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
  const uint16_t* at = vals + (k0 + key) * D + (chunk ^ KeyTile<D, T, 1>::swz_v(key)) * 8 + (i & 1) * 4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * D));
  const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(typename Half<F16>::vec, v);
}

// The V^T operands of 32 keys at once: the reads of values16 and their wait in
// one block. The builtin's reads would have the compiler wait for every load
// into LDS, the next tile's among them.
template <int D, bool F16>
__device__ __forceinline__ void values32(const uint16_t* vals, int lane, typename Half<F16>::vec (&v)[2][D / 32]) {
  typedef __attribute__((address_space(3))) const uint16_t lds_u16;
  const int i = lane & 15, key = (lane >> 5) * 4 + (i >> 2), low = ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
  const int sw = KeyTile<D, 32, 1>::swz_v(key);
  uint64_t r[D / 32][4];  // keys 0, 8, 16, 24 on
#pragma unroll
  for (int dc = 0; dc < D / 32; dc += 2) {
    const uint32_t a = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((lds_u16*)(vals + key * D + ((dc * 4 + low) ^ sw) * 8 + (i & 1) * 4)));
    const uint32_t b = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((lds_u16*)(vals + key * D + (((dc + 1) * 4 + low) ^ sw) * 8 + (i & 1) * 4)));
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
        "ds_read_b64_tr_b16 %2, %8 offset:%11\n\t"
        "ds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %9\n\t"
        "ds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
        "ds_read_b64_tr_b16 %6, %9 offset:%11\n\t"
        "ds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[dc][0]), "=&v"(r[dc][1]), "=&v"(r[dc][2]), "=&v"(r[dc][3]), "=&v"(r[dc + 1][0]),
          "=&v"(r[dc + 1][1]), "=&v"(r[dc + 1][2]), "=&v"(r[dc + 1][3])
        : "v"(a), "v"(b), "n"(16 * D), "n"(32 * D), "n"(48 * D)
        : "memory");
  }
#pragma unroll
  for (int kg = 0; kg < 2; ++kg)
#pragma unroll
    for (int dc = 0; dc < D / 32; ++dc) {
      const uint64_t lo = r[dc][2 * kg], hi = r[dc][2 * kg + 1];
      v[kg][dc] = __builtin_bit_cast(typename Half<F16>::vec,
                                     make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32),
                                                static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32)));
    }
}

// Order of an MFMA phase of N products with R LDS reads each: the reads run
// four products ahead.
template <int N, int R>
__device__ __forceinline__ void pin_read_ahead() {
  constexpr int kMfma = 0x008, kDsRead = 0x100, kAhead = 4;
  __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead * R, 0);
#pragma unroll
  for (int i = 0; i < N - kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kDsRead, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, kAhead, 0);
}

// A row's reference m, in log2 units: P = 2^(s c - m). It follows the running
// maximum of the scores s[0..N) times c, less kBelow, and O and l follow it,
// when some row's maximum has grown by more than 2^kSlack beyond it, so that most
// tiles leave O alone. bf16 has fp32's exponents: P stays below 2^8, which costs
// neither its relative precision nor the sums' range. f16 holds 11 bits only down
// to 2^-14 and nothing below 2^-25: the row's largest P stands at 2^13 to 2^15
// (65,504 is the largest), so that weights down to 2^-27 of it keep their 11 bits
// and only those below 2^-38 are lost. (At 1, keys 17 nats below a sink counted
// 1.44 times and those 17.4 below not at all.) f16 video 16.0 ms, 15.9 at 1.
template <bool F16>
struct Reference {
  static constexpr float kBelow = F16 ? 13.f : 0.f, kSlack = F16 ? 2.f : 8.f;
};
template <int N, int DCH, bool F16, bool LSE>
__device__ __forceinline__ float follow_max(const f32x16* s, float c, float& m, float& l, float& e, f32x16* o) {
  float mx = -INFINITY;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[k][r]);
  mx = xhalf_max(mx) * c - Reference<F16>::kBelow;
  if (__any(mx > m + Reference<F16>::kSlack)) {
    const float mn = fmaxf(m, mx);
    const float alpha = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
    l *= alpha;
    if (LSE) e *= alpha;
#pragma unroll
    for (int i = 0; i < DCH; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
    m = mn;
  }
  return m == -INFINITY ? 0.f : m;  // rows without a key so far: P = 2^(-inf)
}

// P = 2^(s c - m) of 32 keys as two PV operands; their rounded values are added
// to l, which divides O, and, where the log-sum-exp is wanted, the values as they
// are to e: there is no rounding above that l's could cancel there (two keys in
// tiles apart: 3e-3 with l in bf16). It costs instances that have no lse nothing
// and the others 4% (video 15.05 and 15.7 ms, 32 single tokens 201 and 209 us).
template <bool F16, bool LSE>
__device__ __forceinline__ void weights32(const f32x16& s, float c, float m, typename Half<F16>::vec* pf, float& l,
                                          float& e) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (LSE) {
        const float x = exp2_fast(fmaf(s[h * 8 + 2 * j], c, -m)), y = exp2_fast(fmaf(s[h * 8 + 2 * j + 1], c, -m));
        w[j] = pack2<F16>(x, y);
        e += x + y;
      } else {
        w[j] = pack2<F16>(exp2_fast(fmaf(s[h * 8 + 2 * j], c, -m)), exp2_fast(fmaf(s[h * 8 + 2 * j + 1], c, -m)));
      }
      l = Half<F16>::sum2(__builtin_bit_cast(typename Half<F16>::pair, w[j]), l);
    }
    pf[h] = __builtin_bit_cast(typename Half<F16>::vec, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// Keys first.. of the scores that the row does not see get -inf.
__device__ __forceinline__ void mask32(f32x16& s, int first, int hl, int klo, int khi, int sinks) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int key = first + (r >> 2) * 8 + hl * 4 + (r & 3);
    const bool hidden = (key > khi) | ((key < klo) & (key >= sinks));  // no branches
    s[r] = hidden ? -INFINITY : s[r];
  }
}

template <bool F16>
__device__ __forceinline__ float lse_of(float m, float e) {
  constexpr float kBelow = Reference<F16>::kBelow, kUnit = F16 ? 0x1p-13f : 1.f;  // 2^-kBelow
  return e == 0.f ? -INFINITY : ((m + kBelow) + log2f(e * kUnit)) * 0.69314718055994531f;
}

// O^T / l of a lane's row: the halves of a lane pair are joined into 8
// consecutive channels, 16-byte stores.
template <int D, bool F16>
__device__ __forceinline__ void store_row(uint16_t* out, const f32x16* o, float inv, bool live, int hl) {
#pragma unroll
  for (int dc = 0; dc < D / 32; ++dc)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = pack2<F16>(o[dc][g * 8 + 2 * i] * inv, o[dc][g * 8 + 2 * i + 1] * inv);
        b[i] = pack2<F16>(o[dc][g * 8 + 4 + 2 * i] * inv, o[dc][g * 8 + 5 + 2 * i] * inv);
      }
      const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
      if (live) *reinterpret_cast<uint4*>(out + dc * 32 + g * 16 + hl * 8) = make_uint4(x[0], y[0], x[1], y[1]);
    }
}

// A part's O, (m, l) and e of a lane's row as they are, to row `at` of the parts.
template <int D, bool LSE>
__device__ __forceinline__ void store_part(const WindowParams& p, int64_t at, const f32x16* o, float m, float l,
                                           float e, int hl) {
  float* const po = p.part_o + at * D;
#pragma unroll
  for (int dc = 0; dc < D / 32; ++dc)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(po + dc * 32 + g * 8 + hl * 4) =
          make_float4(o[dc][g * 4], o[dc][g * 4 + 1], o[dc][g * 4 + 2], o[dc][g * 4 + 3]);
  if (hl == 0) {
    *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
    if (LSE) p.part_e[at] = e;
  }
}

// Rows of a (sequence, key head): query i of query head g of the group is row
// i * group + g, so that a block's rows share their keys and stand at few
// positions.
struct Row {
  int i, g;
};
__device__ __forceinline__ Row row_of(const WindowParams& p, int r) {
  Row x;
  x.i = r / p.group;
  x.g = r - x.i * p.group;
  return x;
}

// Work item of a workgroup: block `blk` of (sequence, key head) `bh`, part
// `piece` of `pieces`, whose result goes to `slot`.
struct Item {
  int bh, blk, piece, pieces, slot;
};

// Block i of XCD x: its (sequence, key head) and its number there.
__device__ __forceinline__ void block_of(const WindowParams& p, int x, int i, int& bh, int& blk) {
  if (p.short_last) {  // chunks == 1: an XCD has whole heads
    const int full = p.blocks - 1, all = p.B * p.Hkv / 8 * full;
    const int h = i < all ? i / full : i - all;
    bh = h * 8 + x;
    blk = i < all ? full - 1 - (i - h * full) : full;
    return;
  }
  const int per = (p.blocks + p.chunks - 1) / p.chunks;  // blocks of a range
  const int u = i / per * 8 + x;
  bh = u / p.chunks;
  blk = p.blocks - 1 - (u % p.chunks * per + i % per);
}

// Hardware deals workgroup i to XCD i % 8. The blocks of a (sequence, key
// head) are cut into p.chunks ranges and range u of them all belongs to XCD
// u % 8, so neighbouring blocks, which share keys, run on one XCD's L2 and
// sequences of different lengths spread evenly. Of an XCD's list the first
// p.whole blocks are one workgroup each, the rest p.parts, joined by
// window_join_kernel. Late blocks, which see most keys where left has no limit,
// are started first; where left has a limit, a head's last block with rows for
// at most two of its waves comes behind all others and fills places that the
// last round leaves (40 heads, 1,560 rows by 9,360 keys 291 us, in its place 300;
// 3,600 by 14,400 938 and 962; without a limit 8 heads x 12,040 458 and 386).
__device__ __forceinline__ bool item_of(const WindowParams& p, Item& it) {
  const int x = blockIdx.x & 7, j = blockIdx.x >> 3;
  int i = j;
  it.piece = 0;
  it.pieces = 1;
  it.slot = 0;
  if (j >= p.whole && p.parts > 1) {
    const int t = (j - p.whole) / p.parts;
    it.piece = j - p.whole - t * p.parts;
    it.pieces = p.parts;
    it.slot = (t * 8 + x) * p.parts + it.piece;
    i = p.whole + t;
  }
  block_of(p, x, i, it.bh, it.blk);
  return it.bh < p.B * p.Hkv && it.blk >= 0;
}

// 128 rows a workgroup, four waves of 32, tiles of 128 keys; the framework's
// block-sparse schedule: two workgroups a CU, one K and one V buffer each, the
// next K copied under the softmax and P V, the next V under Q K^T. S^T = K Q^T
// leaves a lane with one query, whose P is the second operand of
// O^T += V^T P^T as it lies in the registers; V^T comes from the rows of V by
// transposing LDS reads, so nothing is laid out beforehand. Tiles are aligned;
// a wave masks those that cross its rows' window and passes over those that none
// of its rows sees.
//
// P is rounded to the operands' 8 or 11 bits (the products take no more), and
// the row sum adds the rounded values, so that the rounding cancels where one
// weight dominates; f16's range is at Reference. Statistics and O are fp32.
//
// 75,600 tokens x 40 heads, 10,800 keys a row: 15.0 ms, 1.07 PFLOP/s; matrix
// cores busy 58% of the cycles at 1.8 GHz, the vector units 43%, which overlap
// little between the two workgroups. Tried and slower: two groups of four waves
// half a turn apart over shared tiles (17.5 ms), three workgroups a CU with
// tiles of 64 keys (27 ms, spills), a reference from a row's first tile without
// later maxima (15.8 ms), raised wave priority in either phase (no change).
template <int D, bool F16, bool ROLL, bool LSE>
__global__ void __launch_bounds__(256, 2) window_tile_kernel(WindowParams p) {
  constexpr int DCH = D / 32, T = 128;
  typedef KeyTile<D, T, 4> KT;
  typedef typename Half<F16>::vec vec;
  __shared__ __attribute__((aligned(16))) uint16_t k_lds[T * D];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[T * D];
  Item it;
  if (!item_of(p, it)) return;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int b = it.bh / p.Hkv, g = it.bh - b * p.Hkv;
  const Seq seq = seq_of(p, b);
  const int rows = p.Lq * p.group, r0 = it.blk * 128;
  const Tiles tiles = tiles_of<T>(p, seq, r0 / p.group, min(min(r0 + 127, rows - 1) / p.group, seq.nq - 1));
  const int t0 = static_cast<int64_t>(tiles.n) * it.piece / it.pieces;
  const int t1 = static_cast<int64_t>(tiles.n) * (it.piece + 1) / it.pieces;
  // This wave's rows, and its lane's.
  const int wr = r0 + w * 32;
  const int wq0 = min(wr, rows - 1) / p.group, wq1 = min(min(wr + 31, rows - 1) / p.group, seq.nq - 1);
  const int wlo0 = first_key(p, seq, wq0), wlo1 = first_key(p, seq, wq1);
  // (a wave behind the last row sees nothing and only copies)
  const int whi0 = last_key(p, seq, wq0), whi1 = wq1 < wq0 || wr >= rows ? -1 : last_key(p, seq, wq1);
  const bool in = wr + l32 < rows;
  const Row row = row_of(p, min(wr + l32, rows - 1));
  const int klo = first_key(p, seq, row.i), khi = last_key(p, seq, row.i);
  const int head = g * p.group + row.g;
  f32x16 o[DCH];
#pragma unroll
  for (int i = 0; i < DCH; ++i) o[i] = f32x16{};
  float m = -INFINITY, l = 0.f, e = 0.f;
  if (t0 < t1) {
    const uint16_t* const ks = p.k + b * p.k_sb + g * p.k_sh;
    const uint16_t* const vs = p.v + b * p.v_sb + g * p.v_sh;
    const KT kc(w, lane, false), vc(w, lane, true);
    int tile = tiles.at(t0);
    kc.template issue<ROLL>(p, ks, p.k_sl, seq.nk, tile, k_lds, w);
    vc.template issue<ROLL>(p, vs, p.v_sl, seq.nk, tile, v_lds, w);
    vec qf[D / 16];
    {
      const uint16_t* q = p.q + b * p.q_sb + head * p.q_sh + row.i * p.q_sl;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        qf[i] = __builtin_bit_cast(vec, *reinterpret_cast<const uint4*>(q + (2 * i + hl) * 8));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) asm volatile("" ::"v"(qf[i]));  // arrived: no wait for them in the loop
    }
    for (int t = t0; t < t1; ++t) {
      // The last tile's copies are repeated, unread, so that every turn waits
      // for the same number of loads.
      const int next = t + 1 < t1 ? tiles.at(t + 1) : tile;
      const int first = tile * T;
      const bool seen = first <= whi1 && (first + T > wlo0 || first < p.sinks);
      f32x16 s[4];
      vec pf[8];
      wait_vmcnt<KT::LOADS>();  // this wave's part of K has landed
      block_barrier();          // ... and everybody else's
      if (seen) {
        scores<D, F16, T>(k_lds, qf, l32, hl, s);
        pin_read_ahead<4 * (D / 16), 1>();
      }
      block_barrier();  // K has been read by all
      kc.template issue<ROLL>(p, ks, p.k_sl, seq.nk, next, k_lds, w);
      if (seen) {
        if (first + T - 1 > whi0 || (first < wlo1 && first + T > p.sinks)) {
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) mask32(s[kb], first + kb * 32, hl, klo, khi, p.sinks);
        }
        const float ref = follow_max<4, DCH, F16, LSE>(s, p.scale_log2, m, l, e, o);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) weights32<F16, LSE>(s[kb], p.scale_log2, ref, pf + 2 * kb, l, e);
      }
      wait_vmcnt<KT::LOADS>();  // V has landed
      block_barrier();
      if (seen) {
#pragma unroll
        for (int kg = 0; kg < 8; ++kg)
#pragma unroll
          for (int dc = 0; dc < DCH; ++dc)
            o[dc] = Half<F16>::mfma(values16<D, F16, T>(v_lds, kg * 16, dc, lane), pf[kg], o[dc]);
        pin_read_ahead<8 * DCH, 2>();
      }
      block_barrier();  // V has been read by all
      vc.template issue<ROLL>(p, vs, p.v_sl, seq.nk, next, v_lds, w);
      tile = next;
    }
    wait_vmcnt_0();  // the trailing copies have landed before the workgroup's LDS is released
  }
  l = xhalf_sum(l);
  if (LSE) e = xhalf_sum(e);
  const bool dead = row.i >= seq.nq;
  if (it.pieces > 1) {
    const int64_t at = static_cast<int64_t>(it.slot) * 128 + w * 32 + l32;
    if (in) store_part<D, LSE>(p, at, o, dead ? -INFINITY : m, dead ? 0.f : l, e, hl);
    return;
  }
  const float inv = dead || l == 0.f ? 0.f : 1.f / l;
  if (dead) {
#pragma unroll
    for (int i = 0; i < DCH; ++i) o[i] = f32x16{};
  }
  store_row<D, F16>(p.out + b * p.o_sb + head * p.o_sh + row.i * p.o_sl, o, inv, in, hl);
  // (asked of p.lse although LSE says it: the compiler orders the copies before
  // the loop otherwise, video 15.25 ms for 15.05)
  if (p.lse && in && hl == 0)
    p.lse[(static_cast<int64_t>(b) * p.Hq + head) * p.Lq + row.i] = dead ? -INFINITY : lse_of<F16>(m, e);
}

// At most 32 rows (a token, or a few, of a group's heads) over many keys: a
// wave a workgroup, tiles of 32 keys through two LDS buffers of its own that
// the loads fill directly; no barrier, five waves a CU keep 80 KB in flight.
// The keys are dealt over p.parts waves; reading them is all that counts, past
// the last-level cache with streaming loads (32 sequences x 8 heads x 8,256
// keys: 210 us, 229 with ordinary ones).
template <int D, bool F16, bool ROLL, bool STREAM, bool LSE>
__global__ void __launch_bounds__(64, 2) window_few_kernel(WindowParams p) {
  constexpr int DCH = D / 32, T = 32;
  typedef KeyTile<D, T, 1> KT;
  typedef typename Half<F16>::vec vec;
  __shared__ __attribute__((aligned(16))) uint16_t k0[T * D], v0[T * D], k1[T * D], v1[T * D];
  const int bh = blockIdx.x / p.parts, piece = blockIdx.x - bh * p.parts;
  const int lane = threadIdx.x, l32 = lane & 31, hl = lane >> 5;
  const int b = bh / p.Hkv, g = bh - b * p.Hkv;
  const Seq seq = seq_of(p, b);
  const int rows = p.Lq * p.group;
  const Tiles tiles = tiles_of<T>(p, seq, 0, seq.nq - 1);
  const int t0 = static_cast<int64_t>(tiles.n) * piece / p.parts;
  const int t1 = static_cast<int64_t>(tiles.n) * (piece + 1) / p.parts;
  const bool in = l32 < rows;
  const Row row = row_of(p, min(l32, rows - 1));
  const int klo = first_key(p, seq, row.i), khi = last_key(p, seq, row.i);
  const int head = g * p.group + row.g;
  f32x16 o[DCH];
#pragma unroll
  for (int i = 0; i < DCH; ++i) o[i] = f32x16{};
  float m = -INFINITY, l = 0.f, e = 0.f;
  if (t0 < t1) {
    const uint16_t* const ks = p.k + b * p.k_sb + g * p.k_sh;
    const uint16_t* const vs = p.v + b * p.v_sb + g * p.v_sh;
    const KT kc(0, lane, false), vc(0, lane, true);
    auto load = [&](int t, uint16_t* kb, uint16_t* vb) {
      const int tile = tiles.at(min(t, t1 - 1));  // past the last one: that again, unread
      kc.template issue<ROLL, STREAM>(p, ks, p.k_sl, seq.nk, tile, kb, 0);
      vc.template issue<ROLL, STREAM>(p, vs, p.v_sl, seq.nk, tile, vb, 0);
    };
    vec qf[D / 16];
    const uint16_t* q = p.q + b * p.q_sb + head * p.q_sh + row.i * p.q_sl;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      qf[i] = __builtin_bit_cast(vec, *reinterpret_cast<const uint4*>(q + (2 * i + hl) * 8));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" ::"v"(qf[i]));
    load(t0, k0, v0);
    load(t0 + 1, k1, v1);
    auto step = [&](int t, uint16_t* kb, uint16_t* vb) {
      wait_vmcnt<2 * KT::LOADS>();  // this tile has landed, the next may be in flight
      const int first = tiles.at(t) * T;
      f32x16 s;
      scores<D, F16, T>(kb, qf, l32, hl, &s);
      mask32(s, first, hl, klo, khi, p.sinks);
      const float ref = follow_max<1, DCH, F16, LSE>(&s, p.scale_log2, m, l, e, o);
      vec pf[2];
      weights32<F16, LSE>(s, p.scale_log2, ref, pf, l, e);
      vec vf[2][DCH];
      values32<D, F16>(vb, lane, vf);
#pragma unroll
      for (int kg = 0; kg < 2; ++kg)
#pragma unroll
        for (int dc = 0; dc < DCH; ++dc) o[dc] = Half<F16>::mfma(vf[kg][dc], pf[kg], o[dc]);
      wait_lgkm_0();  // the buffers have been read
      load(t + 2, kb, vb);
    };
    for (int t = t0; t < t1; t += 2) {
      step(t, k0, v0);
      if (t + 1 >= t1) break;
      step(t + 1, k1, v1);
    }
    wait_vmcnt_0();
  }
  l = xhalf_sum(l);
  if (LSE) e = xhalf_sum(e);
  const bool dead = row.i >= seq.nq;
  if (p.parts > 1) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * rows + l32;
    if (in) store_part<D, LSE>(p, at, o, dead ? -INFINITY : m, dead ? 0.f : l, e, hl);
    return;
  }
  const float inv = dead || l == 0.f ? 0.f : 1.f / l;
  if (dead) {
#pragma unroll
    for (int i = 0; i < DCH; ++i) o[i] = f32x16{};
  }
  store_row<D, F16>(p.out + b * p.o_sb + head * p.o_sh + row.i * p.o_sl, o, inv, in, hl);
  if (LSE && in && hl == 0)
    p.lse[(static_cast<int64_t>(b) * p.Hq + head) * p.Lq + row.i] = dead ? -INFINITY : lse_of<F16>(m, e);
}

// Joins the parts of a row: O = sum 2^(m_i - M) O_i over the same sum of l_i.
// A part without keys (l = 0) has no weight; NaN reaches its row. WAVES: one
// wave a row, or four where the parts are many (a row by 32,768 keys in 256
// parts: 4 us, 32 with one). Groups of D / 4 lanes share the parts and are added
// up in a fixed order.
template <int D, bool F16, bool FEW, int WAVES>
__global__ void __launch_bounds__(256) window_join_kernel(WindowParams p) {
  constexpr int LANES = D / 4, GROUPS = 64 * WAVES / LANES;
  __shared__ float4 so[4][LANES];
  __shared__ float sl[4], se[4], sm[4];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane % LANES;
  const int grp = (WAVES == 4 ? static_cast<int>(threadIdx.x) : lane) / LANES;
  const int64_t id = WAVES == 4 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + w;
  const int rows = p.Lq * p.group;
  int bh, r;
  int64_t first, step;  // row of the first part, rows between parts
  if (FEW) {
    bh = static_cast<int>(id / rows);
    r = static_cast<int>(id - static_cast<int64_t>(bh) * rows);
    first = static_cast<int64_t>(bh) * p.parts * rows + r;
    step = rows;
  } else {
    const int block = static_cast<int>(id >> 7), x = block & 7, i = p.whole + (block >> 3);
    int blk;
    block_of(p, x, i, bh, blk);
    r = blk * 128 + static_cast<int>(id & 127);
    if (bh >= p.B * p.Hkv || blk < 0 || r >= rows) return;
    first = static_cast<int64_t>(block) * p.parts * 128 + (id & 127);
    step = 128;
  }
  float M = -INFINITY;
  for (int i = WAVES == 4 ? threadIdx.x : lane; i < p.parts; i += 64 * WAVES) M = fmaxf(M, p.part_ml[(first + i * step) * 2]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  if (WAVES == 4) {
    if (lane == 0) sm[w] = M;
    __syncthreads();
    M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  }
  const float ref = M == -INFINITY ? 0.f : M;
  float l = 0.f, e = 0.f, o[4] = {};
#pragma unroll 8
  for (int i = grp; i < p.parts; i += GROUPS) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (first + i * step) * 2);
    float4 v = *reinterpret_cast<const float4*>(p.part_o + (first + i * step) * D + sub * 4);
    const bool none = ml.y == 0.f;  // rows behind a sequence may hold anything
    const float a = none ? 0.f : exp2_fast(ml.x - ref);
    if (none) v = make_float4(0.f, 0.f, 0.f, 0.f);
    l += a * ml.y;
    if (p.lse && !none) e += a * p.part_e[first + i * step];
    o[0] += a * v.x; o[1] += a * v.y; o[2] += a * v.z; o[3] += a * v.w;
  }
#pragma unroll
  for (int off = LANES; off < 64; off *= 2) {
    l += __shfl_xor(l, off, 64);
    e += __shfl_xor(e, off, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], off, 64);
  }
  if (WAVES == 4) {
    if (lane < LANES) so[w][sub] = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) sl[w] = l, se[w] = e;
    __syncthreads();
    if (threadIdx.x >= LANES) return;
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    e = (se[0] + se[1]) + (se[2] + se[3]);
    const float4 a = so[0][sub], b = so[1][sub], c = so[2][sub], d = so[3][sub];
    o[0] = (a.x + b.x) + (c.x + d.x);
    o[1] = (a.y + b.y) + (c.y + d.y);
    o[2] = (a.z + b.z) + (c.z + d.z);
    o[3] = (a.w + b.w) + (c.w + d.w);
  } else if (lane >= LANES) {
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int b = bh / p.Hkv, g = bh - b * p.Hkv;
  const Row row = row_of(p, r);
  const int head = g * p.group + row.g;
  *reinterpret_cast<uint2*>(p.out + b * p.o_sb + head * p.o_sh + row.i * p.o_sl + sub * 4) =
      make_uint2(pack2<F16>(o[0] * inv, o[1] * inv), pack2<F16>(o[2] * inv, o[3] * inv));
  if (p.lse && sub == 0) p.lse[(static_cast<int64_t>(b) * p.Hq + head) * p.Lq + row.i] = lse_of<F16>(M, e);
}

// How a call is cut. Slots for two workgroups on each of 256 CUs; the blocks
// left over behind full rounds of an XCD's 64 slots are cut into parts so that
// the last round fills the chip too, each part at least two tiles.
void plan(const dfs_window_args* a, WindowParams& p) {
  constexpr int kSlots = 64;  // of an XCD
  p.group = static_cast<int>(a->q_heads / a->kv_heads);
  const int64_t rows = a->q_rows * p.group, heads = a->batch * a->kv_heads;
  auto limit = [](int64_t n) { return n < 0 || n > kNoLimit ? int64_t(kNoLimit) : n; };
  const int64_t keys_all = a->rolling ? a->sinks + limit(a->left) + a->q_rows : a->slots;  // some query may see
  p.few = rows <= 32;
  if (p.few) {
    const int64_t keys = std::min(keys_all, std::min(limit(a->sinks), a->slots) + limit(a->left) + a->q_rows + limit(a->right));
    // Five waves of 32 KB a CU; at least four tiles a wave.
    p.parts = static_cast<int>(std::max(int64_t(1), std::min(1280 / heads, (keys + 127) / 128)));
    p.split = 0;
    p.stream = heads * keys * a->head_dim * 4 > kLastLevelCache;
    return;
  }
  p.blocks = static_cast<int>((rows + 127) / 128);
  int64_t g = heads, e = 8;
  while (e) { const int64_t t = g % e; g = e; e = t; }
  p.chunks = static_cast<int>(8 / g);
  const int64_t per = (p.blocks + p.chunks - 1) / p.chunks;  // blocks of a range
  const int64_t list = (heads * p.chunks + 7) / 8 * per;     // of an XCD
  const int64_t near = limit(a->left) + limit(a->right) + 128 / p.group + 128;
  const int64_t tiles = std::min((keys_all + 127) / 128,
                                 (near + 127) / 128 + (std::min(limit(a->sinks), a->slots) + 127) / 128);
  p.whole = static_cast<int>(list);
  p.parts = 1;
  p.split = 0;
  const int64_t rest = list % kSlots;
  p.short_last = a->left >= 0 && p.chunks == 1 && p.blocks > 1 && rows % 128 > 0 && rows % 128 <= 64 && list < 16 * kSlots;
  if (rest == 0 || list >= 16 * kSlots || tiles < 4) return;
  // Time of the last round in whole blocks: rounds / parts, and a part's own
  // start and store, worth about a tile.
  double best = 1.0;
  for (int64_t n = 2; n <= std::min<int64_t>(tiles / 2, 32); ++n) {
    const double cost = static_cast<double>((rest * n + kSlots - 1) / kSlots) *
                        (1.0 / static_cast<double>(n) + 1.0 / static_cast<double>(tiles));
    if (cost < best * 0.95) {
      best = cost;
      p.parts = static_cast<int>(n);
    }
  }
  if (p.parts > 1) {
    p.whole = static_cast<int>(list - rest);
    p.split = static_cast<int>(rest);
  }
}

int64_t part_rows(const dfs_window_args* a, const WindowParams& p) {
  if (p.parts <= 1) return 0;
  return p.few ? a->batch * a->kv_heads * p.parts * a->q_rows * p.group : int64_t(8) * p.split * p.parts * 128;
}

template <int D, bool F16, bool ROLL, bool LSE>
void launch(const WindowParams& p, hipStream_t st) {
  const unsigned heads = static_cast<unsigned>(p.B * p.Hkv);
  if (p.few) {
    if (p.stream)
      window_few_kernel<D, F16, ROLL, true, LSE><<<heads * p.parts, 64, 0, st>>>(p);
    else
      window_few_kernel<D, F16, ROLL, false, LSE><<<heads * p.parts, 64, 0, st>>>(p);
    const int64_t rows = static_cast<int64_t>(heads) * p.Lq * p.group;
    if (p.parts > 1) window_join_kernel<D, F16, true, 4><<<static_cast<unsigned>(rows), 256, 0, st>>>(p);
    return;
  }
  window_tile_kernel<D, F16, ROLL, LSE><<<8u * (p.whole + p.split * p.parts), 256, 0, st>>>(p);
  const unsigned cut = static_cast<unsigned>(p.split) * 8 * 128;  // rows of the blocks that were
  if (p.parts > 8)
    window_join_kernel<D, F16, false, 4><<<cut, 256, 0, st>>>(p);
  else if (p.parts > 1)
    window_join_kernel<D, F16, false, 1><<<cut / 4, 256, 0, st>>>(p);
}

}  // namespace
}  // namespace dfs

extern "C" int64_t dfs_window_attention_workspace_size(const dfs_window_args* a) {
  using namespace dfs;
  if (!a || a->batch <= 0 || a->kv_heads <= 0 || a->q_heads < a->kv_heads || a->q_rows <= 0 || a->slots <= 0) {
    set_error("window_attention: batch, heads, q_rows and slots must be positive");
    return -1;
  }
  WindowParams p{};
  plan(a, p);
  return part_rows(a, p) * (a->head_dim + 3) * 4;
}

extern "C" int dfs_window_attention_form(const dfs_window_args* a) {
  using namespace dfs;
  if (!a || a->batch <= 0 || a->kv_heads <= 0 || a->q_heads < a->kv_heads || a->q_rows <= 0 || a->slots <= 0) {
    set_error("window_attention: batch, heads, q_rows and slots must be positive");
    return -1;
  }
  WindowParams p{};
  plan(a, p);
  return (p.few ? DFS_WINDOW_FEW : DFS_WINDOW_BLOCKS) | (p.parts > 1 ? DFS_FORM_PARTS : 0) |
         (p.stream ? DFS_FORM_STREAM : 0) | (p.short_last ? DFS_WINDOW_SHORT_LAST : 0);
}

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
  // (a scale of 0 in fp32 would make a hidden key's minus infinity NaN)
  DFS_REQUIRE(a->scale >= 1e-30 && a->scale < 1e30, "%s: scale must lie from 1e-30 to 1e30", name);
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
  constexpr int64_t kTileBytes = int64_t(1) << 31;
  DFS_REQUIRE(a->k_row_stride * 256 < kTileBytes && a->v_row_stride * 256 < kTileBytes,
              "%s: row strides of k and v are too large", name);
  DFS_REQUIRE(!a->rolling || (a->k_row_stride * a->slots * 2 < 2 * kTileBytes - 65536 &&
                              a->v_row_stride * a->slots * 2 < 2 * kTileBytes - 65536),
              "%s: a rolling cache's rows of one head must lie within 4 GB", name);
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
  plan(a, p);
  const int64_t spare = part_rows(a, p), need = spare * (a->head_dim + 3) * 4;
  DFS_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need &&
                            reinterpret_cast<uintptr_t>(a->workspace) % 16 == 0),
              "%s: a 16-byte aligned workspace of %lld bytes is needed", name, (long long)need);
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = p.part_o + spare * a->head_dim;
  p.part_e = p.part_ml + spare * 2;
  // A launch holds fewer than 2^32 threads.
  DFS_REQUIRE((p.whole + static_cast<int64_t>(p.split) * p.parts) * 8 < (1 << 24) &&
                  a->batch * a->kv_heads * p.parts < (1 << 26) && a->q_rows * p.group < kNoLimit,
              "%s: too many rows", name);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = a->dtype == DFS_DTYPE_F16, roll = p.rolling;
  auto run = [&](auto wide, auto half, auto ring) {
    constexpr int D = decltype(wide)::value ? 128 : 64;
    if (p.lse)
      launch<D, decltype(half)::value, decltype(ring)::value, true>(p, st);
    else
      launch<D, decltype(half)::value, decltype(ring)::value, false>(p, st);
  };
  auto with = [](bool b, auto&& f) { b ? f(std::true_type{}) : f(std::false_type{}); };
  with(a->head_dim == 128, [&](auto wide) {
    with(f16, [&](auto half) { with(roll, [&](auto ring) { run(wide, half, ring); }); });
  });
  return check_launch(name);
}
