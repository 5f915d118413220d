// Rows of 16-bit values to 8-bit codes with a scale for every 128 channels (the
// definition is in fp8_block.h).
#include <algorithm>

#include "fp8_block.h"
#include "lds_copy.h"

namespace dfs {
namespace {

struct QuantizeParams {
  const uint16_t* x;
  uint8_t *values, *scales;
  int64_t ldx, ldv, lds;
  int rows, k, fill, blocks;  // blocks: of a row
};

// Sixteen lanes a block, eight channels each, so that a wave reads a KB in one
// piece; x's rows may lie anywhere. Bound by memory: 75,600 x 5,120 197 us, 5.9
// TB/s of two bytes read and one written. The largest magnitude is taken on the
// values' bits as integers and pairs are converted with their scale by one
// instruction; in fp32, value by value, it was 204.
template <bool F16>
__device__ __forceinline__ void quantize_group(const QuantizeParams& p) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (id >= static_cast<int64_t>(p.rows) * p.blocks) return;  // whole groups of sixteen lanes
  const int row = static_cast<int>(id / p.blocks), block = static_cast<int>(id - static_cast<int64_t>(row) * p.blocks);
  const int l16 = threadIdx.x & 15, c = block * kScaleBlock + l16 * 8;
  const uint16_t* const src = p.x + row * p.ldx;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (c + 8 <= p.k) {
    __builtin_memcpy(&v, src + c, 16);
  } else if (c < p.k) {
    uint16_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = src[min(c + i, p.k - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = c + i < p.k ? t[i] : 0;
    __builtin_memcpy(&v, t, 16);
  }
  const uint4 values[1] = {v};
  uint2 code[1];
  const uint32_t scale = encode<F16, 16, 1>(values, code);
  const uint2 codes = code[0];
  uint8_t* const dst = p.values + row * p.ldv + c;
  if (c + 8 <= p.fill) {
    __builtin_memcpy(dst, &codes, 8);
  } else {
    uint8_t b[8];
    __builtin_memcpy(b, &codes, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < p.fill) dst[i] = b[i];
  }
  if (l16 == 0) p.scales[block * p.lds + row] = static_cast<uint8_t>(scale);
}

template <bool F16>
__global__ void __launch_bounds__(256) quantize_kernel(QuantizeParams p) {
  quantize_group<F16>(p);
}
// With codes to be laid out by the workgroups behind those of the values: a
// launch less where a product needs both (333 rows by 1,017 x 709 in f16 16.4 us with
// two, 13.2 with one).
template <bool F16>
__global__ void __launch_bounds__(256) quantize_pad_kernel(QuantizeParams p, int groups, PadCodes codes) {
  const int group = static_cast<int>(blockIdx.x);
  if (group < groups)
    quantize_group<F16>(p);
  else
    pad_codes(codes, group - groups, static_cast<int>(gridDim.x) - groups);
}

}  // namespace

void launch_quantize(const uint16_t* x, int64_t rows, int64_t k, int64_t ldx, bool f16, uint8_t* values, int64_t ldv,
                     int64_t fill, uint8_t* scales, int64_t lds, hipStream_t stream, const PadCodes* also) {
  QuantizeParams p{x, values, scales, ldx, ldv, lds, static_cast<int>(rows), static_cast<int>(k),
                   static_cast<int>(fill), static_cast<int>((k + kScaleBlock - 1) / kScaleBlock)};
  const int groups = static_cast<int>((rows * p.blocks + 15) / 16);
  if (also) {
    const int more = static_cast<int>(pad_groups(*also));
    const dim3 grid(static_cast<unsigned>(groups) + static_cast<unsigned>(more));
    f16 ? quantize_pad_kernel<true><<<grid, 256, 0, stream>>>(p, groups, *also)
        : quantize_pad_kernel<false><<<grid, 256, 0, stream>>>(p, groups, *also);
    return;
  }
  const dim3 grid(static_cast<unsigned>(groups));
  if (f16)
    quantize_kernel<true><<<grid, 256, 0, stream>>>(p);
  else
    quantize_kernel<false><<<grid, 256, 0, stream>>>(p);
}

}  // namespace dfs

extern "C" int dfs_quantize_fp8(const dfs_quantize_fp8_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "quantize_fp8";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  DFS_REQUIRE(a->x && a->values && a->scales, "%s: NULL operand", name);
  const int64_t blocks = (a->k + kScaleBlock - 1) / kScaleBlock;
  DFS_REQUIRE(a->rows > 0 && a->k > 0 && a->rows < (int64_t(1) << 30) && a->k < (int64_t(1) << 21),
              "%s: rows=%lld k=%lld must be positive, below 2^30 and 2^21", name, (long long)a->rows, (long long)a->k);
  // A launch holds fewer than 2^32 threads: 2^24 - 1 workgroups, of sixteen blocks each.
  DFS_REQUIRE(a->rows * blocks <= (int64_t(1) << 28) - 16, "%s: too many blocks", name);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(reinterpret_cast<uintptr_t>(a->x) % 2 == 0, "%s: x must be aligned to its elements", name);
  DFS_REQUIRE(a->x_stride >= 0 && a->values_stride >= a->k && a->scales_stride >= a->rows,
              "%s: x's stride must not be negative, the results' rows must not overlap", name);
  launch_quantize(static_cast<const uint16_t*>(a->x), a->rows, a->k, a->x_stride, a->dtype == DFS_DTYPE_F16,
                  static_cast<uint8_t*>(a->values), a->values_stride, a->k, static_cast<uint8_t*>(a->scales),
                  a->scales_stride, reinterpret_cast<hipStream_t>(stream));
  return check_launch(name);
}
