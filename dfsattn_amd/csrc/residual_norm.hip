// The C entry of residual_norm.h and its bf16 kernels.
#include "residual_norm.h"

#include <cfloat>
#include <cmath>

namespace dfs {
void run_residual_norm_bf16(const NormParams& p, hipStream_t stream) { run<false>(p, stream); }
}  // namespace dfs

extern "C" int dfs_residual_norm(const dfs_residual_norm_args* a, dfs_stream_t stream) {
  using namespace dfs;
  const char* name = "residual_norm";
  DFS_REQUIRE(a != nullptr, "%s: args is NULL", name);
  const int64_t rows = a->rows, C = a->channels;
  DFS_REQUIRE(a->x && (a->y == nullptr) == (a->out == nullptr) && (a->h != nullptr) != (a->h8 != nullptr) &&
                  (a->h8 == nullptr) == (a->h8_scales == nullptr),
              "%s: x and h, or h8 with its scales, must be non-NULL, and y and out go together", name);
  // A launch holds fewer than 2^32 threads: 2^24 - 1 workgroups, of four rows each.
  DFS_REQUIRE(rows > 0 && rows <= (int64_t(1) << 26) - 4 && C > 0 && C <= 512 * kMaxChunks,
              "%s: rows=%lld channels=%lld must be positive, up to 2^26 - 4 and up to %d", name, (long long)rows,
              (long long)C, 512 * kMaxChunks);
  DFS_REQUIRE(C % 8 == 0 || rows < (int64_t(1) << 24), "%s: too many rows of %lld channels", name, (long long)C);
  DFS_REQUIRE(a->dtype == DFS_DTYPE_BF16 || a->dtype == DFS_DTYPE_F16, "%s: dtype must be bf16 or f16", name);
  DFS_REQUIRE(a->norm == DFS_NORM_RMS || a->norm == DFS_NORM_LAYER, "%s: norm code %lld is not supported", name,
              (long long)a->norm);
  DFS_REQUIRE(a->post_norm >= DFS_NORM_NONE && a->post_norm <= DFS_NORM_LAYER, "%s: norm code %lld is not supported",
              name, (long long)a->post_norm);
  DFS_REQUIRE(a->y || (!a->gate && a->post_norm == DFS_NORM_NONE), "%s: a gate or norm of y without it", name);
  DFS_REQUIRE(a->post_norm != DFS_NORM_NONE || (!a->post_weight && !a->post_bias), "%s: a weight without its norm", name);
  DFS_REQUIRE(a->eps >= 0. && a->post_eps >= 0., "%s: eps must not be negative", name);
  DFS_REQUIRE(a->eps <= FLT_MAX && a->post_eps <= FLT_MAX && (!a->y || std::fabs(a->residual_scale) <= FLT_MAX),
              "%s: eps and the residual's scale must be in fp32's range", name);
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
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  a->dtype == DFS_DTYPE_F16 ? run_residual_norm_f16(p, st) : run_residual_norm_bf16(p, st);
  return check_launch(name);
}
