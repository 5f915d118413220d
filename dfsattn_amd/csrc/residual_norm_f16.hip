// The f16 kernels of residual_norm.h.
#include "residual_norm.h"

namespace dfs {
void run_residual_norm_f16(const NormParams& p, hipStream_t stream) { run<true>(p, stream); }
}  // namespace dfs
