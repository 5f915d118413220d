// The f16 results of linear_fp8_large.h.
#include "linear_fp8_large.h"

namespace dfs {
void run_fp8_large_f16(const Fp8Params& p, int64_t rest, hipStream_t stream) { run_fp8_large<true>(p, rest, stream); }
}  // namespace dfs
