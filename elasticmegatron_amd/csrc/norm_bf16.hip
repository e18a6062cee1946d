// The norm kernels on bf16 operands.
#include "norm.h"

namespace emrs_internal {

void norm_bf16(const emrs_norm_kernels::Norm &p, bool wide_stream, bool backward, bool full, bool is_wide, uint32_t blocks, hipStream_t st) {
  if (wide_stream)
    emrs_norm_kernels::launch<__bf16, float>(p, backward, full, is_wide, blocks, st);
  else
    emrs_norm_kernels::launch<__bf16, __bf16>(p, backward, full, is_wide, blocks, st);
}

}  // namespace emrs_internal
