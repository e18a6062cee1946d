// The norm kernels on fp16 operands.
#include "norm.h"

namespace emrs_internal {

void norm_fp16(const emrs_norm_kernels::Norm &p, bool wide_stream, bool backward, bool full, bool is_wide, uint32_t blocks, hipStream_t st) {
  if (wide_stream)
    emrs_norm_kernels::launch<_Float16, float>(p, backward, full, is_wide, blocks, st);
  else
    emrs_norm_kernels::launch<_Float16, _Float16>(p, backward, full, is_wide, blocks, st);
}

}  // namespace emrs_internal
