// Library-internal helpers shared by the translation units of libemrs.
#ifndef EMRS_INTERNAL_H
#define EMRS_INTERNAL_H

#include <string>

#include "emrs.h"

namespace emrs_internal {
// Record `msg` as this thread's last error (read by emrs_last_error) and return `code`.
int fail(int code, const std::string &msg);
void clear_error();
// EMRS_OK, or EMRS_ERR_NO_DEVICE where no HIP device is visible.
int need_device();
// f(), or EMRS_ERR_TOO_LARGE where memory for a message ran out: nothing is thrown through a C entry point.
template <class F>
int guarded(F &&f) noexcept {
  try {
    return f();
  } catch (...) {
    return EMRS_ERR_TOO_LARGE;
  }
}
}  // namespace emrs_internal

#endif
