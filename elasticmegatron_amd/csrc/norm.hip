// The calls of the norms around a block: checks, shapes, launches.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "emrs.h"
#include "internal.h"
#include "norm.h"

namespace {

using emrs_internal::fail;
using emrs_norm_kernels::kMaxHidden;
using emrs_norm_kernels::Norm;
using emrs_norm_kernels::parts_of;

bool on(const void *p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether every row that is read or written lies on 16 bytes (rows of 32 bits: on 32).
bool wide(const emrs_norm *a) {
  for (const void *p : {a->residual, a->branch, a->gate, a->branch_weight, a->weight, (const void *)a->stream, (const void *)a->normed, a->grad_stream,
                        a->grad_normed, (const void *)a->grad_residual, (const void *)a->grad_branch, (const void *)a->grad_gate})
    if (!on(p, 32) && !(on(p, 16) && a->residual_dtype != EMRS_FP32)) return false;
  return a->hidden % 8 == 0 && a->residual_stride % 8 == 0 && a->branch_stride % 8 == 0 && a->gate_stride % 8 == 0 && a->stream_stride % 8 == 0;
}

// Of the shape that has more parts.
uint64_t workspace_of(const emrs_norm *a) { return (uint64_t)std::max(parts_of(a, true), parts_of(a, false)) * 3 * a->hidden * 4; }

int check_sizes(const emrs_norm *a) {
  if (!a) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL argument");
  if (a->dtype != EMRS_BF16 && a->dtype != EMRS_FP16) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: operands are bf16 or fp16");
  if (a->residual_dtype != a->dtype && a->residual_dtype != EMRS_FP32)
    return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: the residual stream is of the operands' type or fp32");
  if (a->hidden < 1 || a->hidden > kMaxHidden) return fail(EMRS_ERR_TOO_LARGE, "norm: hidden sizes are 1 to 16384");
  if (a->tokens > 0x7fffffffull) return fail(EMRS_ERR_TOO_LARGE, "norm: at most 2^31 - 1 tokens");
  return EMRS_OK;
}

int run(const emrs_norm *a, bool backward, hipStream_t st) {
  int rc = check_sizes(a);
  if (rc) return rc;
  if (a->gate_kind > EMRS_NORM_GATE_TOKEN) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: unknown kind of gate");
  if (a->reserved) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: reserved is not 0");
  const uint64_t h = a->hidden;
  const bool full = a->gate_kind || a->branch_weight;
  if (!a->branch && (full || a->grad_gate || a->grad_branch_weight))
    return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a gate or a branch's norm without a branch");
  if (a->gate_kind && !a->gate) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL gate");
  if (a->grad_gate && !a->gate_kind) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a gradient of no gate");
  if (a->grad_branch_weight && !a->branch_weight) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a gradient of no branch weight");
  if ((a->branch && a->branch_stride < h) || (a->gate_kind == EMRS_NORM_GATE_TOKEN && a->gate_stride < h))
    return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: rows overlap");
  if (!backward) {
    if (!a->stream && !a->normed) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: nothing is wanted");
    if (a->normed && !a->weight) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL weight");
    if (!a->residual && a->tokens) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL residual");
    if (a->residual_stride < h) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: rows overlap");
  } else {
    if (!a->grad_stream && !a->grad_normed) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: no gradient is given");
    if (a->grad_normed && (!a->weight || !a->stream || !a->stream_rms || a->stream_stride < h))
      return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: the norm's gradient wants its weight, the stream and its rms");
    if (a->branch_weight && !a->branch_rms) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL branch_rms");
    if (a->grad_weight && !a->grad_normed) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a weight's gradient without grad_normed");
  }
  for (const void *p : {a->branch, a->gate, a->branch_weight, a->weight, (const void *)a->normed, a->grad_normed, (const void *)a->grad_branch,
                        (const void *)a->grad_gate, (const void *)a->grad_weight, (const void *)a->grad_branch_weight})
    if (!on(p, 2)) return fail(EMRS_ERR_MISALIGNED, "norm: a buffer off its type's alignment");
  for (const void *p : {a->residual, (const void *)a->stream, a->grad_stream, (const void *)a->grad_residual})
    if (!on(p, a->residual_dtype == EMRS_FP32 ? 4 : 2)) return fail(EMRS_ERR_MISALIGNED, "norm: a buffer off its type's alignment");
  if (!on(a->stream_rms, 4) || !on(a->branch_rms, 4)) return fail(EMRS_ERR_MISALIGNED, "norm: a buffer off its type's alignment");
  const bool sums = backward && (a->grad_weight || a->grad_branch_weight || (a->gate_kind == EMRS_NORM_GATE_CHANNEL && a->grad_gate));
  if (sums && a->tokens) {
    if (!a->workspace || a->workspace_bytes < workspace_of(a)) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: the workspace is too small");
    if (!on(a->workspace, 256)) return fail(EMRS_ERR_MISALIGNED, "norm: the workspace is off 256 bytes");
  }
  if (a->tokens == 0) {
    if (!sums) return EMRS_OK;
    return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: sums over no tokens");
  }
  rc = emrs_internal::need_device();
  if (rc) return rc;
  Norm p{a->tokens, (int)h, (int)a->gate_kind, a->residual, a->branch, a->gate, (int64_t)a->residual_stride, (int64_t)a->branch_stride,
         (int64_t)a->gate_stride, (int64_t)a->stream_stride, a->branch_weight, a->weight, a->residual_scale, a->eps, 1.f / (float)h, a->stream, a->normed,
         a->stream_rms, a->branch_rms, a->grad_stream, a->grad_normed, a->grad_residual, a->grad_branch, a->grad_gate,
         sums ? static_cast<float *>(a->workspace) : nullptr};
  const bool w = wide(a);
  const uint32_t blocks = parts_of(a, w);
  (a->dtype == EMRS_BF16 ? emrs_internal::norm_bf16 : emrs_internal::norm_fp16)(p, a->residual_dtype == EMRS_FP32, backward, full, w, blocks, st);
  if (sums) {
    void *const gate = a->gate_kind == EMRS_NORM_GATE_CHANNEL ? a->grad_gate : nullptr;
    if (a->dtype == EMRS_BF16)
      emrs_norm_kernels::launch_sums<__bf16>(p, full, blocks, a->grad_weight, a->grad_branch_weight, gate, st);
    else
      emrs_norm_kernels::launch_sums<_Float16>(p, full, blocks, a->grad_weight, a->grad_branch_weight, gate, st);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? EMRS_OK : fail(EMRS_ERR_HIP, std::string("norm: ") + hipGetErrorString(e));
}

}  // namespace

extern "C" int emrs_norm_workspace(const emrs_norm *a, uint64_t *bytes) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    if (!bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL argument");
    const int rc = check_sizes(a);
    if (rc) return rc;
    *bytes = workspace_of(a);
    return EMRS_OK;
  });
}

extern "C" int emrs_norm_forward(const emrs_norm *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    return run(a, false, static_cast<hipStream_t>(stream));
  });
}

extern "C" int emrs_norm_backward(const emrs_norm *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    return run(a, true, static_cast<hipStream_t>(stream));
  });
}
