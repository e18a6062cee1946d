// The AdamW update of a flat run of elements: one pass, every value read and written once.
//
// 28 to 30 bytes an element with an fp32 gradient (three fp32 values read and written, the gradient read,
// the bf16 image written) against a few operations: bound by memory.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "emrs.h"
#include "internal.h"

namespace {

using emrs_internal::fail;

typedef __attribute__((ext_vector_type(4))) float f32x4;
constexpr int kThreads = 128;  // 131 million elements: 603 us; 64 lanes 609, 256 to 1024 646 to 654

template <class T>
struct Four {
  typedef __attribute__((ext_vector_type(4))) T type;
};

struct Factors {
  float beta1, rest1, beta2, rest2, eps, keep, rate, over2;  // rate: lr / (1 - beta1^step); over2: 1 / (1 - beta2^step)
};

__device__ inline void update(float &w, float &m, float &v, float g, const Factors &f) {
  m = f.beta1 * m + f.rest1 * g;
  v = f.beta2 * v + f.rest2 * g * g;
  w = w * f.keep - f.rate * m / (sqrtf(v * f.over2) + f.eps);
}

template <class V>
__device__ inline V stream_in(const V *p) {
  return __builtin_nontemporal_load(p);
}

// Four elements a lane where they lie on their vectors, and the last three by a lane each.  Nothing is read
// twice: the accesses bypass the caches' retention.
template <class G, bool kImage, bool kWide>
__global__ __launch_bounds__(kThreads) void adamw_kernel(uint64_t fours, uint64_t n, float *w, float *m, float *v, const G *g, __bf16 *image,
                                                         Factors f) {
  using g4 = typename Four<G>::type;
  using h4 = typename Four<__bf16>::type;
  uint64_t i = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * kThreads + threadIdx.x;
  if (kWide && i < fours) {
    f32x4 a = stream_in(reinterpret_cast<const f32x4 *>(w) + i), b = stream_in(reinterpret_cast<const f32x4 *>(m) + i);
    f32x4 c = stream_in(reinterpret_cast<const f32x4 *>(v) + i);
    const g4 d = stream_in(reinterpret_cast<const g4 *>(g) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float x = a[k], y = b[k], z = c[k];
      update(x, y, z, (float)d[k], f);
      a[k] = x, b[k] = y, c[k] = z;
    }
    __builtin_nontemporal_store(a, reinterpret_cast<f32x4 *>(w) + i);
    __builtin_nontemporal_store(b, reinterpret_cast<f32x4 *>(m) + i);
    __builtin_nontemporal_store(c, reinterpret_cast<f32x4 *>(v) + i);
    if (kImage) {
      h4 h;
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = (__bf16)a[k];
      __builtin_nontemporal_store(h, reinterpret_cast<h4 *>(image) + i);
    }
    return;
  }
  if (kWide) i += fours * 3;  // element 4 fours + (i - fours)
  if (i >= n) return;
  float x = w[i], y = m[i], z = v[i];
  update(x, y, z, (float)g[i], f);
  w[i] = x, m[i] = y, v[i] = z;
  if (kImage) image[i] = (__bf16)x;
}

bool on(const void *p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <class G, bool kImage>
int launch(const emrs_adamw *a, const Factors &f, hipStream_t st) {
  const G *g = static_cast<const G *>(a->grad);
  __bf16 *image = static_cast<__bf16 *>(a->image);
  const bool wide = on(a->main, 16) && on(a->exp_avg, 16) && on(a->exp_avg_sq, 16) && on(g, 4 * sizeof(G)) && on(image, 8);
  const uint64_t fours = wide ? a->n / 4 : 0, lanes = fours + (a->n - fours * 4);
  // A row of the grid holds less than 2^32 lanes; rows of equal length, so that the last one is not empty for the most part.
  constexpr uint64_t most = 0xffffffffull / kThreads;
  const uint64_t all = (lanes + kThreads - 1) / kThreads, rows = (all + most - 1) / most;
  const dim3 blocks((uint32_t)((all + rows - 1) / rows), (uint32_t)rows);
  if (wide)
    adamw_kernel<G, kImage, true><<<blocks, kThreads, 0, st>>>(fours, a->n, a->main, a->exp_avg, a->exp_avg_sq, g, image, f);
  else
    adamw_kernel<G, kImage, false><<<blocks, kThreads, 0, st>>>(0, a->n, a->main, a->exp_avg, a->exp_avg_sq, g, image, f);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? EMRS_OK : fail(EMRS_ERR_HIP, std::string("adamw: ") + hipGetErrorString(e));
}

template <class G>
int launch(const emrs_adamw *a, const Factors &f, hipStream_t st) {
  return a->image ? launch<G, true>(a, f, st) : launch<G, false>(a, f, st);
}

}  // namespace

extern "C" int emrs_adamw_step(const emrs_adamw *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    if (!a) return fail(EMRS_ERR_INVALID_ARGUMENT, "adamw: NULL argument");
    if (a->grad_dtype > EMRS_FP16) return fail(EMRS_ERR_INVALID_ARGUMENT, "adamw: gradients are fp32, bf16 or fp16");
    if (a->step == 0) return fail(EMRS_ERR_INVALID_ARGUMENT, "adamw: steps count from 1");
    if (!(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1))
      return fail(EMRS_ERR_INVALID_ARGUMENT, "adamw: betas lie in [0, 1)");
    if (a->n == 0) return EMRS_OK;
    if (a->n > (1ull << 38)) return fail(EMRS_ERR_TOO_LARGE, "adamw: at most 2^38 elements");
    if (!a->main || !a->exp_avg || !a->exp_avg_sq || !a->grad) return fail(EMRS_ERR_INVALID_ARGUMENT, "adamw: NULL buffer");
    const uint64_t grad_bytes = a->grad_dtype == EMRS_FP32 ? 4 : 2;
    if (!on(a->main, 4) || !on(a->exp_avg, 4) || !on(a->exp_avg_sq, 4) || !on(a->grad, grad_bytes) || !on(a->image, 2))
      return fail(EMRS_ERR_MISALIGNED, "adamw: a buffer off its type's alignment");
    const int rc = emrs_internal::need_device();
    if (rc) return rc;
    const double c1 = 1.0 - std::pow(a->beta1, (double)a->step), c2 = 1.0 - std::pow(a->beta2, (double)a->step);
    const Factors f{(float)a->beta1, (float)(1.0 - a->beta1), (float)a->beta2, (float)(1.0 - a->beta2), (float)a->eps,
                    (float)(1.0 - a->lr * a->weight_decay), (float)(a->lr / c1), (float)(1.0 / c2)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    return a->grad_dtype == EMRS_FP32   ? launch<float>(a, f, st)
           : a->grad_dtype == EMRS_BF16 ? launch<__bf16>(a, f, st)
                                        : launch<_Float16>(a, f, st);
  });
}
