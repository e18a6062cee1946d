// Newton-Schulz orthogonalisation, and the Muon update around it.
//
// X_0 = U / (|U|_F + eps) has singular values in [0, 1]; a step X <- a X + (b A + c A^2) X, A = X X^T, maps
// each of them by s -> a s + b s^3 + c s^5 and keeps the singular vectors.  With S the shorter side and L the
// longer, A is S x S, and a step costs three products:
//   A = X X^T          S S L multiply-adds by half: symmetric, tiles on and below the diagonal are computed
//   B = b A + c A A    S S S by half, b A in the epilogue
//   X = a X + B X      S S L, a X in the epilogue
// Each product wants its summed index contiguous: X [S][L] for the first, X^T [L][S] for the last, so the
// epilogue of the last writes both.  All live in the workspace, with rows and columns padded to 64 by zeros,
// which the products keep zero.
//
// Operands are fp16: X, A and B are bounded (singular values stay under 1.3 with the usual coefficients), so
// powers of two keep their entries near 1, and fp16's 11 bits then round 8 times finer than bf16's 8 at the
// same rate.  A rounding of X is noise over all directions, and directions of small singular values grow by
// a in each step that follows, noise and all: so X is held as the sum of two fp16 parts (22 bits) in every
// step but the last two, where the noise has two steps at most to grow.  There a X goes into the polynomial,
// P = a I + b A + c A^2: near the end P is close to 0.7 I where b A + c A^2 is close to -2.7 I, and has a
// quarter of its rounding; before, P's rounding on the diagonal would be such noise itself.  An error of A
// enters by the polynomial's slope, b + 2 c A, of size 0.7 at the end.  Against 64 bits five steps' result is then
// below 2e-3 off in norm for spectra from flat to s_i ~ i^-3 and 3.4e-3 for a matrix of rank one (4e-2 with one
// part throughout, 3e-1 with bf16), about the rounding of the bf16 that it is written in.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "emrs.h"
#include "gemm.h"
#include "internal.h"

namespace {

using emrs_gemm::f32x4;
using emrs_gemm::Product;
using emrs_gemm::Where;
using emrs_internal::fail;
using half = _Float16;
using half4 = emrs_gemm::Vec<_Float16>::x4;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;

constexpr float kGramScale = 64.f;  // of A and B: entries of a Gram matrix with spectrum in [0, 1.7]
constexpr int kSide = 64;
constexpr int kMaxMatrices = EMRS_MUON_MAX_MATRICES;
constexpr int kNormBlocks = 2048;  // of all matrices together

template <class P>
struct Table {
  P p[kMaxMatrices];
};

struct Update {  // where the matrix that is orthogonalised comes from
  Table<const void *> grad;
  Table<float *> momentum;
  int64_t grad_stride, momentum_stride;
  int32_t rows, cols;
  uint32_t grad_dtype;
  int32_t has_momentum, nesterov;
  float mu;
};

__device__ inline float grad_at(const void *p, uint32_t dtype, int64_t i) {
  return dtype == EMRS_FP32 ? static_cast<const float *>(p)[i]
                            : dtype == EMRS_BF16 ? (float)static_cast<const __bf16 *>(p)[i] : (float)static_cast<const half *>(p)[i];
}

__device__ inline f32x4 grad4_at(const void *p, uint32_t dtype, int64_t i) {
  if (dtype == EMRS_FP32) return *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i);
  f32x4 v;
  if (dtype == EMRS_BF16) {
    const bf16x4 g = *reinterpret_cast<const bf16x4 *>(static_cast<const __bf16 *>(p) + i);
    for (int r = 0; r < 4; ++r) v[r] = (float)g[r];
  } else {
    const half4 g = *reinterpret_cast<const half4 *>(static_cast<const half *>(p) + i);
    for (int r = 0; r < 4; ++r) v[r] = (float)g[r];
  }
  return v;
}

__device__ inline float block_sum(float v) {
  __shared__ float part[4];
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

// The first part of a value, or a value whose parts are taken at two places, held in a register: the compiler
// may otherwise round the product that it comes from to 16 bits at once in one place and by way of 32 in
// another, and the first part that is stored is not always the one that the second part completes.
template <class V>
__device__ __forceinline__ V settled(V v) {
  asm("" : "+v"(v));
  return v;
}

// momentum = mu momentum + grad, and each workgroup's share of |update|^2.  Rows go to the workgroups in
// turn.  No atomics: the sums are the same on every run.  One pass: 805 MB for four fp32 4096 x 4096 in 155
// us, 5.2 TB/s; with 512 workgroups in place of 2048, 3.0.
template <bool kWide>
__global__ __launch_bounds__(256) void momentum_kernel(Update u, float *norms) {
  const int b = blockIdx.y;
  const void *grad = u.grad.p[b];
  float *buf = u.has_momentum ? u.momentum.p[b] : nullptr;
  float sum = 0.f;
  for (int64_t r = blockIdx.x; r < u.rows; r += gridDim.x) {
    const int64_t g0 = r * u.grad_stride, m0 = r * u.momentum_stride;
    if (kWide) {
      for (int c = threadIdx.x * 4; c < u.cols; c += 1024) {
        f32x4 g = grad4_at(grad, u.grad_dtype, g0 + c);
        if (buf) {
          f32x4 m = *reinterpret_cast<const f32x4 *>(buf + m0 + c);
          m = u.mu * m + g;
          *reinterpret_cast<f32x4 *>(buf + m0 + c) = m;
          g = u.nesterov ? g + u.mu * m : m;
        }
        for (int i = 0; i < 4; ++i) sum += g[i] * g[i];
      }
    } else {
      for (int c = threadIdx.x; c < u.cols; c += 256) {
        float g = grad_at(grad, u.grad_dtype, g0 + c);
        if (buf) {
          const float m = u.mu * buf[m0 + c] + g;
          buf[m0 + c] = m;
          g = u.nesterov ? g + u.mu * m : m;
        }
        sum += g * g;
      }
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) norms[b * gridDim.x + blockIdx.x] = sum;
}

// One orientation of X in the workspace: [rows][stride] fp16, the second part (if any) `low` elements on in
// the same row.
struct Image {
  half *p;
  int64_t stride, batch, low;
};

// X_0 in both orientations, its two parts, and the padding's zeros.  A workgroup turns a 64 x 64 tile over in
// LDS; its elements are loaded before it adds up the norm.  Bound by its bytes: 1.07 GB
// for four fp32 4096 x 4096 with momentum in 225 us, 4.7 TB/s, the rate of a copy.
template <bool kWide>
__global__ __launch_bounds__(256) void pack_kernel(Update u, const float *norms, int blocks, float eps, float scale, Image straight,
                                                   Image across, int parts) {
  __shared__ float tile[kSide][kSide + 1];
  const int b = blockIdx.z, r0 = blockIdx.y * kSide, c0 = blockIdx.x * kSide;
  const int quad = threadIdx.x % 16 * 4, line = threadIdx.x / 16;
  const void *grad = u.grad.p[b];
  const float *buf = u.has_momentum ? u.momentum.p[b] : nullptr;
  if (kWide) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t r = r0 + line + q * 16;
      const int c = c0 + quad;
      f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
      if (r < u.rows && c < u.cols) {
        if (!buf || u.nesterov) v = grad4_at(grad, u.grad_dtype, r * u.grad_stride + c);
        if (buf) {
          const f32x4 m = *reinterpret_cast<const f32x4 *>(buf + r * u.momentum_stride + c);
          v = u.nesterov ? v + u.mu * m : m;
        }
      }
      for (int i = 0; i < 4; ++i) tile[line + q * 16][quad + i] = v[i];
    }
  } else {
    const int c = c0 + threadIdx.x % kSide;
#pragma unroll 4
    for (int y = threadIdx.x / kSide; y < kSide; y += 256 / kSide) {
      const int64_t r = r0 + y;
      float v = 0.f;
      if (r < u.rows && c < u.cols) {
        if (!buf || u.nesterov) v = grad_at(grad, u.grad_dtype, r * u.grad_stride + c);
        if (buf) {
          const float m = buf[r * u.momentum_stride + c];
          v = u.nesterov ? v + u.mu * m : m;
        }
      }
      tile[y][c - c0] = v;
    }
  }
  float norm = 0.f;
  for (int i = threadIdx.x; i < blocks; i += 256) norm += norms[b * blocks + i];
  norm = sqrtf(block_sum(norm));
  const float by = scale / (norm + eps);
  auto store = [&](half *o, int64_t low, f32x4 x) __attribute__((always_inline)) {
    half4 hi, lo;
    for (int i = 0; i < 4; ++i) hi[i] = (half)x[i];
    hi = settled(hi);
    for (int i = 0; i < 4; ++i) lo[i] = (half)(x[i] - (float)hi[i]);
    *reinterpret_cast<half4 *>(o) = hi;
    if (parts > 1) *reinterpret_cast<half4 *>(o + low) = lo;
  };
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int y = line + q * 16;
    f32x4 v, t;
    for (int i = 0; i < 4; ++i) v[i] = tile[y][quad + i], t[i] = tile[quad + i][y];
    store(straight.p + b * straight.batch + (r0 + y) * straight.stride + c0 + quad, straight.low, v * by);
    store(across.p + b * across.batch + (c0 + y) * across.stride + r0 + quad, across.low, t * by);
  }
}

using half8 = emrs_gemm::fp16x8;

// An offset from a wave's corner, held inside the matrix: what is read there is not stored, but is read with
// no branch, so that many such loads are on their way together.  (A corner may lie outside: then it is negative.)
__device__ __forceinline__ int inside(int at, int corner, int last) { return min(at, last - corner); }

// A wave's tile of a symmetric matrix, from LDS to its place and, off the diagonal, to the place across it.
// (A tile on the diagonal holds both: with two parts they differ in their sums' order, and are stored once.)
template <class Cfg>
__device__ __forceinline__ void store_symmetric(half *out, int64_t stride, const Where &w, int m0, int n0, int lane, const Product &p,
                                                const char *own) {
  // From a wave's corner on, offsets are 32 bits: 256 rows of 2^22 elements at most.
  const int step = (int)stride;
  half *const here = out + n0 * stride + m0;
  emrs_gemm::Turn<Cfg>::along_m(own, lane, [&](int x, int y, half8 v) __attribute__((always_inline)) {
    if (m0 + x < p.m && n0 + y < p.n) *reinterpret_cast<half8 *>(here + (y * step + x)) = v;
  });
  if (w.m0 == w.n0) return;
  half *const across = out + m0 * stride + n0;
  emrs_gemm::Turn<Cfg>::along_n(own, lane, [&](int x, int y, half8 v) __attribute__((always_inline)) {
    if (m0 + x < p.m && n0 + y < p.n) *reinterpret_cast<half8 *>(across + (x * step + y)) = v;
  });
}

struct StoreGram : emrs_gemm::Operand {
  half *out;
  int64_t stride, batch;
  float by;

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        half4 v;
        for (int r = 0; r < 4; ++r) v[r] = (half)(acc[i][j][r] * by);
        emrs_gemm::Turn<Cfg>::put(own, i, j, lane, v);
      }
    store_symmetric<Cfg>(out + w.batch * batch, stride, w, m0, n0, lane, p, own);
  }
};

// a I + b A + c A A, the polynomial of the steps with one part; without a I (a = 0) of the others.
struct StorePolynomial : emrs_gemm::Operand {
  half *out;
  const half *gram;
  int64_t stride, batch;
  float a, b, c;  // a times the scale of A, c over it

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    const half *const in = gram + w.batch * batch + n0 * stride + m0;
    const int step = (int)stride;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int m = i * 16 + (lane >> 4) * 4, n = j * 16 + (lane & 15);
        const half4 x = *reinterpret_cast<const half4 *>(in + inside(m, m0, p.m - 4) + inside(n, n0, p.n - 1) * step);
        half4 v;
        for (int r = 0; r < 4; ++r) v[r] = (half)((m0 + m + r == n0 + n ? a : 0.f) + b * (float)x[r] + c * acc[i][j][r]);
        emrs_gemm::Turn<Cfg>::put(own, i, j, lane, v);
      }
    store_symmetric<Cfg>(out + w.batch * batch, stride, w, m0, n0, lane, p, own);
  }
};

// A product of symmetric matrices that commute, in two parts like its operands (side by side in a row, the
// second `stride` / 2 on): a I + b A + c A A for the polynomial, c alone for the others.
struct StoreSquare : emrs_gemm::Operand {
  half *out, *second_out;
  const half *in;         // A, or NULL
  const half *second;     // the first operand of matrices from `count` on, which share the second operand with
  int32_t count;          // the first `count`, and whose product goes to second_out
  int64_t stride, batch;
  float a, b, c;

  __device__ __forceinline__ const void *operand_a(const Product &p, int i) const {
    return i < count ? static_cast<const half *>(p.a) + i * p.a_batch : second + (i - count) * p.a_batch;
  }
  __device__ __forceinline__ const void *operand_b(const Product &p, int i) const {
    return static_cast<const half *>(p.b) + (i < count ? i : i - count) * p.b_batch;
  }

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    const int step = (int)stride, low = step / 2;
    const half *const from = in ? in + w.batch * batch + n0 * stride + m0 : nullptr;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      __builtin_amdgcn_sched_barrier(0);  // the loads of one column at a time: registers
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int m = i * 16 + (lane >> 4) * 4, n = j * 16 + (lane & 15);
        acc[i][j] *= c;
        if (from) {
          const half *const x = from + inside(m, m0, p.m - 4) + inside(n, n0, p.n - 1) * step;
          const half4 hi = *reinterpret_cast<const half4 *>(x), lo = *reinterpret_cast<const half4 *>(x + low);
          for (int r = 0; r < 4; ++r) acc[i][j][r] += (m0 + m + r == n0 + n ? a : 0.f) + b * ((float)hi[r] + (float)lo[r]);
        }
        acc[i][j] = settled(acc[i][j]);
        half4 v;
        for (int r = 0; r < 4; ++r) v[r] = (half)acc[i][j][r];
        emrs_gemm::Turn<Cfg>::put(own, i, j, lane, v);
      }
    }
    half *const to = w.batch < count ? out + w.batch * batch : second_out + (w.batch - count) * batch;
    store_symmetric<Cfg>(to, stride, w, m0, n0, lane, p, own);
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        half4 v;
        for (int r = 0; r < 4; ++r) v[r] = (half)(acc[i][j][r] - (float)(half)acc[i][j][r]);
        emrs_gemm::Turn<Cfg>::put(own, i, j, lane, v);
      }
    store_symmetric<Cfg>(to + low, stride, w, m0, n0, lane, p, own);
  }
};

// The product, plus a X from both its parts where the polynomial is without it.
__device__ __forceinline__ f32x4 applied(const half *x, int at, int low, int parts, float a, f32x4 acc) {
  if (parts == 1) return acc * (1.f / kGramScale);
  const half4 hi = *reinterpret_cast<const half4 *>(x + at);
  const half4 lo = *reinterpret_cast<const half4 *>(x + (at + low));
  f32x4 v;
  for (int r = 0; r < 4; ++r) v[r] = a * ((float)hi[r] + (float)lo[r]) + acc[r] * (1.f / kGramScale);
  return v;
}

// The next X (m: the longer side), in both orientations: its first part, then, where it has one, its second.
// Units of 16 bytes through LDS (four elements a lane: 995 us for four 4096 x 4096 from two parts to two, 880
// with, at the clock of that day); reading X and writing both orientations is a fifth of the time.
struct StoreIterate : emrs_gemm::Operand {
  Image in, out, across;
  int32_t in_parts, out_parts;
  float a;

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    using Turn = emrs_gemm::Turn<Cfg>;
    const half *const x = in.p + w.batch * in.batch + n0 * in.stride + m0;
    const int step = (int)in.stride, low = (int)in.low;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      __builtin_amdgcn_sched_barrier(0);  // the loads of one column at a time: registers
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int m = inside(i * 16 + (lane >> 4) * 4, m0, p.m - 4), n = inside(j * 16 + (lane & 15), n0, p.n - 1);
        acc[i][j] = settled(applied(x, n * step + m, low, in_parts, a, acc[i][j]));
        half4 v;
        for (int r = 0; r < 4; ++r) v[r] = (half)acc[i][j][r];
        Turn::put(own, i, j, lane, v);
      }
    }
    half *const o = out.p + w.batch * out.batch + n0 * out.stride + m0, *const t = across.p + w.batch * across.batch + m0 * across.stride + n0;
    store(o, t, m0, n0, lane, p, own, Turn{});
    if (out_parts == 1) return;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        half4 v;
        for (int r = 0; r < 4; ++r) v[r] = (half)(acc[i][j][r] - (float)(half)acc[i][j][r]);
        Turn::put(own, i, j, lane, v);
      }
    store(o + out.low, t + across.low, m0, n0, lane, p, own, Turn{});
  }
  template <class Turn>
  __device__ __forceinline__ void store(half *o, half *t, int m0, int n0, int lane, const Product &p, const char *own, Turn) const {
    const int o_step = (int)out.stride, t_step = (int)across.stride;
    Turn::along_m(own, lane, [&](int x, int y, half8 v) __attribute__((always_inline)) {
      if (m0 + x < p.m && n0 + y < p.n) *reinterpret_cast<half8 *>(o + (y * o_step + x)) = v;
    });
    Turn::along_n(own, lane, [&](int x, int y, half8 v) __attribute__((always_inline)) {
      if (m0 + x < p.m && n0 + y < p.n) *reinterpret_cast<half8 *>(t + (x * t_step + y)) = v;
    });
  }
};

// The last X: the result, or the update of the weights and their bf16 image.  m runs along the caller's rows,
// which are written four elements at a time where they lie so (kWide).
template <bool kWide>
struct StoreResult : emrs_gemm::Operand {
  Image in;
  int32_t in_parts;
  float a, by;  // by: over the scale of X
  int32_t rows, cols;
  Table<void *> out, image;
  Table<float *> main;
  int64_t out_stride, image_stride, main_stride;
  int32_t has_out, has_image, has_main;
  float keep, rate;

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *) const {
    const half *const x = in.p + w.batch * in.batch + n0 * in.stride + m0;
    __bf16 *o = has_out ? static_cast<__bf16 *>(out.p[w.batch]) : nullptr;
    __bf16 *img = has_image ? static_cast<__bf16 *>(image.p[w.batch]) : nullptr;
    float *mn = has_main ? main.p[w.batch] : nullptr;
    const int step = (int)in.stride, low = (int)in.low;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      __builtin_amdgcn_sched_barrier(0);  // the loads of one column at a time: registers
      f32x4 before[Cfg::MI];
      if (kWide && mn)
#pragma unroll
        for (int i = 0; i < Cfg::MI; ++i)
          before[i] = *reinterpret_cast<const f32x4 *>(mn + min(n0 + j * 16 + (lane & 15), rows - 1) * main_stride +
                                                       min(m0 + i * 16 + (lane >> 4) * 4, cols - 4));
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int c = m0 + i * 16 + (lane >> 4) * 4;
        const int64_t r = n0 + j * 16 + (lane & 15);
        // The workspace's rows and columns go on with zeros to multiples of 64, and past them this reads others.
        f32x4 v = applied(x, inside(j * 16 + (lane & 15), n0, p.n - 1) * step + inside(i * 16 + (lane >> 4) * 4, m0, p.m - 4), low, in_parts, a,
                          acc[i][j]) * by;
        if (c >= cols || r >= rows) continue;
        if (kWide) {
          if (mn) {
            v = before[i] * keep - rate * v;
            *reinterpret_cast<f32x4 *>(mn + r * main_stride + c) = v;
          }
          bf16x4 h;
          for (int k = 0; k < 4; ++k) h[k] = (__bf16)v[k];
          if (o) *reinterpret_cast<bf16x4 *>(o + r * out_stride + c) = h;
          if (img) *reinterpret_cast<bf16x4 *>(img + r * image_stride + c) = h;
          continue;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c + k >= cols) continue;
          float u = v[k];
          if (mn) {
            float *at = mn + r * main_stride + c + k;
            u = *at * keep - rate * u;
            *at = u;
          }
          if (o) o[r * out_stride + c + k] = (__bf16)u;
          if (img) img[r * image_stride + c + k] = (__bf16)u;
        }
      }
    }
  }
};

// ---- small matrices: the whole update of one in one workgroup ----
//
// A matrix whose X, in two parts, fits in a CU's LDS beside the polynomial stays there for all its steps: one
// launch and no memory traffic in place of three launches a step, which cost 5 us each whatever their work.
// X lies [s][l] (s: the shorter side, padded to 32; l to 64), units of 16 bytes permuted by s; the product
// X <- P X takes the columns of X as rows through the transposing LDS read.  LDS reads bound it, so a
// wave of the S x S products computes 32 x 32, on or below the diagonal; where that leaves waves over, KS of
// them share one over k.  For P X a wave has all S of every 16th 16 of L.  128 x 128 takes 41 us, one or two
// of them; as launches of the large kernels, 108.

struct Small {
  Update u;
  Table<void *> out, image;
  Table<float *> main;
  int64_t out_stride, image_stride, main_stride;
  int32_t has_out, has_image, has_main, tall, fours;
  int32_t s, l, steps;
  float eps, scale, keep, rate;
  float coefficients[3 * EMRS_MUON_MAX_STEPS];
};

constexpr int kSmallLds = 160 * 1024, kSmallWaves = 16;

constexpr int small_poly_stride(int s) { return s <= 64 ? 64 : 128; }
constexpr int small_blocks(int s) { return (s / 32) * (s / 32 + 1) / 2; }         // of 32 x 32, with the diagonal's
constexpr int small_shares(int s) { return s <= 32 ? 8 : s <= 64 ? 4 : 1; }       // waves of one over k
constexpr int small_fixed(int s) { return 2 * s * small_poly_stride(s) + (small_shares(s) - 1) * small_blocks(s) * 4096; }
constexpr int64_t small_bytes(int64_t s, int64_t l) { return 4 * s * l + small_fixed((int)s); }

// Rows of tiles of P X that a wave may have, for S = 16 ST: as many as LDS can hold.
template <int ST>
constexpr int small_rounds() {
  constexpr int s = 16 * ST, l = (kSmallLds - small_fixed(s)) / (4 * s) / 64 * 64;
  return (l / 16 + kSmallWaves - 1) / kSmallWaves;
}

template <int ST>
__global__ __launch_bounds__(kSmallWaves * 64) void small_kernel(Small a) {
  constexpr int S = 16 * ST, PS = small_poly_stride(S), R = small_rounds<ST>();
  constexpr int KS = small_shares(S), BLOCKS = small_blocks(S);
  static_assert(KS * BLOCKS <= kSmallWaves, "a wave each");
  __shared__ __attribute__((aligned(1024))) char lds[kSmallLds];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lp = (a.l + 63) / 64 * 64;
  half *const hi = reinterpret_cast<half *>(lds), *const lo = hi + S * lp, *const poly = lo + S * lp;
  f32x4 *const shares = reinterpret_cast<f32x4 *>(poly + S * PS);
  // Rows of a multiple of 256 bytes begin in the same bank: 16 units take part in the permutation, else 8.
  const int x_mask = lp % 128 == 0 ? 15 : 7;
  constexpr int p_mask = PS == 128 ? 15 : 7;
  auto x_at = [&](int s, int l) { return s * lp + (((l >> 3) ^ (s & x_mask)) << 3) + (l & 7); };
  auto p_at = [&](int s, int k) { return s * PS + (((k >> 3) ^ (s & p_mask)) << 3) + (k & 7); };

  // The momentum, and the norm.  Eight elements a thread at once: their loads are on their way together.
  constexpr int kThreads = kSmallWaves * 64, kBatch = 8;
  const int rows = a.u.rows, cols = a.u.cols, n = rows * cols;
  const void *const grad = a.u.grad.p[b];
  float *const buf = a.u.has_momentum ? a.u.momentum.p[b] : nullptr;
  const float over_cols = 1.f / (float)cols;  // n is below 2^16: the product's floor is the quotient
  auto row_of = [&](int at, float over) { return (int)(((float)at + 0.5f) * over); };
  float sum = 0.f;
  for (int from = threadIdx.x; from < n; from += kThreads * kBatch) {
    float g[kBatch], m[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = from + i * kThreads, r = row_of(at, over_cols), c = at - r * cols;
      g[i] = at < n ? grad_at(grad, a.u.grad_dtype, r * a.u.grad_stride + c) : 0.f;
      m[i] = buf && at < n ? buf[r * a.u.momentum_stride + c] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = from + i * kThreads, r = row_of(at, over_cols), c = at - r * cols;
      float v = g[i];
      if (buf) {
        m[i] = a.u.mu * m[i] + g[i];
        if (at < n) buf[r * a.u.momentum_stride + c] = m[i];
        v = a.u.nesterov ? g[i] + a.u.mu * m[i] : m[i];
      }
      sum += v * v;
    }
  }
  float *const part = reinterpret_cast<float *>(lds);
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  float norm = 0.f;
  for (int i = 0; i < kSmallWaves; ++i) norm += part[i];
  __syncthreads();
  const float by = a.scale / (sqrtf(norm) + a.eps);
  // X_0, with zeros in its padding.  Lanes run along the caller's rows.
  const int all_cols = a.tall ? S : lp, all = S * lp;
  const float over_all = 1.f / (float)all_cols;
  for (int from = threadIdx.x; from < all; from += kThreads * kBatch) {
    float g[kBatch], m[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = from + i * kThreads, r = row_of(at, over_all), c = at - r * all_cols;
      const bool in = r < rows && c < cols;
      g[i] = in ? grad_at(grad, a.u.grad_dtype, r * a.u.grad_stride + c) : 0.f;
      m[i] = buf && in ? buf[r * a.u.momentum_stride + c] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = from + i * kThreads, r = row_of(at, over_all), c = at - r * all_cols;
      if (at >= all) continue;
      const float v = (buf ? a.u.nesterov ? g[i] + a.u.mu * m[i] : m[i] : g[i]) * by;
      const half h = settled((half)v);
      const int o = a.tall ? x_at(c, r) : x_at(r, c);
      hi[o] = h;
      lo[o] = (half)(v - (float)h);
    }
  }
  __syncthreads();

  typedef __attribute__((ext_vector_type(4))) short s16x4;
  typedef __attribute__((ext_vector_type(8))) short s16x8;
  typedef __attribute__((address_space(3))) s16x4 *lds4;
  const int t = lane & 15, q = lane >> 4;
  // This wave's block of the S x S products, rows from `bi` and columns from `bj` on, and its share of k.
  const int share = wave / BLOCKS, block = wave % BLOCKS;
  int bi = 0;
  while ((bi + 1) * (bi + 2) / 2 <= block) ++bi;
  const int bj = (block - bi * (bi + 1) / 2) * 32;
  bi *= 32;
  auto from_rows = [&](const half *x, int s, int k) { return *reinterpret_cast<const emrs_gemm::fp16x8 *>(x + x_at(s, k)); };
  auto from_columns = [&](half *x, int l, int s) __attribute__((always_inline)) {  // eight s of column l + t
    const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(x + x_at(s + (t >> 2), l + (t & 3) * 4)));
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(x + x_at(s + 4 + (t >> 2), l + (t & 3) * 4)));
    return __builtin_bit_cast(emrs_gemm::fp16x8, (s16x8)__builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x4 acc[R][ST];
#pragma unroll 1
  for (int step = 0; step < a.steps; ++step) {
    const float fa = a.coefficients[3 * step], fb = a.coefficients[3 * step + 1], fc = a.coefficients[3 * step + 2];
    const bool split = a.steps - step > 2;
    f32x4 gram[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) gram[i / 2][i % 2] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (share < KS) {
#pragma unroll 1
      for (int k = share * 32; k < lp; k += KS * 32) {
        emrs_gemm::fp16x8 m[2], n[2], m_lo[2], n_lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[i] = from_rows(hi, bi + i * 16 + t, k + q * 8), n[i] = from_rows(hi, bj + i * 16 + t, k + q * 8);
          if (split) m_lo[i] = from_rows(lo, bi + i * 16 + t, k + q * 8), n_lo[i] = from_rows(lo, bj + i * 16 + t, k + q * 8);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 &c = gram[i / 2][i % 2];
          c = emrs_gemm::mfma(m[i / 2], n[i % 2], c);
          if (split) c = emrs_gemm::mfma(m_lo[i / 2], n[i % 2], emrs_gemm::mfma(m[i / 2], n_lo[i % 2], c));
        }
      }
    }
    if (KS > 1) {
      if (share > 0 && share < KS)
#pragma unroll
        for (int i = 0; i < 4; ++i) shares[(((share - 1) * BLOCKS + block) * 4 + i) * 64 + lane] = gram[i / 2][i % 2];
      __syncthreads();
      if (share == 0)
#pragma unroll
        for (int k = 1; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) gram[i / 2][i % 2] += shares[(((k - 1) * BLOCKS + block) * 4 + i) * 64 + lane];
    }
    // Entry (m, n) of a block goes to its place and, off the diagonal, across it.
    auto put = [&](int i, half4 v) __attribute__((always_inline)) {
      const int m = bi + i / 2 * 16 + q * 4, n = bj + i % 2 * 16 + t;
      *reinterpret_cast<half4 *>(poly + p_at(n, m)) = v;
      if (bi != bj)
        for (int r = 0; r < 4; ++r) poly[p_at(m + r, n)] = v[r];
    };
    if (share == 0) {
      const float g = kGramScale / (a.scale * a.scale);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        half4 v;  // rounded as the product that squares it sees it
        for (int r = 0; r < 4; ++r) v[r] = (half)(gram[i / 2][i % 2][r] * g), gram[i / 2][i % 2][r] = (float)v[r];
        put(i, v);
      }
    }
    __syncthreads();
    f32x4 square[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) square[i / 2][i % 2] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto from_poly = [&](int s, int k) { return *reinterpret_cast<const emrs_gemm::fp16x8 *>(poly + p_at(s, k)); };
    if (share == 0) {
#pragma unroll 2
      for (int k = 0; k < S; k += 32) {
        emrs_gemm::fp16x8 m[2], n[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) m[i] = from_poly(bi + i * 16 + t, k + q * 8), n[i] = from_poly(bj + i * 16 + t, k + q * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) square[i / 2][i % 2] = emrs_gemm::mfma(m[i / 2], n[i % 2], square[i / 2][i % 2]);
      }
    }
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = bi + i / 2 * 16 + q * 4, n = bj + i % 2 * 16 + t;
        half4 v;
        for (int r = 0; r < 4; ++r)
          v[r] = (half)((!split && m + r == n ? fa * kGramScale : 0.f) + fb * gram[i / 2][i % 2][r] + fc / kGramScale * square[i / 2][i % 2][r]);
        put(i, v);
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int l = (wave + r * kSmallWaves) * 16;
#pragma unroll
      for (int j = 0; j < ST; ++j) acc[r][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (l < lp) {
#pragma unroll 1
        for (int k = 0; k < S; k += 32) {
          const emrs_gemm::fp16x8 m = from_columns(hi, l, k + q * 8);
          emrs_gemm::fp16x8 m_lo;
          if (split) m_lo = from_columns(lo, l, k + q * 8);
#pragma unroll
          for (int j = 0; j < ST; ++j) {
            const emrs_gemm::fp16x8 n = from_poly(j * 16 + t, k + q * 8);
            acc[r][j] = emrs_gemm::mfma(m, n, acc[r][j]);
            if (split) acc[r][j] = emrs_gemm::mfma(m_lo, n, acc[r][j]);
          }
        }
#pragma unroll
        for (int j = 0; j < ST; ++j) {
          const int o = x_at(j * 16 + t, l + q * 4);
          acc[r][j] *= 1.f / kGramScale;
          if (split) {
            const half4 x = *reinterpret_cast<const half4 *>(hi + o), y = *reinterpret_cast<const half4 *>(lo + o);
            for (int i = 0; i < 4; ++i) acc[r][j][i] += fa * ((float)x[i] + (float)y[i]);
          }
        }
      }
    }
    __syncthreads();
    if (step + 1 == a.steps) break;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int l = (wave + r * kSmallWaves) * 16;
      if (l >= lp) continue;
#pragma unroll
      for (int j = 0; j < ST; ++j) {
        const int o = x_at(j * 16 + t, l + q * 4);
        half4 x, y;
        for (int i = 0; i < 4; ++i) x[i] = (half)acc[r][j][i];
        x = settled(x);
        for (int i = 0; i < 4; ++i) y[i] = (half)(acc[r][j][i] - (float)x[i]);
        *reinterpret_cast<half4 *>(hi + o) = x;
        *reinterpret_cast<half4 *>(lo + o) = y;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < ST; ++j) {
      __builtin_amdgcn_sched_barrier(0);  // one tile's addresses at a time: registers
      if (a.fours) {  // four of a row's elements, which lie so
        const int l = (wave + r * kSmallWaves) * 16 + q * 4, s = j * 16 + t;
        if (s >= a.s || l >= a.l) continue;
        f32x4 v = acc[r][j] * (1.f / a.scale);
        if (a.has_main) {
          f32x4 *const w = reinterpret_cast<f32x4 *>(a.main.p[b] + s * a.main_stride + l);
          v = *w * a.keep - a.rate * v;
          *w = v;
        }
        bf16x4 h;
        for (int i = 0; i < 4; ++i) h[i] = (__bf16)v[i];
        if (a.has_out) *reinterpret_cast<bf16x4 *>(static_cast<__bf16 *>(a.out.p[b]) + s * a.out_stride + l) = h;
        if (a.has_image) *reinterpret_cast<bf16x4 *>(static_cast<__bf16 *>(a.image.p[b]) + s * a.image_stride + l) = h;
        continue;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int l = (wave + r * kSmallWaves) * 16 + q * 4 + i, s = j * 16 + t;
        if (s >= a.s || l >= a.l) continue;
        const int64_t row = a.tall ? l : s, col = a.tall ? s : l;
        float v = acc[r][j][i] * (1.f / a.scale);
        if (a.has_main) {
          float *const w = a.main.p[b] + row * a.main_stride + col;
          v = *w * a.keep - a.rate * v;
          *w = v;
        }
        if (a.has_out) static_cast<__bf16 *>(a.out.p[b])[row * a.out_stride + col] = (__bf16)v;
        if (a.has_image) static_cast<__bf16 *>(a.image.p[b])[row * a.image_stride + col] = (__bf16)v;
      }
    }
}

struct Sizes {
  uint64_t s, l;                             // padded sides
  uint64_t x[2], xt[2], gram, poly, squares, norms, total;  // offsets; x and xt hold both parts of every matrix
  uint32_t blocks;                           // workgroups of the norm, a matrix
};

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Whether the steps with two parts work on S x S matrices alone.  All of a step's polynomials commute:
// A <- P A P and Q <- P Q take the place of X <- P X, and X <- Q X follows once.  With r = L / S that is
// 4.5 r + 13.5 products of S S S for three steps in place of 10.5 r + 6, by the multiply-adds; where two more
// launches and triangles that fill their last round badly count too, it pays from r = 2.5 on.  (Not for the
// steps with one part: there the rounding of A, which grows by a^2 a step, would double the error.)
//
// Q's size is the product of the polynomials' largest values, and where there are no singular values that is
// the product of the a: held times 64 in fp16 it must stay under 65504.  (The default triple's product is 41
// in five steps, 485 in seven, 1669 in eight.)  Steps on X itself have no such growth: past a product of 512
// they run instead.
constexpr int kSquares = 5;
constexpr double kMostGrowth = 512;

// The largest values of the polynomials of the steps with two parts, multiplied: of the first step over
// singular values in [0, 1], of each later one over what the step before can make of them.
double growth(const emrs_muon *a) {
  double product = 1, top = 1;  // of singular values
  for (uint32_t k = 0; k + 2 < a->steps; ++k) {
    const double c0 = a->coefficients[3 * k], c1 = a->coefficients[3 * k + 1], c2 = a->coefficients[3 * k + 2];
    const double end = top * top;
    auto p = [&](double t) { return std::abs(c0 + t * (c1 + t * c2)); };  // of t = s s
    // Both extremes lie at an end or where the derivative is 0: of p at -c1 / 2 c2, of s p at 0 = c0 + 3 c1 t + 5 c2 t t.
    double most = std::max(p(0), p(end)), next = top * p(end);
    auto inner = [&](double t) {
      if (t > 0 && t < end) most = std::max(most, p(t)), next = std::max(next, std::sqrt(t) * p(t));
    };
    if (c2 != 0) {
      inner(-c1 / (2 * c2));
      const double root = std::sqrt(std::max(0.0, 9 * c1 * c1 - 20 * c0 * c2));
      inner((-3 * c1 + root) / (10 * c2));
      inner((-3 * c1 - root) / (10 * c2));
    } else if (c1 != 0) {
      inner(-c0 / (3 * c1));
    }
    product *= std::max(1.0, most);
    top = next;
  }
  return product;
}

// Without coefficients (a workspace may be asked for before they are known) what the shape alone allows.
bool by_squares(const emrs_muon *a) {
  const uint64_t s = std::min(a->rows, a->cols), l = std::max(a->rows, a->cols);
  return a->steps > 3 && 2 * l >= 5 * s && (!a->coefficients || growth(a) <= kMostGrowth);
}

Sizes sizes_of(const emrs_muon *a) {
  Sizes z{};
  z.s = round_up(std::min(a->rows, a->cols), kSide);
  z.l = round_up(std::max(a->rows, a->cols), kSide);
  z.blocks = (uint32_t)std::min<uint64_t>(a->rows, std::max<uint64_t>(kNormBlocks / a->count, 256));
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  for (int i = 0; i < 2; ++i) z.x[i] = take(2 * a->count * z.s * z.l * 2);
  for (int i = 0; i < 2; ++i) z.xt[i] = take(2 * a->count * z.s * z.l * 2);
  z.gram = take(a->count * z.s * z.s * 2);
  z.poly = take(a->count * z.s * z.s * 2);
  z.squares = take(by_squares(a) ? kSquares * a->count * z.s * 2 * z.s * 2 : 0);
  z.norms = take((uint64_t)a->count * z.blocks * 4);
  z.total = at;
  return z;
}

int check(const emrs_muon *a) {
  if (!a) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: NULL argument");
  if (a->count == 0 || a->count > kMaxMatrices) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: 1 to 32 matrices wanted");
  if (a->grad_dtype > EMRS_FP16) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: gradients are fp32, bf16 or fp16");
  // Rows of a tile lie within 32-bit byte offsets of each other.
  if (a->rows == 0 || a->cols == 0 || a->rows > (1u << 20) || a->cols > (1u << 20))
    return fail(EMRS_ERR_TOO_LARGE, "muon: sides of 1 to 2^20 wanted");
  if (std::min(a->rows, a->cols) > 32768) return fail(EMRS_ERR_TOO_LARGE, "muon: the shorter side is at most 32768");
  if (a->steps == 0 || a->steps > EMRS_MUON_MAX_STEPS) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: 1 to 16 steps wanted");
  return EMRS_OK;
}

int check_matrices(const emrs_muon *a) {
  if (!a->coefficients || !a->grad) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: NULL coefficients or gradients");
  if (!a->out && !a->main) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: neither out nor main is given");
  if (a->out && a->main) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: out and main exclude each other");
  if (a->image && !a->main) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: an image needs main");
  const uint64_t grad_bytes = a->grad_dtype == EMRS_FP32 ? 4 : 2;
  auto each = [&](const void *const *p, uint64_t stride, uint64_t bytes, const char *what) {
    if (!p) return (int)EMRS_OK;
    if (a->rows > 1 && (stride < a->cols || stride > (1ull << 40)))
      return fail(EMRS_ERR_INVALID_ARGUMENT, std::string("muon: rows of ") + what + " overlap or lie too far apart");
    for (uint32_t i = 0; i < a->count; ++i) {
      if (!p[i]) return fail(EMRS_ERR_INVALID_ARGUMENT, std::string("muon: a NULL matrix in ") + what);
      if (reinterpret_cast<uintptr_t>(p[i]) % bytes)
        return fail(EMRS_ERR_MISALIGNED, std::string("muon: ") + what + " is off its type's alignment");
    }
    return (int)EMRS_OK;
  };
  int rc = each(a->grad, a->grad_stride, grad_bytes, "grad");
  if (!rc) rc = each(reinterpret_cast<const void *const *>(a->momentum), a->momentum_stride, 4, "momentum");
  if (!rc) rc = each(reinterpret_cast<const void *const *>(a->main), a->main_stride, 4, "main");
  if (!rc) rc = each(reinterpret_cast<const void *const *>(a->image), a->image_stride, 2, "image");
  if (!rc) rc = each(reinterpret_cast<const void *const *>(a->out), a->out_stride, 2, "out");
  return rc;
}

// Whether groups of four elements of every row lie on their own size.
bool fours(const emrs_muon *a, const void *const *p, uint64_t stride, uint64_t bytes) {
  if (!p) return true;
  if (a->cols % 4 || (a->rows > 1 && stride % 4)) return false;
  for (uint32_t i = 0; i < a->count; ++i)
    if (reinterpret_cast<uintptr_t>(p[i]) % (4 * bytes)) return false;
  return true;
}

#define TRY(expr)                                                                                   \
  do {                                                                                              \
    const hipError_t e_ = (expr);                                                                   \
    if (e_ != hipSuccess) return fail(EMRS_ERR_HIP, std::string("muon: ") + hipGetErrorString(e_)); \
  } while (0)

Small small_of(const emrs_muon *a, const Update &u, float scale, bool fours) {
  Small k{};
  k.u = u;
  for (uint32_t i = 0; i < a->count; ++i) {
    if (a->out) k.out.p[i] = a->out[i];
    if (a->image) k.image.p[i] = a->image[i];
    if (a->main) k.main.p[i] = a->main[i];
  }
  k.out_stride = a->out_stride, k.image_stride = a->image_stride, k.main_stride = a->main_stride;
  k.has_out = a->out != nullptr, k.has_image = a->image != nullptr, k.has_main = a->main != nullptr;
  k.tall = a->rows > a->cols, k.fours = fours && !k.tall;
  k.s = (int)std::min(a->rows, a->cols), k.l = (int)std::max(a->rows, a->cols);
  k.steps = (int)a->steps;
  k.eps = a->eps, k.scale = scale, k.keep = 1.f - a->decay, k.rate = a->rate;
  std::copy(a->coefficients, a->coefficients + 3 * a->steps, k.coefficients);
  return k;
}

template <bool kWide>
StoreResult<kWide> result(const emrs_muon *a, const Image &in, int parts, float factor, float scale) {
  StoreResult<kWide> e{};
  e.in = in, e.in_parts = parts;
  e.a = factor, e.by = 1.f / scale;
  e.rows = (int)a->rows, e.cols = (int)a->cols;
  for (uint32_t i = 0; i < a->count; ++i) {
    if (a->out) e.out.p[i] = a->out[i];
    if (a->image) e.image.p[i] = a->image[i];
    if (a->main) e.main.p[i] = a->main[i];
  }
  e.out_stride = a->out_stride, e.image_stride = a->image_stride, e.main_stride = a->main_stride;
  e.has_out = a->out != nullptr, e.has_image = a->image != nullptr, e.has_main = a->main != nullptr;
  e.keep = 1.f - a->decay, e.rate = a->rate;
  return e;
}

int step(const emrs_muon *a, hipStream_t st) {
  const Sizes z = sizes_of(a);
  char *ws = static_cast<char *>(a->workspace);
  const bool tall = a->rows > a->cols;
  const uint64_t grad_bytes = a->grad_dtype == EMRS_FP32 ? 4 : 2;

  Update u{};
  for (uint32_t i = 0; i < a->count; ++i) {
    u.grad.p[i] = a->grad[i];
    if (a->momentum) u.momentum.p[i] = a->momentum[i];
  }
  u.grad_stride = a->grad_stride, u.momentum_stride = a->momentum_stride;
  u.rows = (int)a->rows, u.cols = (int)a->cols;
  u.grad_dtype = a->grad_dtype;
  u.has_momentum = a->momentum != nullptr, u.nesterov = a->nesterov != 0;
  u.mu = a->mu;
  float *norms = reinterpret_cast<float *>(ws + z.norms);
  // Entries of an orthogonal S x L matrix are 1 / sqrt(L): the scale of X brings them to 1.
  const float scale = std::ldexp(1.f, (int)std::lround(0.5 * std::log2((double)z.l)));
  const bool wide_rows = fours(a, reinterpret_cast<const void *const *>(a->main), a->main_stride, 4) &&
                         fours(a, reinterpret_cast<const void *const *>(a->image), a->image_stride, 2) &&
                         fours(a, reinterpret_cast<const void *const *>(a->out), a->out_stride, 2);
  const int small = (int)round_up(std::min(a->rows, a->cols), 32);
  if (small <= 128 && small_bytes(small, (int64_t)z.l) <= kSmallLds) {
    const Small k = small_of(a, u, scale, wide_rows);
    switch (small) {
      case 32: small_kernel<2><<<a->count, kSmallWaves * 64, 0, st>>>(k); break;
      case 64: small_kernel<4><<<a->count, kSmallWaves * 64, 0, st>>>(k); break;
      case 96: small_kernel<6><<<a->count, kSmallWaves * 64, 0, st>>>(k); break;
      default: small_kernel<8><<<a->count, kSmallWaves * 64, 0, st>>>(k); break;
    }
    TRY(hipGetLastError());
    return EMRS_OK;
  }
  const bool wide = fours(a, a->grad, a->grad_stride, grad_bytes) &&
                    fours(a, reinterpret_cast<const void *const *>(a->momentum), a->momentum_stride, 4);
  const dim3 grid(z.blocks, a->count);
  if (wide)
    momentum_kernel<true><<<grid, 256, 0, st>>>(u, norms);
  else
    momentum_kernel<false><<<grid, 256, 0, st>>>(u, norms);
  TRY(hipGetLastError());

  auto parts_of = [&](uint32_t k) { return a->steps - k > 2 ? 2 : 1; };
  const int64_t area = 2 * (int64_t)(z.s * z.l);
  auto x = [&](int i) { return Image{reinterpret_cast<half *>(ws + z.x[i]), 2 * (int64_t)z.l, area, (int64_t)z.l}; };
  auto xt = [&](int i) { return Image{reinterpret_cast<half *>(ws + z.xt[i]), 2 * (int64_t)z.s, area, (int64_t)z.s}; };
  half *gram = reinterpret_cast<half *>(ws + z.gram), *poly = reinterpret_cast<half *>(ws + z.poly);
  const int64_t square = (int64_t)(z.s * z.s);

  const dim3 tiles(round_up(a->cols, kSide) / kSide, round_up(a->rows, kSide) / kSide, a->count);
  const Image straight = tall ? xt(0) : x(0), across = tall ? x(0) : xt(0);
  if (wide)
    pack_kernel<true><<<tiles, 256, 0, st>>>(u, norms, (int)z.blocks, a->eps, scale, straight, across, parts_of(0));
  else
    pack_kernel<false><<<tiles, 256, 0, st>>>(u, norms, (int)z.blocks, a->eps, scale, straight, across, parts_of(0));
  TRY(hipGetLastError());

  int now = 0;
  uint32_t done = 0;
  if (by_squares(a)) {
    const int64_t two = 2 * (int64_t)z.s, each = (int64_t)z.s * two;
    half *const squares = reinterpret_cast<half *>(ws + z.squares);
    auto matrix = [&](int i) { return squares + i * (int64_t)a->count * each; };
    half *gram_of = matrix(0), *const p_of = matrix(1), *spare = matrix(2), *q_of = matrix(3), *q_next = matrix(4);
    // hi hi + hi lo + lo hi
    // With a second m, its product with n too: launches of small matrices are bound by their number.
    auto square = [&](const half *m, const half *n, half *out, const half *poly_of, float fa, float fb, float fc,
                      const half *second = nullptr, half *second_out = nullptr) {
      Product g{};
      g.a = m, g.b = n;
      g.a_stride = g.b_stride = two, g.a_batch = g.b_batch = each;
      g.m = g.n = (int)z.s, g.k = 3 * (int)z.s;
      g.a_wrap = (int)z.s, g.b_wrap = 2 * (int)z.s;
      g.batch = (int)a->count * (second ? 2 : 1), g.symmetric = 1;
      return emrs_gemm::launch<half>(g, StoreSquare{{}, out, second_out, poly_of, second, (int)a->count, two, each, fa, fb, fc}, st);
    };
    const Image in = x(0), in_t = xt(0);
    Product g{};
    g.a = g.b = in.p;
    g.a_stride = g.b_stride = in.stride, g.a_batch = g.b_batch = in.batch;
    g.m = g.n = (int)z.s, g.k = 3 * (int)z.l;
    g.a_wrap = (int)z.l, g.b_wrap = 2 * (int)z.l;
    g.batch = (int)a->count, g.symmetric = 1;
    TRY((emrs_gemm::launch<half>(g, StoreSquare{{}, gram_of, nullptr, nullptr, nullptr, (int)a->count, two, each, 0.f, 0.f, kGramScale / (scale * scale)}, st)));
    constexpr float one = 1.f / kGramScale;
    for (; parts_of(done) == 2; ++done) {
      const float *f = a->coefficients + 3 * done;
      half *const p = done == 0 ? q_of : p_of;
      TRY(square(gram_of, gram_of, p, gram_of, f[0] * kGramScale, f[1], f[2] * one));
      const bool again = parts_of(done + 1) == 2;
      if (done == 0) {
        TRY(square(gram_of, p, spare, nullptr, 0.f, 0.f, one));
      } else {
        TRY(again ? square(q_of, p, q_next, nullptr, 0.f, 0.f, one, gram_of, spare) : square(q_of, p, q_next, nullptr, 0.f, 0.f, one));
        std::swap(q_of, q_next);
      }
      if (again) TRY(square(spare, p, gram_of, nullptr, 0.f, 0.f, one));
    }
    Product r{};
    r.a = in_t.p, r.b = q_of;
    r.a_stride = in_t.stride, r.b_stride = two;
    r.a_batch = in_t.batch, r.b_batch = each;
    r.m = (int)z.l, r.n = (int)z.s, r.k = 3 * (int)z.s;
    r.a_wrap = (int)z.s, r.b_wrap = 2 * (int)z.s;
    r.batch = (int)a->count;
    TRY((emrs_gemm::launch<half>(r, StoreIterate{{}, in, x(1), xt(1), 1, 1, 0.f}, st)));
    now = 1;
  }
  for (uint32_t k = done; k < a->steps; ++k, now ^= 1) {
    const float *f = a->coefficients + 3 * k;
    const int parts = parts_of(k);
    const Image in = x(now), in_t = xt(now);
    Product g{};
    g.a = g.b = in.p;
    g.a_stride = g.b_stride = in.stride, g.a_batch = g.b_batch = area;
    g.m = g.n = (int)z.s, g.k = (int)z.l * (parts == 2 ? 3 : 1);
    // hi hi + hi lo + lo hi
    g.a_wrap = parts == 2 ? (int)z.l : emrs_gemm::kNoWrap, g.b_wrap = parts == 2 ? 2 * (int)z.l : emrs_gemm::kNoWrap;
    g.batch = (int)a->count, g.symmetric = 1;
    TRY((emrs_gemm::launch<half>(g, StoreGram{{}, gram, (int64_t)z.s, square, kGramScale / (scale * scale)}, st)));

    Product q{};
    q.a = q.b = gram;
    q.a_stride = q.b_stride = (int64_t)z.s, q.a_batch = q.b_batch = square;
    q.m = q.n = q.k = (int)z.s;
    q.a_wrap = q.b_wrap = emrs_gemm::kNoWrap;
    q.batch = (int)a->count, q.symmetric = 1;
    TRY((emrs_gemm::launch<half>(q, StorePolynomial{{}, poly, gram, (int64_t)z.s, square, parts == 1 ? f[0] * kGramScale : 0.f, f[1], f[2] / kGramScale}, st)));

    Product r{};
    const bool last = k + 1 == a->steps, turned = last && tall;
    // P hi + P lo
    const int32_t wrap = parts == 2 ? (int)z.s : emrs_gemm::kNoWrap;
    r.a = turned ? poly : in_t.p, r.b = turned ? in_t.p : poly;
    r.a_stride = turned ? (int64_t)z.s : in_t.stride, r.b_stride = turned ? in_t.stride : (int64_t)z.s;
    r.a_batch = turned ? square : area, r.b_batch = turned ? area : square;
    r.a_wrap = turned ? wrap : emrs_gemm::kNoWrap, r.b_wrap = turned ? emrs_gemm::kNoWrap : wrap;
    r.m = (int)(turned ? z.s : z.l), r.n = (int)(turned ? z.l : z.s), r.k = (int)z.s * parts;
    r.batch = (int)a->count;
    if (!last) {
      TRY((emrs_gemm::launch<half>(r, StoreIterate{{}, in, x(now ^ 1), xt(now ^ 1), parts, parts_of(k + 1), f[0]}, st)));
      continue;
    }
    const Image &from = turned ? in_t : in;
    const hipError_t e = wide_rows ? emrs_gemm::launch<half>(r, result<true>(a, from, parts, f[0], scale), st)
                                   : emrs_gemm::launch<half>(r, result<false>(a, from, parts, f[0], scale), st);
    TRY(e);
  }
  return EMRS_OK;
}

}  // namespace

extern "C" {

int emrs_muon_workspace(const emrs_muon *a, uint64_t *bytes) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    const int rc = check(a);
    if (rc) return rc;
    if (!bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "muon: NULL argument");
    *bytes = sizes_of(a).total;
    return EMRS_OK;
  });
}

int emrs_muon_step(const emrs_muon *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    int rc = check(a);
    if (!rc) rc = check_matrices(a);
    if (rc) return rc;
    const uint64_t want = sizes_of(a).total;
    if (!a->workspace || a->workspace_bytes < want)
      return fail(EMRS_ERR_INVALID_ARGUMENT,
                  "muon: the workspace holds " + std::to_string(a->workspace_bytes) + " bytes of " + std::to_string(want));
    if (reinterpret_cast<uintptr_t>(a->workspace) % 256) return fail(EMRS_ERR_MISALIGNED, "muon: the workspace is off 256 bytes");
    rc = emrs_internal::need_device();
    if (rc) return rc;
    return step(a, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
