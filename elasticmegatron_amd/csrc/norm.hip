// The norm before a block and what joins the block before it to the residual stream, in one pass each way.
//
// With n(b) = b / rms(b) branch_weight (or b itself), rms(x) = sqrt(mean x^2 + eps):
//   stream = residual_scale residual + gate n(branch),  normed = stream / rms(stream) weight.
// Backward, with hat = stream / rms(stream), d = grad_normed weight, dS the whole gradient of the stream:
//   dS = grad_stream + (d - hat mean(d hat)) / rms(stream);  grad_residual = residual_scale dS
//   grad_gate = dS n(branch) (summed over tokens where all share one);  dn = gate dS
//   with bh = branch / rms(branch), e = dn branch_weight:  grad_branch = (e - bh mean(e bh)) / rms(branch), or dn
//   grad_weight = sum_t grad_normed hat,  grad_branch_weight = sum_t dn bh.
//
// Everything is bound by memory: a row is read once into registers, where its sums are taken and its results
// made, and written once.  A row belongs to one wave up to 2048 elements and to two, four or eight above, in
// units of eight elements a lane.  Statistics, sums and products are in 32 bits; the norm is of the stream before
// its rounding, and backward takes hat from the rounded stream, which saves reading residual and branch again.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "emrs.h"
#include "internal.h"

namespace {

using emrs_internal::fail;

constexpr int kMaxHidden = 16384;
constexpr uint32_t kParts = 512;  // workgroups of a backward launch, each with its own sums over tokens

template <class T>
struct Unit {
  typedef __attribute__((ext_vector_type(8))) T x8;
};

// A row's place: `lanes` lanes, each with UNITS units of eight elements, `lanes` units apart.
template <class T, bool kWide>
__device__ __forceinline__ typename Unit<T>::x8 load_unit(const T *row, int at, int hidden) {
  using x8 = typename Unit<T>::x8;
  x8 v;
  if (kWide) {
    if (at < hidden) return *reinterpret_cast<const x8 *>(row + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
    return v;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = at + e < hidden ? row[at + e] : (T)0.f;
  return v;
}

template <class T, bool kWide>
__device__ __forceinline__ void store_unit(T *row, int at, int hidden, const float (&v)[8]) {
  if (kWide) {
    typename Unit<T>::x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (T)v[e];
    if (at < hidden) *reinterpret_cast<typename Unit<T>::x8 *>(row + at) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (at + e < hidden) row[at + e] = (T)v[e];
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o /= 2) v += __shfl_xor(v, o);
  return v;
}

// The sum over a row's waves, the same in every lane.  `room` alternates between two calls' places, so that one
// barrier a call is enough.
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float (*room)[WAVES], int &turn, int wave) {
  v = wave_sum(v);
  if (WAVES == 1) return v;
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) room[turn][wave] = v;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) sum += room[turn][i];
  return sum;
}

template <int WAVES>
constexpr int rows_of_block() {
  return WAVES == 1 ? 4 : 1;
}
template <int WAVES>
constexpr int threads_of() {
  return 64 * WAVES * rows_of_block<WAVES>();
}

struct Norm {
  uint64_t tokens;
  int hidden, gate_kind;
  const void *residual, *branch, *gate;
  int64_t residual_stride, branch_stride, gate_stride, stream_stride;
  const void *branch_weight, *weight;
  float scale, eps, share;  // share: 1 / hidden
  void *stream, *normed;
  float *stream_rms, *branch_rms;  // 1 / rms
  const void *grad_stream, *grad_normed;
  void *grad_residual, *grad_branch, *grad_gate;
  float *parts;              // [workgroups][3][hidden]: weight, branch_weight, gate
};

template <class T, class R, int WAVES, int UNITS, bool kWide>
__global__ __launch_bounds__(threads_of<WAVES>()) void norm_forward_kernel(Norm p) {
  using x8 = typename Unit<T>::x8;
  constexpr int lanes = 64 * WAVES;
  __shared__ float room[2][WAVES];
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
  const uint64_t row = (uint64_t)blockIdx.x * rows_of_block<WAVES>() + (WAVES == 1 ? wave : 0);
  if (row >= p.tokens) return;  // whole waves, and with several waves a row whole workgroups
  int turn = 0;
  const int hidden = p.hidden;
  const R *const residual = static_cast<const R *>(p.residual) + row * p.residual_stride;
  typename Unit<R>::x8 r[UNITS];
  x8 b[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) r[u] = load_unit<R, kWide>(residual, (u * lanes + lane) * 8, hidden);
  float s[UNITS][8];
  if (p.branch) {
    const T *const branch = static_cast<const T *>(p.branch) + row * p.branch_stride;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) b[u] = load_unit<T, kWide>(branch, (u * lanes + lane) * 8, hidden);
    float rms = 1.f;
    if (p.branch_weight) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf((float)b[u][e], (float)b[u][e], sum);
      rms = 1.f / sqrtf(row_sum<WAVES>(sum, room, turn, wave) * p.share + p.eps);
      if (lane == 0 && p.branch_rms) p.branch_rms[row] = rms;
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int at = (u * lanes + lane) * 8;
      float n[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = (float)b[u][e];
      if (p.branch_weight) {
        const x8 w = load_unit<T, kWide>(static_cast<const T *>(p.branch_weight), at, hidden);
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] = n[e] * rms * (float)w[e];
      }
      if (p.gate_kind) {
        const x8 g = load_unit<T, kWide>(static_cast<const T *>(p.gate) + (p.gate_kind == EMRS_NORM_GATE_TOKEN ? row * p.gate_stride : 0), at, hidden);
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] *= (float)g[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s[u][e] = fmaf(p.scale, (float)r[u][e], n[e]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[u][e] = p.scale * (float)r[u][e];
  }
  if (p.stream) {
    R *const to = static_cast<R *>(p.stream) + row * hidden;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) store_unit<R, kWide>(to, (u * lanes + lane) * 8, hidden, s[u]);
  }
  if (!p.normed) return;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(s[u][e], s[u][e], sum);
  const float rms = 1.f / sqrtf(row_sum<WAVES>(sum, room, turn, wave) * p.share + p.eps);
  if (lane == 0 && p.stream_rms) p.stream_rms[row] = rms;
  T *const to = static_cast<T *>(p.normed) + row * hidden;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int at = (u * lanes + lane) * 8;
    const x8 w = load_unit<T, kWide>(static_cast<const T *>(p.weight), at, hidden);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[u][e] *= rms * (float)w[e];
    store_unit<T, kWide>(to, at, hidden, s[u]);
  }
}

// A workgroup's rows are those of its own index and every gridDim.x-th from there; it keeps its sums over them in
// registers and leaves them in its own place of `parts`, where sum_parts_kernel joins them in a fixed order.
// kFull: with a branch norm or a gate.
template <class T, class R, int WAVES, int UNITS, bool kWide, bool kFull>
__global__ __launch_bounds__(threads_of<WAVES>()) void norm_backward_kernel(Norm p) {
  using x8 = typename Unit<T>::x8;
  constexpr int lanes = 64 * WAVES, rows = rows_of_block<WAVES>();
  constexpr int kSums = kFull ? 3 : 1;
  __shared__ float room[2][WAVES];
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
  int turn = 0;
  const int hidden = p.hidden;
  float sums[kSums][UNITS][8];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[k][u][e] = 0.f;
  x8 w[UNITS];
  if (p.grad_normed)
#pragma unroll
    for (int u = 0; u < UNITS; ++u) w[u] = load_unit<T, kWide>(static_cast<const T *>(p.weight), (u * lanes + lane) * 8, hidden);

  for (uint64_t row = (uint64_t)blockIdx.x * rows + (WAVES == 1 ? wave : 0); row < p.tokens; row += (uint64_t)gridDim.x * rows) {
    float ds[UNITS][8];
    typename Unit<R>::x8 s[UNITS], gs[UNITS];
    x8 go[UNITS], b[UNITS];
    if (p.grad_stream) {
      const R *const from = static_cast<const R *>(p.grad_stream) + row * hidden;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) gs[u] = load_unit<R, kWide>(from, (u * lanes + lane) * 8, hidden);
    }
    if (p.grad_normed) {
      const R *const from = static_cast<const R *>(p.stream) + row * p.stream_stride;
      const T *const grad = static_cast<const T *>(p.grad_normed) + row * hidden;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        s[u] = load_unit<R, kWide>(from, (u * lanes + lane) * 8, hidden);
        go[u] = load_unit<T, kWide>(grad, (u * lanes + lane) * 8, hidden);
      }
    }
    if (kFull) {
      const T *const branch = static_cast<const T *>(p.branch) + row * p.branch_stride;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) b[u] = load_unit<T, kWide>(branch, (u * lanes + lane) * 8, hidden);
    }
    if (p.grad_normed) {
      const float rms = p.stream_rms[row];
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float hat = (float)s[u][e] * rms, g = (float)go[u][e];
          sums[0][u][e] = fmaf(g, hat, sums[0][u][e]);
          sum = fmaf(g * (float)w[u][e], hat, sum);
        }
      const float mean = row_sum<WAVES>(sum, room, turn, wave) * p.share;
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float hat = (float)s[u][e] * rms;
          ds[u][e] = rms * ((float)go[u][e] * (float)w[u][e] - hat * mean);
        }
      if (p.grad_stream)
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) ds[u][e] += (float)gs[u][e];
    } else {
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) ds[u][e] = (float)gs[u][e];
    }
    if (p.grad_residual) {
      R *const to = static_cast<R *>(p.grad_residual) + row * hidden;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p.scale * ds[u][e];
        store_unit<R, kWide>(to, (u * lanes + lane) * 8, hidden, v);
      }
    }
    if (!p.branch) continue;
    T *const to = static_cast<T *>(p.grad_branch) + row * hidden;
    if (kFull) {
      const float rms = p.branch_weight ? p.branch_rms[row] : 1.f;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int at = (u * lanes + lane) * 8;
        x8 bw, g;
        if (p.branch_weight) bw = load_unit<T, kWide>(static_cast<const T *>(p.branch_weight), at, hidden);
        if (p.gate_kind) {
          g = load_unit<T, kWide>(static_cast<const T *>(p.gate) + (p.gate_kind == EMRS_NORM_GATE_TOKEN ? row * p.gate_stride : 0), at, hidden);
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = ds[u][e] * (float)b[u][e] * rms;
            if (p.branch_weight) v[e] *= (float)bw[e];
          }
          if (p.gate_kind == EMRS_NORM_GATE_TOKEN) {
            if (p.grad_gate) store_unit<T, kWide>(static_cast<T *>(p.grad_gate) + row * hidden, at, hidden, v);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[kSums - 1][u][e] += v[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) ds[u][e] *= (float)g[e];
        }
        if (p.branch_weight)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float hat = (float)b[u][e] * rms;
            sums[kSums / 2][u][e] = fmaf(ds[u][e], hat, sums[kSums / 2][u][e]);
            ds[u][e] *= (float)bw[e];
            sum = fmaf(ds[u][e], hat, sum);
          }
      }
      if (p.branch_weight) {
        const float mean = row_sum<WAVES>(sum, room, turn, wave) * p.share;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) ds[u][e] = rms * (ds[u][e] - (float)b[u][e] * rms * mean);
      }
    }
    if (p.grad_branch)
#pragma unroll
      for (int u = 0; u < UNITS; ++u) store_unit<T, kWide>(to, (u * lanes + lane) * 8, hidden, ds[u]);
  }

  if (!p.parts) return;
  float *const parts = p.parts + (uint64_t)blockIdx.x * 3 * hidden;
  // The rows of a workgroup of single waves meet in LDS first.
  constexpr int kUnit = rows == 1 ? 1 : lanes * 8;
  __shared__ float meet[rows][kUnit];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int at = (u * lanes + lane) * 8;
      if (rows > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) meet[wave % rows][(rows == 1 ? 0 : e * lanes + lane)] = sums[k][u][e];
        __syncthreads();
        if (wave == 0)
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 1; i < rows; ++i) sums[k][u][e] += meet[i][(rows == 1 ? 0 : e * lanes + lane)];
      }
      if (rows == 1 || wave == 0)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at + e < hidden) parts[(uint64_t)k * hidden + at + e] = sums[k][u][e];
    }
}

// Sums of the workgroups' parts, 32 columns of one of the three vectors to a workgroup: eight rows of lanes add
// every eighth part, and meet in LDS.
constexpr int kSumColumns = 32, kSumRows = 8;

template <class T>
__global__ __launch_bounds__(kSumColumns * kSumRows) void sum_parts_kernel(const float *parts, uint32_t count, int hidden, T *weight,
                                                                           T *branch_weight, T *gate) {
  __shared__ float meet[kSumRows][kSumColumns];
  T *const to = blockIdx.y == 0 ? weight : blockIdx.y == 1 ? branch_weight : gate;
  if (!to) return;
  const int column = blockIdx.x * kSumColumns + threadIdx.x % kSumColumns, row = threadIdx.x / kSumColumns;
  float sum = 0.f;
  if (column < hidden)
#pragma unroll 8
    for (uint32_t i = row; i < count; i += kSumRows) sum += parts[((uint64_t)i * 3 + blockIdx.y) * hidden + column];
  meet[row][threadIdx.x % kSumColumns] = sum;
  __syncthreads();
  if (row || column >= hidden) return;
#pragma unroll
  for (int i = 1; i < kSumRows; ++i) sum += meet[i][threadIdx.x];
  to[column] = (T)sum;
}

bool on(const void *p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether every row that is read or written lies on 16 bytes (rows of 32 bits: on 32).
bool wide(const emrs_norm *a) {
  for (const void *p : {a->residual, a->branch, a->gate, a->branch_weight, a->weight, (const void *)a->stream, (const void *)a->normed, a->grad_stream,
                        a->grad_normed, (const void *)a->grad_residual, (const void *)a->grad_branch, (const void *)a->grad_gate})
    if (!on(p, 32) && !(on(p, 16) && a->residual_dtype != EMRS_FP32)) return false;
  return a->hidden % 8 == 0 && a->residual_stride % 8 == 0 && a->branch_stride % 8 == 0 && a->gate_stride % 8 == 0 && a->stream_stride % 8 == 0;
}

template <int WAVES>
uint32_t blocks_of(uint64_t tokens) {
  return (uint32_t)((tokens + rows_of_block<WAVES>() - 1) / rows_of_block<WAVES>());
}

uint32_t parts_of(uint64_t tokens, int waves) { return (uint32_t)std::min<uint64_t>(kParts, waves == 1 ? (tokens + 3) / 4 : tokens); }
int waves_of(uint64_t hidden) { return hidden <= 2048 ? 1 : hidden <= 4096 ? 2 : hidden <= 8192 ? 4 : 8; }

template <class T, class R, int WAVES, int UNITS, bool kWide>
void launch(const Norm &p, bool backward, bool full, hipStream_t st) {
  constexpr int threads = threads_of<WAVES>();
  if (!backward)
    norm_forward_kernel<T, R, WAVES, UNITS, kWide><<<blocks_of<WAVES>(p.tokens), threads, 0, st>>>(p);
  else if (full)
    norm_backward_kernel<T, R, WAVES, UNITS, kWide, true><<<parts_of(p.tokens, WAVES), threads, 0, st>>>(p);
  else
    norm_backward_kernel<T, R, WAVES, UNITS, kWide, false><<<parts_of(p.tokens, WAVES), threads, 0, st>>>(p);
}

// Rows off their units take one shape a wave count: its element accesses bound it anyway.
template <class T, class R>
void launch(const Norm &p, bool backward, bool full, bool is_wide, hipStream_t st) {
  const int units = (p.hidden + 7) / 8;
  switch (waves_of(p.hidden)) {
    case 1:
      if (!is_wide) return launch<T, R, 1, 4, false>(p, backward, full, st);
      if (units <= 64) return launch<T, R, 1, 1, true>(p, backward, full, st);
      if (units <= 128) return launch<T, R, 1, 2, true>(p, backward, full, st);
      return launch<T, R, 1, 4, true>(p, backward, full, st);
    case 2: return is_wide ? launch<T, R, 2, 4, true>(p, backward, full, st) : launch<T, R, 2, 4, false>(p, backward, full, st);
    case 4: return is_wide ? launch<T, R, 4, 4, true>(p, backward, full, st) : launch<T, R, 4, 4, false>(p, backward, full, st);
    default: return is_wide ? launch<T, R, 8, 4, true>(p, backward, full, st) : launch<T, R, 8, 4, false>(p, backward, full, st);
  }
}

uint64_t workspace_of(const emrs_norm *a) { return (uint64_t)parts_of(a->tokens, waves_of(a->hidden)) * 3 * a->hidden * 4; }

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
  const uint64_t h = a->hidden;
  if (!a->branch && (a->gate_kind || a->branch_weight || a->grad_branch || a->grad_gate || a->grad_branch_weight))
    return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a gate or a branch's norm without a branch");
  if (a->gate_kind && !a->gate) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: NULL gate");
  if (a->grad_gate && !a->gate_kind) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a gradient of no gate");
  if (a->grad_branch_weight && !a->branch_weight) return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: a gradient of no branch weight");
  if ((a->branch && a->branch_stride < h) || (a->gate_kind == EMRS_NORM_GATE_TOKEN && a->gate_stride < h))
    return fail(EMRS_ERR_INVALID_ARGUMENT, "norm: rows overlap");
  const bool full = a->branch && (a->gate_kind || a->branch_weight);
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
  if (a->dtype == EMRS_BF16)
    a->residual_dtype == EMRS_FP32 ? launch<__bf16, float>(p, backward, full, w, st) : launch<__bf16, __bf16>(p, backward, full, w, st);
  else
    a->residual_dtype == EMRS_FP32 ? launch<_Float16, float>(p, backward, full, w, st) : launch<_Float16, _Float16>(p, backward, full, w, st);
  if (sums) {
    const dim3 grid((uint32_t)((h + kSumColumns - 1) / kSumColumns), full ? 3 : 1);
    const uint32_t count = parts_of(a->tokens, waves_of(h));
    void *const gate = a->gate_kind == EMRS_NORM_GATE_CHANNEL ? a->grad_gate : nullptr;
    if (a->dtype == EMRS_BF16)
      sum_parts_kernel<<<grid, kSumColumns * kSumRows, 0, st>>>(p.parts, count, p.hidden, static_cast<__bf16 *>(a->grad_weight),
                                                                static_cast<__bf16 *>(a->grad_branch_weight), static_cast<__bf16 *>(gate));
    else
      sum_parts_kernel<<<grid, kSumColumns * kSumRows, 0, st>>>(p.parts, count, p.hidden, static_cast<_Float16 *>(a->grad_weight),
                                                                static_cast<_Float16 *>(a->grad_branch_weight), static_cast<_Float16 *>(gate));
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
