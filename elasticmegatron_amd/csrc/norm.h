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
// made, and written once.  A row belongs to one wave as long as four units of eight elements a lane hold it forward
// (2048 elements) and two backward (1024), and to two, four or eight above; up to 256 elements, two or four rows share one.  Statistics, sums and products are in 32 bits;
// the norm is of the stream before its rounding, and backward takes hat from the rounded stream, which saves reading
// residual and branch again (a quarter more bytes for a plain sum) and is one rounding more in grad_weight.
//
// Measured: 4096 x 4096 in bf16, a plain sum, forward 24 us (5.6 TB/s) and backward 29 us (4.7 TB/s; 5 us more to sum
// the parts); 8192 x 8192, the stream in 32 bits, a norm and a gate for each channel on
// the branch, forward 154 us (5.2 TB/s) and backward 249 us (4.9 TB/s); a contiguous copy reaches 6.65 TB/s.  500 x 512 takes
// 3 to 4 us a kernel, and the call's host time is most of it.

#ifndef EMRS_NORM_H
#define EMRS_NORM_H

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "emrs.h"

namespace emrs_norm_kernels {

constexpr int kMaxHidden = 16384;
constexpr uint32_t kWavesOfSums = 2048;  // waves of a backward launch: eight for each CU, each workgroup with its own sums

// A lane's units of a row are E elements, 16 bytes of the widest type among its arrays, and a wave's lie side by side:
// every access is to whole lines.  (With eight fp32 elements a lane, two accesses of every other 16 bytes, backward of
// 8192 x 8192 takes 255 us against 249; forward, which holds the whole row, is not slower with eight.)
template <class R>
constexpr int unit_of() {
  return 16 / sizeof(R);
}

template <class T, int E>
struct Unit {
  typedef __attribute__((ext_vector_type(E))) T type;
};

template <class T, int E, bool kWide>
__device__ __forceinline__ typename Unit<T, E>::type load_unit(const T *row, int at, int hidden) {
  using V = typename Unit<T, E>::type;
  V v;
  if (kWide) {
    if (at < hidden) return *reinterpret_cast<const V *>(row + at);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (T)0.f;
    return v;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = at + e < hidden ? row[at + e] : (T)0.f;
  return v;
}

template <class T, int E, bool kWide>
__device__ __forceinline__ void store_unit(T *row, int at, int hidden, const float (&v)[E]) {
  if (kWide) {
    using V = typename Unit<T, E>::type;
    V o;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = (T)v[e];
    if (at < hidden) *reinterpret_cast<V *>(row + at) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (at + e < hidden) row[at + e] = (T)v[e];
}

// Over a row's lanes of one wave, all of which have it.
template <int LANES>
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = LANES < 64 ? LANES / 2 : 32; o; o /= 2) v += __shfl_xor(v, o);
  return v;
}

// The sum over a row's waves, the same in every lane.  `room` alternates between two calls' places, so that one
// barrier a call is enough.
template <int LANES>
constexpr int waves_of_row() {
  return LANES <= 64 ? 1 : LANES / 64;
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float (*room)[waves_of_row<LANES>()], int &turn, int wave) {
  constexpr int WAVES = waves_of_row<LANES>();
  v = wave_sum<LANES>(v);
  if (WAVES == 1) return v;
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) room[turn][wave] = v;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) sum += room[turn][i];
  return sum;
}

// Rows of up to a wave's lanes share a workgroup of four waves.
template <int LANES>
constexpr int rows_of_block() {
  return LANES <= 64 ? 256 / LANES : 1;
}
template <int LANES>
__device__ __forceinline__ int row_of_block() {
  return LANES <= 64 ? threadIdx.x / LANES : 0;  // the 0 keeps what goes by the row scalar
}
template <int LANES>
constexpr int threads_of() {
  return LANES * rows_of_block<LANES>();
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

template <class T, class R, int LANES, int UNITS, bool kWide>
__global__ __launch_bounds__(threads_of<LANES>()) void norm_forward_kernel(Norm p) {
  constexpr int E = 8, N = UNITS;
  using V = typename Unit<T, E>::type;
  constexpr int lanes = LANES;
  __shared__ float room[2][waves_of_row<LANES>()];
  const int lane = LANES <= 64 ? threadIdx.x % LANES : threadIdx.x, wave = threadIdx.x >> 6;
  const uint64_t row = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * rows_of_block<LANES>() + row_of_block<LANES>();
  if (row >= p.tokens) return;  // whole rows, and with several waves a row whole workgroups
  int turn = 0;
  const int hidden = p.hidden;
  const R *const residual = static_cast<const R *>(p.residual) + row * p.residual_stride;
  typename Unit<R, E>::type r[N];
  V b[N];
#pragma unroll
  for (int u = 0; u < N; ++u) r[u] = load_unit<R, E, kWide>(residual, (u * lanes + lane) * E, hidden);
  float s[N][E];
  if (p.branch) {
    const T *const branch = static_cast<const T *>(p.branch) + row * p.branch_stride;
#pragma unroll
    for (int u = 0; u < N; ++u) b[u] = load_unit<T, E, kWide>(branch, (u * lanes + lane) * E, hidden);
    float rms = 1.f;
    if (p.branch_weight) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) sum = fmaf((float)b[u][e], (float)b[u][e], sum);
      rms = 1.f / sqrtf(row_sum<LANES>(sum, room, turn, wave) * p.share + p.eps);
      if (lane == 0 && p.branch_rms) p.branch_rms[row] = rms;
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int at = (u * lanes + lane) * E;
      float n[E];
#pragma unroll
      for (int e = 0; e < E; ++e) n[e] = (float)b[u][e];
      if (p.branch_weight) {
        const V w = load_unit<T, E, kWide>(static_cast<const T *>(p.branch_weight), at, hidden);
#pragma unroll
        for (int e = 0; e < E; ++e) n[e] = n[e] * rms * (float)w[e];
      }
      if (p.gate_kind) {
        const V g = load_unit<T, E, kWide>(static_cast<const T *>(p.gate) + (p.gate_kind == EMRS_NORM_GATE_TOKEN ? row * p.gate_stride : 0), at, hidden);
#pragma unroll
        for (int e = 0; e < E; ++e) n[e] *= (float)g[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) s[u][e] = fmaf(p.scale, (float)r[u][e], n[e]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) s[u][e] = p.scale * (float)r[u][e];
  }
  if (p.stream) {
    R *const to = static_cast<R *>(p.stream) + row * hidden;
#pragma unroll
    for (int u = 0; u < N; ++u) store_unit<R, E, kWide>(to, (u * lanes + lane) * E, hidden, s[u]);
  }
  if (!p.normed) return;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) sum = fmaf(s[u][e], s[u][e], sum);
  const float rms = 1.f / sqrtf(row_sum<LANES>(sum, room, turn, wave) * p.share + p.eps);
  if (lane == 0 && p.stream_rms) p.stream_rms[row] = rms;
  T *const to = static_cast<T *>(p.normed) + row * hidden;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int at = (u * lanes + lane) * E;
    const V w = load_unit<T, E, kWide>(static_cast<const T *>(p.weight), at, hidden);
#pragma unroll
    for (int e = 0; e < E; ++e) s[u][e] *= rms * (float)w[e];
    store_unit<T, E, kWide>(to, at, hidden, s[u]);
  }
}

// What stands between a branch and the stream.
enum Kind { kPlain, kShared, kToken };  // nothing; a norm, a gate for each channel or both; a gate for each token, and maybe a norm

// What a lane reads of a row.
template <class T, class R, int N, Kind kKind>
struct RowOf {
  static constexpr int E = unit_of<R>();
  typename Unit<R, E>::type s[N], gs[N];
  typename Unit<T, E>::type go[N], b[kKind == kPlain ? 1 : N], g[kKind == kToken ? N : 1];
};

// A workgroup's rows are those of its own index and every gridDim.x-th from there; it keeps its sums over them in
// registers and leaves them in its own place of `parts`, where sum_parts_kernel joins them in a fixed order.  A row is
// read while the one before it is worked on: with two sums over the row in a chain, a workgroup that reads and works in
// turn leaves memory idle half of the time, and registers hold too few workgroups to fill that.  (Four units a lane
// leave no registers for it.)
template <class T, class R, int LANES, int UNITS, bool kWide, Kind kKind>
__global__ __launch_bounds__(threads_of<LANES>()) void norm_backward_kernel(Norm p) {
  constexpr int E = unit_of<R>(), N = UNITS * 8 / E;
  using V = typename Unit<T, E>::type;
  using Row = RowOf<T, R, N, kKind>;
  constexpr int lanes = LANES, rows = rows_of_block<LANES>();
  constexpr int kSums = kKind == kPlain ? 1 : kKind == kToken ? 2 : 3;  // weight, branch_weight, gate
  constexpr bool kFull = kKind != kPlain, by_token = kKind == kToken, kAhead = UNITS <= 2;
  __shared__ float room[2][waves_of_row<LANES>()];
  const int lane = LANES <= 64 ? threadIdx.x % LANES : threadIdx.x, wave = threadIdx.x >> 6, mine = row_of_block<LANES>();
  int turn = 0;
  const int hidden = p.hidden;
  auto at = [&](int u) { return (u * lanes + lane) * E; };
  float sums[kSums][N][E];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) sums[k][u][e] = 0.f;
  // What all rows share stays in registers; with four units a lane it is read again for every row.
  V weights[3][kAhead ? N : 1];
  const bool by_channel = kKind == kShared && p.gate_kind;
  auto shared = [&](int which, int u) __attribute__((always_inline)) {
    return load_unit<T, E, kWide>(static_cast<const T *>(which == 0 ? p.weight : which == 1 ? p.branch_weight : p.gate), at(u), hidden);
  };
  if constexpr (kAhead)
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (p.grad_normed) weights[0][u] = shared(0, u);
      if (kFull && p.branch_weight) weights[1][u] = shared(1, u);
      if (by_channel) weights[2][u] = shared(2, u);
    }
  auto of_all = [&](int which, int u) __attribute__((always_inline)) {
    if constexpr (kAhead) {
      V v = weights[which][u];
      asm("" : "+v"(v));  // widened anew for every row: 32-bit copies would take twice the registers
      return v;
    } else {
      return shared(which, u);
    }
  };

  auto read = [&](Row &r, uint64_t row) __attribute__((always_inline)) {
    if (row >= p.tokens) return;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (p.grad_normed) {
        r.s[u] = load_unit<R, E, kWide>(static_cast<const R *>(p.stream) + row * p.stream_stride, at(u), hidden);
        r.go[u] = load_unit<T, E, kWide>(static_cast<const T *>(p.grad_normed) + row * hidden, at(u), hidden);
      }
      if (p.grad_stream) r.gs[u] = load_unit<R, E, kWide>(static_cast<const R *>(p.grad_stream) + row * hidden, at(u), hidden);
      if (kFull) r.b[kFull ? u : 0] = load_unit<T, E, kWide>(static_cast<const T *>(p.branch) + row * p.branch_stride, at(u), hidden);
      if (by_token) r.g[by_token ? u : 0] = load_unit<T, E, kWide>(static_cast<const T *>(p.gate) + row * p.gate_stride, at(u), hidden);
    }
  };

  auto work = [&](const Row &r, uint64_t row) __attribute__((always_inline)) {
    float ds[N][E];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) ds[u][e] = p.grad_stream ? (float)r.gs[u][e] : 0.f;
    if (p.grad_normed) {
      const float rms = p.stream_rms[row];
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const V w = of_all(0, u);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float hat = (float)r.s[u][e] * rms, g = (float)r.go[u][e];
          sums[0][u][e] = fmaf(g, hat, sums[0][u][e]);
          sum = fmaf(g * (float)w[e], hat, sum);
        }
      }
      const float mean = row_sum<LANES>(sum, room, turn, wave) * p.share;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const V w = of_all(0, u);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float hat = (float)r.s[u][e] * rms;
          ds[u][e] = fmaf(rms, (float)r.go[u][e] * (float)w[e] - hat * mean, ds[u][e]);
        }
      }
    }
    if (p.grad_residual) {
      R *const to = static_cast<R *>(p.grad_residual) + row * hidden;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = p.scale * ds[u][e];
        store_unit<R, E, kWide>(to, at(u), hidden, v);
      }
    }
    if (kFull) {
      const float rms = p.branch_weight ? p.branch_rms[row] : 1.f;
      if (by_channel || by_token) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
          float v[E];
          V bw, g;
          if (p.branch_weight) bw = of_all(1, u);
          if (by_token)
            g = r.g[by_token ? u : 0];
          else
            g = of_all(2, u);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            v[e] = ds[u][e] * (float)r.b[kFull ? u : 0][e] * rms;
            if (p.branch_weight) v[e] *= (float)bw[e];
            if (!by_token) sums[kSums - 1][u][e] += v[e];
            ds[u][e] *= (float)g[e];
          }
          if (by_token && p.grad_gate) store_unit<T, E, kWide>(static_cast<T *>(p.grad_gate) + row * hidden, at(u), hidden, v);
        }
      }
      if (p.branch_weight) {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const V bw = of_all(1, u);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float hat = (float)r.b[kFull ? u : 0][e] * rms;
            sums[kFull ? 1 : 0][u][e] = fmaf(ds[u][e], hat, sums[kFull ? 1 : 0][u][e]);
            ds[u][e] *= (float)bw[e];
            sum = fmaf(ds[u][e], hat, sum);
          }
        }
        const float mean = row_sum<LANES>(sum, room, turn, wave) * p.share;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) ds[u][e] = rms * (ds[u][e] - (float)r.b[kFull ? u : 0][e] * rms * mean);
      }
    }
    if (p.grad_branch)
#pragma unroll
      for (int u = 0; u < N; ++u) store_unit<T, E, kWide>(static_cast<T *>(p.grad_branch) + row * hidden, at(u), hidden, ds[u]);
  };

  const uint64_t step = (uint64_t)gridDim.x * rows;
  uint64_t row = (uint64_t)blockIdx.x * rows + mine;
  Row even;
  if constexpr (kAhead) {
    Row odd;
    read(even, row);
    for (; row < p.tokens; row += 2 * step) {
      read(odd, row + step);
      work(even, row);
      if (row + step >= p.tokens) break;
      read(even, row + 2 * step);
      work(odd, row + step);
    }
  } else {
#pragma unroll 1
    for (; row < p.tokens; row += step) {
      read(even, row);
      work(even, row);
    }
  }

  if (!p.parts) return;
  float *const parts = p.parts + (uint64_t)blockIdx.x * 3 * hidden;
  // A workgroup's rows meet in LDS first.
  constexpr int kUnit = rows == 1 ? 1 : lanes * E;
  __shared__ float meet[rows][kUnit];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (rows > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) meet[mine % rows][(rows == 1 ? 0 : e * lanes + lane)] = sums[k][u][e];
        __syncthreads();
        if (mine == 0)
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 1; i < rows; ++i) sums[k][u][e] += meet[i][(rows == 1 ? 0 : e * lanes + lane)];
      }
      if (rows == 1 || mine == 0)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at(u) + e < hidden) parts[(uint64_t)k * hidden + at(u) + e] = sums[k][u][e];
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

// ---- launches ----

// Lines of 2^20 workgroups: a launch has less than 2^32 threads along a line.
template <int LANES>
dim3 lines_of(uint64_t tokens) {
  constexpr uint64_t line = 1u << 20;
  const uint64_t all = (tokens + rows_of_block<LANES>() - 1) / rows_of_block<LANES>();
  return dim3((uint32_t)std::min(all, line), (uint32_t)((all + line - 1) / line));
}

// Lanes of a row: of a wave, forward with up to four units a lane, backward with two (its sums take registers), up to
// eight waves; and 16 or 32 where one unit a lane of those is enough, as for the heads of queries and keys (100000 rows of
// 128 forward 11 us against 24 with a wave for each, 500000 of 64 29 against 102).
inline int lanes_of(uint64_t hidden, bool backward, bool is_wide) {
  if (is_wide && hidden <= 256) return hidden <= 128 ? 16 : 32;
  int waves = 1;
  while (waves < 8 && hidden > (uint64_t)waves * 64 * 8 * (backward ? 2 : 4)) waves *= is_wide ? 2 : 8;
  return waves * 64;
}
// As many as each CU has room for eight waves.
inline uint32_t parts_of(const emrs_norm *a, bool is_wide) {
  const int lanes = lanes_of(a->hidden, true, is_wide), rows = lanes <= 64 ? 256 / lanes : 1;
  return (uint32_t)std::min<uint64_t>(kWavesOfSums * 64 / (lanes * rows), (a->tokens + rows - 1) / rows);
}

template <class T, class R, int LANES, int UNITS, bool kWide>
void launch_forward(const Norm &p, hipStream_t st) {
  norm_forward_kernel<T, R, LANES, UNITS, kWide><<<lines_of<LANES>(p.tokens), threads_of<LANES>(), 0, st>>>(p);
}
template <class T, class R, int LANES, int UNITS, bool kWide>
void launch_backward(const Norm &p, bool full, uint32_t blocks, hipStream_t st) {
  if (p.gate_kind == EMRS_NORM_GATE_TOKEN)
    norm_backward_kernel<T, R, LANES, UNITS, kWide, kToken><<<blocks, threads_of<LANES>(), 0, st>>>(p);
  else if (full)
    norm_backward_kernel<T, R, LANES, UNITS, kWide, kShared><<<blocks, threads_of<LANES>(), 0, st>>>(p);
  else
    norm_backward_kernel<T, R, LANES, UNITS, kWide, kPlain><<<blocks, threads_of<LANES>(), 0, st>>>(p);
}

// Rows off their units have two shapes: their accesses by elements bound them anyway.
template <class T, class R>
void launch(const Norm &p, bool backward, bool full, bool is_wide, uint32_t blocks, hipStream_t st) {
  const int lanes = lanes_of(p.hidden, backward, is_wide), units = (p.hidden + 511) / 512;
  if (!is_wide) {
    if (lanes == 64) return backward ? launch_backward<T, R, 64, 2, false>(p, full, blocks, st) : launch_forward<T, R, 64, 4, false>(p, st);
    return backward ? launch_backward<T, R, 512, 4, false>(p, full, blocks, st) : launch_forward<T, R, 512, 4, false>(p, st);
  }
  if (backward) {
    if (lanes == 16) return launch_backward<T, R, 16, 1, true>(p, full, blocks, st);
    if (lanes == 32) return launch_backward<T, R, 32, 1, true>(p, full, blocks, st);
    if (units <= 1) return launch_backward<T, R, 64, 1, true>(p, full, blocks, st);
    if (lanes == 64) return launch_backward<T, R, 64, 2, true>(p, full, blocks, st);
    if (lanes == 128) return launch_backward<T, R, 128, 2, true>(p, full, blocks, st);
    if (lanes == 256) return launch_backward<T, R, 256, 2, true>(p, full, blocks, st);
    if (units <= 16) return launch_backward<T, R, 512, 2, true>(p, full, blocks, st);
    return launch_backward<T, R, 512, 4, true>(p, full, blocks, st);
  }
  if (lanes == 16) return launch_forward<T, R, 16, 1, true>(p, st);
  if (lanes == 32) return launch_forward<T, R, 32, 1, true>(p, st);
  if (units <= 1) return launch_forward<T, R, 64, 1, true>(p, st);
  if (units <= 2) return launch_forward<T, R, 64, 2, true>(p, st);
  if (lanes == 64) return launch_forward<T, R, 64, 4, true>(p, st);
  if (lanes == 128) return launch_forward<T, R, 128, 4, true>(p, st);
  if (lanes == 256) return launch_forward<T, R, 256, 4, true>(p, st);
  return launch_forward<T, R, 512, 4, true>(p, st);
}

// The sums over tokens that were wanted.
template <class T>
void launch_sums(const Norm &p, bool full, uint32_t parts, void *weight, void *branch_weight, void *gate, hipStream_t st) {
  const dim3 grid((uint32_t)((p.hidden + kSumColumns - 1) / kSumColumns), full ? 3 : 1);
  sum_parts_kernel<<<grid, kSumColumns * kSumRows, 0, st>>>(p.parts, parts, p.hidden, static_cast<T *>(weight), static_cast<T *>(branch_weight),
                                                            static_cast<T *>(gate));
}

}  // namespace emrs_norm_kernels

// Each in a source of its own, so that they compile side by side.
namespace emrs_internal {
void norm_bf16(const emrs_norm_kernels::Norm &p, bool wide_stream, bool backward, bool full, bool is_wide, uint32_t blocks, hipStream_t st);
void norm_fp16(const emrs_norm_kernels::Norm &p, bool wide_stream, bool backward, bool full, bool is_wide, uint32_t blocks, hipStream_t st);
}  // namespace emrs_internal

#endif
