// Cross entropy over a large vocabulary from the output layer's weight, without keeping the logits.
//
// With x_tv = h_t . w_v:  lse_t = log sum_v exp(x_tv),  loss_t = lse_t - x_t,target.
// Forward: one product per vocabulary shard, whose epilogue reduces its tile of x in registers to a
// maximum and a sum of exponentials for each token (and picks out the target's x); a second kernel joins
// the tiles' pairs.  Nothing of size tokens x vocabulary is written.
// Backward: x is computed again, a piece of the vocabulary at a time.  The product's epilogue turns it into
// d_tv = g_t (exp(x_tv - lse_t) - [v = target_t]) in the operands' type, in both orientations, and two
// products read that: grad_h = d w (summed over the pieces in 32 bits) and grad_w = d^T h.
//
// d is rounded to 16 bits because it is an operand of the matrix instructions, as the gradients that it
// makes are; in fp16 it is scaled first, so that the gradient weight of a long batch does not underflow.

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

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kPieceBytes = 64ull << 20;  // of d in one orientation: both, and what reads them, stay near the caches

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// ---- forward ----

// Reduces a tile of x (m: vocabulary rows, n: tokens) to one (maximum, sum) pair per token and wave row.
struct TileStatistics {
  float2 *pairs;          // [slots][tokens]
  float *target_logit;    // [tokens]
  const int64_t *target;
  int64_t first;          // vocabulary index of m = 0
  int32_t valid;          // rows m < valid count

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int wm, int lane, const Product &p) const {
    const int64_t slot = (int64_t)(w.m0 / Cfg::BM) * Cfg::WAVES_M + wm;
    const int m = m0 + (lane >> 4) * 4;
    if (m0 + Cfg::WM > valid) {
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m + i * 16 + r >= valid)
#pragma unroll
            for (int j = 0; j < Cfg::NI; ++j) acc[i][j][r] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      const int t = n0 + j * 16 + (lane & 15);
      const bool in = t < p.n;
      const int64_t at = (in ? target[t] : -1) - first - m;  // among this lane's rows: 16 i + r
      if (__any(at >= 0 && at < Cfg::WM && at % 16 < 4)) {
#pragma unroll
        for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (in && at == i * 16 + r && m + i * 16 + r < valid) target_logit[t] = acc[i][j][r];
      }
      float top = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      // No row that counts: the exponentials below are then of -inf, 0.  fmaxf drops NaN; the sum has it.
      const float shift = top == -INFINITY ? 0.f : top * kLog2e;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], kLog2e, -shift));
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (in && lane < 16) pairs[slot * p.n + t] = float2{top, sum};
    }
  }
};

constexpr int kMergeTokens = 16, kMergeThreads = 256;

// Joins the pairs of every tile: one workgroup for 16 tokens, 16 lanes apart over the slots.
__global__ __launch_bounds__(kMergeThreads) void merge_statistics_kernel(const float2 *pairs, int64_t slots, int tokens,
                                                                         const int64_t *target, int64_t ignore, int64_t first,
                                                                         int64_t last, float *lse, float *target_logit,
                                                                         float *loss) {
  __shared__ float2 part[kMergeThreads];
  const int t = blockIdx.x * kMergeTokens + threadIdx.x % kMergeTokens;
  float top = -INFINITY, sum = 0.f;
  if (t < tokens)
    for (int64_t s = threadIdx.x / kMergeTokens; s < slots; s += kMergeThreads / kMergeTokens) {
      const float2 v = pairs[s * tokens + t];
      const float up = fmaxf(top, v.x), shift = up == -INFINITY ? 0.f : up;
      sum = sum * exp_of(top - shift) + v.y * exp_of(v.x - shift);
      top = up;
    }
  part[threadIdx.x] = float2{top, sum};
  __syncthreads();
  if (threadIdx.x >= kMergeTokens || t >= tokens) return;
  for (int i = 1; i < kMergeThreads / kMergeTokens; ++i) {
    const float2 v = part[i * kMergeTokens + threadIdx.x];
    const float up = fmaxf(top, v.x), shift = up == -INFINITY ? 0.f : up;
    sum = sum * exp_of(top - shift) + v.y * exp_of(v.x - shift);
    top = up;
  }
  const float l = (top == -INFINITY ? 0.f : top) + logf(sum);
  const int64_t at = target[t];
  const float x = at >= first && at < last ? target_logit[t] : -INFINITY;
  lse[t] = l;
  target_logit[t] = x;
  if (loss) loss[t] = at == ignore ? 0.f : l - x;
}

// ---- backward ----

// d of a piece, in both orientations, with zeros up to the padded sizes (the next products sum over them).
template <class T>
struct LogitGradients {
  T *d;                   // [tokens][d_stride]: m contiguous
  T *dt;                  // [rows][dt_stride]: n contiguous
  int32_t d_stride, dt_stride;
  const float *lse, *grad_loss;
  const int64_t *target;
  int64_t ignore, first;
  int32_t valid;
  const float *scale;     // fp16: what d is multiplied by; NULL: 1

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &, int m0, int n0, int, int lane, const Product &p) const {
    using x4 = typename emrs_gemm::Vec<T>::x4;
    const int m = m0 + (lane >> 4) * 4;
    const float by = scale ? scale[0] : 1.f;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      const int t = n0 + j * 16 + (lane & 15);
      const bool in = t < p.n;
      const int64_t label = in ? target[t] : ignore;
      const bool counts = label != ignore;
      const int64_t at = label - first;
      const float g = counts ? grad_loss[t] * by : 0.f, l = counts ? lse[t] : 0.f;
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int v = m + i * 16;
        x4 out;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = exp_of(acc[i][j][r] - l) - (v + r == at ? 1.f : 0.f);
          out[r] = (T)(counts && v + r < valid ? e * g : 0.f);
          if (dt && v + r < p.m && t < dt_stride) dt[(int64_t)(v + r) * dt_stride + t] = out[r];
        }
        if (d && in && v < d_stride) *reinterpret_cast<x4 *>(d + (int64_t)t * d_stride + v) = out;
      }
    }
  }
};

// C as 16-bit rows out[n][m], scaled; `sum` (32 bits, same layout) carries a sum over several products.
template <class T>
struct StoreRows {
  T *out;                 // NULL: only the running sum is kept
  float *sum;             // NULL: C alone
  int32_t add;            // the sum holds a value already
  int64_t stride;         // elements between rows of out and of sum
  int32_t wide;           // four elements can be stored at once
  const float *scale;     // what C is divided by; NULL: 1

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &, int m0, int n0, int, int lane, const Product &p) const {
    using x4 = typename emrs_gemm::Vec<T>::x4;
    const int m = m0 + (lane >> 4) * 4;
    const float by = scale ? 1.f / scale[0] : 1.f;  // a power of two
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      const int n = n0 + j * 16 + (lane & 15);
      if (n >= p.n) continue;
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int at = m + i * 16;
        if (at >= p.m) continue;
        const int64_t o = (int64_t)n * stride + at;
        f32x4 c = acc[i][j];
        if (wide) {
          if (sum) {
            if (add) c += *reinterpret_cast<const f32x4 *>(sum + o);
            if (!out) *reinterpret_cast<f32x4 *>(sum + o) = c;
          }
          if (out) {
            x4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (T)(c[r] * by);
            *reinterpret_cast<x4 *>(out + o) = v;
          }
          continue;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (at + r >= p.m) continue;
          float v = c[r];
          if (sum) {
            if (add) v += sum[o + r];
            if (!out) sum[o + r] = v;
          }
          if (out) out[o + r] = (T)(v * by);
        }
      }
    }
  }
};

// A power of two that brings the largest |grad_loss| to 2^15: fp16 then keeps d of probabilities down to
// 2^-29 of it out of the subnormals.  1 where there is nothing to scale.
__global__ __launch_bounds__(1024) void gradient_scale_kernel(const float *grad_loss, const int64_t *target, int64_t ignore,
                                                             int tokens, float *scale) {
  __shared__ float part[16];
  float top = 0.f;
  for (int t = threadIdx.x; t < tokens; t += 1024)
    if (target[t] != ignore) top = fmaxf(top, fabsf(grad_loss[t]));
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, part[i]);
  int e = 0;
  if (top > 0.f && top < INFINITY) frexpf(top, &e);  // top <= 2^e
  scale[0] = ldexpf(1.f, min(max(15 - e, -100), 100));
}

// ---- operands in the layout that the products read ----

constexpr int kSide = 64;

// out[c][r] = in[r][c] for r < rows and c < cols, with zeros up to `padded` r and where keep says so.
template <class T>
__global__ __launch_bounds__(256) void transpose_kernel(const T *in, int64_t in_stride, int rows, int cols, T *out,
                                                        int64_t out_stride, int padded, const int64_t *target, int64_t ignore) {
  __shared__ T tile[kSide][kSide + 2];
  const int r0 = blockIdx.x * kSide, c0 = blockIdx.y * kSide;
  const int x = threadIdx.x % kSide;
  for (int y = threadIdx.x / kSide; y < kSide; y += 256 / kSide) {
    const int r = r0 + y, c = c0 + x;
    const bool keep = r < rows && c < cols && !(target && target[r] == ignore);
    tile[y][x] = keep ? in[(int64_t)r * in_stride + c] : (T)0.f;
  }
  __syncthreads();
  for (int y = threadIdx.x / kSide; y < kSide; y += 256 / kSide) {
    const int c = c0 + y, r = r0 + x;
    if (c < cols && r < padded) out[(int64_t)c * out_stride + r] = tile[x][y];
  }
}

// out[r][c] = in[r][c], with zeros from `cols` up to the padded row: operands whose rows do not lie on 16 bytes.
template <class T>
__global__ __launch_bounds__(256) void pad_kernel(const T *in, int64_t in_stride, int cols, T *out, int64_t out_stride) {
  const int64_t r = blockIdx.x;
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c < out_stride) out[r * out_stride + c] = c < cols ? in[r * in_stride + c] : (T)0.f;
}

bool on_16(const void *p, uint64_t stride, uint64_t k) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && k % 8 == 0;
}

// Where the workspace's parts lie, and how the vocabulary is cut.
struct Sizes {
  uint64_t k;              // the hidden size, padded where an operand is copied
  bool pad_hidden, pad_weight;
  uint64_t piece;          // vocabulary rows that are worked on at once
  uint64_t tokens_padded;
  uint64_t pairs, hidden, weight, sum, d, dt, ht, wt, scale, total;  // offsets
};

int check(const emrs_loss *a) {
  if (!a) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: NULL argument");
  if (a->dtype != EMRS_BF16 && a->dtype != EMRS_FP16) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: bf16 or fp16 wanted");
  if (a->n_shards == 0 || a->n_shards > EMRS_LOSS_MAX_SHARDS)
    return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: 1 to 64 vocabulary shards wanted");
  if (!a->weights || !a->weight_strides || !a->shard_rows)
    return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: NULL shard table");
  // Row offsets inside a tile, and element offsets inside a row, are 32-bit byte offsets.
  constexpr uint64_t most_columns = 1u << 20, most_rows = 1u << 30, most_tokens = 1u << 21, most_stride = 1u << 21;
  if (a->hidden_size == 0 || a->hidden_size > most_columns) return fail(EMRS_ERR_TOO_LARGE, "loss: hidden size 1 to 2^20 wanted");
  if (a->tokens > most_tokens) return fail(EMRS_ERR_TOO_LARGE, "loss: at most 2^21 tokens");
  if (a->tokens > 1 && (a->hidden_stride < a->hidden_size || a->hidden_stride > most_stride))
    return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: hidden rows overlap, or lie over 2^21 elements apart");
  if (a->tokens && (!a->hidden || !a->target)) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: NULL hidden states or targets");
  if (reinterpret_cast<uintptr_t>(a->hidden) % 2 || reinterpret_cast<uintptr_t>(a->target) % 8)
    return fail(EMRS_ERR_MISALIGNED, "loss: hidden states or targets off their type's alignment");
  for (uint32_t s = 0; s < a->n_shards; ++s) {
    if (!a->weights[s] && a->shard_rows[s]) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: NULL shard");
    if (reinterpret_cast<uintptr_t>(a->weights[s]) % 2) return fail(EMRS_ERR_MISALIGNED, "loss: a shard off its type's alignment");
    if (a->shard_rows[s] > most_rows) return fail(EMRS_ERR_TOO_LARGE, "loss: at most 2^30 rows a shard");
    if (a->shard_rows[s] > 1 && (a->weight_strides[s] < a->hidden_size || a->weight_strides[s] > most_stride))
      return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: a shard's rows overlap, or lie over 2^21 elements apart");
  }
  return EMRS_OK;
}

Sizes sizes_of(const emrs_loss *a, bool backward) {
  Sizes s{};
  uint64_t most = 0, slots = 0;
  s.pad_hidden = !on_16(a->hidden, a->tokens > 1 ? a->hidden_stride : 8, a->hidden_size);
  for (uint32_t i = 0; i < a->n_shards; ++i) {
    most = std::max(most, a->shard_rows[i]);
    s.pad_weight |= !on_16(a->weights[i], a->shard_rows[i] > 1 ? a->weight_strides[i] : 8, a->hidden_size);
  }
  s.k = a->hidden_size % 8 ? round_up(a->hidden_size, 64) : a->hidden_size;
  s.tokens_padded = round_up(std::max<uint64_t>(a->tokens, 1), 64);
  s.piece = round_up(std::max<uint64_t>(most, 1), 256);
  if (backward || s.pad_weight)
    s.piece = std::min(s.piece, std::max<uint64_t>(kPieceBytes / 2 / s.tokens_padded / 256, 4) * 256);
  for (uint32_t i = 0; i < a->n_shards; ++i)
    for (uint64_t lo = 0; lo < a->shard_rows[i]; lo += s.piece) {
      Product p{};
      p.m = std::min(s.piece, a->shard_rows[i] - lo), p.n = a->tokens, p.batch = 1;
      slots += emrs_gemm::wave_rows(p);
    }
  uint64_t at = 0;
  auto take = [&](bool wanted, uint64_t bytes) {
    const uint64_t here = at;
    if (wanted) at += round_up(bytes, 256);
    return here;
  };
  s.pairs = take(!backward, slots * a->tokens * sizeof(float2));
  s.hidden = take(s.pad_hidden, a->tokens * s.k * 2);
  s.weight = take(s.pad_weight, s.piece * s.k * 2);
  s.sum = take(backward && a->grad_hidden, a->tokens * a->hidden_size * 4);
  s.d = take(backward && a->grad_hidden, a->tokens * s.piece * 2);
  s.wt = take(backward && a->grad_hidden, a->hidden_size * s.piece * 2);
  s.dt = take(backward && a->grad_weights, s.piece * s.tokens_padded * 2);
  s.ht = take(backward && a->grad_weights, a->hidden_size * s.tokens_padded * 2);
  s.scale = take(backward, 256);
  s.total = at;
  return s;
}

#define TRY(expr)                                                                                       \
  do {                                                                                                  \
    const hipError_t e_ = (expr);                                                                       \
    if (e_ != hipSuccess) return fail(EMRS_ERR_HIP, std::string("loss: ") + hipGetErrorString(e_));     \
  } while (0)

// The operands of one piece: its weight rows, copied into padded rows where they do not lie on 16 bytes.
template <class T>
int piece_operands(const emrs_loss *a, const Sizes &s, uint32_t shard, uint64_t lo, uint64_t rows, hipStream_t st, Product *p) {
  char *ws = static_cast<char *>(a->workspace);
  const T *w = static_cast<const T *>(a->weights[shard]) + lo * a->weight_strides[shard];
  *p = Product{};
  p->b = s.pad_hidden ? ws + s.hidden : a->hidden;
  p->b_stride = s.pad_hidden ? s.k : a->tokens > 1 ? a->hidden_stride : s.k;
  p->a = w;
  p->a_stride = a->shard_rows[shard] > 1 ? a->weight_strides[shard] : s.k;
  if (s.pad_weight) {
    pad_kernel<T><<<dim3(rows, (s.k + 255) / 256), 256, 0, st>>>(w, a->weight_strides[shard], a->hidden_size,
                                                                 reinterpret_cast<T *>(ws + s.weight), s.k);
    TRY(hipGetLastError());
    p->a = ws + s.weight;
    p->a_stride = s.k;
  }
  p->m = rows;
  p->n = a->tokens;
  p->k = s.k;
  p->batch = 1;
  p->a_wrap = p->b_wrap = emrs_gemm::kNoWrap;
  return EMRS_OK;
}

template <class T>
int pad_hidden(const emrs_loss *a, const Sizes &s, hipStream_t st) {
  if (!s.pad_hidden) return EMRS_OK;
  pad_kernel<T><<<dim3(a->tokens, (s.k + 255) / 256), 256, 0, st>>>(static_cast<const T *>(a->hidden), a->hidden_stride, a->hidden_size,
                                                                    reinterpret_cast<T *>(static_cast<char *>(a->workspace) + s.hidden), s.k);
  TRY(hipGetLastError());
  return EMRS_OK;
}

int32_t valid_rows(const emrs_loss *a, uint64_t first, uint64_t rows) {
  return (int32_t)(a->vocab_size <= first ? 0 : std::min(rows, a->vocab_size - first));
}

template <class T>
int forward(const emrs_loss *a, hipStream_t st) {
  const Sizes s = sizes_of(a, false);
  char *ws = static_cast<char *>(a->workspace);
  float2 *pairs = reinterpret_cast<float2 *>(ws + s.pairs);
  int rc = pad_hidden<T>(a, s, st);
  if (rc) return rc;
  uint64_t first = a->vocab_start;
  int64_t slots = 0;
  for (uint32_t i = 0; i < a->n_shards; first += a->shard_rows[i], ++i)
    for (uint64_t lo = 0; lo < a->shard_rows[i]; lo += s.piece) {
      const uint64_t rows = std::min(s.piece, a->shard_rows[i] - lo);
      Product p;
      rc = piece_operands<T>(a, s, i, lo, rows, st, &p);
      if (rc) return rc;
      const TileStatistics e{pairs + slots * (int64_t)a->tokens, a->target_logit, a->target, (int64_t)(first + lo),
                             valid_rows(a, first + lo, rows)};
      TRY((emrs_gemm::launch<T>(p, e, st)));
      slots += emrs_gemm::wave_rows(p);
    }
  const int64_t last = (int64_t)std::max(a->vocab_start, std::min(first, a->vocab_size));
  merge_statistics_kernel<<<(a->tokens + kMergeTokens - 1) / kMergeTokens, kMergeThreads, 0, st>>>(
      pairs, slots, (int)a->tokens, a->target, a->ignore_index, (int64_t)a->vocab_start, last, a->lse, a->target_logit, a->loss);
  TRY(hipGetLastError());
  return EMRS_OK;
}

template <class T>
int transpose(const T *in, int64_t in_stride, int64_t rows, int64_t cols, T *out, int64_t out_stride, const int64_t *target,
              int64_t ignore, hipStream_t st) {
  const dim3 grid((out_stride + kSide - 1) / kSide, (cols + kSide - 1) / kSide);
  transpose_kernel<T><<<grid, 256, 0, st>>>(in, in_stride, (int)rows, (int)cols, out, out_stride, (int)out_stride, target, ignore);
  TRY(hipGetLastError());
  return EMRS_OK;
}

template <class T>
int backward(const emrs_loss *a, hipStream_t st) {
  const Sizes s = sizes_of(a, true);
  char *ws = static_cast<char *>(a->workspace);
  T *d = reinterpret_cast<T *>(ws + s.d), *wt = reinterpret_cast<T *>(ws + s.wt);
  T *dt = reinterpret_cast<T *>(ws + s.dt), *ht = reinterpret_cast<T *>(ws + s.ht);
  float *sum = reinterpret_cast<float *>(ws + s.sum), *scale = nullptr;
  int rc = pad_hidden<T>(a, s, st);
  if (rc) return rc;
  if (a->dtype == EMRS_FP16) {
    scale = reinterpret_cast<float *>(ws + s.scale);
    gradient_scale_kernel<<<1, 1024, 0, st>>>(a->grad_loss, a->target, a->ignore_index, (int)a->tokens, scale);
    TRY(hipGetLastError());
  }
  if (a->grad_weights) {
    rc = transpose<T>(static_cast<const T *>(a->hidden), a->hidden_stride, a->tokens, a->hidden_size, ht, s.tokens_padded, a->target,
                      a->ignore_index, st);
    if (rc) return rc;
  }
  uint64_t first = a->vocab_start, left = 0;
  for (uint32_t i = 0; i < a->n_shards; ++i) left += (a->shard_rows[i] + s.piece - 1) / s.piece;
  bool begun = false;
  for (uint32_t i = 0; i < a->n_shards; first += a->shard_rows[i], ++i)
    for (uint64_t lo = 0; lo < a->shard_rows[i]; lo += s.piece) {
      const uint64_t rows = std::min(s.piece, a->shard_rows[i] - lo), padded = round_up(rows, 64);
      T *gw = a->grad_weights ? static_cast<T *>(a->grad_weights[i]) : nullptr;
      const int32_t valid = valid_rows(a, first + lo, rows);
      --left;
      Product p;
      rc = piece_operands<T>(a, s, i, lo, rows, st, &p);
      if (rc) return rc;
      if (!a->grad_hidden && !gw) continue;
      const LogitGradients<T> e{a->grad_hidden ? d : nullptr, gw ? dt : nullptr, (int32_t)padded, (int32_t)s.tokens_padded,
                                a->lse, a->grad_loss, a->target, a->ignore_index, (int64_t)(first + lo), valid, scale};
      TRY((emrs_gemm::launch<T>(p, e, st)));
      const bool wide = a->hidden_size % 4 == 0;
      if (a->grad_hidden) {
        rc = transpose<T>(static_cast<const T *>(a->weights[i]) + lo * a->weight_strides[i], a->weight_strides[i], valid,
                          a->hidden_size, wt, padded, nullptr, 0, st);
        if (rc) return rc;
        Product q{};
        q.a = wt, q.b = d;
        q.a_stride = q.b_stride = padded;
        q.m = a->hidden_size, q.n = a->tokens, q.k = padded;
        q.batch = 1;
        q.a_wrap = q.b_wrap = emrs_gemm::kNoWrap;
        const StoreRows<T> out{left ? nullptr : static_cast<T *>(a->grad_hidden), left || begun ? sum : nullptr, begun,
                               (int64_t)a->hidden_size, wide && reinterpret_cast<uintptr_t>(a->grad_hidden) % 8 == 0, scale};
        TRY((emrs_gemm::launch<T>(q, out, st)));
        begun = true;
      }
      if (gw) {
        Product q{};
        q.a = ht, q.b = dt;
        q.a_stride = q.b_stride = s.tokens_padded;
        q.m = a->hidden_size, q.n = rows, q.k = s.tokens_padded;
        q.batch = 1;
        q.a_wrap = q.b_wrap = emrs_gemm::kNoWrap;
        const StoreRows<T> out{gw + lo * a->hidden_size, nullptr, 0, (int64_t)a->hidden_size,
                               wide && reinterpret_cast<uintptr_t>(gw) % 8 == 0, scale};
        TRY((emrs_gemm::launch<T>(q, out, st)));
      }
    }
  return EMRS_OK;
}

int check_workspace(const emrs_loss *a, bool backward) {
  const Sizes s = sizes_of(a, backward);
  if (s.total && (!a->workspace || a->workspace_bytes < s.total))
    return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: the workspace holds " + std::to_string(a->workspace_bytes) + " bytes of " +
                                               std::to_string(s.total));
  if (reinterpret_cast<uintptr_t>(a->workspace) % 256) return fail(EMRS_ERR_MISALIGNED, "loss: the workspace is off 256 bytes");
  return EMRS_OK;
}

}  // namespace

extern "C" {

int emrs_loss_workspace(const emrs_loss *a, int backward, uint64_t *bytes) {
  emrs_internal::clear_error();
  const int rc = check(a);
  if (rc) return rc;
  if (!bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: NULL argument");
  *bytes = sizes_of(a, backward != 0).total;
  return EMRS_OK;
}

int emrs_loss_forward(const emrs_loss *a, void *stream) {
  emrs_internal::clear_error();
  int rc = check(a);
  if (rc) return rc;
  if (a->tokens == 0) return EMRS_OK;
  if (!a->lse || !a->target_logit) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: forward wants lse and target_logit");
  rc = check_workspace(a, false);
  if (rc) return rc;
  rc = emrs_internal::need_device();
  if (rc) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == EMRS_BF16 ? forward<__bf16>(a, st) : forward<_Float16>(a, st);
}

int emrs_loss_backward(const emrs_loss *a, void *stream) {
  emrs_internal::clear_error();
  int rc = check(a);
  if (rc) return rc;
  if (a->tokens && (!a->lse || !a->grad_loss)) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: backward wants lse and grad_loss");
  uint64_t rows = 0;
  for (uint32_t i = 0; i < a->n_shards; ++i) rows += a->shard_rows[i];
  if (a->tokens == 0 || rows == 0)
    return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: no tokens or no vocabulary rows: the gradients are zeros, which the caller fills");
  rc = check_workspace(a, true);
  if (rc) return rc;
  rc = emrs_internal::need_device();
  if (rc) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == EMRS_BF16 ? backward<__bf16>(a, st) : backward<_Float16>(a, st);
}

}  // extern "C"
