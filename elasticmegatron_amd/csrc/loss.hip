// Cross entropy over a large vocabulary from the output layer's weight, without keeping the logits.
//
// With x_tv = h_t . w_v:  lse_t = log sum_v exp(x_tv),  loss_t = lse_t - x_t,target.
// Forward: one product per vocabulary shard, whose epilogue reduces its tile of x in registers to a
// maximum and a sum of exponentials for each token (and picks out the target's x); a second kernel joins
// the tiles' pairs.  Nothing of size tokens x vocabulary is written.
// Backward: x is computed again, a piece of the vocabulary at a time.  The product's epilogue turns it into
// d_tv = g_t (exp(x_tv - lse_t) - [v = target_t]), in both orientations, and two products read that:
// grad_h = d w (summed over the pieces in 32 bits) and grad_w = d^T h.
//
// d is an operand of the matrix instructions, and so rounded to 16 bits: to fp16, whose 11 bits leave the
// gradients with the rounding of their own type alone (in bf16, d's rounding would be as large as theirs).
// fp16's range is met by powers of two: each token's d is scaled by its own |g|, and copies of w and h, which the
// products want transposed anyway, by their largest entry; bf16's 8 bits lose nothing in them.  grad_h takes a
// token's scale off its row.  grad_w sums over tokens: h carries there what a token's |g| is below the largest, so
// that h's entries keep all bits down to 2^-27 of the largest |g| times the largest |h|, and below 2^-38 are lost.
// So do d's: where a probability is below 2^-27 bits of it are lost, and below 2^-38 all.
//
// Equal vocabulary shards (those of tensor parallelism are) go through every kernel together, as a batch.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "emrs.h"
#include "gemm.h"
#include "internal.h"

namespace {

using emrs_gemm::f32x4;
using emrs_gemm::Product;
using emrs_gemm::Where;
using emrs_internal::fail;

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kPieceBytes = 128ull << 20;  // of d in one orientation
// Of a copy of weights, transposed or padded: with few tokens a piece of d would let it be the whole weight
// (128256 x 4096, 512 tokens: 1321 MiB of workspace; bounded to this 388, and 2614 us against 2350; to half of it
// 180 and 3080).
constexpr uint64_t kCopyBytes = 256ull << 20;

// Whether grad_hidden's product takes the weights as they lie: no search of their largest entry, no transposed
// copy, but smaller tiles, and for bf16 twice the rows of d, in two parts.  What both read and compute grows alike
// with rows and hidden size, so that tokens decide.  All gradients, this against the other, us:
//   bf16       64 tokens   256          512          1024            fp16  256 tokens   512          1024
//   32000 x 512     69/76    102/100      123/113      208/165              89/95        102/109      161/163
//   8000 x 4096     86/108   141/152      192/178      342/259             132/140       157/169      246/253
//   32000 x 4096   253/423   486/559      698/641     1220/950             399/504       543/589      902/896
//   128256 x 4096  914/1744 1550/2278    2578/2594    4781/3789           1259/2035     1961/2361    3507/3584
//   32000 x 8192   510/866   890/1104    1316/1384    2351/1832            746/982      1010/1270    1745/1725
bool takes_weights(uint32_t dtype, uint64_t tokens) { return tokens <= (dtype == EMRS_BF16 ? 256 : 768); }

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

using half = _Float16;
using half4 = emrs_gemm::Vec<_Float16>::x4;

struct Table {
  const void *p[EMRS_LOSS_MAX_SHARDS];
};

// A piece of the vocabulary: the same `rows` rows of every shard of a group.
struct Piece {
  static constexpr bool kRowsOfK = false, kBy32 = true;
  Table weights;          // first row of the piece in each shard
  int64_t first, shard;   // vocabulary index of the first shard's first row here; rows from a shard to the next
  int64_t vocab;          // rows from this vocabulary index on do not count

  __device__ __forceinline__ const void *operand_a(const Product &, int batch) const { return weights.p[batch]; }
  __device__ __forceinline__ const void *operand_b(const Product &p, int batch) const { return emrs_gemm::Operand{}.operand_b(p, batch); }
  __host__ __device__ int64_t first_of(int batch) const { return first + batch * shard; }
  __device__ __forceinline__ int valid(int batch, int rows) const {
    return (int)min((int64_t)rows, max((int64_t)0, vocab - first_of(batch)));
  }
};

// ---- forward ----

// Reduces a tile of x (m: vocabulary rows, n: tokens) to one (maximum, sum) pair per token and wave row: of
// 128 logits of a token in a large tile 8 bytes are left.
struct TileStatistics : Piece {
  float2 *pairs;          // [batch x slots][tokens]
  float *target_logit;    // [tokens]
  const int64_t *target;
  int64_t slots;          // of one shard

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int wm, int lane, const Product &p, char *) const {
    const int64_t slot = w.batch * slots + (int64_t)(w.m0 / Cfg::BM) * Cfg::WAVES_M + wm, first = first_of(w.batch);
    const int valid = this->valid(w.batch, p.m);
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

// ---- forward, one token ----
//
// The weight's bytes bound the call, and vector arithmetic keeps up with one token (with two it does not: 55 us
// against the tiles' 51 on 32000 rows of 4096).  A workgroup reads 32 rows of a shard, eight at a time, each in
// whole consecutive kilobytes, the order that memory serves fastest: 6.2 TB/s on 128256 rows of 4096 (tiles:
// 4.6; a wave's 16 rows straight into fragments: 3.7).  Every thread multiplies 8 of each 2048 k for all eight
// rows; the 256 partial sums of a row meet in LDS.

constexpr int kOneRows = 32, kOneAtOnce = 8, kOneThreads = 256;

template <class T>
__global__ __launch_bounds__(kOneThreads) void one_token_kernel(Piece piece, int64_t stride, int rows, const T *hidden, int k, float2 *pairs,
                                                                float *target_logit, const int64_t *target) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  constexpr int lanes = kOneThreads / kOneAtOnce;  // threads that add one row's parts
  __shared__ float part[kOneAtOnce][kOneThreads];
  __shared__ float x[kOneRows];
  const int m0 = blockIdx.x * kOneRows, batch = blockIdx.y, tid = threadIdx.x;
  const T *const w = static_cast<const T *>(piece.weights.p[batch]);
#pragma unroll 1
  for (int pass = 0; pass < kOneRows; pass += kOneAtOnce) {
    float acc[kOneAtOnce];
#pragma unroll
    for (int i = 0; i < kOneAtOnce; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int at = tid * 8; at < k; at += kOneThreads * 8) {
      x8 a[kOneAtOnce];  // rows past the last one read it again, and are left out below
#pragma unroll
      for (int i = 0; i < kOneAtOnce; ++i)
        a[i] = __builtin_nontemporal_load(reinterpret_cast<const x8 *>(w + min(m0 + pass + i, rows - 1) * stride + at));
      const x8 b = *reinterpret_cast<const x8 *>(hidden + at);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < kOneAtOnce; ++i) acc[i] = fmaf((float)a[i][e], (float)b[e], acc[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOneAtOnce; ++i) part[i][tid] = acc[i];
    __syncthreads();
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kOneThreads / lanes; ++i) v += part[tid / lanes][tid % lanes + i * lanes];
#pragma unroll
    for (int o = lanes / 2; o; o /= 2) v += __shfl_xor(v, o);
    if (tid % lanes == 0) x[pass + tid / lanes] = v;
  }
  __syncthreads();
  if (tid >= kOneRows) return;
  const int valid = piece.valid(batch, rows);
  const int64_t at = target[0] - piece.first_of(batch) - m0;
  if (m0 + tid < valid && at == tid) target_logit[0] = x[tid];
  const float own = m0 + tid < valid ? x[tid] : -INFINITY;
  float top = own;
  for (int o = kOneRows / 2; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
  float sum = exp_of(own - (top == -INFINITY ? 0.f : top));
  for (int o = kOneRows / 2; o; o /= 2) sum += __shfl_xor(sum, o);
  if (tid == 0) pairs[(int64_t)batch * gridDim.x + blockIdx.x] = float2{top, sum};
}

// Joins the pairs of every tile: a workgroup for kTokens tokens, the lanes of one token spread over the
// slots, four of them at once.
constexpr int kMergeThreads = 256;

__device__ inline void join_pair(float &top, float &sum, float2 v) {
  const float up = fmaxf(top, v.x), shift = up == -INFINITY ? 0.f : up;
  sum = sum * exp_of(top - shift) + v.y * exp_of(v.x - shift);
  top = up;
}

template <int kTokens>
__global__ __launch_bounds__(kMergeThreads) void merge_statistics_kernel(const float2 *pairs, int64_t slots, int tokens,
                                                                         const int64_t *target, int64_t ignore, int64_t first,
                                                                         int64_t last, float *lse, float *target_logit,
                                                                         float *loss) {
  constexpr int lanes = kMergeThreads / kTokens;
  __shared__ float2 part[kMergeThreads];
  const int t = blockIdx.x * kTokens + threadIdx.x % kTokens;
  float top = -INFINITY, sum = 0.f;
  if (t < tokens)
    for (int64_t s = threadIdx.x / kTokens; s < slots; s += 4 * lanes) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = s + i * lanes < slots ? pairs[(s + i * lanes) * tokens + t] : float2{-INFINITY, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) join_pair(top, sum, v[i]);
    }
  part[threadIdx.x] = float2{top, sum};
  for (int half = lanes / 2; half; half /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < half * kTokens) {
      join_pair(top, sum, part[threadIdx.x + half * kTokens]);
      part[threadIdx.x] = float2{top, sum};
    }
  }
  if (threadIdx.x >= kTokens || t >= tokens) return;
  const float l = (top == -INFINITY ? 0.f : top) + logf(sum);
  const int64_t at = target[t];
  const float x = at >= first && at < last ? target_logit[t] : -INFINITY;
  lse[t] = l;
  target_logit[t] = x;
  if (loss) loss[t] = at == ignore ? 0.f : l - x;
}

// ---- backward ----

// Of a scale, a power of two; NULL: 1.
__device__ inline int exponent_of(const float *scale) { return scale ? __builtin_amdgcn_frexp_expf(scale[0]) - 1 : 0; }

// The power of two that brings |x| to [2^13, 2^14); `otherwise` for 0 and for what is not finite.
__device__ inline int exponent_for(float x, int otherwise) {
  x = fabsf(x);
  return x > 0.f && x < INFINITY ? min(max(14 - __builtin_amdgcn_frexp_expf(x), -120), 120) : otherwise;
}

__device__ inline float scale_of(float top) { return __builtin_amdgcn_ldexpf(1.f, exponent_for(top, 14)); }

// d of a piece, in both orientations, with zeros up to the padded sizes (the next products sum over them).  Its
// 512 KB a large tile of exponentials and stores are what it is slower by than the statistics.
// With kParts d is in two bf16 parts, [2][tokens]: what the product with bf16 weights as they lie takes.
template <bool kParts>
struct LogitGradients : Piece {
  static constexpr bool kBy32 = false;  // writes zeros up to multiples of 64
  half *d;                // [tokens][shards x padded rows]: m contiguous; NULL: not wanted
  half *dt;               // [shards x padded rows][padded tokens]: n contiguous; NULL: not wanted
  int32_t d_stride, dt_stride, padded;
  const float *lse, *grad_loss;
  const int64_t *target;
  int64_t ignore;
  const float *scale;     // of the largest |grad_loss|

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    const int m = m0 + (lane >> 4) * 4, valid = this->valid(w.batch, p.m);
    const int64_t first = first_of(w.batch);
    const int largest = exponent_of(scale);
    using Turn = emrs_gemm::Turn<Cfg>;
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      const int t = n0 + j * 16 + (lane & 15);
      const int64_t label = t < p.n ? target[t] : ignore;
      const bool counts = label != ignore;
      const int64_t at = label - first;
      const float weight = counts ? grad_loss[t] : 0.f, g = __builtin_amdgcn_ldexpf(weight, exponent_for(weight, largest)), l = counts ? lse[t] * kLog2e : 0.f;
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int v = m + i * 16;
        half4 out;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], kLog2e, -l)) - (v + r == at ? 1.f : 0.f);
          acc[i][j][r] = counts && v + r < valid ? e * g : 0.f;
          out[r] = (half)acc[i][j][r];
        }
        Turn::put(own, i, j, lane, out);
      }
    }
    // From a wave's corner on, offsets are 32 bits: 256 rows of 2^22 elements at most.
    auto rows = [&](half *to) __attribute__((always_inline)) {
      Turn::along_m(own, lane, [&](int x, int t, emrs_gemm::fp16x8 v) __attribute__((always_inline)) {
        if (m0 + x < padded && n0 + t < p.n) *reinterpret_cast<emrs_gemm::fp16x8 *>(to + (t * d_stride + x)) = v;
      });
    };
    half *const to = d + (int64_t)n0 * d_stride + w.batch * padded + m0;
    if (d && !kParts) rows(to);
    if (dt) {
      half *const to = dt + (int64_t)(w.batch * padded + m0) * dt_stride + n0;
      Turn::along_n(own, lane, [&](int x, int t, emrs_gemm::fp16x8 v) __attribute__((always_inline)) {
        if (m0 + x < padded && n0 + t < dt_stride) *reinterpret_cast<emrs_gemm::fp16x8 *>(to + (x * dt_stride + t)) = v;
      });
    }
    if constexpr (kParts) {
      if (!d) return;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
#pragma unroll
        for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
          for (int i = 0; i < Cfg::MI; ++i) {
            emrs_gemm::Vec<__bf16>::x4 v;
            for (int r = 0; r < 4; ++r) v[r] = (__bf16)acc[i][j][r];
            asm("" : "+v"(v));  // one rounding for the part that is stored and the part that is taken off
            for (int r = 0; r < 4; ++r) acc[i][j][r] -= (float)v[r];
            Turn::put(own, i, j, lane, v);
          }
        rows(to + part * (int64_t)p.n * d_stride);
      }
    }
  }
};

// A product with the weight's own rows as rows of k: of every shard in turn, padded.
template <class Base>
struct OfWeights : Base {
  static constexpr bool kRowsOfK = true, kBy32 = false;
  Piece piece;
  int32_t padded, rows, all;  // of a shard; of all of them, padded

  template <class T>
  __device__ __forceinline__ void rows_from(const Product &p, int k, const T *&first, int &count) const {
    const int shard = k < all ? k / padded : 0, row = k - shard * padded;
    first = static_cast<const T *>(piece.weights.p[shard]) + row * p.a_stride;
    count = k < all ? piece.valid(shard, rows) - row : 0;
  }
};

// What the sums are to be divided by, as a power of two: the scales of both operands, and where row n is a token's
// (or that of its second part), the token's own in place of the largest.
struct Scales {
  const float *a, *b;
  const float *grad_loss;  // NULL: no tokens
  int32_t tokens;

  // Both read once, before a tile's stores.  The product of the scales may be out of range: exponents.
  struct Exponents {
    int a, b;
  };
  __device__ __forceinline__ Exponents exponents() const { return {exponent_of(a), exponent_of(b)}; }
  __device__ __forceinline__ int of(int n, const Exponents &e) const {
    return e.b + (grad_loss ? exponent_for(grad_loss[min(n < tokens ? n : n - tokens, tokens - 1)], e.a) : e.a);
  }
};

// A run of k of each product for itself: C of run b goes to sum[b], in 32 bits and unscaled, on top of what
// an earlier piece left there.
struct StoreSums : emrs_gemm::Operand {
  float *sum;             // [batch][n][stride]
  int64_t stride, batch;
  int32_t add;
  int32_t wide;
  Scales scales;

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    const int m = m0 + (lane >> 4) * 4;
    float *const to = sum + w.batch * batch;
    const auto exponents = scales.exponents();
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      const int n = n0 + j * 16 + (lane & 15), by = scales.of(n, exponents);
      // What lies outside reads the last element inside: with no branch, these loads are on their way together.
      f32x4 before[Cfg::MI];
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) before[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (wide && add)
#pragma unroll
        for (int i = 0; i < Cfg::MI; ++i)
          before[i] = *reinterpret_cast<const f32x4 *>(to + min(n, p.n - 1) * stride + min(m + i * 16, p.m - 4));
      if (n >= p.n) continue;
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int at = m + i * 16;
        if (at >= p.m) continue;
        float *const o = to + n * stride + at;
        f32x4 c = before[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] += __builtin_amdgcn_ldexpf(acc[i][j][r], -by);
        if (wide) {
          *reinterpret_cast<f32x4 *>(o) = c;
          continue;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (at + r < p.m) o[r] = c[r] + (add ? o[r] : 0.f);
      }
    }
  }
};

// C as 16-bit rows out[n][m], on top of a sum of earlier pieces if there is one; through LDS, so that rows are
// stored in whole lines (262 MB of gradients of few tokens: 87 us; with four elements a lane, 104).
template <class T>
struct StoreRows : emrs_gemm::Operand {
  Table out;              // of each matrix of the batch
  const float *sum;       // NULL: C alone (a batch of one)
  int64_t stride;         // elements between rows of out and of sum
  int32_t wide;           // eight elements can be stored at once
  Scales scales;

  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    using x4 = typename emrs_gemm::Vec<T>::x4;
    using Turn = emrs_gemm::Turn<Cfg>;
    const int m = m0 + (lane >> 4) * 4;
    T *const to = static_cast<T *>(const_cast<void *>(out.p[w.batch]));
    const auto exponents = scales.exponents();
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) {
      const int n = n0 + j * 16 + (lane & 15), by = scales.of(n, exponents);
      f32x4 before[Cfg::MI];
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) before[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (wide && sum)
#pragma unroll
        for (int i = 0; i < Cfg::MI; ++i)
          before[i] = *reinterpret_cast<const f32x4 *>(sum + min(n, p.n - 1) * stride + min(m + i * 16, p.m - 4));
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        f32x4 c = before[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] += __builtin_amdgcn_ldexpf(acc[i][j][r], -by);
        if (wide) {
          x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = (T)c[r];
          Turn::put(own, i, j, lane, v);
          continue;
        }
        const int at = m + i * 16;
        const int64_t o = n * stride + at;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n < p.n && at + r < p.m) to[o + r] = (T)(c[r] + (sum ? sum[o + r] : 0.f));
      }
    }
    if (!wide) return;
    T *const corner = to + n0 * stride + m0;
    const int step = (int)stride;  // 256 rows of 2^20 elements at most
    Turn::along_m(own, lane, [&](int x, int y, emrs_gemm::fp16x8 v) __attribute__((always_inline)) {
      if (m0 + x < p.m && n0 + y < p.n) *reinterpret_cast<emrs_gemm::fp16x8 *>(corner + (y * step + x)) = v;
    });
  }
};

// The sum of several sums, as 16 bits: 5.5 us for 16 sums of 500 x 512, most of it the launch.
template <class T>
__global__ __launch_bounds__(256) void join_sums_kernel(const float *sum, int sums, int64_t each, T *out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= each) return;
  float v = sum[i];
  for (int s = 1; s < sums; ++s) v += sum[s * each + i];
  out[i] = (T)v;
}

// ---- scales: powers of two that bring the largest finite entry, or |grad_loss|, to [2^13, 2^14) ----

constexpr int kScaleBlocks = 1024;  // workgroups that look for the largest entries of one kind

__device__ inline float block_max(float v) {
  __shared__ float part[4];
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// Rows of one kind that become a transposed operand: a group's weight rows, or the hidden states.
struct Rows {
  Piece piece;
  int64_t stride;
  int32_t rows, count;    // of each matrix; matrices
  int32_t blocks;         // workgroups that look for a matrix's largest entry; 0: copied unscaled
  const int64_t *target;  // NULL, or: rows whose target is `ignore` do not count
  int64_t ignore;
  const float *grad_loss; // NULL, or: a row carries what its |grad_loss| is below the largest, whose scale is d_scale
  const float *d_scale;
  float *largest;         // [count x blocks]
  float *scale;           // written by the transposition
};

template <class T>
__device__ float largest_of(const Rows &a, int matrix, int block, int cols) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  const T *in = static_cast<const T *>(a.piece.weights.p[matrix]);
  const int valid = a.piece.valid(matrix, a.rows);
  const bool wide = cols % 8 == 0 && a.stride % 8 == 0 && reinterpret_cast<uintptr_t>(in) % 16 == 0;
  float top = 0.f;
  if (wide) {
    // A run of consecutive rows a workgroup, four 16-byte units a thread on their way at a time.
    const int units = cols / 8, each = (valid + a.blocks - 1) / a.blocks, r0 = block * each;
    const int64_t n = (int64_t)max(0, min(each, valid - r0)) * units;
    for (int64_t u = threadIdx.x; u < n; u += 4 * 256) {
      x8 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t at = min(u + k * 256, n - 1);
        const int r = r0 + (int)(at / units);
        v[k] = *reinterpret_cast<const x8 *>(in + r * a.stride + at % units * 8);
        if (a.target && a.target[r] == a.ignore)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[k][i] = (T)0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = fabsf((float)v[k][i]);
          top = x < INFINITY ? fmaxf(top, x) : top;
        }
    }
  } else {
    for (int r = block; r < valid; r += a.blocks) {
      if (a.target && a.target[r] == a.ignore) continue;
      const T *row = in + r * a.stride;
      for (int c = threadIdx.x; c < cols; c += 256) {
        const float x = fabsf((float)row[c]);
        top = x < INFINITY ? fmaxf(top, x) : top;
      }
    }
  }
  return block_max(top);
}

// Largest finite |entry| of what the next transpositions copy, one value a workgroup; and, by the last
// workgroup, the scale of grad_loss (only with the first piece).  One read of them: 134 MB in 37 us, 3.6 TB/s.
template <class T>
__global__ __launch_bounds__(256) void largest_kernel(Rows weights, Rows hidden, int cols, const float *grad_loss, const int64_t *target,
                                                      int64_t ignore, int tokens, float *d_scale) {
  int b = blockIdx.x;
  const int w = weights.count * weights.blocks, h = hidden.count * hidden.blocks;
  if (b < w) {
    const float top = largest_of<T>(weights, b / weights.blocks, b % weights.blocks, cols);
    if (threadIdx.x == 0) weights.largest[b] = top;
    return;
  }
  b -= w;
  if (b < h) {
    const float top = largest_of<T>(hidden, 0, b, cols);
    if (threadIdx.x == 0) hidden.largest[b] = top;
    return;
  }
  float top = 0.f;
  for (int t = threadIdx.x; t < tokens; t += 256) {
    const float a = fabsf(grad_loss[t]);
    if (target[t] != ignore && a < INFINITY) top = fmaxf(top, a);
  }
  top = block_max(top);
  if (threadIdx.x == 0) d_scale[0] = scale_of(top);
}

// ---- operands in the layout that the products read ----

constexpr int kSide = 64;

// out[c][r] = scale in[r][c] for the rows that count and every c, with zeros in the others, up to `padded` r
// for each matrix, one beside the other.
struct Turned {
  Rows rows;
  half *out;
  int64_t out_stride;
  int32_t padded;

  __host__ __device__ uint32_t across() const { return (uint32_t)(padded + kSide - 1) / kSide; }
  __host__ __device__ uint32_t tiles(int cols) const { return rows.count * across() * ((uint32_t)(cols + kSide - 1) / kSide); }
};

// Column c of the tile in row c of LDS; a row's 16-byte units of eight r are permuted by c, so that the eight
// columns that a lane reads in one row meet no other lane's bank.
template <class T>
__device__ __forceinline__ void turn(const Turned &to, uint32_t id, int cols, half (&tile)[kSide][kSide]) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  const Rows &a = to.rows;
  const uint32_t matrix = id % (uint32_t)a.count, tile_at = id / (uint32_t)a.count;
  const int r0 = (int)(tile_at % to.across()) * kSide, c0 = (int)(tile_at / to.across()) * kSide;
  const T *in = static_cast<const T *>(a.piece.weights.p[matrix]);
  const int valid = a.piece.valid(matrix, a.rows);
  float by = 1.f;
  const int largest = exponent_of(a.d_scale);
  if (a.blocks) {
    float top = 0.f;
    for (int i = threadIdx.x; i < a.count * a.blocks; i += 256) top = fmaxf(top, a.largest[i]);
    by = scale_of(block_max(top));
  }
  if (id + threadIdx.x == 0) a.scale[0] = by;
  const bool wide = cols % 8 == 0 && a.stride % 8 == 0 && reinterpret_cast<uintptr_t>(in) % 16 == 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = threadIdx.x + h * 256, r = at / 8, c = at % 8 * 8;
    const bool keep = r0 + r < valid && !(a.target && a.target[r0 + r] == a.ignore);
    float own = by;
    if (a.grad_loss && keep) own = __builtin_amdgcn_ldexpf(by, min(0, largest - exponent_for(a.grad_loss[r0 + r], largest)));
    const T *row = in + (r0 + r) * a.stride + c0 + c;
    x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)0.f;
    if (keep && wide && c0 + c < cols) {
      v = *reinterpret_cast<const x8 *>(row);
    } else if (keep) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + c + i < cols) v[i] = row[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) tile[c + i][((r / 8 ^ (c / 8)) * 8) + r % 8] = (half)((float)v[i] * own);
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = threadIdx.x + h * 256, c = at / 8, unit = at % 8, r = r0 + unit * 8;
    if (c0 + c < cols && r < to.padded)
      *reinterpret_cast<emrs_gemm::fp16x8 *>(to.out + (c0 + c) * to.out_stride + (int64_t)matrix * to.padded + r) =
          *reinterpret_cast<const emrs_gemm::fp16x8 *>(&tile[c][(unit ^ (c / 8)) * 8]);
  }
}

// Both kinds in one launch.  Bound by its bytes: 16384 x 4096 in 56 us, 4.8 TB/s of reads and writes.
template <class T>
__global__ __launch_bounds__(256) void transpose_kernel(Turned weights, Turned hidden, int cols) {
  __shared__ __attribute__((aligned(16))) half tile[kSide][kSide];
  const uint32_t firsts = weights.tiles(cols);
  if (blockIdx.x < firsts)
    turn<T>(weights, blockIdx.x, cols, tile);
  else
    turn<T>(hidden, blockIdx.x - firsts, cols, tile);
}

// out[r][c] = in[r][c], with zeros from `cols` up to the padded row: operands whose rows do not lie on 16 bytes,
// which loads into LDS cannot take.
template <class T>
__global__ __launch_bounds__(256) void pad_kernel(const T *in, int64_t in_stride, int cols, T *out, int64_t out_stride) {
  const int64_t r = blockIdx.x;
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c < out_stride) out[r * out_stride + c] = c < cols ? in[r * in_stride + c] : (T)0.f;
}

bool on_16(const void *p, uint64_t stride, uint64_t k) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && k % 8 == 0;
}

// Shards that go through every kernel together: equal ones, or one.
struct Group {
  uint32_t first, count;
};

// Where the workspace's parts lie, and how the vocabulary is cut.
struct Sizes {
  uint64_t k;              // the hidden size, padded where an operand is copied
  bool pad_hidden, pad_weight;
  Group groups[EMRS_LOSS_MAX_SHARDS];
  uint32_t n_groups;
  uint64_t piece;          // rows of each shard of a group that are worked on at once
  uint64_t tokens_padded;
  uint64_t splits;         // runs of k that grad_hidden's products are cut into
  bool direct;             // these take the weights as they lie
  uint64_t parts, sums;    // of d there; partial sums of grad_hidden, splits x parts
  uint64_t pairs, hidden, weight, sum, d, dt, ht, wt, scales, largest, total;  // offsets
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

Product logits_of(const emrs_loss *a, const Sizes &s, const Group &g, uint64_t rows) {
  Product p{};
  p.b_stride = s.pad_hidden ? s.k : a->tokens > 1 ? a->hidden_stride : s.k;
  p.a_stride = s.pad_weight || a->shard_rows[g.first] == 1 ? s.k : a->weight_strides[g.first];
  p.m = rows, p.n = a->tokens, p.k = s.k;
  p.a_wrap = p.b_wrap = emrs_gemm::kNoWrap;
  p.batch = g.count;
  return p;
}

// Partial statistics that a shard's `rows` rows leave for each token.
int64_t slots_of(const emrs_loss *a, const Product &p) {
  return a->tokens == 1 ? emrs_gemm::tiles_of(p.m, kOneRows) : emrs_gemm::wave_rows(p);
}

Sizes sizes_of(const emrs_loss *a, bool backward) {
  Sizes s{};
  uint64_t most = 1, shards = 1;
  s.pad_hidden = !on_16(a->hidden, a->tokens > 1 ? a->hidden_stride : 8, a->hidden_size);
  bool equal = true;
  for (uint32_t i = 0; i < a->n_shards; ++i) {
    most = std::max(most, a->shard_rows[i]);
    s.pad_weight |= !on_16(a->weights[i], a->shard_rows[i] > 1 ? a->weight_strides[i] : 8, a->hidden_size);
    equal &= a->shard_rows[i] == a->shard_rows[0] && a->weight_strides[i] == a->weight_strides[0];
  }
  s.n_groups = equal ? 1 : a->n_shards;
  for (uint32_t i = 0; i < s.n_groups; ++i) s.groups[i] = equal ? Group{0, a->n_shards} : Group{i, 1};
  if (equal) shards = a->n_shards;
  s.k = a->hidden_size % 8 ? round_up(a->hidden_size, 64) : a->hidden_size;
  s.tokens_padded = round_up(std::max<uint64_t>(a->tokens, 1), 64);
  s.piece = round_up(most, 256);
  if (backward || s.pad_weight)
    s.piece = std::min(s.piece, std::max<uint64_t>(kPieceBytes / 2 / s.tokens_padded / shards / 256, 1) * 256);
  s.direct = takes_weights(a->dtype, a->tokens);
  if (s.pad_weight || (backward && a->grad_hidden && !s.direct))
    s.piece = std::min(s.piece, std::max<uint64_t>(kCopyBytes / 2 / s.k / shards / 256, 1) * 256);
  uint64_t slots = 0;
  for (uint32_t i = 0; i < s.n_groups; ++i)
    for (uint64_t lo = 0; lo < a->shard_rows[s.groups[i].first]; lo += s.piece)
      slots += slots_of(a, logits_of(a, s, s.groups[i], std::min(s.piece, a->shard_rows[s.groups[i].first] - lo))) * s.groups[i].count;
  // grad_hidden's product has few tiles where there are few tokens: its sum over the vocabulary is cut into
  // runs of at least 1024 rows, as many as the product and the sums' way through memory take least time with.
  const uint64_t k = round_up(std::min(s.piece, most), 64) * shards;
  s.parts = s.direct && a->dtype == EMRS_BF16 ? 2 : 1;
  s.splits = 1;
  double best = 0;
  for (uint64_t n = 1; n <= std::min<uint64_t>(256, std::max<uint64_t>(1, k / 1024)); n += n < 16 ? 1 : n / 8) {
    Product q{};
    q.m = (int32_t)a->hidden_size, q.n = (int32_t)(s.parts * a->tokens), q.k = (int32_t)round_up((k + n - 1) / n, 64);
    q.batch = (int32_t)n;
    const double cost = emrs_gemm::choice_of(q, s.direct, !s.direct).cost + (n * s.parts > 1 ? 6 + 8e-6 * n * q.m * q.n / 4 : 0);
    if (n == 1 || cost < best) best = cost, s.splits = n;
  }
  s.sums = s.splits * s.parts;
  uint64_t at = 0;
  auto take = [&](bool wanted, uint64_t bytes) {
    const uint64_t here = at;
    if (wanted) at += round_up(bytes, 256);
    return here;
  };
  s.pairs = take(!backward, slots * a->tokens * sizeof(float2));
  s.hidden = take(s.pad_hidden, a->tokens * s.k * 2);
  s.weight = take(s.pad_weight, shards * s.piece * s.k * 2);
  s.sum = take(backward && a->grad_hidden, s.sums * a->tokens * a->hidden_size * 4);
  s.d = take(backward && a->grad_hidden, s.parts * a->tokens * shards * s.piece * 2);
  s.wt = take(backward && a->grad_hidden && !s.direct, a->hidden_size * shards * s.piece * 2);
  s.dt = take(backward && a->grad_weights, shards * s.piece * s.tokens_padded * 2);
  s.ht = take(backward && a->grad_weights, a->hidden_size * s.tokens_padded * 2);
  s.scales = take(backward, 256);
  s.largest = take(backward, 2 * kScaleBlocks * 4);
  s.total = at;
  return s;
}

#define TRY(expr)                                                                                       \
  do {                                                                                                  \
    const hipError_t e_ = (expr);                                                                       \
    if (e_ != hipSuccess) return fail(EMRS_ERR_HIP, std::string("loss: ") + hipGetErrorString(e_));     \
  } while (0)

Piece piece_of(const emrs_loss *a, const Group &g, uint64_t first, uint64_t lo) {
  Piece c{};
  for (uint32_t i = 0; i < g.count; ++i)
    c.weights.p[i] = static_cast<const char *>(a->weights[g.first + i]) + lo * a->weight_strides[g.first + i] * 2;
  c.first = (int64_t)(first + lo), c.shard = (int64_t)a->shard_rows[g.first], c.vocab = (int64_t)a->vocab_size;
  return c;
}

// The same piece as an operand of the logits' product: copied into padded rows where its own do not lie on 16 bytes.
template <class T>
int aligned_piece(const emrs_loss *a, const Sizes &s, const Group &g, uint64_t rows, Piece *c, hipStream_t st) {
  if (!s.pad_weight) return EMRS_OK;
  T *out = reinterpret_cast<T *>(static_cast<char *>(a->workspace) + s.weight);
  for (uint32_t i = 0; i < g.count; ++i, out += rows * s.k) {
    pad_kernel<T><<<dim3(rows, (s.k + 255) / 256), 256, 0, st>>>(static_cast<const T *>(c->weights.p[i]), a->weight_strides[g.first + i],
                                                                 (int)a->hidden_size, out, s.k);
    TRY(hipGetLastError());
    c->weights.p[i] = out;
  }
  return EMRS_OK;
}

template <class T>
int aligned_hidden(const emrs_loss *a, const Sizes &s, const void **hidden, hipStream_t st) {
  *hidden = a->hidden;
  if (!s.pad_hidden) return EMRS_OK;
  T *out = reinterpret_cast<T *>(static_cast<char *>(a->workspace) + s.hidden);
  pad_kernel<T><<<dim3(a->tokens, (s.k + 255) / 256), 256, 0, st>>>(static_cast<const T *>(a->hidden), a->hidden_stride, (int)a->hidden_size,
                                                                    out, s.k);
  TRY(hipGetLastError());
  *hidden = out;
  return EMRS_OK;
}

template <class T>
int forward(const emrs_loss *a, hipStream_t st) {
  const Sizes s = sizes_of(a, false);
  float2 *pairs = reinterpret_cast<float2 *>(static_cast<char *>(a->workspace) + s.pairs);
  const void *hidden;
  int rc = aligned_hidden<T>(a, s, &hidden, st);
  if (rc) return rc;
  uint64_t first = a->vocab_start;
  int64_t slots = 0;
  for (uint32_t i = 0; i < s.n_groups; ++i) {
    const Group &g = s.groups[i];
    const uint64_t all = a->shard_rows[g.first];
    for (uint64_t lo = 0; lo < all; lo += s.piece) {
      const uint64_t rows = std::min(s.piece, all - lo);
      Piece c = piece_of(a, g, first, lo);
      rc = aligned_piece<T>(a, s, g, rows, &c, st);
      if (rc) return rc;
      Product p = logits_of(a, s, g, rows);
      p.b = hidden;
      const int64_t each = slots_of(a, p);
      float2 *const out = pairs + slots * (int64_t)a->tokens;
      if (a->tokens == 1) {
        one_token_kernel<T><<<dim3((uint32_t)each, g.count), kOneThreads, 0, st>>>(c, p.a_stride, p.m, static_cast<const T *>(hidden), p.k, out,
                                                                                a->target_logit, a->target);
        TRY(hipGetLastError());
      } else {
        TRY((emrs_gemm::launch<T>(p, TileStatistics{c, out, a->target_logit, a->target, each}, st)));
      }
      slots += each * g.count;
    }
    first += all * g.count;
  }
  const int64_t last = (int64_t)std::max(a->vocab_start, std::min(first, a->vocab_size));
  // Few tokens: all of a workgroup on one, so that its many slots are not read one after another.
  const auto merge = a->tokens <= 256 ? merge_statistics_kernel<1> : merge_statistics_kernel<16>;
  const uint64_t each = a->tokens <= 256 ? 1 : 16;
  merge<<<(a->tokens + each - 1) / each, kMergeThreads, 0, st>>>(pairs, slots, (int)a->tokens, a->target, a->ignore_index, (int64_t)a->vocab_start,
                                                              last, a->lse, a->target_logit, a->loss);
  TRY(hipGetLastError());
  return EMRS_OK;
}

Rows rows_of(const Piece &c, uint32_t count, int64_t stride, int64_t rows, bool scaled, float *largest, float *scale) {
  Rows r{};
  r.piece = c, r.stride = stride, r.rows = (int32_t)rows, r.count = (int32_t)count;
  r.blocks = scaled ? (int32_t)std::max<int64_t>(1, std::min<int64_t>(rows, kScaleBlocks / count)) : 0;
  r.largest = largest, r.scale = scale;
  return r;
}

template <class T>
int backward(const emrs_loss *a, hipStream_t st) {
  const Sizes s = sizes_of(a, true);
  char *ws = static_cast<char *>(a->workspace);
  half *d = reinterpret_cast<half *>(ws + s.d), *wt = reinterpret_cast<half *>(ws + s.wt);
  half *dt = reinterpret_cast<half *>(ws + s.dt), *ht = reinterpret_cast<half *>(ws + s.ht);
  float *sum = reinterpret_cast<float *>(ws + s.sum), *largest = reinterpret_cast<float *>(ws + s.largest);
  float *d_scale = reinterpret_cast<float *>(ws + s.scales), *h_scale = d_scale + 1, *w_scale = d_scale + 2;
  const int64_t h = (int64_t)a->hidden_size, tokens = (int64_t)a->tokens;
  const void *hidden;
  int rc = aligned_hidden<T>(a, s, &hidden, st);
  if (rc) return rc;
  Piece every{};
  every.weights.p[0] = a->hidden, every.vocab = tokens;
  Rows h_rows = rows_of(every, 1, (int64_t)a->hidden_stride, tokens, true, largest + kScaleBlocks, h_scale);
  h_rows.target = a->target, h_rows.ignore = a->ignore_index;
  h_rows.grad_loss = a->grad_loss, h_rows.d_scale = d_scale;
  const bool fours = h % 4 == 0;
  uint64_t first = a->vocab_start, left = 0;
  for (uint32_t i = 0; i < s.n_groups; ++i) left += (a->shard_rows[s.groups[i].first] + s.piece - 1) / s.piece;
  bool begun = false, scaled = false;
  for (uint32_t i = 0; i < s.n_groups; ++i) {
    const Group &g = s.groups[i];
    const uint64_t all = a->shard_rows[g.first];
    uint32_t wanted = 0;
    for (uint32_t k = 0; a->grad_weights && k < g.count; ++k) wanted += a->grad_weights[g.first + k] != nullptr;
    for (uint64_t lo = 0; lo < all; lo += s.piece) {
      const uint64_t rows = std::min(s.piece, all - lo), padded = round_up(rows, 64);
      --left;
      if (!a->grad_hidden && !wanted) continue;
      const Piece own = piece_of(a, g, first, lo);
      const Rows w_rows = rows_of(own, g.count, (int64_t)a->weight_strides[g.first], (int64_t)rows, !std::is_same<T, half>::value, largest, w_scale);
      Rows none = h_rows;
      none.count = 0;
      const bool copied = a->grad_hidden && !s.direct;
      const int blocks = (copied ? w_rows.count * w_rows.blocks : 0) + (scaled ? 0 : (a->grad_weights ? h_rows.blocks : 0) + 1);
      if (blocks) {
        largest_kernel<T><<<blocks, 256, 0, st>>>(copied ? w_rows : none, scaled || !a->grad_weights ? none : h_rows, (int)h, a->grad_loss,
                                                  a->target, a->ignore_index, (int)tokens, d_scale);
        TRY(hipGetLastError());
      }
      const Turned w_turned{copied ? w_rows : none, wt, (int64_t)(g.count * padded), (int32_t)padded};
      const Turned h_turned{scaled || !a->grad_weights ? none : h_rows, ht, (int64_t)s.tokens_padded, (int32_t)s.tokens_padded};
      if (const uint32_t tiles = w_turned.tiles((int)h) + h_turned.tiles((int)h)) {
        transpose_kernel<T><<<tiles, 256, 0, st>>>(w_turned, h_turned, (int)h);
        TRY(hipGetLastError());
      }
      scaled = true;
      Piece c = own;
      rc = aligned_piece<T>(a, s, g, rows, &c, st);
      if (rc) return rc;
      Product p = logits_of(a, s, g, rows);
      p.b = hidden;
      const int32_t sum_k = (int32_t)(g.count * padded);
      auto gradients = [&](auto e) {
        static_cast<Piece &>(e) = c;
        e.d = a->grad_hidden ? d : nullptr, e.dt = wanted ? dt : nullptr;
        e.d_stride = sum_k, e.dt_stride = (int32_t)s.tokens_padded, e.padded = (int32_t)padded;
        e.lse = a->lse, e.grad_loss = a->grad_loss, e.target = a->target, e.ignore = a->ignore_index, e.scale = d_scale;
        return emrs_gemm::launch<T>(p, e, st);
      };
      TRY(s.parts == 2 ? gradients(LogitGradients<true>{}) : gradients(LogitGradients<false>{}));
      if (a->grad_hidden) {
        Product q{};
        q.a = wt, q.b = d;
        q.a_stride = s.direct ? p.a_stride : sum_k, q.b_stride = sum_k;
        q.m = h, q.n = (int32_t)(s.parts * a->tokens);
        q.a_wrap = q.b_wrap = emrs_gemm::kNoWrap;
        auto product = [&](const auto &e) {
          if (s.direct) return emrs_gemm::launch<T>(q, OfWeights<std::decay_t<decltype(e)>>{e, c, (int32_t)padded, (int32_t)rows, sum_k}, st);
          return emrs_gemm::launch<half>(q, e, st);
        };
        q.batch = 1, q.k = sum_k;
        if (s.splits > 1) {
          // Runs of k as a batch: multiples of 64, the last one shorter (its stages past the end are zeros).
          q.k_end = q.k;
          q.batch = (int32_t)s.splits;
          q.k = (int32_t)round_up((q.k + s.splits - 1) / s.splits, 64);
          q.a_batch = q.b_batch = q.k;
        }
        const Scales scales{d_scale, s.direct ? nullptr : w_scale, a->grad_loss, (int32_t)tokens};
        if (s.sums > 1 || left) {
          TRY(product(StoreSums{{}, sum, h, q.n * h, begun, fours, scales}));
        } else {
          StoreRows<T> out{};
          out.out.p[0] = a->grad_hidden, out.sum = begun ? sum : nullptr, out.stride = h;
          out.wide = h % 8 == 0 && reinterpret_cast<uintptr_t>(a->grad_hidden) % 16 == 0;
          out.scales = scales;
          TRY(product(out));
        }
        begun = true;
      }
      for (uint32_t k = 0; wanted && k < g.count; k += wanted == g.count ? g.count : 1) {
        const uint32_t n = wanted == g.count ? g.count : 1;
        if (!a->grad_weights[g.first + k]) continue;
        Product q{};
        q.a = ht, q.b = dt + (int64_t)k * padded * s.tokens_padded;
        q.a_stride = q.b_stride = s.tokens_padded, q.b_batch = (int64_t)padded * s.tokens_padded;
        q.m = h, q.n = rows, q.k = s.tokens_padded;
        q.a_wrap = q.b_wrap = emrs_gemm::kNoWrap;
        q.batch = n;
        StoreRows<T> out{};
        out.wide = h % 8 == 0;
        for (uint32_t b = 0; b < n; ++b) {
          T *gw = static_cast<T *>(a->grad_weights[g.first + k + b]) + lo * h;
          out.out.p[b] = gw;
          out.wide &= reinterpret_cast<uintptr_t>(gw) % 16 == 0;
        }
        out.stride = h, out.scales = Scales{d_scale, h_scale, nullptr, 0};
        TRY((emrs_gemm::launch<half>(q, out, st)));
      }
    }
    first += all * g.count;
  }
  if (a->grad_hidden && s.sums > 1) {
    join_sums_kernel<T><<<(uint32_t)((tokens * h + 255) / 256), 256, 0, st>>>(sum, (int)s.sums, tokens * h, static_cast<T *>(a->grad_hidden));
    TRY(hipGetLastError());
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
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    const int rc = check(a);
    if (rc) return rc;
    if (!bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "loss: NULL argument");
    *bytes = sizes_of(a, backward != 0).total;
    return EMRS_OK;
  });
}

int emrs_loss_forward(const emrs_loss *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
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
  });
}

int emrs_loss_backward(const emrs_loss *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
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
  });
}

}  // extern "C"
