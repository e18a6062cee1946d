// Products of every token with its expert's weight matrix, over experts of ragged sizes.
//
// Rows lie by expert: the first counts[0] are expert 0's, and so on; rows behind the last expert's belong to none.
//   y_t = W_e x_t,  grad_x_t = W_e^T grad_y_t,  grad_W_e = sum_t grad_y_t x_t^T
// The counts stay on the device.  A launch has as many workgroups as tiles there can be at the most (every expert
// may add one that is not full); each finds its expert by a prefix sum over the counts, one a lane, and those past the
// last tile end at once.  So nothing is sorted, padded or read back, and no expert waits for another.
//
// All three are products of gemm.h, bound by its matrix instructions where experts have many tokens and by the bytes
// of the weights where they have few.  Outputs have m contiguous, m the weights' other side: rows of x and grad_y are
// operand b.  grad_x sums over rows of W_e, and grad_W over tokens, along which operands lie in rows of k:
// transposing reads from LDS, which cost less than copies the other way round.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "emrs.h"
#include "gemm.h"
#include "internal.h"

namespace {

using emrs_gemm::f32x4;
using emrs_gemm::kGroup;
using emrs_gemm::kXcds;
using emrs_gemm::Product;
using emrs_gemm::Where;
using emrs_internal::fail;

constexpr uint64_t kMaxRows = (1u << 30) - 1;  // the sum of two counts fits 32 bits
// k from which on the tiles of a last round are cut along it: it has to be long enough to pay for 64 MB of parts (4096
// rows, m 4096, k 14336: 272 tiles in 443 us, uncut 705; k of 4096 loses what it gains).
constexpr uint64_t kCutFrom = 8192;
// Rows up to which weights are read by rows, in vector arithmetic (2 experts' 28672 x 4096 with a row each, 84 us against
// 110 in tiles; one expert's with two rows, 59 against 58).
constexpr uint64_t kFew = 2;

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

struct Table {
  const void *p[EMRS_EXPERTS_MAX];
};

// The rows of every expert, and behind them those of none.
struct Counts {
  const void *counts;
  int32_t wide;     // 64-bit counts
  int32_t experts, rows;

  // A count as it counts: none below 0, none past the rows (sums below stay within 32 bits).
  __device__ __forceinline__ int of(int e) const {
    if (e >= experts) return 0;
    if (wide) return (int)min(max(static_cast<const int64_t *>(counts)[e], (int64_t)0), (int64_t)rows);
    return min(max(static_cast<const int32_t *>(counts)[e], 0), rows);
  }
};

__device__ __forceinline__ int lane_of() { return threadIdx.x & 63; }

// Inclusive prefix sum over a wave, held at `most`: of values in [0, most], most < 2^30.
__device__ __forceinline__ int prefix(int v, int most) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int before = __shfl_up(v, o);
    if (lane_of() >= o) v = min(v + before, most);
  }
  return v;
}

struct Segment {
  int expert, first, end;  // expert == experts: the rows of none
};

// Tiles of `size` rows over the experts' rows, and over those of none behind them (kRest).
struct Walk {
  int first, end, tiles;   // of this lane's segment of the current 64, tiles up to and with it
  int rows_before, tiles_before;

  __device__ __forceinline__ void begin() { rows_before = tiles_before = 0; }
  template <bool kRest>
  __device__ __forceinline__ void step(const Counts &c, int from, int size) {
    const int e = from + lane_of(), upto = min(prefix(c.of(e), c.rows) + rows_before, c.rows);
    end = upto;
    const int last = __builtin_amdgcn_readlane(upto, 63), below = __shfl_up(upto, 1);
    first = lane_of() ? below : rows_before;
    if (kRest && e == c.experts) end = c.rows;
    if (e > c.experts) first = end = c.rows;
    tiles = prefix((end - first + size - 1) / size, 0x3fffffff) + tiles_before;
    rows_before = last;
    tiles_before = __builtin_amdgcn_readlane(tiles, 63);
  }
};

// Tiles that fill no round of 256 workgroups, cut along a long k: `whole` tiles go as they are, and each of the others
// is as many parts as there are workgroups for, whose sums a second kernel joins.  The same in both kernels.
struct Cut {
  uint32_t total, whole, parts;
};
constexpr uint32_t kRound = 256, kLeastStages = 16;

__device__ __forceinline__ Cut cut_of(uint32_t total, int k, bool cuts) {
  const uint32_t rest = total % kRound, stages = (k + emrs_gemm::kStage - 1) / emrs_gemm::kStage;
  const uint32_t parts = cuts && rest ? min(kRound / rest, stages / kLeastStages) : 1;
  return parts > 1 ? Cut{total, total - rest, parts} : Cut{total, total, 1};
}

// Tiles along n of all segments; `walk` is then at the last 64.
template <class Cfg>
__device__ __forceinline__ uint32_t tiles_of(const Counts &c, Walk &walk) {
  walk.begin();
  for (int from = 0; from <= c.experts; from += 64) walk.step<true>(c, from, Cfg::BN);
  return (uint32_t)walk.tiles_before;
}

// Tile t of the experts' rows (n) and of the weights' side m.
template <class Cfg>
__device__ __forceinline__ void locate(const Counts &c, const Product &p, Walk &walk, uint32_t t, Where &w, Segment &s) {
  const uint32_t tm = (p.m + Cfg::BM - 1) / Cfg::BM;
  if (c.experts >= 64) walk.begin();  // of more than one 64, find the one
  for (int from = 0;; from += 64) {
    if (c.experts >= 64) walk.step<true>(c, from, Cfg::BN);
    const uint64_t past = __ballot(t < (uint32_t)walk.tiles * tm);
    if (!past) continue;  // never of the last 64: t is less than all tiles
    const int lane = __builtin_ctzll(past);
    s.expert = from + lane;
    s.first = __builtin_amdgcn_readlane(walk.first, lane);
    s.end = __builtin_amdgcn_readlane(walk.end, lane);
    t -= (uint32_t)(__builtin_amdgcn_readlane(walk.tiles, lane) - (s.end - s.first + Cfg::BN - 1) / Cfg::BN) * tm;
    break;
  }
  const uint32_t tn = (s.end - s.first + Cfg::BN - 1) / Cfg::BN;
  const uint32_t group = t / (kGroup * tn), first = group * kGroup, rows = min((uint32_t)kGroup, tm - first);
  const uint32_t in = t - group * kGroup * tn;
  w.m0 = (int)(first + in % rows) * Cfg::BM;
  w.n0 = (int)(in / rows) * Cfg::BN;
  w.first = s.first;
}

// The workgroup's tile, or its part of one; false: there is none.  Each XCD has a run of consecutive tiles.
template <class Cfg>
__device__ __forceinline__ bool find(const Counts &c, Product &p, bool cuts, Where &w, Segment &s) {
  Walk walk;
  const uint32_t tm = (p.m + Cfg::BM - 1) / Cfg::BM;
  const Cut cut = cut_of(tiles_of<Cfg>(c, walk) * tm, p.k, cuts);  // checked on the host to fit
  const bool whole = blockIdx.x < cut.whole;
  const uint32_t id = whole ? blockIdx.x : blockIdx.x - cut.whole, units = whole ? cut.whole : (cut.total - cut.whole) * cut.parts;
  const uint32_t q = units / kXcds, r = units % kXcds, x = id % kXcds, at = id / kXcds;
  if (at >= q + (x < r ? 1 : 0)) return false;
  const uint32_t unit = x * q + min(x, r) + at;
  locate<Cfg>(c, p, walk, whole ? unit : cut.whole + unit / cut.parts, w, s);
  w.k_from = 0;
  w.part = -1;
  if (!whole) {
    const int stages = (p.k + emrs_gemm::kStage - 1) / emrs_gemm::kStage, part = unit % cut.parts;
    w.k_from = stages * part / (int)cut.parts * emrs_gemm::kStage;
    w.part = unit;
    p.k = min(p.k, stages * (part + 1) / (int)cut.parts * emrs_gemm::kStage) - w.k_from;
  }
  if (s.expert == c.experts) p.k = 0;  // zeros
  return true;
}

// The rows of one expert.
__device__ __forceinline__ Segment rows_of(const Counts &c, int expert) {
  Walk walk;
  walk.begin();
  for (int from = 0; from <= expert; from += 64) walk.step<false>(c, from, 1);
  const int lane = expert & 63;
  return {expert, __builtin_amdgcn_readlane(walk.first, lane), __builtin_amdgcn_readlane(walk.end, lane)};
}

// C as 16-bit rows to[n][m], through LDS where eight elements can be stored at once.
template <class T, class Cfg>
__device__ __forceinline__ void store_rows(const f32x4 (&acc)[Cfg::MI][Cfg::NI], T *to, int64_t stride, bool wide, int m0, int n0, int lane, const Product &p,
                                           char *own) {
  using x4 = typename emrs_gemm::Vec<T>::x4;
  using Turn = emrs_gemm::Turn<Cfg>;
  if (wide) {
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = (T)acc[i][j][r];
        Turn::put(own, i, j, lane, v);
      }
    T *const corner = to + n0 * stride + m0;
    const int step = (int)stride;  // 256 rows of 2^20 elements at most
    Turn::along_m(own, lane, [&](int x, int y, emrs_gemm::fp16x8 v) __attribute__((always_inline)) {
      if (m0 + x < p.m && n0 + y < p.n) *reinterpret_cast<emrs_gemm::fp16x8 *>(corner + (y * step + x)) = v;
    });
    return;
  }
#pragma unroll
  for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
    for (int i = 0; i < Cfg::MI; ++i) {
      const int n = n0 + j * 16 + (lane & 15), m = m0 + i * 16 + (lane >> 4) * 4;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n < p.n && m + r < p.m) to[n * stride + m + r] = (T)acc[i][j][r];
    }
}

// y, or with kTransposed (the weights' rows are rows of k) grad_x.
template <class T, bool kTransposed>
struct OfTokens {
  static constexpr bool kRowsOfK = kTransposed, kBy32 = !kTransposed, kColumnsOfK = false, kPlaced = true;
  Table weights;
  Counts counts;
  int32_t wide, n_out;    // n_out: rows of a weight
  T *out;                 // [rows][m]
  float *parts;           // [part][BN][BM], where tiles may be cut along k; NULL: they are not

  template <class Cfg>
  __device__ __forceinline__ bool place(Product &p, Where &w) const {
    Segment s;
    if (!find<Cfg>(counts, p, parts != nullptr, w, s)) return false;
    p.n = s.end - s.first;
    p.b = static_cast<const T *>(p.b) + s.first * p.b_stride + w.k_from;
    w.batch = min(s.expert, counts.experts - 1);
    p.a = static_cast<const T *>(weights.p[w.batch]) + w.k_from * (kTransposed ? p.a_stride : 1);
    return true;
  }
  __device__ __forceinline__ const void *operand_a(const Product &p, int) const { return p.a; }
  __device__ __forceinline__ const void *operand_b(const Product &p, int) const { return p.b; }
  template <class U>
  __device__ __forceinline__ void rows_from(const Product &p, const Where &w, int k, const U *&first, int &count) const {
    first = static_cast<const U *>(p.a) + k * p.a_stride;
    count = n_out - w.k_from - k;
  }
  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    if (w.part < 0) return store_rows<T, Cfg>(acc, out + (int64_t)w.first * p.m, p.m, wide, m0, n0, lane, p, own);
    float *const to = parts + (int64_t)w.part * (Cfg::BN * Cfg::BM);
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const int n = n0 - w.n0 + j * 16 + (lane & 15), m = m0 - w.m0 + i * 16 + (lane >> 4) * 4;
        *reinterpret_cast<f32x4 *>(to + n * Cfg::BM + m) = acc[i][j];
      }
  }
};

// Joins the parts of the tiles that were cut: 32 of a tile's rows to a workgroup, in the order of k.
constexpr int kJoinRows = 32;

template <class T, class Cfg>
__global__ __launch_bounds__(256) void join_tiles_kernel(Product p, Counts counts, const float *parts, T *out) {
  constexpr int each = Cfg::BN / kJoinRows;
  Walk walk;
  const uint32_t tm = (p.m + Cfg::BM - 1) / Cfg::BM;
  const Cut cut = cut_of(tiles_of<Cfg>(counts, walk) * tm, p.k, true);
  const uint32_t nth = blockIdx.x / each;
  if (nth >= cut.total - cut.whole) return;
  Where w;
  Segment s;
  locate<Cfg>(counts, p, walk, cut.whole + nth, w, s);
  static_assert(Cfg::BM == 256, "a row of a tile is four elements of each lane of a wave");
  const int m = (threadIdx.x & 63) * 4, n0 = blockIdx.x % each * kJoinRows + (threadIdx.x >> 6) * (kJoinRows / 4);
  const float *const from = parts + (int64_t)nth * cut.parts * (Cfg::BN * Cfg::BM) + m;
#pragma unroll 1
  for (int n = n0; n < n0 + kJoinRows / 4 && w.n0 + n < s.end - s.first; ++n) {
    f32x4 v = *reinterpret_cast<const f32x4 *>(from + n * Cfg::BM);
#pragma unroll 4
    for (uint32_t i = 1; i < cut.parts; ++i) v += *reinterpret_cast<const f32x4 *>(from + (int64_t)i * (Cfg::BN * Cfg::BM) + n * Cfg::BM);
    T *const to = out + (int64_t)(s.first + w.n0 + n) * p.m + w.m0 + m;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (w.m0 + m + e < p.m) to[e] = (T)v[e];
  }
}

// Few rows: a token's experts are read once, in vector arithmetic.  A wave takes four of a weight's rows, each in whole
// consecutive kilobytes and many of them on their way at a time, for up to two of the expert's rows.
constexpr int kFewRows = 2, kFewWeights = 4, kFewWaves = 4;

template <class T>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(Table weights, int64_t weight_stride, Counts counts, const T *x, int64_t x_stride, int k,
                                                                  int n_out, T *y) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  Walk walk;
  walk.begin();
  Segment s{};
  int at = 0;
  bool found = false;
  for (int from = 0; from <= counts.experts && !found; from += 64) {
    walk.step<true>(counts, from, kFewRows);
    const uint64_t past = __ballot((int)blockIdx.y < walk.tiles);
    if (!past) continue;
    const int lane = __builtin_ctzll(past);
    s = {from + lane, __builtin_amdgcn_readlane(walk.first, lane), __builtin_amdgcn_readlane(walk.end, lane)};
    at = s.first + ((int)blockIdx.y - __builtin_amdgcn_readlane(walk.tiles, lane) + (s.end - s.first + kFewRows - 1) / kFewRows) * kFewRows;
    found = true;
  }
  const int m0 = ((int)blockIdx.x * kFewWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kFewWeights, lane = lane_of();
  if (!found || m0 >= n_out) return;
  const int count = min(kFewRows, s.end - at);
  const T *const w = static_cast<const T *>(weights.p[min(s.expert, counts.experts - 1)]);
  const T *const row = x + at * x_stride, *const second = row + (count > 1 ? x_stride : 0);
  float acc[kFewRows][kFewWeights];
#pragma unroll
  for (int r = 0; r < kFewRows; ++r)
#pragma unroll
    for (int i = 0; i < kFewWeights; ++i) acc[r][i] = 0.f;
  if (s.expert < counts.experts)
#pragma unroll 4
    for (int c = lane * 8; c < k; c += 64 * 8) {
      x8 a[kFewWeights];  // rows past the last one read it again, and are left out below
#pragma unroll
      for (int i = 0; i < kFewWeights; ++i) a[i] = __builtin_nontemporal_load(reinterpret_cast<const x8 *>(w + min(m0 + i, n_out - 1) * weight_stride + c));
      const x8 b = *reinterpret_cast<const x8 *>(row + c);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < kFewWeights; ++i) acc[0][i] = fmaf((float)a[i][e], (float)b[e], acc[0][i]);
      if (count > 1) {
        const x8 d = *reinterpret_cast<const x8 *>(second + c);
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < kFewWeights; ++i) acc[1][i] = fmaf((float)a[i][e], (float)d[e], acc[1][i]);
      }
    }
#pragma unroll
  for (int r = 0; r < kFewRows; ++r)
#pragma unroll
    for (int i = 0; i < kFewWeights; ++i) {
      if (r >= count) continue;
      float v = acc[r][i];
#pragma unroll
      for (int o = 32; o; o /= 2) v += __shfl_xor(v, o);
      if (lane == 0 && m0 + i < n_out) y[(int64_t)(at + r) * n_out + m0 + i] = (T)v;
    }
}

// grad_W: both operands are rows of k.
template <class T>
struct OfWeights {
  static constexpr bool kRowsOfK = true, kBy32 = false, kColumnsOfK = true, kPlaced = true;
  Table out;
  Counts counts;
  int32_t wide;

  template <class Cfg>
  __device__ __forceinline__ bool place(Product &p, Where &w) const {
    // One expert after the other, each over all XCDs: how long a tile takes is its expert's rows.
    const uint32_t tm = (p.m + Cfg::BM - 1) / Cfg::BM, tn = (p.n + Cfg::BN - 1) / Cfg::BN, each = (tm * tn + kXcds - 1) / kXcds;
    const uint32_t t = blockIdx.x % kXcds * each + blockIdx.x / kXcds % each;
    if (t >= tm * tn) return false;
    w.batch = blockIdx.x / (each * kXcds);
    const uint32_t group = t / (kGroup * tn), first = group * kGroup, rows = min((uint32_t)kGroup, tm - first);
    const uint32_t in = t - group * kGroup * tn;
    w.m0 = (int)(first + in % rows) * Cfg::BM;
    w.n0 = (int)(in / rows) * Cfg::BN;
    const Segment s = rows_of(counts, w.batch);
    p.k = s.end - s.first;
    p.a = static_cast<const T *>(p.a) + s.first * p.a_stride;
    p.b = static_cast<const T *>(p.b) + s.first * p.b_stride;
    return true;
  }
  template <class U>
  __device__ __forceinline__ void rows_from(const Product &p, const Where &, int k, const U *&first, int &count) const {
    first = static_cast<const U *>(p.a) + k * p.a_stride;
    count = p.k - k;
  }
  template <class U>
  __device__ __forceinline__ void columns_from(const Product &p, const Where &, int k, const U *&first, int &count) const {
    first = static_cast<const U *>(p.b) + k * p.b_stride;
    count = p.k - k;
  }
  template <class Cfg>
  __device__ __forceinline__ void run(f32x4 (&acc)[Cfg::MI][Cfg::NI], const Where &w, int m0, int n0, int, int lane, const Product &p, char *own) const {
    store_rows<T, Cfg>(acc, static_cast<T *>(const_cast<void *>(out.p[w.batch])), p.m, wide, m0, n0, lane, p, own);
  }
};

// Rows as operands want them: on 16 bytes, with zeros up to the next multiple of eight.
template <class T>
__global__ __launch_bounds__(256) void pad_rows_kernel(Table from, int64_t stride, uint64_t rows, int columns, int padded, T *to) {
  typedef __attribute__((ext_vector_type(8))) T x8;
  const T *const in = static_cast<const T *>(from.p[blockIdx.y]);
  x8 *const out = reinterpret_cast<x8 *>(to + blockIdx.y * rows * padded);
  const int units = padded / 8;
  const uint64_t all = rows * units;
  for (uint64_t u = (uint64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += (uint64_t)gridDim.x * 256) {
    const T *const row = in + u / units * stride;
    const int at = (int)(u % units) * 8;
    x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < columns ? row[at + e] : (T)0.f;
    out[u] = v;
  }
}

bool on(const void *p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether a product over k may cut the tiles of its last round, and the room that their parts take.
bool may_cut(uint64_t k, uint64_t rows) { return k >= kCutFrom && rows >= emrs_gemm::Large::BN; }
constexpr uint64_t kPartsBytes = (uint64_t)kRound * emrs_gemm::Large::BN * emrs_gemm::Large::BM * 4;

// Of the three inputs, which have to be copied, and where in the workspace the copies and the tiles' parts lie.
struct Copies {
  bool x, weights, grad_y, cuts;
  uint64_t at_weights, at_grad_y, at_parts, bytes;
};

Copies copies_of(const emrs_experts *a, bool backward) {
  Copies c{};
  const uint64_t in8 = round_up(a->n_in, 8), out8 = round_up(a->n_out, 8);
  const bool want_x = !backward || a->grad_weights, want_w = !backward || a->grad_x;
  c.x = want_x && (a->n_in % 8 || a->x_stride % 8 || !on(a->x, 16));
  c.weights = want_w && (a->n_in % 8 || a->weight_stride % 8);
  for (uint32_t e = 0; want_w && a->weights && e < a->n_experts; ++e) c.weights |= !on(a->weights[e], 16);
  c.grad_y = backward && (a->n_out % 8 || a->grad_y_stride % 8 || !on(a->grad_y, 16));
  c.at_weights = c.x ? round_up(a->rows * in8 * 2, 256) : 0;
  c.at_grad_y = c.at_weights + (c.weights ? round_up((uint64_t)a->n_experts * a->n_out * in8 * 2, 256) : 0);
  c.cuts = (!backward && may_cut(a->n_in, a->rows)) || (backward && a->grad_x && may_cut(a->n_out, a->rows));
  c.at_parts = c.at_grad_y + (c.grad_y ? round_up(a->rows * out8 * 2, 256) : 0);
  c.bytes = c.at_parts + (c.cuts ? kPartsBytes : 0);
  return c;
}

int check_sizes(const emrs_experts *a) {
  if (!a) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL argument");
  if (a->dtype != EMRS_BF16 && a->dtype != EMRS_FP16) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: operands are bf16 or fp16");
  if (a->n_experts < 1 || a->n_experts > EMRS_EXPERTS_MAX) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: 1 to 256 experts");
  if (a->n_in < 1 || a->n_out < 1 || a->n_in > (1u << 20) || a->n_out > (1u << 20)) return fail(EMRS_ERR_TOO_LARGE, "experts: sides are 1 to 2^20");
  if (a->rows > kMaxRows) return fail(EMRS_ERR_TOO_LARGE, "experts: at most 2^30 - 1 rows");
  return EMRS_OK;
}

// What launches take is estimated, in microseconds, as rounds of workgroups of `fixed` + `stage` for each of a group's
// stages; the constants are fitted to 18 sets of experts, 1 to 256 of them with 16 to 8192 rows in all, at all tiles.  On
// these sets the choice was at most 4% from the best of y, 15% of grad_x, 1% of grad_W; what it decides, for instance:
// 64 uneven experts' 8192 rows, k 1024, m 1376: y 57 us in tiles of 256, 61 of 192, 74 of 128, 132 of 64; 8 experts of
// 30 rows, k and m 4096: 88, 73, 53 and 55; 2 of 128 rows: 73, 58, 37 and 25; 1500 rows, k 4096, m 128: 70, 46, 27, 17 and,
// of 32, 12.

// Tiles of the tokens' rows: of every expert that can have rows one at the least, and half a tile that is not full.
template <class Cfg>
double tiles_expected(const Product &p, uint64_t rows, uint64_t experts) {
  const double most = (double)std::min<uint64_t>(rows, experts), each = (double)rows / Cfg::BN / most;
  return std::min(most * std::max(1.0, each + 0.5), (double)rows) * (double)emrs_gemm::tiles_of(p.m, Cfg::BM);
}

template <class Cfg>
double cost_of(double tiles, double k, double stage, double fixed, bool cuts = false) {
  const double rounds = std::max(1.0, tiles / kRound), stages = std::ceil(std::ceil(k / emrs_gemm::kStage) / Cfg::GROUPS);
  return (rounds < 4 && !cuts ? std::ceil(rounds) : rounds) * (fixed + stage * stages) + (cuts ? 40 : 0);
}

template <class Cfg, class T, bool kTransposed>
int launch_tokens(const Product &p, OfTokens<T, kTransposed> e, uint64_t rows, uint64_t experts, hipStream_t st) {
  // Every segment, that of the rows of none among them, may have one tile that is not full.
  const uint64_t tiles = std::min(rows, rows / Cfg::BN + experts + 1) * (uint64_t)emrs_gemm::tiles_of(p.m, Cfg::BM);
  if (tiles > 0x3fffffff) return fail(EMRS_ERR_TOO_LARGE, "experts: too many tiles for one launch");
  constexpr bool cuts = std::is_same<Cfg, emrs_gemm::Large>::value;
  if (!cuts) e.parts = nullptr;
  emrs_gemm::product_kernel<T, Cfg><<<(uint32_t)tiles + (e.parts ? kRound : 0), Cfg::THREADS, 0, st>>>(p, e);
  if constexpr (cuts)
    if (e.parts) join_tiles_kernel<T, Cfg><<<(kRound - 1) * (Cfg::BN / kJoinRows), 256, 0, st>>>(p, e.counts, e.parts, e.out);
  return EMRS_OK;
}

template <class T, bool kTransposed>
int launch(const Product &p, const OfTokens<T, kTransposed> &e, uint64_t rows, uint64_t experts, hipStream_t st) {
  using namespace emrs_gemm;
  const double k = p.k;
  const double cost[5] = {cost_of<Large>(tiles_expected<Large>(p, rows, experts), k, kTransposed ? 1.45 : 1.5, kTransposed ? 8 : 5.5, e.parts),
                          cost_of<Broad>(tiles_expected<Broad>(p, rows, experts), k, 1.3, 6.5),
                          cost_of<Medium>(tiles_expected<Medium>(p, rows, experts), k, kTransposed ? 1.4 : 1.5, kTransposed ? 4.5 : 5.5),
                          cost_of<Small>(tiles_expected<Small>(p, rows, experts), k, kTransposed ? 1.2 : 1.25, 4),
                          cost_of<Tiny>(tiles_expected<Tiny>(p, rows, experts), k, 0.95, 5)};
  int best = kLarge;
  for (int i = kBroad; i <= kTiny; ++i)
    if (cost[i] < cost[best] && !(kTransposed && (i == kBroad || i == kTiny))) best = i;
  if (best == kLarge) return launch_tokens<Large>(p, e, rows, experts, st);
  if constexpr (!kTransposed) {
    if (best == kBroad) return launch_tokens<Broad>(p, e, rows, experts, st);
    if (best == kTiny) return launch_tokens<Tiny>(p, e, rows, experts, st);
  }
  if (best == kMedium) return launch_tokens<Medium>(p, e, rows, experts, st);
  return launch_tokens<Small>(p, e, rows, experts, st);
}

template <class Cfg, class T>
int launch_weights(const Product &p, const OfWeights<T> &e, hipStream_t st) {
  const int64_t each = emrs_gemm::tiles_of(emrs_gemm::tiles_of(p.m, Cfg::BM) * emrs_gemm::tiles_of(p.n, Cfg::BN), kXcds) * kXcds;
  if (each * p.batch > 0x3fffffff) return fail(EMRS_ERR_TOO_LARGE, "experts: too many tiles for one launch");
  emrs_gemm::product_kernel<T, Cfg><<<(uint32_t)(each * p.batch), Cfg::THREADS, 0, st>>>(p, e);
  return EMRS_OK;
}

template <class T>
int launch(const Product &p, const OfWeights<T> &e, uint64_t rows, hipStream_t st) {
  using namespace emrs_gemm;
  const double k = (double)rows / p.batch;
  const double cost[3] = {cost_of<Large>((double)tile_count<Large>(p), k, 1.7, 8.5), cost_of<Medium>((double)tile_count<Medium>(p), k, 1.8, 3),
                          cost_of<Small>((double)tile_count<Small>(p), k, 2.15, 3.5)};
  const int best = (int)(std::min_element(cost, cost + 3) - cost);
  if (best == 0) return launch_weights<Large>(p, e, st);
  if (best == 1) return launch_weights<Medium>(p, e, st);
  return launch_weights<Small>(p, e, st);
}

template <class T>
void pad(const Table &from, uint32_t matrices, int64_t stride, uint64_t rows, uint64_t columns, T *to, hipStream_t st) {
  const uint64_t padded = round_up(columns, 8), units = rows * (padded / 8);
  const dim3 grid((uint32_t)std::min<uint64_t>((units + 255) / 256, std::max<uint64_t>(1, 8192 / matrices)), matrices);
  pad_rows_kernel<T><<<grid, 256, 0, st>>>(from, stride, rows, (int)columns, (int)padded, to);
}

template <class T>
int run_as(const emrs_experts *a, bool backward, hipStream_t st) {
  const uint64_t in8 = round_up(a->n_in, 8), out8 = round_up(a->n_out, 8);
  const Copies copies = copies_of(a, backward);
  char *const room = static_cast<char *>(a->workspace);
  Counts counts{a->counts, a->counts_bytes == 8, (int32_t)a->n_experts, (int32_t)a->rows};
  Table weights{};
  for (uint32_t e = 0; (!backward || a->grad_x) && e < a->n_experts; ++e) weights.p[e] = a->weights[e];
  const T *x = static_cast<const T *>(a->x), *grad_y = static_cast<const T *>(a->grad_y);
  int64_t x_stride = (int64_t)a->x_stride, weight_stride = (int64_t)a->weight_stride, grad_y_stride = (int64_t)a->grad_y_stride;
  if (copies.x && a->rows) {
    T *const to = reinterpret_cast<T *>(room);
    pad<T>(Table{{x}}, 1, x_stride, a->rows, a->n_in, to, st);
    x = to, x_stride = (int64_t)in8;
  }
  if (copies.weights && a->rows) {
    T *const to = reinterpret_cast<T *>(room + copies.at_weights);
    pad<T>(weights, a->n_experts, weight_stride, a->n_out, a->n_in, to, st);
    for (uint32_t e = 0; e < a->n_experts; ++e) weights.p[e] = to + e * a->n_out * in8;
    weight_stride = (int64_t)in8;
  }
  if (copies.grad_y && a->rows) {
    T *const to = reinterpret_cast<T *>(room + copies.at_grad_y);
    pad<T>(Table{{grad_y}}, 1, grad_y_stride, a->rows, a->n_out, to, st);
    grad_y = to, grad_y_stride = (int64_t)out8;
  }
  float *const parts = copies.cuts ? reinterpret_cast<float *>(room + copies.at_parts) : nullptr;
  int rc = EMRS_OK;
  if (!backward && a->rows) {
    const Product p{nullptr, x, weight_stride, x_stride, 0, 0, (int32_t)a->n_out, 0, (int32_t)in8, emrs_gemm::kNoWrap, emrs_gemm::kNoWrap, 0, 1, 0};
    const OfTokens<T, false> e{weights, counts, a->n_out % 8 == 0 && on(a->y, 16), (int32_t)a->n_out, static_cast<T *>(a->y), parts};
    if (a->rows <= kFew) {
      const uint64_t groups = std::min<uint64_t>(a->rows, a->rows / kFewRows + a->n_experts + 1);
      few_rows_kernel<T><<<dim3((uint32_t)((a->n_out + kFewWeights * kFewWaves - 1) / (kFewWeights * kFewWaves)), (uint32_t)groups), 64 * kFewWaves, 0, st>>>(
          weights, weight_stride, counts, x, x_stride, (int)in8, (int)a->n_out, static_cast<T *>(a->y));
    } else {
      rc = launch<T, false>(p, e, a->rows, a->n_experts, st);
    }
  }
  if (backward && a->grad_x && a->rows) {
    const Product p{nullptr, grad_y, weight_stride, grad_y_stride, 0, 0, (int32_t)a->n_in, 0, (int32_t)out8, emrs_gemm::kNoWrap, emrs_gemm::kNoWrap, 0, 1, 0};
    const OfTokens<T, true> e{weights, counts, a->n_in % 8 == 0 && on(a->grad_x, 16), (int32_t)a->n_out, static_cast<T *>(a->grad_x), parts};
    rc = launch<T, true>(p, e, a->rows, a->n_experts, st);
  }
  if (rc == EMRS_OK && backward && a->grad_weights) {
    const Product p{x, grad_y, x_stride, grad_y_stride, 0, 0, (int32_t)a->n_in, (int32_t)a->n_out, 0, emrs_gemm::kNoWrap, emrs_gemm::kNoWrap, 0,
                    (int32_t)a->n_experts, 0};
    OfWeights<T> e{{}, counts, a->n_in % 8 == 0};
    for (uint32_t i = 0; i < a->n_experts; ++i) e.out.p[i] = a->grad_weights[i], e.wide = e.wide && on(a->grad_weights[i], 16);
    rc = launch<T>(p, e, a->rows, st);
  }
  if (rc) return rc;
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? EMRS_OK : fail(EMRS_ERR_HIP, std::string("experts: ") + hipGetErrorString(e));
}

int run(const emrs_experts *a, bool backward, hipStream_t st) {
  int rc = check_sizes(a);
  if (rc) return rc;
  if (a->counts_bytes != 4 && a->counts_bytes != 8) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: counts are of 4 or 8 bytes");
  if (a->reserved) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: reserved is not 0");
  if (!a->counts) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL counts");
  if (!on(a->counts, a->counts_bytes)) return fail(EMRS_ERR_MISALIGNED, "experts: counts off their type's alignment");
  const bool want_x = !backward || a->grad_weights, want_w = !backward || a->grad_x;
  if (backward && !a->grad_x && !a->grad_weights) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: no gradient is wanted");
  if (want_w) {
    if (!a->weights) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL weights");
    if (a->weight_stride < a->n_in || a->weight_stride > (1u << 21)) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: row strides are from n_in to 2^21");
    for (uint32_t e = 0; e < a->n_experts; ++e) {
      if (!a->weights[e]) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL weight");
      if (!on(a->weights[e], 2)) return fail(EMRS_ERR_MISALIGNED, "experts: a weight off its type's alignment");
    }
  }
  if (backward && a->grad_weights)
    for (uint32_t e = 0; e < a->n_experts; ++e) {
      if (!a->grad_weights[e]) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL gradient of a weight");
      if (!on(a->grad_weights[e], 2)) return fail(EMRS_ERR_MISALIGNED, "experts: a gradient off its type's alignment");
    }
  if (a->rows) {
    if (want_x && !a->x) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL x");
    if (!backward && !a->y) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL y");
    if (backward && !a->grad_y) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL grad_y");
    if (want_x && (a->x_stride < a->n_in || a->x_stride > (1u << 21))) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: row strides are from n_in to 2^21");
    if (backward && (a->grad_y_stride < a->n_out || a->grad_y_stride > (1u << 21)))
      return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: row strides are from n_out to 2^21");
    if (!on(a->x, 2) || !on(a->y, 2) || !on(a->grad_y, 2) || !on(a->grad_x, 2))
      return fail(EMRS_ERR_MISALIGNED, "experts: a buffer off its type's alignment");
    const Copies copies = copies_of(a, backward);
    if (copies.bytes) {
      if (!a->workspace || a->workspace_bytes < copies.bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: the workspace is too small");
      if (!on(a->workspace, 256)) return fail(EMRS_ERR_MISALIGNED, "experts: the workspace is off 256 bytes");
    }
  } else if (!backward || !a->grad_weights) {
    return EMRS_OK;
  }
  rc = emrs_internal::need_device();
  if (rc) return rc;
  return a->dtype == EMRS_BF16 ? run_as<__bf16>(a, backward, st) : run_as<_Float16>(a, backward, st);
}

}  // namespace

extern "C" int emrs_experts_workspace(const emrs_experts *a, int backward, uint64_t *bytes) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    if (!bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "experts: NULL argument");
    const int rc = check_sizes(a);
    if (rc) return rc;
    *bytes = copies_of(a, backward != 0).bytes;
    return EMRS_OK;
  });
}

extern "C" int emrs_experts_forward(const emrs_experts *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    return run(a, false, static_cast<hipStream_t>(stream));
  });
}

extern "C" int emrs_experts_backward(const emrs_experts *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    return run(a, true, static_cast<hipStream_t>(stream));
  });
}
