// Attention within documents, and its gradients, which compute the probabilities again.
//
// For every query i of a document with n queries and m keys (causal: i sees the keys j <= i + m - n):
//   s_ij = scale q_i . k_j,  lse_i = log sum_j exp(s_ij),  p_ij = exp(s_ij - lse_i),  out_i = sum_j p_ij v_j
//   delta_i = grad_out_i . out_i,  d_ij = p_ij (grad_out_i . v_j - delta_i)
//   grad_q_i = scale sum_j d_ij k_j,  grad_k_j = scale sum_i d_ij q_i,  grad_v_j = sum_i p_ij grad_out_i
// where keys of a head get the sums over all query heads that share it.  Nothing of size queries x keys is written.
//
// All three kernels are one scheme.  A wave owns 32 rows of one side (queries; for grad_k and grad_v keys), whose
// operands and sums stay in its registers, and the workgroup walks the other side in tiles that buffer loads put into
// LDS, the next one while this one is worked on.  The product with the tile's rows as m and the wave's as n (32x32x16)
// leaves each lane with 16 values of its own row: softmax sums need one exchange with the other half of the wave, and
// the values, rounded to 16 bits, are where the next product wants its operand b, if that product's k (the tile's
// rows) is taken in the order 0..3, 8..11 | 4..7, 12..15 of each 16.  Operand a, the tile's columns, comes through
// transposing LDS reads in the same order.  So probabilities never leave registers.
//
// Statistics and sums are in 32 bits; p and d are rounded to the operands' type, as the matrix instructions take
// them (two parts of every d would be a third more products in grad_q, and there are no registers for them in grad_k).
// fp16 holds p and d scaled by powers of two.  Of p, forward keeps all bits down to 2^-21 of a row's largest (scaled by
// 2^7, with room for a maximum that grows) and grad_v down to 2^-29 (by 2^15); of d, each row of grad_q and of grad_k down
// to 2^-20 of the largest of its own sum (Lift).  No result passes through atomics: the same call gives the same bits.
//
// What bounds it: the matrix units, with the arithmetic of the softmax beside them.  4096 rows, 32 heads of 128, causal, one
// call behind the other: forward 145 to 147 us (0.94 PFLOP/s), the two backward kernels 472 to 487 (1.0 PFLOP/s of what they
// execute); in fp16 152 and 531 to 540.  Under the profiler, mean and least: forward 172 and 158 us, with matrix instructions in
// 51% of the cycles that a CU is busy, grad_q 236 and 218, 57%, grad_k and grad_v 297 and 273, 60%.  With a query or a few to
// many keys, reading these: 64 single tokens to 8192 keys each, 5.9 TB/s.

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

using emrs_gemm::arrive;
using emrs_gemm::kXcds;
using emrs_internal::fail;

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int kWaves = 4, kThreads = kWaves * 64;
constexpr int kOwn = 32 * kWaves;  // rows of a workgroup's own side
constexpr int kTile = 64;          // rows of the other side in LDS
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ inline f32x16 mfma(emrs_gemm::bf16x8 a, emrs_gemm::bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma(emrs_gemm::fp16x8 a, emrs_gemm::fp16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ int lane_of() { return threadIdx.x & 63; }
// The row, among a product's 32, of a lane's value r.
__device__ __forceinline__ int row_of(int r) { return (r >> 2) * 8 + (lane_of() >> 5) * 4 + (r & 3); }

// ---- documents ----

// Where documents begin and end in one side's rows.  Segment 0 are the rows before the first document, segment i the
// i-th document, the last one the rows behind all documents; those of no document see nothing.
struct Bounds {
  const void *offsets;  // [documents + 1]; NULL: documents of equal length
  int32_t bytes, documents, rows, each;
  int32_t fold;  // of a row here, heads of a query that count as rows

  __device__ __forceinline__ int all() const { return rows * fold; }
  __device__ __forceinline__ int at(int i) const {  // i <= documents
    if (!offsets) return i * each * fold;
    if (bytes == 8) return (int)min(max(static_cast<const int64_t *>(offsets)[i], (int64_t)0), (int64_t)rows) * fold;
    return min(max(static_cast<const int32_t *>(offsets)[i], 0), rows) * fold;
  }
};

struct Span {
  int first, end;
};

// This lane's segment, of at most 64: ends that never go back, and tiles up to and with it.
struct Walk {
  int first, end, tiles;

  __device__ __forceinline__ explicit Walk(const Bounds &b) {
    const int e = lane_of();
    end = e <= b.documents ? b.at(e) : b.all();
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int before = __shfl_up(end, o);
      if (lane_of() >= o) end = max(end, before);
    }
    const int below = __shfl_up(end, 1);
    first = lane_of() ? below : 0;
    tiles = (end - first + kOwn - 1) / kOwn;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int before = __shfl_up(tiles, o);
      if (lane_of() >= o) tiles += before;
    }
  }
  __device__ __forceinline__ Span span(int lane) const { return {__builtin_amdgcn_readlane(first, lane), __builtin_amdgcn_readlane(end, lane)}; }
};
// Documents that are walked; with the rows before and behind them they are a wave's lanes.  More of them have their
// tiles listed by a launch of its own.  (Forward and backward of 32 heads of 128, listed and walked: 60 documents of 64
// rows 183 us and 172; walked in steps of 64, 100 documents 229 and 266, 256 documents 519 and 826, 1024 of 8 rows 1180
// and 4199.)
constexpr uint64_t kWalked = 62;

struct Place {
  Span own, other;  // the document's rows on both sides
  int row;          // the workgroup's first row, from the document's first
  int head, split;
};

// Where a tile's rows lie, as attention_places_kernel leaves it for every tile of a side with many documents.
struct Entry {
  Span own, other;
  int row;
};
struct Places {
  int tiles;
  Entry tile[1];
};

// The workgroup's place in a launch of any size: see lines_of().
__device__ __forceinline__ uint32_t block_of() { return blockIdx.y * gridDim.x + blockIdx.x; }

// The workgroup's tile, of `tiles` for each head and split, its head and its split; false: there is none for it.  Each
// XCD gets a run of consecutive places, heads that share keys one after the other: whole heads where they divide by the
// XCDs.  Within it the last rows come first, whose causal work is the longest (grad_k: the first).
template <bool kLastFirst>
__device__ __forceinline__ bool pick(uint32_t tiles, int heads, int splits, Place &at, int &own_tile) {
  const uint32_t block = block_of(), total = tiles * heads * splits;
  const uint32_t q = total / kXcds, r = total % kXcds, x = block % kXcds, nth = block / kXcds;
  if (nth >= q + (x < r ? 1 : 0)) return false;
  // Causal work falls along the places: of those that fill a XCD's CUs twice, the second half goes backwards, so that
  // each CU begins with the same sum (4096 rows, 32 heads: 157 us against 161, grad_q 207 against 214).
  constexpr uint32_t kCus = 32;
  uint32_t t = x * q + min(x, r) + (q >= 2 * kCus && nth >= kCus && nth < 2 * kCus ? 3 * kCus - 1 - nth : nth);
  const uint32_t chunk = (heads % kXcds ? 1 : heads / kXcds) * splits, each = chunk * tiles;
  const uint32_t first_head = t / each * chunk;
  t -= t / each * each;
  const uint32_t tile = t / chunk, unit = first_head + t % chunk;
  at.head = unit / splits, at.split = unit % splits;
  own_tile = (int)(kLastFirst ? tiles - 1 - tile : tile);
  return true;
}

// The workgroup's rows, head and share of the other side; false: there are none for it.  Documents of one length are
// counted off, others are walked by every workgroup for itself, one a lane, or, more than there are lanes, looked up.
template <bool kLastFirst>
__device__ __forceinline__ bool find(const Bounds &own, const Bounds &other, const Places *places, int heads, int splits, Place &at) {
  int tile;
  if (!own.offsets) {
    const int each_has = (own.each * own.fold + kOwn - 1) / kOwn;
    if (!pick<kLastFirst>((uint32_t)each_has * own.documents, heads, splits, at, tile)) return false;
    const int document = tile / each_has;
    at.own = {own.at(document), own.at(document + 1)}, at.other = {other.at(document), other.at(document + 1)};
    at.row = (tile - document * each_has) * kOwn;
    return true;
  }
  if (places) {
    if (!pick<kLastFirst>((uint32_t)places->tiles, heads, splits, at, tile)) return false;
    const Entry &e = places->tile[tile];
    at.own = e.own, at.other = e.other, at.row = e.row;
    return true;
  }
  const Walk walk(own);
  if (!pick<kLastFirst>((uint32_t)__builtin_amdgcn_readlane(walk.tiles, 63), heads, splits, at, tile)) return false;
  const int segment = __builtin_ctzll(__ballot(tile < walk.tiles));  // tile is less than all tiles
  at.own = walk.span(segment);
  at.row = (tile - __builtin_amdgcn_readlane(walk.tiles, segment) + (at.own.end - at.own.first + kOwn - 1) / kOwn) * kOwn;
  at.other = {0, 0};
  if (segment > 0 && segment <= own.documents) {
    // One tensor of offsets, held within as many rows of as many heads each, gives one span.
    const bool one = own.offsets == other.offsets && own.rows == other.rows && own.fold == other.fold;
    at.other = one ? at.own : Walk(other).span(segment);
  }
  return true;
}

// Inclusive maximum or sum over a workgroup's threads, and over all of them.
constexpr int kPlaceThreads = 1024;
template <class Op>
__device__ __forceinline__ int scan(int v, int *room, int &all, Op op) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int before = __shfl_up(v, o);
    if (lane_of() >= o) v = op(v, before);
  }
  const int wave = threadIdx.x / 64;
  __syncthreads();
  if (lane_of() == 63) room[wave] = v;
  __syncthreads();
  for (int i = 0; i < wave; ++i) v = op(v, room[i]);
  all = room[0];
  for (int i = 1; i < kPlaceThreads / 64; ++i) all = op(all, room[i]);
  return v;
}

// The tiles of the queries' side (workgroup 0) and of the keys' (1), each document's by a thread.
__global__ __launch_bounds__(kPlaceThreads) void attention_places_kernel(Bounds queries, Bounds keys, Places *of_queries, Places *of_keys) {
  __shared__ int room[kPlaceThreads / 64], last[2];  // last: ends of the thread before
  __shared__ int ends[2][kPlaceThreads];
  const Bounds &own = blockIdx.x ? keys : queries, &other = blockIdx.x ? queries : keys;
  Places *const places = blockIdx.x ? of_keys : of_queries;
  if (threadIdx.x < 2) last[threadIdx.x] = 0;
  const int segments = own.documents + 2;
  auto most = [](int a, int b) { return max(a, b); };
  auto sum = [](int a, int b) { return a + b; };
  int tiles_before = 0;
  for (int from = 0; from < segments; from += kPlaceThreads) {
    const int segment = from + (int)threadIdx.x;
    __syncthreads();
    const int own_before = last[0], other_before = last[1];
    int all_own, all_other, all_tiles;
    const int end = max(scan(segment <= own.documents ? own.at(segment) : own.all(), room, all_own, most), own_before);
    const int other_end = max(scan(segment <= own.documents ? other.at(segment) : other.all(), room, all_other, most), other_before);
    ends[0][threadIdx.x] = end, ends[1][threadIdx.x] = other_end;
    __syncthreads();
    Entry e;
    e.own = {threadIdx.x ? ends[0][threadIdx.x - 1] : own_before, end};
    const bool document = segment > 0 && segment <= own.documents;
    e.other = {document ? (threadIdx.x ? ends[1][threadIdx.x - 1] : other_before) : 0, document ? other_end : 0};
    const int tiles = (e.own.end - e.own.first + kOwn - 1) / kOwn, upto = scan(tiles, room, all_tiles, sum) + tiles_before;
    for (int i = 0; i < tiles; ++i) {
      e.row = i * kOwn;
      places->tile[upto - tiles + i] = e;
    }
    tiles_before += all_tiles;
    if (threadIdx.x == 0) last[0] = max(own_before, all_own), last[1] = max(other_before, all_other);
  }
  if (threadIdx.x == 0) places->tiles = tiles_before;
}

// ---- tiles ----

// A tile's rows in LDS: DIM 16-bit elements each, in units of 16 bytes that are permuted by the row.  Both kinds of
// reads then meet 16 different units of the 64 banks: 16 rows at one unit (a product's operand of rows), and four rows
// at four units (one of columns).
template <int DIM>
__device__ __forceinline__ int permuted(int row) {
  return DIM == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

// What a lane loads of every tile of ROWS rows of an operand: 16 bytes of each of its wave's kilobytes.
template <class T, int DIM, int WAVES = kWaves, int ROWS = kTile>
struct TileLoader {
  static constexpr int kUnits = DIM / 8, kRows = 64 / kUnits, kLoads = ROWS / (kRows * WAVES);
  int offset, step, stride, dim;
  __device__ __forceinline__ void init(int64_t row_stride, int dim_, int wave) {
    const int row = wave * kRows + lane_of() / kUnits, unit = lane_of() % kUnits ^ permuted<DIM>(row);
    static_assert(kRows * WAVES % 16 == 0 && kLoads * kRows * WAVES == ROWS, "a lane's rows are permuted alike");
    stride = (int)row_stride * 2, dim = dim_ * 2, step = kRows * WAVES * stride;
    offset = unit * 8 < dim_ ? row * stride + unit * 16 : (int)0x80000000;  // past the end: zeros
  }
  // `rows` rows from `first` on (more than a tile's: a tile's; less: zeros behind them; none: zeros).
  __device__ __forceinline__ void load(char *lds, const T *first, int rows, int wave) const {
    rows = min(rows, ROWS);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(first), 0, rows > 0 ? (rows - 1) * stride + dim : 0, 0x00020000);
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + (j * WAVES + wave) * 1024), 16,
                                               offset < 0 ? offset : offset + j * step, 0, 0, 0);
  }
};

// A lane's places in a tile for the reads of both kinds.
template <class T, int DIM>
struct TileReader {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  static constexpr int kRow = DIM * 2;
  int by_rows, by_columns;
  __device__ __forceinline__ void init() {
    const int lane = lane_of(), row = lane & 31, half = lane >> 5, t = lane & 15;
    by_rows = row * kRow + ((half ^ permuted<DIM>(row)) << 4);
    const int four = half * 4 + (t >> 2);  // the row of the first four; those of the second four are 8 further
    by_columns = four * kRow + ((((lane >> 4 & 1) * 2 + (t >> 1 & 1)) ^ permuted<DIM>(four)) << 4) + (t & 1) * 8;
  }
  // Rows block * 32 .. + 31 as operand a, 16 of their elements from 16 c on.
  __device__ __forceinline__ x8 rows(const char *tile, int block, int c) const {
    return *reinterpret_cast<const x8 *>(tile + (by_rows ^ c << 5) + block * 32 * kRow);
  }
  // Columns 32 d .. + 31 as operand a: 16 rows from 16 c on, in the order in which a lane holds its values.
  __device__ __forceinline__ x8 columns(const char *tile, int d, int c) const {
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    typedef __attribute__((address_space(3))) s16x4 *lds4;
    char *const at = const_cast<char *>(tile) + c * 16 * kRow;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + (by_columns ^ d << 6)));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * kRow + (by_columns ^ d << 6 ^ 32)));
    return __builtin_bit_cast(x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// A wave's own rows as operand b: row lane % 32, eight elements from 16 c + 8 (lane / 32) on.
template <class T, int DIM>
struct OwnRows {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  x8 v[DIM / 16];
  __device__ __forceinline__ void load(const T *row, bool valid, int dim) {
#pragma unroll
    for (int c = 0; c < DIM / 16; ++c) {
      const int at = c * 16 + (lane_of() >> 5) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = (T)0.f;
      if (valid && at < dim) v[c] = *reinterpret_cast<const x8 *>(row + at);
    }
  }
};

// Products in a row: use(i, fragment) of each, with what comes D products later read right behind it, so that no
// product waits for its own read.  The order is pinned: left to itself, where registers are short, the compiler reads
// every fragment just before its product.  first(): the reads of the first D, to be started earlier.
template <int N, int D, class F>
struct Products {
  F f[D];
  template <class Read>
  __device__ __forceinline__ void first(Read read) {
#pragma unroll
    for (int i = 0; i < D; ++i) f[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
  }
  template <class Read, class Use>
  __device__ __forceinline__ void run(Read read, Use use) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      use(i, f[i % D]);
      if (i + D < N) f[i % D] = read(i + D);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Eight of a lane's 16 values, in 16 bits, as operand b of the next product.
template <class T>
__device__ __forceinline__ typename emrs_gemm::Vec<T>::x8 eight_of(const f32x16 &v, int half) {
  typename emrs_gemm::Vec<T>::x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (T)v[half * 8 + e];
  return o;
}

// What that rounding left over.
template <class T>
__device__ __forceinline__ typename emrs_gemm::Vec<T>::x8 rest_of_eight(const f32x16 &v, int half) {
  typename emrs_gemm::Vec<T>::x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (T)(v[half * 8 + e] - (float)(T)v[half * 8 + e]);
  return o;
}

// Both halves of the wave's values, exchanged without a way through LDS.
__device__ __forceinline__ float2 both_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ float sum_of_halves(float v) {
  const float2 x = both_halves(v);
  return x.x + x.y;
}
__device__ __forceinline__ float most_of_halves(float v) {
  const float2 x = both_halves(v);
  return fmaxf(x.x, x.y);
}

struct Strides {
  int64_t row, head;
};

struct Attention {
  Bounds queries, keys;
  const Places *query_places, *key_places;  // NULL: they are found without
  const void *q, *k, *v, *grad_out;
  Strides q_at, k_at, v_at, grad_out_at;
  int32_t heads, group, dim, real_dim, causal, splits, wide_out, wide_grads;  // dim: of the operands' rows, a multiple of 8; real_dim: of the outputs'
  float scale;           // of the scores
  void *out, *rest;      // [rows][heads][real_dim]: the output, and what its rounding left over
  float *lse;            // [heads][rows]
  float *exponent, *delta;  // the same, backward: lse in units of log 2 (infinity where a query sees nothing), and delta
  void *grad_q, *grad_k, *grad_v;
  float *parts, *parts2, *part_lse;  // of every split, where there are several
};

// What rounding x to `rounded` left over (nothing of infinities and NaN).
template <class T>
__device__ __forceinline__ T rest_of(float x, T rounded) {
  const float left = x - (float)rounded;
  return fabsf(left) < INFINITY ? (T)left : (T)0.f;
}

// A wave's sums, held as [column][row], to the rows of an output: turned over in the wave's own part of LDS, whose
// units of 16 bytes are permuted by the row, so that rows are stored in whole lines (straight from registers, eight
// bytes a lane, the two outputs of 8192 x 32 x 128 took 25 us longer).
template <class V, int DIM>
struct RowStore {
  static constexpr int kEach = 16 / sizeof(V), kUnits = DIM / kEach, kMask = kUnits < 16 ? kUnits - 1 : 15;
  static __device__ __forceinline__ int at(int row, int unit) { return (row * kUnits + (unit ^ (row & kMask))) * 16; }
  // value(d, r): of the lane's row, in 32 bits.  rows: how many of the wave's rows there are; from(row): where one is.
  template <class Value, class From>
  static __device__ __forceinline__ void store(char *room, Value value, V *to, From from, int rows, int dim, bool wide) {
    typedef __attribute__((ext_vector_type(4))) V v4;
    typedef __attribute__((ext_vector_type(kEach))) V unit_t;
    const int lane = lane_of();
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        v4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (V)value(d, r + e);
        const int column = d * 32 + row_of(r);
        *reinterpret_cast<v4 *>(room + at(lane & 31, column / kEach) + column % kEach * sizeof(V)) = v;
      }
#pragma unroll
    for (int pass = 0; pass < kUnits / 2; ++pass) {
      const int row = pass * (64 / kUnits) + lane / kUnits, unit = lane % kUnits;
      const unit_t v = *reinterpret_cast<const unit_t *>(room + at(row, unit));
      if (row >= rows || unit * kEach >= dim) continue;
      V *const out = to + from(row) + unit * kEach;
      if (wide) {
        *reinterpret_cast<unit_t *>(out) = v;
      } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (unit * kEach + e < dim) out[e] = v[e];
      }
    }
  }
};

// A split's run of tiles.
__device__ __forceinline__ Span share_of(int tiles, int split, int splits) {
  return {(int)((int64_t)tiles * split / splits), (int)((int64_t)tiles * (split + 1) / splits)};
}

// ---- forward ----

// kFold: the heads that share a key are rows of one tile, whose queries' documents are short.
template <class T, int DIM, bool kFold>
__global__ __launch_bounds__(kThreads, DIM == 64 ? 4 : 2) void attention_forward_kernel(Attention p) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  constexpr int kBytes = kTile * DIM * 2;
  __shared__ __attribute__((aligned(1024))) char k_even[kBytes];
  __shared__ __attribute__((aligned(1024))) char k_odd[kBytes];
  __shared__ __attribute__((aligned(1024))) char v_even[kBytes];
  __shared__ __attribute__((aligned(1024))) char v_odd[kBytes];
  Place at;
  const int fold = kFold ? p.group : 1;
  if (!find<true>(p.queries, p.keys, p.query_places, kFold ? p.heads / p.group : p.heads, p.splits, at)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_of();
  const int queries = at.own.end - at.own.first, keys = at.other.end - at.other.first;
  const int mine = at.row + wave * 32, query = mine + (lane & 31), kv_head = kFold ? at.head : at.head / p.group;
  const bool valid = query < queries;
  const int64_t row = (at.own.first + query) / fold;
  const int head = at.head * fold + (at.own.first + query) % fold;

  OwnRows<T, DIM> q;
  q.load(static_cast<const T *>(p.q) + row * p.q_at.row + head * p.q_at.head, valid, p.dim);

  // Keys that the workgroup's, the wave's and the lane's last query sees.
  const int shift = keys - queries / fold;
  auto seen_by = [&](int i) { return p.causal ? min(max(min(i, queries - 1) / fold + shift + 1, 0), keys) : keys; };
  const int seen = seen_by(at.row + kOwn - 1), seen_wave = mine < queries ? seen_by(mine + 31) : 0, seen_lane = seen_by(query), seen_by_all = seen_by(mine);
  const Span tiles = share_of((seen + kTile - 1) / kTile, at.split, p.splits);

  TileLoader<T, DIM> k_loader, v_loader;
  k_loader.init(p.k_at.row, p.dim, wave);
  v_loader.init(p.v_at.row, p.dim, wave);
  TileReader<T, DIM> reader;
  reader.init();
  const T *const k = static_cast<const T *>(p.k) + at.other.first * p.k_at.row + kv_head * p.k_at.head;
  const T *const v = static_cast<const T *>(p.v) + at.other.first * p.v_at.row + kv_head * p.v_at.head;
  auto load = [&](char *to_k, char *to_v, int t) __attribute__((always_inline)) {
    const int rows = t < tiles.end ? keys - t * kTile : 0;
    const int64_t from = rows > 0 ? t * kTile : 0;
    k_loader.load(to_k, k + from * p.k_at.row, rows, wave);
    v_loader.load(to_v, v + from * p.v_at.row, rows, wave);
  };

  const float by = p.scale * kLog2e;
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  constexpr float kLift = kHalf ? 7.f : 0.f, kSlack = 8.f;  // exponents are kept below kLift + kSlack
  f32x16 out[DIM / 32];
#pragma unroll
  for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) out[d][r] = 0.f;
  float top = -INFINITY, sum = 0.f;  // top: what exponents are taken off, in units of log 2; sum: this lane's part

  auto work = [&](const char *kt, const char *vt, int t) __attribute__((always_inline)) {
    const int from = t * kTile;
    if (from >= seen_wave) return;
    constexpr int kC = DIM / 16, kD = DIM / 32;
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
    Products<2 * kC, 4, x8> scores;
    auto key_rows = [&](int i) __attribute__((always_inline)) { return reader.rows(kt, i % 2, i / 2); };
    scores.first(key_rows);
    scores.run(key_rows, [&](int i, const x8 &f) __attribute__((always_inline)) { s[i % 2] = mfma(f, q.v[i / 2], s[i % 2]); });
    Products<4 * kD, 4, x8> sums;
    auto columns = [&](int i) __attribute__((always_inline)) { return reader.columns(vt, i % kD, i / kD); };
    sums.first(columns);
    if (from + kTile > seen_by_all) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (from + b * 32 + row_of(r) >= seen_lane) s[b][r] = -INFINITY;
    }
    float tops[4];  // in four chains: one would be 16 dependent instructions
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      tops[i] = s[i >> 1][(i & 1) * 8];
#pragma unroll
      for (int r = 1; r < 8; ++r) tops[i] = fmaxf(tops[i], s[i >> 1][(i & 1) * 8 + r]);
    }
    const float most = most_of_halves(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))) * by;
    // The sums are brought to a new maximum only where exponents would grow past the slack.
    if (__any(most > top + kSlack)) {
      const float next = fmaxf(top, most), less = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - next);
      sum *= less;
#pragma unroll
      for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[d][r] *= less;
      top = next;
    }
    const float off = (top == -INFINITY ? 0.f : top) - kLift;
    // Values 2 n and 2 n + 1 of the tile: the first eight before any product with v, the others between them, eight ahead.
    auto exponentials = [&](int n) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[n / 8][n % 8 * 2 + e], by, -off));
        s[n / 8][n % 8 * 2 + e] = x;
        sum += x;
      }
    };
#pragma unroll
    for (int n = 0; n < 4; ++n) exponentials(n);
    x8 prob = eight_of<T>(s[0], 0);
    sums.run(columns, [&](int i, const x8 &f) __attribute__((always_inline)) {
      const int c = i / kD, d = i % kD;
      if (i && d == 0) prob = eight_of<T>(s[c >> 1], c & 1);
      out[d] = mfma(f, prob, out[d]);
      if (c < 3)
#pragma unroll
        for (int n = 0; n < 4 / kD; ++n) exponentials((c + 1) * 4 + d * (4 / kD) + n);
    });
  };

  load(k_even, v_even, tiles.first);
  for (int t = tiles.first; t < tiles.end; t += 2) {
    arrive();
    load(k_odd, v_odd, t + 1);
    work(k_even, v_even, t);
    if (t + 1 >= tiles.end) break;
    arrive();
    load(k_even, v_even, t + 2);
    work(k_odd, v_odd, t + 1);
  }
  arrive();  // no load may still be on its way into LDS that another workgroup gets

  sum = sum_of_halves(sum);
  const float lse = sum == 0.f ? -INFINITY : (top - kLift) * kLn2 + logf(sum);
  const float norm = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t stride = (int64_t)p.heads * p.real_dim;
  auto place = [&](int i) __attribute__((always_inline)) {  // of the wave's row i
    const int at_row = at.own.first + mine + i;
    return ((int64_t)(at_row / fold) * p.heads + at.head * fold + at_row % fold) * p.real_dim;
  };
  char *const room = wave == 0 ? k_even : wave == 1 ? k_odd : wave == 2 ? v_even : v_odd;
  const int rows = queries - mine;
  auto value = [&](int d, int r) { return out[d][r] * norm; };
  if (p.splits > 1) {
    if (valid && lane < 32) p.part_lse[((int64_t)at.split * p.heads + head) * p.queries.rows + row] = lse;
    RowStore<float, DIM>::store(room, value, p.parts + (int64_t)at.split * p.queries.rows * stride, place, rows, p.real_dim, p.real_dim % 4 == 0);
    return;
  }
  if (valid && lane < 32 && p.lse) p.lse[(int64_t)head * p.queries.rows + row] = lse;
  RowStore<T, DIM>::store(room, value, static_cast<T *>(p.out), place, rows, p.real_dim, p.wide_out);
  if (p.rest)
    RowStore<T, DIM>::store(room, [&](int d, int r) { return (float)rest_of<T>(value(d, r), (T)value(d, r)); }, static_cast<T *>(p.rest), place, rows, p.real_dim,
                            p.wide_out);
}

// Joins the splits' outputs: four elements a thread where heads are whole units of four, and one else.
template <class T, int E>
__global__ __launch_bounds__(256) void attention_join_kernel(const float *parts, const float *part_lse, int splits, int64_t rows, int heads, int dim, T *out,
                                                             T *rest, float *lse) {
  typedef __attribute__((ext_vector_type(E))) float fE;
  typedef __attribute__((ext_vector_type(E))) T tE;
  const int units = dim / E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = rows * heads * units, unit = i / units;  // row * heads + head
  if (i >= all) return;
  const int64_t row = unit / heads, head = unit % heads;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, part_lse[(s * heads + head) * rows + row]);
  const float shift = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  fE v;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float w = __builtin_amdgcn_exp2f((part_lse[(s * heads + head) * rows + row] - shift) * kLog2e);
    const fE x = *reinterpret_cast<const fE *>(parts + (s * all + i) * E);
    sum += w;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = w == 0.f ? v[e] : fmaf(w, x[e], v[e]);  // NaN is not 0
  }
  const float norm = sum == 0.f ? 0.f : 1.f / sum;
  tE o, left;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    o[e] = (T)(v[e] * norm);
    left[e] = rest_of<T>(v[e] * norm, o[e]);
  }
  *reinterpret_cast<tE *>(out + i * E) = o;
  if (rest) *reinterpret_cast<tE *>(rest + i * E) = left;
  if (i % units == 0 && lse) lse[head * rows + row] = sum == 0.f ? -INFINITY : shift + logf(sum);
}

// Sums of every split's part, E elements a thread.
template <class T, int E>
__global__ __launch_bounds__(256) void attention_sum_kernel(const float *parts, int splits, int64_t each, T *out) {
  typedef __attribute__((ext_vector_type(E))) float fE;
  typedef __attribute__((ext_vector_type(E))) T tE;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * E;
  if (i >= each) return;
  fE v = *reinterpret_cast<const fE *>(parts + i);
#pragma unroll 4
  for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const fE *>(parts + s * each + i);
  tE o;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = (T)v[e];
  *reinterpret_cast<tE *>(out + i) = o;
}

// ---- backward ----

// fp16: the power of two that a lane's d are multiplied by on their way into products.  It goes by the largest |d| of the
// lane's own row (of its key in grad_k) so far, with room for a 2^8 times larger one: beyond that the row's sums are
// brought to a new one, as those of forward to a new maximum.  Other rows, and what stands in rows of no document, do not
// count.  (With one power of two for all rows, from the largest entries of grad_out and v, grad_q of rows whose grad_out
// was 2^-16 of the largest was 9.7e-3 off, now 3.1e-4; 6e4 in rows of no document changed all gradients; and the search for
// these entries cost more: 4096 rows, 32 heads of 128, forward and backward 781 us against 700.)
template <class T>
struct Lift {
  static constexpr bool kAny = std::is_same<T, _Float16>::value;
  static constexpr int kMost = 15, kRoom = 8, kLeast = -85;
  float limit = 0x1p-85f;  // a power of two: |d| up to it become 2^15 at most
  __device__ __forceinline__ float by() const { return kAny ? __uint_as_float(((254u + kMost) << 23) - __float_as_uint(limit)) : 1.f; }  // 2^15 / limit

  template <int N>
  __device__ __forceinline__ void apply(f32x16 &d, f32x16 (&sums)[N]) {
    if constexpr (kAny) {
      float most = fabsf(d[0]);
#pragma unroll
      for (int r = 1; r < 16; ++r) most = fmaxf(most, fabsf(d[r]));  // NaN is passed over
      most = most_of_halves(most);
      if (__any(most > limit)) {
        const float before = limit;  // (the exponent of an infinity is 0)
        if (most > limit) limit = fmaxf(limit, __builtin_amdgcn_ldexpf(1.f, max(__builtin_amdgcn_frexp_expf(most) + kRoom, kLeast)));
        const float less = before / limit;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) sums[n][r] *= less;
      }
      const float x = by();
#pragma unroll
      for (int r = 0; r < 16; ++r) d[r] *= x;
    }
  }
};

// grad_q, and on the way delta and the exponent (split 0 leaves them for grad_k).
template <class T, int DIM>
__global__ __launch_bounds__(kThreads, DIM == 64 ? 3 : 2) void attention_grad_q_kernel(Attention p) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  constexpr int kBytes = kTile * DIM * 2;
  __shared__ __attribute__((aligned(1024))) char k_even[kBytes];
  __shared__ __attribute__((aligned(1024))) char k_odd[kBytes];
  __shared__ __attribute__((aligned(1024))) char v_even[kBytes];
  __shared__ __attribute__((aligned(1024))) char v_odd[kBytes];
  Place at;
  if (!find<true>(p.queries, p.keys, p.query_places, p.heads, p.splits, at)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_of();
  const int queries = at.own.end - at.own.first, keys = at.other.end - at.other.first;
  const int mine = at.row + wave * 32, query = mine + (lane & 31), kv_head = at.head / p.group;
  const bool valid = query < queries;
  const int64_t row = at.own.first + query, place = (row * p.heads + at.head) * p.real_dim;

  OwnRows<T, DIM> q, g;
  q.load(static_cast<const T *>(p.q) + row * p.q_at.row + at.head * p.q_at.head, valid, p.dim);
  g.load(static_cast<const T *>(p.grad_out) + row * p.grad_out_at.row + at.head * p.grad_out_at.head, valid, p.dim);
  float delta = 0.f, lse = INFINITY;
  if (valid) {
    // Of the output before its rounding, as far as it was kept: delta's error is one of every d of the row.
    const T *const out = static_cast<const T *>(p.out) + place, *const rest = p.rest ? static_cast<const T *>(p.rest) + place : nullptr;
    if (p.wide_out) {
      OwnRows<T, DIM> a, b;
      a.load(out, true, p.real_dim);
      b.load(rest, rest != nullptr, p.real_dim);
#pragma unroll
      for (int c = 0; c < DIM / 16; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)g.v[c][e], (float)a.v[c][e] + (float)b.v[c][e], delta);
    } else {
#pragma unroll
      for (int c = 0; c < DIM / 16; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = c * 16 + (lane >> 5) * 8 + e;
          if (d < p.real_dim) delta = fmaf((float)g.v[c][e], (float)out[d] + (rest ? (float)rest[d] : 0.f), delta);
        }
    }
    lse = p.lse[(int64_t)at.head * p.queries.rows + row] * kLog2e;
    if (lse == -INFINITY) lse = INFINITY;  // sees nothing: probabilities of 0
  }
  delta = sum_of_halves(delta);
  if (valid && lane < 32 && at.split == 0) {
    p.exponent[(int64_t)at.head * p.queries.rows + row] = lse;
    p.delta[(int64_t)at.head * p.queries.rows + row] = delta;
  }
  if (!p.grad_q) return;  // of gradients of keys and values alone, these are all that is wanted

  const int shift = keys - queries;
  auto seen_by = [&](int i) { return p.causal ? min(max(min(i, queries - 1) + shift + 1, 0), keys) : keys; };
  const int seen = seen_by(at.row + kOwn - 1), seen_wave = mine < queries ? seen_by(mine + 31) : 0, seen_lane = seen_by(query), seen_by_all = seen_by(mine);
  const Span tiles = share_of((seen + kTile - 1) / kTile, at.split, p.splits);

  TileLoader<T, DIM> k_loader, v_loader;
  k_loader.init(p.k_at.row, p.dim, wave);
  v_loader.init(p.v_at.row, p.dim, wave);
  TileReader<T, DIM> reader;
  reader.init();
  const T *const k = static_cast<const T *>(p.k) + at.other.first * p.k_at.row + kv_head * p.k_at.head;
  const T *const v = static_cast<const T *>(p.v) + at.other.first * p.v_at.row + kv_head * p.v_at.head;
  auto load = [&](char *to_k, char *to_v, int t) __attribute__((always_inline)) {
    const int rows = t < tiles.end ? keys - t * kTile : 0;
    const int64_t from = rows > 0 ? t * kTile : 0;
    k_loader.load(to_k, k + from * p.k_at.row, rows, wave);
    v_loader.load(to_v, v + from * p.v_at.row, rows, wave);
  };
  const float by = p.scale * kLog2e;
  Lift<T> lift;

  f32x16 acc[DIM / 32];
#pragma unroll
  for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;

  auto work = [&](const char *kt, const char *vt, int t) __attribute__((always_inline)) {
    const int from = t * kTile;
    if (from >= seen_wave) return;
    constexpr int kC = DIM / 16, kD = DIM / 32;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
      Products<2 * kC, 4, x8> scores;
      auto rows = [&](int i) __attribute__((always_inline)) { return reader.rows(i % 2 ? vt : kt, b, i / 2); };
      scores.first(rows);
      scores.run(rows, [&](int i, const x8 &f) __attribute__((always_inline)) {
        if (i % 2)
          dp = mfma(f, g.v[i / 2], dp);
        else
          s = mfma(f, q.v[i / 2], s);
      });
      Products<2 * kD, 4, x8> sums;
      auto columns = [&](int i) __attribute__((always_inline)) { return reader.columns(kt, i % kD, b * 2 + i / kD); };
      sums.first(columns);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], by, -lse)) * (dp[r] - delta);
      if (from + kTile > seen_by_all) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (from + b * 32 + row_of(r) >= seen_lane) s[r] = 0.f;
      }
      lift.apply(s, acc);
      if (from + kTile > seen_by_all) {
        // Tiles that the mask cuts hold all that the first queries of a document see, whose gradients are the largest:
        // here d is taken in two parts (4096 rows, 32 heads of 128: error 2.43e-3 against 2.50e-3, 209 us against 204).
#pragma unroll
        for (int i = 0; i < 2 * kD; ++i) acc[i % kD] = mfma(columns(i), rest_of_eight<T>(s, i / kD), acc[i % kD]);
      }
      const x8 ds[2] = {eight_of<T>(s, 0), eight_of<T>(s, 1)};
      sums.run(columns, [&](int i, const x8 &f) __attribute__((always_inline)) { acc[i % kD] = mfma(f, ds[i / kD], acc[i % kD]); });
    }
  };

  load(k_even, v_even, tiles.first);
  for (int t = tiles.first; t < tiles.end; t += 2) {
    arrive();
    load(k_odd, v_odd, t + 1);
    work(k_even, v_even, t);
    if (t + 1 >= tiles.end) break;
    arrive();
    load(k_even, v_even, t + 2);
    work(k_odd, v_odd, t + 1);
  }
  arrive();
  const int64_t corner = ((int64_t)(at.own.first + mine) * p.heads + at.head) * p.real_dim, stride = (int64_t)p.heads * p.real_dim;
  char *const room = wave == 0 ? k_even : wave == 1 ? k_odd : wave == 2 ? v_even : v_odd;
  const float back = p.scale / lift.by();
  auto value = [&](int d, int r) { return acc[d][r] * back; };
  auto place_of = [&](int i) { return i * stride; };
  if (p.splits > 1)
    RowStore<float, DIM>::store(room, value, p.parts + (int64_t)at.split * p.queries.rows * stride + corner, place_of, queries - mine, p.real_dim, p.real_dim % 4 == 0);
  else
    RowStore<T, DIM>::store(room, value, static_cast<T *>(p.grad_q) + corner, place_of, queries - mine, p.real_dim, p.wide_grads);
}

// grad_k and grad_v of one head of keys: the sums over the queries of every head that shares it, or, with splits, of
// a run of these heads.  Tiles of 32 queries, and v in LDS: what a wave holds of its keys and both sums leaves no
// registers for it.  So two workgroups fit a CU, and the two waves of a SIMD, which no barrier joins, fill each other's
// waits.  (One workgroup of two waves for each 32 keys, which take the same turns at the matrix units: 4096 rows, 32
// heads of 128 in 296 us; one wave for each SIMD, v in registers: 357.)
constexpr int kQueries = 32;

template <class T, int DIM>
__global__ __launch_bounds__(kThreads, 2) void attention_grad_kv_kernel(Attention p) {
  using x8 = typename emrs_gemm::Vec<T>::x8;
  constexpr int kBytes = kQueries * DIM * 2;
  __shared__ __attribute__((aligned(1024))) char even[2 * kBytes];  // rows of q and of grad_out
  __shared__ __attribute__((aligned(1024))) char odd[2 * kBytes];
  __shared__ __attribute__((aligned(1024))) char v_own[kOwn * DIM * 2];
  __shared__ __attribute__((aligned(256))) float sums_even[2][64];  // exponent and delta of the tile's queries, and zeros
  __shared__ __attribute__((aligned(256))) float sums_odd[2][64];
  const int kv_heads = p.heads / p.group;
  Place at;
  if (!find<false>(p.keys, p.queries, p.key_places, kv_heads, p.splits, at)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_of();
  const int keys = at.own.end - at.own.first, queries = at.other.end - at.other.first;
  const int mine = at.row + wave * 32, key = mine + (lane & 31);
  const bool valid = key < keys;
  const int64_t row = at.own.first + key;

  {
    TileLoader<T, DIM, kWaves, kOwn> loader;
    loader.init(p.v_at.row, p.dim, wave);
    loader.load(v_own, static_cast<const T *>(p.v) + (int64_t)(at.own.first + at.row) * p.v_at.row + at.head * p.v_at.head, keys - at.row, wave);
  }
  OwnRows<T, DIM> k;
  k.load(static_cast<const T *>(p.k) + row * p.k_at.row + at.head * p.k_at.head, valid, p.dim);

  // The first query that sees the workgroup's, the wave's and the lane's key, and the one from which on all of the
  // wave's are seen.
  const int shift = keys - queries;
  auto first_for = [&](int j) { return p.causal ? min(max(j - shift, 0), queries) : 0; };
  const int first = first_for(at.row), first_wave = mine < keys ? first_for(mine) : queries, first_lane = first_for(key), all_from = first_for(mine + 31);
  const bool all_valid = mine + 32 <= keys;
  const int from_tile = first / kQueries, tiles = (queries + kQueries - 1) / kQueries - from_tile;  // of a head
  const Span heads = share_of(p.group, at.split, p.splits);
  const int total = max(tiles, 0) * (heads.end - heads.first);

  TileLoader<T, DIM, kWaves, kQueries> q_loader, g_loader;
  q_loader.init(p.q_at.row, p.dim, wave);
  g_loader.init(p.grad_out_at.row, p.dim, wave);
  // Of a tile, and of the wave's keys, whose place is far above the bits that exclusive ors change.
  TileReader<T, DIM> reader, own_reader;
  reader.init();
  own_reader = reader;
  own_reader.by_rows += wave * 32 * reader.kRow;
  const T *const q = static_cast<const T *>(p.q) + at.other.first * p.q_at.row;
  const T *const g = static_cast<const T *>(p.grad_out) + at.other.first * p.grad_out_at.row;
  // The next tile to be loaded and the one that is worked on: tile of a head, head.
  int load_tile = 0, load_head = at.head * p.group + heads.first, work_tile = 0;
  auto load = [&](char *to, float (*sums)[64], bool any) __attribute__((always_inline)) {
    const int64_t from = any ? (from_tile + load_tile) * kQueries : 0;
    const int rows = any ? queries - (int)from : 0, head = any ? load_head : 0;
    q_loader.load(to, q + from * p.q_at.row + head * p.q_at.head, rows, wave);
    g_loader.load(to + kBytes, g + from * p.grad_out_at.row + head * p.grad_out_at.head, rows, wave);
    if (wave < 2) {  // zeros where there is no query: its operands are zeros
      const float *const of = (wave ? p.delta : p.exponent) + (int64_t)head * p.queries.rows + at.other.first + from;
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(of), 0, max(0, min(rows, kQueries)) * 4, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)sums[wave], 4, lane * 4, 0, 0, 0);
    }
    if (++load_tile == tiles) load_tile = 0, ++load_head;
  };
  const float by = p.scale * kLog2e;
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  Lift<T> lift;

  f32x16 grad_k[DIM / 32], grad_v[DIM / 32];
#pragma unroll
  for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) grad_k[d][r] = grad_v[d][r] = 0.f;

  auto work = [&](const char *qt, const float (*sums)[64]) __attribute__((always_inline)) {
    const char *const gt = qt + kBytes;
    const int from = (from_tile + work_tile) * kQueries;
    if (++work_tile == tiles) work_tile = 0;
    if (from + kQueries <= first_wave) return;
    asm("" : "+v"(reader.by_rows), "+v"(reader.by_columns), "+v"(own_reader.by_rows));  // their exclusive ors are taken again: registers
    f32x16 s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
    constexpr int kC = DIM / 16, kD = DIM / 32;
    struct Rows {
      x8 q, g, v;
    };
    Products<kC, 2, Rows> scores;
    auto rows = [&](int c) __attribute__((always_inline)) { return Rows{reader.rows(qt, 0, c), reader.rows(gt, 0, c), own_reader.rows(v_own, 0, c)}; };
    // What the matrix units wait for goes first: the other wave's arithmetic fills what is left (2.5%).
    __builtin_amdgcn_s_setprio(1);
    scores.first(rows);
    scores.run(rows, [&](int c, const Rows &f) __attribute__((always_inline)) {
      s = mfma(f.q, k.v[c], s);
      dp = mfma(f.g, f.v, dp);
    });
    __builtin_amdgcn_s_setprio(0);
    struct Sums {
      f32x4 exponent, delta;
    };
    Products<4, 2, Sums> values;
    auto sums_of = [&](int i) __attribute__((always_inline)) {
      return Sums{*reinterpret_cast<const f32x4 *>(&sums[0][row_of(i * 4)]), *reinterpret_cast<const f32x4 *>(&sums[1][row_of(i * 4)])};
    };
    values.first(sums_of);
    Products<4 * kD, 3, x8> products;
    auto columns = [&](int i) __attribute__((always_inline)) { return reader.columns(i % 2 ? qt : gt, i / 2 % kD, i / (2 * kD)); };
    products.first(columns);
    values.run(sums_of, [&](int i, const Sums &f) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[i * 4 + e], by, -f.exponent[e]));
        dp[i * 4 + e] = x * (dp[i * 4 + e] - f.delta[e]);
        s[i * 4 + e] = kHalf ? x * 32768.f : x;
      }
    });
    if (from < all_from || !all_valid) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (from + row_of(r) < first_lane || !valid) s[r] = dp[r] = 0.f;
    }
    lift.apply(dp, grad_k);
    if (DIM == 64 && (from < all_from || !all_valid)) {
      // As in grad_q, d in two parts where queries see few keys.  (At 128 registers run out: 300 us against 266.)
#pragma unroll
      for (int i = 0; i < 2 * kD; ++i) grad_k[i % kD] = mfma(reader.columns(qt, i % kD, i / kD), rest_of_eight<T>(dp, i / kD), grad_k[i % kD]);
    }
    const x8 prob[2] = {eight_of<T>(s, 0), eight_of<T>(s, 1)}, ds[2] = {eight_of<T>(dp, 0), eight_of<T>(dp, 1)};
    __builtin_amdgcn_s_setprio(1);
    products.run(columns, [&](int i, const x8 &f) __attribute__((always_inline)) {
      const int c = i / (2 * kD), d = i / 2 % kD;
      if (i % 2)
        grad_k[d] = mfma(f, ds[c], grad_k[d]);
      else
        grad_v[d] = mfma(f, prob[c], grad_v[d]);
    });
    __builtin_amdgcn_s_setprio(0);
  };

  load(even, sums_even, total > 0);
  for (int n = 0; n < total; n += 2) {
    arrive();
    load(odd, sums_odd, n + 1 < total);
    work(even, sums_even);
    if (n + 1 >= total) break;
    arrive();
    load(even, sums_even, n + 2 < total);
    work(odd, sums_odd);
  }
  arrive();

  char *const room = wave == 0 ? v_own : wave == 1 ? v_own + 2 * kBytes : wave == 2 ? even : odd;
  const int64_t stride = (int64_t)kv_heads * p.real_dim, corner = (int64_t)(at.own.first + mine) * stride + at.head * p.real_dim, part = at.split * (p.keys.rows * stride);
  const float back_k = p.scale / lift.by(), back_v = kHalf ? 1.f / 32768.f : 1.f;
  auto value_k = [&](int d, int r) { return grad_k[d][r] * back_k; };
  auto value_v = [&](int d, int r) { return grad_v[d][r] * back_v; };
  auto place_of = [&](int i) { return i * stride; };
  if (p.splits > 1) {
    RowStore<float, DIM>::store(room, value_k, p.parts + part + corner, place_of, keys - mine, p.real_dim, p.real_dim % 4 == 0);
    RowStore<float, DIM>::store(room, value_v, p.parts2 + part + corner, place_of, keys - mine, p.real_dim, p.real_dim % 4 == 0);
  } else {
    RowStore<T, DIM>::store(room, value_k, static_cast<T *>(p.grad_k) + corner, place_of, keys - mine, p.real_dim, p.wide_grads);
    RowStore<T, DIM>::store(room, value_v, static_cast<T *>(p.grad_v) + corner, place_of, keys - mine, p.real_dim, p.wide_grads);
  }
}

// Rows as operands want them: on 16 bytes, with zeros up to the next multiple of eight.
template <class T>
__global__ __launch_bounds__(256) void attention_pad_kernel(const T *from, Strides at, int64_t rows, int heads, int dim, int padded, T *to) {
  typedef __attribute__((ext_vector_type(8))) T x8;
  const int units = padded / 8;
  const int64_t all = rows * heads * units;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += (int64_t)gridDim.x * 256) {
    const int64_t row = u / (heads * units);
    const int rest = (int)(u % (heads * units)), c = rest % units * 8;
    const T *const in = from + row * at.row + rest / units * at.head;
    x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < dim ? in[c + e] : (T)0.f;
    reinterpret_cast<x8 *>(to)[u] = v;
  }
}

// ---- calls ----

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }
bool on(const void *p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Workgroups that a launch ought to have: as many as the card holds at a time.  (Twice as many make twice the parts to
// be joined: 2048 queries of 8 heads to 16384 keys, 760 us for all kernels against 700.)
constexpr uint64_t kWanted = 512;
constexpr uint64_t kMostSplits = 32;  // (a token of 32 heads to 131072 keys of 8 heads, 120 us; with 64, 128)

// Whether forward takes the heads that share a key's as rows of one tile: where documents have few queries, tiles of
// one head would be empty for the most part, and every head would read the keys again.  (32 heads of 128, 8 of keys: 64
// single tokens to 8192 keys each, 366 us against 733; 16 documents of 64 queries to 2048 keys, 53 against 57, of 96, 68
// against 63.)
bool folds(const emrs_attention *a) {
  const uint64_t group = a->heads / a->kv_heads;
  return group > 1 && a->rows * 2 <= a->documents * kOwn && a->rows * group < (1u << 30);
}
// Splits of the keys that queries walk: as many as fill the card, with four tiles for each at the least.
uint32_t key_splits(const emrs_attention *a, bool backward) {
  const bool fold = !backward && folds(a);
  const uint64_t rows = a->rows * (fold ? a->heads / a->kv_heads : 1), heads = fold ? a->kv_heads : a->heads;
  const uint64_t tiles = std::max<uint64_t>({1, (rows + kOwn - 1) / kOwn, std::min(a->rows, a->documents)}), each = a->key_rows / std::max<uint64_t>(1, a->documents);
  if (tiles * heads >= kWanted) return 1;
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({kWanted / (tiles * heads), each / (4 * kTile), kMostSplits}));
}
// Of the heads that share a key's.  Where keys are seen by very different numbers of queries, one round of workgroups
// would take as long as its longest (8192 rows, 8 heads of keys: 446 us against 330 with two parts).
uint32_t head_splits(const emrs_attention *a) {
  const uint32_t group = a->heads / a->kv_heads, wanted = a->causal && a->rows * 2 > a->key_rows ? 2 * kWanted : kWanted;
  const uint64_t units = std::max<uint64_t>(1, (a->key_rows + kOwn - 1) / kOwn) * a->kv_heads;
  uint32_t splits = 1;
  while (splits < group && units * splits < wanted) {
    do ++splits;
    while (group % splits);
  }
  return splits;
}

// What lies in the workspace, and where.
struct Room {
  bool pad_q, pad_k, pad_v, pad_g;
  uint64_t q, k, v, g, parts, parts2, part_lse, exponent, delta, query_places, key_places, bytes;
};

bool lists(const emrs_attention *a) { return a->offsets && a->documents > kWalked; }
uint64_t most_tiles(uint64_t rows, uint64_t documents) { return std::min(rows, rows / kOwn + documents + 2); }

// Rows that a tile's loads cannot take as they lie: off 16 bytes, too far apart, or (expanded tensors) one over the
// other, so that what is past the last of them is not past the end of their buffer.
bool off_units(const emrs_attention *a, const void *p, const uint64_t *strides) {
  return a->dim % 8 || strides[0] < a->dim || strides[0] % 8 || strides[1] % 8 || !on(p, 16) || strides[0] > (1u << 22);
}

Room room_of(const emrs_attention *a, bool backward) {
  Room r{};
  const uint64_t dim8 = round_up(a->dim, 8), own = a->rows * a->heads, other = a->key_rows * a->kv_heads;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  r.pad_q = off_units(a, a->q, a->q_strides), r.pad_k = off_units(a, a->k, a->k_strides), r.pad_v = off_units(a, a->v, a->v_strides);
  r.pad_g = backward && off_units(a, a->grad_out, a->grad_out_strides);
  if (r.pad_q) r.q = take(own * dim8 * 2);
  if (r.pad_k) r.k = take(other * dim8 * 2);
  if (r.pad_v) r.v = take(other * dim8 * 2);
  if (r.pad_g) r.g = take(own * dim8 * 2);
  if (backward) {
    r.exponent = take(own * 4);
    r.delta = take(own * 4);
  }
  const uint64_t keys = key_splits(a, backward), heads = backward ? head_splits(a) : 1;
  // grad_q's parts are summed before grad_k's and grad_v's are written.
  const uint64_t parts = std::max(keys > 1 ? keys * own * a->dim * 4 : 0, heads > 1 ? heads * other * a->dim * 4 : 0);
  if (lists(a)) {
    r.query_places = take(sizeof(Places) + most_tiles(a->rows * (!backward && folds(a) ? a->heads / a->kv_heads : 1), a->documents) * sizeof(Entry));
    if (backward) r.key_places = take(sizeof(Places) + most_tiles(a->key_rows, a->documents) * sizeof(Entry));
  }
  r.parts = take(parts);
  if (heads > 1) r.parts2 = take(heads * other * a->dim * 4);
  if (!backward && keys > 1) r.part_lse = take(keys * own * 4);
  r.bytes = at;
  return r;
}

int check_sizes(const emrs_attention *a) {
  if (!a) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: NULL argument");
  if (a->dtype != EMRS_BF16 && a->dtype != EMRS_FP16) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: operands are bf16 or fp16");
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: heads are a multiple of kv_heads");
  if (a->heads > 4096) return fail(EMRS_ERR_TOO_LARGE, "attention: at most 4096 heads");
  if (a->dim < 1 || a->dim > EMRS_ATTENTION_MAX_DIM) return fail(EMRS_ERR_TOO_LARGE, "attention: heads of 1 to 128 elements");
  if (a->documents < 1 || a->documents > (1u << 20)) return fail(EMRS_ERR_TOO_LARGE, "attention: 1 to 2^20 documents");
  if (a->rows > (1u << 28) || a->key_rows > (1u << 28)) return fail(EMRS_ERR_TOO_LARGE, "attention: at most 2^28 rows");
  const uint64_t heads = (uint64_t)a->heads * kMostSplits;
  if ((a->rows / kOwn + a->documents + 2) * heads > 0x3fffffffull || (a->key_rows / kOwn + a->documents + 2) * heads > 0x3fffffffull)
    return fail(EMRS_ERR_TOO_LARGE, "attention: too many tiles for one launch");
  return EMRS_OK;
}

// Lines of 2^20 workgroups: a launch has less than 2^32 threads along a line.
dim3 lines_of(uint64_t rows, uint64_t documents, uint64_t heads, uint64_t splits) {
  constexpr uint64_t line = 1u << 20;
  static_assert(line % kXcds == 0, "every line begins at the same XCD");
  const uint64_t all = most_tiles(rows, documents) * heads * splits;
  return dim3((uint32_t)std::min(all, line), (uint32_t)((all + line - 1) / line));
}

template <class T>
const T *pad(const void *from, const uint64_t *strides, uint64_t rows, uint32_t heads, uint32_t dim, char *to, Strides &at, hipStream_t st) {
  const uint32_t dim8 = (uint32_t)round_up(dim, 8);
  const uint64_t units = rows * heads * (dim8 / 8);
  if (units)
    attention_pad_kernel<T><<<(uint32_t)std::min<uint64_t>((units + 255) / 256, 8192), 256, 0, st>>>(
        static_cast<const T *>(from), Strides{(int64_t)strides[0], (int64_t)strides[1]}, (int64_t)rows, (int)heads, (int)dim, (int)dim8, reinterpret_cast<T *>(to));
  at = {(int64_t)heads * dim8, (int64_t)dim8};
  return reinterpret_cast<const T *>(to);
}

template <class T>
void sum_parts(const float *parts, uint32_t splits, uint64_t each, void *out, hipStream_t st) {
  if (each % 4 == 0)  // outputs lie on 8 bytes
    attention_sum_kernel<T, 4><<<(uint32_t)((each / 4 + 255) / 256), 256, 0, st>>>(parts, (int)splits, (int64_t)each, static_cast<T *>(out));
  else
    attention_sum_kernel<T, 1><<<(uint32_t)((each + 255) / 256), 256, 0, st>>>(parts, (int)splits, (int64_t)each, static_cast<T *>(out));
}

template <class T, int DIM>
int run_as(const emrs_attention *a, bool backward, hipStream_t st) {
  const Room room = room_of(a, backward);
  char *const w = static_cast<char *>(a->workspace);
  const uint32_t dim8 = (uint32_t)round_up(a->dim, 8);
  Attention p{};
  const bool uniform = !a->offsets;
  const int32_t fold = !backward && folds(a) ? (int32_t)(a->heads / a->kv_heads) : 1;
  p.queries = {a->offsets, (int32_t)a->offset_bytes, (int32_t)a->documents, (int32_t)a->rows, uniform ? (int32_t)(a->rows / a->documents) : 0, fold};
  p.keys = {a->key_offsets, (int32_t)a->offset_bytes, (int32_t)a->documents, (int32_t)a->key_rows, uniform ? (int32_t)(a->key_rows / a->documents) : 0, 1};
  auto strides = [](const uint64_t *s) { return Strides{(int64_t)s[0], (int64_t)s[1]}; };
  p.q = a->q, p.k = a->k, p.v = a->v, p.grad_out = a->grad_out;
  p.q_at = strides(a->q_strides), p.k_at = strides(a->k_strides), p.v_at = strides(a->v_strides), p.grad_out_at = strides(a->grad_out_strides);
  if (room.pad_q) p.q = pad<T>(a->q, a->q_strides, a->rows, a->heads, a->dim, w + room.q, p.q_at, st);
  if (room.pad_k) p.k = pad<T>(a->k, a->k_strides, a->key_rows, a->kv_heads, a->dim, w + room.k, p.k_at, st);
  if (room.pad_v) p.v = pad<T>(a->v, a->v_strides, a->key_rows, a->kv_heads, a->dim, w + room.v, p.v_at, st);
  if (room.pad_g) p.grad_out = pad<T>(a->grad_out, a->grad_out_strides, a->rows, a->heads, a->dim, w + room.g, p.grad_out_at, st);
  p.heads = (int32_t)a->heads, p.group = (int32_t)(a->heads / a->kv_heads), p.dim = (int32_t)dim8, p.real_dim = (int32_t)a->dim, p.causal = a->causal != 0;
  p.scale = a->scale, p.out = a->out, p.rest = a->out_rest, p.lse = a->lse;
  p.wide_out = a->dim % 8 == 0 && on(a->out, 16) && on(a->out_rest, 16);
  p.wide_grads = a->dim % 8 == 0 && on(a->grad_q, 16) && on(a->grad_k, 16) && on(a->grad_v, 16);
  if (lists(a) && a->rows + a->key_rows) {
    Places *const of_queries = reinterpret_cast<Places *>(w + room.query_places), *const of_keys = backward ? reinterpret_cast<Places *>(w + room.key_places) : nullptr;
    attention_places_kernel<<<backward ? 2 : 1, kPlaceThreads, 0, st>>>(p.queries, p.keys, of_queries, of_keys);
    p.query_places = of_queries, p.key_places = of_keys;
  }
  p.splits = (int32_t)key_splits(a, backward);
  p.parts = p.splits > 1 ? reinterpret_cast<float *>(w + room.parts) : nullptr;
  if (!backward) {
    if (a->rows == 0) return EMRS_OK;
    p.part_lse = reinterpret_cast<float *>(w + room.part_lse);
    if (fold > 1)
      attention_forward_kernel<T, DIM, true><<<lines_of(a->rows * fold, a->documents, a->kv_heads, p.splits), kThreads, 0, st>>>(p);
    else
      attention_forward_kernel<T, DIM, false><<<lines_of(a->rows, a->documents, a->heads, p.splits), kThreads, 0, st>>>(p);
    if (p.splits > 1) {
      const uint32_t e = a->dim % 4 ? 1 : 4, blocks = (uint32_t)((a->rows * a->heads * (a->dim / e) + 255) / 256);
      (e == 4 ? attention_join_kernel<T, 4> : attention_join_kernel<T, 1>)<<<blocks, 256, 0, st>>>(p.parts, p.part_lse, p.splits, (int64_t)a->rows, (int)a->heads,
                                                                                                 (int)a->dim, static_cast<T *>(a->out), static_cast<T *>(a->out_rest), a->lse);
    }
  } else {
    p.exponent = reinterpret_cast<float *>(w + room.exponent);
    p.delta = reinterpret_cast<float *>(w + room.delta);
    // delta and exponent come out of grad_q's kernel, so that it runs in any case; without grad_q it ends there.
    p.grad_q = a->grad_q;
    if (!a->grad_q && p.splits > 1) p.splits = 1, p.parts = nullptr;
    if (a->rows) {
      attention_grad_q_kernel<T, DIM><<<lines_of(a->rows, a->documents, a->heads, p.splits), kThreads, 0, st>>>(p);
      if (p.splits > 1) sum_parts<T>(p.parts, p.splits, a->rows * a->heads * a->dim, a->grad_q, st);
    }
    if (a->grad_k && a->key_rows) {
      p.grad_k = a->grad_k, p.grad_v = a->grad_v;
      p.splits = (int32_t)head_splits(a);
      p.parts = p.splits > 1 ? reinterpret_cast<float *>(w + room.parts) : nullptr;
      p.parts2 = p.splits > 1 ? reinterpret_cast<float *>(w + room.parts2) : nullptr;
      attention_grad_kv_kernel<T, DIM><<<lines_of(a->key_rows, a->documents, a->kv_heads, p.splits), kThreads, 0, st>>>(p);
      if (p.splits > 1) {
        sum_parts<T>(p.parts, p.splits, a->key_rows * a->kv_heads * a->dim, a->grad_k, st);
        sum_parts<T>(p.parts2, p.splits, a->key_rows * a->kv_heads * a->dim, a->grad_v, st);
      }
    }
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? EMRS_OK : fail(EMRS_ERR_HIP, std::string("attention: ") + hipGetErrorString(e));
}

int run(const emrs_attention *a, bool backward, hipStream_t st) {
  int rc = check_sizes(a);
  if (rc) return rc;
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: the scale is positive and finite");
  if (a->reserved) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: reserved is not 0");
  if (!a->offsets != !a->key_offsets) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: offsets of both sides, or of none");
  if (a->offsets) {
    if (a->offset_bytes != 4 && a->offset_bytes != 8) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: offsets are of 4 or 8 bytes");
    if (!on(a->offsets, a->offset_bytes) || !on(a->key_offsets, a->offset_bytes))
      return fail(EMRS_ERR_MISALIGNED, "attention: offsets off their type's alignment");
  } else if (a->rows % a->documents || a->key_rows % a->documents) {
    return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: documents of equal length do not fill the rows");
  }
  auto operand = [&](const void *p, uint64_t rows, const uint64_t *strides) {
    if (!rows) return EMRS_OK;
    if (!p) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: NULL operand");
    if (!on(p, 2)) return fail(EMRS_ERR_MISALIGNED, "attention: an operand off its type's alignment");
    if (strides[0] > (1ull << 40) || strides[1] > (1ull << 40)) return fail(EMRS_ERR_TOO_LARGE, "attention: strides are at most 2^40");
    return (int)EMRS_OK;
  };
  if ((rc = operand(a->q, a->rows, a->q_strides)) || (rc = operand(a->k, a->key_rows, a->k_strides)) || (rc = operand(a->v, a->key_rows, a->v_strides)))
    return rc;
  if (a->rows && !a->out) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: NULL out");
  if (!on(a->out, 8) || !on(a->out_rest, 8) || !on(a->lse, 4)) return fail(EMRS_ERR_MISALIGNED, "attention: out is off 8 bytes");
  if (backward) {
    if ((rc = operand(a->grad_out, a->rows, a->grad_out_strides))) return rc;
    if (a->rows && !a->lse) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: NULL lse");
    if (!a->grad_q && !a->grad_k) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: no gradient is wanted");
    if (!a->grad_k != !a->grad_v) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: grad_k and grad_v come together");
    if (!on(a->grad_q, 8) || !on(a->grad_k, 8) || !on(a->grad_v, 8)) return fail(EMRS_ERR_MISALIGNED, "attention: a gradient is off 8 bytes");
  }
  const uint64_t wanted = room_of(a, backward).bytes;
  if (wanted) {
    if (!a->workspace || a->workspace_bytes < wanted) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: the workspace is too small");
    if (!on(a->workspace, 256)) return fail(EMRS_ERR_MISALIGNED, "attention: the workspace is off 256 bytes");
  }
  if (!a->rows && (!backward || !a->grad_k || !a->key_rows)) return EMRS_OK;
  rc = emrs_internal::need_device();
  if (rc) return rc;
  if (a->dtype == EMRS_BF16) return a->dim <= 64 ? run_as<__bf16, 64>(a, backward, st) : run_as<__bf16, 128>(a, backward, st);
  return a->dim <= 64 ? run_as<_Float16, 64>(a, backward, st) : run_as<_Float16, 128>(a, backward, st);
}

}  // namespace

extern "C" int emrs_attention_workspace(const emrs_attention *a, int backward, uint64_t *bytes) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    if (!bytes) return fail(EMRS_ERR_INVALID_ARGUMENT, "attention: NULL argument");
    const int rc = check_sizes(a);
    if (rc) return rc;
    *bytes = room_of(a, backward != 0).bytes;
    return EMRS_OK;
  });
}

extern "C" int emrs_attention_forward(const emrs_attention *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    return run(a, false, static_cast<hipStream_t>(stream));
  });
}

extern "C" int emrs_attention_backward(const emrs_attention *a, void *stream) {
  return emrs_internal::guarded([&]() -> int {
    emrs_internal::clear_error();
    return run(a, true, static_cast<hipStream_t>(stream));
  });
}
