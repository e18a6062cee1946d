// Matrix products of the training operators: C[n][m] = sum_k A[m][k] B[n][k], 16-bit operands, sums in 32 bits.
//
// Both operands hold the summed index contiguously, and what an operator does with C is a functor (the
// epilogue) that gets the accumulators in registers, so that no product goes through memory only to be
// read again.  A lane of a 16x16x32 matrix instruction ends up with four consecutive m of one n: outputs
// are laid out with m contiguous, where those four make one store.
//
// A workgroup computes a BM x BN tile.  Its operands pass through two LDS stages of 64 k each, which
// buffer loads fill directly: the loads of the next stage are in flight while the matrix instructions
// consume this one.  Such a load writes 64 lanes x 16 bytes to consecutive LDS addresses (8 rows of 128
// bytes), so a row's eight 16-byte units are permuted on the global side, unit c of row r in slot
// c ^ swizzle(r): what 16 lanes of a fragment read take at a time then lies in 16 different slots of the
// 64 banks.  Rows past the operand's last are past the buffer's end and read as zeros, and so are, by
// their lane's offset, units past the last k.
//
// In large products matrix instructions issue in 63 to 68% of the cycles that a CU is busy, start and epilogue
// included (74% where k is 12288, 56% where the epilogue reads X and writes it twice), at 1.9 to 2.1 GHz of 2.4.
// Measured with what the epilogues do, on two cards: statistics of 4096 x 32000 logits, k 4096, 780 and 832 us (1.38 and 1.29 PFLOP/s); d
// of 4096 x 16384, 450 and 472 us; the gradients' products of that d, 425 to 458 us.
#ifndef EMRS_GEMM_H
#define EMRS_GEMM_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace emrs_gemm {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 fp16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

__device__ inline f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma(fp16x8 a, fp16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <class T>
struct Vec;
template <>
struct Vec<__bf16> {
  using x8 = bf16x8;
  typedef __attribute__((ext_vector_type(4))) __bf16 x4;
};
template <>
struct Vec<_Float16> {
  using x8 = fp16x8;
  typedef __attribute__((ext_vector_type(4))) _Float16 x4;
};

constexpr int kStage = 64;  // k of one LDS stage: rows of 128 bytes
constexpr int kXcds = 8;
constexpr int kGroup = 8;   // tiles of m that are walked before the next n: what one XCD's CUs share

// An operand that is held as a sum of two 16-bit parts has them side by side in its rows, hi | lo, and
// multiplies as hi hi + hi lo + lo hi, which is only more k: the operand's own k starts again where k
// reaches its wrap.
struct Product {
  const void *a, *b;
  int64_t a_stride, b_stride;      // elements between rows, multiples of 8
  int64_t a_batch, b_batch;        // elements between the matrices of a batch
  int32_t m, n, k;                 // k a multiple of 8, and of 64 where an operand wraps
  int32_t a_wrap, b_wrap;          // multiples of 64; kNoWrap
  int32_t k_end;                   // 0, or where batches are runs of k: all of k, which the last run may pass
  int32_t batch;
  int32_t symmetric;               // only tiles on and below the diagonal (m >= n) are computed
};
constexpr int32_t kNoWrap = 0x7fffffff;

template <int BM_, int BN_, int WM_, int WN_, int GROUPS_ = 1>
struct Tile {
  static constexpr int BM = BM_, BN = BN_;
  static constexpr int WAVES_M = BM / WM_, WAVES_N = BN / WN_, WAVES = WAVES_M * WAVES_N;
  static constexpr int WM = WM_, WN = WN_;
  static constexpr int MI = WM / 16, NI = WN / 16;
  static constexpr int GROUPS = GROUPS_;  // of waves that share a tile, each over its own run of k
  static constexpr int THREADS = WAVES * GROUPS * 64;
  static constexpr int A_LOADS = BM / 8 / WAVES, B_LOADS = BN / 8 / WAVES;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole 1 KB loads per wave");
};

// 256 x 256 with 8 waves of 128 x 64: a stage is 64 KB, and its 2^23 multiply-adds are 2048 cycles of the
// CU's matrix units against 96 KB of fragment reads.  192 x 192 with 12 waves reads 1.33 times the bytes for a
// multiply-add, and is for products whose large tiles would fill their last round badly: 253 of them take
// 207 us where 136 large ones take 255 (4096 x 4096 by half, k 12288).  The smaller tiles are for products
// that would not give every CU one of these: what bounds them is how often a stage's loads are waited for, so
// the smaller a tile, the more groups of waves share its k (Newton-Schulz on 512 x 512: 112 us, with tiles of
// 64 at the least 147).
using Large = Tile<256, 256, 128, 64>;
using Broad = Tile<192, 192, 64, 48>;
using Medium = Tile<128, 128, 64, 64, 2>;
using Small = Tile<64, 64, 32, 32, 4>;
using Tiny = Tile<32, 32, 32, 32, 8>;

__host__ __device__ inline int64_t tiles_of(int64_t n, int64_t t) { return (n + t - 1) / t; }
template <class Cfg>
__host__ inline int64_t tile_count(const Product &p) {
  const int64_t tm = tiles_of(p.m, Cfg::BM), tn = tiles_of(p.n, Cfg::BN);
  return (p.symmetric ? tm * (tm + 1) / 2 : tm * tn) * p.batch;
}

struct Where {
  int m0, n0, batch;
  // Of place(): the tile's first row, the first k, and which part of a tile's k it is (-1: the whole).
  int first, k_from, part;
};

// What an epilogue is beside its run(): where the operands of a matrix of the batch begin.
struct Operand {
  static constexpr bool kRowsOfK = false;  // whether operand a is [k][m]
  static constexpr bool kBy32 = true;      // whether tiles of 32 will do; else they reach the next multiples of 64
  __device__ __forceinline__ const void *operand_a(const Product &p, int batch) const {
    return static_cast<const char *>(p.a) + batch * p.a_batch * 2;
  }
  __device__ __forceinline__ const void *operand_b(const Product &p, int batch) const {
    return static_cast<const char *>(p.b) + batch * p.b_batch * 2;
  }
};

// What an epilogue may have besides.  kColumnsOfK: operand b is [k][n].  kPlaced: place() finds the workgroup's tile
// and may narrow the product to a part of it (rows of n, or k), or says that there is none; rows of k then come from
// rows_from() and columns_from() by that tile.
template <class E, class = void>
struct Extras {
  static constexpr bool kColumnsOfK = false, kPlaced = false;
};
template <class E>
struct Extras<E, std::void_t<decltype(E::kPlaced)>> {
  static constexpr bool kColumnsOfK = E::kColumnsOfK, kPlaced = E::kPlaced;
};

// The row that holds place t of a triangle, whose row i holds i + 1.
__device__ inline uint32_t triangle_row(uint32_t t) {
  uint32_t i = (uint32_t)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
  while (i * (i + 1) / 2 > t) --i;
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  return i;
}

// The tile of a workgroup.  Workgroups go to the XCDs in turn; each XCD gets a run of consecutive tiles,
// and a run walks kGroup tiles of m for each n, so that its CUs share operand rows in the XCD's L2.
template <class Cfg>
__device__ inline Where tile_of(const Product &p) {
  const uint32_t total = gridDim.x, id = blockIdx.x;
  const uint32_t q = total / kXcds, r = total % kXcds, x = id % kXcds;
  uint32_t t = x * q + min(x, r) + id / kXcds;
  const uint32_t tm = (p.m + Cfg::BM - 1) / Cfg::BM, tn = (p.n + Cfg::BN - 1) / Cfg::BN;
  const uint32_t per = p.symmetric ? tm * (tm + 1) / 2 : tm * tn;
  Where w;
  w.batch = t / per;
  t %= per;
  uint32_t i, j;
  if (p.symmetric) {  // bands of kGroup rows: the columns left of the diagonal block, then that block
    const uint32_t first = triangle_row(t) / kGroup * kGroup, rows = min((uint32_t)kGroup, tm - first);
    uint32_t at = t - first * (first + 1) / 2;
    if (at < first * rows) {
      i = first + at % rows;
      j = at / rows;
    } else {
      at -= first * rows;
      const uint32_t r = triangle_row(at);
      i = first + r;
      j = first + at - r * (r + 1) / 2;
    }
  } else {
    const uint32_t group = t / (kGroup * tn), first = group * kGroup, rows = min((uint32_t)kGroup, tm - first);
    const uint32_t at = t - group * kGroup * tn;
    i = first + at % rows;
    j = at / rows;
  }
  w.m0 = (int)i * Cfg::BM;
  w.n0 = (int)j * Cfg::BN;
  return w;
}

// Of the row's place among eight alone, so that a wave reads its fragments at constant offsets of one address.  The 16
// lanes that LDS serves at a time are those of rows 0 to 3 and 12 to 15 at one unit and of rows 4 to 11 at its
// neighbour (or the other way round): their units differ where the rows' halves of eight are told apart.  (Permuted as
// for 16 lanes in a row, LDS spent a quarter of the cycles of products of 8192 x 4096 x 28672 in conflicts; without them
// they take 1% fewer.)
__device__ inline int swizzle(int row) { return (row ^ (row >> 2 & 1)) & 7; }

// What a lane loads of an operand's stage: the same 16 bytes of row `lane / 8` of each of its wave's groups
// of eight rows, which lie a constant apart.  Every group has a buffer of its own, from its first row to the
// operand's last k: the hardware checks a lane's offset against a buffer's size, but not the scalar offset
// (where k goes), so what places a row must not be scalar.
template <class T, int LOADS, int WAVES>
struct Loader {
  int voffset;
  int unit;        // first k, within a stage, of its 16 bytes
  const T *base[LOADS];
  int bytes[LOADS];  // 0: no row of the group is the operand's
  // first: the tile's first row; rows: how many of its rows there are; columns: what a row holds.
  __device__ __forceinline__ void init(const T *first, int64_t stride, int rows, int columns, int wave, int lane) {
    const int row = lane >> 3, c = (lane & 7) ^ swizzle(row);
    unit = c * 8;
    voffset = (int)(row * stride * 2) + (c << 4);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int at = (wave + j * WAVES) * 8, here = rows - at;
      base[j] = first + at * stride;
      bytes[j] = here > 0 ? (int)(((here - 1) * stride + columns) * 2) : 0;
    }
  }
  // Fewer than a stage's k are left: lanes whose 16 bytes are past them go past the buffer's end instead.
  __device__ __forceinline__ void cut(int left) {
    voffset = unit < left ? voffset : (int)0x80000000;
  }
  // Load j of the stage from k0 on; none: zeros.
  __device__ __forceinline__ void load(char *lds, int j, int k0, bool none, int wave) const {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base[j]), 0, none ? 0 : bytes[j], 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + (wave + j * WAVES) * 1024), 16,
                                             voffset, k0 * 2, 0, 0);
  }
};

// The same of an operand that is [k][m] or [k][n]: a stage is 64 of its rows, B (a tile's m or n) long each, 16-byte
// units permuted by the row so that the transposing reads of 32 lanes, eight rows of 32 bytes, meet in different
// banks.  Rows that do not count are past the end of their buffer.
template <class T, int B, int WAVES>
struct RowLoader {
  static constexpr int kUnits = B / 8, kRows = 64 / kUnits;  // of a row; of one load
  int voffset, columns, stride;
  const T *first;  // the stage's first row, at the tile's first m
  int rows;        // that count from there on
  static __device__ __forceinline__ int permuted(int row) {
    return B == 64 ? (row >> 1 & 1) | (row >> 3 & 1) << 1 : (row & 3) | (row >> 3 & 1) << 2;
  }
  __device__ __forceinline__ void init(int64_t row_stride, int columns_here, int wave, int lane) {
    static_assert(B == 256 || B == 128 || B == 64, "whole rows in a load");
    static_assert(WAVES * kRows % 16 == 0, "a wave's loads are permuted alike");
    const int row = lane / kUnits, unit = lane % kUnits;
    stride = (int)row_stride, columns = columns_here;
    voffset = (int)(row * stride * 2) + ((unit ^ permuted(wave * kRows + row) << 1) << 4);
  }
  __device__ __forceinline__ void cut(int) {}
  __device__ __forceinline__ void load(char *lds, int j, int, bool none, int wave) const {
    // No branches: the loads are started between matrix instructions.  (columns <= stride.)  The median is a
    // vector instruction; a buffer that might differ between lanes would cost the load a loop.
    const int from = (wave + j * WAVES) * kRows, here = __builtin_amdgcn_readfirstlane(none ? 0 : min(max(rows - from, 0), kRows));
    const int bytes = max(0, (here - 1) * stride + columns) * 2;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(first + from * stride), 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + (wave + j * WAVES) * 1024), 16,
                                             voffset, 0, 0, 0);
  }
};

// This wave's loads into LDS have landed and its LDS reads are in registers, and so are every other wave's:
// a barrier alone waits for neither.
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  __builtin_amdgcn_sched_barrier(0);
}

// The loads of one stage, to be started one by one.
template <class Cfg, class LoaderA, class LoaderB>
struct Loads {
  static constexpr int kCount = Cfg::A_LOADS + Cfg::B_LOADS;
  const LoaderA &loader_a;
  const LoaderB &loader_b;
  char *a, *b;
  int a_k, b_k;
  bool none;
  int wave;
  __device__ __forceinline__ void operator()(int q) const {
    if (q < Cfg::A_LOADS)
      loader_a.load(a, q, a_k, none, wave);
    else
      loader_b.load(b, q - Cfg::A_LOADS, b_k, none, wave);
  }
};

struct NoLoads {
  static constexpr int kCount = 0;
  __device__ void operator()(int) const {}
};

// Eight consecutive k of a lane's m from rows of k: sixteen lanes read a block of 4 k x 16 m as it lies, twice.
template <class X8>
__device__ __forceinline__ X8 along_k(const char *at, int four_rows) {
  typedef __attribute__((ext_vector_type(4))) short s16x4;
  typedef __attribute__((address_space(3))) s16x4 *lds4;
  char *const lo = const_cast<char *>(at);
  const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)lo), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lo + four_rows));
  return __builtin_bit_cast(X8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Where a group after the first leaves sum q of its lanes: the stages' arrays, one after the other.
template <class Cfg>
__device__ __forceinline__ f32x4 &left_sum(char *a, char *b, char *c, char *d, int group, int q, int wave, int lane) {
  constexpr int block = Cfg::WAVES * 1024, each = Cfg::GROUPS * 128 * (Cfg::BM < Cfg::BN ? Cfg::BM : Cfg::BN) / block;
  static_assert((Cfg::GROUPS - 1) * Cfg::MI * Cfg::NI <= 4 * each, "they fit");
  const int at = (group - 1) * Cfg::MI * Cfg::NI + q;
  char *const base = at < each ? a : at < 2 * each ? b : at < 3 * each ? c : d;
  return reinterpret_cast<f32x4 *>(base + at % each * block + wave * 1024)[lane];
}

// A wave's tile in 16 bits, turned over in its part of LDS: accumulators go in, and 16-byte units of eight
// consecutive m of an n, or of eight consecutive n of an m, come out.  Rows are of n; a row's units are
// permuted by n, so that 16 lanes of different n meet different banks.  Nothing here waits for other waves.
template <class Cfg>
struct Turn {
  static constexpr int kRow = Cfg::WM / 8, kMask = kRow - 1;  // units of a row
  static constexpr int kPasses = Cfg::WM * Cfg::WN / 512;
  static __device__ __forceinline__ int at(int n, int m) { return n * Cfg::WM * 2 + (((m >> 3) ^ n) & kMask) * 16 + (m & 7) * 2; }
  template <class V>
  static __device__ __forceinline__ void put(char *own, int i, int j, int lane, V v) {
    static_assert(sizeof(V) == 8, "four values");
    *reinterpret_cast<V *>(own + at(j * 16 + (lane & 15), i * 16 + (lane >> 4) * 4)) = v;
  }
  // store(m, n, unit): eight consecutive m.
  template <class Store>
  static __device__ __forceinline__ void along_m(const char *own, int lane, Store store) {
#pragma unroll 4
    for (int q = 0; q < kPasses; ++q) {
      const int u = q * 64 + lane, n = u / kRow, m = u % kRow * 8;
      store(m, n, *reinterpret_cast<const fp16x8 *>(own + at(n, m)));
    }
  }
  // store(m, n, unit): eight consecutive n.  Sixteen lanes read a block of 4 n x 16 m as it lies, and each gets
  // the four n of one m.
  template <class Store>
  static __device__ __forceinline__ void along_n(const char *own, int lane, Store store) {
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    typedef __attribute__((address_space(3))) s16x4 *lds4;
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    const int t = lane & 15;
#pragma unroll 4
    for (int q = 0; q < kPasses; ++q) {
      const int b = q * 4 + (lane >> 4), n = b % (Cfg::WN / 8) * 8, m = b / (Cfg::WN / 8) * 16;
      char *const lo = const_cast<char *>(own) + at(n + (t >> 2), m + (t & 3) * 4);
      char *const hi = const_cast<char *>(own) + at(n + 4 + (t >> 2), m + (t & 3) * 4);
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)lo), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)hi);
      const s16x8 v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
      store(m + t, n, __builtin_bit_cast(fp16x8, v));
    }
  }
};

template <class T, class Cfg, class Epilogue>
__global__ __launch_bounds__(Cfg::THREADS) void product_kernel(Product p, Epilogue epilogue) {
  using x8 = typename Vec<T>::x8;
  // One array for each stage: the compiler then knows which of them a load into LDS and a read have in common.
  __shared__ __attribute__((aligned(1024))) char a_evens[Cfg::GROUPS][Cfg::BM * 128];
  __shared__ __attribute__((aligned(1024))) char a_odds[Cfg::GROUPS][Cfg::BM * 128];
  __shared__ __attribute__((aligned(1024))) char b_evens[Cfg::GROUPS][Cfg::BN * 128];
  __shared__ __attribute__((aligned(1024))) char b_odds[Cfg::GROUPS][Cfg::BN * 128];
  constexpr bool rows_of_k = Epilogue::kRowsOfK, columns_of_k = Extras<Epilogue>::kColumnsOfK;
  Where w;
  if constexpr (Extras<Epilogue>::kPlaced) {
    if (!epilogue.template place<Cfg>(p, w)) return;
  } else {
    w = tile_of<Cfg>(p);
  }
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = Cfg::GROUPS > 1 ? all / Cfg::WAVES : 0, wave = Cfg::GROUPS > 1 ? all % Cfg::WAVES : all;
  char *const a_even = a_evens[group], *const a_odd = a_odds[group], *const b_even = b_evens[group], *const b_odd = b_odds[group];
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;

  const int k = p.k_end ? min(p.k, max(0, p.k_end - w.batch * p.k)) : p.k;
  auto columns = [&](int wrap) { return k <= wrap ? k : max(wrap, k - wrap); };
  typename std::conditional<rows_of_k, RowLoader<T, Cfg::BM, Cfg::WAVES>, Loader<T, Cfg::A_LOADS, Cfg::WAVES>>::type la;
  typename std::conditional<columns_of_k, RowLoader<T, Cfg::BN, Cfg::WAVES>, Loader<T, Cfg::B_LOADS, Cfg::WAVES>>::type lb;
  using NextLoads = Loads<Cfg, decltype(la), decltype(lb)>;
  if constexpr (rows_of_k)
    la.init(p.a_stride, min(Cfg::BM, ((p.m + 7) & ~7) - w.m0), wave, lane);
  else
    la.init(static_cast<const T *>(epilogue.operand_a(p, w.batch)) + w.m0 * p.a_stride, p.a_stride, min(Cfg::BM, p.m - w.m0), columns(p.a_wrap), wave, lane);
  if constexpr (columns_of_k)
    lb.init(p.b_stride, min(Cfg::BN, ((p.n + 7) & ~7) - w.n0), wave, lane);
  else
    lb.init(static_cast<const T *>(epilogue.operand_b(p, w.batch)) + w.n0 * p.b_stride, p.b_stride, min(Cfg::BN, p.n - w.n0), columns(p.b_wrap), wave, lane);
  // Stages of a group; those past the last k are zeros.
  const int total = ((p.k + kStage - 1) / kStage + Cfg::GROUPS - 1) / Cfg::GROUPS;
  int k0 = group * total * kStage;
  const int k_to = min(k, k0 + total * kStage);
  // The next stage's loads; past the last stage they read zeros.
  auto next_stage = [&](char *a, char *b) __attribute__((always_inline)) {
    const int left = k - k0;
    const bool none = k0 >= k_to;
    const int from = none ? 0 : k0;  // a scalar offset past a buffer's end is not to be relied on
    if constexpr (rows_of_k) {
      if constexpr (Extras<Epilogue>::kPlaced)
        epilogue.rows_from(p, w, from, la.first, la.rows);
      else
        epilogue.rows_from(p, w.batch * p.k + from, la.first, la.rows);
      la.first += w.m0;
    }
    if constexpr (columns_of_k) {
      epilogue.columns_from(p, w, from, lb.first, lb.rows);
      lb.first += w.n0;
    }
    const NextLoads n{la, lb, a, b, from >= p.a_wrap ? from - p.a_wrap : from, from >= p.b_wrap ? from - p.b_wrap : from, none, wave};
    k0 += kStage;
    if (!none && left < kStage) la.cut(left), lb.cut(left);
    return n;
  };
  auto load = [&](char *a, char *b) __attribute__((always_inline)) {
    const NextLoads n = next_stage(a, b);
#pragma unroll
    for (int q = 0; q < NextLoads::kCount; ++q) n(q);
  };

  f32x4 acc[Cfg::MI][Cfg::NI];
#pragma unroll
  for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int row = lane & 15, c = lane >> 4;
  const int unit[2] = {(c ^ swizzle(row)) << 4, ((4 + c) ^ swizzle(row)) << 4};
  const int a_at = (wm * Cfg::WM + row) * 128, b_at = (wn * Cfg::WN + row) * 128;
  // The first of the wave's 32-byte pieces of its rows of k; piece i lies where i is added to it before the
  // permutation, and both are exclusive ors: the wave's first piece is a multiple of MI.
  const int a_k = c * 8 + (row >> 2);
  int a_piece = rows_of_k ? a_k * Cfg::BM * 2 + ((wm * Cfg::MI) ^ RowLoader<T, rows_of_k ? Cfg::BM : 64, Cfg::WAVES>::permuted(a_k)) * 32 + (row & 3) * 8 : 0;
  int b_piece = columns_of_k ? a_k * Cfg::BN * 2 + ((wn * Cfg::NI) ^ RowLoader<T, columns_of_k ? Cfg::BN : 64, Cfg::WAVES>::permuted(a_k)) * 32 + (row & 3) * 8 : 0;
  struct Fragments {
    x8 a[Cfg::MI], b[Cfg::NI];
  } even, odd;  // of the first and the second 32 k of a stage
  auto read_one = [&](Fragments &f, const char *a, const char *b, int kk, int r) __attribute__((always_inline)) {
    if (r < Cfg::NI) {
      if constexpr (columns_of_k)
        f.b[r] = along_k<x8>(b + (b_piece ^ r << 5) + kk * 64 * Cfg::BN, 8 * Cfg::BN);
      else
        f.b[r] = *reinterpret_cast<const x8 *>(b + b_at + unit[kk] + r * 2048);
    } else if constexpr (rows_of_k)
      f.a[r - Cfg::NI] = along_k<x8>(a + (a_piece ^ (r - Cfg::NI) << 5) + kk * 64 * Cfg::BM, 8 * Cfg::BM);
    else
      f.a[r - Cfg::NI] = *reinterpret_cast<const x8 *>(a + a_at + unit[kk] + (r - Cfg::NI) * 2048);
  };
  // 32 k of a stage: multiplies `now` while it reads `next`, and starts the loads of another stage.  Pinned in
  // this order: LDS reads in the shadow of every second or third matrix instruction, done well before the
  // end, and the loads spread over all of them, at the rate at which the CU can take them.
  auto half = [&](const Fragments &now, Fragments &next, const char *a, const char *b, int kk, auto start) __attribute__((always_inline)) {
    constexpr int products = Cfg::MI * Cfg::NI, reads = Cfg::MI + Cfg::NI, loads = decltype(start)::kCount;
    constexpr int per = products * 3 / 4 / reads > 0 ? products * 3 / 4 / reads : 1;
    if constexpr (rows_of_k) asm("" : "+v"(a_piece));  // its MI exclusive ors are taken again: registers
    if constexpr (columns_of_k) asm("" : "+v"(b_piece));
#pragma unroll
    for (int q = 0; q < products; ++q) {
      acc[q / Cfg::NI][q % Cfg::NI] = mfma(now.a[q / Cfg::NI], now.b[q % Cfg::NI], acc[q / Cfg::NI][q % Cfg::NI]);
      if (q % per == 0 && q / per < reads) read_one(next, a, b, kk, q / per);
#pragma unroll
      for (int l = (q * loads + products - 1) / products; l < ((q + 1) * loads + products - 1) / products; ++l) start(l);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = (products + per - 1) / per; r < reads; ++r) read_one(next, a, b, kk, r);
  };
  // A stage.  Its first fragments are in registers: the second ones are read while the first multiply.  Then
  // every wave has read all of it, and the next stage has arrived: the loads of the one after that go into
  // its place, and the next stage's first fragments are read while the second ones multiply.
  auto stage = [&](char *a, char *b, const char *a_next, const char *b_next) __attribute__((always_inline)) {
    half(even, odd, a, b, 1, NoLoads{});
    arrive();
    half(odd, even, a_next, b_next, 0, next_stage(a, b));
  };

  load(a_even, b_even);
  load(a_odd, b_odd);
  arrive();
#pragma unroll
  for (int r = 0; r < Cfg::MI + Cfg::NI; ++r) read_one(even, a_even, b_even, 0, r);
  int it = 0;
  for (; it + 1 < total; it += 2) {
    stage(a_even, b_even, a_odd, b_odd);
    stage(a_odd, b_odd, a_even, b_even);
  }
  if (it < total) stage(a_even, b_even, a_odd, b_odd);
  arrive();  // no load may still be on its way into LDS that another workgroup gets
  if constexpr (Cfg::GROUPS > 1) {
    // The groups' sums pass through the stages' LDS to the first group, in the order of k.
    if (group > 0) {
#pragma unroll
      for (int q = 0; q < Cfg::MI * Cfg::NI; ++q)
        left_sum<Cfg>(a_evens[0], b_evens[0], a_odds[0], b_odds[0], group, q, wave, lane) = acc[q / Cfg::NI][q % Cfg::NI];
    }
    arrive();
    if (group == 0) {
#pragma unroll
      for (int g = 1; g < Cfg::GROUPS; ++g)
#pragma unroll
        for (int q = 0; q < Cfg::MI * Cfg::NI; ++q)
          acc[q / Cfg::NI][q % Cfg::NI] += left_sum<Cfg>(a_evens[0], b_evens[0], a_odds[0], b_odds[0], g, q, wave, lane);
    }
    arrive();
    if (group > 0) return;
  }
  // Each wave's own part of the stages' LDS, for its tile in 16 bits.
  constexpr int part = Cfg::WM * Cfg::WN * 2, each = Cfg::GROUPS * 128 * (Cfg::BM < Cfg::BN ? Cfg::BM : Cfg::BN) / part;
  static_assert(4 * each >= Cfg::WAVES, "they fit");
  char *const own = (wave < each ? a_evens[0] : wave < 2 * each ? b_evens[0] : wave < 3 * each ? a_odds[0] : b_odds[0]) + wave % each * part;
  epilogue.template run<Cfg>(acc, w, w.m0 + wm * Cfg::WM, w.n0 + wn * Cfg::WN, wm, lane, p, own);
}

enum Shape { kLarge, kBroad, kMedium, kSmall, kTiny };

// What a launch of one tile size takes, in microseconds, by its rounds of 256 workgroups (each has a CU's LDS
// for itself): measured are 1.25 for a large tile's stage, 1.05 for a broad one's and for the stage that each
// of a medium tile's two groups works on, 0.95 for a small tile's four, 0.9 for the smallest's eight, and what a workgroup takes beside; 1.7
// for a large tile's with rows of k, whose reads leave it short of registers.
// (A last round split along k instead, its pieces' sums joined by the last of them to end, was slower but for
// the longest k: the sums of 240 pieces took 50 us on their way through memory.)
template <class Cfg>
inline double cost_of(const Product &p, double stage, double fixed) {
  const int64_t rounds = (tile_count<Cfg>(p) + 255) / 256, stages = (tiles_of(p.k, kStage) + Cfg::GROUPS - 1) / Cfg::GROUPS;
  return (double)rounds * (fixed + stage * (double)stages);
}

// Large tiles read the operands fewer times; smaller ones give more CUs work, and their waves share a long k.
struct Choice {
  Shape shape;
  double cost;
};
inline Choice choice_of(const Product &p, bool rows_of_k, bool by_32) {
  const double cost[5] = {cost_of<Large>(p, rows_of_k ? 1.7 : 1.25, 8), cost_of<Broad>(p, 1.05, 6), cost_of<Medium>(p, 1.05, 4), cost_of<Small>(p, 0.95, 3),
                          cost_of<Tiny>(p, 0.9, 3)};
  int best = kLarge;
  for (int i = kBroad; i <= kTiny; ++i)
    if (cost[i] < cost[best] && !(rows_of_k && i == kBroad) && (by_32 || i != kTiny)) best = i;
  return {(Shape)best, cost[best]};
}
inline Shape shape_of(const Product &p) { return choice_of(p, false, true).shape; }

template <class T, class Cfg, class Epilogue>
void launch_as(const Product &p, const Epilogue &e, hipStream_t stream) {
  product_kernel<T, Cfg><<<(uint32_t)tile_count<Cfg>(p), Cfg::THREADS, 0, stream>>>(p, e);
}

template <class T, class Epilogue>
hipError_t launch(const Product &p, const Epilogue &e, hipStream_t stream) {
  switch (choice_of(p, Epilogue::kRowsOfK, Epilogue::kBy32).shape) {
    case kLarge: launch_as<T, Large>(p, e, stream); break;
    case kBroad:  // rows of 192 are no whole loads
      if constexpr (!Epilogue::kRowsOfK) launch_as<T, Broad>(p, e, stream);
      break;
    case kMedium: launch_as<T, Medium>(p, e, stream); break;
    case kSmall: launch_as<T, Small>(p, e, stream); break;
    case kTiny:
      if constexpr (Epilogue::kBy32) launch_as<T, Tiny>(p, e, stream);
      break;
  }
  return hipGetLastError();
}

// Wave rows of m in the launch of `p`: how many partial results along m an epilogue makes.
inline int64_t wave_rows(const Product &p) {
  switch (shape_of(p)) {
    case kLarge: return tiles_of(p.m, Large::BM) * Large::WAVES_M;
    case kBroad: return tiles_of(p.m, Broad::BM) * Broad::WAVES_M;
    case kMedium: return tiles_of(p.m, Medium::BM) * Medium::WAVES_M;
    case kTiny: return tiles_of(p.m, Tiny::BM) * Tiny::WAVES_M;
    default: return tiles_of(p.m, Small::BM) * Small::WAVES_M;
  }
}

}  // namespace emrs_gemm

#endif
