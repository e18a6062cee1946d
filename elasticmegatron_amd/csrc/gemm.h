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
// c ^ swizzle(r): the 16 rows that a fragment read takes at one c then lie in 16 different slots of the
// 64 banks.  Rows past the operand's last are past the buffer's end and read as zeros, and so are, by
// their lane's offset, units past the last k.
#ifndef EMRS_GEMM_H
#define EMRS_GEMM_H

#include <hip/hip_runtime.h>

#include <cstdint>

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

// Up to three products that are summed into one C: operands that are held as a sum of two 16-bit parts
// multiply as hi*hi + hi*lo + lo*hi, which is only more k.
struct Product {
  const void *a[3];
  const void *b[3];
  int64_t a_stride, b_stride;      // elements between rows, multiples of 8
  int64_t a_batch, b_batch;        // elements between the matrices of a batch
  int32_t m, n, k;                 // k a multiple of 8
  int32_t parts;                   // 1 to 3
  int32_t batch;
  int32_t symmetric;               // only tiles on and below the diagonal (m >= n) are computed
};

template <int BM_, int BN_, int WM_, int WN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_;
  static constexpr int WAVES_M = BM / WM_, WAVES_N = BN / WN_, WAVES = WAVES_M * WAVES_N;
  static constexpr int WM = WM_, WN = WN_;
  static constexpr int MI = WM / 16, NI = WN / 16;
  static constexpr int THREADS = WAVES * 64;
  static constexpr int A_LOADS = BM / 8 / WAVES, B_LOADS = BN / 8 / WAVES;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole 1 KB loads per wave");
};

// 256 x 256 with 8 waves of 128 x 64: a stage is 64 KB, and its 2^23 multiply-adds are 2048 cycles of the
// CU's matrix units against 96 KB of fragment reads.  The smaller tiles are for products that would not
// give every CU a large one.
using Large = Tile<256, 256, 128, 64>;
using Medium = Tile<128, 128, 64, 64>;
using Small = Tile<64, 64, 32, 32>;

__host__ __device__ inline int64_t tiles_of(int64_t n, int64_t t) { return (n + t - 1) / t; }
template <class Cfg>
__host__ inline int64_t tile_count(const Product &p) {
  const int64_t tm = tiles_of(p.m, Cfg::BM), tn = tiles_of(p.n, Cfg::BN);
  return (p.symmetric ? tm * (tm + 1) / 2 : tm * tn) * p.batch;
}

struct Where {
  int m0, n0, batch;
};

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
  if (p.symmetric) {  // row i of the triangle holds i + 1 tiles
    i = (uint32_t)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > t) --i;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    j = t - i * (i + 1) / 2;
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

// Of the row's place among 16 alone, so that a wave reads its fragments at constant offsets of one address.
__device__ inline int swizzle(int row) { return (row ^ ((row >> 3) & 1)) & 7; }

template <class T, int LOADS, int WAVES>
struct Loader {
  int voffset[LOADS];
  int unit;  // the 16-byte unit of a row that this lane loads, per load: alternates with the row group
  __device__ void init(int64_t stride, int wave, int lane) {
    for (int j = 0; j < LOADS; ++j) {
      const int row = (wave + j * WAVES) * 8 + (lane >> 3);
      voffset[j] = (int)(row * stride * 2) + (((lane & 7) ^ swizzle(row)) << 4);
    }
  }
  // k0: first k of the stage; tail: k that are left from there, when fewer than a stage.
  __device__ void load(__amdgpu_buffer_rsrc_t r, char *lds, int k0, int k, int wave, int lane) const {
    for (int j = 0; j < LOADS; ++j) {
      const int group = wave + j * WAVES;
      int v = voffset[j];
      if (k - k0 < kStage) {
        const int c = (lane & 7) ^ swizzle(group * 8 + (lane >> 3));
        v = c * 8 < k - k0 ? v : (int)0x80000000;  // past the buffer's end: reads zeros
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + group * 1024), 16, v,
                                               k0 * 2, 0, 0);
    }
  }
};

// The buffer that holds a tile's rows of one operand: nothing past its last row's last k is read.
template <class T>
__device__ inline __amdgpu_buffer_rsrc_t rows_buffer(const void *base, int64_t batch, int64_t first, int rows, int64_t stride,
                                                     int k) {
  const T *p = static_cast<const T *>(base) + batch + first * stride;
  const int64_t bytes = ((int64_t)(rows - 1) * stride + k) * 2;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(p), 0, (int)bytes, 0x00020000);
}

template <class T, class Cfg, class Epilogue>
__global__ __launch_bounds__(Cfg::THREADS) void product_kernel(Product p, Epilogue epilogue) {
  using x8 = typename Vec<T>::x8;
  __shared__ __attribute__((aligned(1024))) char a_even[Cfg::BM * 128];
  __shared__ __attribute__((aligned(1024))) char a_odd[Cfg::BM * 128];
  __shared__ __attribute__((aligned(1024))) char b_even[Cfg::BN * 128];
  __shared__ __attribute__((aligned(1024))) char b_odd[Cfg::BN * 128];
  const Where w = tile_of<Cfg>(p);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;

  Loader<T, Cfg::A_LOADS, Cfg::WAVES> la;
  Loader<T, Cfg::B_LOADS, Cfg::WAVES> lb;
  la.init(p.a_stride, wave, lane);
  lb.init(p.b_stride, wave, lane);
  const int a_rows = min(Cfg::BM, p.m - w.m0), b_rows = min(Cfg::BN, p.n - w.n0);
  const int stages = (p.k + kStage - 1) / kStage, total = stages * p.parts;
  int part = 0, stage = 0;
  auto load = [&](char *a, char *b) {
    const int k0 = stage * kStage;
    la.load(rows_buffer<T>(p.a[part], w.batch * p.a_batch, w.m0, a_rows, p.a_stride, p.k), a, k0, p.k, wave, lane);
    lb.load(rows_buffer<T>(p.b[part], w.batch * p.b_batch, w.n0, b_rows, p.b_stride, p.k), b, k0, p.k, wave, lane);
    if (++stage == stages) {
      stage = 0;
      ++part;
    }
  };

  f32x4 acc[Cfg::MI][Cfg::NI];
#pragma unroll
  for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
    for (int j = 0; j < Cfg::NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int row = lane & 15, c = lane >> 4;
  const int unit[2] = {(c ^ swizzle(row)) << 4, ((4 + c) ^ swizzle(row)) << 4};
  const int a_at = (wm * Cfg::WM + row) * 128, b_at = (wn * Cfg::WN + row) * 128;
  auto compute = [&](const char *a, const char *b) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      x8 fa[Cfg::MI], fb[Cfg::NI];
#pragma unroll
      for (int j = 0; j < Cfg::NI; ++j) fb[j] = *reinterpret_cast<const x8 *>(b + b_at + unit[kk] + j * 2048);
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) fa[i] = *reinterpret_cast<const x8 *>(a + a_at + unit[kk] + i * 2048);
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
        for (int j = 0; j < Cfg::NI; ++j) acc[i][j] = mfma(fa[i], fb[j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  load(a_even, b_even);
  int it = 0;
  for (; it + 1 < total; it += 2) {
    __syncthreads();  // the even stage is filled, and every wave is done with the odd one
    load(a_odd, b_odd);
    compute(a_even, b_even);
    __syncthreads();
    if (it + 2 < total) load(a_even, b_even);
    compute(a_odd, b_odd);
  }
  if (it < total) {
    __syncthreads();
    compute(a_even, b_even);
  }
  epilogue.template run<Cfg>(acc, w, w.m0 + wm * Cfg::WM, w.n0 + wn * Cfg::WN, wm, lane, p);
}

enum Shape { kLarge, kMedium, kSmall };

// The largest tile that keeps most CUs busy: a larger one reads its operands fewer times from the caches.
inline Shape shape_of(const Product &p) {
  return tile_count<Large>(p) >= 192 ? kLarge : tile_count<Medium>(p) >= 128 ? kMedium : kSmall;
}

template <class T, class Epilogue>
hipError_t launch(const Product &p, const Epilogue &e, hipStream_t stream) {
  switch (shape_of(p)) {
    case kLarge:
      product_kernel<T, Large, Epilogue><<<(uint32_t)tile_count<Large>(p), Large::THREADS, 0, stream>>>(p, e);
      break;
    case kMedium:
      product_kernel<T, Medium, Epilogue><<<(uint32_t)tile_count<Medium>(p), Medium::THREADS, 0, stream>>>(p, e);
      break;
    case kSmall:
      product_kernel<T, Small, Epilogue><<<(uint32_t)tile_count<Small>(p), Small::THREADS, 0, stream>>>(p, e);
  }
  return hipGetLastError();
}

// Wave rows of m in the launch of `p`: how many partial results along m an epilogue makes.
inline int64_t wave_rows(const Product &p) {
  switch (shape_of(p)) {
    case kLarge: return tiles_of(p.m, Large::BM) * Large::WAVES_M;
    case kMedium: return tiles_of(p.m, Medium::BM) * Medium::WAVES_M;
    default: return tiles_of(p.m, Small::BM) * Small::WAVES_M;
  }
}

}  // namespace emrs_gemm

#endif
