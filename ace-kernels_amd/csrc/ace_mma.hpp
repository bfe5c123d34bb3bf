// Tiles of a matrix product on the matrix cores of gfx950: the main loop that
// the vocabulary loss's kernels share (ace_vocab.hpp).
//
// A block of WM x WN waves forms a BM x BN tile of
//
//     C[m][n] = sum_k A(m, k) B(n, k)
//
// from two operands in device memory that are each stored one of two ways:
//
//   k contiguous  rows of k, one per m (or n): LDS holds 128 bytes of k of
//                 each row, read as 16-byte fragments (ds_read_b128);
//   m contiguous  rows of m (or n), one per k: LDS holds the rows of one step
//                 of k, read through the transposing LDS load
//                 (ds_read_b64_tr_b16: lane n of a group of 16 gets column n of
//                 the group's 4 x 16 block), so no operand is ever transposed
//                 in memory.
//
// A step of k is 128 bytes wide (64 elements of 16 bits, 32 floats).  Operands
// go from memory to LDS directly (global_load_lds, 16 bytes a lane), one step
// ahead of the products, into the other of two buffers.  Rows of LDS are
// swizzled in units of 16 bytes (k contiguous) or of 16 columns (m contiguous),
// on the side of the global address because the LDS side of such a load is
// fixed, so that the lanes one LDS cycle serves touch different banks.
//
// Accumulators are float32 throughout.  In C, lane l of a wave holds, for each
// 16 x 16 piece, column n = l % 16 and the four rows m = 4 (l / 16) + 0..3.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ace {
namespace mma {

using f32x4 = float __attribute__((ext_vector_type(4)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));

constexpr int kStepBytes = 128;  // bytes of k in one step

template <typename T>
constexpr int kStep = kStepBytes / (int)sizeof(T);  // elements of k in one step

__device__ inline char* lds_base() {
  extern __shared__ __align__(1024) char ace_mma_lds[];
  return ace_mma_lds;
}

// 16 bytes a lane from `src` (the lane's own address) to LDS at `dst` (the
// wave's) + 16 lane.
__device__ inline void load_to_lds(const char* src, char* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// Every load to LDS of this wave has landed, and every wave has come here.
__device__ inline void landed_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
}

// One operand's side of a tile: R rows (free index) by one step of k.
template <typename T, int R, bool KC, int THREADS>
struct Operand {
  static constexpr int kBytes = R * kStepBytes;
  static constexpr int kChunks = KC ? kStepBytes / 16 : R * (int)sizeof(T) / 16;  // per LDS row
  static constexpr int kLoads = (kBytes + 16 * THREADS - 1) / (16 * THREADS);
  static_assert(kBytes % 1024 == 0, "whole waves load");
  static_assert(KC || R * (int)sizeof(T) >= 64, "rows of at least 64 bytes");

  // Which 16-byte chunk of the row holds logical chunk c (its own inverse).
  __device__ static int swizzle(int row, int c) {
    if constexpr (KC) {
      return c ^ (row & 7);
    } else if constexpr (sizeof(T) == 2) {
      // units of 16 columns: the 16 rows of one transposing read are
      // 8 g + j (+ 4), g and j in 0..3
      constexpr int units = R / 16;
      const int f = ((row & 3) | ((row >> 1) & 12)) & (units - 1);
      return c ^ (f << 1);
    } else {
      constexpr int units = R / 16;
      return c ^ (((row >> 2) & 3 & (units - 1)) << 2);
    }
  }

  uint32_t off[kLoads];  // from the operand's base at k = 0 of a step

  // `stride`: bytes between rows in memory; `first`, `limit`: the tile's first
  // free index and how many there are (> first).  Indices past the limit read
  // the last valid row or chunk: their results are not used.
  __device__ void init(int64_t stride, int64_t first, int64_t limit) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = i * THREADS + (int)threadIdx.x;
      const int row = c / kChunks, lc = swizzle(row, c % kChunks);
      if constexpr (KC) {
        const int64_t last = limit - 1 - first;
        off[i] = (uint32_t)((row < last ? row : last) * stride + lc * 16);
      } else {
        const int64_t last = (limit - first) * (int64_t)sizeof(T) - 16;
        const int64_t at = lc * 16;
        off[i] = (uint32_t)(row * stride + (at < last ? at : last));
      }
    }
  }

  // Loads one step into LDS at `lds`.  `base`: the operand at the tile's first
  // free index and the step's first k.  With TAIL, `left` k's are left (fewer
  // than a step); the others are read from `zeros` (16 zero bytes).
  template <bool TAIL>
  __device__ void load(const char* base, char* lds, int left, const char* zeros) const {
    const int wave = (int)threadIdx.x / 64;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (kBytes % (16 * THREADS) != 0 && i == kLoads - 1 &&
          (i * THREADS + wave * 64) * 16 >= kBytes)
        break;  // whole waves have nothing to load
      const char* src = base + off[i];
      if constexpr (TAIL) {
        const int c = i * THREADS + (int)threadIdx.x;
        const int row = c / kChunks;
        const int k = KC ? swizzle(row, c % kChunks) * (16 / (int)sizeof(T)) : row;
        if (k >= left) src = zeros;
      }
      load_to_lds(src, lds + (i * THREADS + wave * 64) * 16);
    }
  }
};

// Fragments of the matrix instructions.  16 bits: 32 k's an instruction, lane
// group g = l / 16 holds k = 8 g + 0..7.  float32: four instructions of 4 k's
// for 16 k's, instruction j takes k = 4 g + j of lane group g.
template <typename T>
struct Frag {
  s16x8 v;
};
template <>
struct Frag<float> {
  f32x4 v;
};

constexpr int kSub = 2;  // fragments of k per step

// The fragment `kk` of the 16 rows that begin at `row`.
template <typename T, int R, bool KC>
__device__ inline Frag<T> read_frag(const char* lds, int row, int kk) {
  using Op = Operand<T, R, KC, 64>;
  const int lane = (int)threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  Frag<T> f;
  if constexpr (KC) {
    const int r = row + n;
    const char* at = lds + r * kStepBytes + Op::swizzle(r, kk * 4 + g) * 16;
    f.v = *reinterpret_cast<const decltype(f.v)*>(at);
  } else if constexpr (sizeof(T) == 2) {
    s16x4 h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = kk * 32 + 8 * g + 4 * i + (n >> 2);  // the lane's row of the 4 x 16 block
      const char* at =
          lds + k * (R * 2) + Op::swizzle(k, row / 8 + ((n >> 1) & 1)) * 16 + (n & 1) * 8;
      h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(at));
    }
    f.v = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = kk * 16 + 4 * g + j;
      const int c = row + n;
      f.v[j] = *reinterpret_cast<const float*>(lds + k * (R * 4) + Op::swizzle(k, c / 4) * 16 +
                                               (c & 3) * 4);
    }
  }
  return f;
}

template <typename T>
__device__ inline f32x4 multiply(Frag<T> a, Frag<T> b, f32x4 c);
template <>
__device__ inline f32x4 multiply<__bf16>(Frag<__bf16> a, Frag<__bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v),
                                                 __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
}
template <>
__device__ inline f32x4 multiply<_Float16>(Frag<_Float16> a, Frag<_Float16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v),
                                                __builtin_bit_cast(f16x8, b.v), c, 0, 0, 0);
}
template <>
__device__ inline f32x4 multiply<float>(Frag<float> a, Frag<float> b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// A BM x BN tile by WM x WN waves.
template <typename T_, int BM_, int BN_, int WM_, int WN_, bool AKC_, bool BKC_>
struct Tile {
  using T = T_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // 16 x 16 pieces of a wave
  static constexpr int kStageBytes = (BM + BN) * kStepBytes;
  static constexpr int kLdsBytes = 2 * kStageBytes;
  static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "whole pieces");
  using OpA = Operand<T, BM, AKC_, kThreads>;
  using OpB = Operand<T, BN, BKC_, kThreads>;

  // What one operand needs of memory: its address at the tile's first free
  // index and k = 0, and the bytes from one step of k to the next.
  struct Source {
    const char* base;
    int64_t step;
  };

  __device__ static int wave_m() { return ((int)threadIdx.x / 64 / WN) * (BM / WM); }
  __device__ static int wave_n() { return ((int)threadIdx.x / 64 % WN) * (BN / WN); }

  __device__ static void clear(f32x4 (&acc)[MT][NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  __device__ static void load(const OpA& a, const OpB& b, Source sa, Source sb, int step, int k,
                              char* lds, const char* zeros) {
    const int left = k - step * kStep<T>;
    const char* pa = sa.base + step * sa.step;
    const char* pb = sb.base + step * sb.step;
    if (left >= kStep<T>) {
      a.template load<false>(pa, lds, left, zeros);
      b.template load<false>(pb, lds + OpA::kBytes, left, zeros);
    } else {
      a.template load<true>(pa, lds, left, zeros);
      b.template load<true>(pb, lds + OpA::kBytes, left, zeros);
    }
  }

  __device__ static void step(const char* lds, f32x4 (&acc)[MT][NT]) {
    const int m0 = wave_m(), n0 = wave_n();
#pragma unroll
    for (int kk = 0; kk < kSub; ++kk) {
      Frag<T> a[MT], b[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
        b[j] = read_frag<T, BN, BKC_>(lds + OpA::kBytes, n0 + 16 * j, kk);
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = read_frag<T, BM, AKC_>(lds, m0 + 16 * i, kk);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = multiply<T>(a[i], b[j], acc[i][j]);
    }
  }

  // acc += the product over steps first..last-1 of a k values long product.  The
  // caller's waves all come here with the same arguments, with nothing reading
  // LDS any more.
  __device__ static void product(const OpA& a, const OpB& b, Source sa, Source sb, int first,
                                 int last, int k, const char* zeros, f32x4 (&acc)[MT][NT]) {
    char* lds = lds_base();
    if (first >= last) return;
    load(a, b, sa, sb, first, k, lds, zeros);
    for (int s = first; s < last; ++s) {
      char* here = lds + ((s - first) & 1) * kStageBytes;
      landed_barrier();  // step s is in LDS, and nothing reads the other buffer
      if (s + 1 < last)
        load(a, b, sa, sb, s + 1, k, lds + ((s + 1 - first) & 1) * kStageBytes, zeros);
      step(here, acc);
    }
  }
};

// Work of a kernel in `total` equal units spread evenly over `blocks` blocks:
// block b does units [begin(b), begin(b + 1)).  Units are dealt in order, so a
// block's units are neighbours; consecutive launch indices go to the 8 XCDs in
// turn, and `order` gives each XCD a run of neighbouring blocks, which then share
// its L2.
struct Spread {
  int64_t total;
  int blocks;
  __device__ int64_t begin(int b) const { return b * total / blocks; }
  __device__ int owner(int64_t unit) const {
    return (int)(((unit + 1) * blocks - 1) / total);
  }
};

__device__ inline int xcd_order(int b, int blocks) {
  const int x = b & 7, base = blocks >> 3, rest = blocks & 7;
  return x * base + (x < rest ? x : rest) + (b >> 3);
}

}  // namespace mma
}  // namespace ace
