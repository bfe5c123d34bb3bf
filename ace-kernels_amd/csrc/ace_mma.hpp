// Tiles of a matrix product on the matrix cores of gfx950: the main loop that
// the vocabulary loss's kernels share (ace_vocab.hpp).
//
// A block of WM x WN waves forms a BM x BN tile of
//
//     C[m][n] = sum_k A(m, k) B(n, k)
//
// from two operands in device memory that are each stored one of two ways:
//
//   k contiguous  rows of k, one per m (or n): LDS holds 64 bytes of k of
//                 each row, read as 16-byte fragments (ds_read_b128);
//   m contiguous  rows of m (or n), one per k: LDS holds the rows of one step
//                 of k, read through the transposing LDS load
//                 (ds_read_b64_tr_b16: lane n of a group of 16 gets column n of
//                 the group's 4 x 16 block), so no operand is ever transposed
//                 in memory.
//
// A step of k is 64 bytes wide (32 elements of 16 bits, 16 floats).  LDS holds a
// ring of steps, four in the large tiles: while the products of step s run, step
// s + 1 goes from LDS to registers and step s + 3 from memory to LDS directly (global_load_lds, 16
// bytes a lane), so that neither latency is waited for; one barrier a step.  Rows
// of LDS are swizzled in units of 16 bytes (k contiguous) or of 16 columns (m
// contiguous), on the side of the global address because the LDS side of such a
// load is fixed, so that the lanes one LDS cycle serves touch different banks.
//
// Accumulators are float32 throughout.  In C, lane l of a wave holds, for each
// 16 x 16 piece, column n = l % 16 and the four rows m = 4 (l / 16) + 0..3.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ace_deal.hpp"

namespace ace {
namespace mma {

using f32x4 = float __attribute__((ext_vector_type(4)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));

template <typename T>
constexpr int kStep = kStepBytes / (int)sizeof(T);  // elements of k in one step

__device__ inline char* lds_base() {
  extern __shared__ __align__(1024) char ace_mma_lds[];
  return ace_mma_lds;
}

// 16 bytes a lane from memory to LDS at `dst` (the wave's) + 16 lane: from a
// uniform base and the lane's offset, or from the lane's own address.  With ASM
// it is written as assembler: the compiler waits for every load to LDS that it
// knows of before each transposing LDS read, which takes the whole pipeline away
// (8192 x 8192 x 4096 in bfloat16: 820 TFLOP/s instead of 1146).  Nothing here has
// an output, and the waits for the data are landed_barrier's.  What the compiler
// would do for an instruction of its own is done in the block: a vector memory
// instruction may read scalar registers that a vector instruction wrote
// (v_readfirstlane) no sooner than five wait states later, which is the move and
// four of s_nop 3 (the load that follows a write of m0 needs one of them).  Where no
// transposing reads are, the builtin leaves the compiler more freedom (1200 instead
// of 1140).
__device__ inline uint32_t lds_address(const char* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane(
      (int)(uintptr_t)(__attribute__((address_space(3))) const char*)p);
}
__device__ inline const char* uniform(const char* p) {
  const uint64_t a = (uint64_t)p;
  const uint32_t low = (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
  const uint32_t high = (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32));
  return (const char*)((uint64_t)high << 32 | low);
}
template <bool ASM>
__device__ inline void load_to_lds(const char* base, uint32_t off, char* dst) {
  if constexpr (ASM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                     lds_address(dst)),
                 "v"(off), "s"(uniform(base))
                 : "m0");
  else
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + off),
                                     (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
template <bool ASM>
__device__ inline void load_to_lds(const char* src, char* dst) {
  if constexpr (ASM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                     lds_address(dst)),
                 "v"(src)
                 : "m0");
  else
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// All but the wave's last N memory operations are done, its LDS reads are, and
// every wave has come here.
template <int N>
__device__ inline void landed_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// One operand's side of a tile: R rows (free index) by one step of k.
// PAIRED: fragments come in pairs of 32 rows, in which the first has rows
// 8 q + 0..3 and the second 8 q + 4..7 (q = 0..3), so that a lane's eight values of
// the pair are neighbours in C.
template <typename T, int R, bool KC, int THREADS, bool ASM, bool PAIRED = false>
struct Operand {
  static constexpr int kBytes = R * kStepBytes;
  static constexpr int kChunks = KC ? kStepBytes / 16 : R * (int)sizeof(T) / 16;  // per LDS row
  static constexpr int kLoads = (kBytes + 16 * THREADS - 1) / (16 * THREADS);
  static_assert(kBytes % 1024 == 0, "whole waves load");
  static_assert(KC || R * (int)sizeof(T) >= 64, "rows of at least 64 bytes");

  // Which 16-byte chunk of the row holds logical chunk c (its own inverse).
  __device__ static int swizzle(int row, int c) {
    if constexpr (KC) {
      // a cycle of 16-byte reads serves lanes l..l+7 and l+16..l+23: eight rows,
      // two neighbouring chunks of each; rows 4 (paired: 8) apart share banks
      return c ^ ((row >> (PAIRED ? 2 : 1)) & 2);
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

  // Whether this wave has a part in load i.
  __device__ static bool has(int i) {
    return kBytes % (16 * THREADS) == 0 || i < kLoads - 1 ||
           (i * THREADS + (int)threadIdx.x / 64 * 64) * 16 < kBytes;
  }
  __device__ static char* at(char* lds, int i) {
    return lds + (i * THREADS + (int)threadIdx.x / 64 * 64) * 16;
  }

  // Load i of one step into LDS at `lds`.  `base` (uniform): the operand at the
  // tile's first free index and the step's first k.
  __device__ void load(int i, const char* base, char* lds) const {
    if (has(i)) load_to_lds<ASM>(base, off[i], at(lds, i));
  }

  // All loads of a step of which only `left` k's exist; the others are read from
  // `zeros` (16 zero bytes).
  __device__ void load_tail(const char* base, char* lds, int left, const char* zeros) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = i * THREADS + (int)threadIdx.x;
      const int row = c / kChunks;
      const int k = KC ? swizzle(row, c % kChunks) * (16 / (int)sizeof(T)) : row;
      if (has(i)) load_to_lds<ASM>(k < left ? base + off[i] : zeros, at(lds, i));
    }
  }
};

// Fragments of the matrix instructions, one a step.  16 bits: 32 k's an
// instruction, lane group g = l / 16 holds k = 8 g + 0..7.  float32: four
// instructions of 4 k's, instruction j takes k = 4 g + j of lane group g.
template <typename T>
struct Frag {
  s16x8 v;
};
template <>
struct Frag<float> {
  f32x4 v;
};

// Fragment i of the rows that begin at `row`.
template <typename T, int R, bool KC, bool PAIRED = false>
__device__ inline Frag<T> read_frag(const char* lds, int row, int i) {
  static_assert(KC || sizeof(T) == 2 || !PAIRED, "pairs: not through single floats");
  using Op = Operand<T, R, KC, 64, false, PAIRED>;
  if constexpr (!PAIRED) row += 16 * i;
  const int lane = (int)threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  Frag<T> f;
  if constexpr (KC) {
    const int r = PAIRED ? row + 32 * (i >> 1) + 8 * (n >> 2) + 4 * (i & 1) + (n & 3) : row + n;
    const char* at = lds + r * kStepBytes + Op::swizzle(r, g) * 16;
    f.v = *reinterpret_cast<const decltype(f.v)*>(at);
  } else if constexpr (sizeof(T) == 2) {
    s16x4 h[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int k = 8 * g + 4 * half + (n >> 2);  // the lane's row of the 4 x 16 block
      const int c = PAIRED ? row / 8 + 4 * (i >> 1) + (n & 3) : row / 8 + ((n >> 1) & 1);
      const char* at =
          lds + k * (R * 2) + Op::swizzle(k, c) * 16 + (PAIRED ? i & 1 : n & 1) * 8;
      h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(at));
    }
    f.v = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 4 * g + j;
      const int c = row + n;
      f.v[j] = *reinterpret_cast<const float*>(lds + k * (R * 4) + Op::swizzle(k, c / 4) * 16 +
                                               (c & 3) * 4);
    }
  }
  return f;
}

// Instruction j of kParts<T> that multiply two fragments.
template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 4 : 1;
template <typename T>
__device__ inline f32x4 multiply(const Frag<T>& a, const Frag<T>& b, f32x4 c, int j);
template <>
__device__ inline f32x4 multiply<__bf16>(const Frag<__bf16>& a, const Frag<__bf16>& b, f32x4 c,
                                         int) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v),
                                                 __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
}
template <>
__device__ inline f32x4 multiply<_Float16>(const Frag<_Float16>& a, const Frag<_Float16>& b,
                                           f32x4 c, int) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v),
                                                __builtin_bit_cast(f16x8, b.v), c, 0, 0, 0);
}
template <>
__device__ inline f32x4 multiply<float>(const Frag<float>& a, const Frag<float>& b, f32x4 c,
                                        int j) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
}

// A BM x BN tile by WM x WN waves.
template <typename T_, int BM_, int BN_, int WM_, int WN_, bool AKC_, bool BKC_,
          bool PAIRED_ = false>
struct Tile {
  using T = T_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // 16 x 16 pieces of a wave
  static constexpr int kStageBytes = (BM + BN) * kStepBytes;
  // steps in LDS, and between loading one and multiplying it: the narrowest tiles have
  // little to do in a step, and wait for memory unless more of them are on the way
  static constexpr int kRing = BN <= 32 ? 7 : 4, kAhead = kRing - 1;
  static constexpr int kLdsBytes = kRing * kStageBytes;
  static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "whole pieces");
  // waves a SIMD that the registers must allow: two, or as many blocks as LDS holds
  static constexpr int kWaves = BN == 64 ? 3 : 2;
  static constexpr bool kAsm = sizeof(T) == 2 && !(AKC_ && BKC_);  // transposing reads
  static constexpr bool kPaired = PAIRED_;  // the first operand's fragments
  using OpA = Operand<T, BM, AKC_, kThreads, kAsm, PAIRED_>;
  using OpB = Operand<T, BN, BKC_, kThreads, kAsm>;

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
    if (left >= kStep<T>) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load_one(i, a, b, sa, sb, step, lds);
    } else {
      a.load_tail(sa.base + step * sa.step, lds, left, zeros);
      b.load_tail(sb.base + step * sb.step, lds + OpA::kBytes, left, zeros);
    }
  }
  static constexpr int kLoads = OpA::kLoads + OpB::kLoads;  // of a step
  __device__ static void load_one(int i, const OpA& a, const OpB& b, Source sa, Source sb, int step,
                                  char* lds) {
    if (i < OpA::kLoads)
      a.load(i, sa.base + step * sa.step, lds);
    else
      b.load(i - OpA::kLoads, sb.base + step * sb.step, lds + OpA::kBytes);
  }

  struct Frags {
    Frag<T> a[MT], b[NT];
  };

  // Fragments first..last-1 of a step, those of b before those of a.
  __device__ static void read(const char* lds, Frags& f, int first = 0, int last = MT + NT) {
    const int m0 = wave_m(), n0 = wave_n();
#pragma unroll
    for (int i = first; i < last; ++i) {
      if (i < NT)
        f.b[i] = read_frag<T, BN, BKC_>(lds + OpA::kBytes, n0, i);
      else
        f.a[i - NT] = read_frag<T, BM, AKC_, PAIRED_>(lds, m0, i - NT);
    }
  }

  // Neighbouring instructions add to different pieces: one that waits for the
  // result of the one before takes longer.
  __device__ static void multiply_all(const Frags& f, f32x4 (&acc)[MT][NT]) {
#pragma unroll
    for (int q = 0; q < kParts<T>; ++q)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = multiply<T>(f.a[i], f.b[j], acc[i][j], q);
  }

  // False: this wave has no part in the last load of a step.
  __device__ static bool loads_all() {
    static_assert(OpA::kBytes % (16 * kThreads) == 0, "whole loads of the first operand");
    return OpB::has(OpB::kLoads - 1);
  }

  // Spreads a step's LDS reads (and with them the loads between them) evenly among
  // its matrix instructions, so that the matrix cores do not wait for a burst.
  __device__ static void interleave() {
    constexpr int reads_a = MT * (AKC_ ? 1 : sizeof(T) == 4 ? 4 : 2);
    constexpr int reads_b = NT * (BKC_ ? 1 : sizeof(T) == 4 ? 4 : 2);
    constexpr int n = MT * NT * kParts<T>, reads = reads_a + reads_b;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
      const int r = (i + 1) * reads / n - i * reads / n;
      if (r == 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS reads
      if (r == 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      if (r > 2) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      if (!kAsm && (i + 1) * kLoads / n > i * kLoads / n)
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // a load
    }
  }

  // The main loop over a sequence of steps that may span tiles.
  struct Pipe {
    int fed = 0, done = 0;  // steps loaded, and multiplied
    Frags now;

    __device__ char* slot(int step) const { return lds_base() + (step % kRing) * kStageBytes; }

    // Nothing else may be reading LDS.  `feed(lds)` loads the next step of the
    // sequence to `lds` and says whether there was one.
    template <typename Feed>
    __device__ void begin(Feed feed) {
      for (int i = 0; i < kAhead; ++i)
        if (feed(slot(fed))) ++fed;
      landed_barrier<0>();
      if (fed) read(slot(0), now);
    }

    // `n` steps into acc, of which at least the first `plain` have a `simple(i, lds)`
    // in place of the feed: it makes load i of a whole step, without a condition.
    template <typename Simple, typename Feed>
    __device__ void run(int n, int plain, Simple simple, Feed feed, f32x4 (&acc)[MT][NT]) {
      Frags next;
      int s = 0;
      for (; s + 2 <= plain; s += 2) {
        plain_step(simple, now, next, acc);
        plain_step(simple, next, now, acc);
      }
      for (; s + 2 <= n; s += 2) {
        any_step(feed, now, next, acc);
        any_step(feed, next, now, acc);
      }
      if (s < n) {
        any_step(feed, now, next, acc);
        now = next;
      }
    }

    template <typename Simple>
    __device__ void plain_step(Simple simple, const Frags& f, Frags& next, f32x4 (&acc)[MT][NT]) {
      if (loads_all())  // step done + 1 has landed
        landed_barrier<kLoads*(kAhead - 2)>();
      else
        landed_barrier<(kLoads - 1) * (kAhead - 2)>();
      // loads and reads in turn: neither is moved past the other
      constexpr int all = MT + NT;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        simple(i, slot(fed));
        read(slot(done + 1), next, i * all / kLoads, (i + 1) * all / kLoads);
      }
      multiply_all(f, acc);
      interleave();
      ++fed;
      ++done;
    }

    template <typename Feed>
    __device__ void any_step(Feed feed, const Frags& f, Frags& next, f32x4 (&acc)[MT][NT]) {
      if (fed - done < kAhead)  // the end of the sequence
        landed_barrier<0>();
      else if (loads_all())
        landed_barrier<kLoads*(kAhead - 2)>();
      else
        landed_barrier<(kLoads - 1) * (kAhead - 2)>();
      if (feed(slot(fed))) ++fed;
      read(slot(done + 1), next);  // past the end: whatever the slot holds, unused
      multiply_all(f, acc);
      ++done;
    }
  };

  // How many of a tile's steps first..last-1 of k values may feed simply: those
  // whose step kAhead on is whole and in the tile.
  __device__ static int plain_steps(int first, int last, int k) {
    const int whole = k / kStep<T> < last ? k / kStep<T> : last;
    const int n = whole - first - kAhead;
    return n > 0 ? n : 0;
  }
};

// Consecutive launch indices go to the 8 XCDs in turn: this numbers the blocks so
// that each XCD has a run of neighbours, which share its L2.
__device__ inline int xcd_order(int b, int blocks) {
  const int x = b & 7, base = blocks >> 3, rest = blocks & 7;
  return x * base + (x < rest ? x : rest) + (b >> 3);
}

}  // namespace mma
}  // namespace ace
