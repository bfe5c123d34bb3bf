// Tokens sorted by expert, their rows in that order, and the experts' rows added
// back to their tokens (ace_expert_order, ace_to_experts, ace_from_experts and
// ace_from_experts_backward, declared in include/ace_hip.h).
//
// A token's k choices are its slots, slot s = token k + j.  The order is a stable
// counting sort of the slots by expert, slots without an expert left out:
//
//   place_s = offset_e + |{s' < s : e_s' = e_s}|,   source_place_s = s
//
//   to:    rows[place_tj] = x_t                 dx_t  = sum_j drows[place_tj]
//   from:  out_t = sum_j w_tj rows[place_tj]    drows[place_tj] = w_tj dout_t
//                                               dw_tj = <rows[place_tj], dout_t>
//
// A slot is at a row where place and source agree on it, so that no two slots are at
// one, whatever a caller has made of them (choices are dropped by a place of -1).
// Rows without a slot are 0 where they are written, and not read.
// Everything is a copy's work: bytes of rows at the rate of memory.  Where they do not
// fit the last-level cache, stores go past it (8192 x 8 rows of 2048 in bfloat16 back to
// their tokens and their gradients: 153 us instead of 180).
//
// Sums over a token's rows and over a row's width are float32, in an order that the
// sizes alone decide; no atomic's order reaches a result (the order's counts are
// integers).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ace_core.hpp"  // wave_sync
#include "ace_piece.hpp"

namespace ace {
namespace experts {

constexpr int kMaxExperts = 512;
constexpr int kBlock = 256, kWaves = kBlock / 64;
constexpr int kOrderBlock = 1024;
constexpr int kMaxBlocks = 256;  // of the order: each adds up the counts of those before it

// -------------------------------------------------------------------- order

struct OrderParams {
  const int64_t* chosen;  // [slots]
  int64_t slots;
  int experts;
  int blocks;
  int64_t per_block;      // slots, whole rounds of the block
  int* counts;            // [blocks][experts]
  int64_t* offsets;       // [experts + 1]
  int64_t* source;        // [slots]
  int64_t* place;         // [slots]
};

// The choice at slot s, -1: none.
__device__ inline int choice(const OrderParams& p, int64_t s, int64_t end) {
  if (s >= end) return -1;
  const int64_t e = p.chosen[s];
  return e >= 0 && e < p.experts ? (int)e : -1;
}

// How often each expert is chosen in a block's slots.
__global__ __launch_bounds__(kOrderBlock) void count_kernel(OrderParams p) {
  __shared__ int s_count[kMaxExperts];
  const int tid = (int)threadIdx.x;
  for (int e = tid; e < p.experts; e += kOrderBlock) s_count[e] = 0;
  __syncthreads();
  const int64_t s0 = blockIdx.x * p.per_block;
  const int64_t s1 = s0 + p.per_block < p.slots ? s0 + p.per_block : p.slots;
  for (int64_t s = s0 + tid; s < s1; s += kOrderBlock) {
    const int e = choice(p, s, s1);
    if (e >= 0) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  for (int e = tid; e < p.experts; e += kOrderBlock)
    p.counts[(int64_t)blockIdx.x * p.experts + e] = s_count[e];
}

// The slots' places.  Each wave has a run of the block's slots, and for each expert
// the place that its next slot takes; among 64 slots, those of one expert are found by
// ballots over the bits of its number.  Every block adds up the counts of the others by
// itself, eight loads at a time: 2^20 slots of 256 experts take 25 us, and 95 where a block
// of 256 threads loads one after another.
__global__ __launch_bounds__(kOrderBlock) void place_kernel(OrderParams p) {
  constexpr int kWaves = kOrderBlock / 64;
  __shared__ int s_next[kWaves][kMaxExperts];
  __shared__ int s_all[kMaxExperts], s_before[kMaxExperts];
  __shared__ int s_sum[kWaves];
  __shared__ int64_t s_total;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t per_wave = p.per_block / kWaves;
  const int64_t s0 = blockIdx.x * p.per_block + wave * per_wave;
  const int64_t s1 = s0 + per_wave < p.slots ? s0 + per_wave : p.slots;
  for (int e = tid; e < kMaxExperts; e += kOrderBlock) s_all[e] = s_before[e] = 0;
  for (int i = tid; i < kWaves * kMaxExperts; i += kOrderBlock) (&s_next[0][0])[i] = 0;
  __syncthreads();
  for (int64_t s = s0 + lane; s < s1; s += 64) {
    const int e = choice(p, s, s1);
    if (e >= 0) atomicAdd(&s_next[wave][e], 1);
  }
  if (p.blocks > 1) {  // the blocks' counts, added up over all and over those before
    constexpr int kAhead = 8;
    const uint32_t experts = (uint32_t)p.experts;
    const uint32_t step_e = kOrderBlock % experts, step_b = kOrderBlock / experts;
    uint32_t e = (uint32_t)tid % experts, b = (uint32_t)tid / experts;
    const int n = p.blocks * p.experts;
    for (int i = tid; i < n; i += kAhead * kOrderBlock) {
      int c[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int at = i + a * kOrderBlock;
        c[a] = at < n ? p.counts[at] : 0;
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (c[a]) {
          atomicAdd(&s_all[e], c[a]);
          if (b < blockIdx.x) atomicAdd(&s_before[e], c[a]);
        }
        e += step_e;
        b += step_b;
        if (e >= experts) {
          e -= experts;
          ++b;
        }
      }
    }
  }
  __syncthreads();
  // thread e has expert e
  static_assert(kOrderBlock >= kMaxExperts, "all experts have a thread");
  int before = 0, all = 0;
  if (tid < p.experts) {
    before = s_before[tid];
    all = s_all[tid];
    if (p.blocks == 1) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all += s_next[w][tid];
    }
  }
  int upto = all;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += s_sum[w];
  if (tid == kOrderBlock - 1) s_total = upto;
  if (tid < p.experts) {
    if (blockIdx.x == 0) {
      if (tid == 0) p.offsets[0] = 0;
      p.offsets[tid + 1] = upto;
    }
    int next = upto - all + before;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int n = s_next[w][tid];
      s_next[w][tid] = next;
      next += n;
    }
  }
  __syncthreads();
  int bits = 0;
  while (1 << bits < p.experts) ++bits;
  for (int64_t s = s0; s < s1; s += 64) {
    const int e = choice(p, s + lane, s1);
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long set = __ballot(e >> b & 1);
      same &= e >> b & 1 ? set : ~set;
    }
    int64_t at = -1;
    if (e >= 0) {
      const int earlier = __popcll(same & ((1ull << lane) - 1));
      const int first = s_next[wave][e];
      wave_sync();  // all lanes have read before one writes
      if (earlier == 0) s_next[wave][e] = first + __popcll(same);
      wave_sync();
      at = first + earlier;
      p.source[at] = s + lane;
    }
    if (s + lane < s1) p.place[s + lane] = at;
  }
  for (int64_t s = s_total + (int64_t)blockIdx.x * kOrderBlock + tid; s < p.slots;
       s += (int64_t)p.blocks * kOrderBlock)
    p.source[s] = -1;
}

// --------------------------------------------------------------------- rows

struct RowsParams {
  const void* in;         // to: x [tokens, width]; from: rows [slots, width]
  const void* grad;       // from's backward: dout [tokens, width]
  void* out;              // to: rows; from: out; from's backward: drows
  const int64_t* source;  // [slots]
  const int64_t* place;   // [slots]
  const float* weights;   // [slots] or null: 1
  float* d_weights;       // [slots]
  int64_t tokens, slots;
  int width, top_k;
  int pieces;             // of a row that waves share
  int lanes_log2;         // narrow rows: lanes of one
};

template <typename T>
constexpr int kV = 16 / (int)sizeof(T);
// Pieces of 16 bytes that a lane holds of a row: a wave takes spans of 64 of them.
constexpr int kDeepTo = 4, kDeepFrom = 2, kDeepBack = 4;
constexpr int kAtOnce = 4;  // rows that a wave has on the way
constexpr int kMany = 2;    // slots that a lane takes of narrow rows

template <typename T, int D>
struct Span {
  static constexpr int V = kV<T>, kWidth = 64 * D * V;
  Piece<T> x[D];

  __device__ void clear() {
#pragma unroll
    for (int u = 0; u < D; ++u) x[u].fill((T)0.f);
  }
  // From element `first` of a row; what is behind the row's end reads as 0 and is
  // not written.
  __device__ void load(const T* row, int first, int width) {
#pragma unroll
    for (int u = 0; u < D; ++u) {
      const int at = first + (u * 64 + ((int)threadIdx.x & 63)) * V;
      if (at + V <= width)
        x[u].load(row + at);
      else
        x[u].load_some(row + at, width - at, (T)0.f);
    }
  }
  template <bool STREAM>
  __device__ void store(T* row, int first, int width) const {
#pragma unroll
    for (int u = 0; u < D; ++u) {
      const int at = first + (u * 64 + ((int)threadIdx.x & 63)) * V;
      if (at + V <= width)
        x[u].template store<STREAM>(row + at);
      else
        x[u].store_some(row + at, width - at);
    }
  }
};

// The same for the whole wave, in a scalar register.
__device__ inline int wave_number() {
  return __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kWaves + threadIdx.x / 64));
}
__device__ inline float lane_value(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}
// The row that a slot is at (below 2^26), -1: none.
__device__ inline int place_of(const RowsParams& p, int64_t slot) {
  const int64_t at = p.place[slot];
  return at >= 0 && at < p.slots && p.source[at] == slot ? (int)at : -1;
}
// The slot that is at a row, -1: none.
__device__ inline int slot_at(const RowsParams& p, int64_t row) {
  const int64_t slot = p.source[row];
  return slot >= 0 && slot < p.slots && p.place[slot] == row ? (int)slot : -1;
}

// A wave copies one span of a token's row to its places.  Rows without a slot belong
// to the wave of the slot that has their number.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kBlock) void to_kernel(RowsParams p) {
  using S = Span<T, kDeepTo>;
  const int task = wave_number(), lane = (int)threadIdx.x & 63;
  const int64_t token = task / p.pieces;
  const int first = task % p.pieces * S::kWidth;
  if (token >= p.tokens) return;
  S x, none;
  x.load(static_cast<const T*>(p.in) + token * p.width, first, p.width);
  none.clear();
  T* rows = static_cast<T*>(p.out);
  for (int j0 = 0; j0 < p.top_k; j0 += 64) {
    const int64_t slot0 = token * p.top_k + j0;  // lane j has choice j0 + j
    const int n = p.top_k - j0 < 64 ? p.top_k - j0 : 64;
    int place = -1;
    bool empty = false;
    if (lane < n) {
      place = place_of(p, slot0 + lane);
      empty = slot_at(p, slot0 + lane) < 0;
    }
    const unsigned long long clear = __ballot(empty);
    for (int j = 0; j < n; ++j) {
      const int at = __builtin_amdgcn_readlane(place, j);
      if (at >= 0) x.template store<STREAM>(rows + (int64_t)at * p.width, first, p.width);
      if (clear >> j & 1) none.template store<STREAM>(rows + (slot0 + j) * p.width, first, p.width);
    }
  }
}

// A wave adds up one span of a token's rows.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kBlock) void from_kernel(RowsParams p) {
  using S = Span<T, kDeepFrom>;
  const int task = wave_number(), lane = (int)threadIdx.x & 63;
  const int64_t token = task / p.pieces;
  const int first = task % p.pieces * S::kWidth;
  if (token >= p.tokens) return;
  const T* rows = static_cast<const T*>(p.in);
  float sum[kDeepFrom][S::V];
#pragma unroll
  for (int u = 0; u < kDeepFrom; ++u)
#pragma unroll
    for (int e = 0; e < S::V; ++e) sum[u][e] = 0.f;
  for (int j0 = 0; j0 < p.top_k; j0 += 64) {
    const int64_t slot = token * p.top_k + j0 + lane;  // lane j has choice j0 + j
    int place = -1;
    float weight = 1.f;
    if (j0 + lane < p.top_k) {
      place = place_of(p, slot);
      if (p.weights) weight = p.weights[slot];
    }
    for (unsigned long long left = __ballot(place >= 0); left;) {
      S x[kAtOnce];
      int from[kAtOnce], n = 0;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        from[i] = 0;
        if (!left) continue;
        from[i] = __builtin_ctzll(left);
        left &= left - 1;
        n = i + 1;
        x[i].load(rows + (int64_t)__builtin_amdgcn_readlane(place, from[i]) * p.width, first, p.width);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (i >= n) continue;
        const float w = lane_value(weight, from[i]);
#pragma unroll
        for (int u = 0; u < kDeepFrom; ++u)
#pragma unroll
          for (int e = 0; e < S::V; ++e) sum[u][e] = fmaf(w, x[i].x[u][e], sum[u][e]);
      }
    }
  }
  S out;
#pragma unroll
  for (int u = 0; u < kDeepFrom; ++u) out.x[u].set(sum[u]);
  out.template store<STREAM>(static_cast<T*>(p.out) + token * p.width, first, p.width);
}

// A wave takes a slot: its row's gradient and its weight's.
template <typename T, bool ROWS, bool WEIGHTS, bool STREAM>
__global__ __launch_bounds__(kBlock) void from_backward_kernel(RowsParams p) {
  using S = Span<T, kDeepBack>;
  const int64_t slot = wave_number();
  if (slot >= p.slots) return;
  const T* grad = static_cast<const T*>(p.grad) + (int64_t)((int)slot / p.top_k) * p.width;
  const int64_t at = place_of(p, slot);
  const bool empty = ROWS && slot_at(p, slot) < 0;
  const float w = p.weights ? p.weights[slot] : 1.f;
  float dot = 0.f;
  for (int first = 0; first < p.width; first += S::kWidth) {
    S x;
    x.load(grad, first, p.width);
    if (at >= 0) {
      if (WEIGHTS) {
        S y;
        y.load(static_cast<const T*>(p.in) + at * p.width, first, p.width);
        float more = 0.f;
#pragma unroll
        for (int u = 0; u < kDeepBack; ++u)
#pragma unroll
          for (int e = 0; e < S::V; ++e) more = fmaf(x.x[u][e], y.x[u][e], more);
        dot += more;
      }
      if (ROWS) {
#pragma unroll
        for (int u = 0; u < kDeepBack; ++u) {
          float d[S::V];
#pragma unroll
          for (int e = 0; e < S::V; ++e) d[e] = w * x.x[u][e];
          x.x[u].set(d);
        }
        x.template store<STREAM>(static_cast<T*>(p.out) + at * p.width, first, p.width);
      }
    }
    if (empty) {
      x.clear();
      x.template store<STREAM>(static_cast<T*>(p.out) + slot * p.width, first, p.width);
    }
  }
  if (WEIGHTS) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
    if ((threadIdx.x & 63) == 0) p.d_weights[slot] = dot;
  }
}

// Narrow rows: of at most 64 pieces, so that a wave takes several slots or tokens at
// once, L lanes each, and kMany in turn, whose loads are on the way together (34933 x 7 rows
// of 128 in bfloat16, to, from and back: 21, 19 and 36 us; 52, 39 and 195 with a wave a row).
struct Narrow {
  int lanes, per_wave, first;  // L, units a wave takes at once, the lane's first unit
  int at, left;                // the lane's first element, and how many of its piece exist

  __device__ explicit Narrow(const RowsParams& p, int vector) {
    const int lane = (int)threadIdx.x & 63;
    lanes = 1 << p.lanes_log2;
    per_wave = 64 >> p.lanes_log2;
    first = wave_number() * per_wave * kMany + (lane >> p.lanes_log2);
    at = (lane & (lanes - 1)) * vector;
    left = p.width - at;
  }
  __device__ int unit(int i) const { return first + i * per_wave; }

  template <typename T>
  __device__ void load(Piece<T>& x, const T* row) const {
    if (left >= kV<T>)
      x.load(row + at);
    else
      x.load_some(row + at, left, (T)0.f);
  }
  template <bool STREAM, typename T>
  __device__ void store(const Piece<T>& x, T* row) const {
    if (left >= kV<T>)
      x.template store<STREAM>(row + at);
    else
      x.store_some(row + at, left);
  }
};

// L lanes fill a row: a token's row is read for each of its slots, from the caches, but
// rows are written in their order (65536 x 4 rows of 256 in bfloat16: 46 us; 60 by slots.
// Wide rows are better read once: 16384 x 4 of 4096 112 us by tokens, 153 by rows).
template <typename T, bool STREAM>
__global__ __launch_bounds__(kBlock) void to_narrow_kernel(RowsParams p) {
  const Narrow n(p, kV<T>);
  Piece<T> x[kMany];
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    const int row = n.unit(i), slot = row < p.slots ? slot_at(p, row) : -1;
    x[i].fill((T)0.f);
    if (slot >= 0) n.load(x[i], static_cast<const T*>(p.in) + (int64_t)(slot / p.top_k) * p.width);
  }
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    const int row = n.unit(i);
    if (row < p.slots) n.store<STREAM>(x[i], static_cast<T*>(p.out) + (int64_t)row * p.width);
  }
}

// L lanes add up a token's rows, kAtOnce of them on the way.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kBlock) void from_narrow_kernel(RowsParams p) {
  const Narrow n(p, kV<T>);
  const T* rows = static_cast<const T*>(p.in);
  const int lane = (int)threadIdx.x & 63;
  const int token = wave_number() * n.per_wave + (lane >> p.lanes_log2);
  if (token >= p.tokens) return;
  float sum[kV<T>];
#pragma unroll
  for (int e = 0; e < kV<T>; ++e) sum[e] = 0.f;
  for (int j0 = 0; j0 < p.top_k; j0 += kAtOnce) {
    Piece<T> x[kAtOnce];
    float w[kAtOnce];
    bool on[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t slot = (int64_t)token * p.top_k + j0 + i;
      const int at = j0 + i < p.top_k ? place_of(p, slot) : -1;
      on[i] = at >= 0;
      if (!on[i]) continue;
      w[i] = p.weights ? p.weights[slot] : 1.f;
      n.load(x[i], rows + (int64_t)at * p.width);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (!on[i]) continue;
#pragma unroll
      for (int e = 0; e < kV<T>; ++e) sum[e] = fmaf(w[i], x[i][e], sum[e]);
    }
  }
  Piece<T> out;
  out.set(sum);
  n.store<STREAM>(out, static_cast<T*>(p.out) + (int64_t)token * p.width);
}

// L lanes take a slot's row and weight.
template <typename T, bool ROWS, bool WEIGHTS, bool STREAM>
__global__ __launch_bounds__(kBlock) void from_backward_narrow_kernel(RowsParams p) {
  constexpr int V = kV<T>;
  const Narrow n(p, V);
  const T* grads = static_cast<const T*>(p.grad);
  const T* in = static_cast<const T*>(p.in);
  T* rows = static_cast<T*>(p.out);
  Piece<T> x[kMany], y[kMany], none;
  none.fill((T)0.f);
  int place[kMany];
  bool empty[kMany];
  float w[kMany];
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    const int slot = n.unit(i);
    const bool in_range = slot < p.slots;
    place[i] = in_range ? place_of(p, slot) : -1;
    empty[i] = ROWS && in_range && slot_at(p, slot) < 0;
    w[i] = ROWS && in_range && p.weights ? p.weights[slot] : 1.f;
    x[i].fill((T)0.f);
    y[i].fill((T)0.f);
    if (place[i] >= 0) {
      n.load(x[i], grads + (int64_t)(slot / p.top_k) * p.width);
      if (WEIGHTS) n.load(y[i], in + (int64_t)place[i] * p.width);
    }
  }
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    if (WEIGHTS) {
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) dot = fmaf(x[i][e], y[i][e], dot);
      for (int d = 1; d < n.lanes; d *= 2) dot += __shfl_xor(dot, d);
      if (n.at == 0 && n.unit(i) < p.slots) p.d_weights[n.unit(i)] = dot;
    }
    if (ROWS) {
      if (place[i] >= 0) {
        float d[V];
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = w[i] * x[i][e];
        x[i].set(d);
        n.store<STREAM>(x[i], rows + (int64_t)place[i] * p.width);
      }
      if (empty[i]) n.store<STREAM>(none, rows + (int64_t)n.unit(i) * p.width);
    }
  }
}

}  // namespace experts
}  // namespace ace
