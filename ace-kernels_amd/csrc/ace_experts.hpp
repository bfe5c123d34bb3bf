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
// Rows behind the last routed one are 0 where they are written, and not read.
// Everything is a copy's work: bytes of rows at the rate of memory.
//
// Sums over a token's rows and over a row's width are float32, in an order that the
// sizes alone decide; no atomic's order reaches a result (the order's counts are
// integers).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ace_core.hpp"  // wave_sync

namespace ace {
namespace experts {

constexpr int kMaxExperts = 512;
constexpr int kBlock = 256, kWaves = kBlock / 64;
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
__global__ __launch_bounds__(kBlock) void count_kernel(OrderParams p) {
  __shared__ int s_count[kMaxExperts];
  const int tid = (int)threadIdx.x;
  for (int e = tid; e < p.experts; e += kBlock) s_count[e] = 0;
  __syncthreads();
  const int64_t s0 = blockIdx.x * p.per_block;
  const int64_t s1 = s0 + p.per_block < p.slots ? s0 + p.per_block : p.slots;
  for (int64_t s = s0 + tid; s < s1; s += kBlock) {
    const int e = choice(p, s, s1);
    if (e >= 0) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  for (int e = tid; e < p.experts; e += kBlock)
    p.counts[(int64_t)blockIdx.x * p.experts + e] = s_count[e];
}

// The slots' places.  Each wave has a run of the block's slots, and for each expert
// the place that its next slot takes; among 64 slots, those of one expert are found by
// ballots over the bits of its number.
__global__ __launch_bounds__(kBlock) void place_kernel(OrderParams p) {
  __shared__ int s_next[kWaves][kMaxExperts];
  __shared__ int s_sum[kWaves];
  __shared__ int64_t s_total;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t per_wave = p.per_block / kWaves;
  const int64_t s0 = blockIdx.x * p.per_block + wave * per_wave;
  const int64_t s1 = s0 + per_wave < p.slots ? s0 + per_wave : p.slots;
  for (int i = tid; i < kWaves * kMaxExperts; i += kBlock) (&s_next[0][0])[i] = 0;
  __syncthreads();
  for (int64_t s = s0 + lane; s < s1; s += 64) {
    const int e = choice(p, s, s1);
    if (e >= 0) atomicAdd(&s_next[wave][e], 1);
  }
  __syncthreads();
  // thread t has experts 2 t and 2 t + 1
  static_assert(2 * kBlock == kMaxExperts, "all experts have a thread");
  int before[2], all[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * tid + i;
    before[i] = all[i] = 0;
    if (e >= p.experts) continue;
    if (p.blocks > 1) {
      for (int b = 0; b < p.blocks; ++b) {
        const int n = p.counts[(int64_t)b * p.experts + e];
        all[i] += n;
        if (b < (int)blockIdx.x) before[i] += n;
      }
    } else {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all[i] += s_next[w][e];
    }
  }
  int upto = all[0] + all[1];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  int start = upto - all[0] - all[1];
  for (int w = 0; w < wave; ++w) start += s_sum[w];
  if (tid == kBlock - 1) s_total = start + all[0] + all[1];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * tid + i;
    if (e < p.experts) {
      if (blockIdx.x == 0) {
        if (e == 0) p.offsets[0] = 0;
        p.offsets[e + 1] = start + all[i];
      }
      int next = start + before[i];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int n = s_next[w][e];
        s_next[w][e] = next;
        next += n;
      }
    }
    start += all[i];
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
  for (int64_t s = s_total + (int64_t)blockIdx.x * kBlock + tid; s < p.slots;
       s += (int64_t)p.blocks * kBlock)
    p.source[s] = -1;
}

// --------------------------------------------------------------------- rows

struct RowsParams {
  const void* in;         // to: x [tokens, width]; from: rows [slots, width]
  const void* grad;       // from's backward: dout [tokens, width]
  void* out;              // to: rows; from: out; from's backward: drows
  const int64_t* place;   // [slots]
  const int64_t* offsets; // the last of them: routed slots
  const float* weights;   // [slots] or null: 1
  float* d_weights;       // [slots]
  int64_t tokens, slots;
  int width, top_k;
  int pieces;             // of a row that waves share
};

template <typename T>
constexpr int kV = 16 / (int)sizeof(T);
constexpr int kDeep = 4;  // pieces of 16 bytes a lane holds
template <typename T>
constexpr int kSpan = 64 * kDeep * kV<T>;  // elements of a row that a wave takes at once

// A wave's span of a row from element `first` on; what is behind the row's end
// reads as 0 and is not written.
template <typename T>
__device__ inline void load_span(const T* row, int first, int width, T (&x)[kDeep][kV<T>]) {
  constexpr int V = kV<T>;
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < kDeep; ++u) {
    const int at = first + (u * 64 + lane) * V;
    if (at + V <= width) {
      __builtin_memcpy(x[u], row + at, 16);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x[u][e] = at + e < width ? row[at + e] : (T)0.f;
    }
  }
}
template <typename T>
__device__ inline void store_span(T* row, int first, int width, const T (&x)[kDeep][kV<T>]) {
  constexpr int V = kV<T>;
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < kDeep; ++u) {
    const int at = first + (u * 64 + lane) * V;
    if (at + V <= width) {
      __builtin_memcpy(row + at, x[u], 16);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (at + e < width) row[at + e] = x[u][e];
    }
  }
}

// The same for the whole wave, in a scalar register.
__device__ inline int wave_number() {
  return __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kWaves + threadIdx.x / 64));
}
// A slot's place, -1: none (or none that exists).
__device__ inline int64_t place_of(const RowsParams& p, int64_t slot) {
  const int64_t at = p.place[slot];
  return at >= 0 && at < p.slots ? at : -1;
}

// A wave copies one span of a token's row to its places.  Of the rows behind the
// last, each belongs to the wave of the slot with its number.
template <typename T>
__global__ __launch_bounds__(kBlock) void to_kernel(RowsParams p) {
  const int task = wave_number();
  const int64_t token = task / p.pieces;
  const int first = task % p.pieces * kSpan<T>;
  if (token >= p.tokens) return;
  T x[kDeep][kV<T>], none[kDeep][kV<T>];
  load_span<T>(static_cast<const T*>(p.in) + token * p.width, first, p.width, x);
#pragma unroll
  for (int u = 0; u < kDeep; ++u)
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) none[u][e] = (T)0.f;
  T* rows = static_cast<T*>(p.out);
  const int64_t routed = *p.offsets;
  for (int j = 0; j < p.top_k; ++j) {
    const int64_t slot = token * p.top_k + j, at = place_of(p, slot);
    if (at >= 0) store_span<T>(rows + at * p.width, first, p.width, x);
    if (slot >= routed) store_span<T>(rows + slot * p.width, first, p.width, none);
  }
}

// A wave adds up one span of a token's rows.
template <typename T>
__global__ __launch_bounds__(kBlock) void from_kernel(RowsParams p) {
  const int task = wave_number();
  const int64_t token = task / p.pieces;
  const int first = task % p.pieces * kSpan<T>;
  if (token >= p.tokens) return;
  const T* rows = static_cast<const T*>(p.in);
  float sum[kDeep][kV<T>];
#pragma unroll
  for (int u = 0; u < kDeep; ++u)
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) sum[u][e] = 0.f;
  for (int j = 0; j < p.top_k; ++j) {
    const int64_t slot = token * p.top_k + j, at = place_of(p, slot);
    if (at < 0) continue;
    const float w = p.weights ? p.weights[slot] : 1.f;
    T x[kDeep][kV<T>];
    load_span<T>(rows + at * p.width, first, p.width, x);
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
#pragma unroll
      for (int e = 0; e < kV<T>; ++e) sum[u][e] = fmaf(w, (float)x[u][e], sum[u][e]);
  }
  T out[kDeep][kV<T>];
#pragma unroll
  for (int u = 0; u < kDeep; ++u)
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) out[u][e] = (T)sum[u][e];
  store_span<T>(static_cast<T*>(p.out) + token * p.width, first, p.width, out);
}

// A wave takes a slot: its row's gradient and its weight's.
template <typename T, bool ROWS, bool WEIGHTS>
__global__ __launch_bounds__(kBlock) void from_backward_kernel(RowsParams p) {
  const int64_t slot = wave_number();
  if (slot >= p.slots) return;
  const int64_t at = place_of(p, slot), routed = *p.offsets;
  const T* grad = static_cast<const T*>(p.grad) + slot / p.top_k * p.width;
  const float w = p.weights ? p.weights[slot] : 1.f;
  float dot = 0.f;
  T x[kDeep][kV<T>], y[kDeep][kV<T>];
  for (int first = 0; first < p.width; first += kSpan<T>) {
    if (at >= 0) {
      load_span<T>(grad, first, p.width, x);
      if (WEIGHTS) {
        load_span<T>(static_cast<const T*>(p.in) + at * p.width, first, p.width, y);
        float more = 0.f;
#pragma unroll
        for (int u = 0; u < kDeep; ++u)
#pragma unroll
          for (int e = 0; e < kV<T>; ++e) more = fmaf((float)x[u][e], (float)y[u][e], more);
        dot += more;
      }
      if (ROWS) {
#pragma unroll
        for (int u = 0; u < kDeep; ++u)
#pragma unroll
          for (int e = 0; e < kV<T>; ++e) x[u][e] = (T)(w * (float)x[u][e]);
        store_span<T>(static_cast<T*>(p.out) + at * p.width, first, p.width, x);
      }
    }
    if (ROWS && slot >= routed) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u)
#pragma unroll
        for (int e = 0; e < kV<T>; ++e) x[u][e] = (T)0.f;
      store_span<T>(static_cast<T*>(p.out) + slot * p.width, first, p.width, x);
    }
  }
  if (WEIGHTS) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
    if ((threadIdx.x & 63) == 0) p.d_weights[slot] = dot;
  }
}

}  // namespace experts
}  // namespace ace
