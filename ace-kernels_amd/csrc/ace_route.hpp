// A router's choice of experts with their weights, and the gradient
// (ace_route_forward / ace_route_backward, declared in include/ace_hip.h).  For a
// token with scores x [experts], of which it takes the k largest, c_1 .. c_k in order:
//
//   p = softmax(x),   w_r = p_c_r              or, normalised, p_c_r / sum_s p_c_s
//   dx_e = [e = c_r] w_r g_r - p_e sum_s w_s g_s              (normalised: p is w)
//
// As in the balance loss (ace_balance.hpp), whose choice this is: L lanes share a
// token, each holds C of its scores in registers, and the k largest are a sorted
// list that lanes merge by exchanges.  A 16-bit score's key holds its expert, so the
// list is the answer; in float32 the lanes that hold the taken scores say which they
// are.  Normalised weights need the chosen scores only, and their gradient no score.
//
// What bounds it (131072 x 256, top 8, in a trace): the forward of many experts its
// instructions, 59 us for 147 MB in float32 and 41 for 80 in bfloat16 (normalised 54 and
// 35).  A float32 token's lists are about 275 vector instructions; some 370 stand before
// the loop, for two trips of it, 142 of them spills of scalars that say which score a lane
// has, which the trips read back.  The backward memory: 53 us for 285 MB, 5.4 TB/s
// (normalised 37 us for 151).  Where a token has at least as many lanes as choices, each lane writes one of
// them: with every lane writing its share of all, the forward took 65 us.
#pragma once

#include "ace_balance.hpp"

namespace ace {
namespace route {

using balance::kAdd;
using balance::kMin;
using balance::over_lanes;
using balance::Row;

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void* logits;   // [tokens, experts]
  const uint8_t* mask;  // [tokens] or null
  int64_t tokens;
  int experts, top_k;
  int lanes_log2;       // L
  int64_t per_block;    // tokens of a block
  int normalize;
  int64_t* chosen;      // [tokens, top_k]
  float* weights;       // [tokens, top_k]
  // backward
  const float* grad;    // [tokens, top_k]
  void* d_logits;
};

// The score of a key.
__device__ inline float score_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
template <typename T>
__device__ inline float key_score(uint32_t key) {
  if constexpr (sizeof(T) == 4) return key == 0xffffffffu ? NAN : score_of(key);
  if (key >= 0xffff0000u) return NAN;
  // a 16-bit score is the upper half (of a negative key the lower half's complement is 0)
  const uint32_t b = key & 0x80000000u ? (key & 0xffff0000u) ^ 0x80000000u : ~(key | 0xffffu);
  if constexpr (std::is_same_v<T, __bf16>)
    return __uint_as_float(b);
  else
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(b >> 16));
}

template <typename T, int C, int K>
__global__ __launch_bounds__(kThreads, K <= 8 ? 5 : 4) void forward_kernel(Params p) {
  constexpr bool numbered = sizeof(T) == 2;
  __shared__ int s_expert[numbered ? 1 : kThreads];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lanes = 1 << p.lanes_log2, j = lane & (lanes - 1);
  const int E = p.experts;
  const int64_t t0 = blockIdx.x * p.per_block;
  const int64_t t1 = t0 + p.per_block < p.tokens ? t0 + p.per_block : p.tokens;
  const int per_wave = 64 >> p.lanes_log2;
  Row<T, C> row;
  row.init(E, j, lanes);
  const T* logits = static_cast<const T*>(p.logits);
  for (int64_t t = t0 + wave * per_wave; t < t1; t += kThreads / 64 * per_wave) {
    const int64_t mine = t + (lane >> p.lanes_log2);
    const bool in = mine < t1, counted = in && (!p.mask || p.mask[mine]);
    T x[C];
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = (T)0.f;
    if (counted) row.load(logits + mine * E, E, x);
    bool nan = false;
#pragma unroll
    for (int i = 0; i < C; ++i) nan |= x[i] != x[i];
    float by = 0.f;
    if (!p.normalize) {
      float e[C];
      by = balance::exponentials<T, C>(row, x, lanes, e);
    }
    uint32_t key[C], list[K];
    balance::largest<T, C, K>(row, x, lanes, __ballot(nan) != 0, key, list);
    const float top = key_score<T>(list[0]);
    const bool dead = top == -INFINITY;  // every expert is closed
    const auto raw = [&](uint32_t k) {
      return __builtin_amdgcn_exp2f((key_score<T>(k) - top) * kLog2e);
    };
    int64_t* chosen = p.chosen + mine * p.top_k;
    float* weights = p.weights + mine * p.top_k;
    // float32's keys have no numbers: the place of each score that is taken.  Equal
    // scores among them, or beyond the last, are seldom, and looked for one by one.
    bool tied = false;
    uint32_t taken = 0;
    if constexpr (!numbered) {
      uint32_t least = list[0];
#pragma unroll
      for (int r = 1; r < K; ++r) {
        tied |= r < p.top_k && list[r] == list[r - 1];
        least = r < p.top_k ? list[r] : least;
      }
#pragma unroll
      for (int i = 0; i < C; ++i) taken |= key[i] >= least ? 1u << i : 0u;
      if (!counted) taken = 0;
      tied |= over_lanes(__popc(taken), lanes, kAdd) > p.top_k;
    }
    if (lanes >= K && !__ballot(tied && counted)) {  // lane r writes the r-th
      uint32_t own = list[0];
#pragma unroll
      for (int r = 1; r < K; ++r) own = j == r ? list[r] : own;
      int expert = (int)(0xffffu ^ (own & 0xffffu));
      if constexpr (!numbered) {
        int* place_of = s_expert + wave * 64 + (lane & ~(lanes - 1));
        wave_sync();
        while (__ballot(taken != 0)) {
          const int at = __builtin_ctz(taken | 1u << (C - 1));
          uint32_t k = key[0];
          int e = row.expert(0), place = 0;
#pragma unroll
          for (int i = 1; i < C; ++i) {
            k = at == i ? key[i] : k;
            e = at == i ? row.expert(i) : e;
          }
#pragma unroll
          for (int r = 0; r < K; ++r) place += list[r] > k;
          if (taken) place_of[place] = e;
          taken &= taken - 1;
        }
        wave_sync();
        expert = place_of[j];
      }
      float weight = j < p.top_k && !dead ? raw(own) : 0.f;
      if (p.normalize) by = 1.f / over_lanes(weight, lanes, kAdd);
      if (in && j < p.top_k) {
        chosen[j] = counted ? expert : -1;
        weights[j] = counted && !dead ? weight * by : 0.f;
      }
      continue;
    }
    float weight[K], total = 0.f;
#pragma unroll
    for (int r = 0; r < K; ++r) {
      weight[r] = r < p.top_k && !dead ? raw(list[r]) : 0.f;
      total += weight[r];
    }
    if (p.normalize) by = 1.f / total;
    int last = -1;
#pragma unroll
    for (int r = 0; r < K; ++r) {
      int expert = (int)(0xffffu ^ (list[r] & 0xffffu));
      if (!numbered && r < p.top_k) {  // the lowest that no place before has
        if (r > 0 && list[r] != list[r > 0 ? r - 1 : 0]) last = -1;
        int next = balance::kMaxExperts;
#pragma unroll
        for (int i = C - 1; i >= 0; --i)
          if (key[i] == list[r] && row.expert(i) > last) next = row.expert(i);
        expert = last = over_lanes(next, lanes, kMin);
      }
      if (in && r < p.top_k && (r & (lanes - 1)) == j) {
        chosen[r] = counted ? expert : -1;
        weights[r] = counted && !dead ? weight[r] * by : 0.f;
      }
    }
  }
}

// The chosen experts' terms go through LDS, a row of scores a token that is 0 in
// between: looking for them among each lane's scores takes 16 x top_k comparisons, and
// loads that wait for each other (131072 x 256, top 8, normalised: 56 us instead of 37).
template <typename T, int C>
__global__ __launch_bounds__(kThreads, 4) void backward_kernel(Params p) {
  constexpr int V = Row<T, C>::V;
  __shared__ float s_rows[kThreads / 64][64 * C];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lanes = 1 << p.lanes_log2, j = lane & (lanes - 1);
  const int E = p.experts;
  const int64_t t0 = blockIdx.x * p.per_block;
  const int64_t t1 = t0 + p.per_block < p.tokens ? t0 + p.per_block : p.tokens;
  const int per_wave = 64 >> p.lanes_log2;
  Row<T, C> row;
  row.init(E, j, lanes);
  const T* logits = static_cast<const T*>(p.logits);
  T* out = static_cast<T*>(p.d_logits);
  float* own = s_rows[wave] + (lane >> p.lanes_log2) * E;  // a token's row
#pragma unroll
  for (int i = 0; i < C; ++i) s_rows[wave][i * 64 + lane] = 0.f;
  for (int64_t t = t0 + wave * per_wave; t < t1; t += kThreads / 64 * per_wave) {
    const int64_t mine = t + (lane >> p.lanes_log2);
    const bool in = mine < t1;
    // lane j has the choices j, j + L, ...
    float pull = 0.f, total = 0.f;
    for (int r = j; in && r < p.top_k; r += lanes) {
      const float w = p.weights[mine * p.top_k + r];
      pull = fmaf(w, p.grad[mine * p.top_k + r], pull);
      total += w;
    }
    T x[C];
    float d[C];
    bool on = in && p.chosen[mine * p.top_k] >= 0;
    if (!p.normalize) {
#pragma unroll
      for (int i = 0; i < C; ++i) x[i] = (T)0.f;
      if (on) row.load(logits + mine * E, E, x);
    }
    pull = over_lanes(pull, lanes, kAdd);
    total = over_lanes(total, lanes, kAdd);
    // a token that is masked, or whose experts are all closed, has weights of 0
    on = on && total != 0.f;
    const auto choices = [&](auto term) {
      wave_sync();
      for (int r = j; on && r < p.top_k; r += lanes) {
        const int expert = (int)p.chosen[mine * p.top_k + r];
        const float w = p.weights[mine * p.top_k + r], g = p.grad[mine * p.top_k + r];
        if (expert >= 0 && expert < E) own[expert] = term(w * (p.normalize ? g - pull : g));
      }
      wave_sync();
    };
    choices([](float x) { return x; });
    if (!p.normalize) {
      const float inv = balance::exponentials<T, C>(row, x, lanes, d);
#pragma unroll
      for (int i = 0; i < C; ++i) d[i] *= -inv * pull;
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) d[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      // scores that do not exist read others': fewer than V scores are the first of a row,
      // all others a piece within it
      d[i] += own[(row.at[i / V] >= 0 ? row.at[i / V] : 0) + i % V];
      x[i] = on ? (T)d[i] : (T)0.f;
    }
    choices([](float) { return 0.f; });
    if (in) row.store(out + mine * E, E, x);
  }
}

}  // namespace route
}  // namespace ace
