// The balance loss of an expert router, with the experts' token counts, and its
// gradient (ace_balance_forward / ace_balance_backward, declared in
// include/ace_hip.h).  For each group (a layer, or a sequence) of M counted
// tokens with scores l [tokens, E], of which each token takes the k largest:
//
//   p_t = softmax(l_t),  n_e = tokens that take e,  q_e = E n_e / (k M^2)
//   loss = sum_e q_e sum_t p_te,      dl_te = u p_te (q_e - sum_j q_j p_tj)
//
// Both directions are one pass over the scores.  The backward is bound by it (131072
// tokens of 256 experts in float32: 45 us for 268 MB, 6 TB/s).  The forward (69 us for
// 134 MB, top 8; 23 us for 32 x 4096 x 64 in bfloat16, top 6; 27 us for 16 x 8191 x 100, top
// 1) waits: its vector units work for a half, a third and two fifths of that time, and
// its waves stand still for half of theirs, for their first scores (a wave has two
// to four rounds of them in the smaller two) and for the blocks' joins, two or three one
// after another.  L lanes share a token, each holding C = 8 (up to 8 experts) or 16 scores
// in registers as interleaved 16-byte pieces.  With 32 scores a lane fewer lanes
// exchange, but half of the waves fit: 158 us instead of 69.
//
// Choosing: the k largest of a lane are a sorted list, into which a score x goes
// with one instruction an entry, list[i] = median(list[i - 1], list[i], x); L
// lists become one by exchanging them.  What comes out is the k-th largest, the
// threshold that every score is then compared with.  Scores are compared as
// unsigned keys of the same order; a 16-bit score's key holds the expert's number
// below it, so that equal scores rank by number, lowest first.  float32 has no
// room for that: where more scores equal the threshold than are left to take
// (rare), the lowest numbers among them are taken one by one.
//
// Sums: per lane over its tokens, then across lanes, waves and blocks, in an order
// that depends on the sizes alone; the last blocks to finish (tickets) add the
// others' partial sums, 32 at a time, passed device-coherently (ace_core.hpp): with
// fences, which write back whole caches, the forward took 290 us instead of 160.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ace_core.hpp"  // device-coherent accesses

namespace ace {
namespace balance {

constexpr int kFan = 32;             // partial sums that one block adds
constexpr int kMaxBlocks = kFan * kFan;  // blocks of a group
constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;

struct Params {
  const void* logits;     // [groups, tokens, experts]
  const uint8_t* mask;    // [groups, tokens] or null
  int64_t tokens;
  int groups, experts, top_k;
  int lanes_log2;         // L
  int blocks;             // per group
  int64_t per_block;      // tokens of a block
  int reduction;          // 0 mean, 1 sum, 2 none
  // forward
  unsigned long long* part;  // where groups have several blocks: [groups][blocks + fans]
                             // [experts + 1]: count << 32 | the sum of p; the last entry's
                             // count is the counted tokens
  double* part_loss;      // [groups + ceil(groups / kFan)]
  int* tickets;           // zero, left zero: [groups][fans + 1] where groups have several
                          // blocks, [ceil(groups / kFan)], [1]
  float* loss;            // one value, or [groups]
  int64_t* counts;        // [groups, experts]
  float* share;           // [groups, experts]: q
  // backward
  const float* grad;      // one value, or [groups]
  void* d_logits;
};

// The 16-byte pieces of a row of E scores that a lane holds, C scores in all.
// Piece i of lane j (of L) is chunk j + L i of V scores.  The last chunk of a
// row whose length is no multiple of V is read from the row's last V scores
// instead (no read leaves the row); those it shares with the chunk before are
// not counted twice (`fresh`).
template <typename T, int C>
struct Row {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int P = C / V;
  static_assert(C % V == 0, "whole pieces");
  int at[P];       // first expert of a piece, or -1: none
  uint32_t fresh;  // bit i: score i counts
  bool ragged;     // some lane has a piece that is partly fresh
  bool partial;    // some lane has fewer than C scores

  __device__ void init(int experts, int lane, int lanes) {
    fresh = 0;
    ragged = experts % V != 0;
    partial = lanes * C != experts;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int first = (lane + lanes * i) * V;
      at[i] = first >= experts ? -1 : first + V <= experts || experts < V ? first : experts - V;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (at[i] >= 0 && at[i] + e >= first && at[i] + e < experts) fresh |= 1u << (i * V + e);
    }
  }
  __device__ bool is_fresh(int i) const { return fresh >> i & 1; }
  __device__ int expert(int i) const { return at[i / V] + i % V; }

  __device__ void load(const T* row, int experts, T (&x)[C]) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (at[i] < 0) continue;
      if (experts >= V) {
        struct Piece {
          T v[V];
        } piece;
        __builtin_memcpy(&piece, row + at[i], 16);
#pragma unroll
        for (int e = 0; e < V; ++e) x[i * V + e] = piece.v[e];
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i * V + e] = e < experts ? row[e] : (T)-INFINITY;
      }
    }
  }
  __device__ void store(T* row, int experts, const T (&x)[C]) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (at[i] < 0) continue;
      if (experts >= V) {
        struct Piece {
          T v[V];
        } piece;
#pragma unroll
        for (int e = 0; e < V; ++e) piece.v[e] = x[i * V + e];
        __builtin_memcpy(row + at[i], &piece, 16);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < experts) row[e] = x[i * V + e];
      }
    }
  }
};

// What the lane D away among a token's lanes holds, where lanes that differ below
// D already agree: neighbours, pairs, then mirror images of 8 and of 16 lanes.
template <int D>
__device__ inline uint32_t across(uint32_t x) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16, "at most 32 lanes");
  if constexpr (D == 16) return (uint32_t)__shfl_xor((int)x, 16);
  constexpr int ctrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, ctrl, 0xf, 0xf, false);
}

// x joined over a token's lanes by `op`, in every lane.
template <typename X, typename Op>
__device__ inline X over_lanes(X x, int lanes, Op op) {
  static_assert(sizeof(X) == 4, "one register");
  const auto other = [&](auto d) {
    return __builtin_bit_cast(X, across<decltype(d)::value>(__builtin_bit_cast(uint32_t, x)));
  };
  if (lanes > 1) x = op(x, other(std::integral_constant<int, 1>{}));
  if (lanes > 2) x = op(x, other(std::integral_constant<int, 2>{}));
  if (lanes > 4) x = op(x, other(std::integral_constant<int, 4>{}));
  if (lanes > 8) x = op(x, other(std::integral_constant<int, 8>{}));
  if (lanes > 16) x = op(x, other(std::integral_constant<int, 16>{}));
  return x;
}

constexpr auto kAdd = [](auto a, auto b) { return a + b; };
constexpr auto kMin = [](auto a, auto b) { return a < b ? a : b; };
constexpr auto kFmax = [](float a, float b) { return fmaxf(a, b); };

// Unsigned, in the scores' order, -0 as 0.  NaN is somewhere: `choose` puts it
// above everything where there is one.  For 16-bit scores the upper half
// suffices.
__device__ inline uint32_t ordered(uint32_t b) {
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ inline uint32_t key_of(float x) { return ordered(__float_as_uint(x + 0.f)); }
__device__ inline uint32_t key_of(__bf16 x) { return key_of((float)x) & 0xffff0000u; }
__device__ inline uint32_t key_of(_Float16 x) {
  const _Float16 y = x + (_Float16)0.f;
  return ordered((uint32_t)__builtin_bit_cast(uint16_t, y) << 16) & 0xffff0000u;
}

__device__ inline uint32_t median(uint32_t a, uint32_t b, uint32_t c) {
  return max(min(a, b), min(max(a, b), c));  // v_med3_u32
}

// The scores' keys, and the K largest of all of a token's in order.  `nans`: some
// score of the wave may be NaN.
template <typename T, int C, int K>
__device__ inline void largest(const Row<T, C>& row, const T (&x)[C], int lanes, bool nans,
                               uint32_t (&key)[C], uint32_t (&list)[K]) {
  constexpr bool numbered = sizeof(T) == 2;
#pragma unroll
  for (int k = 0; k < K; ++k) list[k] = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    key[i] = key_of(x[i]);
    if constexpr (numbered) key[i] |= 0xffffu ^ (uint32_t)row.expert(i);
  }
  if (nans) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (x[i] != x[i]) key[i] |= 0xffff0000u | (numbered ? 0u : 0xffffu);
  }
  if (row.partial) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (!row.is_fresh(i)) key[i] = 0;  // below every score's key
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int k = K - 1; k > 0; --k) list[k] = median(list[k - 1], list[k], key[i]);
    list[0] = max(list[0], key[i]);
  }
  // the K largest of two sorted lists: the larger of each entry and the other's
  // mirror image, sorted again by halves
  const auto merge = [&](auto d) {
    uint32_t other[K];
#pragma unroll
    for (int k = 0; k < K; ++k) other[k] = across<decltype(d)::value>(list[k]);
#pragma unroll
    for (int k = 0; k < K; ++k) list[k] = max(list[k], other[K - 1 - k]);
#pragma unroll
    for (int h = K / 2; h > 0; h /= 2)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (!(k & h)) {
          const uint32_t low = min(list[k], list[k + h]);
          list[k] = max(list[k], list[k + h]);
          list[k + h] = low;
        }
  };
  if (lanes > 1) merge(std::integral_constant<int, 1>{});
  if (lanes > 2) merge(std::integral_constant<int, 2>{});
  if (lanes > 4) merge(std::integral_constant<int, 4>{});
  if (lanes > 8) merge(std::integral_constant<int, 8>{});
  if (lanes > 16) merge(std::integral_constant<int, 16>{});
}

// The scores' keys and the threshold that the k largest reach: score i is taken
// where key[i] >= the result.  `on`: the token is counted, its scores are there;
// others take nothing.
template <typename T, int C, int K>
__device__ inline uint32_t choose(const Row<T, C>& row, const T (&x)[C], int lanes, int top_k,
                                  bool on, bool nans, uint32_t (&key)[C]) {
  constexpr bool numbered = sizeof(T) == 2;
  uint32_t list[K];
  largest<T, C, K>(row, x, lanes, nans, key, list);
  uint32_t least = list[0];
#pragma unroll
  for (int k = 1; k < K; ++k) least = k < top_k ? list[k] : least;
  if constexpr (!numbered) {
    int reach = 0, above = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) reach += key[i] >= least;
    reach = over_lanes(reach, lanes, kAdd);
    const bool tied = on && reach > top_k;
    if (__ballot(tied)) {
#pragma unroll
      for (int i = 0; i < C; ++i) above += key[i] > least;
      int left = tied ? top_k - over_lanes(above, lanes, kAdd) : 0;
      uint32_t taken = 0;
      while (__ballot(left > 0)) {  // the lowest number that is left, at most k times
        int next = kMaxExperts;
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (key[i] == least && !(taken >> i & 1)) next = min(next, row.expert(i));
        next = over_lanes(next, lanes, kMin);
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (left > 0 && key[i] == least && row.expert(i) == next) taken |= 1u << i;
        --left;
      }
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (tied && key[i] == least && !(taken >> i & 1)) key[i] = 0;
    }
  }
  return on ? least : 0xffffffffu;
}

// exp(x - the token's largest score) of a lane's scores, and the reciprocal of the
// token's sum of them.  Scores that do not exist are 0; those that a last piece
// repeats have their value (their gradient is stored twice) and are not summed.
template <typename T, int C>
__device__ inline float exponentials(const Row<T, C>& row, const T (&x)[C], int lanes,
                                     float (&e)[C]) {
  constexpr int V = Row<T, C>::V;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < C; ++i) e[i] = (float)x[i];
  if (row.partial) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (row.at[i / V] < 0) e[i] = -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < C; ++i) top = fmaxf(top, e[i]);
  top = over_lanes(top, lanes, kFmax);
#pragma unroll
  for (int i = 0; i < C; ++i) e[i] = __builtin_amdgcn_exp2f((e[i] - top) * 1.4426950408889634f);
  float sum = 0.f;
  if (row.ragged) {
#pragma unroll
    for (int i = 0; i < C; ++i) sum += row.is_fresh(i) ? e[i] : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) sum += e[i];
  }
  return 1.f / over_lanes(sum, lanes, kAdd);
}

__device__ inline void store_dev(double* p, double v) {
  ace::store_dev(reinterpret_cast<long long*>(p), __double_as_longlong(v));
}
__device__ inline double load_dev(const double* p) {
  return __longlong_as_double(
      (long long)ace::load_dev(reinterpret_cast<const unsigned long long*>(p)));
}

template <typename T, int C, int K>
__global__ __launch_bounds__(kThreads, 4) void forward_kernel(Params p) {
  __shared__ float s_sum[kMaxExperts];
  __shared__ int s_count[kMaxExperts + 1];
  __shared__ double s_loss[kThreads / 64];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lanes = 1 << p.lanes_log2, j = lane & (lanes - 1);
  const int E = p.experts;
  const int group = (int)blockIdx.x / p.blocks, block = (int)blockIdx.x % p.blocks;
  const int64_t t0 = block * p.per_block;
  const int64_t t1 = t0 + p.per_block < p.tokens ? t0 + p.per_block : p.tokens;
  const int per_wave = 64 >> p.lanes_log2;  // tokens a wave takes at a time
  Row<T, C> row;
  row.init(E, j, lanes);
  float sum[C];
  int count[C], tokens = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    sum[i] = 0.f;
    count[i] = 0;
  }
  const T* logits = static_cast<const T*>(p.logits) + (int64_t)group * p.tokens * E;
  const uint8_t* mask = p.mask ? p.mask + group * p.tokens : nullptr;
  for (int64_t t = t0 + wave * per_wave; t < t1; t += kThreads / 64 * per_wave) {
    const int64_t mine = t + (lane >> p.lanes_log2);
    const bool counted = mine < t1 && (!mask || mask[mine]);
    T x[C];
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = (T)0.f;
    if (counted) row.load(logits + mine * E, E, x);
    float e[C];
    const float inv = exponentials<T, C>(row, x, lanes, e);
    const float of = counted ? inv : 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) sum[i] = fmaf(e[i], of, sum[i]);
    tokens += counted && j == 0;
    uint32_t key[C];
    const uint32_t least =
        choose<T, C, K>(row, x, lanes, p.top_k, counted, __ballot(inv != inv) != 0, key);
#pragma unroll
    for (int i = 0; i < C; ++i) count[i] += key[i] >= least;
  }
  // across the wave's tokens, then the waves in turn
  for (int d = lanes; d < 64; d *= 2) {
    tokens += __shfl_xor(tokens, d);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      sum[i] += __shfl_xor(sum[i], d);
      count[i] += __shfl_xor(count[i], d);
    }
  }
  for (int w = 0; w < kThreads / 64; ++w) {
    if (wave == w && lane < lanes) {
      if (lane == 0) s_count[E] = tokens + (w ? s_count[E] : 0);
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (row.is_fresh(i)) {
          const int e = row.expert(i);
          s_sum[e] = sum[i] + (w ? s_sum[e] : 0.f);
          s_count[e] = count[i] + (w ? s_count[e] : 0);
        }
    }
    __syncthreads();
  }
  // across the group's blocks: kFan of them, then those sums
  const int fans = (p.blocks + kFan - 1) / kFan;
  unsigned long long* part = p.part + (int64_t)group * (p.blocks + fans) * (E + 1);
  const int group_tickets = p.blocks > 1 ? fans + 1 : 0;
  int* tickets = p.tickets + (int64_t)group * group_tickets * kTicketStride;
  const auto put = [&](int at) {
    for (int e = tid; e <= E; e += kThreads)
      ace::store_dev(part + (int64_t)at * (E + 1) + e,
                     (unsigned long long)(unsigned)s_count[e] << 32 |
                         (e < E ? __float_as_uint(s_sum[e]) : 0u));
  };
  const auto add = [&](int first, int n) {
    for (int e = tid; e <= E; e += kThreads) {
      const unsigned long long* at = part + (int64_t)first * (E + 1) + e;
      float s = 0.f;
      int c = 0;
      for (int i0 = 0; i0 < n; i0 += 8) {
        unsigned long long w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = i0 + i < n ? ace::load_dev(at + (int64_t)(i0 + i) * (E + 1)) : 0ull;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s += __uint_as_float((unsigned)w[i]);
          c += (int)(w[i] >> 32);
        }
      }
      if (e < E) s_sum[e] = s;
      s_count[e] = c;
    }
    __syncthreads();
  };
  if (p.blocks > 1) {
    const int fan = block / kFan;
    const int in_fan = p.blocks - fan * kFan < kFan ? p.blocks - fan * kFan : kFan;
    put(block);
    if (!last_of(tickets + fan * kTicketStride, in_fan)) return;
    add(fan * kFan, in_fan);
    if (fans > 1) {
      put(p.blocks + fan);
      if (!last_of(tickets + fans * kTicketStride, fans)) return;
      add(p.blocks, fans);
    }
  }
  // the group's loss
  const double m = s_count[E] > 0 ? (double)s_count[E] : 1.0;
  double loss = 0.0;
  for (int e = tid; e < E; e += kThreads) {
    const double q = (double)E * (double)s_count[e] / ((double)p.top_k * m * m);
    p.counts[(int64_t)group * E + e] = s_count[e];
    p.share[(int64_t)group * E + e] = (float)q;
    loss += q * (double)s_sum[e];
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) loss += __shfl_xor(loss, d);
  if (lane == 0) s_loss[wave] = loss;
  __syncthreads();
  loss = s_loss[0] + s_loss[1] + s_loss[2] + s_loss[3];
  if (p.reduction == 2 || p.groups == 1) {
    if (tid == 0) p.loss[group] = (float)loss;
    return;
  }
  // across the groups: kFan of them, then those sums
  const int sets = (p.groups + kFan - 1) / kFan, set = group / kFan;
  const int in_set = p.groups - set * kFan < kFan ? p.groups - set * kFan : kFan;
  int* loss_tickets = p.tickets + (int64_t)p.groups * group_tickets * kTicketStride;
  const auto sum_of = [&](const double* x, int n) {  // by the first wave
    double all = 0.0;
    for (int g = lane; g < n; g += 64) all += load_dev(x + g);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
    return all;
  };
  if (tid == 0) store_dev(p.part_loss + group, loss);
  if (!last_of(loss_tickets + set * kTicketStride, in_set)) return;
  double all = wave == 0 ? sum_of(p.part_loss + set * kFan, in_set) : 0.0;
  if (sets > 1) {
    if (tid == 0) store_dev(p.part_loss + p.groups + set, all);
    if (!last_of(loss_tickets + sets * kTicketStride, sets)) return;
    if (wave == 0) all = sum_of(p.part_loss + p.groups, sets);
  }
  if (tid == 0) *p.loss = (float)(p.reduction == 0 ? all / p.groups : all);
}

template <typename T, int C>
__global__ __launch_bounds__(kThreads, 4) void backward_kernel(Params p) {
  constexpr int V = Row<T, C>::V;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lanes = 1 << p.lanes_log2, j = lane & (lanes - 1);
  const int E = p.experts;
  const int group = (int)blockIdx.x / p.blocks, block = (int)blockIdx.x % p.blocks;
  const int64_t t0 = block * p.per_block;
  const int64_t t1 = t0 + p.per_block < p.tokens ? t0 + p.per_block : p.tokens;
  const int per_wave = 64 >> p.lanes_log2;
  Row<T, C> row;
  row.init(E, j, lanes);
  const float up = p.reduction == 2 ? p.grad[group]
                                    : p.grad[0] * (p.reduction == 0 ? 1.f / (float)p.groups : 1.f);
  float q[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int e = row.expert(i);
    q[i] = row.at[i / V] >= 0 && e < E ? p.share[(int64_t)group * E + e] : 0.f;
  }
  const int64_t base = (int64_t)group * p.tokens * E;
  const T* logits = static_cast<const T*>(p.logits) + base;
  T* out = static_cast<T*>(p.d_logits) + base;
  const uint8_t* mask = p.mask ? p.mask + group * p.tokens : nullptr;
  for (int64_t t = t0 + wave * per_wave; t < t1; t += kThreads / 64 * per_wave) {
    const int64_t mine = t + (lane >> p.lanes_log2);
    const bool in = mine < t1, counted = in && (!mask || mask[mine]);
    T x[C];
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = (T)0.f;
    if (counted) row.load(logits + mine * E, E, x);
    float e[C];
    const float inv = exponentials<T, C>(row, x, lanes, e);
    float pull = 0.f;
    if (row.ragged) {
#pragma unroll
      for (int i = 0; i < C; ++i) pull = fmaf(row.is_fresh(i) ? q[i] : 0.f, e[i], pull);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) pull = fmaf(q[i], e[i], pull);
    }
    pull = over_lanes(pull, lanes, kAdd) * inv;
    const float of = up * inv;
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = counted ? (T)(e[i] * (q[i] - pull) * of) : (T)0.f;
    if (in) row.store(out + mine * E, E, x);
  }
}

}  // namespace balance
}  // namespace ace
