// Log probabilities of given tokens from logits, with the entropy and the largest
// alternatives, and their gradient (ace_logprob_forward / ace_logprob_backward,
// declared in include/ace_hip.h).  For a row x of V logits, temperature t, token y:
//
//   z_v = (x_v - max x) / t,   l = log sum_v exp z_v,   lp_v = z_v - l,   p_v = exp lp_v
//   logprob = lp_y,            H = -sum_v p_v lp_v = l - sum_v p_v z_v
//   dx_v = -p_v (g + h (lp_v + H)) / t,   dx_y = (g (1 - p_y) - p_y h (lp_y + H)) / t
//
// with g and h the upstream gradients of logprob and H.  Both directions are one
// pass over the logits.
//
// Forward: a team of one wave (short rows) or four reads a row, or a part of one
// where there are few rows.  Each lane keeps a running maximum, sum of exp z and sum
// of z exp z; these are joined across lanes, waves and, through the workspace, the
// row's parts, by the part that ends last.  The largest word's e^0 is in the sum, and
// where it is most of it (a word that is all but certain) l is what the others add to that
// 1.  So groups, lanes and parts are added in float64, and where a wave's sum is below 2,
// so that one word has its 1 alone, the words that its lane had added to it in float32 are
// read once more, by a lane each, and added up without it.  (With float32 throughout, what
// words below 2^-25 of the largest add was lost in its lane: log probabilities near 0 of a
// row of 131072 were off by 6e-6 of themselves, now 2e-7.)
//
// Alternatives: a key is a logit's bits in their order above the complement of its
// number, so keys differ and equal logits rank by number, lowest first.  The k
// largest words are among the k pieces (16 bytes of words) with the largest maxima:
// each piece before a word's own has a word before it.  The maxima are there anyway, so
// pieces are what is looked for.  The k-th largest of the lanes' maxima over the
// team's first words bounds the k-th largest from below; pieces that reach it are
// kept as candidates, in LDS.  At the end every
// candidate counts those above it, which is its place; then the same for the words
// of the k best.  A wave whose candidates outgrow its LDS (logits in ascending
// order, say) keeps its k best and raises the bound.
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ace_balance.hpp"  // keys in the scores' order
#include "ace_core.hpp"     // device-coherent accesses
#include "ace_piece.hpp"

namespace ace {
namespace logprob {

using balance::key_of;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kBlock = 256;
constexpr int kPieces = 4;    // of 16 bytes that a lane reads at a time
constexpr int kMaxTop = 32;
constexpr int kMaxParts = 32;
constexpr int kRoom = 128;    // candidates of a wave
constexpr int kHeld = kRoom + kMaxTop;  // keys of its LDS
constexpr float kFar = 200.f;  // 2^-200 is 0 in float32: exponents beyond it count as it
template <typename T>
constexpr int kV = 16 / (int)sizeof(T);  // words of a piece
template <typename T>
constexpr int kTile = 64 * kV<T>;        // words a wave reads with one piece a lane
template <typename T>
constexpr int kGroup = kPieces * kTile<T>;

// What the backward needs of a row: 16 bytes.  label -1: not counted, or no logit
// above -inf; its gradient is 0.
struct Saved {
  float top, log_sum, entropy;
  int label;
};

struct Params {
  const void* logits;    // rows of `stride` elements
  int64_t stride;
  const int64_t* tokens;
  int64_t rows, vocab, ignore;
  float inv_t, scale;    // 1 / t, log2(e) / t
  int top;
  int parts;             // of a row
  int64_t per_part;      // words, whole tiles
  Saved* saved;
  float* logprob;
  float* entropy;
  float* top_logprobs;   // [rows, top]
  int64_t* top_tokens;
  unsigned long long* part;  // [rows][parts][2 + top]: a part's sums, and its best keys in order
  int* tickets;          // [rows], zero, left zero
  // backward
  const float* grad_logprob;
  const float* grad_entropy;
  void* d_logits;        // [rows, vocab]
  int tiles;             // groups of a row
};

// Takes NaN along.
__device__ inline float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ inline float exponent(float x, float top, float scale) {
  return fmaxf((x - top) * scale, -kFar);
}

// e^x - 1 for x of a probability's logarithm: near 0 its series, whose next term is
// x^8 / 9! of it (below 2^-26 up to 1/2); below, where nothing cancels, the difference.
__device__ inline float exp_less_1(float x) {
  float r = 1.f;
#pragma unroll
  for (int n = 8; n > 1; --n) r = fmaf(r, x * (1.f / (float)n), 1.f);
  return x > -0.5f ? r * x : exp2_of(x * kLog2e) - 1.f;
}

// Running maximum of x, sum of e = 2^((x - top) scale), sum of e (x - top) scale.
struct Sums {
  double sum;
  float top, pull;

  __device__ void clear() {
    top = -FLT_MAX;  // not -inf: e of a logit of -inf is then 0
    sum = 0.0;
    pull = 0.f;
  }
  // moved to another, larger maximum
  __device__ void raise(float to, float scale) {
    const float d = fminf((to - top) * scale, kFar), f = exp2_of(-d);
    pull = f * (pull - d * (float)sum);
    sum *= (double)f;
    top = to;
  }
  __device__ void over_wave(float scale);
};

// x joined over the wave's lanes by `op`, in every lane.
template <typename Op>
__device__ inline float over_lanes(float x, Op op) {
  x = balance::over_lanes(x, 32, op);
  return op(x, __shfl_xor(x, 32));
}
__device__ inline void Sums::over_wave(float scale) {
  raise(over_lanes(top, [](float a, float b) { return max_of(a, b); }), scale);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  pull = over_lanes(pull, balance::kAdd);
}

// The piece of words that begins at `at`; words from `end` on are -inf.
template <typename T>
__device__ inline void load_piece(const T* row, int64_t at, int64_t end, Piece<T>& x) {
  if (at + kV<T> <= end)
    x.load(row + at);
  else
    x.load_some(row + at, end - at, (T)-INFINITY);
}
// The lane's pieces of the group that begins at `first`.
template <typename T>
__device__ inline void load_group(const T* row, int64_t first, int64_t end,
                                  Piece<T> (&x)[kPieces]) {
  const int64_t mine = first + ((int)threadIdx.x & 63) * kV<T>;
  if (first + kGroup<T> <= end) {
#pragma unroll
    for (int u = 0; u < kPieces; ++u) x[u].load(row + mine + u * kTile<T>);
  } else {
#pragma unroll
    for (int u = 0; u < kPieces; ++u) load_piece<T>(row, mine + u * kTile<T>, end, x[u]);
  }
}

// Order among all of a row's words: the larger logit, then the lower number; NaN
// above all.  0 is no word's.
__device__ inline uint32_t order_of(float x) { return x != x ? 0xffffffffu : key_of(x); }
__device__ inline float logit_of(uint32_t order) {  // NaN also where it is no logit's
  return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
__device__ inline uint64_t number_key(uint32_t order, uint32_t number) {
  return (uint64_t)order << 32 | (0xffffffffu - number);
}

// A wave's candidates, in its part of LDS.
struct Candidates {
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  uint64_t* keys;   // [kRoom], and room for the best of them
  Words* pieces;    // what belongs to a key
  int count;        // uniform
  uint64_t least;   // what a key has to reach; uniform

  // How many of n keys at `at` are above `key`; all lanes read the same ones.
  __device__ static int above(const uint64_t* at, int n, uint64_t key) {
    int r = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) r += at[i] > key;
    return r;
  }
  // Keeps the `top` best, in order.
  template <bool PIECES>
  __device__ void shrink(int top) {
    const int lane = (int)threadIdx.x & 63;
    wave_sync();
    for (int i = lane; i < count; i += 64) {
      const uint64_t key = keys[i];
      const int place = above(keys, count, key);
      if (place < top) {
        keys[kRoom + place] = key;
        if (PIECES) pieces[kRoom + place] = pieces[i];
      }
    }
    wave_sync();
    if (count > top) count = top;
    if (lane < count) {
      keys[lane] = keys[kRoom + lane];
      if (PIECES) pieces[lane] = pieces[kRoom + lane];
    }
    wave_sync();
    if (count == top) least = keys[top - 1];
  }
  // One key a lane, where `on`, with its piece.
  template <bool PIECES>
  __device__ void push(uint64_t key, Words piece, bool on, int top) {
    on = on && key >= least;
    unsigned long long m = __ballot(on);
    if (!m) return;
    if (count + __popcll(m) > kRoom) {
      shrink<PIECES>(top);
      on = on && key >= least;
      m = __ballot(on);
    }
    const int lane = (int)threadIdx.x & 63;
    if (on) {
      const int at = count + __popcll(m & ((1ull << lane) - 1));
      keys[at] = key;
      if (PIECES) pieces[at] = piece;
    }
    count += __popcll(m);
  }
};

// A bound of the k-th largest of the wave's N values a lane, from below: its upper
// half, which 16 bits have all of and a float 7 bits behind the exponent.
template <int N>
__device__ inline uint32_t kth_largest(const uint32_t (&x)[N], int k) {
  uint32_t found = 0;
  for (int b = 31; b >= 16; --b) {
    const uint32_t next = found | 1u << b;
    int reach = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) reach += __popcll(__ballot(x[i] >= next));
    if (reach >= k) found = next;
    if (reach == k) break;
  }
  return found;
}

// W waves share a row or a part of one.
template <typename T, int W, bool TOP>
__global__ __launch_bounds__(kBlock) void forward_kernel(Params p) {
  constexpr int V = kV<T>, kTeams = kBlock / 64 / W;
  __shared__ uint64_t s_keys[TOP ? kBlock / 64 * kHeld : 1];
  __shared__ Candidates::Words s_pieces[TOP ? kBlock / 64 * kHeld : 1];
  __shared__ int s_slot[TOP ? kTeams * kMaxTop : 1];
  __shared__ uint32_t s_max[TOP && W > 1 ? kBlock : 1];
  __shared__ int s_count[TOP ? kBlock / 64 : 1];
  __shared__ Sums s_sums[W > 1 ? W : 1];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x / 64;
  const int team = wave / W, mate = wave % W, thread = mate * 64 + lane;
  const auto team_sync = [] {
    if constexpr (W > 1)
      __syncthreads();
    else
      wave_sync();
  };
  const int64_t row = W > 1 ? (int64_t)blockIdx.x / p.parts : (int64_t)blockIdx.x * kTeams + team;
  const int part = W > 1 ? (int)((int64_t)blockIdx.x % p.parts) : 0;
  if (row >= p.rows) return;  // a whole team
  const int64_t y = p.tokens[row];
  if (y < 0 || y >= p.vocab || y == p.ignore) {
    if (part == 0) {
      if (TOP && thread < p.top) {
        p.top_logprobs[row * p.top + thread] = 0.f;
        p.top_tokens[row * p.top + thread] = -1;
      }
      if (thread == 0) {
        p.logprob[row] = p.entropy[row] = 0.f;
        p.saved[row] = Saved{0.f, 0.f, 0.f, -1};
      }
    }
    return;
  }
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride;
  const float x_y = (float)logits[y];
  const int64_t v0 = part * p.per_part;
  const int64_t v1 = v0 + p.per_part < p.vocab ? v0 + p.per_part : p.vocab;

  Sums sums;
  sums.clear();
  Candidates best{s_keys + (TOP ? wave * kHeld : 0), s_pieces + (TOP ? wave * kHeld : 0), 0, 0};
  int highest = 0;      // the group of the lane's largest word, from v0
  float beside = 0.f;   // what the lane added there
  float reach = 0.f;  // pieces with a smaller maximum are no candidates; NaN: all are
  bool first = true;
  for (int64_t v = v0; v < v1; v += W * kGroup<T>) {
    Piece<T> x[kPieces];
    const int64_t mine = v + mate * kGroup<T>;
    load_group<T>(logits, mine, v1, x);
    float tops[kPieces], t = -INFINITY;
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      tops[u] = max_of(x[u][0], x[u][1]);
#pragma unroll
      for (int e = 2; e < V; e += 2)
        tops[u] = max_of(max_of(tops[u], x[u][e]), x[u][e + 1]);
      t = max_of(t, tops[u]);
      // unpacked again for the exponentials: with all floats kept beside the pieces,
      // four waves fit a SIMD instead of seven (4096 x 32000, top 20: 68 us instead of 61)
      if constexpr (TOP) asm volatile("" : "+v"(x[u].words));
    }
    const bool raised = t > sums.top;
    sums.raise(max_of(sums.top, t), p.scale);
    float sum = 0.f, pull = 0.f;
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float z = exponent(x[u][e], sums.top, p.scale), ex = exp2_of(z);
        sum += ex;
        pull = fmaf(ex, z, pull);
      }
    sums.sum += (double)sum;
    sums.pull += pull;
    if (raised) {
      highest = (int)(v - v0);
      beside = sum;
    }
    if constexpr (TOP) {
      if (first) {
        const uint32_t order = order_of(t);
        uint32_t least;
        if constexpr (W > 1) {
          s_max[threadIdx.x] = order;
          __syncthreads();
          uint32_t all[W];
#pragma unroll
          for (int i = 0; i < W; ++i) all[i] = s_max[i * 64 + lane];
          least = kth_largest<W>(all, p.top);
        } else {
          const uint32_t all[1] = {order};
          least = kth_largest<1>(all, p.top);
        }
        best.least = (uint64_t)least << 32;
        reach = logit_of(least);
      }
      if (__ballot(!(t < reach))) {
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
          if (!__ballot(!(tops[u] < reach))) continue;
          const int64_t at = mine + u * kTile<T> + lane * V;
          best.push<true>(number_key(order_of(tops[u]), (uint32_t)(at / V)), x[u].words, at < v1,
                          p.top);
        }
        // pieces that follow have higher numbers: an equal logit is no candidate
        if ((uint32_t)best.least) reach = logit_of((uint32_t)(best.least >> 32) + 1);
      }
    }
    first = false;
  }
  const float own = sums.top;
  sums.over_wave(p.scale);
  // one word's 1, and less than 1 of all others; at -FLT_MAX all others are -inf, and
  // lanes that have no word have that maximum too
  if (sums.sum >= 1.0 && sums.sum < 2.0 && sums.top > -FLT_MAX) {
    static_assert(kPieces * V <= 64, "the holder's words have a lane each");
    const int holder = __builtin_ctzll(__ballot(own == sums.top));
    const int64_t at = v0 + __builtin_amdgcn_readlane(highest, holder) + mate * kGroup<T> +
                       lane / V * kTile<T> + holder * V + lane % V;
    float rest = 0.f;
    if (lane < kPieces * V && at < v1) {
      const float ex = exp2_of(exponent((float)logits[at], sums.top, p.scale));
      rest = ex == 1.f ? 0.f : ex;
    }
    rest = over_lanes(rest, balance::kAdd);
    const float added = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(beside), holder));
    sums.sum += 1.0 + (double)rest - (double)added;
  }
  if constexpr (W > 1) {
    if (lane == 0) s_sums[mate] = sums;
  }
  if constexpr (TOP) {
    if (lane == 0) s_count[wave] = best.count;
  }
  team_sync();
  if constexpr (W > 1) {
    float t = s_sums[0].top;
#pragma unroll
    for (int i = 1; i < W; ++i) t = max_of(t, s_sums[i].top);
    sums.sum = 0.0;
    sums.pull = 0.f;
    sums.top = t;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Sums o = s_sums[i];
      o.raise(t, p.scale);
      sums.sum += o.sum;
      sums.pull += o.pull;
    }
  }

  // Every candidate's place among the team's: `put(place, key, slot)` for the first
  // `top`.
  const auto rank = [&](auto put) {
    const uint64_t* keys = s_keys + team * W * kHeld;
    const int* count = s_count + team * W;
    for (int i = lane; i < best.count; i += 64) {  // each wave its own
      const uint64_t key = best.keys[i];
      int place = 0;
      for (int o = 0; o < W; ++o) place += Candidates::above(keys + o * kHeld, count[o], key);
      if (place < p.top) put(place, key, mate * kHeld + i);
    }
  };
  if constexpr (TOP) {  // pieces are ranked, then the words of the best
    constexpr int kRounds = (kMaxTop * V + W * 64 - 1) / (W * 64);
    const uint64_t* keys = s_keys + team * W * kHeld;
    const Candidates::Words* pieces = s_pieces + team * W * kHeld;
    int* slots = s_slot + team * kMaxTop;
    int held = 0;
    for (int w = 0; w < W; ++w) held += s_count[team * W + w];
    if (held > p.top) held = p.top;
    rank([&](int place, uint64_t, int slot) { slots[place] = slot; });
    team_sync();
    uint64_t words[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = r * W * 64 + thread;
      words[r] = 0;
      if (i >= held * V) continue;
      const int slot = slots[i / V];
      const int64_t word = (int64_t)(0xffffffffu - (uint32_t)keys[slot]) * V + i % V;
      const float l = (float)reinterpret_cast<const T*>(pieces + slot)[i % V];
      if (word < v1) words[r] = number_key(order_of(l), (uint32_t)word);
    }
    best.least = held == p.top ? keys[slots[p.top - 1]] & 0xffffffff00000000u : 0;
    team_sync();
    best.count = 0;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) best.push<false>(words[r], {}, words[r] != 0, p.top);
    if (lane == 0) s_count[wave] = best.count;
    team_sync();
  }

  if constexpr (W > 1) {
    if (p.parts > 1) {
      unsigned long long* all = p.part + row * p.parts * (2 + p.top);
      unsigned long long* own = all + part * (2 + p.top);
      if (thread == 0) {
        ace::store_dev(own, (unsigned long long)__double_as_longlong(sums.sum));
        ace::store_dev(own + 1, (unsigned long long)__float_as_uint(sums.top) << 32 |
                                    __float_as_uint(sums.pull));
      }
      if constexpr (TOP) {
        int held = 0;
        for (int w = 0; w < W; ++w) held += s_count[w];
        rank([&](int place, uint64_t key, int) {
          ace::store_dev(own + 2 + place, (unsigned long long)key);
        });
        if (thread >= held && thread < p.top) ace::store_dev(own + 2 + thread, 0ull);
      }
      if (!ace::last_of(p.tickets + row * kTicketStride, p.parts)) return;
      // each part's d-th best, of which the m-th largest has at least d m >= top words
      // that reach it
      const int d = TOP ? (p.top + p.parts - 1) / p.parts : 0;
      const unsigned long long* at = all + (lane < p.parts ? lane : 0) * (2 + p.top);
      const unsigned long long a = ace::load_dev(at), b = ace::load_dev(at + 1);
      const uint64_t key = TOP ? ace::load_dev(at + 1 + d) : 0ull;
      sums.clear();
      if (lane < p.parts)
        sums = Sums{__longlong_as_double((long long)a), __uint_as_float((uint32_t)(b >> 32)),
                    __uint_as_float((uint32_t)b)};
      if constexpr (TOP) {
        const int m = (p.top + d - 1) / d, n = p.parts * p.top;
        uint64_t held[kMaxParts * kMaxTop / kBlock];
#pragma unroll
        for (int i = 0; i < kMaxParts * kMaxTop / kBlock; ++i) {
          const uint32_t word = (uint32_t)(i * kBlock + thread);
          held[i] = (int)word < n ? ace::load_dev(all + word / (uint32_t)p.top * (2 + p.top) + 2 +
                                                  word % (uint32_t)p.top)
                                  : 0ull;
        }
        const uint32_t orders[1] = {lane < p.parts ? (uint32_t)(key >> 32) : 0u};
        best.count = 0;
        best.least = (uint64_t)kth_largest<1>(orders, m) << 32;
#pragma unroll
        for (int i = 0; i < kMaxParts * kMaxTop / kBlock; ++i)
          best.push<false>(held[i], {}, held[i] != 0, p.top);
        __syncthreads();
        if (lane == 0) s_count[wave] = best.count;
        __syncthreads();
      }
      sums.over_wave(p.scale);
    }
  }

  const bool defined = sums.top < INFINITY;  // not NaN, not +inf
  const bool dead = sums.sum == 0.0;         // every logit is -inf
  // log(hi + lo) = log hi + lo / hi, lo being less than a step of hi
  const float hi = (float)sums.sum, lo = (float)(sums.sum - (double)hi);
  const float log_sum = logf(hi) + lo * __builtin_amdgcn_rcpf(hi);
  const auto logprob_of = [&](float x) {
    return !defined ? NAN : dead ? -INFINITY : (x - sums.top) * p.inv_t - log_sum;
  };
  if (thread == 0) {
    const float entropy = !defined ? NAN : dead ? 0.f : log_sum - kLn2 * (sums.pull / (float)sums.sum);
    p.logprob[row] = logprob_of(x_y);
    p.entropy[row] = entropy;
    p.saved[row] = Saved{defined ? sums.top : NAN, log_sum, entropy, dead && defined ? -1 : (int)y};
  }
  if constexpr (TOP)
    rank([&](int place, uint64_t key, int) {
      p.top_logprobs[row * p.top + place] = logprob_of(logit_of((uint32_t)(key >> 32)));
      p.top_tokens[row * p.top + place] = (int64_t)(0xffffffffu - (uint32_t)key);
    });
}

// A wave does one group of a row.  Gradients that the last-level cache has no room for
// are stored past it (8192 x 65536 in bfloat16, forward and backward: 541 us instead of
// 560).
template <typename T, bool STREAM>
__global__ __launch_bounds__(kBlock) void backward_kernel(Params p) {
  constexpr int V = kV<T>;
  const int lane = (int)threadIdx.x & 63;
  // fewer than 2^28 of them, and one for the wave: a 32-bit scalar division
  const uint32_t task = (uint32_t)__builtin_amdgcn_readfirstlane(
      (int)(blockIdx.x * (kBlock / 64) + threadIdx.x / 64));
  const int64_t row = task / (uint32_t)p.tiles;
  const int64_t first = (int64_t)(task % (uint32_t)p.tiles) * kGroup<T>;
  if (row >= p.rows) return;
  const Saved s = p.saved[row];
  T* out = static_cast<T*>(p.d_logits) + row * p.vocab;
  Piece<T> x[kPieces];
  bool given = false;  // the given word is in the group
  float own = 0.f;     // its gradient
  if (s.label >= 0) {
    const T* logits = static_cast<const T*>(p.logits) + row * p.stride;
    given = s.label >= first && s.label < first + kGroup<T>;
    const T x_y = given ? logits[s.label] : (T)0.f;
    load_group<T>(logits, first, p.vocab, x);
    const float g = (p.grad_logprob ? p.grad_logprob[row] : 0.f) * p.inv_t;
    const float h = (p.grad_entropy ? p.grad_entropy[row] : 0.f) * p.inv_t;
    const float whole = s.top == s.top ? g : NAN;  // NaN anywhere in the row: everywhere
    // at most kFar below: p is 0 there, and lp times it too
    const auto logprob_of = [&](float x) {
      return fmaxf((x - s.top) * p.inv_t - s.log_sum, -kFar);
    };
    const auto entropy_term = [&](float lp, float more) {
      return -exp2_of(lp * kLog2e) * fmaf(h, lp + s.entropy, more);
    };
    // The given word's g (1 - p) keeps its digits where p is almost 1, as the others' p g do.
    if (given) {
      const float lp = logprob_of((float)x_y);
      own = fmaf(-whole, exp_less_1(lp), entropy_term(lp, 0.f));
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = entropy_term(logprob_of(x[u][e]), whole);
      x[u].set(d);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kPieces; ++u) x[u].fill((T)0.f);
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t at = first + u * kTile<T> + lane * V;
    if (at + V <= p.vocab)
      x[u].template store<STREAM>(out + at);
    else
      x[u].store_some(out + at, p.vocab - at);
  }
  // over its piece's, by the lane that stored that one (memcpy: of the same memory as the
  // piece's words; 30000 x 1000 in bfloat16 37 us, 42 with a choice at each word)
  if (given && lane == (int)(s.label - first) / V % 64) {
    const T v = (T)own;
    __builtin_memcpy(out + s.label, &v, sizeof v);
  }
}

}  // namespace logprob
}  // namespace ace
