// Softmax cross entropy of hidden states against a vocabulary, with each
// token's top-label confidence, and its gradients (ace_vocab_forward /
// ace_vocab_backward, declared in include/ace_hip.h).
//
//   s_tv  = h_t . w_v                         never kept: formed tile by tile
//   lse_t = log sum_v exp s_tv,  nll_t = lse_t - s_t,y
//   a_t   = argmax_v s_tv,       conf_t = exp(s_t,a - lse_t)
//   dS_tv = g_t (p_tv - [v = y_t]) + c_t conf_t ([v = a_t] - p_tv)
//   dh_t  = sum_v dS_tv w_v,     dw_v = sum_t dS_tv h_t
//
// with g and c the upstream gradients of nll and conf.  Tokens whose label is
// not counted are left out at the start: the others' hidden states are copied
// together (`rows`), so ignored tokens cost nothing and whatever they hold, NaN
// included, reaches no result.  How many there are is known on the device only;
// grids are sized for all tokens and the kernels spread the work that there is.
//
// Forward: every block forms tiles of vocabulary x tokens (ace_mma.hpp) and
// folds each into a running maximum and sum per token, held per lane and joined
// across lanes, waves and blocks at the end.
// Backward: for each piece of the vocabulary, one kernel forms the tiles again,
// takes dS from the kept maximum and sum and stores it (in the inputs' type: the
// matrix cores' operand), one forms the piece's dw, and one adds its part of dh.
//
// All sums, the running maxima, the logits and the partial dh are float32.  The one
// rounding beside the results' own is dS's to the inputs' type, at most half a step of
// each entry (2^-8 of it in bfloat16, 2^-11 in float16), because the matrix cores take
// both operands of a product in one type: two products of halves of dS would keep more
// digits for twice the time.  The gradients' errors against 64 bits are 1.15 to 1.2
// times those of a gradient that is only rounded at the end (8192 x 4096 x 65536 in
// bfloat16: 1.93e-3 against 1.66e-3 of the gradient's norm).
//
// What bounds it: the matrix cores.  8192 tokens (5 % ignored) x 4096 x 65536 words
// in bfloat16 take 13.2 ms for four products of 4.2 TFLOP, 1.27 PFLOP/s, the rate
// of the library's products of this size (1.1 to 1.4 PFLOP/s); the logits are
// formed twice because they are not kept.  With few tokens it is the weight, which
// is read three times and whose gradient is written: 96 tokens x 2048 x 50304 words
// in float16 take 0.27 ms for 0.83 GB.
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "ace_mma.hpp"
#include "ace_vocab_plan.hpp"

namespace ace {
namespace vocab {

using mma::f32x4;
using mma::kStep;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNone = 0x7fffffff;  // no index

// What a forward leaves for its backward, in one allocation of 4-byte words:
// the number of counted tokens (`rows`), then n words each of
struct Saved {
  int* count;    // [0]: counted tokens
  int* token;    // row -> token
  int* row;      // token -> row, -1 if not counted
  int* label;    // row -> label
  int* best;     // row -> argmax
  float* top;    // row -> largest logit
  float* inv;    // row -> 1 / sum of exp(s - top)
};

constexpr int kSavedHead = 64;  // words before the arrays

__host__ __device__ inline Saved saved_of(void* p, int64_t n) {
  int* w = static_cast<int*>(p);
  int* a = w + kSavedHead;
  return Saved{w,         a,         a + n, a + 2 * n, a + 3 * n, reinterpret_cast<float*>(a + 4 * n),
               reinterpret_cast<float*>(a + 5 * n)};
}

template <typename T>
struct Four {
  typedef T type __attribute__((ext_vector_type(4)));
};

// The first `left` of four neighbouring values at `at`, in T; one store where
// the row allows it (`vec`: rows are whole aligned groups of four).
template <typename T>
__device__ inline void store4(T* at, f32x4 x, int64_t left, bool vec) {
  const typename Four<T>::type v{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
  if (vec && left >= 4) {
    *reinterpret_cast<typename Four<T>::type*>(at) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) at[e] = v[e];
  }
}

// Eight neighbouring values at `at` (a multiple of 16 bytes), in T.
template <typename T>
__device__ inline void store8(T* at, f32x4 x, f32x4 y) {
  if constexpr (sizeof(T) == 2) {
    typedef T Eight __attribute__((ext_vector_type(8)));
    *reinterpret_cast<Eight*>(at) = Eight{(T)x[0], (T)x[1], (T)x[2], (T)x[3],
                                          (T)y[0], (T)y[1], (T)y[2], (T)y[3]};
  } else {
    reinterpret_cast<f32x4*>(at)[0] = x;
    reinterpret_cast<f32x4*>(at)[1] = y;
  }
}

// A block's share of one token's softmax.
struct Part {
  float top, sum;
  int best, pad;
};
static_assert(sizeof(Part) == kPartBytes, "the workspace holds them");

// Both take NaN along.
__device__ inline float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// (top, sum, best) of two disjoint sets of words: the larger logit, the lower
// index where they are equal.
__device__ inline void join(float& top, float& sum, int& best, float top2, float sum2, int best2) {
  const float t = fmaxf(top, top2);
  best = top2 > top || (top2 == top && best2 < best) ? best2 : best;
  // a set without a logit has sum 0 and the lowest top: its factor is 0 or 1
  sum = sum * exp_of(top - t) + sum2 * exp_of(top2 - t);
  top = t;
}

// ----------------------------------------------------------- rows of tokens

struct PrepParams {
  const int64_t* labels;
  int64_t ignore, vocab;
  const void* hidden;
  void* rows;          // [n, width] the counted tokens' hidden states
  int64_t n;
  int hidden_size, width;  // width: hidden_size rounded up to 16 bytes
  int vec;             // rows of `hidden` are whole aligned 16-byte chunks
  int per_block;       // tokens (forward) or rows (backward) a block handles
  Saved saved;
  float* nll;          // outputs of tokens that are not counted: 0 (or null)
  float* confidence;
  float* correct;
  char* zeros;         // 16 zero bytes for the kernels that follow
  int* ticket;
};

// Copies the rows `token[0..count)` of `hidden` (LDS list) to rows at..
template <typename T>
__device__ inline void copy_rows(const void* hidden, void* rows, int hidden_size, int width,
                                 int vec, const int* token, int count, int64_t at) {
  if (vec) {
    // at most 256 rows of 2^18 chunks: 32 bits
    const uint32_t chunks = (uint32_t)(width * (int)sizeof(T) / 16);
    for (uint32_t i = threadIdx.x; i < (uint32_t)count * chunks; i += blockDim.x) {
      const uint32_t j = i / chunks, c = i % chunks;
      reinterpret_cast<uint4*>(rows)[(at + j) * chunks + c] =
          reinterpret_cast<const uint4*>(hidden)[(int64_t)token[j] * chunks + c];
    }
  } else {
    for (uint32_t i = threadIdx.x; i < (uint32_t)count * (uint32_t)width; i += blockDim.x) {
      const uint32_t j = i / (uint32_t)width, c = i % (uint32_t)width;
      T v{};
      if (c < (uint32_t)hidden_size) v = static_cast<const T*>(hidden)[(int64_t)token[j] * hidden_size + c];
      static_cast<T*>(rows)[(at + j) * width + c] = v;
    }
  }
}

// Numbers the counted tokens, and copies their labels and hidden states
// together.  Each block counts the labels before its own by itself: cheaper than
// another launch, as the labels are few and in the caches.
template <typename T>
__global__ __launch_bounds__(256) void prep_kernel(PrepParams p) {
  __shared__ int s_count[4], s_token[256];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)blockIdx.x * p.per_block;
  const int64_t last = first + p.per_block < p.n ? first + p.per_block : p.n;
  auto counted = [&](int64_t t) {
    const int64_t y = p.labels[t];
    return y >= 0 && y < p.vocab && y != p.ignore;
  };
  if (blockIdx.x == 0 && tid < 4) {
    reinterpret_cast<int*>(p.zeros)[tid] = 0;
    if (tid == 0) *p.ticket = 0;
  }
  int before = 0;
  for (int64_t t = tid; t < first; t += 256) before += counted(t);
  for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d);
  if (lane == 0) s_count[wave] = before;
  __syncthreads();
  int64_t row = s_count[0] + s_count[1] + s_count[2] + s_count[3];
  for (int64_t t0 = first; t0 < last; t0 += 256) {
    __syncthreads();
    const int64_t t = t0 + tid;
    const bool in = t < last, yes = in && counted(t);
    const unsigned long long m = __ballot(yes);
    if (lane == 0) s_count[wave] = __popcll(m);
    __syncthreads();
    int at = __popcll(m & ((1ull << lane) - 1));
    for (int w = 0; w < wave; ++w) at += s_count[w];
    const int here = s_count[0] + s_count[1] + s_count[2] + s_count[3];
    if (yes) {
      s_token[at] = (int)t;
      p.saved.token[row + at] = (int)t;
      p.saved.label[row + at] = (int)p.labels[t];
      p.saved.row[t] = (int)(row + at);
    } else if (in) {
      p.saved.row[t] = -1;
      if (p.nll) p.nll[t] = 0.f;
      if (p.confidence) p.confidence[t] = 0.f;
      if (p.correct) p.correct[t] = 0.f;
    }
    __syncthreads();
    copy_rows<T>(p.hidden, p.rows, p.hidden_size, p.width, p.vec, s_token, here, row);
    row += here;
  }
  if (blockIdx.x == gridDim.x - 1 && tid == 0) *p.saved.count = (int)row;
}

// Rows of a weight whose rows are not whole aligned 16-byte chunks, padded to
// `width` with zeros.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* src, T* dst, int64_t rows, int size,
                                                  int width) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = (int)threadIdx.x; c < width; c += 256)
      dst[r * width + c] = c < size ? src[r * size + c] : T{};
}

// ------------------------------------------------------------------ forward

struct ScoreParams {
  const char* weight;  // [vocab, width]
  const char* rows;    // [n, width]
  int64_t vocab;
  int width;
  Saved saved;
  const char* zeros;
  // forward
  Part* part;          // [parts][BN]
  float* label_logit;  // row -> s_ty
  int want_best;       // somebody asks for the top label
  // backward
  int64_t v0;          // first word of this piece
  int64_t v1;          // end of it
  int64_t stride;      // elements of a row of ds
  void* ds;            // [n, stride]
  const float* g;      // row -> upstream of nll
  const float* c;      // row -> upstream of conf, times conf; null: none
  int one_g;           // g is the same for all rows
  const float* bound;  // blocks' largest |g| + |c|, then (float16) their smallest
                       // that is not 0, and how many blocks
  int bounds;
  int scaling;         // float16: kTogether, kEach or kEachOrNone
  float* scale;        // 16 bits (out): what ds is multiplied by, and whether the
                       // rows of the hidden gradient's ds have scales of their own
};

// How the score kernels deal (token tile) x (vocabulary tiles): part s of a token
// tile has the vocabulary tiles s, s + splits, ..., so that all blocks of an XCD
// walk the same few vocabulary tiles at a time (4 to 8 of them and 4 to 8 token
// tiles): 1250 TFLOP/s at 8192 x 4096 x 65536, against 995 where each block had a
// run of vocabulary tiles of its own.
__device__ inline mma::Deal score_deal(int tts, int vts, int blocks) {
  return mma::deal(tts, vts, blocks, 0, kScoreRounds);
}

// The tile walk that forward and backward share: `fold(tt, vt, acc)` takes a
// finished tile, `enter(tt)` and `leave(part)` a part's run of them.  The pipeline
// runs on across tiles: the next one's first steps load while `fold` works.
template <class TL, class Enter, class Fold, class Leave>
__device__ inline void walk_tiles(const ScoreParams& p, int64_t v0, int64_t v1, Enter enter,
                                  Fold fold, Leave leave) {
  using T = typename TL::T;
  const int count = *p.saved.count;
  const int tts = (count + TL::BN - 1) / TL::BN;
  const int vts = (int)((v1 - v0 + TL::BM - 1) / TL::BM);
  if (tts == 0) return;
  const int blocks = (int)gridDim.x;
  const mma::Deal d = score_deal(tts, vts, blocks);
  const int first = mma::xcd_order((int)blockIdx.x, blocks);
  const int64_t row_bytes = (int64_t)p.width * sizeof(T);
  const int k = p.width;
  const int steps = (k + kStep<T> - 1) / kStep<T>;
  // what is loaded next: step `at` of vocabulary tile `to_vt` of part `to`
  typename TL::OpA a;
  typename TL::OpB bo;
  typename TL::Source sa, sb;
  sa.step = sb.step = mma::kStepBytes;
  int at = steps, to = first - blocks, to_vt = vts;
  const auto feed = [&](char* lds) {
    if (at == steps) {
      to_vt += d.splits;
      const bool turn = to_vt >= vts;
      if (turn) {
        if (to + blocks >= d.parts()) return false;
        to += blocks;
        to_vt = to % d.splits;
        const int tt = to / d.splits;
        bo.init(row_bytes, (int64_t)tt * TL::BN, count);
        sb.base = p.rows + (int64_t)tt * TL::BN * row_bytes;
      }
      const int64_t v = v0 + (int64_t)to_vt * TL::BM;
      a.init(row_bytes, v, v1);
      sa.base = p.weight + v * row_bytes;
      at = 0;
    }
    TL::load(a, bo, sa, sb, at, k, lds, p.zeros);
    ++at;
    return true;
  };
  const auto simple = [&](int i, char* lds) {
    TL::load_one(i, a, bo, sa, sb, at, lds);
    if (i == TL::kLoads - 1) ++at;
  };
  typename TL::Pipe pipe;
  pipe.begin(feed);
  f32x4 acc[TL::MT][TL::NT];
  for (int part = first; part < d.parts(); part += blocks) {
    const int tt = part / d.splits;
    enter(tt);
    for (int vt = part % d.splits; vt < vts; vt += d.splits) {
      TL::clear(acc);
      pipe.run(steps, TL::plain_steps(0, steps, k), simple, feed, acc);
      fold(tt, vt, acc);
    }
    leave(part);
  }
}

// The forward: each lane keeps a running maximum and sum for each of its tokens
// over the words that it holds, without an exchange until its part ends.  Per
// tile of 256 x 256 the exponentials cost about 8 us of which nothing overlaps the
// products (28 us at a hidden size of 1024, 113 us at 4096).
template <class TL>
__global__ __launch_bounds__(TL::kThreads, TL::kWaves) void score_kernel(ScoreParams p) {
  constexpr int NT = TL::NT, MT = TL::MT;
  __shared__ Part s_part[TL::WM][TL::BN];
  const int lane = (int)threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int count = *p.saved.count;
  float top[NT], sum[NT];
  int best[NT], label[NT];
  auto enter = [&](int tt) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      top[j] = -FLT_MAX;
      sum[j] = 0.f;
      best[j] = kNone;
      const int r = tt * TL::BN + TL::wave_n() + 16 * j + n;
      label[j] = r < count ? p.saved.label[r] : -1;
    }
  };
  auto fold = [&](int tt, int vt, f32x4(&acc)[MT][NT]) {
    const int v_wave = vt * TL::BM + TL::wave_m();  // the wave's first word
    const int left = (int)(p.vocab - v_wave) - 4 * g;
    if (p.vocab - v_wave < TL::BM / TL::WM) {  // ragged end: words that do not exist
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * i + e >= left) acc[i][j][e] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float t = top[j];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; e += 2) t = max_of(max_of(t, acc[i][j][e]), acc[i][j][e + 1]);
      if (p.want_best && __ballot(t > top[j])) {
        // a new largest logit somewhere in the wave: where it stands.  Words
        // come in ascending order, so the first place that has it stays.
        int at = kNone;
#pragma unroll
        for (int i = MT - 1; i >= 0; --i)
#pragma unroll
          for (int e = 3; e >= 0; --e) at = acc[i][j][e] == t ? 16 * i + e : at;
        if (t > top[j]) best[j] = v_wave + 4 * g + at;
      }
      // the lane's words that the label may be among: v_wave + 4 g + 16 i + e
      const int y = label[j] - v_wave - 4 * g;
      if (__ballot(y >= 0 && y < TL::BM / TL::WM && (y & 12) == 0)) {
        float s = 0.f;
        bool mine = false;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (y == 16 * i + e) {
              s = acc[i][j][e];
              mine = true;
            }
        if (mine) p.label_logit[tt * TL::BN + TL::wave_n() + 16 * j + n] = s;
      }
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) l += exp_of(acc[i][j][e] - t);
      sum[j] = sum[j] * exp_of(top[j] - t) + l;
      top[j] = t;
    }
  };
  auto leave = [&](int part) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int d = 16; d < 64; d *= 2)
        join(top[j], sum[j], best[j], __shfl_xor(top[j], d), __shfl_xor(sum[j], d),
             __shfl_xor(best[j], d));
      if (g == 0)
        s_part[(int)threadIdx.x / 64 / TL::WN][TL::wave_n() + 16 * j + n] =
            Part{top[j], sum[j], best[j], 0};
    }
    __syncthreads();
    for (int c = (int)threadIdx.x; c < TL::BN; c += TL::kThreads) {
      Part q = s_part[0][c];
#pragma unroll
      for (int w = 1; w < TL::WM; ++w)
        join(q.top, q.sum, q.best, s_part[w][c].top, s_part[w][c].sum, s_part[w][c].best);
      p.part[(int64_t)part * TL::BN + c] = q;
    }
    __syncthreads();
  };
  walk_tiles<TL>(p, 0, p.vocab, enter, fold, leave);
}

// ----------------------------------------------------------------- backward

struct UpstreamParams {
  PrepParams copy;
  int reduction;
  const float* grad_loss;  // one value, or [n] for none; null: 0
  const float* grad_conf;  // [n] or null
  float* g;
  float* c;
  float* bound;            // [blocks], float16: [2][blocks]
};

// The rows' upstream gradients, and the counted tokens' hidden states together
// again (cheaper to copy twice than to keep).
template <typename T>
__global__ __launch_bounds__(256) void upstream_kernel(UpstreamParams p) {
  __shared__ int s_token[256];
  __shared__ float s_max[4];
  const PrepParams& q = p.copy;
  const int tid = (int)threadIdx.x, count = *q.saved.count;
  if (blockIdx.x == 0 && tid < 4) reinterpret_cast<int*>(q.zeros)[tid] = 0;
  const int64_t first = (int64_t)blockIdx.x * q.per_block;
  const int64_t last = first + q.per_block < count ? first + q.per_block : count;
  float most = 0.f, least = FLT_MAX;
  for (int64_t r0 = first; r0 < last; r0 += 256) {
    __syncthreads();
    const int64_t r = r0 + tid;
    if (r < last) {
      const int t = q.saved.token[r];
      s_token[tid] = t;
      float g = 0.f, c = 0.f;
      if (p.grad_loss) {
        g = p.reduction == 2 ? p.grad_loss[t] : p.grad_loss[0];
        if (p.reduction == 0) g /= (float)count;
      }
      if (p.c) p.c[r] = c = p.grad_conf[t] * q.saved.inv[r];
      p.g[r] = g;
      const float bound = fabsf(g) + fabsf(c);
      most = fmaxf(most, bound);
      if (bound > 0.f) least = fminf(least, bound);
    }
    __syncthreads();
    if (q.rows)
      copy_rows<T>(q.hidden, q.rows, q.hidden_size, q.width, q.vec, s_token,
                   (int)(last - r0 < 256 ? last - r0 : 256), r0);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
  if ((tid & 63) == 0) s_max[tid >> 6] = most;
  __syncthreads();
  if (tid == 0) p.bound[blockIdx.x] = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  if constexpr (__is_same(T, _Float16)) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) least = fminf(least, __shfl_xor(least, d));
    __syncthreads();
    if ((tid & 63) == 0) s_max[tid >> 6] = least;
    __syncthreads();
    if (tid == 0)
      p.bound[gridDim.x + blockIdx.x] = fminf(fminf(s_max[0], s_max[1]), fminf(s_max[2], s_max[3]));
  }
}

// dS is held times a scale that its products are divided by at the end.
// Where all tokens have the same upstream gradient (mean, sum), the scale is its
// reciprocal, so that the label's entry, p - 1, is near a number that the type
// holds exactly: every token's largest entry would else be rounded alike.
// float16 takes 2^13 of that, or for other upstream gradients a power of two that
// takes the largest |g| + |c|, dS's bound, to 2^13..2^14: without it the
// probabilities of a large vocabulary are below float16's smallest numbers.
// bfloat16 has float32's range: with confidences whose upstream gradients are
// larger by more than kMostScaled it takes none, as the products' sums would
// leave that range.
//
// One scale serves all tokens in float16 while their |g| + |c| are within kApart
// of each other: an entry is then off by at most half of float16's smallest step,
// 2^-25, against a bound of 2^7, which summed over 2^18 words is below float16's
// own rounding of the token's gradient.  Where they are further apart, the
// probabilities of tokens with small upstream gradients would be lost, so the hidden
// gradient has a dS of its own, each row scaled by a power of two to 2^13..2^14, which
// finish_kernel takes out.  The weight's gradient sums over tokens, beside whose
// largest those entries do not count.
constexpr float kMostScaled = 0x1p40f;
constexpr float kApart = 64.f;
// What one launch of dscore_kernel makes: dS with one scale; dS for the hidden
// gradient, with scales by row where they are needed; or that, and nothing where
// they are not (the dS that is there serves).
enum { kTogether = 0, kEach = 1, kEachOrNone = 2 };
template <typename T>
constexpr float kHalfScale = __is_same(T, _Float16) ? 8192.f : 1.f;

__device__ inline float scale_of(float bound) {
  if (!(bound > 0.f) || bound > FLT_MAX) return 1.f;
  int e;
  frexpf(bound, &e);  // bound < 2^e
  e = 14 - e;
  return ldexpf(1.f, e > 100 ? 100 : e < -100 ? -100 : e);
}

// dS of a piece.  The first operand's rows are paired (ace_mma.hpp), so that a lane
// stores 16 bytes at a time and four lanes 64: with the label, the top label and
// the ragged end out of the common path this took 163 us instead of 194 at 2048 x
// 1024 x 32768.
template <class TL>
__global__ __launch_bounds__(TL::kThreads, TL::kWaves) void dscore_kernel(ScoreParams p) {
  using T = typename TL::T;
  constexpr int NT = TL::NT, MT = TL::MT;
  const int lane = (int)threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int count = *p.saved.count;
  float scale = 1.f;
  bool by_row = false;
  if constexpr (sizeof(T) == 2) {
    constexpr bool half = __is_same(T, _Float16);
    const float g0 = p.one_g && count > 0 ? fabsf(p.g[0]) : 0.f;
    if (g0 >= FLT_MIN * 8192.f && g0 <= FLT_MAX / 8192.f) {
      scale = kHalfScale<T> / g0;
    }
    if (p.c || (half && scale == 1.f)) {
      float most = 0.f;  // every wave on its own
      for (int i = lane; i < p.bounds; i += 64) most = fmaxf(most, p.bound[i]);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
      // with confidences: no more than the largest |g| + |c| allows
      if constexpr (half) {
        if (p.scaling != kTogether) {
          float least = FLT_MAX;
          for (int i = lane; i < p.bounds; i += 64) least = fminf(least, p.bound[p.bounds + i]);
#pragma unroll
          for (int d = 1; d < 64; d *= 2) least = fminf(least, __shfl_xor(least, d));
          by_row = least * kApart < most;
        }
        if (scale == 1.f || !(most * scale <= 32768.f)) scale = scale_of(most);
      } else {
        if (!(most * scale <= kMostScaled)) scale = 1.f;
      }
    }
    if (p.scaling == kEachOrNone && !by_row) {
      if (blockIdx.x == 0 && threadIdx.x == 0) p.scale[1] = 0.f;
      return;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      p.scale[0] = scale;
      p.scale[1] = by_row ? 1.f : 0.f;
    }
  }
  float top[NT], of_p[NT], of_label[NT], of_best[NT];
  int label[NT], best[NT];
  auto enter = [&](int tt) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = tt * TL::BN + TL::wave_n() + 16 * j + n;
      const bool in = r < count;
      float gr = in ? p.g[r] : 0.f, cr = in && p.c ? p.c[r] : 0.f;
      const float by = by_row ? scale_of(fabsf(gr) + fabsf(cr)) : scale;
      gr *= by;
      cr *= by;
      top[j] = in ? p.saved.top[r] : 0.f;
      of_p[j] = in ? (gr - cr) * p.saved.inv[r] : 0.f;
      of_label[j] = gr;
      of_best[j] = cr;
      label[j] = in ? p.saved.label[r] : -1;
      best[j] = in && p.c ? p.saved.best[r] : -1;
    }
  };
  // the lane's words of a wave's piece: of pair h, 32 h + 8 g + 0..7
  static_assert(TL::kPaired && MT % 2 == 0, "pairs of fragments");
  auto fold = [&](int tt, int vt, f32x4(&acc)[MT][NT]) {
    const int v_wave = (int)(p.v0 + (int64_t)vt * TL::BM + TL::wave_m());
    const int left = (int)(p.vocab - v_wave) - 8 * g;  // words that exist from the lane's first
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = of_p[j] * exp_of(acc[i][j][e] - top[j]);
      // the two words that have more to them are rarely in the wave's piece
      const int y = label[j] - v_wave - 8 * g, z = best[j] - v_wave - 8 * g;
      const bool here = (y >= 0 && y < TL::BM / TL::WM && (y & 24) == 0) ||
                        (z >= 0 && z < TL::BM / TL::WM && (z & 24) == 0);
      if (__ballot(here)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int w = 32 * (i >> 1) + 4 * (i & 1) + e;
            acc[i][j][e] -= y == w ? of_label[j] : 0.f;
            acc[i][j][e] += z == w ? of_best[j] : 0.f;
          }
      }
      if (p.vocab - v_wave < TL::BM / TL::WM) {  // ragged end: words that do not exist
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (32 * (i >> 1) + 4 * (i & 1) + e >= left) acc[i][j][e] = 0.f;
      }
      const int64_t r = (int64_t)tt * TL::BN + TL::wave_n() + 16 * j + n;
      if (r < count) {
        T* out = static_cast<T*>(p.ds) + r * p.stride + (v_wave + 8 * g - p.v0);
#pragma unroll
        for (int h = 0; h < MT / 2; ++h) store8(out + 32 * h, acc[2 * h][j], acc[2 * h + 1][j]);
      }
    }
  };
  walk_tiles<TL>(p, p.v0, p.v1, enter, fold, [](int) {});
}

struct GradParams {
  const char* a;        // m contiguous: the weight's piece, or the rows
  int64_t a_stride;     // bytes
  const char* b;        // ds
  int64_t b_stride;
  const int* count;
  int64_t m;            // hidden size rounded up to 16 bytes
  int64_t n;            // words of the piece (dw), unused for dh
  int64_t k;            // words of the piece (dh), unused for dw
  int64_t k_map;        // dh: words of a whole piece: every piece is cut alike
  int accumulate;       // dh: not the first piece
  float* seg;           // partial tiles [parts][BN][BM], or null: store `out`
  void* out;            // [n, out_stride]
  int64_t out_stride;   // elements: the hidden size
  int out_vec;          // rows of `out` are whole aligned groups of four
  int out_vec8;         // and of eight
  const float* scale;   // 16 bits
  const char* zeros;
};


// dh (DW = false): C[h][row] = sum over words of w[v][h] ds[row][v];
// dw (DW = true):  C[h][v] = sum over rows of rows[row][h] ds[row][v].
// With `seg`, tiles are cut along k where that fills the CUs better, and each
// part's sum goes to (or is added to) a partial tile of its own, which
// finish_kernel adds in order.  Without it blocks take whole tiles.  Parts that run
// at once are at the same place along k: 1194 TFLOP/s for dh at 8192 x 4096 x 65536,
// against 913 with the work cut evenly wherever that fell.  dw: 1.25 PFLOP/s.
template <class TL, bool DW>
__global__ __launch_bounds__(TL::kThreads, TL::kWaves) void grad_kernel(GradParams p) {
  using T = typename TL::T;
  constexpr int NT = TL::NT, MT = TL::MT, es = (int)sizeof(T);
  const int lane = (int)threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int count = *p.count;
  const int64_t nn = DW ? p.n : count;
  const int k = DW ? count : (int)p.k;
  const int mts = (int)((p.m + TL::BM - 1) / TL::BM), nts = (int)((nn + TL::BN - 1) / TL::BN);
  const int all = (k + kStep<T> - 1) / kStep<T>;  // steps there are
  // steps by which tiles are cut
  const int ks = DW ? all : (int)((p.k_map + kStep<T> - 1) / kStep<T>);
  if (nts == 0) return;
  const int blocks = (int)gridDim.x;
  const mma::Deal d = p.seg ? mma::deal(mts * nts, ks, blocks, part_steps(sizeof(T)), kGradRounds)
                            : mma::Deal{mts * nts, 1};
  const int start = mma::xcd_order((int)blockIdx.x, blocks);

  struct Part {
    int first, last;  // steps
    int64_t m0, n0;
  };
  const auto part_at = [&](int part) {
    Part q;
    const int tile = part % d.tiles, s = part / d.tiles;
    const int each = ks / d.splits, more = ks % d.splits;  // the first `more` parts have one more
    q.first = s * each + (s < more ? s : more);
    q.last = q.first + each + (s < more);
    if (q.last > all) q.last = all;
    // tiles in groups of 8 along n: a group's operands are shared in L2
    constexpr int kGroup = 8;
    const int group = tile / (kGroup * mts), from = group * kGroup;
    const int width = nts - from < kGroup ? nts - from : kGroup;
    const int in_group = tile - from * mts;
    q.n0 = (int64_t)(from + in_group % width) * TL::BN;
    q.m0 = (int64_t)(in_group / width) * TL::BM;
    return q;
  };

  typename TL::OpA a;
  typename TL::OpB b;
  typename TL::Source sa, sb;
  sa.step = kStep<T> * p.a_stride;
  sb.step = DW ? kStep<T> * p.b_stride : mma::kStepBytes;
  int to = start;  // what is loaded next: steps at..upto-1 of the part before `to`
  int at = 0, upto = 0;
  const auto feed = [&](char* lds) {
    while (at >= upto) {
      if (to >= d.parts()) return false;
      const Part q = part_at(to);
      to += blocks;
      at = q.first;
      upto = q.last;
      if (at >= upto) continue;
      a.init(p.a_stride, q.m0, p.m);
      b.init(p.b_stride, q.n0, DW ? (nn + 16 / es - 1) / (16 / es) * (16 / es) : nn);
      sa.base = p.a + q.m0 * es;
      sb.base = p.b + q.n0 * (DW ? (int64_t)es : p.b_stride);
    }
    TL::load(a, b, sa, sb, at, k, lds, p.zeros);
    ++at;
    return true;
  };
  const auto simple = [&](int i, char* lds) {
    TL::load_one(i, a, b, sa, sb, at, lds);
    if (i == TL::kLoads - 1) ++at;
  };
  typename TL::Pipe pipe;
  pipe.begin(feed);
  for (int index = start; index < d.parts(); index += blocks) {
    const Part q = part_at(index);
    const int first = q.first, last = q.last;
    float* part = p.seg ? p.seg + (int64_t)index * (TL::BM * TL::BN) : nullptr;
    const auto place = [&](int i, int j) {
      return reinterpret_cast<f32x4*>(
          part + (TL::wave_n() + 16 * j + col) * TL::BM + TL::wave_m() +
          (TL::kPaired ? 32 * (i >> 1) + 8 * g + 4 * (i & 1) : 16 * i + 4 * g));
    };
    f32x4 acc[MT][NT];
    TL::clear(acc);
    if (first < last) pipe.run(last - first, TL::plain_steps(first, last, k), simple, feed, acc);
    if (p.seg) {
      if (p.accumulate && first >= last) continue;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) *place(i, j) = p.accumulate ? *place(i, j) + acc[i][j] : acc[i][j];
    } else {
      const float inv = p.scale ? 1.f / *p.scale : 1.f;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int64_t n = q.n0 + TL::wave_n() + 16 * j + col;
        if (n >= nn) continue;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int64_t m = q.m0 + TL::wave_m() +
                            (TL::kPaired ? 32 * (i >> 1) + 8 * g + 4 * (i & 1) : 16 * i + 4 * g);
          T* at = static_cast<T*>(p.out) + n * p.out_stride + m;
          if (TL::kPaired && p.out_vec8 && m + (i & 1 ? 4 : 8) <= p.out_stride) {
            if (!(i & 1)) store8(at, acc[i][j] * inv, acc[i ^ 1][j] * inv);
          } else {
            store4(at, acc[i][j] * inv, p.out_stride - m, p.out_vec);
          }
        }
      }
    }
  }
}

struct FinishParams {
  const float* seg;
  const int* count;
  const int* row;     // dh: token -> row or -1; dw: null (row = index)
  int64_t out_rows;   // tokens, or words
  int64_t n;          // dw: words
  int64_t k_map;      // dh: words of a whole piece
  int64_t m, hidden_size;
  int bm, bn, grad_blocks;
  void* out;
  int out_vec;
  const float* scale;
  const float* g;     // dh in float16, where rows may have scales of their own: the
  const float* c;     // rows' upstream gradients (c may be null), else null
};

// out = the sum of each tile's partial tiles in order, in the output's type.  Where
// there are many for few results (few tokens, a long vocabulary), eight threads share
// a group of four values: 20 tokens of a hidden size of 256 have 1280 such groups
// of up to 384 parts, which took one thread each 29 us, and takes eight 7 us.  Backward
// in us with the rule, always one thread, always eight: 4 x 256 x 40000 38 / 45 / 38, 60 x 512
// x 11000 38 / 43 / 38, 1000 x 256 x 4000 69 / 68 / 79, 2048 x 1024 x 32768 411 / 409 / 431.
template <typename T, bool DW>
__global__ __launch_bounds__(256) void finish_kernel(FinishParams p) {
  __shared__ f32x4 s_sum[8][32];
  const int count = *p.count;
  const int64_t nn = DW ? p.n : count;
  const int k = DW ? count : (int)p.k_map;
  const int mts = ((int)p.m + p.bm - 1) / p.bm, nts = ((int)nn + p.bn - 1) / p.bn;
  const int ks = (k + kStep<T> - 1) / kStep<T>;
  const mma::Deal d = mma::deal(mts * nts, ks, p.grad_blocks, part_steps(sizeof(T)), kGradRounds);
  const float inv = p.scale ? 1.f / *p.scale : 1.f;
  const bool by_row = p.g && p.scale[1] != 0.f;
  const uint32_t quads = (uint32_t)((p.hidden_size + 3) / 4);
  const int64_t all = p.out_rows * quads;
  const int64_t stride = (int64_t)d.tiles * p.bm * p.bn;  // from a split to the next
  const auto place = [&](int64_t i, int64_t& o, int& m) {
    if (all <= UINT32_MAX) {  // a 64-bit division costs more than the rest
      o = (uint32_t)i / quads;
      m = (int)((uint32_t)i % quads) * 4;
    } else {
      o = i / quads;
      m = (int)(i % quads) * 4;
    }
  };
  // parts first, first + by, ... of group i
  const auto sum_of = [&](int64_t i, int first, int by) {
    int64_t o;
    int m;
    place(i, o, m);
    const int n = DW ? (int)o : p.row[o];
    f32x4 sum{0.f, 0.f, 0.f, 0.f};
    if (n < 0 || ks == 0) return sum;
    constexpr int kGroup = 8;
    const int nt = n / p.bn, mt = m / p.bm, from = nt / kGroup * kGroup;
    const int width = nts - from < kGroup ? nts - from : kGroup;
    const int64_t tile = (int64_t)from * mts + mt * width + (nt - from);
    const float* at = p.seg + tile * p.bm * p.bn + (n % p.bn) * p.bm + m % p.bm;
    for (int s0 = first; s0 < d.splits; s0 += 8 * by) {
      f32x4 x[8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        x[s] = s0 + s * by < d.splits ? *reinterpret_cast<const f32x4*>(at + (s0 + s * by) * stride)
                                      : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 8; ++s) sum += x[s];
    }
    return sum;
  };
  const auto put = [&](int64_t i, f32x4 sum) {
    int64_t o;
    int m;
    place(i, o, m);
    float of = inv;
    if constexpr (!DW && __is_same(T, _Float16)) {
      if (by_row) {
        const int r = p.row[o];
        if (r >= 0) of = 1.f / scale_of(fabsf(p.g[r]) + (p.c ? fabsf(p.c[r]) : 0.f));
      }
    }
    store4(static_cast<T*>(p.out) + o * p.hidden_size + m, sum * of, p.hidden_size - m, p.out_vec);
  };
  if (d.splits <= 8 || all >= 32768) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256)
      put(i, sum_of(i, 0, 1));
    return;
  }
  const int z = (int)threadIdx.x / 32, q = (int)threadIdx.x % 32;
  for (int64_t i0 = (int64_t)blockIdx.x * 32; i0 < all; i0 += (int64_t)gridDim.x * 32) {
    if (i0 + q < all) s_sum[z][q] = sum_of(i0 + q, z, 8);
    __syncthreads();
    if (z == 0 && i0 + q < all) {
      f32x4 sum = s_sum[0][q];
#pragma unroll
      for (int y = 1; y < 8; ++y) sum += s_sum[y][q];
      put(i0 + q, sum);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ launches

// Implemented per element type by ACE_DEFINE_VOCAB in the ace_k_vocab_*.hip
// units.
template <typename T>
struct Launch {
  static hipError_t prep(const PrepParams&, int blocks, hipStream_t);
  static hipError_t pad(const void* src, void* dst, int64_t rows, int size, int width, hipStream_t);
  static hipError_t score(int tile, const ScoreParams&, int blocks, hipStream_t);
  static hipError_t upstream(const UpstreamParams&, int blocks, hipStream_t);
  static hipError_t dscore(int tile, const ScoreParams&, int blocks, hipStream_t);
  static hipError_t grad(int tile, bool dw, const GradParams&, int blocks, hipStream_t);
  static hipError_t finish(bool dw, const FinishParams&, int blocks, hipStream_t);
};

template <auto KERNEL, typename P>
inline hipError_t launch(int blocks, int threads, size_t lds, hipStream_t s, const P& p) {
  if (lds > 64 * 1024) {  // asked for once per kernel and device
    static std::atomic<uint64_t> asked{0};
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (device & 63);
    if (device > 63 || !(asked.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return e;
      asked.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3((unsigned)threads), lds, s, p);
  return hipGetLastError();
}

template <typename T, bool AKC, bool BKC, bool PAIRED = false, typename F>
inline hipError_t with_tile(int tile, F f) {
  if constexpr (sizeof(T) == 2)
    if (tile == kTile256) return f(mma::Tile<T, 256, 256, 2, 4, AKC, BKC, PAIRED>{});
  switch (tile) {
    case kTile128: return f(mma::Tile<T, 128, 128, 2, 2, AKC, BKC, PAIRED>{});
    case kTile64: return f(mma::Tile<T, 128, 64, 4, 1, AKC, BKC, PAIRED>{});
    default: return f(mma::Tile<T, 128, 32, 4, 1, AKC, BKC, PAIRED>{});
  }
}

#define ACE_DEFINE_VOCAB(T)                                                                      \
  template <>                                                                                    \
  hipError_t Launch<T>::prep(const PrepParams& p, int blocks, hipStream_t s) {                   \
    return launch<prep_kernel<T>>(blocks, 256, 0, s, p);                                         \
  }                                                                                              \
  template <>                                                                                    \
  hipError_t Launch<T>::pad(const void* src, void* dst, int64_t rows, int size, int width,       \
                            hipStream_t s) {                                                     \
    const int blocks = (int)(rows < 4096 ? rows : 4096);                                         \
    hipLaunchKernelGGL(pad_kernel<T>, dim3(blocks), dim3(256), 0, s, static_cast<const T*>(src), \
                       static_cast<T*>(dst), rows, size, width);                                 \
    return hipGetLastError();                                                                    \
  }                                                                                              \
  template <>                                                                                    \
  hipError_t Launch<T>::score(int tile, const ScoreParams& p, int blocks, hipStream_t s) {       \
    return with_tile<T, true, true>(tile, [&](auto t) {                                          \
      using TL = decltype(t);                                                                    \
      return launch<score_kernel<TL>>(blocks, TL::kThreads, TL::kLdsBytes, s, p);                \
    });                                                                                          \
  }                                                                                              \
  template <>                                                                                    \
  hipError_t Launch<T>::upstream(const UpstreamParams& p, int blocks, hipStream_t s) {           \
    return launch<upstream_kernel<T>>(blocks, 256, 0, s, p);                                     \
  }                                                                                              \
  template <>                                                                                    \
  hipError_t Launch<T>::dscore(int tile, const ScoreParams& p, int blocks, hipStream_t s) {      \
    return with_tile<T, true, true, true>(tile, [&](auto t) {                                    \
      using TL = decltype(t);                                                                    \
      return launch<dscore_kernel<TL>>(blocks, TL::kThreads, TL::kLdsBytes, s, p);               \
    });                                                                                          \
  }                                                                                              \
  template <>                                                                                    \
  hipError_t Launch<T>::grad(int tile, bool dw, const GradParams& p, int blocks,                 \
                             hipStream_t s) {                                                    \
    if (dw)                                                                                      \
      return with_tile<T, false, false, sizeof(T) == 2>(tile, [&](auto t) {                      \
        using TL = decltype(t);                                                                  \
        return launch<grad_kernel<TL, true>>(blocks, TL::kThreads, TL::kLdsBytes, s, p);         \
      });                                                                                        \
    return with_tile<T, false, true>(tile, [&](auto t) {                                         \
      using TL = decltype(t);                                                                    \
      return launch<grad_kernel<TL, false>>(blocks, TL::kThreads, TL::kLdsBytes, s, p);          \
    });                                                                                          \
  }                                                                                              \
  template <>                                                                                    \
  hipError_t Launch<T>::finish(bool dw, const FinishParams& p, int blocks, hipStream_t s) {      \
    return dw ? launch<finish_kernel<T, true>>(blocks, 256, 0, s, p)                             \
              : launch<finish_kernel<T, false>>(blocks, 256, 0, s, p);                           \
  }

}  // namespace vocab
}  // namespace ace
