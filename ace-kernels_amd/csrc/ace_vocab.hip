// Host side of the vocabulary loss (ace_vocab_forward / ace_vocab_backward,
// declared in include/ace_hip.h): argument checks, the choice of tiles, the
// layout of the workspace, and the launches.  Nothing here allocates, copies
// or synchronises.
#include "ace_vocab.hpp"

#include "ace_core.hpp"  // device-coherent accesses

#include "ace_hip.h"

namespace ace {
namespace vocab {

#define ACE_DECLARE_VOCAB(T)                                                                       \
  template <> hipError_t Launch<T>::prep(const PrepParams&, int, hipStream_t);                     \
  template <> hipError_t Launch<T>::pad(const void*, void*, int64_t, int, int, hipStream_t);       \
  template <> hipError_t Launch<T>::score(int, const ScoreParams&, int, hipStream_t);              \
  template <> hipError_t Launch<T>::upstream(const UpstreamParams&, int, hipStream_t);             \
  template <> hipError_t Launch<T>::dscore(int, const ScoreParams&, int, hipStream_t);             \
  template <> hipError_t Launch<T>::grad(int, bool, const GradParams&, int, hipStream_t);          \
  template <> hipError_t Launch<T>::finish(bool, const FinishParams&, int, hipStream_t);
ACE_DECLARE_VOCAB(float)
ACE_DECLARE_VOCAB(__bf16)
ACE_DECLARE_VOCAB(_Float16)
#undef ACE_DECLARE_VOCAB

namespace {

struct JoinParams {
  const Part* part;
  const float* label_logit;
  Saved saved;
  int64_t vocab;
  int bm, bn, score_blocks;  // the score kernel's tile and grid
  int reduction;             // 0 mean, 1 sum, 2 none
  float* loss;               // one value, or [n] for none
  float* confidence;         // [n] or null
  float* correct;
  double* sums;              // [blocks]
  int* ticket;
};

// One wave per row joins the blocks' parts; the block that finishes last adds
// the blocks' sums of nll in order (double: the result does not depend on which
// block that is).
__global__ __launch_bounds__(256) void join_kernel(JoinParams p) {
  __shared__ double s_sum[256];
  __shared__ int s_last;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int count = *p.saved.count;
  const int tts = (count + p.bn - 1) / p.bn;
  const int64_t vts = (p.vocab + p.bm - 1) / p.bm;
  const mma::Deal d = score_deal(tts, (int)vts, p.score_blocks);
  const int per = (count + (int)gridDim.x * 4 - 1) / ((int)gridDim.x * 4);
  const int first = ((int)blockIdx.x * 4 + wave) * per;
  const int last = first + per < count ? first + per : count;
  double total = 0.0;
  for (int r = first; r < last; ++r) {
    const int tt = r / p.bn;
    float top = -FLT_MAX, sum = 0.f;
    int best = kNone;
    for (int s = lane; s < d.splits; s += 64) {
      const Part q = p.part[((int64_t)tt * d.splits + s) * p.bn + r % p.bn];
      join(top, sum, best, q.top, q.sum, q.best);
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2)
      join(top, sum, best, __shfl_xor(top, x), __shfl_xor(sum, x), __shfl_xor(best, x));
    if (lane == 0) {
      // log(sum) and top - label apart: a confident token's nll keeps its digits
      const float nll = logf(sum) + (top - p.label_logit[r]);
      const float inv = 1.f / sum;
      p.saved.top[r] = top;
      p.saved.inv[r] = inv;
      p.saved.best[r] = best;
      const int t = p.saved.token[r];
      if (p.reduction == 2) p.loss[t] = nll;
      if (p.confidence) p.confidence[t] = inv;
      if (p.correct) p.correct[t] = best == p.saved.label[r] ? 1.f : 0.f;
      total += (double)nll;
    }
  }
  if (p.reduction == 2) return;
  s_sum[tid] = total;
  __syncthreads();
  if (tid == 0) {
    const double s = s_sum[0] + s_sum[64] + s_sum[128] + s_sum[192];
    __hip_atomic_store(&p.sums[blockIdx.x], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_own_writes();
    s_last = ticket(p.ticket) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  double s = 0.0;
  for (int b = tid; b < (int)gridDim.x; b += 256)
    s += __hip_atomic_load(&p.sums[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s_sum[tid] = s;
  __syncthreads();
  for (int d = 128; d; d >>= 1) {
    if (tid < d) s_sum[tid] += s_sum[tid + d];
    __syncthreads();
  }
  if (tid == 0) *p.loss = (float)(p.reduction == 0 ? s_sum[0] / (count > 0 ? count : 1) : s_sum[0]);
}

constexpr int kCus = 256;
constexpr int64_t kMaxTokens = (int64_t)1 << 30, kMaxVocab = (int64_t)1 << 30;
constexpr int64_t kMaxHidden = (int64_t)1 << 20;
// Bytes of dS that one piece of the vocabulary may take: what the last-level
// cache holds.
constexpr int64_t kPieceBytes = (int64_t)256 << 20;

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t parts(int64_t x, int64_t of) { return (x + of - 1) / of; }
int elem_size(int dtype) { return dtype == ACE_F32 ? 4 : 2; }

// Rates of the tiles relative to each other, measured on large products: with 16
// bits 1146, 870 and less (TFLOP/s), which small tiles lose to the traffic of LDS;
// with float32 the matrix cores alone bound them (125 to 140).
float rate_of(int es, int tile) {
  constexpr float half[kTiles] = {1.2f, 0.85f, 0.65f, 0.4f}, single[kTiles] = {0.95f, 1.f, 0.95f, 0.85f};
  return es == 2 ? half[tile] : single[tile];
}

// The tile for m x n results: the one that takes the least time, counting what
// its edges waste.  `whole`: tiles are not cut, so that a round of blocks counts
// in full however few they are.
int pick_tile(int es, int64_t m, int64_t n, bool whole, int first = kTile256) {
  int best = first;
  double least = 0.0;
  for (int t = first; t < kTiles; ++t) {
    const TileShape s = kShape[t];
    const double slots = (double)kCus * s.per_cu;
    double rounds = (double)(parts(m, s.bm) * parts(n, s.bn)) / slots;
    if (whole) rounds = (double)(int64_t)(rounds + 1.0 - 1e-9);
    const double cost = rounds * s.per_cu * s.bm * s.bn / rate_of(es, t);
    if (t == first || cost < least) {
      best = t;
      least = cost;
    }
  }
  return best;
}

// Most parts that mma::deal makes of at most `tiles` tiles.
int64_t parts_of(int blocks, int rounds, int64_t tiles) {
  const int64_t cut = (int64_t)blocks * rounds;
  return tiles > cut ? tiles : cut;
}

struct Cursor {  // lays out a workspace
  size_t at = 0;
  size_t take(size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  }
};

// Everything that follows from the sizes alone.
struct Plan {
  int64_t n, h, v, width;
  int es;
  bool pad;            // the weight's rows are copied to a padded width
  int score_tile, score_blocks;
  int prep_blocks, prep_per, join_blocks;
  // backward
  int64_t piece;       // words of a piece (a multiple of 256)
  int dscore_blocks;
  int dh_tile, dh_blocks;
  int dw_tile, dw_blocks;
  bool dw_seg;
  int64_t dh_segs, dw_segs;
};

Plan make_plan(int dtype, int64_t n, int64_t h, int64_t v) {
  Plan p{};
  p.n = n;
  p.h = h;
  p.v = v;
  p.es = elem_size(dtype);
  p.width = up(h, 16 / p.es);
  p.pad = p.width != h;
  p.score_tile = pick_tile(p.es, v, n, true);
  const auto blocks_of = [](int tile, int64_t tiles) {
    const int64_t most = (int64_t)kCus * kShape[tile].per_cu;
    return (int)(tiles < most ? (tiles > 0 ? tiles : 1) : most);
  };
  const TileShape st = kShape[p.score_tile];
  p.score_blocks = blocks_of(p.score_tile, parts(v, st.bm) * parts(n, st.bn));
  p.prep_per = (int)parts(n > 0 ? n : 1, kPrepBlocks);
  p.prep_blocks = (int)parts(n > 0 ? n : 1, p.prep_per);
  p.join_blocks = (int)(n < 4 * kPrepBlocks ? parts(n > 0 ? n : 1, 4) : kPrepBlocks);
  // equal pieces, of no more than kPieceBytes unless a piece would be narrow
  int64_t most = kPieceBytes / ((n > 0 ? n : 1) * p.es) / 256 * 256;
  if (most < 2048) most = 2048;
  p.piece = up(parts(v, parts(v, most)), 256);
  p.dscore_blocks = blocks_of(p.score_tile, parts(p.piece, st.bm) * parts(n, st.bn));
  p.dh_tile = pick_tile(p.es, p.width, n, false);
  const TileShape ht = kShape[p.dh_tile];
  const int64_t dh_tiles = parts(p.width, ht.bm) * parts(n, ht.bn);
  p.dh_blocks = blocks_of(p.dh_tile, dh_tiles * parts(p.piece, mma::kStepBytes / p.es));
  p.dh_segs = parts_of(p.dh_blocks, kGradRounds, dh_tiles);
  // few tokens: what is written bounds it, and blocks that share a CU overlap
  p.dw_tile = pick_tile(p.es, p.width, p.piece, true, n > 256 ? kTile256 : kTile128);
  // the tokens are shared out as well where whole tiles leave half of the CUs idle
  p.dw_seg = n >= 512 && parts(p.width, 128) * parts(p.piece, 128) < kCus;
  if (p.dw_seg) p.dw_tile = kTile128;
  const TileShape wt = kShape[p.dw_tile];
  const int64_t dw_tiles = parts(p.width, wt.bm) * parts(p.piece, wt.bn);
  p.dw_blocks = p.dw_seg ? kCus * wt.per_cu : blocks_of(p.dw_tile, dw_tiles);
  p.dw_segs = p.dw_seg ? parts_of(p.dw_blocks, kGradRounds, dw_tiles) : 0;
  return p;
}

struct ForwardSpace {
  size_t zeros, ticket, rows, weight, part, label_logit, sums, bytes;
};
ForwardSpace forward_space(const Plan& p) {
  Cursor c;
  ForwardSpace s{};
  const TileShape st = kShape[p.score_tile];
  s.zeros = c.take(16);
  s.ticket = c.take(4);
  s.sums = c.take((size_t)p.join_blocks * 8);
  s.label_logit = c.take((size_t)p.n * 4);
  const size_t score_parts = parts_of(p.score_blocks, kScoreRounds, parts(p.n, st.bn));
  s.part = c.take(score_parts * st.bn * sizeof(Part));
  s.rows = c.take((size_t)(p.n * p.width) * p.es);
  s.weight = c.take(p.pad ? (size_t)(p.v * p.width) * p.es : 0);
  s.bytes = c.at;
  return s;
}

struct BackwardSpace {
  size_t zeros, scale, bound, g, c, rows, weight, ds, dh, dw, bytes;
};
BackwardSpace backward_space(const Plan& p) {
  Cursor c;
  BackwardSpace s{};
  const TileShape ht = kShape[p.dh_tile], wt = kShape[p.dw_tile];
  s.zeros = c.take(16);
  s.scale = c.take(8);
  s.bound = c.take((size_t)p.prep_blocks * 8);
  s.g = c.take((size_t)p.n * 4);
  s.c = c.take((size_t)p.n * 4);
  s.rows = c.take((size_t)(p.n * p.width) * p.es);
  s.weight = c.take(p.pad ? (size_t)(p.v * p.width) * p.es : 0);
  s.ds = c.take((size_t)(p.n * p.piece) * p.es);
  s.dh = c.take((size_t)p.dh_segs * ht.bm * ht.bn * 4);
  s.dw = c.take((size_t)p.dw_segs * wt.bm * wt.bn * 4);
  s.bytes = c.at;
  return s;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check(const void* hidden, const void* weight, int dtype, int64_t n, int64_t h, int64_t v,
          int reduction, const void* saved, const void* workspace) {
  if (dtype != ACE_F32 && dtype != ACE_BF16 && dtype != ACE_F16) return ACE_EINVAL;
  if (n < 0 || h < 1 || v < 1) return ACE_EINVAL;
  if (reduction != ACE_RED_MEAN && reduction != ACE_RED_SUM && reduction != ACE_RED_NONE)
    return ACE_EINVAL;
  if (!weight || !saved || !workspace || (!hidden && n > 0)) return ACE_EINVAL;
  if (!aligned16(hidden) || !aligned16(weight) || !aligned16(workspace) || !aligned16(saved))
    return ACE_EINVAL;
  if (n > kMaxTokens || v > kMaxVocab || h > kMaxHidden) return ACE_EUNSUPPORTED;
  return ACE_OK;
}

int code_of(hipError_t e) { return e == hipSuccess ? ACE_OK : ACE_EHIP + (int)e; }

#define ACE_TRY(call)                          \
  do {                                         \
    const hipError_t e_ = (call);              \
    if (e_ != hipSuccess) return code_of(e_);  \
  } while (0)

template <typename T>
int forward(const Plan& p, const void* hidden, const void* weight, const int64_t* labels,
            int64_t ignore_index, int reduction, void* saved, float* loss, float* confidence,
            float* correct, char* ws, hipStream_t s) {
  const ForwardSpace at = forward_space(p);
  PrepParams q{};
  q.labels = labels;
  q.ignore = ignore_index;
  q.vocab = p.v;
  q.hidden = hidden;
  q.rows = ws + at.rows;
  q.n = p.n;
  q.hidden_size = (int)p.h;
  q.width = (int)p.width;
  q.vec = !p.pad;
  q.per_block = p.prep_per;
  q.saved = saved_of(saved, p.n);
  q.nll = reduction == ACE_RED_NONE ? loss : nullptr;
  q.confidence = confidence;
  q.correct = correct;
  q.zeros = ws + at.zeros;
  q.ticket = reinterpret_cast<int*>(ws + at.ticket);
  ACE_TRY(Launch<T>::prep(q, p.prep_blocks, s));
  if (p.n > 0) {
    if (p.pad) {
      ACE_TRY(Launch<T>::pad(weight, ws + at.weight, p.v, (int)p.h, (int)p.width, s));
      weight = ws + at.weight;
    }
    ScoreParams r{};
    r.weight = static_cast<const char*>(weight);
    r.rows = ws + at.rows;
    r.vocab = p.v;
    r.hidden_size = (int)p.h;
    r.width = (int)p.width;
    r.saved = q.saved;
    r.zeros = q.zeros;
    r.part = reinterpret_cast<Part*>(ws + at.part);
    r.label_logit = reinterpret_cast<float*>(ws + at.label_logit);
    r.want_best = confidence || correct;
    ACE_TRY(Launch<T>::score(p.score_tile, r, p.score_blocks, s));
  }
  JoinParams j{};
  j.part = reinterpret_cast<const Part*>(ws + at.part);
  j.label_logit = reinterpret_cast<const float*>(ws + at.label_logit);
  j.saved = q.saved;
  j.vocab = p.v;
  j.bm = kShape[p.score_tile].bm;
  j.bn = kShape[p.score_tile].bn;
  j.score_blocks = p.score_blocks;
  j.reduction = reduction;
  j.loss = loss;
  j.confidence = confidence;
  j.correct = correct;
  j.sums = reinterpret_cast<double*>(ws + at.sums);
  j.ticket = q.ticket;
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)p.join_blocks), dim3(256), 0, s, j);
  return code_of(hipGetLastError());
}

template <typename T>
int backward(const Plan& p, const void* hidden, const void* weight, int reduction,
             const void* saved, const float* grad_loss, const float* grad_confidence,
             void* d_hidden, void* d_weight, char* ws, hipStream_t s) {
  const BackwardSpace at = backward_space(p);
  UpstreamParams q{};
  q.copy.hidden = hidden;
  q.copy.rows = ws + at.rows;
  q.copy.n = p.n;
  q.copy.hidden_size = (int)p.h;
  q.copy.width = (int)p.width;
  q.copy.vec = !p.pad;
  q.copy.per_block = p.prep_per;
  q.copy.saved = saved_of(const_cast<void*>(saved), p.n);
  q.copy.zeros = ws + at.zeros;
  q.reduction = reduction;
  q.grad_loss = grad_loss;
  q.grad_conf = grad_confidence;
  q.g = reinterpret_cast<float*>(ws + at.g);
  q.c = grad_confidence ? reinterpret_cast<float*>(ws + at.c) : nullptr;
  q.bound = reinterpret_cast<float*>(ws + at.bound);
  ACE_TRY(Launch<T>::upstream(q, p.prep_blocks, s));
  if (p.pad) {
    ACE_TRY(Launch<T>::pad(weight, ws + at.weight, p.v, (int)p.h, (int)p.width, s));
    weight = ws + at.weight;
  }
  float* scale = sizeof(T) == 2 ? reinterpret_cast<float*>(ws + at.scale) : nullptr;
  // float16: tokens' upstream gradients may be far apart (kApart)
  const bool apart = __is_same(T, _Float16) && d_hidden && p.n > 0 &&
                     (reduction == ACE_RED_NONE || grad_confidence);
  const TileShape ht = kShape[p.dh_tile], wt = kShape[p.dw_tile];
  const int64_t row_bytes = p.width * p.es;
  for (int64_t v0 = 0; v0 < p.v; v0 += p.piece) {
    const int64_t v1 = v0 + p.piece < p.v ? v0 + p.piece : p.v;
    const char* w = static_cast<const char*>(weight) + v0 * row_bytes;
    ScoreParams r{};
    r.weight = static_cast<const char*>(weight);
    r.rows = ws + at.rows;
    r.vocab = p.v;
    r.hidden_size = (int)p.h;
    r.width = (int)p.width;
    r.saved = q.copy.saved;
    r.zeros = q.copy.zeros;
    r.v0 = v0;
    r.v1 = v1;
    r.stride = p.piece;
    r.ds = ws + at.ds;
    r.g = q.g;
    r.c = q.c;
    r.one_g = grad_loss && reduction != ACE_RED_NONE;
    r.bound = q.bound;
    r.bounds = p.prep_blocks;
    r.scale = scale;
    r.scaling = apart && !d_weight ? kEach : kTogether;
    ACE_TRY(Launch<T>::dscore(p.score_tile, r, p.dscore_blocks, s));
    GradParams g{};
    g.b = ws + at.ds;
    g.b_stride = p.piece * p.es;
    g.count = q.copy.saved.count;
    g.m = p.width;
    g.zeros = q.copy.zeros;
    g.scale = scale;
    g.out_stride = p.h;
    if (d_weight) {
      g.a = ws + at.rows;
      g.a_stride = row_bytes;
      g.n = v1 - v0;
      g.seg = p.dw_seg ? reinterpret_cast<float*>(ws + at.dw) : nullptr;
      g.out = static_cast<char*>(d_weight) + v0 * p.h * p.es;
      g.out_vec = p.h % 4 == 0;
      g.out_vec8 = p.h % 8 == 0;
      const int blocks = p.dw_blocks;
      ACE_TRY(Launch<T>::grad(p.dw_tile, true, g, blocks, s));
      if (p.dw_seg) {
        FinishParams f{};
        f.seg = g.seg;
        f.count = g.count;
        f.out_rows = f.n = v1 - v0;
        f.m = p.width;
        f.hidden_size = p.h;
        f.bm = wt.bm;
        f.bn = wt.bn;
        f.grad_blocks = blocks;
        f.out = g.out;
        f.out_vec = g.out_vec;
        f.scale = scale;
        const int64_t need = parts((v1 - v0) * parts(p.h, 4), 32);
        ACE_TRY(Launch<T>::finish(true, f, (int)(need < 4096 ? need : 4096), s));
      }
    }
    if (d_hidden && p.n > 0) {
      if (apart && d_weight) {
        r.scaling = kEachOrNone;
        ACE_TRY(Launch<T>::dscore(p.score_tile, r, p.dscore_blocks, s));
      }
      g.a = w;
      g.a_stride = row_bytes;
      g.k = v1 - v0;
      g.k_map = p.piece < p.v ? p.piece : p.v;
      g.accumulate = v0 > 0;
      g.seg = reinterpret_cast<float*>(ws + at.dh);
      ACE_TRY(Launch<T>::grad(p.dh_tile, false, g, p.dh_blocks, s));
      if (v1 == p.v) {
        FinishParams f{};
        f.seg = g.seg;
        f.count = g.count;
        f.row = q.copy.saved.row;
        f.out_rows = p.n;
        f.k_map = g.k_map;
        f.m = p.width;
        f.hidden_size = p.h;
        f.bm = ht.bm;
        f.bn = ht.bn;
        f.grad_blocks = p.dh_blocks;
        f.out = d_hidden;
        f.out_vec = p.h % 4 == 0;
        f.scale = scale;
        if (apart) {
          f.g = q.g;
          f.c = q.c;
        }
        const int64_t need = parts(p.n * parts(p.h, 4), 32);
        ACE_TRY(Launch<T>::finish(false, f, (int)(need < 4096 ? need : 4096), s));
      }
    }
  }
  return ACE_OK;
}

}  // namespace
}  // namespace vocab
}  // namespace ace

using namespace ace::vocab;

extern "C" {

size_t ace_vocab_saved_bytes(int64_t tokens) {
  return tokens < 0 || tokens > kMaxTokens ? 0 : (size_t)(kSavedHead + 6 * tokens) * 4;
}

size_t ace_vocab_workspace_bytes(int dtype, int64_t tokens, int64_t hidden_size, int64_t vocab,
                                 int backward) {
  if (dtype != ACE_F32 && dtype != ACE_BF16 && dtype != ACE_F16) return 0;
  if (tokens < 0 || hidden_size < 1 || vocab < 1 || tokens > kMaxTokens || vocab > kMaxVocab ||
      hidden_size > kMaxHidden)
    return 0;
  const Plan p = make_plan(dtype, tokens, hidden_size, vocab);
  return backward ? backward_space(p).bytes : forward_space(p).bytes;
}

int ace_vocab_forward(const void* hidden, const void* weight, int dtype, const int64_t* labels,
                      int64_t tokens, int64_t hidden_size, int64_t vocab, int64_t ignore_index,
                      int reduction, void* saved, float* loss, float* confidence, float* correct,
                      void* workspace, size_t workspace_bytes, void* stream) {
  const int bad =
      check(hidden, weight, dtype, tokens, hidden_size, vocab, reduction, saved, workspace);
  if (bad) return bad;
  if ((!labels && tokens > 0) || (!loss && (tokens > 0 || reduction != ACE_RED_NONE)))
    return ACE_EINVAL;
  const Plan p = make_plan(dtype, tokens, hidden_size, vocab);
  if (workspace_bytes < forward_space(p).bytes) return ACE_EWORKSPACE;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  switch (dtype) {
    case ACE_F32:
      return forward<float>(p, hidden, weight, labels, ignore_index, reduction, saved, loss,
                            confidence, correct, ws, s);
    case ACE_BF16:
      return forward<__bf16>(p, hidden, weight, labels, ignore_index, reduction, saved, loss,
                             confidence, correct, ws, s);
    default:
      return forward<_Float16>(p, hidden, weight, labels, ignore_index, reduction, saved, loss,
                               confidence, correct, ws, s);
  }
}

int ace_vocab_backward(const void* hidden, const void* weight, int dtype, int64_t tokens,
                       int64_t hidden_size, int64_t vocab, int reduction, const void* saved,
                       const float* grad_loss, const float* grad_confidence, void* d_hidden,
                       void* d_weight, void* workspace, size_t workspace_bytes, void* stream) {
  const int bad =
      check(hidden, weight, dtype, tokens, hidden_size, vocab, reduction, saved, workspace);
  if (bad) return bad;
  if (!aligned16(d_hidden) || !aligned16(d_weight)) return ACE_EINVAL;
  const Plan p = make_plan(dtype, tokens, hidden_size, vocab);
  if (workspace_bytes < backward_space(p).bytes) return ACE_EWORKSPACE;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  switch (dtype) {
    case ACE_F32:
      return backward<float>(p, hidden, weight, reduction, saved, grad_loss, grad_confidence,
                             d_hidden, d_weight, ws, s);
    case ACE_BF16:
      return backward<__bf16>(p, hidden, weight, reduction, saved, grad_loss, grad_confidence,
                              d_hidden, d_weight, ws, s);
    default:
      return backward<_Float16>(p, hidden, weight, reduction, saved, grad_loss, grad_confidence,
                                d_hidden, d_weight, ws, s);
  }
}

}  // extern "C"
