// Host side of the vocabulary loss (ace_vocab_forward / ace_vocab_backward,
// declared in include/ace_hip.h): argument checks and the launches; the choice of
// tiles and the layout of the workspace are ace_vocab_plan.hpp's.  Nothing here allocates, copies
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

int elem_size(int dtype) { return dtype == ACE_F32 ? 4 : 2; }

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
  const Plan p = make_plan(elem_size(dtype), tokens, hidden_size, vocab);
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
  const Plan p = make_plan(elem_size(dtype), tokens, hidden_size, vocab);
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
  const Plan p = make_plan(elem_size(dtype), tokens, hidden_size, vocab);
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
