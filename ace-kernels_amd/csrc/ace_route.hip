// The expert choice's entry points (declared in include/ace_hip.h): argument
// checks, launch geometry, instantiations.
#include "ace_route.hpp"

#include "ace_hip.h"

namespace ace {
namespace route {
namespace {

constexpr int64_t kMaxTokens = (int64_t)1 << 30;
constexpr int64_t kTarget = 4096;  // blocks to aim at: sixteen on each CU

int check(const void* logits, int dtype, int64_t tokens, int64_t experts, int top_k) {
  if (dtype != ACE_F32 && dtype != ACE_BF16 && dtype != ACE_F16) return ACE_EINVAL;
  if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts) return ACE_EINVAL;
  if (!logits && tokens > 0) return ACE_EINVAL;
  if (experts > balance::kMaxExperts || top_k > balance::kMaxTopK || tokens > kMaxTokens)
    return ACE_EUNSUPPORTED;
  return ACE_OK;
}

struct Launch {
  Params p;
  int c;
  unsigned blocks;
};

Launch launch_of(const void* logits, int64_t tokens, int64_t experts, int top_k, int normalize) {
  Launch l{};
  Params& p = l.p;
  p.logits = logits;
  p.tokens = tokens;
  p.experts = (int)experts;
  p.top_k = top_k;
  p.normalize = normalize != 0;
  l.c = experts <= 8 ? 8 : 16;
  while ((l.c << p.lanes_log2) < experts) ++p.lanes_log2;
  const int64_t at_once = kThreads >> p.lanes_log2;
  const int64_t most = (tokens + at_once - 1) / at_once;
  const int64_t rounds = (most + kTarget - 1) / kTarget;
  p.per_block = rounds * at_once;
  l.blocks = (unsigned)((tokens + p.per_block - 1) / p.per_block);
  return l;
}

template <typename T, int C>
void forward(const Launch& l, hipStream_t s) {
  const dim3 grid(l.blocks), block(kThreads);
  if (l.p.top_k <= 1)
    hipLaunchKernelGGL((forward_kernel<T, C, 1>), grid, block, 0, s, l.p);
  else if (l.p.top_k <= 2)
    hipLaunchKernelGGL((forward_kernel<T, C, 2>), grid, block, 0, s, l.p);
  else if (l.p.top_k <= 4)
    hipLaunchKernelGGL((forward_kernel<T, C, 4>), grid, block, 0, s, l.p);
  else if (l.p.top_k <= 8)
    hipLaunchKernelGGL((forward_kernel<T, C, 8>), grid, block, 0, s, l.p);
  else
    hipLaunchKernelGGL((forward_kernel<T, C, 16>), grid, block, 0, s, l.p);
}

template <typename T>
int launch(const Launch& l, bool backward, hipStream_t s) {
  const dim3 grid(l.blocks), block(kThreads);
  if (!backward)
    l.c == 8 ? forward<T, 8>(l, s) : forward<T, 16>(l, s);
  else if (l.c == 8)
    hipLaunchKernelGGL((backward_kernel<T, 8>), grid, block, 0, s, l.p);
  else
    hipLaunchKernelGGL((backward_kernel<T, 16>), grid, block, 0, s, l.p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ACE_OK : ACE_EHIP + (int)e;
}

int launch_type(int dtype, const Launch& l, bool backward, hipStream_t s) {
  switch (dtype) {
    case ACE_F32: return launch<float>(l, backward, s);
    case ACE_BF16: return launch<__bf16>(l, backward, s);
    default: return launch<_Float16>(l, backward, s);
  }
}

}  // namespace
}  // namespace route
}  // namespace ace

using namespace ace::route;

extern "C" {

int ace_route_forward(const void* logits, int dtype, const uint8_t* mask, int64_t tokens,
                      int64_t experts, int top_k, int normalize, int64_t* chosen, float* weights,
                      void* stream) {
  const int bad = check(logits, dtype, tokens, experts, top_k);
  if (bad) return bad;
  if (tokens == 0) return ACE_OK;
  if (!chosen || !weights) return ACE_EINVAL;
  Launch l = launch_of(logits, tokens, experts, top_k, normalize);
  l.p.mask = mask;
  l.p.chosen = chosen;
  l.p.weights = weights;
  return launch_type(dtype, l, false, static_cast<hipStream_t>(stream));
}

int ace_route_backward(const void* logits, int dtype, int64_t tokens, int64_t experts, int top_k,
                       int normalize, const int64_t* chosen, const float* weights,
                       const float* grad_weights, void* d_logits, void* stream) {
  const int bad = check(logits, dtype, tokens, experts, top_k);
  if (bad) return bad;
  if (tokens == 0) return ACE_OK;
  if (!chosen || !weights || !grad_weights || !d_logits) return ACE_EINVAL;
  Launch l = launch_of(logits, tokens, experts, top_k, normalize);
  l.p.chosen = const_cast<int64_t*>(chosen);
  l.p.weights = const_cast<float*>(weights);
  l.p.grad = grad_weights;
  l.p.d_logits = d_logits;
  return launch_type(dtype, l, true, static_cast<hipStream_t>(stream));
}

}  // extern "C"
