// The balance loss's entry points (declared in include/ace_hip.h): argument
// checks, launch geometry, instantiations.
#include "ace_balance.hpp"

#include "ace_hip.h"

namespace ace {
namespace balance {
namespace {

constexpr int64_t kMaxTokens = (int64_t)1 << 30;  // counts are 32 bits on the way
constexpr int kMaxGroups = 1 << 20;
constexpr int kTarget = 1024;  // blocks to aim at: four on each CU

struct Geometry {
  int c, lanes_log2, blocks;  // scores a lane, lanes a token, blocks a group
  int64_t per_block;
};

Geometry geometry(int64_t groups, int64_t tokens, int experts) {
  Geometry g{};
  // 8 scores a lane up to 8 experts, else 16: fewer lanes mean fewer exchanges, more
  // registers
  g.c = experts <= 8 ? 8 : 16;
  while ((g.c << g.lanes_log2) < experts) ++g.lanes_log2;
  const int64_t at_once = kThreads >> g.lanes_log2;  // tokens of a block at a time
  const int64_t most = (tokens + at_once - 1) / at_once;
  int64_t blocks = (kTarget + groups - 1) / groups;
  if (blocks > most) blocks = most;
  if (blocks > kMaxBlocks) blocks = kMaxBlocks;
  // A few rounds cost less than joining blocks: forward in us with one block a group up
  // to 1, 4 and 16 rounds, 300 x 200 tokens of 64 experts 26 / 16 / 16, 8 x 512 13 / 13 / 20, 32 x
  // 1024 16 / 16 / 34, 4 x 1024 of 16 experts 13.7 / 14.8 / 15.1.
  if (blocks < 1 || most <= 4) blocks = 1;
  const int64_t rounds = (most + blocks - 1) / blocks;
  g.per_block = (rounds > 0 ? rounds : 1) * at_once;
  g.blocks = (int)((tokens + g.per_block - 1) / g.per_block);
  if (g.blocks < 1) g.blocks = 1;
  return g;
}

struct Space {
  size_t loss, bytes, ticket_bytes;
};
Space space(int64_t groups, int experts, const Geometry& g) {
  const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
  const size_t fans = (size_t)(g.blocks + kFan - 1) / kFan;
  const size_t sets = (size_t)(groups + kFan - 1) / kFan;
  Space s{};
  const bool cut = g.blocks > 1;
  s.loss = cut ? round((size_t)groups * (g.blocks + fans) * (size_t)(experts + 1) * 8) : 0;
  s.bytes = s.loss + round(((size_t)groups + sets) * 8);
  s.ticket_bytes = ((cut ? (size_t)groups * (fans + 1) : 0) + sets + 1) * kTicketStride * 4;
  return s;
}

int check(const void* logits, int dtype, int64_t groups, int64_t tokens, int64_t experts,
          int reduction) {
  if (dtype != ACE_F32 && dtype != ACE_BF16 && dtype != ACE_F16) return ACE_EINVAL;
  if (groups < 1 || tokens < 0 || experts < 1) return ACE_EINVAL;
  if (reduction != ACE_RED_MEAN && reduction != ACE_RED_SUM && reduction != ACE_RED_NONE)
    return ACE_EINVAL;
  if (!logits && tokens > 0) return ACE_EINVAL;
  if (experts > kMaxExperts || groups > kMaxGroups || tokens > kMaxTokens) return ACE_EUNSUPPORTED;
  return ACE_OK;
}

Params params(const void* logits, const uint8_t* mask, int64_t groups, int64_t tokens,
              int64_t experts, int reduction, const Geometry& g) {
  Params p{};
  p.logits = logits;
  p.mask = mask;
  p.tokens = tokens;
  p.groups = (int)groups;
  p.experts = (int)experts;
  p.lanes_log2 = g.lanes_log2;
  p.blocks = g.blocks;
  p.per_block = g.per_block;
  p.reduction = reduction;
  return p;
}

template <typename T, int C>
void launch_forward(const Params& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.groups * p.blocks)), block(kThreads);
  if (p.top_k <= 1)
    hipLaunchKernelGGL((forward_kernel<T, C, 1>), grid, block, 0, s, p);
  else if (p.top_k <= 2)
    hipLaunchKernelGGL((forward_kernel<T, C, 2>), grid, block, 0, s, p);
  else if (p.top_k <= 4)
    hipLaunchKernelGGL((forward_kernel<T, C, 4>), grid, block, 0, s, p);
  else if (p.top_k <= 8)
    hipLaunchKernelGGL((forward_kernel<T, C, 8>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((forward_kernel<T, C, 16>), grid, block, 0, s, p);
}

template <typename T>
int launch(const Params& p, int c, bool backward, hipStream_t s) {
  const dim3 grid((unsigned)(p.groups * p.blocks)), block(kThreads);
  if (!backward)
    c == 8 ? launch_forward<T, 8>(p, s) : launch_forward<T, 16>(p, s);
  else if (c == 8)
    hipLaunchKernelGGL((backward_kernel<T, 8>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((backward_kernel<T, 16>), grid, block, 0, s, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ACE_OK : ACE_EHIP + (int)e;
}

int launch_type(int dtype, const Params& p, int c, bool backward, hipStream_t s) {
  switch (dtype) {
    case ACE_F32: return launch<float>(p, c, backward, s);
    case ACE_BF16: return launch<__bf16>(p, c, backward, s);
    default: return launch<_Float16>(p, c, backward, s);
  }
}

}  // namespace
}  // namespace balance
}  // namespace ace

using namespace ace::balance;

extern "C" {

size_t ace_balance_workspace_bytes(int64_t groups, int64_t tokens, int64_t experts) {
  if (groups < 1 || tokens < 0 || experts < 1 || experts > kMaxExperts || groups > kMaxGroups ||
      tokens > kMaxTokens)
    return 0;
  return space(groups, (int)experts, geometry(groups, tokens, (int)experts)).bytes;
}

size_t ace_balance_ticket_bytes(int64_t groups, int64_t tokens, int64_t experts) {
  if (!ace_balance_workspace_bytes(groups, tokens, experts)) return 0;
  return space(groups, (int)experts, geometry(groups, tokens, (int)experts)).ticket_bytes;
}

int ace_balance_forward(const void* logits, int dtype, const uint8_t* mask, int64_t groups,
                        int64_t tokens, int64_t experts, int top_k, int reduction, float* loss,
                        int64_t* counts, float* share, void* tickets, size_t ticket_bytes,
                        void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check(logits, dtype, groups, tokens, experts, reduction);
  if (bad) return bad;
  if (top_k < 1 || top_k > experts || !loss || !counts || !share || !tickets || !workspace)
    return ACE_EINVAL;
  if (top_k > kMaxTopK) return ACE_EUNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 || reinterpret_cast<uintptr_t>(tickets) % 4)
    return ACE_EINVAL;
  const Geometry g = geometry(groups, tokens, (int)experts);
  const Space at = space(groups, (int)experts, g);
  if (workspace_bytes < at.bytes || ticket_bytes < at.ticket_bytes) return ACE_EWORKSPACE;
  Params p = params(logits, mask, groups, tokens, experts, reduction, g);
  char* ws = static_cast<char*>(workspace);
  p.top_k = top_k;
  p.part = reinterpret_cast<unsigned long long*>(ws);
  p.part_loss = reinterpret_cast<double*>(ws + at.loss);
  p.tickets = static_cast<int*>(tickets);
  p.loss = loss;
  p.counts = counts;
  p.share = share;
  return launch_type(dtype, p, g.c, false, static_cast<hipStream_t>(stream));
}

int ace_balance_backward(const void* logits, int dtype, const uint8_t* mask, int64_t groups,
                         int64_t tokens, int64_t experts, int reduction, const float* share,
                         const float* grad_loss, void* d_logits, void* stream) {
  const int bad = check(logits, dtype, groups, tokens, experts, reduction);
  if (bad) return bad;
  if (tokens == 0) return ACE_OK;
  if (!share || !grad_loss || !d_logits) return ACE_EINVAL;
  const Geometry g = geometry(groups, tokens, (int)experts);
  Params p = params(logits, mask, groups, tokens, experts, reduction, g);
  p.share = const_cast<float*>(share);
  p.grad = grad_loss;
  p.d_logits = d_logits;
  return launch_type(dtype, p, g.c, true, static_cast<hipStream_t>(stream));
}

}  // extern "C"
