// The token log probabilities' entry points (declared in include/ace_hip.h):
// argument checks, launch geometry, instantiations.
#include "ace_logprob.hpp"

#include "ace_hip.h"

namespace ace {
namespace logprob {
namespace {

constexpr int64_t kMaxSize = (int64_t)1 << 30;
constexpr int64_t kMaxRows = (int64_t)1 << 24;   // a launch has less than 2^32 threads
// A wave each, and whole blocks of four of them: below 2^32 threads too.
constexpr int64_t kMaxGroups = ((int64_t)1 << 26) - kBlock / 64;
constexpr int64_t kTarget = 1024;  // blocks to aim at: four on each CU

int words_of(int dtype) { return dtype == ACE_F32 ? kGroup<float> : kGroup<__bf16>; }

struct Geometry {
  int waves, parts;
  int64_t per_part;
};

Geometry geometry(int64_t rows, int64_t vocab, int dtype) {
  const int64_t group = words_of(dtype), whole = 4 * group;
  Geometry g{4, 1, vocab};
  // Rows that four waves would take in one go or less, and enough of them: a wave each.
  // Forward in us with four waves and with one: 30000 x 1000 top 5 124 / 34, 8000 x 8000
  // 48 / 37, 2000 x 8000 18 / 14; 8000 x 16000 65 / 70.
  if (rows >= kTarget && vocab <= whole) {
    g.waves = 1;
    return g;
  }
  // Parts cost a join each, so rows are cut only as far as it takes to fill the chip: in
  // us with 256, 512, 1024 and 2048 blocks to aim at, 400 x 131072 top 20 55 / 45 / 38 / -, 200 x
  // 100000 top 5 22 / 21 / 21 / 25, 1500 x 65536 top 5 46 / 46 / 46 / 55; to the nearest: 700 x
  // 32000 top 5 whole 16, in halves 19.
  int64_t parts = (kTarget + rows / 2) / rows;
  const int64_t most = (vocab + whole - 1) / whole;  // a group a wave
  if (parts > most) parts = most;
  if (parts > kMaxParts) parts = kMaxParts;
  if (parts < 1) parts = 1;
  const int64_t tile = group / kPieces;
  g.per_part = ((vocab + parts - 1) / parts + tile - 1) / tile * tile;
  g.parts = (int)((vocab + g.per_part - 1) / g.per_part);
  return g;
}

int64_t groups_of(int64_t vocab, int dtype) {
  return (vocab + words_of(dtype) - 1) / words_of(dtype);
}
bool fits(int64_t rows, int64_t vocab, int dtype) {
  return rows < kMaxRows && vocab <= kMaxSize && rows * groups_of(vocab, dtype) <= kMaxGroups;
}
bool sizes(int64_t rows, int64_t vocab, int dtype) {
  return (dtype == ACE_F32 || dtype == ACE_BF16 || dtype == ACE_F16) && rows >= 0 && vocab >= 1 &&
         fits(rows, vocab, dtype);
}

int check(const void* logits, int dtype, int64_t stride, int64_t rows, int64_t vocab, float t,
          const void* saved) {
  if (dtype != ACE_F32 && dtype != ACE_BF16 && dtype != ACE_F16) return ACE_EINVAL;
  if (rows < 0 || vocab < 1 || !(t >= 1e-3f && t <= 1e3f)) return ACE_EINVAL;
  if (!fits(rows, vocab, dtype)) return ACE_EUNSUPPORTED;
  if (rows > 0 && (!logits || !saved)) return ACE_EINVAL;
  if (stride < 0 || reinterpret_cast<uintptr_t>(saved) % 16) return ACE_EINVAL;
  const int size = dtype == ACE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return ACE_EINVAL;
  return ACE_OK;
}

Params params(const void* logits, int64_t stride, int64_t rows, int64_t vocab, float t,
              const void* saved) {
  Params p{};
  p.logits = logits;
  p.stride = stride;
  p.rows = rows;
  p.vocab = vocab;
  p.inv_t = (float)(1.0 / (double)t);
  p.scale = (float)(1.4426950408889634 / (double)t);
  p.saved = static_cast<Saved*>(const_cast<void*>(saved));
  return p;
}

template <typename T>
void launch_forward(const Params& p, int waves, hipStream_t s) {
  const int teams = kBlock / 64 / waves;
  const dim3 grid((unsigned)((p.rows * p.parts + teams - 1) / teams)), block(kBlock);
  if (waves == 1) {
    if (p.top)
      hipLaunchKernelGGL((forward_kernel<T, 1, true>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((forward_kernel<T, 1, false>), grid, block, 0, s, p);
  } else {
    if (p.top)
      hipLaunchKernelGGL((forward_kernel<T, 4, true>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((forward_kernel<T, 4, false>), grid, block, 0, s, p);
  }
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ACE_OK : ACE_EHIP + (int)e;
}

}  // namespace
}  // namespace logprob
}  // namespace ace

using namespace ace::logprob;
using ace::kStreamBytes;

extern "C" {

size_t ace_logprob_saved_bytes(int64_t rows) {
  return rows < 0 || rows >= kMaxRows ? 0 : (size_t)(rows < 1 ? 1 : rows) * sizeof(Saved);
}

size_t ace_logprob_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int top) {
  if (!sizes(rows, vocab, dtype) || rows == 0 || top < 0 || top > kMaxTop) return 0;
  const Geometry g = geometry(rows, vocab, dtype);
  return g.parts > 1 ? (size_t)rows * (size_t)g.parts * (size_t)(2 + top) * 8 : 0;
}

size_t ace_logprob_ticket_bytes(int dtype, int64_t rows, int64_t vocab) {
  if (!sizes(rows, vocab, dtype) || rows == 0) return 0;
  const Geometry g = geometry(rows, vocab, dtype);
  return g.parts > 1 ? (size_t)rows * ace::kTicketStride * 4 : 0;
}

int ace_logprob_forward(const void* logits, int dtype, int64_t stride, const int64_t* tokens,
                        int64_t rows, int64_t vocab, int64_t ignore_index, float temperature,
                        int top, void* saved, float* logprob, float* entropy, float* top_logprobs,
                        int64_t* top_tokens, void* tickets, size_t ticket_bytes, void* workspace,
                        size_t workspace_bytes, void* stream) {
  const int bad = check(logits, dtype, stride, rows, vocab, temperature, saved);
  if (bad) return bad;
  if (top < 0 || top > vocab) return ACE_EINVAL;
  if (top > kMaxTop) return ACE_EUNSUPPORTED;
  if (rows == 0) return ACE_OK;
  if (!tokens || !logprob || !entropy || (top && (!top_logprobs || !top_tokens))) return ACE_EINVAL;
  const Geometry g = geometry(rows, vocab, dtype);
  if (g.parts > 1) {
    if (!tickets || !workspace || reinterpret_cast<uintptr_t>(tickets) % 4 ||
        reinterpret_cast<uintptr_t>(workspace) % 8)
      return ACE_EINVAL;
    if (workspace_bytes < ace_logprob_workspace_bytes(dtype, rows, vocab, top) ||
        ticket_bytes < ace_logprob_ticket_bytes(dtype, rows, vocab))
      return ACE_EWORKSPACE;
  }
  Params p = params(logits, stride, rows, vocab, temperature, saved);
  p.tokens = tokens;
  p.ignore = ignore_index;
  p.top = top;
  p.parts = g.parts;
  p.per_part = g.per_part;
  p.logprob = logprob;
  p.entropy = entropy;
  p.top_logprobs = top_logprobs;
  p.top_tokens = top_tokens;
  p.part = static_cast<unsigned long long*>(workspace);
  p.tickets = static_cast<int*>(tickets);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case ACE_F32: launch_forward<float>(p, g.waves, s); break;
    case ACE_BF16: launch_forward<__bf16>(p, g.waves, s); break;
    default: launch_forward<_Float16>(p, g.waves, s);
  }
  return launched();
}

int ace_logprob_backward(const void* logits, int dtype, int64_t stride, int64_t rows, int64_t vocab,
                         float temperature, const void* saved, const float* grad_logprob,
                         const float* grad_entropy, void* d_logits, void* stream) {
  const int bad = check(logits, dtype, stride, rows, vocab, temperature, saved);
  if (bad) return bad;
  if (rows == 0) return ACE_OK;
  if (!d_logits) return ACE_EINVAL;
  Params p = params(logits, stride, rows, vocab, temperature, saved);
  p.grad_logprob = grad_logprob;
  p.grad_entropy = grad_entropy;
  p.d_logits = d_logits;
  p.tiles = (int)groups_of(vocab, dtype);
  const dim3 grid((unsigned)((rows * p.tiles + kBlock / 64 - 1) / (kBlock / 64))), block(kBlock);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool stream_stores = (size_t)(2 * rows * vocab) * (dtype == ACE_F32 ? 4 : 2) > kStreamBytes;
  const auto launch = [&](auto plain, auto streamed) {
    hipLaunchKernelGGL(stream_stores ? streamed : plain, grid, block, 0, s, p);
  };
  switch (dtype) {
    case ACE_F32: launch(backward_kernel<float, false>, backward_kernel<float, true>); break;
    case ACE_BF16: launch(backward_kernel<__bf16, false>, backward_kernel<__bf16, true>); break;
    default: launch(backward_kernel<_Float16, false>, backward_kernel<_Float16, true>);
  }
  return launched();
}

}  // extern "C"
