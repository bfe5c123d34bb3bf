// The entry points of tokens sorted by expert and back (declared in
// include/ace_hip.h): argument checks, launch geometry, instantiations.
#include "ace_experts.hpp"

#include <type_traits>

#include "ace_hip.h"

namespace ace {
namespace experts {
namespace {

constexpr int64_t kMaxSlots = (int64_t)1 << 30;
constexpr int64_t kMaxWidth = (int64_t)1 << 20;
// A launch has fewer than 2^32 threads, in whole blocks.
constexpr int64_t kMaxWaves = ((int64_t)1 << 26) - kWaves;

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ACE_OK : ACE_EHIP + (int)e;
}

int64_t order_blocks(int64_t slots, int64_t* per_block) {
  // A slot a thread, more where that would be too many blocks.  One block alone needs one
  // launch instead of two: up to eight slots a thread (8000 slots 9.5 us instead of 10.4, 2000
  // 7.3 instead of 10.2; 16000 17 instead of 10).
  int64_t each = 1;
  if (slots <= 8 * kOrderBlock) each = slots;
  if (slots > kOrderBlock * kMaxBlocks) each = (slots + kMaxBlocks - 1) / kMaxBlocks;
  *per_block = (each + kOrderBlock - 1) / kOrderBlock * kOrderBlock;
  if (*per_block < 1) *per_block = kOrderBlock;
  const int64_t blocks = (slots + *per_block - 1) / *per_block;
  return blocks < 1 ? 1 : blocks;
}

int64_t pieces_of(int64_t width, int dtype, int deep) {
  const int64_t span = 64 * deep * (dtype == ACE_F32 ? kV<float> : kV<__bf16>);
  return (width + span - 1) / span;
}

int check(const void* in, int dtype, int64_t tokens, int64_t width, int64_t top_k,
          const int64_t* source, const int64_t* place) {
  if (dtype != ACE_F32 && dtype != ACE_BF16 && dtype != ACE_F16) return ACE_EINVAL;
  if (tokens < 0 || width < 1 || top_k < 1) return ACE_EINVAL;
  if (tokens > 0 && (!in || !source || !place)) return ACE_EINVAL;
  if (width > kMaxWidth || top_k > kMaxSlots || tokens > kMaxSlots || tokens * top_k > kMaxSlots)
    return ACE_EUNSUPPORTED;
  if (tokens * pieces_of(width, dtype, kDeepFrom) > kMaxWaves || tokens * top_k > kMaxWaves)
    return ACE_EUNSUPPORTED;
  return ACE_OK;
}

// Whether so many rows read and written exceed the last-level cache.
bool streams(int64_t rows, int64_t width, int dtype) {
  return (size_t)(rows * width) * (dtype == ACE_F32 ? 4 : 2) > kStreamBytes;
}

RowsParams params(const void* in, int dtype, int64_t tokens, int64_t width, int64_t top_k,
                  const int64_t* source, const int64_t* place, const float* weights) {
  RowsParams p{};
  p.in = in;
  p.tokens = tokens;
  p.slots = tokens * top_k;
  p.width = (int)width;
  p.top_k = (int)top_k;
  p.source = source;
  p.place = place;
  p.weights = weights;
  const int vector = dtype == ACE_F32 ? kV<float> : kV<__bf16>;
  while (p.lanes_log2 < 6 && (vector << p.lanes_log2) < width) ++p.lanes_log2;
  return p;
}

dim3 grid_of(int64_t waves) { return dim3((unsigned)((waves + kWaves - 1) / kWaves)); }

// Waves of narrow rows that take `each` of n units a lane.
int64_t narrow_waves(const RowsParams& p, int64_t n, int each) {
  const int64_t units = (int64_t)(64 >> p.lanes_log2) * each;
  return (n + units - 1) / units;
}

// Rows of at most a piece a lane are narrow: several of them share a wave.
template <typename T>
bool narrow(const RowsParams& p) {
  return p.width <= 64 * kV<T>;
}

template <typename T, bool STREAM>
void launch_to(RowsParams p, hipStream_t s) {
  const dim3 block(kBlock);
  if (narrow<T>(p)) {
    const int64_t waves = narrow_waves(p, p.slots, kMany);
    hipLaunchKernelGGL((to_narrow_kernel<T, STREAM>), grid_of(waves), block, 0, s, p);
  } else {
    hipLaunchKernelGGL((to_kernel<T, STREAM>), grid_of(p.tokens * p.pieces), block, 0, s, p);
  }
}

template <typename T, bool STREAM>
void launch_from(RowsParams p, hipStream_t s) {
  const dim3 block(kBlock);
  if (narrow<T>(p)) {
    const int64_t waves = narrow_waves(p, p.tokens, 1);
    hipLaunchKernelGGL((from_narrow_kernel<T, STREAM>), grid_of(waves), block, 0, s, p);
  } else {
    hipLaunchKernelGGL((from_kernel<T, STREAM>), grid_of(p.tokens * p.pieces), block, 0, s, p);
  }
}

template <typename T, bool ROWS, bool WEIGHTS, bool STREAM>
void launch_back(RowsParams p, hipStream_t s) {
  const dim3 block(kBlock);
  if (narrow<T>(p)) {
    const int64_t waves = narrow_waves(p, p.slots, kMany);
    hipLaunchKernelGGL((from_backward_narrow_kernel<T, ROWS, WEIGHTS, STREAM>), grid_of(waves), block, 0,
                       s, p);
  } else {
    hipLaunchKernelGGL((from_backward_kernel<T, ROWS, WEIGHTS, STREAM>), grid_of(p.slots), block, 0, s, p);
  }
}
template <typename T, bool STREAM>
void launch_back(const RowsParams& p, hipStream_t s) {
  if (p.out && p.d_weights)
    launch_back<T, true, true, STREAM>(p, s);
  else if (p.out)
    launch_back<T, true, false, STREAM>(p, s);
  else
    launch_back<T, false, true, false>(p, s);
}

// `launch` with the rows' type and whether stores go past the caches.
template <typename Launch>
int by_type(int dtype, bool past, Launch launch) {
  switch (dtype) {
    case ACE_F32: past ? launch(float{}, std::true_type{}) : launch(float{}, std::false_type{}); break;
    case ACE_BF16: past ? launch(__bf16{}, std::true_type{}) : launch(__bf16{}, std::false_type{}); break;
    default: past ? launch(_Float16{}, std::true_type{}) : launch(_Float16{}, std::false_type{});
  }
  return launched();
}

}  // namespace
}  // namespace experts
}  // namespace ace

using namespace ace::experts;

extern "C" {

size_t ace_expert_order_workspace_bytes(int64_t slots, int64_t experts) {
  if (slots < 0 || slots > kMaxSlots || experts < 1 || experts > kMaxExperts) return 0;
  int64_t per_block;
  const int64_t blocks = order_blocks(slots, &per_block);
  return blocks > 1 ? (size_t)blocks * (size_t)experts * 4 : 0;
}

int ace_expert_order(const int64_t* chosen, int64_t slots, int64_t experts, int64_t* offsets,
                     int64_t* source, int64_t* place, void* workspace, size_t workspace_bytes,
                     void* stream) {
  if (slots < 0 || experts < 1 || !offsets) return ACE_EINVAL;
  if (slots > kMaxSlots || experts > kMaxExperts) return ACE_EUNSUPPORTED;
  if (slots > 0 && (!chosen || !source || !place)) return ACE_EINVAL;
  OrderParams p{};
  p.blocks = (int)order_blocks(slots, &p.per_block);
  if (p.blocks > 1) {
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 4) return ACE_EINVAL;
    if (workspace_bytes < ace_expert_order_workspace_bytes(slots, experts)) return ACE_EWORKSPACE;
  }
  p.chosen = chosen;
  p.slots = slots;
  p.experts = (int)experts;
  p.counts = static_cast<int*>(workspace);
  p.offsets = offsets;
  p.source = source;
  p.place = place;
  const dim3 grid((unsigned)p.blocks), block(kOrderBlock);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.blocks > 1) {
    hipLaunchKernelGGL(count_kernel, grid, block, 0, s, p);
    const int rc = launched();
    if (rc) return rc;
  }
  hipLaunchKernelGGL(place_kernel, grid, block, 0, s, p);
  return launched();
}

int ace_to_experts(const void* x, int dtype, int64_t tokens, int64_t width, int64_t top_k,
                   const int64_t* source, const int64_t* place, void* rows, void* stream) {
  const int bad = check(x, dtype, tokens, width, top_k, source, place);
  if (bad) return bad;
  if (tokens == 0) return ACE_OK;
  if (!rows) return ACE_EINVAL;
  RowsParams p = params(x, dtype, tokens, width, top_k, source, place, nullptr);
  p.out = rows;
  p.pieces = (int)pieces_of(width, dtype, kDeepTo);
  const bool past = streams(p.slots + tokens, width, dtype);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, past, [&](auto t, auto past_caches) {
    launch_to<decltype(t), decltype(past_caches)::value>(p, s);
  });
}

int ace_from_experts(const void* rows, int dtype, int64_t tokens, int64_t width, int64_t top_k,
                     const int64_t* source, const int64_t* place, const float* weights, void* out,
                     void* stream) {
  const int bad = check(rows, dtype, tokens, width, top_k, source, place);
  if (bad) return bad;
  if (tokens == 0) return ACE_OK;
  if (!out) return ACE_EINVAL;
  RowsParams p = params(rows, dtype, tokens, width, top_k, source, place, weights);
  p.out = out;
  p.pieces = (int)pieces_of(width, dtype, kDeepFrom);
  const bool past = streams(p.slots + tokens, width, dtype);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, past, [&](auto t, auto past_caches) {
    launch_from<decltype(t), decltype(past_caches)::value>(p, s);
  });
}

int ace_from_experts_backward(const void* rows, const void* grad, int dtype, int64_t tokens,
                              int64_t width, int64_t top_k, const int64_t* source,
                              const int64_t* place, const float* weights, void* d_rows,
                              float* d_weights, void* stream) {
  // without the weights' gradient the rows are not read
  const int bad = check(d_weights ? rows : grad, dtype, tokens, width, top_k, source, place);
  if (bad) return bad;
  if (tokens == 0 || (!d_rows && !d_weights)) return ACE_OK;
  if (!grad) return ACE_EINVAL;
  RowsParams p = params(rows, dtype, tokens, width, top_k, source, place, weights);
  p.grad = grad;
  p.out = d_rows;
  p.d_weights = d_weights;
  const bool past = streams((d_weights ? 2 : 1) * p.slots + tokens, width, dtype);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, past, [&](auto t, auto past_caches) {
    launch_back<decltype(t), decltype(past_caches)::value>(p, s);
  });
}

}  // extern "C"
