// How the tiles of a matrix product (ace_mma.hpp) are dealt to blocks.  Host and
// device: the host sizes buffers for what the kernels will make of it.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define ACE_DEAL_HD __host__ __device__
#else
#define ACE_DEAL_HD
#endif

namespace ace {
namespace mma {

constexpr int kStepBytes = 64;  // bytes of k in one step

// How work of `tiles` tiles, each `units` long, is dealt to `blocks` blocks: every
// tile is cut into `splits` equal parts, and block b takes parts b, b + blocks,
// and so on.  Whole tiles would leave blocks idle in the last round (or in the
// only one); cutting costs each part `overhead` units (its own start, and a partial
// result that is written), and a little more for each split where the results
// are joined.  At most `rounds` rounds, unless the whole tiles need more.
struct Deal {
  int tiles, splits;
  ACE_DEAL_HD int parts() const { return tiles * splits; }
};

// Every block works this out for itself: 32-bit divisions only, as a 64-bit one takes
// about a microsecond.
ACE_DEAL_HD inline Deal deal(int tiles, int units, int blocks, int overhead, int rounds) {
  Deal d{tiles, 1};
  const uint32_t t = tiles > 0 ? (uint32_t)tiles : 1u, u = (uint32_t)units, n = (uint32_t)blocks;
  const auto cost = [&](uint32_t s) {
    return (float)((t * s + n - 1) / n) * (float)((u + s - 1) / s + (uint32_t)overhead) +
           (overhead ? (float)s / 16.f : 0.f);
  };
  float best = cost(1);
  // a quarter, a half, and whole numbers of rounds
  for (uint32_t q = 1; q <= 4u * (uint32_t)rounds; q += q < 4 ? q : 4) {
    uint32_t s = q * n / (4 * t);
    if (s > u) s = u;
    if (s <= 1) continue;
    const float c = cost(s);
    if (c < best) {
      best = c;
      d.splits = (int)s;
    }
  }
  return d;
}

}  // namespace mma
}  // namespace ace
