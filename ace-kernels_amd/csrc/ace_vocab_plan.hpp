// What follows from the sizes of a vocabulary loss alone (ace_vocab.hpp): the tiles
// and grids of its kernels, the pieces of the vocabulary, and the layout of the
// workspace.  Host arithmetic, no HIP calls.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "ace_deal.hpp"

namespace ace {
namespace vocab {

constexpr int kCus = 256;
constexpr int kPrepBlocks = 512;   // most blocks of the kernels that walk tokens
constexpr int64_t kMaxTokens = (int64_t)1 << 30, kMaxVocab = (int64_t)1 << 30;
constexpr int64_t kMaxHidden = (int64_t)1 << 20;
// Bytes of dS that one piece of the vocabulary may take: what the last-level
// cache holds.  Backward in us with 64 MB, this, 1 GB: 2048 x 1024 x 32768 455 / 409 / 410,
// 1999 x 1000 x 50001 902 / 728 / 733, 8192 x 4096 x 65536 11349 / 10552 / 10494.
constexpr int64_t kPieceBytes = (int64_t)256 << 20;

inline int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline int64_t parts(int64_t x, int64_t of) { return (x + of - 1) / of; }

// The tiles that are built: vocabulary (or hidden) x tokens (or vocabulary).  The
// largest is for 16 bits only: in float32, which the matrix cores bound, it is no
// faster than 128 x 128 (0.95 of its rate) and wastes more at the edges.
enum { kTile256 = 0, kTile128 = 1, kTile64 = 2, kTile32 = 3, kTiles = 4 };
struct TileShape {
  int bm, bn, per_cu;  // per_cu: blocks of it whose LDS fits one of the 256 CUs
};
constexpr TileShape kShape[kTiles] = {{256, 256, 1}, {128, 128, 2}, {128, 64, 3}, {128, 32, 2}};

// Rounds of blocks that tiles are cut into at most, and what a cut costs: a part of
// a gradient's tile takes its partial tile's way to memory and back, about as long
// as this many steps of k.  Forward in us with 1, 2, 4 and 8 rounds: 33000 x 512 x 8000
// 599 / 433 / 398 / 384, 12000 x 1024 x 8000 255 / 251 / 235 / 233, but 1000 x 256 x 4000 20.2 / 20.4 /
// 21.0 / 22.8.  Backward with 1, 2 and 4: 10000 x 1024 x 8000 595 / 560 / 564, 700 x 700 x 3000 80 /
// 82 / 87.  With a quarter of these steps 3300 x 1024 x 8000 takes 228 instead of 214, with
// four times them 10000 x 1024 x 8000 takes 597 instead of 560.
constexpr int kScoreRounds = 4, kGradRounds = 2;
ACE_DEAL_HD constexpr int part_steps(int es) { return es == 2 ? 24 : 8; }
constexpr int kPartBytes = 16;  // a block's share of one token's softmax

// Rates of the tiles relative to each other, measured on large products: with 16
// bits 1146, 870 and less (TFLOP/s), which small tiles lose to the traffic of LDS;
// with float32 the matrix cores alone bound them (125 to 140).
inline float rate_of(int es, int tile) {
  constexpr float half[kTiles] = {1.2f, 0.85f, 0.65f, 0.4f}, single[kTiles] = {0.f, 1.f, 0.95f, 0.85f};
  return es == 2 ? half[tile] : single[tile];
}

// The tile for m x n results: the one that takes the least time, counting what
// its edges waste.  `whole`: tiles are not cut, so that a round of blocks counts
// in full however few they are.
inline int pick_tile(int es, int64_t m, int64_t n, bool whole, int first = kTile256) {
  if (es == 4 && first == kTile256) first = kTile128;
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
inline int64_t parts_of(int blocks, int rounds, int64_t tiles) {
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

inline Plan make_plan(int es, int64_t n, int64_t h, int64_t v) {
  Plan p{};
  p.n = n;
  p.h = h;
  p.v = v;
  p.es = es;
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
  // Few tokens: what is written bounds it, and blocks that share a CU overlap.  Backward
  // in us with 128 x 128 / 256 x 256 tiles at 2048 x 50304: 64 tokens 164 / 173, 96 to 256
  // within 4 % of each other, 512 tokens 412 / 396, 700 tokens 543 / 510.
  p.dw_tile = pick_tile(p.es, p.width, p.piece, true, n > 256 ? kTile256 : kTile128);
  // The tokens are shared out as well (cut) where whole tiles leave CUs idle for long
  // enough to pay for partial tiles and a launch more: 128 x 128 tiles for less than
  // all CUs, and the more steps of k the more CUs the smallest tiles fill by themselves.
  // Where the 128 x 128 tiles alone fill most CUs, float32, which the matrix cores
  // bound, gains from a cut early, 16 bits late.  Backward in us, whole / cut:
  //   bfloat16 512 x 512 x 4000 words 55 / 70, 2048: 89 / 94, 4096: 131 / 122, 9000: 248 /
  //   202; 1500 x 64 x 1000 46 / 45, 2048: 53 / 46; 2500 x 256 x 12000 118 / 129, 9000: 306 / 310
  //   float32 1024 x 512 x 4000 151 / 157, 2048: 252 / 247; 768 x 64 x 1000 54 / 52, 1500: 80 /
  //   59; 512 x 256 x 12000 132 / 136, 1500: 310 / 281
  const int64_t tiles = parts(p.width, 128) * parts(p.piece, 128);
  const int64_t small = parts(p.width, 128) * parts(p.piece, 32), filled = small < kCus ? small : kCus;
  const bool most_cus = p.es == 4 ? 2 * tiles > kCus : 8 * tiles > 5 * kCus;
  const int64_t steps = most_cus ? (p.es == 4 ? 48 : 192) : 34 + filled / 4;
  p.dw_seg = tiles < kCus && parts(n, mma::kStepBytes / p.es) >= steps;
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
inline ForwardSpace forward_space(const Plan& p) {
  Cursor c;
  ForwardSpace s{};
  const TileShape st = kShape[p.score_tile];
  s.zeros = c.take(16);
  s.ticket = c.take(4);
  s.sums = c.take((size_t)p.join_blocks * 8);
  s.label_logit = c.take((size_t)p.n * 4);
  const size_t score_parts = parts_of(p.score_blocks, kScoreRounds, parts(p.n, st.bn));
  s.part = c.take(score_parts * st.bn * kPartBytes);
  s.rows = c.take((size_t)(p.n * p.width) * p.es);
  s.weight = c.take(p.pad ? (size_t)(p.v * p.width) * p.es : 0);
  s.bytes = c.at;
  return s;
}

struct BackwardSpace {
  size_t zeros, scale, bound, g, c, rows, weight, ds, dh, dw, bytes;
};
inline BackwardSpace backward_space(const Plan& p) {
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

}  // namespace vocab
}  // namespace ace
