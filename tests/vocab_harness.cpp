// CPU harness for the plan of the vocabulary loss (ace-kernels_amd/csrc/ace_vocab_plan.hpp):
// its tiles, grids, pieces and workspace.  Built with g++ by tests/test_vocab_plan.py
// and called through ctypes.
#include <cstdint>

#include "ace_vocab_plan.hpp"

using namespace ace;

extern "C" {

// out: score tile, dh tile, dw tile, dw in parts, pieces, rows padded, piece, dh
// blocks, dh partial tiles, dw blocks, dw partial tiles, score blocks, dscore blocks,
// bytes of the workspace forward and backward.
void vocab_plan(int es, long long n, long long h, long long v, long long* out) {
  const vocab::Plan p = vocab::make_plan(es, n, h, v);
  const long long all[] = {p.score_tile, p.dh_tile, p.dw_tile, p.dw_seg, vocab::parts(v, p.piece), p.pad, p.piece,
                           p.dh_blocks, p.dh_segs, p.dw_blocks, p.dw_segs, p.score_blocks, p.dscore_blocks,
                           (long long)vocab::forward_space(p).bytes, (long long)vocab::backward_space(p).bytes};
  for (int i = 0; i < 15; ++i) out[i] = all[i];
}

void vocab_tile(int tile, int* bm, int* bn) {
  *bm = vocab::kShape[tile].bm;
  *bn = vocab::kShape[tile].bn;
}

// Parts that the score kernels (0), the hidden gradient (1) and the weight's (2) make
// of `tiles` tiles that are `units` long.
long long vocab_parts(int kernel, int es, int tiles, int units, int blocks) {
  const mma::Deal d = kernel == 0 ? mma::deal(tiles, units, blocks, 0, vocab::kScoreRounds)
                                  : mma::deal(tiles, units, blocks, vocab::part_steps(es), vocab::kGradRounds);
  return (long long)d.tiles * d.splits;
}

// Most parts of the score kernels that the workspace holds.
long long vocab_score_parts(int es, long long n, long long h, long long v) {
  const vocab::Plan p = vocab::make_plan(es, n, h, v);
  return vocab::parts_of(p.score_blocks, vocab::kScoreRounds, vocab::parts(n, vocab::kShape[p.score_tile].bn));
}

}  // extern "C"
