// How the experts' products are cut into units of work (qx_moe.cu); host code without CUDA.
#pragma once

namespace qx {
namespace moe {

// A unit of the up projection gives 32 inner activations, one of the down projection 64 outputs (for up to eight tokens of an
// expert, or four), one that combines 1024 outputs of a token.
constexpr int kUpWidth = 32, kDownWidth = 64, kCombineWidth = 1024;

// Thread blocks that a pass has work for, of which a launch takes as many as the card has places for. `places`: experts that a
// token takes, shared ones among them; there are no more groups of tokens than pairs of token and expert.
// As many as there are up units, which then go on to the down units; where those are twice as many or more (narrow experts), as
// many as there are units at all, so that the down projections' weights come while the up projections run. One bf16 token, us, as
// many as up units | as all units (296 at most), for (up, down) units: (192, 256) 20.2 | 22.3, (128, 192) 17.8 | 18.3, f32 (144, 192)
// 21.0 | 20.6; (96, 256) 26.1 | 25.4, (64, 256) 22.2 | 18.3, (8, 64) 29.5 | 17.4, (2, 256) 198 | 24, (1, 1024) 1470 | 112; four tokens
// (128, 512) 24.5 | 21.5.
inline long long pass_blocks(long long tokens, long long places, long long dim, long long inner) {
  const long long groups = tokens * places, up = groups * (inner / kUpWidth), down = groups * ((dim + kDownWidth - 1) / kDownWidth);
  return 2 * up > down ? up : up + down + tokens * ((dim + kCombineWidth - 1) / kCombineWidth);
}

}  // namespace moe
}  // namespace qx
