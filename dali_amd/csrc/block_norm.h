// What stands between two blocks of a layer: norm of the block's output, gate, scaled residual, norm before the next block.
//   u = x rstd(x) w_post     v = u silu(g)     h = r + s v     n = h rstd(h) w_pre
// Backward, with z^ = z rstd(z) and <.> the mean over a row's channels:
//   dh <- dh + rstd(h) (dn w_pre - h^ <dn w_pre h^>)          dw_pre  = sum over rows of dn h^
//   dr = dh     dv = dh s                                      ds      = sum over rows of dh v
//   dg = dv u silu'(g)     du = dv silu(g)                     dw_post = sum over rows of du x^
//   dx = rstd(x) (du w_post - x^ <du w_post x^>)
#ifndef DALI_AMD_CSRC_BLOCK_NORM_H_
#define DALI_AMD_CSRC_BLOCK_NORM_H_

#include <algorithm>
#include "sequence_common.h"

namespace daliamd {

// Threads of a row of more than 256 channels: whole waves, with one piece of 4 channels each up to 4096 channels, two up to 8192.
inline int NormRowThreads(int channels) {
  const int pieces = (channels + 3) / 4, each = pieces <= 1024 ? 1 : pieces <= 2048 ? 2 : 4;
  return ((pieces + each - 1) / each + 63) / 64 * 64;
}
// Workgroups of the backward pass, at most: as many as the card holds at once (four waves per SIMD), so that no second round is
// left half empty and the partial sums stay a small part of what it moves.
inline int64_t BackwardWorkgroups(int64_t rows, int channels) {
  const int threads = channels <= 256 ? 256 : NormRowThreads(channels);
  return std::min<int64_t>(rows, 256 * (1024 / threads));
}

// one source file per type of x; `count`: the workgroups that leave partial sums
template <typename XT> void LaunchBlockNorm(hipStream_t s, const daliamdBlockNormArgs &a);
template <typename XT> void LaunchBlockNormBackward(hipStream_t s, const daliamdBlockNormArgs &a, float *partial, int *count);

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_BLOCK_NORM_H_
