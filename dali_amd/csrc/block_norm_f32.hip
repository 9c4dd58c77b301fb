#include "block_norm_kernels.h"

namespace daliamd {
template void LaunchBlockNorm<float>(hipStream_t, const daliamdBlockNormArgs &);
template void LaunchBlockNormBackward<float>(hipStream_t, const daliamdBlockNormArgs &, float *, int *);
}  // namespace daliamd
