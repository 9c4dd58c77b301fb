#include "block_norm_kernels.h"

namespace daliamd {
template void LaunchBlockNorm<F16>(hipStream_t, const daliamdBlockNormArgs &);
template void LaunchBlockNormBackward<F16>(hipStream_t, const daliamdBlockNormArgs &, float *, int *);
}  // namespace daliamd
