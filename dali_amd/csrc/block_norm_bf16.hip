#include "block_norm_kernels.h"

namespace daliamd {
template void LaunchBlockNorm<Bf16>(hipStream_t, const daliamdBlockNormArgs &);
template void LaunchBlockNormBackward<Bf16>(hipStream_t, const daliamdBlockNormArgs &, float *, int *);
}  // namespace daliamd
