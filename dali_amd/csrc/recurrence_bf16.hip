#include "recurrence_kernels.h"

namespace daliamd {
template void LaunchRecurrence<Bf16>(hipStream_t, const RecKernelArgs &);
template void LaunchRecurrenceBackward<Bf16>(hipStream_t, const RecKernelArgs &);
}  // namespace daliamd
