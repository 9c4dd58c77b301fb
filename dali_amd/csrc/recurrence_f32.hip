#include "recurrence_kernels.h"

namespace daliamd {
template void LaunchRecurrence<float>(hipStream_t, const RecKernelArgs &);
template void LaunchRecurrenceBackward<float>(hipStream_t, const RecKernelArgs &);
}  // namespace daliamd
