#include "recurrence_kernels.h"

namespace daliamd {
template void LaunchRecurrence<F16>(hipStream_t, const RecKernelArgs &);
template void LaunchRecurrenceBackward<F16>(hipStream_t, const RecKernelArgs &);
}  // namespace daliamd
