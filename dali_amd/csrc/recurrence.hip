// Linear recurrence along sequences, h_t = a_t h_{t-1} + b_t per channel, and its backward pass.
#include "sequence_common.h"

namespace daliamd {

constexpr int kRecThreads = 256;

struct RecArgs : daliamdRecurrenceArgs {
  float *workspace;   // backward: per-channel gradients [sequences][channels]
};

__device__ __forceinline__ int64_t RowAt(const daliamdSequenceRows &q, int64_t row, int64_t row_stride, int64_t seq_stride) {
  if (q.offsets) return row * row_stride;
  const int64_t s = (uint32_t)row / (uint32_t)q.steps;
  return s * seq_stride + (row - s * q.steps) * row_stride;
}

// a_t and the factor of x_t
__device__ __forceinline__ void Coefficients(const RecArgs &p, int64_t row, int c, float *a, float *k) {
  const float g = LoadElement(p.decay, p.per_channel ? c : RowAt(p.seq, row, p.decay_row, p.decay_seq) + c, p.decay_dtype);
  if (p.form == DALIAMD_RECURRENCE_GATE) Logistic(g, a, k);
  else *a = g, *k = 1.0f;
}

__global__ __launch_bounds__(kRecThreads) void RecurrenceForwardKernel(RecArgs p) {
  const int c = blockIdx.x * kRecThreads + threadIdx.x, s = blockIdx.y;
  if (c >= p.channels) return;
  int64_t begin, end;
  SequenceRange(p.seq, s, &begin, &end);
  double h = p.initial ? p.initial[(int64_t)s * p.channels + c] : 0.0f;
  for (int64_t row = begin; row < end; row++) {
    float a, k;
    Coefficients(p, row, c, &a, &k);
    const double x = LoadElement(p.x, RowAt(p.seq, row, p.x_row, p.x_seq) + c, p.dtype);
    if (p.saved) p.saved[row * p.channels + c] = (float)h;
    h = p.form == DALIAMD_RECURRENCE_GATE ? h + (double)k * (x - h) : (double)a * h + x;
    StoreElement(p.y, row * p.channels + c, p.dtype, (float)h);
  }
  if (p.final_state) p.final_state[(int64_t)s * p.channels + c] = (float)h;
}

__global__ __launch_bounds__(kRecThreads) void RecurrenceBackwardKernel(RecArgs p) {
  const int c = blockIdx.x * kRecThreads + threadIdx.x, s = blockIdx.y;
  if (c >= p.channels) return;
  int64_t begin, end;
  SequenceRange(p.seq, s, &begin, &end);
  double carry = p.dfinal ? p.dfinal[(int64_t)s * p.channels + c] : 0.0f, sum = 0;
  for (int64_t row = end - 1; row >= begin; row--) {
    float a, k;
    Coefficients(p, row, c, &a, &k);
    const double lambda = carry + (p.dy ? LoadElement(p.dy, RowAt(p.seq, row, p.dy_row, p.dy_seq) + c, p.dtype) : 0.0f);
    const double before = p.saved[row * p.channels + c];
    double dx = lambda, da = lambda * before;
    if (p.form == DALIAMD_RECURRENCE_GATE) {
      dx *= k;
      da = lambda * (before - LoadElement(p.x, RowAt(p.seq, row, p.x_row, p.x_seq) + c, p.dtype)) * ((double)a * k);
    }
    StoreElement(p.dx, row * p.channels + c, p.dtype, (float)dx);
    if (p.per_channel) sum += da;
    else StoreElement(p.ddecay, row * p.channels + c, p.decay_dtype, (float)da);
    carry = p.form == DALIAMD_RECURRENCE_GATE ? lambda - k * lambda : a * lambda;
  }
  if (p.dinitial) p.dinitial[(int64_t)s * p.channels + c] = (float)carry;
  if (p.per_channel) p.workspace[(int64_t)s * p.channels + c] = (float)sum;
}

// zeros where no sequence is
__global__ __launch_bounds__(kRecThreads) void RecurrenceDeadRowsKernel(RecArgs p, int backward) {
  const int64_t row = blockIdx.x;
  int64_t begin, end;
  if (FindSequence(p.seq, row, &begin, &end) >= 0) return;
  for (int c = threadIdx.x; c < p.channels; c += kRecThreads) {
    StoreElement(backward ? p.dx : p.y, row * p.channels + c, p.dtype, 0.0f);
    if (backward && !p.per_channel) StoreElement(p.ddecay, row * p.channels + c, p.decay_dtype, 0.0f);
  }
}

__global__ __launch_bounds__(kRecThreads) void RecurrenceChannelSumKernel(RecArgs p) {
  const int c = blockIdx.x * kRecThreads + threadIdx.x;
  if (c >= p.channels) return;
  double sum = 0;
  for (int s = 0; s < p.seq.sequences; s++) sum += p.workspace[(int64_t)s * p.channels + c];
  StoreElement(p.ddecay, c, p.decay_dtype, (float)sum);
}

static daliamdResult_t CheckRows(const daliamdSequenceRows &q, const char *what) {
  DALIAMD_REQUIRE(q.rows >= 0 && q.rows < ((int64_t)1 << 31) && q.sequences >= 0, DALIAMD_ERROR_OUT_OF_RANGE,
                  "%s: rows and sequences must be in [0, 2^31)", what);
  DALIAMD_REQUIRE(!(q.offsets && q.lengths), DALIAMD_ERROR_INVALID_ARGUMENT, "%s: offsets and lengths exclude each other", what);
  DALIAMD_REQUIRE(!(q.offsets || q.lengths) || q.index_dtype == DALIAMD_INT32 || q.index_dtype == DALIAMD_INT64, DALIAMD_ERROR_UNSUPPORTED,
                  "%s: offsets and lengths must be INT32 or INT64", what);
  DALIAMD_REQUIRE(q.offsets || (q.steps >= 0 && q.steps < ((int64_t)1 << 31) && q.rows == q.steps * q.sequences),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "%s: rows must be sequences * steps", what);
  DALIAMD_REQUIRE(!q.offsets || q.sequences > 0 || q.rows == 0, DALIAMD_ERROR_INVALID_ARGUMENT, "%s: rows without a sequence", what);
  return DALIAMD_SUCCESS;
}

static daliamdResult_t CheckRecurrence(const daliamdRecurrenceArgs *args, daliamdRecurrencePlan *plan) {
  DALIAMD_REQUIRE(args, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrence: NULL argument");
  const daliamdRecurrenceArgs &a = *args;
  if (daliamdResult_t r = CheckRows(a.seq, "daliamdRecurrence")) return r;
  DALIAMD_REQUIRE(a.channels >= 1 && a.channels <= (1 << 24), DALIAMD_ERROR_OUT_OF_RANGE, "daliamdRecurrence: channels must be in [1, 2^24]");
  DALIAMD_REQUIRE(IsSequenceType(a.dtype), DALIAMD_ERROR_UNSUPPORTED, "daliamdRecurrence: x must be FLOAT, FLOAT16 or BFLOAT16");
  DALIAMD_REQUIRE(a.decay_dtype == a.dtype || a.decay_dtype == DALIAMD_FLOAT, DALIAMD_ERROR_UNSUPPORTED,
                  "daliamdRecurrence: decay must have x's type or be FLOAT");
  DALIAMD_REQUIRE(a.form == DALIAMD_RECURRENCE_DECAY || a.form == DALIAMD_RECURRENCE_GATE, DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdRecurrence: unknown form %d", a.form);
  plan->saved_bytes = sizeof(float) * (size_t)a.seq.rows * a.channels;
  plan->forward_workspace_bytes = 0;
  plan->backward_workspace_bytes = a.per_channel ? sizeof(float) * (size_t)a.seq.sequences * a.channels : 0;
  return DALIAMD_SUCCESS;
}

}  // namespace daliamd

extern "C" {

daliamdResult_t daliamdRecurrenceSetup(const daliamdRecurrenceArgs *args, daliamdRecurrencePlan *plan) {
  DALIAMD_REQUIRE(plan, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceSetup: NULL argument");
  return daliamd::CheckRecurrence(args, plan);
}

daliamdResult_t daliamdRecurrenceRun(daliamdStream_t stream, const daliamdRecurrenceArgs *args, void *workspace, size_t workspace_bytes) {
  using namespace daliamd;
  daliamdRecurrencePlan plan;
  if (daliamdResult_t r = CheckRecurrence(args, &plan)) return r;
  const daliamdSequenceRows &q = args->seq;
  DALIAMD_REQUIRE(q.rows == 0 || (args->x && args->decay && args->y), DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceRun: NULL tensor");
  DALIAMD_REQUIRE(workspace_bytes >= plan.forward_workspace_bytes && (workspace || !plan.forward_workspace_bytes),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceRun: the workspace is too small");
  if (!q.sequences) return DALIAMD_SUCCESS;
  hipStream_t s = (hipStream_t)stream;
  RecArgs p;
  static_cast<daliamdRecurrenceArgs &>(p) = *args;
  p.workspace = nullptr;
  {
    KernelTimer timer("RecurrenceForwardKernel", s);
    hipLaunchKernelGGL(RecurrenceForwardKernel, dim3((p.channels + kRecThreads - 1) / kRecThreads, q.sequences), dim3(kRecThreads), 0, s, p);
  }
  if ((q.offsets || q.lengths) && q.rows) hipLaunchKernelGGL(RecurrenceDeadRowsKernel, dim3((unsigned)q.rows), dim3(kRecThreads), 0, s, p, 0);
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

daliamdResult_t daliamdRecurrenceBackwardRun(daliamdStream_t stream, const daliamdRecurrenceArgs *args, void *workspace,
                                             size_t workspace_bytes) {
  using namespace daliamd;
  daliamdRecurrencePlan plan;
  if (daliamdResult_t r = CheckRecurrence(args, &plan)) return r;
  const daliamdSequenceRows &q = args->seq;
  DALIAMD_REQUIRE((args->ddecay || (q.rows == 0 && !args->per_channel)) && (q.rows == 0 || (args->x && args->decay && args->dx && args->saved)), DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdRecurrenceBackwardRun: NULL tensor");
  DALIAMD_REQUIRE(workspace_bytes >= plan.backward_workspace_bytes && (workspace || !plan.backward_workspace_bytes),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceBackwardRun: the workspace is too small");
  hipStream_t s = (hipStream_t)stream;
  RecArgs p;
  static_cast<daliamdRecurrenceArgs &>(p) = *args;
  p.workspace = static_cast<float *>(workspace);
  const unsigned ctiles = (p.channels + kRecThreads - 1) / kRecThreads;
  if (q.sequences) {
    KernelTimer timer("RecurrenceBackwardKernel", s);
    hipLaunchKernelGGL(RecurrenceBackwardKernel, dim3(ctiles, q.sequences), dim3(kRecThreads), 0, s, p);
  }
  if (p.per_channel) hipLaunchKernelGGL(RecurrenceChannelSumKernel, dim3(ctiles), dim3(kRecThreads), 0, s, p);
  if ((q.offsets || q.lengths) && q.rows) hipLaunchKernelGGL(RecurrenceDeadRowsKernel, dim3((unsigned)q.rows), dim3(kRecThreads), 0, s, p, 1);
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

}  // extern "C"
