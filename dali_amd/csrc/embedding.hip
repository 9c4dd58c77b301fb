// Embedding lookup with a scale, and its gradient: the tokens' gradients summed per row of the table.
#include "sequence_common.h"

namespace daliamd {

constexpr int kEmbThreads = 256;

__global__ __launch_bounds__(kEmbThreads) void EmbeddingKernel(daliamdEmbeddingArgs p) {
  const int64_t token = blockIdx.x;
  const int64_t id = LoadIndex(p.ids, token, p.index_dtype);
  const bool in_table = id >= 0 && id < p.vocab;
  for (int c = threadIdx.x; c < p.channels; c += kEmbThreads)
    StoreElement(p.out, token * p.channels + c, p.out_dtype, in_table ? LoadElement(p.table, id * p.table_row + c, p.dtype) * p.scale : 0.0f);
}

// one workgroup per row of the table looks through all tokens
__global__ __launch_bounds__(kEmbThreads) void EmbeddingBackwardKernel(daliamdEmbeddingArgs p) {
  const int64_t id = blockIdx.x;
  for (int c = threadIdx.x; c < p.channels; c += kEmbThreads) {
    float sum = 0;
    if (id != p.padding)
      for (int64_t t = 0; t < p.tokens; t++)
        if (LoadIndex(p.ids, t, p.index_dtype) == id) sum += LoadElement(p.dout, t * p.dout_row + c, p.out_dtype);
    StoreElement(p.dtable, id * p.channels + c, p.dtype, sum * p.scale);
  }
}

static daliamdResult_t CheckEmbedding(const daliamdEmbeddingArgs *args, daliamdEmbeddingPlan *plan) {
  DALIAMD_REQUIRE(args, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdEmbedding: NULL argument");
  const daliamdEmbeddingArgs &a = *args;
  DALIAMD_REQUIRE(a.tokens >= 0 && a.tokens < ((int64_t)1 << 31) && a.vocab >= 1 && a.vocab < ((int64_t)1 << 31), DALIAMD_ERROR_OUT_OF_RANGE,
                  "daliamdEmbedding: tokens must be in [0, 2^31), vocab in [1, 2^31)");
  DALIAMD_REQUIRE(a.channels >= 1 && a.channels <= (1 << 24), DALIAMD_ERROR_OUT_OF_RANGE, "daliamdEmbedding: channels must be in [1, 2^24]");
  DALIAMD_REQUIRE(IsSequenceType(a.dtype) && IsSequenceType(a.out_dtype), DALIAMD_ERROR_UNSUPPORTED,
                  "daliamdEmbedding: table and output must be FLOAT, FLOAT16 or BFLOAT16");
  DALIAMD_REQUIRE(a.index_dtype == DALIAMD_INT32 || a.index_dtype == DALIAMD_INT64, DALIAMD_ERROR_UNSUPPORTED,
                  "daliamdEmbedding: ids must be INT32 or INT64");
  plan->backward_workspace_bytes = 0;
  return DALIAMD_SUCCESS;
}

}  // namespace daliamd

extern "C" {

daliamdResult_t daliamdEmbeddingSetup(const daliamdEmbeddingArgs *args, daliamdEmbeddingPlan *plan) {
  DALIAMD_REQUIRE(plan, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdEmbeddingSetup: NULL argument");
  return daliamd::CheckEmbedding(args, plan);
}

daliamdResult_t daliamdEmbeddingRun(daliamdStream_t stream, const daliamdEmbeddingArgs *args) {
  using namespace daliamd;
  daliamdEmbeddingPlan plan;
  if (daliamdResult_t r = CheckEmbedding(args, &plan)) return r;
  if (!args->tokens) return DALIAMD_SUCCESS;
  DALIAMD_REQUIRE(args->ids && args->table && args->out, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdEmbeddingRun: NULL tensor");
  hipStream_t s = (hipStream_t)stream;
  {
    KernelTimer timer("EmbeddingKernel", s);
    hipLaunchKernelGGL(EmbeddingKernel, dim3((unsigned)args->tokens), dim3(kEmbThreads), 0, s, *args);
  }
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

daliamdResult_t daliamdEmbeddingBackwardRun(daliamdStream_t stream, const daliamdEmbeddingArgs *args, void *workspace, size_t workspace_bytes) {
  using namespace daliamd;
  daliamdEmbeddingPlan plan;
  if (daliamdResult_t r = CheckEmbedding(args, &plan)) return r;
  DALIAMD_REQUIRE(args->dtable && (!args->tokens || (args->ids && args->dout)), DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdEmbeddingBackwardRun: NULL tensor");
  DALIAMD_REQUIRE(workspace_bytes >= plan.backward_workspace_bytes && (workspace || !plan.backward_workspace_bytes),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdEmbeddingBackwardRun: the workspace is too small");
  hipStream_t s = (hipStream_t)stream;
  {
    KernelTimer timer("EmbeddingBackwardKernel", s);
    hipLaunchKernelGGL(EmbeddingBackwardKernel, dim3((unsigned)args->vocab), dim3(kEmbThreads), 0, s, *args);
  }
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

}  // extern "C"
