// C entries of the block norm: checks and workspaces; the sums over rows.  block_norm.h has the formulas.
#include "block_norm.h"

namespace daliamd {

// the sum of each column of `partial`, in a fixed order: kParts threads take every kParts-th row, then one adds them up
constexpr int kSumColumns = 64, kSumParts = 16;
__global__ __launch_bounds__(kSumColumns * kSumParts) void BlockNormWeightsKernel(daliamdBlockNormArgs p, const float *partial, int count) {
  __shared__ float part[kSumParts][kSumColumns];
  const int column = threadIdx.x % kSumColumns, k = threadIdx.x / kSumColumns;
  const int c = blockIdx.x * kSumColumns + column, which = blockIdx.y;
  void *out = which == 0 ? p.dpost_weight : which == 1 ? p.dscale : p.dpre_weight;
  if (!(which == 0 ? p.post_weight : which == 1 ? p.scale : p.pre_weight)) return;
  float sum = 0;
  if (c < p.channels) {
#pragma unroll 8
    for (int n = k; n < count; n += kSumParts) sum += partial[((int64_t)n * 3 + which) * p.channels + c];
  }
  part[k][column] = sum;
  __syncthreads();
  if (k == 0 && c < p.channels) {
    for (int n = 1; n < kSumParts; n++) sum += part[n][column];
    StoreElement(out, c, p.weight_dtype, sum);
  }
}

static daliamdResult_t CheckBlockNorm(const daliamdBlockNormArgs *args, daliamdBlockNormPlan *plan) {
  DALIAMD_REQUIRE(args, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdBlockNorm: NULL argument");
  const daliamdBlockNormArgs &a = *args;
  DALIAMD_REQUIRE(a.rows >= 0 && a.rows < ((int64_t)1 << 31), DALIAMD_ERROR_OUT_OF_RANGE, "daliamdBlockNorm: rows must be in [0, 2^31)");
  DALIAMD_REQUIRE(a.channels >= 1 && a.channels <= DALIAMD_BLOCK_NORM_MAX_CHANNELS, DALIAMD_ERROR_OUT_OF_RANGE,
                  "daliamdBlockNorm: channels must be in [1, %d]", DALIAMD_BLOCK_NORM_MAX_CHANNELS);
  DALIAMD_REQUIRE(IsSequenceType(a.dtype), DALIAMD_ERROR_UNSUPPORTED, "daliamdBlockNorm: x must be FLOAT, FLOAT16 or BFLOAT16");
  DALIAMD_REQUIRE(!a.residual || a.residual_dtype == a.dtype || a.residual_dtype == DALIAMD_FLOAT, DALIAMD_ERROR_UNSUPPORTED,
                  "daliamdBlockNorm: the residual must have x's type or be FLOAT");
  DALIAMD_REQUIRE(!(a.post_weight || a.scale || a.pre_weight) || a.weight_dtype == a.dtype || a.weight_dtype == DALIAMD_FLOAT, DALIAMD_ERROR_UNSUPPORTED,
                  "daliamdBlockNorm: the weights must have x's type or be FLOAT");
  DALIAMD_REQUIRE(a.eps >= 0, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdBlockNorm: eps must not be negative");
  plan->backward_workspace_bytes = sizeof(float) * 3 * (size_t)BackwardWorkgroups(a.rows, a.channels) * a.channels;
  return DALIAMD_SUCCESS;
}

}  // namespace daliamd

extern "C" {

daliamdResult_t daliamdBlockNormSetup(const daliamdBlockNormArgs *args, daliamdBlockNormPlan *plan) {
  DALIAMD_REQUIRE(plan, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdBlockNormSetup: NULL argument");
  return daliamd::CheckBlockNorm(args, plan);
}

daliamdResult_t daliamdBlockNormRun(daliamdStream_t stream, const daliamdBlockNormArgs *args) {
  using namespace daliamd;
  daliamdBlockNormPlan plan;
  if (daliamdResult_t r = CheckBlockNorm(args, &plan)) return r;
  if (!args->rows) return DALIAMD_SUCCESS;
  DALIAMD_REQUIRE(args->x && args->hidden && (!args->pre_weight || args->normed), DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdBlockNormRun: NULL tensor");
  hipStream_t s = (hipStream_t)stream;
  if (args->dtype == DALIAMD_FLOAT) LaunchBlockNorm<float>(s, *args);
  else if (args->dtype == DALIAMD_FLOAT16) LaunchBlockNorm<F16>(s, *args);
  else LaunchBlockNorm<Bf16>(s, *args);
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

daliamdResult_t daliamdBlockNormBackwardRun(daliamdStream_t stream, const daliamdBlockNormArgs *args, void *workspace, size_t workspace_bytes) {
  using namespace daliamd;
  daliamdBlockNormPlan plan;
  if (daliamdResult_t r = CheckBlockNorm(args, &plan)) return r;
  const daliamdBlockNormArgs &a = *args;
  DALIAMD_REQUIRE(!a.rows || (a.x && a.dx && (!a.gate || a.dgate) && (!a.residual || a.dresidual) && (!a.post_weight || a.rstd_post) &&
                              (!a.pre_weight || a.rstd_pre)), DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdBlockNormBackwardRun: NULL tensor");
  DALIAMD_REQUIRE((!a.post_weight || a.dpost_weight) && (!a.scale || a.dscale) && (!a.pre_weight || a.dpre_weight), DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdBlockNormBackwardRun: NULL gradient");
  DALIAMD_REQUIRE(workspace_bytes >= plan.backward_workspace_bytes && (workspace || !plan.backward_workspace_bytes),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdBlockNormBackwardRun: the workspace is too small");
  DALIAMD_REQUIRE((uintptr_t)workspace % 16 == 0, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdBlockNormBackwardRun: the workspace must start at a multiple of 16 bytes");
  hipStream_t s = (hipStream_t)stream;
  const bool weights = a.post_weight || a.scale || a.pre_weight;
  float *partial = weights ? static_cast<float *>(workspace) : nullptr;
  int count = 0;
  if (a.rows) {
    if (a.dtype == DALIAMD_FLOAT) LaunchBlockNormBackward<float>(s, a, partial, &count);
    else if (a.dtype == DALIAMD_FLOAT16) LaunchBlockNormBackward<F16>(s, a, partial, &count);
    else LaunchBlockNormBackward<Bf16>(s, a, partial, &count);
  }
  if (weights) {
    KernelTimer timer("BlockNormWeightsKernel", s);
    hipLaunchKernelGGL(BlockNormWeightsKernel, dim3((a.channels + kSumColumns - 1) / kSumColumns, 3), dim3(kSumColumns * kSumParts), 0, s, a,
                       partial, count);
  }
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

}  // extern "C"
