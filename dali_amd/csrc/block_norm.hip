// What stands between two blocks of a layer: norm of the block's output, gate, scaled residual, norm before the next block.
//   u = x rstd(x) w_post     v = u silu(g)     h = r + s v     n = h rstd(h) w_pre
// Backward, with z^ = z rstd(z) and <.> the mean over a row's channels:
//   dh <- dh + rstd(h) (dn w_pre - h^ <dn w_pre h^>)          dw_pre  = sum over rows of dn h^
//   dr = dh     dv = dh s                                      ds      = sum over rows of dh v
//   dg = dv u silu'(g)     du = dv silu(g)                     dw_post = sum over rows of du x^
//   dx = rstd(x) (du w_post - x^ <du w_post x^>)
#include "sequence_common.h"

namespace daliamd {

constexpr int kNormRowThreads = 256;

// the sum over a workgroup, in every thread
__device__ __forceinline__ float WorkgroupSum(float v, float *shared) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0;
  for (int w = 0; w < kNormRowThreads / 64; w++) t += shared[w];
  return t;
}

struct NormElement { float x, u, v, h, silu, dsilu; };

// the forward formulas of one channel
__device__ __forceinline__ NormElement Forward(const daliamdBlockNormArgs &p, int64_t row, int c, float rstd) {
  NormElement e;
  e.x = LoadElement(p.x, row * p.x_row + c, p.dtype);
  e.u = p.post_weight ? e.x * rstd * LoadElement(p.post_weight, c, p.weight_dtype) : e.x;
  e.silu = 1.0f, e.dsilu = 0.0f;
  if (p.gate) {
    const float g = LoadElement(p.gate, row * p.gate_row + c, p.dtype);
    float f, k;
    Logistic(g, &f, &k);
    e.silu = g * f;
    e.dsilu = f * (1.0f + g * k);
  }
  e.v = e.u * e.silu;
  e.h = p.scale ? e.v * LoadElement(p.scale, c, p.weight_dtype) : e.v;
  if (p.residual) e.h += LoadElement(p.residual, row * p.residual_row + c, p.residual_dtype);
  return e;
}

__global__ __launch_bounds__(kNormRowThreads) void BlockNormKernel(daliamdBlockNormArgs p) {
  __shared__ float shared[kNormRowThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  float rstd = 1.0f;
  if (p.post_weight) {
    float sum = 0;
    for (int c = tid; c < p.channels; c += kNormRowThreads) {
      const float x = LoadElement(p.x, row * p.x_row + c, p.dtype);
      sum += x * x;
    }
    rstd = 1.0f / sqrtf(WorkgroupSum(sum, shared) / p.channels + p.eps);
    if (p.rstd_post && tid == 0) p.rstd_post[row] = rstd;
  }
  float sum = 0;
  for (int c = tid; c < p.channels; c += kNormRowThreads) {
    const float h = Forward(p, row, c, rstd).h;
    sum += h * h;
    StoreElement(p.hidden, row * p.channels + c, p.residual ? p.residual_dtype : p.dtype, h);
  }
  if (!p.pre_weight) return;
  const float rstd2 = 1.0f / sqrtf(WorkgroupSum(sum, shared) / p.channels + p.eps);
  if (p.rstd_pre && tid == 0) p.rstd_pre[row] = rstd2;
  for (int c = tid; c < p.channels; c += kNormRowThreads)
    StoreElement(p.normed, row * p.channels + c, p.dtype, Forward(p, row, c, rstd).h * rstd2 * LoadElement(p.pre_weight, c, p.weight_dtype));
}

// the gradient of h at one channel, with the mean of the norm behind it
__device__ __forceinline__ float HiddenGradient(const daliamdBlockNormArgs &p, int64_t row, int c, float h, float rstd2, float mean) {
  float d = p.dhidden ? LoadElement(p.dhidden, row * p.dhidden_row + c, p.residual ? p.residual_dtype : p.dtype) : 0.0f;
  if (p.pre_weight && p.dnormed)
    d += rstd2 * (LoadElement(p.dnormed, row * p.dnormed_row + c, p.dtype) * LoadElement(p.pre_weight, c, p.weight_dtype) - h * rstd2 * mean);
  return d;
}

__global__ __launch_bounds__(kNormRowThreads) void BlockNormBackwardKernel(daliamdBlockNormArgs p) {
  __shared__ float shared[kNormRowThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const float rstd = p.post_weight ? p.rstd_post[row] : 1.0f, rstd2 = p.pre_weight ? p.rstd_pre[row] : 1.0f;
  float mean = 0;
  if (p.pre_weight && p.dnormed) {
    for (int c = tid; c < p.channels; c += kNormRowThreads)
      mean += LoadElement(p.dnormed, row * p.dnormed_row + c, p.dtype) * LoadElement(p.pre_weight, c, p.weight_dtype) * Forward(p, row, c, rstd).h * rstd2;
    mean = WorkgroupSum(mean, shared) / p.channels;
  }
  float mean1 = 0;
  for (int c = tid; c < p.channels; c += kNormRowThreads) {
    const NormElement e = Forward(p, row, c, rstd);
    const float dh = HiddenGradient(p, row, c, e.h, rstd2, mean);
    if (p.residual) StoreElement(p.dresidual, row * p.channels + c, p.residual_dtype, dh);
    const float dv = p.scale ? dh * LoadElement(p.scale, c, p.weight_dtype) : dh, du = dv * e.silu;
    if (p.gate) StoreElement(p.dgate, row * p.channels + c, p.dtype, dv * e.u * e.dsilu);
    if (p.post_weight) mean1 += du * LoadElement(p.post_weight, c, p.weight_dtype) * e.x * rstd;
    else StoreElement(p.dx, row * p.channels + c, p.dtype, du);
  }
  if (!p.post_weight) return;
  mean1 = WorkgroupSum(mean1, shared) / p.channels;
  for (int c = tid; c < p.channels; c += kNormRowThreads) {
    const NormElement e = Forward(p, row, c, rstd);
    const float dh = HiddenGradient(p, row, c, e.h, rstd2, mean);
    const float du = (p.scale ? dh * LoadElement(p.scale, c, p.weight_dtype) : dh) * e.silu;
    StoreElement(p.dx, row * p.channels + c, p.dtype, rstd * (du * LoadElement(p.post_weight, c, p.weight_dtype) - e.x * rstd * mean1));
  }
}

// the weights' gradients: one thread per channel goes through all rows
__global__ __launch_bounds__(kNormRowThreads) void BlockNormWeightsKernel(daliamdBlockNormArgs p, const float *means) {
  const int c = blockIdx.x * kNormRowThreads + threadIdx.x;
  if (c >= p.channels) return;
  double post = 0, scale = 0, pre = 0;
  for (int64_t row = 0; row < p.rows; row++) {
    const float rstd = p.post_weight ? p.rstd_post[row] : 1.0f, rstd2 = p.pre_weight ? p.rstd_pre[row] : 1.0f;
    const NormElement e = Forward(p, row, c, rstd);
    const float dh = HiddenGradient(p, row, c, e.h, rstd2, means[row]);
    if (p.pre_weight && p.dnormed) pre += LoadElement(p.dnormed, row * p.dnormed_row + c, p.dtype) * (e.h * rstd2);
    scale += dh * e.v;
    post += (p.scale ? dh * LoadElement(p.scale, c, p.weight_dtype) : dh) * e.silu * e.x * rstd;
  }
  if (p.post_weight) StoreElement(p.dpost_weight, c, p.weight_dtype, (float)post);
  if (p.scale) StoreElement(p.dscale, c, p.weight_dtype, (float)scale);
  if (p.pre_weight) StoreElement(p.dpre_weight, c, p.weight_dtype, (float)pre);
}

__global__ __launch_bounds__(kNormRowThreads) void BlockNormMeansKernel(daliamdBlockNormArgs p, float *means) {
  __shared__ float shared[kNormRowThreads / 64];
  const int64_t row = blockIdx.x;
  const float rstd = p.post_weight ? p.rstd_post[row] : 1.0f, rstd2 = p.pre_weight ? p.rstd_pre[row] : 1.0f;
  float mean = 0;
  if (p.pre_weight && p.dnormed)
    for (int c = threadIdx.x; c < p.channels; c += kNormRowThreads)
      mean += LoadElement(p.dnormed, row * p.dnormed_row + c, p.dtype) * LoadElement(p.pre_weight, c, p.weight_dtype) * Forward(p, row, c, rstd).h * rstd2;
  mean = WorkgroupSum(mean, shared) / p.channels;
  if (threadIdx.x == 0) means[row] = mean;
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
  plan->backward_workspace_bytes = sizeof(float) * (size_t)a.rows;
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
  {
    KernelTimer timer("BlockNormKernel", s);
    hipLaunchKernelGGL(BlockNormKernel, dim3((unsigned)args->rows), dim3(kNormRowThreads), 0, s, *args);
  }
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
  hipStream_t s = (hipStream_t)stream;
  float *means = static_cast<float *>(workspace);
  if (a.rows) {
    KernelTimer timer("BlockNormBackwardKernel", s);
    hipLaunchKernelGGL(BlockNormBackwardKernel, dim3((unsigned)a.rows), dim3(kNormRowThreads), 0, s, a);
  }
  if (a.post_weight || a.scale || a.pre_weight) {
    if (a.rows) hipLaunchKernelGGL(BlockNormMeansKernel, dim3((unsigned)a.rows), dim3(kNormRowThreads), 0, s, a, means);
    hipLaunchKernelGGL(BlockNormWeightsKernel, dim3((a.channels + kNormRowThreads - 1) / kNormRowThreads), dim3(kNormRowThreads), 0, s, a, means);
  }
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

}  // extern "C"
