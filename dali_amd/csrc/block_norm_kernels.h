// The kernels of the block norm (block_norm.h has the formulas); included by the source file of each type of x.
#ifndef DALI_AMD_CSRC_BLOCK_NORM_KERNELS_H_
#define DALI_AMD_CSRC_BLOCK_NORM_KERNELS_H_

#include "block_norm.h"

namespace daliamd {

// A row's channels stay in registers, NV pieces of 4 channels per thread: one pass over memory, whatever the number of sums.  Four
// channels - 8 bytes of a 16-bit type - rather than 16 bytes: the backward pass holds a dozen numbers per channel, and with half the
// channels per thread twice the waves fit a compute unit.
// TPR 8 to 64: so many threads per row, 256 / TPR rows in a workgroup, sums by shuffles.  TPR kWaves: a workgroup per row, of as
// many waves as the row needs (a row of 1111 channels five, not eight), sums through LDS; RowPerWave says which rows have one wave.
// Workgroups go through the rows with a stride; the backward pass keeps its sums over rows (three weights) in registers meanwhile and
// leaves one partial sum per workgroup, which BlockNormWeightsKernel adds up in a fixed order.
//
// Memory bounds it.  32768 rows of 2048 channels bf16, residual in float, all parts: forward 196 us for 939 MB (4.8 TB/s), backward
// 292 us for 1.48 GB (5.1 TB/s); a copy of 1 GiB runs at 5.1 TB/s.  Few short rows (5003 of 1111 float16, norm
// and gate: forward 14.8 us, 2.3 TB/s; backward 25.6 us, 2.2 TB/s) are bound by latency: a wave, or the waves of one row, have one row
// on its way, and the next one's loads wait for this one's sums and stores.  That 1111 is no multiple of 4 costs a tenth of it: 1112
// channels take 10 % less forward and 8 % less backward.
constexpr int kNormV = 4, kWaves = 1024, kMaxWaves = 16;
template <int TPR> constexpr int NormThreads() { return TPR == kWaves ? 1024 : 256; }

// the sum over the threads of a row, in each of them; `slot` alternates between calls: one barrier per sum, because a wave
// that writes a slot again has passed the barrier behind the last reads of it.  The places of waves that do not exist hold zeros.
struct alignas(16) NormShared { float wave[2][kMaxWaves]; };
template <int TPR> __device__ __forceinline__ void ClearShared(NormShared &shared) {
  if (TPR == kWaves && threadIdx.x < 2 * kMaxWaves) shared.wave[threadIdx.x / kMaxWaves][threadIdx.x % kMaxWaves] = 0;
  if (TPR == kWaves) __syncthreads();
}
template <int TPR> __device__ __forceinline__ float RowSum(float v, NormShared &shared, int slot) {
#pragma unroll
  for (int off = (TPR > 64 ? 64 : TPR) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if (TPR == kWaves) {
    if ((threadIdx.x & 63) == 0) shared.wave[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    const float4 *w = reinterpret_cast<const float4 *>(shared.wave[slot]);
    const float4 p = w[0], q = w[1], r = w[2], s = w[3];
    v = ((p.x + p.y) + (p.z + p.w)) + ((q.x + q.y) + (q.z + q.w)) + (((r.x + r.y) + (r.z + r.w)) + ((s.x + s.y) + (s.z + s.w)));
  }
  return v;
}

template <typename XT, int V, bool WHOLE> __device__ __forceinline__ void LoadWeights(float *w, const void *p, int dtype, const Channels<V, WHOLE> &m) {
  if (dtype == DALIAMD_FLOAT) {
    Group<float, V> g;
    m.Load(g, static_cast<const float *>(p));
#pragma unroll
    for (int j = 0; j < V; j++) w[j] = g[j];
  } else {
    Group<XT, V> g;
    m.Load(g, static_cast<const XT *>(p));
#pragma unroll
    for (int j = 0; j < V; j++) w[j] = g[j];
  }
}

// The compiler keeps the addresses of every tensor's pieces from row to row, 64 bits each, rather than compute them from a row's
// number in scalar registers and 32 bits per lane; not if it does not know that these are the same in each round.
template <int TPR> __device__ __forceinline__ int64_t AnyRow(int64_t row) {
#if defined(__AMDGCN__)
  if (TPR == kWaves) {
    int r = __builtin_amdgcn_readfirstlane((int)row);
    asm volatile("" : "+s"(r));
    return r;
  }
#endif
  return row;
}
template <int TPR> __device__ __forceinline__ int AnyLane(int lane) {
#if defined(__AMDGCN__)
  if (TPR == kWaves) asm volatile("" : "+v"(lane));
#endif
  return lane;
}

// A thread's weights: with one or two pieces of the row, in registers for all rows; with more, read again (from the L2) for each row.
template <typename XT, int V, int NV, bool WHOLE> struct NormWeights {
  static constexpr bool kKeep = NV <= 2;
  const daliamdBlockNormArgs &p;
  float kept[kKeep ? 3 : 1][kKeep ? NV : 1][V];
  __device__ __forceinline__ NormWeights(const daliamdBlockNormArgs &p_, int lane, int tpr) : p(p_) {
    if constexpr (kKeep) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
        if (p.post_weight) LoadWeights<XT, V, WHOLE>(kept[0][i], p.post_weight, p.weight_dtype, m);
        if (p.scale) LoadWeights<XT, V, WHOLE>(kept[1][i], p.scale, p.weight_dtype, m);
        if (p.pre_weight) LoadWeights<XT, V, WHOLE>(kept[2][i], p.pre_weight, p.weight_dtype, m);
      }
    }
  }
  // of piece i, which has the channels m
  template <int WHICH> __device__ __forceinline__ void Get(float (&w)[V], int i, const Channels<V, WHOLE> &m) const {
    if constexpr (kKeep) {
#pragma unroll
      for (int j = 0; j < V; j++) w[j] = kept[WHICH][i][j];
    } else {
      LoadWeights<XT, V, WHOLE>(w, WHICH == 0 ? p.post_weight : WHICH == 1 ? p.scale : p.pre_weight, p.weight_dtype, m);
    }
  }
};

template <typename XT, typename RT, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(NormThreads<TPR>()) void BlockNormKernel(daliamdBlockNormArgs p) {
  constexpr int V = kNormV, kRows = NormThreads<TPR>() / TPR;
  const int tpr = TPR == kWaves ? (int)blockDim.x : TPR;
  __shared__ NormShared shared;
  ClearShared<TPR>(shared);
  const int lane0 = TPR == kWaves ? (int)threadIdx.x : (int)threadIdx.x % TPR;
  const NormWeights<XT, V, NV, WHOLE> weights(p, lane0, tpr);
  const float inv = 1.0f / p.channels;
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < p.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = TPR == kWaves ? AnyRow<TPR>(base) : base + threadIdx.x / TPR;
    const int lane = AnyLane<TPR>(lane0);
    const bool live = kRows == 1 || row < p.rows;
    const int64_t at = live ? row : base;   // (rows of a wave that do not exist: the first one's again, not written)
    Group<XT, V> x[NV], g[NV];
    Group<RT, V> r[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
      m.Load(x[i], static_cast<const XT *>(p.x) + at * p.x_row);
      if (p.gate) m.Load(g[i], static_cast<const XT *>(p.gate) + at * p.gate_row);
      if (p.residual) m.Load(r[i], static_cast<const RT *>(p.residual) + at * p.residual_row);
    }
    float rstd = 1.0f;
    if (p.post_weight) {
      float sum = 0;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        Channels<V, WHOLE>((i * tpr + lane) * V, p.channels).Mask(x[i]);
#pragma unroll
        for (int j = 0; j < V; j++) sum = fmaf(x[i][j], x[i][j], sum);
        x[i].Repack();
      }
      rstd = 1.0f / sqrtf(RowSum<TPR>(sum, shared, 0) * inv + p.eps);
      if (p.rstd_post && lane == 0 && live) p.rstd_post[row] = rstd;
    }
    float h[NV][V], sum = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
      float post[V], scale[V];
      if (p.post_weight) weights.template Get<0>(post, i, m);
      if (p.scale) weights.template Get<1>(scale, i, m);
#pragma unroll
      for (int j = 0; j < V; j++) {
        float v = x[i][j];
        if (p.post_weight) v = v * rstd * post[j];
        if (p.gate) v *= Silu(g[i][j]);
        if (p.scale) v *= scale[j];
        if (p.residual) v += r[i][j];
        h[i][j] = v;
        sum = j >= m.begin && j < m.end ? fmaf(v, v, sum) : sum;
      }
      if (live) m.Store(static_cast<RT *>(p.hidden) + row * p.channels, h[i]);
    }
    if (p.pre_weight) {
      const float rstd2 = 1.0f / sqrtf(RowSum<TPR>(sum, shared, 1) * inv + p.eps);
      if (p.rstd_pre && lane == 0 && live) p.rstd_pre[row] = rstd2;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
        float pre[V];
        weights.template Get<2>(pre, i, m);
#pragma unroll
        for (int j = 0; j < V; j++) pre[j] = h[i][j] * rstd2 * pre[j];
        if (live) m.Store(static_cast<XT *>(p.normed) + row * p.channels, pre);
      }
    }
    if (TPR == kWaves && (!p.post_weight || !p.pre_weight)) __syncthreads();   // one sum per row: the slot is written again
  }
}

// What a row brings to its gradients, as it is in memory.
template <typename XT, typename RT, int NV, bool WHOLE> struct NormRow {
  static constexpr int V = kNormV;
  Group<XT, V> x[NV], g[NV], dn[NV];
  Group<RT, V> r[NV], dh[NV];
  float rstd, rstd2;
  __device__ __forceinline__ void Load(const daliamdBlockNormArgs &p, int64_t at, int lane, int tpr, bool second) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
      m.Load(x[i], static_cast<const XT *>(p.x) + at * p.x_row);
      if (p.gate) m.Load(g[i], static_cast<const XT *>(p.gate) + at * p.gate_row);
      if (second) {
        m.Load(dn[i], static_cast<const XT *>(p.dnormed) + at * p.dnormed_row);
        if (p.residual) m.Load(r[i], static_cast<const RT *>(p.residual) + at * p.residual_row);
      }
      if (p.dhidden) m.Load(dh[i], static_cast<const RT *>(p.dhidden) + at * p.dhidden_row);
    }
    rstd = p.post_weight ? p.rstd_post[at] : 1.0f;
    rstd2 = second ? p.rstd_pre[at] : 1.0f;
  }
  // zeros for what is another thread's: it then adds nothing to any sum
  __device__ __forceinline__ void Mask(const daliamdBlockNormArgs &p, int lane, int tpr, bool second) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
      if (second) m.Mask(dn[i]);
      if (p.dhidden) m.Mask(dh[i]);
      m.Mask(x[i]);
    }
  }
  __device__ __forceinline__ void Repack() {
#pragma unroll
    for (int i = 0; i < NV; i++) x[i].Repack(), g[i].Repack(), dn[i].Repack(), r[i].Repack(), dh[i].Repack();
  }
};

// The compiler holds a value that it has computed once for a second use; after this it computes it again from v.
template <int V> __device__ __forceinline__ void Forget(float (&v)[V]) {
#if defined(__AMDGCN__)
#pragma unroll
  for (int j = 0; j < V; j++) asm volatile("" : "+v"(v[j]));
#endif
}

// partial: [gridDim.x][3][channels], sums of the workgroup's rows for post_weight, scale and pre_weight
// Rows of more than 4096 channels have up to 16 waves with 128 registers per lane: their sums are in LDS as far as that goes (two of
// three above 8192 channels), each thread's in its own places, and of a row only what is in memory and v stay in registers between
// the sums over its channels.
template <typename XT, typename RT, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(NormThreads<TPR>()) void BlockNormBackwardKernel(daliamdBlockNormArgs p, float *partial) {
  constexpr int V = kNormV, kThreads = NormThreads<TPR>(), kRows = kThreads / TPR;
  constexpr bool kLds = NV > 1;
  const int tpr = TPR == kWaves ? (int)blockDim.x : TPR;
  __shared__ NormShared shared;
  constexpr bool kLdsPre = NV == 2;
  __shared__ float4 lds_sums[kLds ? (kLdsPre ? 3 : 2) * NV : 1][kLds ? kThreads : 1];
  ClearShared<TPR>(shared);
  const int lane0 = TPR == kWaves ? (int)threadIdx.x : (int)threadIdx.x % TPR;
  const NormWeights<XT, V, NV, WHOLE> weights(p, lane0, tpr);
  const float inv = 1.0f / p.channels;
  const bool second = p.pre_weight && p.dnormed;
  float apost[kLds ? 1 : NV][V] = {}, ascale[kLds ? 1 : NV][V] = {}, apre[kLdsPre ? 1 : NV][V] = {};
  if (kLds) {
#pragma unroll
    for (int i = 0; i < (kLdsPre ? 3 : 2) * NV; i++) lds_sums[i][threadIdx.x] = make_float4(0, 0, 0, 0);
  }
  // sum `which` (0: post_weight, 1: scale, 2: pre_weight) of piece i += a b
  auto add = [&](int which, int i, float (&reg)[V], const float (&a)[V], const float (&b)[V]) {
    if (which == 2 ? kLdsPre : kLds) {
      float4 &l = lds_sums[which * NV + i][threadIdx.x];
      float4 f = l;
      f.x = fmaf(a[0], b[0], f.x), f.y = fmaf(a[1], b[1], f.y), f.z = fmaf(a[2], b[2], f.z), f.w = fmaf(a[3], b[3], f.w);
      l = f;
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) reg[j] = fmaf(a[j], b[j], reg[j]);
    }
  };
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < p.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = TPR == kWaves ? AnyRow<TPR>(base) : base + threadIdx.x / TPR;
    const int lane = AnyLane<TPR>(lane0);
    const bool live = kRows == 1 || row < p.rows;
    NormRow<XT, RT, NV, WHOLE> t;
    t.Load(p, live ? row : base, lane, tpr, second);
    t.Mask(p, lane, tpr, second);
    const float rstd = t.rstd, rstd2 = t.rstd2;
    // v, and with the second norm the mean of dn w_pre h^
    float v[NV][V], mean2 = 0;
    auto hat = [&](int i, int j, const float (&scale)[V]) {   // h^ from v
      float e = v[i][j];
      if (p.scale) e *= scale[j];
      if (p.residual) e += t.r[i][j];
      return e * rstd2;
    };
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
      float post[V], scale[V], pre[V];
      if (p.post_weight) weights.template Get<0>(post, i, m);
      if (p.scale) weights.template Get<1>(scale, i, m);
      if (second) weights.template Get<2>(pre, i, m);
#pragma unroll
      for (int j = 0; j < V; j++) {
        float e = t.x[i][j];
        if (p.post_weight) e = e * rstd * post[j];
        if (p.gate) e *= Silu(t.g[i][j]);
        v[i][j] = e;
        if (second) mean2 = fmaf(t.dn[i][j] * pre[j], hat(i, j, scale), mean2);
      }
    }
    if (second) mean2 = RowSum<TPR>(mean2, shared, 0) * inv;
    t.Repack();
    if (kLds) {
#pragma unroll
      for (int i = 0; i < NV; i++) Forget(v[i]);
    }
    float d[NV][V], mean1 = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane) * V, p.channels);
      float post[V], scale[V], pre[V], dgate[V];
      if (p.post_weight) weights.template Get<0>(post, i, m);
      if (p.scale) weights.template Get<1>(scale, i, m);
      if (second) weights.template Get<2>(pre, i, m);
      float counted[V], hat1[V], hat2[V], counted2[V];   // (0 in rows that do not exist)
#pragma unroll
      for (int j = 0; j < V; j++) {
        float e = p.dhidden ? t.dh[i][j] : 0.0f;
        if (second) {
          hat2[j] = hat(i, j, scale);
          e += rstd2 * (t.dn[i][j] * pre[j] - hat2[j] * mean2);
          counted2[j] = live ? t.dn[i][j] : 0.0f;
        }
        d[i][j] = e;
        counted[j] = live ? e : 0.0f;
      }
      if (second) add(2, i, apre[kLdsPre ? 0 : i], counted2, hat2);
      if (p.scale) add(1, i, ascale[kLds ? 0 : i], counted, v[i]);
      if (p.residual && live) m.Store(static_cast<RT *>(p.dresidual) + row * p.channels, d[i]);
#pragma unroll
      for (int j = 0; j < V; j++) {
        float e = d[i][j];
        if (p.scale) e *= scale[j];
        hat1[j] = t.x[i][j] * rstd;
        if (p.gate) {
          float f, k;
          const float gg = t.g[i][j];
          LogisticPair(gg, &f, &k);
          dgate[j] = e * (p.post_weight ? hat1[j] * post[j] : hat1[j]) * (f * fmaf(gg, k, 1.0f));
          e *= gg * f;
        }
        counted[j] = live ? e : 0.0f;
        if (p.post_weight) {
          e *= post[j];
          mean1 = fmaf(e, hat1[j], mean1);
        }
        d[i][j] = e;
      }
      if (p.post_weight) add(0, i, apost[kLds ? 0 : i], counted, hat1);
      if (p.gate && live) m.Store(static_cast<XT *>(p.dgate) + row * p.channels, dgate);
    }
    if (p.post_weight) {
      mean1 = RowSum<TPR>(mean1, shared, 1) * inv;
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < V; j++) d[i][j] = rstd * (d[i][j] - t.x[i][j] * rstd * mean1);
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; i++) Channels<V, WHOLE>((i * tpr + lane) * V, p.channels).Store(static_cast<XT *>(p.dx) + row * p.channels, d[i]);
    }
    if (TPR == kWaves && (!p.post_weight || !second)) __syncthreads();
  }
  if (!partial) return;
  float *out = partial + (int64_t)blockIdx.x * 3 * p.channels;
  if (kRows == 1) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane0) * V, p.channels);
      if (kLds) {
        const float4 f = lds_sums[i][threadIdx.x], g = lds_sums[kLds ? NV + i : 0][threadIdx.x];
        const float post[V] = {f.x, f.y, f.z, f.w}, scale[V] = {g.x, g.y, g.z, g.w};
        if (p.post_weight) m.Store(out, post);
        if (p.scale) m.Store(out + p.channels, scale);
      } else {
        if (p.post_weight) m.Store(out, apost[kLds ? 0 : i]);
        if (p.scale) m.Store(out + p.channels, ascale[kLds ? 0 : i]);
      }
      if (kLdsPre) {
        const float4 f = lds_sums[kLdsPre ? 2 * NV + i : 0][threadIdx.x];
        const float pre[V] = {f.x, f.y, f.z, f.w};
        if (p.pre_weight) m.Store(out + 2 * p.channels, pre);
      } else if (p.pre_weight) {
        m.Store(out + 2 * p.channels, apre[kLdsPre ? 0 : i]);
      }
    }
  } else {
    // the threads with the same channels in all rows of the workgroup: the first row's adds them up
    __shared__ float rows[3][kRows > 1 ? kThreads : 1];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Channels<V, WHOLE> m((i * tpr + lane0) * V, p.channels);
      float post[V], scale[V], pre[V];
#pragma unroll
      for (int j = 0; j < V; j++) {
        __syncthreads();
        rows[0][threadIdx.x] = apost[kLds ? 0 : i][j];
        rows[1][threadIdx.x] = ascale[kLds ? 0 : i][j];
        rows[2][threadIdx.x] = apre[kLdsPre ? 0 : i][j];
        __syncthreads();
        post[j] = scale[j] = pre[j] = 0;
        if (threadIdx.x < TPR)
          for (int k = 0; k < kRows; k++) {
            post[j] += rows[0][k * TPR + threadIdx.x];
            scale[j] += rows[1][k * TPR + threadIdx.x];
            pre[j] += rows[2][k * TPR + threadIdx.x];
          }
      }
      if (threadIdx.x < TPR) {
        if (p.post_weight) m.Store(out, post);
        if (p.scale) m.Store(out + p.channels, scale);
        if (p.pre_weight) m.Store(out + 2 * p.channels, pre);
      }
    }
  }
}

template <typename XT, typename RT, int TPR, int NV> struct NormLaunch {
  static constexpr int kRows = TPR == kWaves ? 1 : 256 / TPR;
  static dim3 Threads(int channels) { return dim3(TPR == kWaves ? NormRowThreads(channels) : 256); }
  static void Forward(hipStream_t s, const daliamdBlockNormArgs &a) {
    const dim3 grid((unsigned)std::min<int64_t>((a.rows + kRows - 1) / kRows, 1 << 20)), block = Threads(a.channels);
    KernelTimer timer("BlockNormKernel", s);
    if (a.channels % kNormV == 0) hipLaunchKernelGGL((BlockNormKernel<XT, RT, TPR, NV, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((BlockNormKernel<XT, RT, TPR, NV, false>), grid, block, 0, s, a);
  }
  static void Backward(hipStream_t s, const daliamdBlockNormArgs &a, float *partial, int *count) {
    *count = (int)std::min((a.rows + kRows - 1) / kRows, BackwardWorkgroups(a.rows, a.channels));
    const dim3 grid((unsigned)*count), block = Threads(a.channels);
    KernelTimer timer("BlockNormBackwardKernel", s);
    if (a.channels % kNormV == 0) hipLaunchKernelGGL((BlockNormBackwardKernel<XT, RT, TPR, NV, true>), grid, block, 0, s, a, partial);
    else hipLaunchKernelGGL((BlockNormBackwardKernel<XT, RT, TPR, NV, false>), grid, block, 0, s, a, partial);
  }
};

template <typename XT, typename RT, typename F> static void WithShape(int channels, F f) {
  const int pieces = (channels + kNormV - 1) / kNormV;
  if (pieces <= 8) f(NormLaunch<XT, RT, 8, 1>());
  else if (pieces <= 16) f(NormLaunch<XT, RT, 16, 1>());
  else if (pieces <= 32) f(NormLaunch<XT, RT, 32, 1>());
  else if (pieces <= 64) f(NormLaunch<XT, RT, 64, 1>());
  else if (pieces <= 1024) f(NormLaunch<XT, RT, kWaves, 1>());
  else if (pieces <= 2048) f(NormLaunch<XT, RT, kWaves, 2>());
  else f(NormLaunch<XT, RT, kWaves, 4>());
}
template <typename XT, typename F> static void WithResidual(const daliamdBlockNormArgs &a, F f) {
  if (a.residual && a.residual_dtype == DALIAMD_FLOAT) WithShape<XT, float>(a.channels, f);
  else WithShape<XT, XT>(a.channels, f);
}

// A row of 257 to 1280 channels of a 16-bit type, forward, with 4096 rows and more: a wave has a whole row, up to five pieces per
// lane and no barrier.  16384 rows, norm, gate, scaled residual and norm, against several waves per row: 57 : 67 us with 1111
// channels, 20.2 : 20.8 with 512.  With 2048 rows they are equal, with 256 the other's chain of loads is shorter (8.2 : 4.1 us);
// with float several waves are faster (82 : 74 us, 1280 channels), as they are in the backward pass (50 : 25 us, 5003 rows of 1111).
constexpr int kWavePieces = 5;
constexpr int64_t kWaveRows = 4096;
template <typename XT> bool RowPerWave(const daliamdBlockNormArgs &a) {
  return sizeof(XT) == 2 && a.rows >= kWaveRows && a.channels > 64 * kNormV && a.channels <= kWavePieces * 64 * kNormV;
}
template <typename XT, typename RT> static void ForwardRowPerWave(hipStream_t s, const daliamdBlockNormArgs &a) {
  const int pieces = (a.channels + 64 * kNormV - 1) / (64 * kNormV);
  if (pieces <= 2) NormLaunch<XT, RT, 64, 2>::Forward(s, a);
  else if (pieces <= 3) NormLaunch<XT, RT, 64, 3>::Forward(s, a);
  else if (pieces <= 4) NormLaunch<XT, RT, 64, 4>::Forward(s, a);
  else NormLaunch<XT, RT, 64, kWavePieces>::Forward(s, a);
}

template <typename XT> void LaunchBlockNorm(hipStream_t s, const daliamdBlockNormArgs &a) {
  if constexpr (sizeof(XT) == 2) {
    if (RowPerWave<XT>(a)) {
      if (a.residual && a.residual_dtype == DALIAMD_FLOAT) ForwardRowPerWave<XT, float>(s, a);
      else ForwardRowPerWave<XT, XT>(s, a);
      return;
    }
  }
  WithResidual<XT>(a, [&](auto launch) { launch.Forward(s, a); });
}
template <typename XT> void LaunchBlockNormBackward(hipStream_t s, const daliamdBlockNormArgs &a, float *partial, int *count) {
  WithResidual<XT>(a, [&](auto launch) { launch.Backward(s, a, partial, count); });
}

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_BLOCK_NORM_KERNELS_H_
