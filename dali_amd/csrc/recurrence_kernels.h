// The kernels of the linear recurrence (recurrence.h says how they work); included by the source file of each type of x.
#ifndef DALI_AMD_CSRC_RECURRENCE_KERNELS_H_
#define DALI_AMD_CSRC_RECURRENCE_KERNELS_H_

#include "recurrence.h"

namespace daliamd {

template <typename XT> constexpr int RecV() { return 16 / (int)sizeof(XT); }
template <typename XT> constexpr int RecChannels() { return kRecLanes * RecV<XT>(); }

// the rows of a thread's stretch in a tensor: blocks of `steps` rows seq apart (dense), or one block
struct RowCursor {
  int64_t s, t, steps;
  __device__ __forceinline__ RowCursor(const daliamdSequenceRows &q, int64_t row) {
    if (q.offsets) {
      s = 0, t = row, steps = q.rows;
    } else {
      s = (uint32_t)row / (uint32_t)q.steps, t = row - s * q.steps, steps = q.steps;
    }
  }
  __device__ __forceinline__ void Next() { if (++t == steps) t = 0, s++; }
  __device__ __forceinline__ int64_t At(int64_t row_stride, int64_t seq_stride) const { return s * seq_stride + t * row_stride; }
};

template <typename T, int V> __device__ __forceinline__ void LoadStep(Group<T, V> &g, const T *p, bool wide, int n) {
  if (wide && n == V) {
    LoadWide(g, p);
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) g.v[j] = j < n ? p[j] : FromFloat<T>(0.0f);
  }
}
template <typename T, int V> __device__ __forceinline__ void StoreStep(T *p, const float *f, bool wide, int n) {
  if (wide && n == V) {
    StoreWide<T, V>(p, f);
  } else {
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j < n) p[j] = FromFloat<T>(f[j]);
  }
}

// what the stretches of a tile leave behind, per wave; two of them, used in turn: one barrier per scan
template <int CH> struct RecShared {
  double a[2][kRecWaves][CH];
  float s[2][kRecWaves][CH];
  int r[2][kRecWaves];
};

// A thread's place and the scans of its workgroup.
template <typename XT> struct RecLane {
  static constexpr int V = RecV<XT>(), CH = RecChannels<XT>();
  int wave, piece, lane_c, channel, n;   // n: its channels that exist
  int turn = 0;
  RecShared<CH> &shared;
  __device__ __forceinline__ RecLane(RecShared<CH> &sh, int channels, int channel_tile) : shared(sh) {
    const int tid = threadIdx.x;
    wave = tid >> 6;
    piece = (tid & 63) / kRecLanes;
    lane_c = tid % kRecLanes * V;
    channel = channel_tile * CH + lane_c;
    n = min(max(channels - channel, 0), V);
  }
  __device__ __forceinline__ int Stretch() const { return wave * kRecPieces + piece; }

  // Scan over the stretches of the workgroup, in the order of time or (REV) against it.  a, s, r: of this thread's stretch; h: the
  // state in front of all of them -> the one behind; start: the state in front of this thread's.  MAY_RESET false: no r is set.
  // total_a / total_r: the product over the workgroup.
  template <bool REV, bool MAY_RESET>
  __device__ __forceinline__ void Scan(double (&a)[V], float (&s)[V], bool r, double (&h)[V], float (&start)[V], double *total_a, bool *total_r) {
    const int order = REV ? kRecPieces - 1 - piece : piece;
    bool any = r;
#pragma unroll
    for (int d = 1; d < kRecPieces; d <<= 1) {
      const bool have = order >= d;
      const bool before = MAY_RESET && (REV ? __shfl_down((int)any, d * kRecLanes, 64) : __shfl_up((int)any, d * kRecLanes, 64)) != 0;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const double a1 = REV ? __shfl_down(a[j], d * kRecLanes, 64) : __shfl_up(a[j], d * kRecLanes, 64);
        const float s1 = REV ? __shfl_down(s[j], d * kRecLanes, 64) : __shfl_up(s[j], d * kRecLanes, 64);
        if (have && !(MAY_RESET && any)) {
          s[j] = (float)fma(a[j], (double)s1, (double)s[j]);
          a[j] *= a1;
        }
      }
      if (MAY_RESET && have) any |= before;
    }
    turn ^= 1;
    if (order == kRecPieces - 1) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        shared.a[turn][wave][lane_c + j] = a[j];
        shared.s[turn][wave][lane_c + j] = s[j];
      }
      if (MAY_RESET && lane_c == 0) shared.r[turn][wave] = any;
    }
    // what is in front of the stretch inside its wave
    const bool front = order > 0;
    const bool any_front = MAY_RESET && (REV ? __shfl_down((int)any, kRecLanes, 64) : __shfl_up((int)any, kRecLanes, 64)) != 0;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const double a1 = REV ? __shfl_down(a[j], kRecLanes, 64) : __shfl_up(a[j], kRecLanes, 64);
      const float s1 = REV ? __shfl_down(s[j], kRecLanes, 64) : __shfl_up(s[j], kRecLanes, 64);
      a[j] = front ? a1 : 1.0;
      s[j] = front ? s1 : 0.0f;
    }
    __syncthreads();
    double in_front[V];
#pragma unroll
    for (int k = 0; k < kRecWaves; k++) {
      const int w = REV ? kRecWaves - 1 - k : k;
      const bool forget = MAY_RESET && shared.r[turn][w] != 0;
      if (MAY_RESET && total_r) *total_r |= forget;
#pragma unroll
      for (int j = 0; j < V; j++) {
        if (w == wave) in_front[j] = h[j];
        const double wa = shared.a[turn][w][lane_c + j], ws = shared.s[turn][w][lane_c + j];
        h[j] = forget ? ws : fma(wa, h[j], ws);
        if (total_a) total_a[j] *= wa;
      }
    }
#pragma unroll
    for (int j = 0; j < V; j++) start[j] = front && any_front ? s[j] : (float)fma(a[j], in_front[j], (double)s[j]);
  }
};

// Where sequences begin and end in a thread's stretch: bit k belongs to its k-th step.
struct RecEvents { uint32_t live, first, last; };
__device__ __forceinline__ RecEvents FindEvents(const daliamdSequenceRows &q, int64_t row, int64_t limit) {
  RecEvents e = {0, 0, 0};
  int64_t begin = 0, end = 0;
  for (int k = 0; k < kRecSteps && row + k < limit; k++) {
    const int64_t at = row + k;
    if (at < begin || at >= end)
      if (FindSequence(q, at, &begin, &end) < 0) continue;
    e.live |= 1u << k;
    e.first |= (uint32_t)(at == begin) << k;
    e.last |= (uint32_t)(at == end - 1) << k;
  }
  return e;
}

// The decay of a thread's channels, as the steps use it: `a` and, for gates, `k` = 1 - a.
template <typename XT, typename GT, int FORM, bool PER_CHANNEL> struct RecDecay {
  static constexpr int V = RecV<XT>();
  float k_fixed[PER_CHANNEL ? V : 1];
  double a_fixed[PER_CHANNEL ? V : 1];

  __device__ __forceinline__ RecDecay(const daliamdRecurrenceArgs &p, int channel, int n) {
    if (!PER_CHANNEL) return;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const double g = j < n ? (double)LoadElement(p.decay, channel + j, p.decay_dtype) : 0.0;
      if (FORM == DALIAMD_RECURRENCE_GATE) {
        const double t = exp(-fabs(g)), big = 1 / (1 + t);
        a_fixed[j] = g < 0 ? t * big : big;
        k_fixed[j] = (float)(g < 0 ? big : t * big);
      } else {
        a_fixed[j] = g;
        k_fixed[j] = (float)g;
      }
    }
  }
  // the number that a step works with: 1 - f, or the decay
  __device__ __forceinline__ float Coefficient(const Group<GT, V> &g, int j) const {
    if (PER_CHANNEL) return k_fixed[j];
    if (FORM == DALIAMD_RECURRENCE_DECAY) return g[j];
    float f, k;
    Logistic(g[j], &f, &k);
    return k;
  }
  __device__ __forceinline__ double Product(float coefficient, int j) const {
    if (PER_CHANNEL) return a_fixed[j];
    return FORM == DALIAMD_RECURRENCE_GATE ? 1.0 - (double)coefficient : (double)coefficient;
  }
  __device__ static __forceinline__ float Step(float coefficient, float x, float h) {
    return FORM == DALIAMD_RECURRENCE_GATE ? fmaf(coefficient, x - h, h) : fmaf(coefficient, h, x);
  }
  // M = a L
  __device__ static __forceinline__ float Back(float coefficient, float l) {
    return FORM == DALIAMD_RECURRENCE_GATE ? fmaf(-coefficient, l, l) : coefficient * l;
  }
};

template <typename XT, typename GT, bool PER_CHANNEL> struct RecTile {
  static constexpr int V = RecV<XT>();
  Group<XT, V> x[kRecSteps];
  Group<GT, V> g[PER_CHANNEL ? 1 : kRecSteps];
};

template <typename XT, typename GT, bool PER_CHANNEL, bool X>
__device__ __forceinline__ void LoadTile(RecTile<XT, GT, PER_CHANNEL> &t, const RecKernelArgs &p, int64_t row, int64_t limit, int channel, int n) {
  constexpr int V = RecV<XT>();
  if (n == 0 || row >= limit) return;
  RowCursor at(p.a.seq, row);
#pragma unroll
  for (int k = 0; k < kRecSteps; k++) {
    if (row + k < limit) {
      if (X) LoadStep<XT, V>(t.x[k], static_cast<const XT *>(p.a.x) + at.At(p.a.x_row, p.a.x_seq) + channel, p.x_wide, n);
      if (!PER_CHANNEL) LoadStep<GT, V>(t.g[k], static_cast<const GT *>(p.a.decay) + at.At(p.a.decay_row, p.a.decay_seq) + channel, p.decay_wide, n);
    }
    at.Next();
  }
}

template <int V> __device__ __forceinline__ void LoadState(float (&h)[V], const float *state, int64_t s, int channels, int channel, int n) {
#pragma unroll
  for (int j = 0; j < V; j++) h[j] = state && j < n ? state[s * channels + channel + j] : 0.0f;
}
template <int V> __device__ __forceinline__ void StoreState(float *state, const float (&h)[V], int64_t s, int channels, int channel, int n) {
  if (!state) return;
#pragma unroll
  for (int j = 0; j < V; j++)
    if (j < n) state[s * channels + channel + j] = h[j];
}

// Sequences of no steps: their state is the initial one, their initial state's gradient that of the state.
template <int V> __device__ __forceinline__ void PassEmpty(const RecKernelArgs &p, int chunk, int stretch, int channel, int n, const float *from, float *to) {
  const daliamdSequenceRows &q = p.a.seq;
  if (!to || !(q.offsets || q.lengths || q.steps == 0)) return;
  constexpr int kStretches = kRecWaves * kRecPieces;
  for (int64_t s = (int64_t)chunk * kStretches + stretch; s < q.sequences; s += (int64_t)p.chunks * kStretches) {
    int64_t begin, end;
    SequenceRange(q, (int)s, &begin, &end);
    if (begin < end) continue;
    float h[V];
    LoadState<V>(h, from, s, p.a.channels, channel, n);
    StoreState<V>(to, h, s, p.a.channels, channel, n);
  }
}

// The state in front of a chunk (REV: behind it) from the products of those before it.
template <bool REV, typename XT> __device__ __forceinline__ void JoinChunks(RecLane<XT> &lane, const RecKernelArgs &p, int chunk, int channel_tile, double (&h)[RecLane<XT>::V]) {
  constexpr int V = RecLane<XT>::V;
  const int count = REV ? p.chunks - 1 - chunk : chunk;
  if (!p.joined || count == 0) return;
  constexpr int kStretches = kRecWaves * kRecPieces;
  const int each = (count + kStretches - 1) / kStretches, base = REV ? chunk + 1 : 0;
  const int from = base + lane.Stretch() * each, to = min(from + each, base + count);
  double a[V];
  float s[V], start[V];
  bool r = false;
#pragma unroll
  for (int j = 0; j < V; j++) a[j] = 1.0, s[j] = 0.0f;
#pragma unroll 4
  for (int k = from; k < to; k++) {
    const int c = REV ? to - 1 - (k - from) : k;
    const bool forget = p.chunk_r[(int64_t)c * p.channel_tiles + channel_tile] != 0;
    r |= forget;
#pragma unroll
    for (int j = 0; j < V; j++) {
      if (j >= lane.n) continue;
      const int64_t at = (int64_t)c * p.a.channels + lane.channel + j;
      const double ca = p.chunk_a[at];
      const float cs = p.chunk_s[at];
      s[j] = forget ? cs : (float)fma(ca, (double)s[j], (double)cs);
      a[j] *= ca;
    }
  }
  lane.template Scan<REV, true>(a, s, r, h, start, nullptr, nullptr);
}

template <typename XT, typename GT, int FORM, bool PER_CHANNEL> struct RecForward {
  static constexpr int V = RecV<XT>();
  typedef RecDecay<XT, GT, FORM, PER_CHANNEL> Decay;
  typedef RecTile<XT, GT, PER_CHANNEL> Tile;

  // (A, S, R) of a thread's stretch; `c`: the steps' coefficients for the second time
  template <bool EVENTS>
  __device__ static __forceinline__ bool Compose(const RecKernelArgs &p, const Decay &decay, const Tile &t, const RecEvents &e, int64_t row, int channel,
                                                 int n, float (&c)[kRecSteps][V], double (&a)[V], float (&s)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) a[j] = 1.0, s[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) {
      if (EVENTS && !(e.live >> k & 1)) continue;
      if (EVENTS && (e.first >> k & 1)) {
        int64_t begin, end;
        const int q = FindSequence(p.a.seq, row + k, &begin, &end);
        LoadState<V>(s, p.a.initial, q, p.a.channels, channel, n);
      }
#pragma unroll
      for (int j = 0; j < V; j++) {
        c[k][j] = decay.Coefficient(t.g[PER_CHANNEL ? 0 : k], j);
        a[j] *= decay.Product(c[k][j], j);
        s[j] = Decay::Step(c[k][j], t.x[k][j], s[j]);
      }
    }
    return EVENTS && e.first != 0;
  }

  template <bool EVENTS>
  __device__ static __forceinline__ void Process(const RecKernelArgs &p, RecLane<XT> &lane, const Decay &decay, const Tile &t, int64_t row, int64_t limit,
                                                 int sequence, bool ends, double (&h)[V]) {
    RecEvents e = {};
    if (EVENTS) e = FindEvents(p.a.seq, row, limit);
    float c[kRecSteps][V], s[V], state[V];
    double a[V];
    const bool r = Compose<EVENTS>(p, decay, t, e, row, lane.channel, lane.n, c, a, s);
    lane.template Scan<false, EVENTS>(a, s, r, h, state, nullptr, nullptr);
    if (lane.n == 0) return;
    XT *y = static_cast<XT *>(p.a.y) + row * p.a.channels + lane.channel;
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) {
      if (EVENTS && row + k >= limit) break;
      if (EVENTS && !(e.live >> k & 1)) {
        const float zero[V] = {};
        StoreStep<XT, V>(y + (int64_t)k * p.a.channels, zero, p.out_wide, lane.n);
        continue;
      }
      int64_t begin, end;
      if (EVENTS && (e.first >> k & 1)) LoadState<V>(state, p.a.initial, FindSequence(p.a.seq, row + k, &begin, &end), p.a.channels, lane.channel, lane.n);
#pragma unroll
      for (int j = 0; j < V; j++) state[j] = Decay::Step(c[k][j], t.x[k][j], state[j]);
      StoreStep<XT, V>(y + (int64_t)k * p.a.channels, state, p.out_wide, lane.n);
      if (EVENTS && (e.last >> k & 1)) StoreState<V>(p.a.final_state, state, FindSequence(p.a.seq, row + k, &begin, &end), p.a.channels, lane.channel, lane.n);
    }
    if (!EVENTS && ends && lane.Stretch() == kRecWaves * kRecPieces - 1) StoreState<V>(p.a.final_state, state, sequence, p.a.channels, lane.channel, lane.n);
  }
};

template <typename XT, typename GT, int FORM, bool PER_CHANNEL>
__global__ __launch_bounds__(kRecThreads) void RecurrenceForwardKernel(RecKernelArgs p) {
  typedef RecForward<XT, GT, FORM, PER_CHANNEL> Op;
  constexpr int V = RecV<XT>();
  __shared__ RecShared<RecChannels<XT>()> shared;
  const int channel_tile = blockIdx.x % p.channel_tiles, chunk = blockIdx.x / p.channel_tiles;
  RecLane<XT> lane(shared, p.a.channels, channel_tile);
  const typename Op::Decay decay(p.a, lane.channel, lane.n);
  double h[V] = {};
  JoinChunks<false>(lane, p, chunk, channel_tile, h);
  const int64_t first = chunk * p.chunk_rows, limit = min(first + p.chunk_rows, p.a.seq.rows);
  int64_t begin = 0, end = 0;
  int sequence = -1;
  typename Op::Tile now, next;
  const int64_t offset = (int64_t)lane.Stretch() * kRecSteps;
  LoadTile<XT, GT, PER_CHANNEL, true>(next, p, first + offset, limit, lane.channel, lane.n);
  int tile = 0;
  for (int64_t row = first; row < limit; row += kRecTile, tile++) {
    now = next;
    LoadTile<XT, GT, PER_CHANNEL, true>(next, p, row + kRecTile + offset, limit, lane.channel, lane.n);
    if (row < begin || row >= end) sequence = FindSequence(p.a.seq, row, &begin, &end);
    const bool interior = sequence >= 0 && row + kRecTile <= end && row + kRecTile <= limit;
    if (interior && row == begin) {
      float state[V];
      LoadState<V>(state, p.a.initial, sequence, p.a.channels, lane.channel, lane.n);
#pragma unroll
      for (int j = 0; j < V; j++) h[j] = state[j];
    }
    if (p.a.saved && lane.Stretch() == 0) {
      float state[V];
#pragma unroll
      for (int j = 0; j < V; j++) state[j] = (float)h[j];
      StoreState<V>(p.a.saved, state, (int64_t)chunk * p.tiles + tile, p.a.channels, lane.channel, lane.n);
    }
    if (interior) Op::template Process<false>(p, lane, decay, now, row + offset, limit, sequence, row + kRecTile == end, h);
    else Op::template Process<true>(p, lane, decay, now, row + offset, limit, 0, false, h);
  }
  PassEmpty<V>(p, chunk, lane.Stretch(), lane.channel, lane.n, p.a.initial, p.a.final_state);
}

// (A, S, R) of a thread's stretch against time; dy NULL: zeros
template <typename XT, typename GT, int FORM, bool PER_CHANNEL, bool EVENTS>
__device__ __forceinline__ bool ComposeBack(const RecKernelArgs &p, const RecDecay<XT, GT, FORM, PER_CHANNEL> &decay, const Group<XT, RecV<XT>()> (&dy)[kRecSteps],
                                            const float (&c)[kRecSteps][RecV<XT>()], const RecEvents &e, int64_t row, int channel, int n,
                                            double (&a)[RecV<XT>()], float (&s)[RecV<XT>()]) {
  constexpr int V = RecV<XT>();
#pragma unroll
  for (int j = 0; j < V; j++) a[j] = 1.0, s[j] = 0.0f;
#pragma unroll
  for (int k = kRecSteps - 1; k >= 0; k--) {
    if (EVENTS && !(e.live >> k & 1)) continue;
    if (EVENTS && (e.last >> k & 1)) {
      int64_t begin, end;
      LoadState<V>(s, p.a.dfinal, FindSequence(p.a.seq, row + k, &begin, &end), p.a.channels, channel, n);
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
      a[j] *= decay.Product(c[k][j], j);
      s[j] = RecDecay<XT, GT, FORM, PER_CHANNEL>::Back(c[k][j], s[j] + dy[k][j]);
    }
  }
  return EVENTS && e.last != 0;
}

template <typename XT> __device__ __forceinline__ void LoadGradient(Group<XT, RecV<XT>()> (&dy)[kRecSteps], const RecKernelArgs &p, int64_t row, int64_t limit,
                                                                    int channel, int n) {
  constexpr int V = RecV<XT>();
  RowCursor at(p.a.seq, row < limit ? row : 0);
#pragma unroll
  for (int k = 0; k < kRecSteps; k++) {
    if (p.a.dy && n && row + k < limit) {
      LoadStep<XT, V>(dy[k], static_cast<const XT *>(p.a.dy) + at.At(p.a.dy_row, p.a.dy_seq) + channel, p.dy_wide, n);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) dy[k].v[j] = FromFloat<XT>(0.0f);
    }
    at.Next();
  }
}

// the product of each chunk, in the order of time or (REV) against it
template <typename XT, typename GT, int FORM, bool PER_CHANNEL, bool REV>
__global__ __launch_bounds__(kRecThreads) void RecurrenceChunkKernel(RecKernelArgs p) {
  typedef RecForward<XT, GT, FORM, PER_CHANNEL> Op;
  constexpr int V = RecV<XT>();
  __shared__ RecShared<RecChannels<XT>()> shared;
  const int channel_tile = blockIdx.x % p.channel_tiles, chunk = blockIdx.x / p.channel_tiles;
  RecLane<XT> lane(shared, p.a.channels, channel_tile);
  const typename Op::Decay decay(p.a, lane.channel, lane.n);
  const int64_t first = chunk * p.chunk_rows, limit = min(first + p.chunk_rows, p.a.seq.rows);
  double h[V] = {}, total[V];
  bool any = false;
#pragma unroll
  for (int j = 0; j < V; j++) total[j] = 1.0;
  int64_t begin = 0, end = 0;
  for (int tile = 0; tile < p.tiles; tile++) {
    const int64_t row = first + (int64_t)(REV ? p.tiles - 1 - tile : tile) * kRecTile;
    if (row >= limit) continue;
    const int64_t at = row + (int64_t)lane.Stretch() * kRecSteps;
    typename Op::Tile t;
    Group<XT, V> dy[kRecSteps];
    LoadTile<XT, GT, PER_CHANNEL, !REV>(t, p, at, limit, lane.channel, lane.n);
    if (REV) LoadGradient(dy, p, at, limit, lane.channel, lane.n);
    const RecEvents e = FindEvents(p.a.seq, at, limit);
    float c[kRecSteps][V], s[V], start[V];
    double a[V];
    bool r;
    if (REV) {
#pragma unroll
      for (int k = 0; k < kRecSteps; k++)
#pragma unroll
        for (int j = 0; j < V; j++) c[k][j] = decay.Coefficient(t.g[PER_CHANNEL ? 0 : k], j);
      r = ComposeBack<XT, GT, FORM, PER_CHANNEL, true>(p, decay, dy, c, e, at, lane.channel, lane.n, a, s);
    } else {
      r = Op::template Compose<true>(p, decay, t, e, at, lane.channel, lane.n, c, a, s);
    }
    lane.template Scan<REV, true>(a, s, r, h, start, total, &any);
  }
  if (lane.Stretch() == 0) {
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j < lane.n) {
        const int64_t at = (int64_t)chunk * p.a.channels + lane.channel + j;
        p.chunk_a[at] = total[j];
        p.chunk_s[at] = (float)h[j];
      }
    if (threadIdx.x == 0) p.chunk_r[(int64_t)chunk * p.channel_tiles + channel_tile] = any;
  }
}

template <typename XT, typename GT, int FORM, bool PER_CHANNEL> struct RecBackward {
  static constexpr int V = RecV<XT>();
  typedef RecForward<XT, GT, FORM, PER_CHANNEL> Forward;
  typedef typename Forward::Decay Decay;
  typedef typename Forward::Tile Tile;

  // in_front: the state in front of the tile; m: M behind it -> M of its first step
  template <bool EVENTS>
  __device__ static __forceinline__ void Process(const RecKernelArgs &p, RecLane<XT> &lane, const Decay &decay, const Tile &t, const Group<XT, V> (&dy)[kRecSteps],
                                                 int64_t row, int64_t limit, int sequence, bool begins, double (&in_front)[V], double (&m)[V], float (&sum)[V]) {
    RecEvents e = {};
    if (EVENTS) e = FindEvents(p.a.seq, row, limit);
    float c[kRecSteps][V], s[V], state[V], back[V];
    double a[V];
    bool r = Forward::template Compose<EVENTS>(p, decay, t, e, row, lane.channel, lane.n, c, a, s);
    lane.template Scan<false, EVENTS>(a, s, r, in_front, state, nullptr, nullptr);
    r = ComposeBack<XT, GT, FORM, PER_CHANNEL, EVENTS>(p, decay, dy, c, e, row, lane.channel, lane.n, a, s);
    lane.template Scan<true, EVENTS>(a, s, r, m, back, nullptr, nullptr);
    if (lane.n == 0) return;
    int64_t begin, end;
    float before[kRecSteps][V];
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) {
      if (EVENTS && !(e.live >> k & 1)) continue;
      if (EVENTS && (e.first >> k & 1)) LoadState<V>(state, p.a.initial, FindSequence(p.a.seq, row + k, &begin, &end), p.a.channels, lane.channel, lane.n);
#pragma unroll
      for (int j = 0; j < V; j++) {
        before[k][j] = state[j];
        state[j] = Decay::Step(c[k][j], t.x[k][j], state[j]);
      }
    }
#pragma unroll
    for (int k = kRecSteps - 1; k >= 0; k--) {
      if (EVENTS && row + k >= limit) continue;
      float dx[V] = {}, dg[V] = {};
      const bool live = !EVENTS || (e.live >> k & 1);
      if (live) {
        if (EVENTS && (e.last >> k & 1)) LoadState<V>(back, p.a.dfinal, FindSequence(p.a.seq, row + k, &begin, &end), p.a.channels, lane.channel, lane.n);
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float l = back[j] + dy[k][j];
          if (FORM == DALIAMD_RECURRENCE_GATE) {
            dx[j] = c[k][j] * l;
            dg[j] = Decay::Back(c[k][j], dx[j]) * (before[k][j] - t.x[k][j]);   // (1 - f) L, then times f
          } else {
            dx[j] = l;
            dg[j] = l * before[k][j];
          }
          if (PER_CHANNEL) sum[j] += dg[j];
          back[j] = Decay::Back(c[k][j], l);
        }
        if (EVENTS && (e.first >> k & 1)) StoreState<V>(p.a.dinitial, back, FindSequence(p.a.seq, row + k, &begin, &end), p.a.channels, lane.channel, lane.n);
      }
      const int64_t at = (row + k) * p.a.channels + lane.channel;
      StoreStep<XT, V>(static_cast<XT *>(p.a.dx) + at, dx, p.out_wide, lane.n);
      if (!PER_CHANNEL) StoreStep<GT, V>(static_cast<GT *>(p.a.ddecay) + at, dg, p.decay_out_wide, lane.n);
    }
    if (!EVENTS && begins && lane.Stretch() == 0) StoreState<V>(p.a.dinitial, back, sequence, p.a.channels, lane.channel, lane.n);
  }
};

template <typename XT, typename GT, int FORM, bool PER_CHANNEL>
__global__ __launch_bounds__(kRecThreads) void RecurrenceBackwardKernel(RecKernelArgs p) {
  typedef RecBackward<XT, GT, FORM, PER_CHANNEL> Op;
  constexpr int V = RecV<XT>();
  __shared__ RecShared<RecChannels<XT>()> shared;
  const int channel_tile = blockIdx.x % p.channel_tiles, chunk = blockIdx.x / p.channel_tiles;
  RecLane<XT> lane(shared, p.a.channels, channel_tile);
  const typename Op::Decay decay(p.a, lane.channel, lane.n);
  double m[V] = {};
  JoinChunks<true>(lane, p, chunk, channel_tile, m);
  const int64_t first = chunk * p.chunk_rows, limit = min(first + p.chunk_rows, p.a.seq.rows);
  const int64_t offset = (int64_t)lane.Stretch() * kRecSteps;
  float sum[V] = {};
  int64_t begin = 0, end = 0;
  int sequence = -1;
  for (int tile = first < limit ? (int)((limit - first + kRecTile - 1) / kRecTile) - 1 : -1; tile >= 0; tile--) {
    const int64_t row = first + (int64_t)tile * kRecTile;
    typename Op::Tile t;
    Group<XT, V> dy[kRecSteps];
    float saved[V];
    LoadTile<XT, GT, PER_CHANNEL, true>(t, p, row + offset, limit, lane.channel, lane.n);
    LoadGradient(dy, p, row + offset, limit, lane.channel, lane.n);
    LoadState<V>(saved, p.a.saved, (int64_t)chunk * p.tiles + tile, p.a.channels, lane.channel, lane.n);
    if (row < begin || row >= end) sequence = FindSequence(p.a.seq, row, &begin, &end);
    const bool interior = sequence >= 0 && row + kRecTile <= end && row + kRecTile <= limit;
    if (interior && row + kRecTile == end) {
      float state[V];
      LoadState<V>(state, p.a.dfinal, sequence, p.a.channels, lane.channel, lane.n);
#pragma unroll
      for (int j = 0; j < V; j++) m[j] = state[j];
    }
    double in_front[V];
#pragma unroll
    for (int j = 0; j < V; j++) in_front[j] = saved[j];
    if (interior) Op::template Process<false>(p, lane, decay, t, dy, row + offset, limit, sequence, row == begin, in_front, m, sum);
    else Op::template Process<true>(p, lane, decay, t, dy, row + offset, limit, 0, false, in_front, m, sum);
  }
  PassEmpty<V>(p, chunk, lane.Stretch(), lane.channel, lane.n, p.a.dfinal, p.a.dinitial);
  if (PER_CHANNEL) {
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int off = kRecLanes; off < 64; off <<= 1) sum[j] += __shfl_xor(sum[j], off, 64);
    }
    __syncthreads();
    if (lane.piece == 0) {
#pragma unroll
      for (int j = 0; j < V; j++) shared.s[0][lane.wave][lane.lane_c + j] = sum[j];
    }
    __syncthreads();
    if (lane.Stretch() == 0) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        float total = 0;
        for (int w = 0; w < kRecWaves; w++) total += shared.s[0][w][lane.lane_c + j];
        if (j < lane.n) p.partial[(int64_t)chunk * p.a.channels + lane.channel + j] = total;
      }
    }
  }
}

// A few steps per sequence (one token for each of many): a thread has 16 bytes of channels of one sequence.
template <typename XT, typename GT, int FORM, bool PER_CHANNEL>
__global__ __launch_bounds__(kRecThreads) void RecurrenceStepKernel(RecKernelArgs p) {
  constexpr int V = RecV<XT>();
  const int groups = (p.a.channels + V - 1) / V;
  const int64_t id = (int64_t)blockIdx.x * kRecThreads + threadIdx.x;
  const int64_t s = (uint32_t)id / (uint32_t)groups;
  if (s >= p.a.seq.sequences) return;
  const int channel = (int)(id - s * groups) * V, n = min(p.a.channels - channel, V);
  const RecDecay<XT, GT, FORM, PER_CHANNEL> decay(p.a, channel, n);
  int64_t begin, end;
  SequenceRange(p.a.seq, (int)s, &begin, &end);
  const int64_t steps = p.a.seq.steps, length = end - begin;
  float h[V];
  LoadState<V>(h, p.a.initial, s, p.a.channels, channel, n);
  for (int64_t t = 0; t < steps; t++) {
    XT *y = static_cast<XT *>(p.a.y) + (s * steps + t) * p.a.channels + channel;
    if (t < length) {
      Group<XT, V> x;
      Group<GT, V> g;
      LoadStep<XT, V>(x, static_cast<const XT *>(p.a.x) + s * p.a.x_seq + t * p.a.x_row + channel, p.x_wide, n);
      if (!PER_CHANNEL) LoadStep<GT, V>(g, static_cast<const GT *>(p.a.decay) + s * p.a.decay_seq + t * p.a.decay_row + channel, p.decay_wide, n);
#pragma unroll
      for (int j = 0; j < V; j++) h[j] = RecDecay<XT, GT, FORM, PER_CHANNEL>::Step(decay.Coefficient(g, j), x[j], h[j]);
      StoreStep<XT, V>(y, h, p.out_wide, n);
    } else {
      const float zero[V] = {};
      StoreStep<XT, V>(y, zero, p.out_wide, n);
    }
  }
  StoreState<V>(p.a.final_state, h, s, p.a.channels, channel, n);
}

template <typename XT, typename GT, int FORM, bool PER_CHANNEL> struct RecLaunch {
  static void Forward(hipStream_t s, const RecKernelArgs &p) {
    const daliamdSequenceRows &q = p.a.seq;
    if (p.few_steps) {
      constexpr int V = RecV<XT>();
      const int64_t threads = (int64_t)q.sequences * ((p.a.channels + V - 1) / V);
      KernelTimer timer("RecurrenceStepKernel", s);
      hipLaunchKernelGGL((RecurrenceStepKernel<XT, GT, FORM, PER_CHANNEL>), dim3((unsigned)((threads + kRecThreads - 1) / kRecThreads)), dim3(kRecThreads), 0, s, p);
      return;
    }
    const dim3 grid((unsigned)p.chunks * p.channel_tiles);
    if (p.joined) {
      KernelTimer timer("RecurrenceChunkKernel", s);
      hipLaunchKernelGGL((RecurrenceChunkKernel<XT, GT, FORM, PER_CHANNEL, false>), grid, dim3(kRecThreads), 0, s, p);
    }
    KernelTimer timer("RecurrenceForwardKernel", s);
    hipLaunchKernelGGL((RecurrenceForwardKernel<XT, GT, FORM, PER_CHANNEL>), grid, dim3(kRecThreads), 0, s, p);
  }
  static void Backward(hipStream_t s, const RecKernelArgs &p) {
    const dim3 grid((unsigned)p.chunks * p.channel_tiles);
    if (p.joined) {
      KernelTimer timer("RecurrenceChunkKernel", s);
      hipLaunchKernelGGL((RecurrenceChunkKernel<XT, GT, FORM, PER_CHANNEL, true>), grid, dim3(kRecThreads), 0, s, p);
    }
    KernelTimer timer("RecurrenceBackwardKernel", s);
    hipLaunchKernelGGL((RecurrenceBackwardKernel<XT, GT, FORM, PER_CHANNEL>), grid, dim3(kRecThreads), 0, s, p);
  }
};
template <typename XT, typename GT, bool PER_CHANNEL, typename F> static void WithForm(const daliamdRecurrenceArgs &a, F f) {
  if (a.form == DALIAMD_RECURRENCE_GATE) f(RecLaunch<XT, GT, DALIAMD_RECURRENCE_GATE, PER_CHANNEL>());
  else f(RecLaunch<XT, GT, DALIAMD_RECURRENCE_DECAY, PER_CHANNEL>());
}
template <typename XT, typename F> static void WithDecay(const daliamdRecurrenceArgs &a, F f) {
  if (a.per_channel) WithForm<XT, float, true>(a, f);
  else if (a.decay_dtype == a.dtype) WithForm<XT, XT, false>(a, f);
  else WithForm<XT, float, false>(a, f);
}

template <typename XT> void LaunchRecurrence(hipStream_t s, const RecKernelArgs &p) {
  WithDecay<XT>(p.a, [&](auto launch) { launch.Forward(s, p); });
}
template <typename XT> void LaunchRecurrenceBackward(hipStream_t s, const RecKernelArgs &p) {
  WithDecay<XT>(p.a, [&](auto launch) { launch.Backward(s, p); });
}

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_RECURRENCE_KERNELS_H_
