// The kernels of the linear recurrence (recurrence.h says how they work); included by the source file of each type of x.
#ifndef DALI_AMD_CSRC_RECURRENCE_KERNELS_H_
#define DALI_AMD_CSRC_RECURRENCE_KERNELS_H_

#include "recurrence.h"

namespace daliamd {

template <typename XT> constexpr int RecV() { return kRecBytes / (int)sizeof(XT); }
template <typename XT> constexpr int RecChannels() { return kRecLanes * RecV<XT>(); }

// The steps of a thread's stretch in a tensor, one group of channels each.  Loads are not conditional - steps behind the last row
// read that row again, lanes without channels the last ones - because a load under a condition is waited for where the
// condition ends: the 16 or 24 of a tile would come one after the other.  Rows: blocks of `steps` rows seq apart, or one block.
// `plain`: a whole tile of one block: a base in scalar registers, a step per row.
template <typename T, int V>
__device__ __forceinline__ void LoadSteps(Group<T, V> (&g)[kRecSteps], const void *base, const daliamdSequenceRows &q, int first, int stretch, int limit,
                                          int64_t row_stride, int64_t seq_stride, const Channels<V> &own, bool plain) {
  if (plain && !own.narrow) {
    const char *p = static_cast<const char *>(base) + (int64_t)first * row_stride * (int)sizeof(T);
    const uint32_t offset = (uint32_t)(stretch * kRecSteps * (int)row_stride + own.base) * (uint32_t)sizeof(T);
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) LoadWide(g[k], reinterpret_cast<const T *>(p + (int64_t)k * row_stride * (int)sizeof(T) + offset));
    return;
  }
  const int row = min(first + stretch * kRecSteps, limit - 1);
  const int steps = (int)(q.offsets ? q.rows : q.steps), s = q.offsets ? 0 : (int)((uint32_t)row / (uint32_t)steps);
  int t = row - s * steps;
  const T *p = static_cast<const T *>(base) + s * seq_stride + t * row_stride;
  const int64_t next_block = seq_stride - (steps - 1) * row_stride;
#pragma unroll
  for (int k = 0; k < kRecSteps; k++) {
    own.Load(g[k], p);
    const bool wrap = ++t == steps;
    p += row + k + 1 < limit ? (wrap ? next_block : row_stride) : 0;
    if (wrap) t = 0;
  }
}

// what the stretches of a tile leave behind, per wave
template <int CH> struct RecShared {
  double a[kRecWaves][CH];
  float s[kRecWaves][CH];
  int r[kRecWaves];
  float front[CH];              // the state in front of the tile
};

// A product of decays, kept finite: of more than 1 in size, hundreds of them pass the 64 bits' range, and infinity times a state of 0
// (or a decay of 0) is NaN.  Any other state is infinite in 32 bits long before.  (Those of one stretch are within the range.)
// GATES: none is more than 1.
template <bool GATES> __device__ __forceinline__ double Bounded(double a) { return GATES ? a : fmin(fmax(a, -1e300), 1e300); }

// A stretch's place in its wave's scan: what is in front of it inside the wave.
template <int V> struct RecFront {
  double a[V];
  float s[V];
  bool r;
};

// A thread's place and the scans of its workgroup.
template <typename XT> struct RecLane {
  static constexpr int V = RecV<XT>(), CH = RecChannels<XT>();
  int wave, piece, lane_c;
  Channels<V> own;   // (where the row ends inside a group, its first channels are computed by two threads alike, and written by one)
  __device__ __forceinline__ RecLane(int channels, int channel_tile) : own(channel_tile * CH + (int)threadIdx.x % kRecLanes * V, channels) {
    const int tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    piece = (tid & 63) / kRecLanes;
    lane_c = tid % kRecLanes * V;
  }
  __device__ __forceinline__ bool Idle() const { return own.begin >= own.end; }
  __device__ __forceinline__ int Stretch() const { return wave * kRecPieces + piece; }

  // Scan over the stretches of a wave, in the order of time or (REV) against it; a, s, r: of this thread's stretch.  The wave's
  // own product goes to `shared`.  MAY_RESET false: no r is set.
  template <bool REV, bool MAY_RESET, bool GATES>
  __device__ __forceinline__ RecFront<V> ScanWave(RecShared<CH> &shared, double (&a)[V], float (&s)[V], bool r) const {
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
          a[j] = Bounded<GATES>(a[j] * a1);
        }
      }
      if (MAY_RESET && have) any |= before;
    }
    if (order == kRecPieces - 1) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        shared.a[wave][lane_c + j] = a[j];
        shared.s[wave][lane_c + j] = s[j];
      }
      if (lane_c == 0) shared.r[wave] = any;
    }
    RecFront<V> front;
    const bool have = order > 0;
    front.r = MAY_RESET && (REV ? __shfl_down((int)any, kRecLanes, 64) : __shfl_up((int)any, kRecLanes, 64)) != 0 && have;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const double a1 = REV ? __shfl_down(a[j], kRecLanes, 64) : __shfl_up(a[j], kRecLanes, 64);
      const float s1 = REV ? __shfl_down(s[j], kRecLanes, 64) : __shfl_up(s[j], kRecLanes, 64);
      front.a[j] = have ? a1 : 1.0;
      front.s[j] = have ? s1 : 0.0f;
    }
    return front;
  }

  // The state in front of this thread's stretch, from the one in front of the tile.
  template <bool REV, bool MAY_RESET>
  __device__ __forceinline__ void Start(const RecShared<CH> &shared, const RecFront<V> &front, const float (&in)[V], float (&start)[V]) const {
    double h[V];
#pragma unroll
    for (int j = 0; j < V; j++) h[j] = in[j];
#pragma unroll
    for (int k = 0; k < kRecWaves - 1; k++) {
      const int w = REV ? kRecWaves - 1 - k : k;
      if (REV ? w <= wave : w >= wave) break;
      const bool forget = MAY_RESET && shared.r[w] != 0;
#pragma unroll
      for (int j = 0; j < V; j++) h[j] = forget ? (double)shared.s[w][lane_c + j] : fma(shared.a[w][lane_c + j], h[j], (double)shared.s[w][lane_c + j]);
    }
#pragma unroll
    for (int j = 0; j < V; j++) start[j] = front.r ? front.s[j] : (float)fma(front.a[j], h[j], (double)front.s[j]);
  }
};

// ---- the chain -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void Say(uint64_t *word, uint32_t value) {
  __hip_atomic_store(word, ((uint64_t)1 << 32) | value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t Hear(const uint64_t *word) { return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ bool Said(uint64_t word) { return (word >> 32) != 0; }
__device__ __forceinline__ float Value(uint64_t word) { return BitsToFloat((uint32_t)word); }

// For one channel of the workgroup's tile (`place`: its place among all tiles' channels): finds the state in front of the tile and says what is behind it.  a, s, r: of the
// whole tile; `known`: nothing in front counts but `state`.  Returns the state in front.
template <bool REV, bool GATES> __device__ __forceinline__ float Chain(const RecKernelArgs &p, int tile, int64_t width, int place, double a, float s, bool r, bool known, float state) {
  uint64_t *mine = p.words + ((int64_t)tile * width + place) * kRecWords;
  const bool joint = (REV ? p.tiles - 1 - tile : tile) % kRecGroup == kRecGroup - 1;
  if (r || known) {
    Say(mine, __builtin_bit_cast(uint32_t, r ? s : (float)fma(a, (double)state, (double)s)));
    if (known) return state;
  } else if (!joint) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, a);
    Say(mine + 1, __builtin_bit_cast(uint32_t, s));
    Say(mine + 2, (uint32_t)(bits >> 32));
    Say(mine + 3, (uint32_t)bits);
  }
  // the product of the tiles between the one looked at and this one
  double pa = 1.0;
  float ps = 0.0f;
  constexpr int kAhead = 4;
  const int64_t step = (REV ? 1 : -1) * kRecWords * width;
  const int last = REV ? p.tiles - 1 : 0;
  const uint64_t *at = mine + step;
  int left = REV ? last - tile : tile;       // tiles in front of this one
  for (bool found = false; !found && left > 0;) {
    uint64_t w[kAhead][kRecWords];
#pragma unroll
    for (int k = 0; k < kAhead; k++)
#pragma unroll
      for (int i = 0; i < kRecWords; i++) w[k][i] = k < left ? Hear(at + k * step + i) : 0;
    int moved = 0;
    bool go = true;
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      if (!go) continue;
      if (Said(w[k][0])) {
        ps = (float)fma(pa, (double)Value(w[k][0]), (double)ps);
        found = true;
        go = false;
      } else if (Said(w[k][1]) && Said(w[k][2]) && Said(w[k][3])) {
        ps = (float)fma(pa, (double)Value(w[k][1]), (double)ps);
        pa = Bounded<GATES>(pa * __builtin_bit_cast(double, (uint64_t)(uint32_t)w[k][2] << 32 | (uint32_t)w[k][3]));
        moved++;
      } else {
        go = false;
      }
    }
    at += moved * step;
    left -= moved;
    if (!found && moved == 0) __builtin_amdgcn_s_sleep(1);
  }
  if (joint && !r) Say(mine, __builtin_bit_cast(uint32_t, (float)fma(a, (double)ps, (double)s)));
  return ps;
}

// The state in front of the tile into shared.front: by the first threads, one per channel.  initial: of `sequence` where that
// begins with the tile (REV: ends with it); `needs`: the row in front belongs to the same sequence.
template <bool REV, bool GATES, typename XT>
__device__ __forceinline__ void FindFront(const RecKernelArgs &p, RecShared<RecChannels<XT>()> &shared, int tile, int channel_tile, bool needs,
                                          const float *initial, int sequence) {
  constexpr int CH = RecChannels<XT>();
  if (threadIdx.x >= CH) return;
  const int first = channel_tile * CH + (int)threadIdx.x / RecV<XT>() * RecV<XT>();
  const Channels<RecV<XT>()> own(first, p.a.channels);
  const int channel = own.base + (int)threadIdx.x % RecV<XT>();
  double a = 1.0;
  float s = 0.0f;
  bool r = false;
#pragma unroll
  for (int k = 0; k < kRecWaves; k++) {
    const int w = REV ? kRecWaves - 1 - k : k;
    const double wa = shared.a[w][threadIdx.x];
    const float ws = shared.s[w][threadIdx.x];
    const bool forget = shared.r[w] != 0;
    s = forget ? ws : (float)fma(wa, (double)s, (double)ws);
    a = Bounded<GATES>(a * wa);
    r |= forget;
  }
  const float state = initial && sequence >= 0 && channel < p.a.channels ? initial[(int64_t)sequence * p.a.channels + channel] : 0.0f;
  shared.front[threadIdx.x] = p.chained ? Chain<REV, GATES>(p, tile, (int64_t)p.channel_tiles * CH, channel_tile * CH + (int)threadIdx.x, a, s, r, !needs, state) : state;
}

// the workgroup's tile: in the order of the chain
template <bool REV> __device__ __forceinline__ void TakeTile(const RecKernelArgs &p, int *slot, int *tile, int *channel_tile) {
  int id = blockIdx.x;
  if (p.chained) {
    if (threadIdx.x == 0) *slot = (int)atomicAdd(p.ticket, 1u);
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(*slot);
  }
  *channel_tile = id % p.channel_tiles;
  *tile = id / p.channel_tiles;
  if (REV) *tile = p.tiles - 1 - *tile;
}

// Where sequences begin and end in a tile, by row: the sequence, or -1.
struct RecMarks {
  int first[kRecTile], last[kRecTile];
  uint8_t live[kRecTile];
};
// ... in a thread's stretch: bit k belongs to its k-th step.
struct RecEvents {
  uint32_t live, first, last;
  const int *first_of, *last_of;
};

// The last sequence that begins at or before `row` (0 if none does), found by a whole wave: 64 places at a time.
__device__ __forceinline__ int FindInWave(const daliamdSequenceRows &q, int row) {
  const int lane = threadIdx.x & 63;
  int base = 0, count = q.sequences;
  while (count > 1) {
    const int stride = (count + 63) / 64, at = lane * stride;
    const bool before = at < count && LoadIndex(q.offsets, base + min(at, count - 1), q.index_dtype) <= row;
    const int found = __popcll(__ballot(before));
    if (found == 0) break;
    base += (found - 1) * stride;
    count = min(stride, count - (found - 1) * stride);
  }
  return base;
}

// What a workgroup knows of its rows: those of one sequence alone, or not.
struct RecPlace {
  int row, limit, begin, end, sequence, near;   // (the same in every thread)  near: packed, a sequence not behind the first row's
  bool interior;
  __device__ __forceinline__ RecPlace(const RecKernelArgs &p, int tile) {
    row = tile * p.tile_rows;
    limit = min(row + p.tile_rows, (int)p.a.seq.rows);
  }
  __device__ __forceinline__ void Find(const RecKernelArgs &p) {
    const daliamdSequenceRows &q = p.a.seq;
    begin = end = near = 0;
    sequence = -1;
    if (row < limit) {
      near = q.offsets ? FindInWave(q, row) : row / (int)q.steps;
      SequenceRange(q, near, &begin, &end);
      begin = __builtin_amdgcn_readfirstlane(begin);
      end = __builtin_amdgcn_readfirstlane(end);
      near = __builtin_amdgcn_readfirstlane(near);
      if (begin <= row && row < end) sequence = near;
    }
    interior = sequence >= 0 && row + kRecTile <= min(end, limit);
  }
};

// Fills the marks of a tile that is not interior; all threads of the workgroup.
__device__ __forceinline__ void Mark(const RecKernelArgs &p, const RecPlace &place, RecMarks &marks) {
  const daliamdSequenceRows &q = p.a.seq;
  const int tid = threadIdx.x, row = place.row + tid;
  static_assert(kRecThreads >= kRecTile, "a thread per row");
  if (q.offsets) {
    if (tid < kRecTile) {
      marks.first[tid] = marks.last[tid] = -1;
      marks.live[tid] = row < place.limit && row >= ClampRow(LoadIndex(q.offsets, 0, q.index_dtype), q.rows) &&
                        row < ClampRow(LoadIndex(q.offsets, q.sequences, q.index_dtype), q.rows);
    }
    __syncthreads();
    for (int s = place.near + tid; s < q.sequences && place.row < place.limit; s += kRecThreads) {
      int begin, end;
      SequenceRange(q, s, &begin, &end);
      if (begin >= place.limit) break;
      if (begin == end) continue;
      if (begin >= place.row) marks.first[begin - place.row] = s;
      if (end > place.row && end <= place.limit) marks.last[end - 1 - place.row] = s;
    }
  } else if (tid < kRecTile) {
    int begin = 0, end = 0;
    const int s = row < place.limit ? FindDenseSequence(q, row, &begin, &end) : -1;
    marks.live[tid] = s >= 0;
    marks.first[tid] = s >= 0 && row == begin ? s : -1;
    marks.last[tid] = s >= 0 && row == end - 1 ? s : -1;
  }
  __syncthreads();
}
__device__ __forceinline__ RecEvents EventsOf(const RecMarks &marks, int stretch) {
  const int at = stretch * kRecSteps;
  RecEvents e = {0, 0, 0, marks.first + at, marks.last + at};
#pragma unroll
  for (int k = 0; k < kRecSteps; k++) {
    e.live |= (uint32_t)marks.live[at + k] << k;
    e.first |= (uint32_t)(marks.first[at + k] >= 0) << k;
    e.last |= (uint32_t)(marks.last[at + k] >= 0) << k;
  }
  e.first &= e.live, e.last &= e.live;
  return e;
}

// The decay of a thread's channels, as the steps use it.  A step works with one number, its coefficient: the decay, or of a gate
// the smaller one of f and 1 - f, negative where that is f (`shut`).  So a gate that is nearly open takes 1 - f of the input, and one that is
// nearly shut leaves f of the state, both exactly: h + (1 - f)(x - h) is x + f (h - x).
// COMPARE: whether a gate is shut is found by comparison.  Otherwise its sign is spread over a register, which is no shorter but leaves
// the scalar registers alone: the backward pass, which asks four times, spills (8 x 4096 x 2048 bf16, 197 : 205 us; ragged prompts
// 144 : 166; the forward pass 129 : 127, with float gates 82 : 78).
template <typename XT, typename GT, int FORM, bool PER_CHANNEL, bool COMPARE> struct RecDecay {
  static constexpr int V = RecV<XT>();
  static constexpr bool kGate = FORM == DALIAMD_RECURRENCE_GATE;
  float c_fixed[PER_CHANNEL ? V : 1];
  double a_fixed[PER_CHANNEL ? V : 1];

  __device__ __forceinline__ RecDecay(const daliamdRecurrenceArgs &p, const Channels<V> &own) {
    if (!PER_CHANNEL) return;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const double g = j < own.end ? (double)LoadElement(p.decay, own.base + j, p.decay_dtype) : 0.0;
      if (kGate) {
        const double t = exp(-fabs(g)), big = 1 / (1 + t);
        a_fixed[j] = g < 0 ? t * big : big;
        c_fixed[j] = copysignf((float)(t * big), (float)g);
      } else {
        a_fixed[j] = g;
        c_fixed[j] = (float)g;
      }
    }
  }
  __device__ __forceinline__ float Coefficient(const Group<GT, V> &g, int j) const {
    if (PER_CHANNEL) return c_fixed[j];
    if (!kGate) return g[j];
    return SmallerOfLogistic<sizeof(GT) == 4>(g[j]);
  }
  // all bits set if f is the smaller one (-0 as well)
  __device__ static __forceinline__ uint32_t Shut(float coefficient) {
    uint32_t m = (uint32_t)(__builtin_bit_cast(int32_t, coefficient) >> 31);
#if defined(__AMDGCN__)
    if (!COMPARE) asm("" : "+v"(m));   // (the compiler would make a comparison of it)
#endif
    return m;
  }
  __device__ static __forceinline__ float PickOf(uint32_t shut, float then, float otherwise) {
    return BitsToFloat((__builtin_bit_cast(uint32_t, then) & shut) | (__builtin_bit_cast(uint32_t, otherwise) & ~shut));
  }
  __device__ __forceinline__ double Product(float coefficient, int j) const {
    if (PER_CHANNEL) return a_fixed[j];
    if (!kGate) return (double)coefficient;
    const uint64_t one = (uint64_t)(0x3ff00000u & ~Shut(coefficient)) << 32;   // 1, or 0 if shut
    return __builtin_bit_cast(double, one) - (double)coefficient;
  }
  __device__ static __forceinline__ float Step(float coefficient, float x, float h) {
    return kGate ? fmaf(coefficient, x - h, PickOf(Shut(coefficient), x, h)) : fmaf(coefficient, h, x);
  }
  // M = a L
  __device__ static __forceinline__ float Back(float coefficient, float l) {
    return kGate ? fmaf(-coefficient, l, PickOf(Shut(coefficient), 0.0f, l)) : coefficient * l;
  }
  // of a gate: f L and (1 - f) L, which are s L and (1 - s) L with the smaller one s, and f (1 - f) L, which is s (1 - s) L either way
  __device__ static __forceinline__ void Shares(float coefficient, float l, float *m, float *dx, float *both) {
    const float s = fabsf(coefficient), p = s * l, q = fmaf(-s, l, l);
    const uint32_t shut = Shut(coefficient);
    *m = PickOf(shut, p, q);
    *dx = PickOf(shut, q, p);
    *both = s * q;
  }
};

template <typename XT, typename GT, bool PER_CHANNEL> struct RecTile {
  static constexpr int V = RecV<XT>();
  Group<XT, V> x[kRecSteps];
  Group<GT, V> g[PER_CHANNEL ? 1 : kRecSteps];
};

template <typename XT, typename GT, bool PER_CHANNEL>
__device__ __forceinline__ void LoadTile(RecTile<XT, GT, PER_CHANNEL> &t, const RecKernelArgs &p, int first, int stretch, int limit, const Channels<RecV<XT>()> &own) {
  constexpr int V = RecV<XT>();
  const bool full = first + kRecTile <= limit;
  LoadSteps<XT, V>(t.x, p.a.x, p.a.seq, first, stretch, limit, p.a.x_row, p.a.x_seq, own, p.x_plain && full);
  if constexpr (!PER_CHANNEL) LoadSteps<GT, V>(t.g, p.a.decay, p.a.seq, first, stretch, limit, p.a.decay_row, p.a.decay_seq, own, p.decay_plain && full);
}

// The coefficients of a stretch's steps: kept, or computed again where they are used again.
template <typename Decay, typename Tile, bool PER_CHANNEL, bool KEEP> struct RecCoefficients {
  static constexpr int V = Tile::V;
  float kept[KEEP ? kRecSteps : 1][V];
  __device__ __forceinline__ float First(const Decay &decay, const Tile &t, int k, int j) {
    const float c = decay.Coefficient(t.g[PER_CHANNEL ? 0 : k], j);
    if constexpr (KEEP) kept[k][j] = c;
    return c;
  }
  __device__ __forceinline__ float Get(const Decay &decay, const Tile &t, int k, int j) const {
    if constexpr (KEEP) return kept[k][j];
    else return decay.Coefficient(t.g[PER_CHANNEL ? 0 : k], j);
  }
  // Which of them are negative the compiler would keep as well, two scalar registers for each, which it then stores in lanes of
  // vector registers and reads back; after this it looks again.
  __device__ __forceinline__ void Forget() {
#if defined(__AMDGCN__)
    if constexpr (KEEP && !PER_CHANNEL) {
#pragma unroll
      for (int k = 0; k < kRecSteps; k++)
#pragma unroll
        for (int j = 0; j < V; j++) asm volatile("" : "+v"(kept[k][j]));
    }
#endif
  }
};

template <int V> __device__ __forceinline__ void LoadState(float (&h)[V], const float *state, int64_t s, int channels, const Channels<V> &own) {
#pragma unroll
  for (int j = 0; j < V; j++) h[j] = state && j < own.end ? state[s * channels + own.base + j] : 0.0f;
}
template <int V> __device__ __forceinline__ void StoreState(float *state, const float (&h)[V], int64_t s, int channels, const Channels<V> &own) {
  if (!state) return;
#pragma unroll
  for (int j = 0; j < V; j++)
    if (j >= own.begin && j < own.end) state[s * channels + own.base + j] = h[j];
}

// Sequences of no steps: their state is the initial one, their initial state's gradient that of the state.
template <int V> __device__ __forceinline__ void PassEmpty(const RecKernelArgs &p, int tile, int stretch, const Channels<V> &own, const float *from, float *to) {
  const daliamdSequenceRows &q = p.a.seq;
  if (!to || !(q.offsets || q.lengths || q.steps == 0)) return;
  constexpr int kStretches = kRecWaves * kRecPieces;
  for (int64_t s = (int64_t)tile * kStretches + stretch; s < q.sequences; s += (int64_t)p.tiles * kStretches) {
    int begin, end;
    SequenceRange(q, (int)s, &begin, &end);
    if (begin < end) continue;
    float h[V];
    LoadState<V>(h, from, s, p.a.channels, own);
    StoreState<V>(to, h, s, p.a.channels, own);
  }
}

constexpr int kForwardWaves = 4;
// Waves per SIMD that the backward pass' registers are to leave room for: two workgroups per compute unit.  16-bit rows with
// decays of 32 bits do not fit (272 bytes spilled: 236 us against 142 for 8 x 4096 x 1024 with one): one.
template <typename XT, typename GT, bool PER_CHANNEL> constexpr int BackwardWaves() { return !PER_CHANNEL && sizeof(GT) > sizeof(XT) ? 2 : 4; }
// Where registers do not decide, the tile's product is said before its states are computed, and coefficients are kept: nothing else
// covers the chain with one workgroup per compute unit (142 : 149 us), and float rows with decays per channel fit (113 : 117 us).
template <typename XT, typename GT, bool PER_CHANNEL> constexpr bool BackwardChainFirst() { return PER_CHANNEL ? sizeof(XT) == 4 : sizeof(GT) > sizeof(XT); }

// The product of a stretch's gates is kept for the composition against time, not computed again; of decays and per channel it is one
// multiplication a step, and keeping it costs registers that they do not have.
template <int FORM, bool PER_CHANNEL> constexpr bool BackwardShared() { return FORM == DALIAMD_RECURRENCE_GATE && !PER_CHANNEL; }

template <typename XT, typename GT, int FORM, bool PER_CHANNEL, bool COMPARE> struct RecForward {
  static constexpr int V = RecV<XT>();
  typedef RecDecay<XT, GT, FORM, PER_CHANNEL, COMPARE> Decay;
  typedef RecTile<XT, GT, PER_CHANNEL> Tile;

  // (A, S, R) of a thread's stretch
  template <bool EVENTS, typename Coefficients>
  __device__ static __forceinline__ bool Compose(const RecKernelArgs &p, const Decay &decay, const Tile &t, const RecEvents &e, int row,
                                                 const Channels<V> &own, Coefficients &c, double (&a)[V], float (&s)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) a[j] = 1.0, s[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) {
      if (EVENTS && !(e.live >> k & 1)) continue;
      if (EVENTS && (e.first >> k & 1)) LoadState<V>(s, p.a.initial, e.first_of[k], p.a.channels, own);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float ck = c.First(decay, t, k, j);
        a[j] *= decay.Product(ck, j);
        s[j] = Decay::Step(ck, t.x[k][j], s[j]);
      }
    }
    return EVENTS && e.first != 0;
  }

  template <bool EVENTS>
  __device__ static __forceinline__ void Process(const RecKernelArgs &p, const RecLane<XT> &lane, RecShared<RecChannels<XT>()> &shared, const Decay &decay,
                                                 Tile &t, const RecPlace &place, const RecMarks &marks, int tile, int channel_tile) {
    const int row = place.row + lane.Stretch() * kRecSteps, limit = place.limit;
    RecEvents e = {};
    if (EVENTS) e = EventsOf(marks, lane.Stretch());
    RecCoefficients<Decay, Tile, PER_CHANNEL, true> c;
    float s[V], state[V];
    double a[V];
    const bool r = Compose<EVENTS>(p, decay, t, e, row, lane.own, c, a, s);
    const RecFront<V> front = lane.template ScanWave<false, EVENTS, Decay::kGate>(shared, a, s, r);
    c.Forget();
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) t.x[k].Repack();
    __syncthreads();
    const bool starts = place.sequence < 0 || place.row == place.begin;
    FindFront<false, Decay::kGate, XT>(p, shared, tile, channel_tile, !starts, starts && !EVENTS ? p.a.initial : nullptr, place.sequence);
    __syncthreads();
    if (lane.Idle()) return;
    float in[V];
#pragma unroll
    for (int j = 0; j < V; j++) in[j] = shared.front[lane.lane_c + j];
    if (p.a.saved && lane.Stretch() == 0) StoreState<V>(p.a.saved, in, tile, p.a.channels, lane.own);
    lane.template Start<false, EVENTS>(shared, front, in, state);
    XT *y = static_cast<XT *>(p.a.y) + (int64_t)place.row * p.a.channels;
    const uint32_t offset = (uint32_t)(lane.Stretch() * kRecSteps * p.a.channels);
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) {
      if (EVENTS && row + k >= limit) break;
      if (EVENTS && !(e.live >> k & 1)) {
        const float zero[V] = {};
        lane.own.Store(y + (int64_t)k * p.a.channels, zero, offset);
        continue;
      }
      if (EVENTS && (e.first >> k & 1)) LoadState<V>(state, p.a.initial, e.first_of[k], p.a.channels, lane.own);
#pragma unroll
      for (int j = 0; j < V; j++) state[j] = Decay::Step(c.Get(decay, t, k, j), t.x[k][j], state[j]);
      lane.own.Store(y + (int64_t)k * p.a.channels, state, offset);
      if (EVENTS && (e.last >> k & 1)) StoreState<V>(p.a.final_state, state, e.last_of[k], p.a.channels, lane.own);
    }
    if (!EVENTS && place.row + kRecTile == place.end && lane.Stretch() == kRecWaves * kRecPieces - 1)
      StoreState<V>(p.a.final_state, state, place.sequence, p.a.channels, lane.own);
  }
};

template <typename XT, typename GT, int FORM, bool PER_CHANNEL>
__global__ __launch_bounds__(kRecThreads, kForwardWaves) void RecurrenceForwardKernel(RecKernelArgs p) {
  typedef RecForward<XT, GT, FORM, PER_CHANNEL, true> Op;
  constexpr int V = RecV<XT>();
  __shared__ RecShared<RecChannels<XT>()> shared;
  __shared__ int slot;
  int tile, channel_tile;
  TakeTile<false>(p, &slot, &tile, &channel_tile);
  const RecLane<XT> lane(p.a.channels, channel_tile);
  __shared__ RecMarks marks;
  RecPlace place(p, tile);
  typename Op::Tile t;
  if (place.row < place.limit) LoadTile<XT, GT, PER_CHANNEL>(t, p, place.row, lane.Stretch(), place.limit, lane.own);
  const typename Op::Decay decay(p.a, lane.own);
  place.Find(p);
  if (place.interior) {
    Op::template Process<false>(p, lane, shared, decay, t, place, marks, tile, channel_tile);
  } else {
    Mark(p, place, marks);
    Op::template Process<true>(p, lane, shared, decay, t, place, marks, tile, channel_tile);
  }
  PassEmpty<V>(p, tile, lane.Stretch(), lane.own, p.a.initial, p.a.final_state);
}

// (A, S, R) of a thread's stretch against time; dy NULL: zeros; SHARED: A is there, the product of the same decays
template <typename XT, bool EVENTS, bool SHARED, typename Decay, typename Tile, typename Coefficients>
__device__ __forceinline__ bool ComposeBack(const RecKernelArgs &p, const Decay &decay, const Group<XT, RecV<XT>()> (&dy)[kRecSteps],
                                            const Tile &t, const Coefficients &c, const RecEvents &e, int row, const Channels<RecV<XT>()> &own,
                                            double (&a)[RecV<XT>()], float (&s)[RecV<XT>()]) {
  constexpr int V = RecV<XT>();
#pragma unroll
  for (int j = 0; j < V; j++) {
    s[j] = 0.0f;
    if (!SHARED) a[j] = 1.0;
  }
#pragma unroll
  for (int k = kRecSteps - 1; k >= 0; k--) {
    if (EVENTS && !(e.live >> k & 1)) continue;
    if (EVENTS && (e.last >> k & 1)) LoadState<V>(s, p.a.dfinal, e.last_of[k], p.a.channels, own);
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float ck = c.Get(decay, t, k, j);
      if (!SHARED) a[j] *= decay.Product(ck, j);
      s[j] = Decay::Back(ck, s[j] + dy[k][j]);
    }
  }
  return EVENTS && e.last != 0;
}

// What the second half of the backward pass needs of each step, in LDS: a thread's own places.
template <int V> struct RecSteps {
  struct alignas(4 * V) Step { float v[V]; };
  Step steps[kRecSteps][kRecThreads];
  __device__ __forceinline__ void Put(int k, const float (&b)[V]) {
    Step s;
#pragma unroll
    for (int j = 0; j < V; j++) s.v[j] = b[j];
    steps[k][threadIdx.x] = s;
  }
  __device__ __forceinline__ void Get(int k, float (&b)[V]) const {
    const Step s = steps[k][threadIdx.x];
#pragma unroll
    for (int j = 0; j < V; j++) b[j] = s.v[j];
  }
};

template <typename XT, typename GT, int FORM, bool PER_CHANNEL> struct RecBackward {
  static constexpr int V = RecV<XT>();
  typedef RecForward<XT, GT, FORM, PER_CHANNEL, PER_CHANNEL> Forward;
  typedef typename Forward::Decay Decay;
  typedef typename Forward::Tile Tile;

  __device__ static __forceinline__ void Repack(Tile &t) {
    if constexpr (!PER_CHANNEL) {
#pragma unroll
      for (int k = 0; k < kRecSteps; k++) t.g[k].Repack();
    }
  }
  template <bool EVENTS>
  __device__ static __forceinline__ void Process(const RecKernelArgs &p, const RecLane<XT> &lane, RecShared<RecChannels<XT>()> (&shared)[2], const Decay &decay,
                                                 Tile &t, Group<XT, V> (&dy)[kRecSteps], const RecPlace &place, const RecMarks &marks, int tile, int channel_tile,
                                                 const float (&saved)[V], float (&sum)[V], RecSteps<V> &before) {
    const int row = place.row + lane.Stretch() * kRecSteps, limit = place.limit;
    RecEvents e = {};
    if (EVENTS) e = EventsOf(marks, lane.Stretch());
    constexpr bool kChainFirst = BackwardChainFirst<XT, GT, PER_CHANNEL>(), kShared = BackwardShared<FORM, PER_CHANNEL>();
    RecCoefficients<Decay, Tile, PER_CHANNEL, kChainFirst> c;
    float s[V], state[V], back[V];
    double a[V];
    // h_{t-1}, or with gates h_{t-1} - x_t: what the decay's gradient takes
    auto states = [&](const RecFront<V> &front) {
      lane.template Start<false, EVENTS>(shared[0], front, saved, state);
#pragma unroll
      for (int k = 0; k < kRecSteps; k++) {
        if (EVENTS && !(e.live >> k & 1)) continue;
        if (EVENTS && (e.first >> k & 1)) LoadState<V>(state, p.a.initial, e.first_of[k], p.a.channels, lane.own);
        float b[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float x = t.x[k][j], ck = c.Get(decay, t, k, j);
          b[j] = FORM == DALIAMD_RECURRENCE_GATE ? state[j] - x : state[j];
          state[j] = Decay::kGate ? fmaf(-ck, b[j], Decay::PickOf(Decay::Shut(ck), x, state[j])) : Decay::Step(ck, x, state[j]);
        }
        before.Put(k, b);
      }
    };
    bool r = Forward::template Compose<EVENTS>(p, decay, t, e, row, lane.own, c, a, s);
    double product[V];
#pragma unroll
    for (int j = 0; j < V; j++) product[j] = a[j];
    const RecFront<V> front = lane.template ScanWave<false, EVENTS, Decay::kGate>(shared[0], a, s, r);
    c.Forget();
    if constexpr (!kChainFirst) {   // x and what its scan needs are then done with
#pragma unroll
      for (int k = 0; k < kRecSteps; k++) t.x[k].Repack(), dy[k].Repack();
      Repack(t);
      __syncthreads();
      states(front);
      Repack(t);
    }
    r = ComposeBack<XT, EVENTS, kShared>(p, decay, dy, t, c, e, row, lane.own, a, s);
    if (kShared) {
#pragma unroll
      for (int j = 0; j < V; j++) a[j] = product[j];
    }
    const RecFront<V> behind = lane.template ScanWave<true, EVENTS, Decay::kGate>(shared[1], a, s, r);
    c.Forget();
#pragma unroll
    for (int k = 0; k < kRecSteps; k++) {
      if (kChainFirst) t.x[k].Repack();
      dy[k].Repack();
    }
    if (!kChainFirst) Repack(t);
    __syncthreads();
    // the last row's sequence goes on behind the tile
    const int last_row = limit - 1 - place.row;
    const bool needs = EVENTS ? limit > place.row && marks.live[last_row] && marks.last[last_row] < 0 : place.row + kRecTile < place.end;
    FindFront<true, Decay::kGate, XT>(p, shared[1], tile, channel_tile, needs, EVENTS ? nullptr : p.a.dfinal, place.sequence);
    if constexpr (kChainFirst) {
      states(front);
      c.Forget();
    }
    __syncthreads();
    if (lane.Idle()) return;
    float in[V];
#pragma unroll
    for (int j = 0; j < V; j++) in[j] = shared[1].front[lane.lane_c + j];
    lane.template Start<true, EVENTS>(shared[1], behind, in, back);
    const uint32_t offset = (uint32_t)(lane.Stretch() * kRecSteps * p.a.channels);
#pragma unroll
    for (int k = kRecSteps - 1; k >= 0; k--) {
      if (EVENTS && row + k >= limit) continue;
      float dx[V] = {}, dg[V] = {};
      const bool live = !EVENTS || (e.live >> k & 1);
      if (live) {
        float b[V];
        before.Get(k, b);
        if (EVENTS && (e.last >> k & 1)) LoadState<V>(back, p.a.dfinal, e.last_of[k], p.a.channels, lane.own);
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float l = back[j] + dy[k][j], ck = c.Get(decay, t, k, j);
          if (FORM == DALIAMD_RECURRENCE_GATE) {
            float both;
            Decay::Shares(ck, l, &back[j], &dx[j], &both);
            dg[j] = both * b[j];
          } else {
            dx[j] = l;
            dg[j] = l * b[j];
            back[j] = Decay::Back(ck, l);
          }
          if (PER_CHANNEL) sum[j] += dg[j];
        }
        if (EVENTS && (e.first >> k & 1)) StoreState<V>(p.a.dinitial, back, e.first_of[k], p.a.channels, lane.own);
      }
      const int64_t at = (int64_t)(place.row + k) * p.a.channels;
      lane.own.Store(static_cast<XT *>(p.a.dx) + at, dx, offset);
      if (!PER_CHANNEL) lane.own.Store(static_cast<GT *>(p.a.ddecay) + at, dg, offset);
    }
    if (!EVENTS && place.row == place.begin && lane.Stretch() == 0) StoreState<V>(p.a.dinitial, back, place.sequence, p.a.channels, lane.own);
  }
};

template <typename XT, typename GT, int FORM, bool PER_CHANNEL>
__global__ __launch_bounds__(kRecThreads, (BackwardWaves<XT, GT, PER_CHANNEL>())) void RecurrenceBackwardKernel(RecKernelArgs p) {
  typedef RecBackward<XT, GT, FORM, PER_CHANNEL> Op;
  constexpr int V = RecV<XT>();
  __shared__ RecShared<RecChannels<XT>()> shared[2];
  __shared__ RecSteps<V> before;
  __shared__ int slot;
  int tile, channel_tile;
  TakeTile<true>(p, &slot, &tile, &channel_tile);
  const RecLane<XT> lane(p.a.channels, channel_tile);
  __shared__ RecMarks marks;
  RecPlace place(p, tile);
  typename Op::Tile t;
  Group<XT, V> dy[kRecSteps];
  float saved[V], sum[V] = {};
  if (place.row < place.limit) {
    LoadTile<XT, GT, PER_CHANNEL>(t, p, place.row, lane.Stretch(), place.limit, lane.own);
    if (p.a.dy)
      LoadSteps<XT, V>(dy, p.a.dy, p.a.seq, place.row, lane.Stretch(), place.limit, p.a.dy_row, p.a.dy_seq, lane.own,
                       p.dy_plain && place.row + kRecTile <= place.limit);
  }
  if (!p.a.dy) {
#pragma unroll
    for (int k = 0; k < kRecSteps; k++)
#pragma unroll
      for (int j = 0; j < V; j++) dy[k].Set(j, FromFloat<XT>(0.0f));
  }
  LoadState<V>(saved, p.a.saved, tile, p.a.channels, lane.own);
  const typename Op::Decay decay(p.a, lane.own);
  place.Find(p);
  if (place.interior) {
    Op::template Process<false>(p, lane, shared, decay, t, dy, place, marks, tile, channel_tile, saved, sum, before);
  } else {
    Mark(p, place, marks);
    Op::template Process<true>(p, lane, shared, decay, t, dy, place, marks, tile, channel_tile, saved, sum, before);
  }
  PassEmpty<V>(p, tile, lane.Stretch(), lane.own, p.a.dfinal, p.a.dinitial);
  if (PER_CHANNEL) {
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int off = kRecLanes; off < 64; off <<= 1) sum[j] += __shfl_xor(sum[j], off, 64);
    }
    __syncthreads();
    if (lane.piece == 0) {
#pragma unroll
      for (int j = 0; j < V; j++) shared[0].s[lane.wave][lane.lane_c + j] = sum[j];
    }
    __syncthreads();
    if (lane.Stretch() == 0) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        float total = 0;
        for (int w = 0; w < kRecWaves; w++) total += shared[0].s[w][lane.lane_c + j];
        if (j >= lane.own.begin && j < lane.own.end) p.partial[(int64_t)tile * p.a.channels + lane.own.base + j] = total;
      }
    }
  }
}

// A few steps per sequence (one token for each of many): a thread has 8 bytes of channels of one sequence.
template <typename XT, typename GT, int FORM, bool PER_CHANNEL>
__global__ __launch_bounds__(kRecThreads) void RecurrenceStepKernel(RecKernelArgs p) {
  constexpr int V = RecV<XT>();
  const int groups = (p.a.channels + V - 1) / V;
  const int64_t id = (int64_t)blockIdx.x * kRecThreads + threadIdx.x;
  int64_t s = (uint32_t)id / (uint32_t)groups;
  if (s >= p.sequences) return;
  // (a state may be written over the one it is read from: threads have no channels in common)
  const int channel = (int)(id - s * groups) * V, n = min(p.a.channels - channel, V);
  Channels<V> own(channel, p.a.channels);
  if (n < V) own.base = channel, own.begin = 0, own.end = n, own.narrow = true;
  typedef RecDecay<XT, GT, FORM, PER_CHANNEL, true> Decay;
  const Decay decay(p.a, own);
  s += p.first_sequence;
  int begin, end;
  SequenceRange(p.a.seq, (int)s, &begin, &end);
  const int steps = (int)p.a.seq.steps, length = end - begin;
  float h[V];
  LoadState<V>(h, p.a.initial, s, p.a.channels, own);
  for (int t = 0; t < steps; t++) {
    XT *y = static_cast<XT *>(p.a.y) + (s * steps + t) * p.a.channels;
    if (t < length) {
      Group<XT, V> x;
      Group<GT, V> g;
      const XT *px = static_cast<const XT *>(p.a.x) + s * p.a.x_seq + t * p.a.x_row;
      const GT *pg = static_cast<const GT *>(p.a.decay) + s * p.a.decay_seq + t * p.a.decay_row;
      own.Load(x, px + (own.narrow ? own.base : 0));
      if (!PER_CHANNEL) own.Load(g, pg + (own.narrow ? own.base : 0));
#pragma unroll
      for (int j = 0; j < V; j++) h[j] = Decay::Step(decay.Coefficient(g, j), x[j], h[j]);
      own.Store(y, h);
    } else {
      const float zero[V] = {};
      own.Store(y, zero);
    }
  }
  StoreState<V>(p.a.final_state, h, s, p.a.channels, own);
}

template <typename XT, typename GT, int FORM, bool PER_CHANNEL> struct RecLaunch {
  static void Forward(hipStream_t s, const RecKernelArgs &p) {
    const daliamdSequenceRows &q = p.a.seq;
    if (p.few_steps) {
      const int64_t groups = (p.a.channels + RecV<XT>() - 1) / RecV<XT>();
      const int most = (int)std::min<int64_t>(q.sequences, MaxWorkgroups(kRecThreads) * kRecThreads / groups);
      KernelTimer timer("RecurrenceStepKernel", s);
      for (int first = 0, n; first < q.sequences; first += n) {   // (a second launch only for more than 2^32 threads)
        n = std::min(most, q.sequences - first);
        RecKernelArgs part = p;
        part.first_sequence = first;
        part.sequences = n;
        const int64_t threads = n * groups;
        hipLaunchKernelGGL((RecurrenceStepKernel<XT, GT, FORM, PER_CHANNEL>), dim3((unsigned)((threads + kRecThreads - 1) / kRecThreads)), dim3(kRecThreads), 0, s,
                           part);
      }
      return;
    }
    const dim3 grid((unsigned)p.tiles * p.channel_tiles);
    KernelTimer timer("RecurrenceForwardKernel", s);
    hipLaunchKernelGGL((RecurrenceForwardKernel<XT, GT, FORM, PER_CHANNEL>), grid, dim3(kRecThreads), 0, s, p);
  }
  static void Backward(hipStream_t s, const RecKernelArgs &p) {
    const dim3 grid((unsigned)p.tiles * p.channel_tiles);
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
