// Embedding lookup with a scale, and its gradient: the tokens' gradients summed per row of the table.
#include <algorithm>
#include "sequence_common.h"

namespace daliamd {

// Memory bounds the lookup and the sums.  65536 tokens, frequent ones thousands of times, of a table of 48000 x 1024 bf16: lookup
// 38 us for 134 MB written and 33 MB of the table read (4.4 TB/s); gradient 64 us for 134 MB read, rows of 2 KB in the order of their
// ids, and 98 MB written (3.6 TB/s), 11 us to join runs, and 24 us for two sorting passes, whose four kernels each wait for a handful
// of loads one after the other.  131072 tokens of 64000 x 2048: lookup 153 us (4.2 TB/s).  A copy of 1 GiB runs at 5.1 TB/s.

// ---- lookup ------------------------------------------------------------------------------------------------------------
// TPR threads per row, 8 channels per thread and step; kTokens rows per thread, whose loads are all in flight at once.
constexpr int kEmbThreads = 256, kEmbV = 8;

template <typename TT, typename OT, typename IT, int kTokens, bool WHOLE>
__global__ __launch_bounds__(kEmbThreads) void EmbeddingKernel(daliamdEmbeddingArgs p, int tpr) {
  const int64_t first = ((int64_t)blockIdx.x * (kEmbThreads / tpr) + threadIdx.x / tpr) * kTokens;
  if (first >= p.tokens) return;
  const TT *row[kTokens];
  bool inside[kTokens];
#pragma unroll
  for (int k = 0; k < kTokens; k++) {
    const int64_t id = static_cast<const IT *>(p.ids)[min(first + k, p.tokens - 1)];
    inside[k] = id >= 0 && id < p.vocab;
    row[k] = static_cast<const TT *>(p.table) + (inside[k] ? id : 0) * p.table_row;
  }
  for (int c = (int)threadIdx.x % tpr * kEmbV; c < p.channels; c += tpr * kEmbV) {
    const Channels<kEmbV, WHOLE> m(c, p.channels);
    Group<TT, kEmbV> g[kTokens];
#pragma unroll
    for (int k = 0; k < kTokens; k++) m.Load(g[k], row[k]);
#pragma unroll
    for (int k = 0; k < kTokens; k++) {
      float v[kEmbV];
#pragma unroll
      for (int j = 0; j < kEmbV; j++) v[j] = inside[k] ? g[k][j] * p.scale : 0.0f;
      if (first + k < p.tokens) m.Store(static_cast<OT *>(p.out) + (first + k) * p.channels, v);
    }
  }
}

// ---- the tokens, sorted ------------------------------------------------------------------------------------------------
// A stable sort of the tokens by id, least significant digit first (so that equal ids stay in the order of the tokens, and the
// sums below have a fixed order).  A token that takes no part (padding, ids outside the table) has the key `vocab`, behind all
// others.  Per digit of up to 9 bits: SortCountKernel counts the digits of each tile of tokens; SortScatterKernel adds up the
// counts in front of its own (all digits below, and this digit in the tiles before: a few hundred numbers per digit, read by
// every workgroup instead of a launch of their own) and moves its tile's tokens.  Up to kSmallTokens: everything in one workgroup.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kTileTokens = 1024, kMaxTiles = 512;
constexpr int kSmallTokens = 4096, kSmallThreads = 1024, kSmallRounds = kSmallTokens / kSmallThreads;

struct EmbSort {
  int64_t tokens, tile;         // tile: tokens per workgroup, a multiple of kSortThreads
  int tiles, passes, bits;      // bits per digit
  uint32_t *key[2], *index[2], *count;
};

__device__ __forceinline__ uint32_t TokenKey(const daliamdEmbeddingArgs &p, int64_t t) {
  const int64_t id = LoadIndex(p.ids, t, p.index_dtype);
  return (uint32_t)(id >= 0 && id < p.vocab && id != p.padding ? id : p.vocab);
}

// the lanes of the wave whose digit is this lane's (those with `valid`)
__device__ __forceinline__ uint64_t SameDigit(uint32_t digit, int bits, bool valid) {
  uint64_t mask = __ballot(valid);
  for (int b = 0; b < bits; b++) {
    const uint64_t set = __ballot((digit >> b) & 1);
    mask &= (digit >> b) & 1 ? set : ~set;
  }
  return mask;
}

// One round of 64 tokens of a wave in their order: the place of each behind those with its digit so far; next[digit] counts.
__device__ __forceinline__ uint32_t TakePlace(uint32_t *next, uint32_t digit, int bits, bool valid) {
  const uint64_t mask = SameDigit(digit, bits, valid);
  const int lane = threadIdx.x & 63;
  const uint32_t before = (uint32_t)__popcll(mask & (((uint64_t)1 << lane) - 1));
  uint32_t place = 0;
  if (valid) place = next[digit] + before;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (valid && before == 0) next[digit] += (uint32_t)__popcll(mask);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return place;
}

__global__ __launch_bounds__(kSortThreads) void SortCountKernel(daliamdEmbeddingArgs p, EmbSort s, int pass) {
  __shared__ uint32_t count[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * s.tile, end = min(begin + s.tile, s.tokens);
  const int shift = pass * s.bits;
  const uint32_t digits = (1u << s.bits) - 1;
  for (int64_t t = begin + threadIdx.x; t < end; t += kSortThreads) {
    const uint32_t key = pass ? s.key[pass & 1][t] : TokenKey(p, t);
    atomicAdd(&count[(key >> shift) & digits], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) s.count[(int64_t)blockIdx.x * kDigits + d] = count[d];
}

// exclusive prefix sums of one number per thread over kSortThreads == kDigits threads
__device__ __forceinline__ uint32_t PrefixOfDigits(uint32_t v, uint32_t *wave_total) {
  uint32_t incl = v;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)incl, off, 64);
    if (lane >= off) incl += u;
  }
  if (lane == 63) wave_total[wave] = incl;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; w++) before += wave_total[w];
  return before + incl - v;
}

__global__ __launch_bounds__(kSortThreads) void SortScatterKernel(daliamdEmbeddingArgs p, EmbSort s, int pass) {
  static_assert(kSortThreads == kDigits, "a thread per digit");
  __shared__ uint32_t next[kSortWaves][kDigits], wave_total[kSortWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int w = 0; w < kSortWaves; w++) next[w][tid] = 0;
  // this digit in the tiles before, and in all of them
  uint32_t before = 0, all = 0;
#pragma unroll 32
  for (int t = 0; t < s.tiles; t++) {
    const uint32_t n = s.count[(int64_t)t * kDigits + tid];
    all += n;
    if (t < (int)blockIdx.x) before += n;
  }
  __syncthreads();
  // the tokens of a wave: one stretch of the tile
  const int64_t begin = blockIdx.x * s.tile + wave * (s.tile / kSortWaves), end = min(begin + s.tile / kSortWaves, s.tokens);
  const int shift = pass * s.bits;
  const uint32_t digits = (1u << s.bits) - 1;
  for (int64_t t = begin + lane; t < end; t += 64) {
    const uint32_t key = pass ? s.key[pass & 1][t] : TokenKey(p, t);
    atomicAdd(&next[wave][(key >> shift) & digits], 1u);
  }
  uint32_t place = PrefixOfDigits(all, wave_total) + before;
  __syncthreads();
  for (int w = 0; w < kSortWaves; w++) {
    const uint32_t n = next[w][tid];
    next[w][tid] = place;
    place += n;
  }
  __syncthreads();
  for (int64_t t = begin; t < end; t += 64) {
    const bool valid = t + lane < end;
    const uint32_t key = !valid ? 0 : pass ? s.key[pass & 1][t + lane] : TokenKey(p, t + lane);
    const uint32_t index = !valid ? 0 : pass ? s.index[pass & 1][t + lane] : (uint32_t)(t + lane);
    const uint32_t to = TakePlace(next[wave], (key >> shift) & digits, s.bits, valid);
    if (valid) {
      s.key[(pass + 1) & 1][to] = key;
      s.index[(pass + 1) & 1][to] = index;
    }
  }
}

__global__ __launch_bounds__(kSmallThreads) void SortSmallKernel(daliamdEmbeddingArgs p, EmbSort s) {
  constexpr int kWaves = kSmallThreads / 64;
  __shared__ uint32_t key[kSmallTokens], next[kWaves][kDigits], wave_total[kWaves];
  __shared__ uint16_t index[kSmallTokens];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, tokens = (int)s.tokens;
  uint32_t k[kSmallRounds], to[kSmallRounds];
  uint16_t at[kSmallRounds];
  for (int pass = 0; pass < s.passes; pass++) {
    const int shift = pass * s.bits;
    const uint32_t digits = (1u << s.bits) - 1;
    for (int d = tid; d < kWaves * kDigits; d += kSmallThreads)
      if ((uint32_t)d % kDigits <= digits) next[d / kDigits][d % kDigits] = 0;
#pragma unroll
    for (int r = 0; r < kSmallRounds; r++) {
      const int t = (wave * kSmallRounds + r) * 64 + lane;
      if (t >= tokens) continue;
      k[r] = pass ? key[t] : TokenKey(p, t);
      at[r] = pass ? index[t] : (uint16_t)t;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; r++) {
      const bool valid = (wave * kSmallRounds + r) * 64 + lane < tokens;
      to[r] = TakePlace(next[wave], valid ? (k[r] >> shift) & digits : 0, s.bits, valid);
    }
    __syncthreads();
    // `next` counts each wave's digits now: to where the first of each goes
    uint32_t all = 0;
    if (tid <= (int)digits)
      for (int w = 0; w < kWaves; w++) all += next[w][tid];
    uint32_t place = PrefixOfDigits(all, wave_total);
    if (tid <= (int)digits)
      for (int w = 0; w < kWaves; w++) {
        const uint32_t n = next[w][tid];
        next[w][tid] = place;
        place += n;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; r++)
      if ((wave * kSmallRounds + r) * 64 + lane < tokens) {
        const uint32_t at_place = next[wave][(k[r] >> shift) & digits] + to[r];
        key[at_place] = k[r], index[at_place] = at[r];
      }
    __syncthreads();
  }
  for (int t = tid; t < tokens; t += kSmallThreads) {
    s.key[s.passes & 1][t] = key[t];
    s.index[s.passes & 1][t] = index[t];
  }
}

// ---- sums of the sorted tokens' gradients --------------------------------------------------------------------------------
// The sorted tokens are cut into chunks of 8 to 32, whatever their ids: a token that fills half a batch is as much work per
// workgroup as rare ones.  A chunk adds up each run of equal ids in it.  A run that lies within a chunk is a row of the result; of
// one that goes on, each chunk leaves its part, and EmbeddingJoinKernel adds those of one run in their order.  Rows without a
// token are filled with zeros by further workgroups of the same launch.
constexpr int kFillRows = 64;

struct EmbSums {
  const uint32_t *key, *index;
  float *part;                  // [chunks][2][part_row]: of the run that came from the chunk before, of the one that goes on behind
  int chunk, chunks, chunk_groups, tpr, part_row;
  int64_t first;                // of a launch: the first row that it may fill with zeros, or the first chunk whose run it may join
};

// the first place whose key is not below `key`
__device__ __forceinline__ int64_t LowerBound(const uint32_t *keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// ... by a whole wave, 64 places at a time
__device__ __forceinline__ int64_t LowerBoundOfWave(const uint32_t *keys, int64_t n, uint32_t key) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = n;   // all in front of lo are below, none from hi on
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
    const int below = __popcll(__ballot(at < hi && keys[min(at, hi - 1)] < key));
    if (below == 0) return lo;
    hi = min(lo + below * step, hi);
    lo += (below - 1) * step + 1;
  }
  return lo;
}

template <typename TT, typename OT, bool WHOLE>
__global__ __launch_bounds__(kEmbThreads) void EmbeddingBackwardKernel(daliamdEmbeddingArgs p, EmbSums s) {
  const int64_t n = p.tokens;
  if ((int)blockIdx.x >= s.chunk_groups) {   // rows without a token
    __shared__ uint8_t none[kFillRows];
    __shared__ int bound[2];
    const int64_t row = s.first + (int64_t)((int)blockIdx.x - s.chunk_groups) * kFillRows;
    const int tid = threadIdx.x;
    if (tid < 128) {
      const int at = (int)LowerBoundOfWave(s.key, n, (uint32_t)(row + (tid >> 6) * kFillRows));
      if ((tid & 63) == 0) bound[tid >> 6] = at;
    }
    __syncthreads();
    if (tid < kFillRows) {
      const int64_t at = bound[0] + LowerBound(s.key + bound[0], bound[1] - bound[0], (uint32_t)(row + tid));
      none[tid] = at >= bound[1] || s.key[at] != (uint32_t)(row + tid);
    }
    __syncthreads();
    const float zero[kEmbV] = {};
    for (int r = tid / s.tpr; r < kFillRows && row + r < p.vocab; r += kEmbThreads / s.tpr) {
      if (!none[r]) continue;
      TT *out = static_cast<TT *>(p.dtable) + (row + r) * p.channels;
      for (int c = tid % s.tpr * kEmbV; c < p.channels; c += s.tpr * kEmbV) Channels<kEmbV, WHOLE>(c, p.channels).Store(out, zero);
    }
    return;
  }
  const int64_t chunk = (int64_t)blockIdx.x * (kEmbThreads / s.tpr) + threadIdx.x / s.tpr;
  const int64_t begin = chunk * s.chunk, end = min(begin + s.chunk, n);
  if (begin >= end) return;
  const uint32_t vocab = (uint32_t)p.vocab;
  const bool from_before = begin > 0 && s.key[begin - 1] == s.key[begin];
  // (not if these are tokens that take no part: the last real run ends in front of them)
  const bool goes_on = end < n && s.key[end] == s.key[end - 1] && s.key[end] < vocab;
  constexpr int kAhead = 8;   // rows in flight
  for (int c = (int)threadIdx.x % s.tpr * kEmbV; c < p.channels; c += s.tpr * kEmbV) {
    const Channels<kEmbV, WHOLE> m(c, p.channels);
    float sum[kEmbV] = {};
    uint32_t run = s.key[begin];
    bool first = true;        // the chunk's first run
    for (int64_t t0 = begin; t0 < end && s.key[t0] < vocab; t0 += kAhead) {
      Group<OT, kEmbV> g[kAhead];
      uint32_t key[kAhead], token[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; a++) {
        const int64_t at = min(t0 + a, end - 1);
        key[a] = s.key[at];
        token[a] = s.index[at];
      }
#pragma unroll
      for (int a = 0; a < kAhead; a++) {
        m.Load(g[a], static_cast<const OT *>(p.dout) + (int64_t)token[a] * p.dout_row);
        if (t0 + a >= end) key[a] = vocab;
      }
#pragma unroll
      for (int a = 0; a < kAhead; a++) {
        if (key[a] != run && run < vocab) {   // a run ends, not the chunk's last
          if (first && from_before) {
            m.Store(s.part + chunk * 2 * s.part_row, sum);
          } else if (t0 + a < end || !goes_on) {
#pragma unroll
            for (int j = 0; j < kEmbV; j++) sum[j] *= p.scale;
            m.Store(static_cast<TT *>(p.dtable) + (int64_t)run * p.channels, sum);
          } else {
            m.Store(s.part + (chunk * 2 + 1) * s.part_row, sum);
          }
          first = false;
#pragma unroll
          for (int j = 0; j < kEmbV; j++) sum[j] = 0;
        }
        run = key[a];
        if (key[a] < vocab) {
#pragma unroll
          for (int j = 0; j < kEmbV; j++) sum[j] += g[a][j];
        }
      }
    }
    if (run < vocab) {        // the chunk's last token was the last of a group of kAhead
      if (first && from_before) {
        m.Store(s.part + chunk * 2 * s.part_row, sum);
      } else if (goes_on) {
        m.Store(s.part + (chunk * 2 + 1) * s.part_row, sum);
      } else {
#pragma unroll
        for (int j = 0; j < kEmbV; j++) sum[j] *= p.scale;
        m.Store(static_cast<TT *>(p.dtable) + (int64_t)run * p.channels, sum);
      }
    }
  }
}

// A run over several chunks: kJoinParts threads for 4 channels, each adding up a stretch of its parts.  Most workgroups find
// nothing to do or two or three parts: small ones, so that a frequent token's long run is the only one that takes time.
constexpr int kJoinLanes = 64, kJoinParts = 4, kJoinColumns = kJoinLanes * 4;
__global__ __launch_bounds__(kJoinLanes * kJoinParts) void EmbeddingJoinKernel(daliamdEmbeddingArgs p, EmbSums s) {
  __shared__ float4 part[kJoinParts][kJoinLanes];
  const int64_t chunk = s.first + blockIdx.x, begin = chunk * s.chunk, end = begin + s.chunk;
  if (end >= p.tokens || s.key[end] != s.key[end - 1]) return;                  // nothing goes on behind this chunk
  const uint32_t key = s.key[end - 1];
  if (key >= (uint32_t)p.vocab) return;
  if (begin > 0 && s.key[begin - 1] == key) return;                             // it began in a chunk before
  const int64_t last = (LowerBoundOfWave(s.key, p.tokens, key + 1) - 1) / s.chunk;   // the chunk that the run ends in
  const int lane = threadIdx.x % kJoinLanes, k = threadIdx.x / kJoinLanes;
  const int64_t count = last - chunk, each = (count + kJoinParts - 1) / kJoinParts;
  const int64_t from = chunk + 1 + k * each, to = min(from + each, last + 1);
  for (int c0 = blockIdx.y * kJoinColumns; c0 < p.channels; c0 += gridDim.y * kJoinColumns) {
    const int c = c0 + lane * 4;
    const float4 *parts = reinterpret_cast<const float4 *>(s.part + min(c, s.part_row - 4));   // (rows of parts are a multiple of 4 long)
    const int64_t row = s.part_row / 4;
    float4 sum = make_float4(0, 0, 0, 0);
    if (k == 0) sum = parts[(chunk * 2 + 1) * row];
#pragma unroll 8
    for (int64_t n = from; n < to; n++) {
      const float4 v = parts[n * 2 * row];
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    __syncthreads();
    part[k][lane] = sum;
    __syncthreads();
    if (k == 0) {
      for (int n = 1; n < kJoinParts; n++) {
        const float4 v = part[n][lane];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      const float f[4] = {sum.x, sum.y, sum.z, sum.w};
      for (int j = 0; j < 4; j++)
        if (c + j < p.channels) StoreElement(p.dtable, (int64_t)key * p.channels + c + j, p.dtype, f[j] * p.scale);
    }
  }
}

// ---- launches ------------------------------------------------------------------------------------------------------------
struct EmbLayout {
  EmbSort sort;
  EmbSums sums;
  size_t bytes;
};

// how the backward pass uses its workspace
static EmbLayout LayOut(const daliamdEmbeddingArgs &a, void *workspace) {
  EmbLayout l = {};
  EmbSort &s = l.sort;
  s.tokens = a.tokens;
  int bits = 1;
  while (bits < 31 && (a.vocab >> bits)) bits++;          // keys 0 .. vocab
  s.passes = (bits + kDigitBits - 1) / kDigitBits;
  s.bits = (bits + s.passes - 1) / s.passes;
  s.tile = kTileTokens;
  if (a.tokens > (int64_t)kTileTokens * kMaxTiles)
    s.tile = ((a.tokens + kMaxTiles - 1) / kMaxTiles + kSortThreads - 1) / kSortThreads * kSortThreads;
  s.tiles = (int)((a.tokens + s.tile - 1) / s.tile);
  EmbSums &u = l.sums;
  u.tpr = 8;
  while (u.tpr < kEmbThreads && u.tpr * kEmbV < a.channels) u.tpr *= 2;
  // Long chunks leave fewer parts, short ones more workgroups: the longest that still gives every compute unit four.
  u.chunk = 32;
  while (u.chunk > 8 && a.tokens / u.chunk / (kEmbThreads / u.tpr) < 1024) u.chunk /= 2;
  u.chunks = (int)((a.tokens + u.chunk - 1) / u.chunk);
  u.part_row = (a.channels + 3) / 4 * 4;
  u.chunk_groups = (u.chunks + kEmbThreads / u.tpr - 1) / (kEmbThreads / u.tpr);
  uint8_t *at = static_cast<uint8_t *>(workspace);
  auto take = [&](size_t bytes) {
    uint8_t *p = at + l.bytes;
    l.bytes += (bytes + 255) & ~(size_t)255;
    return p;
  };
  for (int k = 0; k < 2; k++) {
    s.key[k] = reinterpret_cast<uint32_t *>(take(sizeof(uint32_t) * (size_t)a.tokens));
    s.index[k] = reinterpret_cast<uint32_t *>(take(sizeof(uint32_t) * (size_t)a.tokens));
  }
  s.count = reinterpret_cast<uint32_t *>(take(sizeof(uint32_t) * kDigits * (size_t)s.tiles));
  u.part = reinterpret_cast<float *>(take(sizeof(float) * 2 * (size_t)u.chunks * u.part_row));
  u.key = s.key[s.passes & 1];
  u.index = s.index[s.passes & 1];
  return l;
}

template <typename TT, typename OT> struct EmbLaunch {
  // (a second launch only for more than 2^26 tokens)
  static void Forward(hipStream_t s, const daliamdEmbeddingArgs &all) {
    int tpr = 8;
    while (tpr < kEmbThreads && tpr * kEmbV < all.channels) tpr *= 2;
    const int64_t per_group = kEmbThreads / tpr, most = 4 * MaxWorkgroups(kEmbThreads) * per_group;
    KernelTimer timer("EmbeddingKernel", s);
    for (int64_t first = 0; first < all.tokens; first += most) {
      daliamdEmbeddingArgs a = all;
      a.tokens = std::min(most, all.tokens - first);
      a.ids = static_cast<const char *>(all.ids) + first * (all.index_dtype == DALIAMD_INT64 ? 8 : 4);
      a.out = static_cast<OT *>(all.out) + first * all.channels;
      ForwardPart(s, a, tpr, per_group);
    }
  }
  static void ForwardPart(hipStream_t s, const daliamdEmbeddingArgs &a, int tpr, int64_t per_group) {
    // four rows per thread where that still leaves workgroups for every compute unit
    if (a.tokens >= 4 * per_group * 1024) ForwardOf<4>(s, a, tpr, (a.tokens + 4 * per_group - 1) / (4 * per_group));
    else ForwardOf<1>(s, a, tpr, (a.tokens + per_group - 1) / per_group);
  }
  template <int kTokens> static void ForwardOf(hipStream_t s, const daliamdEmbeddingArgs &a, int tpr, int64_t groups) {
    const dim3 grid((unsigned)groups), block(kEmbThreads);
    const bool whole = a.channels % kEmbV == 0;
    if (a.index_dtype == DALIAMD_INT64) {
      if (whole) hipLaunchKernelGGL((EmbeddingKernel<TT, OT, int64_t, kTokens, true>), grid, block, 0, s, a, tpr);
      else hipLaunchKernelGGL((EmbeddingKernel<TT, OT, int64_t, kTokens, false>), grid, block, 0, s, a, tpr);
    } else {
      if (whole) hipLaunchKernelGGL((EmbeddingKernel<TT, OT, int32_t, kTokens, true>), grid, block, 0, s, a, tpr);
      else hipLaunchKernelGGL((EmbeddingKernel<TT, OT, int32_t, kTokens, false>), grid, block, 0, s, a, tpr);
    }
  }
  static void Backward(hipStream_t s, const daliamdEmbeddingArgs &a, const EmbSums &sums) {
    KernelTimer timer("EmbeddingBackwardKernel", s);
    EmbSums part = sums;
    do {   // (a second launch only for more than 2^29 rows)
      const int64_t rows = (a.vocab - part.first + kFillRows - 1) / kFillRows, fill = std::min(rows, MaxWorkgroups(kEmbThreads) - part.chunk_groups);
      const dim3 grid((unsigned)(part.chunk_groups + fill)), block(kEmbThreads);
      if (a.channels % kEmbV == 0) hipLaunchKernelGGL((EmbeddingBackwardKernel<TT, OT, true>), grid, block, 0, s, a, part);
      else hipLaunchKernelGGL((EmbeddingBackwardKernel<TT, OT, false>), grid, block, 0, s, a, part);
      part.first += fill * kFillRows;
      part.chunk_groups = 0;
    } while (part.first < a.vocab);
  }
};
template <typename F> static void WithTypes(const daliamdEmbeddingArgs &a, F f) {
  auto out = [&](auto table) {
    using TT = decltype(table);
    if (a.out_dtype == DALIAMD_FLOAT) f(EmbLaunch<TT, float>());
    else if (a.out_dtype == DALIAMD_FLOAT16) f(EmbLaunch<TT, F16>());
    else f(EmbLaunch<TT, Bf16>());
  };
  if (a.dtype == DALIAMD_FLOAT) out(float());
  else if (a.dtype == DALIAMD_FLOAT16) out(F16());
  else out(Bf16());
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
  const EmbLayout l = LayOut(a, nullptr);
  DALIAMD_REQUIRE(l.sums.chunk_groups < MaxWorkgroups(kEmbThreads), DALIAMD_ERROR_OUT_OF_RANGE, "daliamdEmbedding: more tokens and channels than one launch may have");
  plan->backward_workspace_bytes = l.bytes;
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
  WithTypes(*args, [&](auto launch) { launch.Forward(s, *args); });
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
  DALIAMD_REQUIRE((uintptr_t)workspace % 16 == 0, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdEmbeddingBackwardRun: the workspace must start at a multiple of 16 bytes");
  hipStream_t s = (hipStream_t)stream;
  const daliamdEmbeddingArgs &a = *args;
  const EmbLayout l = LayOut(a, workspace);
  const EmbSums &sums = l.sums;
  if (a.tokens && a.tokens <= kSmallTokens) {
    KernelTimer timer("EmbeddingSortKernel", s);
    hipLaunchKernelGGL(SortSmallKernel, dim3(1), dim3(kSmallThreads), 0, s, a, l.sort);
  } else if (a.tokens) {
    for (int pass = 0; pass < l.sort.passes; pass++) {
      KernelTimer timer("EmbeddingSortKernel", s);
      hipLaunchKernelGGL(SortCountKernel, dim3(l.sort.tiles), dim3(kSortThreads), 0, s, a, l.sort, pass);
      hipLaunchKernelGGL(SortScatterKernel, dim3(l.sort.tiles), dim3(kSortThreads), 0, s, a, l.sort, pass);
    }
  }
  WithTypes(a, [&](auto launch) { launch.Backward(s, a, sums); });
  if (sums.chunks > 1) {
    KernelTimer timer("EmbeddingJoinKernel", s);
    const int tiles = (a.channels + kJoinColumns - 1) / kJoinColumns;
    EmbSums part = sums;
    while (part.first < sums.chunks - 1) {   // (a second launch only for more than 2^29 tokens)
      const int64_t groups = std::min<int64_t>(sums.chunks - 1 - part.first, MaxWorkgroups(kJoinLanes * kJoinParts));
      hipLaunchKernelGGL(EmbeddingJoinKernel, dim3((unsigned)groups, (unsigned)(tiles < 65535 ? tiles : 65535)), dim3(kJoinLanes * kJoinParts), 0, s, a,
                         part);
      part.first += groups;
    }
  }
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

}  // extern "C"
