// Shared by the sequence operators (recurrence, block norm, embedding): element types, rows of sequences, the logistic
// function.  Internal; not part of the C ABI.
#ifndef DALI_AMD_CSRC_SEQUENCE_COMMON_H_
#define DALI_AMD_CSRC_SEQUENCE_COMMON_H_

#include <type_traits>
#include "common.h"

namespace daliamd {

struct Bf16 { uint16_t bits; };
typedef _Float16 F16;

__device__ __forceinline__ float BitsToFloat(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(F16 v) { return (float)v; }
__device__ __forceinline__ float ToFloat(Bf16 v) { return BitsToFloat((uint32_t)v.bits << 16); }

template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ F16 FromFloat<F16>(float v) { return (F16)v; }
template <> __device__ __forceinline__ Bf16 FromFloat<Bf16>(float v) {
#if defined(__AMDGCN__)
  return Bf16{__builtin_bit_cast(uint16_t, (__bf16)v)};   // one instruction on gfx950: to nearest, ties to even
#else
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return Bf16{(uint16_t)((u >> 16) | 0x40u)};
  return Bf16{(uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16)};
#endif
}

// V adjacent elements in registers, as they are in memory; read and written 8 or 16 bytes at a time where that is possible
template <typename T, int V> struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Group {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  uint32_t word[kWords];
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (sizeof(T) == 4) {
      return BitsToFloat(word[j]);
    } else {
      const uint32_t w = word[j / 2];
      if constexpr (std::is_same<T, Bf16>::value) return BitsToFloat(j & 1 ? w & 0xffff0000u : w << 16);
      else return (float)__builtin_bit_cast(F16, (uint16_t)(j & 1 ? w >> 16 : w));
    }
  }
  __device__ __forceinline__ void Set(int j, T v) {
    if constexpr (sizeof(T) == 4) {
      word[j] = __builtin_bit_cast(uint32_t, v);
    } else {
      const uint32_t h = __builtin_bit_cast(uint16_t, v);
      word[j / 2] = j & 1 ? (word[j / 2] & 0xffffu) | h << 16 : h;   // (in ascending order of j)
    }
  }
  // The compiler keeps elements that it has unpacked once for a second use, in twice as many registers; after this it does not
  // know that they are the same.
  __device__ __forceinline__ void Repack() {
#if defined(__AMDGCN__)
    if constexpr (sizeof(T) < 4) {
#pragma unroll
      for (int k = 0; k < kWords; k++) asm volatile("" : "+v"(word[k]));
    }
#endif
  }
};
template <int BYTES> __device__ __forceinline__ void CopyWide(void *to, const void *from) {
  if (BYTES % 16 == 0) {
#pragma unroll
    for (int k = 0; k < BYTES / 16; k++) static_cast<uint4 *>(to)[k] = static_cast<const uint4 *>(from)[k];
  } else {
    *static_cast<uint2 *>(to) = *static_cast<const uint2 *>(from);
  }
}
template <typename T, int V> __device__ __forceinline__ void LoadWide(Group<T, V> &g, const T *p) { CopyWide<sizeof(g)>(&g, p); }
template <typename T, int V> __device__ __forceinline__ void StoreWide(T *p, const float *f) {
  Group<T, V> g;
#pragma unroll
  for (int j = 0; j < V; j++) g.Set(j, FromFloat<T>(f[j]));
  CopyWide<sizeof(g)>(p, &g);
}

// Which channels a thread of a row has, in `n` pieces of V: adjacent ones where every row of every tensor can be read 16 bytes
// at a time (`wide`), else every `threads`-th, so that a wave's loads of single elements are adjacent.
struct ChannelMap {
  int channels, threads, lane;
  bool wide;
  template <int V> __device__ __forceinline__ int First(int i) const { return wide ? (i * threads + lane) * V : i * V * threads + lane; }
  __device__ __forceinline__ int Step() const { return wide ? 1 : threads; }
};
template <typename T, int V> __device__ __forceinline__ void LoadChannels(Group<T, V> &g, const T *row, const ChannelMap &m, int i) {
  const int c = m.First<V>(i);
  if (m.wide) {
    if (c < m.channels) {
      LoadWide(g, row + c);
      return;
    }
#pragma unroll
    for (int j = 0; j < V; j++) g.Set(j, FromFloat<T>(0.0f));
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) g.Set(j, c + j * m.threads < m.channels ? row[c + j * m.threads] : FromFloat<T>(0.0f));
  }
}
template <typename T, int V> __device__ __forceinline__ void StoreChannels(T *row, const ChannelMap &m, int i, const float *f) {
  const int c = m.First<V>(i);
  if (m.wide) {
    if (c < m.channels) StoreWide<T, V>(row + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < V; j++)
      if (c + j * m.threads < m.channels) row[c + j * m.threads] = FromFloat<T>(f[j]);
  }
}
// whether rows of `elem`-byte elements, `stride` elements apart, all start at multiples of `bytes` bytes
inline bool RowsAligned(const void *p, int64_t stride, int elem, int bytes = 16) {
  return ((reinterpret_cast<uintptr_t>(p) | (uint64_t)(stride * elem)) & (bytes - 1)) == 0;
}

__device__ __forceinline__ float LoadElement(const void *p, int64_t i, int dtype) {
  return dtype == DALIAMD_FLOAT ? static_cast<const float *>(p)[i]
       : dtype == DALIAMD_FLOAT16 ? ToFloat(static_cast<const F16 *>(p)[i]) : ToFloat(static_cast<const Bf16 *>(p)[i]);
}
__device__ __forceinline__ void StoreElement(void *p, int64_t i, int dtype, float v) {
  if (dtype == DALIAMD_FLOAT) static_cast<float *>(p)[i] = v;
  else if (dtype == DALIAMD_FLOAT16) static_cast<F16 *>(p)[i] = FromFloat<F16>(v);
  else static_cast<Bf16 *>(p)[i] = FromFloat<Bf16>(v);
}

inline bool IsSequenceType(int dtype) { return dtype == DALIAMD_FLOAT || dtype == DALIAMD_FLOAT16 || dtype == DALIAMD_BFLOAT16; }
inline int ElementSize(int dtype) { return dtype == DALIAMD_FLOAT ? 4 : 2; }

__device__ __forceinline__ int64_t LoadIndex(const void *p, int64_t i, int dtype) {
  return dtype == DALIAMD_INT64 ? static_cast<const int64_t *>(p)[i] : (int64_t) static_cast<const int32_t *>(p)[i];
}

// the rows [begin, end) of sequence s, whatever the device holds in offsets / lengths
__device__ __forceinline__ int ClampRow(int64_t v, int64_t rows) { return (int)min(max(v, (int64_t)0), rows); }
__device__ __forceinline__ void SequenceRange(const daliamdSequenceRows &q, int s, int *begin, int *end) {
  if (q.offsets) {
    *begin = ClampRow(LoadIndex(q.offsets, s, q.index_dtype), q.rows);
    *end = max(*begin, ClampRow(LoadIndex(q.offsets, s + 1, q.index_dtype), q.rows));
  } else {
    *begin = s * (int)q.steps;
    *end = *begin + (q.lengths ? ClampRow(LoadIndex(q.lengths, s, q.index_dtype), q.steps) : (int)q.steps);
  }
}

// the sequence that `row` belongs to, or -1: with ascending offsets the last one that begins at or before it
__device__ __forceinline__ int FindSequence(const daliamdSequenceRows &q, int row, int *begin, int *end) {
  int s;
  if (q.offsets) {
    int lo = 0, hi = q.sequences - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (LoadIndex(q.offsets, mid, q.index_dtype) <= row) lo = mid; else hi = mid - 1;
    }
    s = lo;
  } else {
    s = (uint32_t)row / (uint32_t)q.steps;
  }
  SequenceRange(q, s, begin, end);
  return *begin <= row && row < *end ? s : -1;
}

__device__ __forceinline__ float Exp(float v) { return expf(v); }
// f = 1 / (1 + exp(-g)) and k = 1 - f, both to the last bits: k is small where a gate holds, and it is what h moves by
__device__ __forceinline__ void Logistic(float g, float *f, float *k) {
  const float t = Exp(-fabsf(g)), big = 1.0f / (1.0f + t), small = t * big;
  *f = g < 0 ? small : big;
  *k = g < 0 ? big : small;
}

// 1 - f alone, in the instructions that the hardware has for it.  The product with log2(e) is off by 2^-24 of itself, which is
// |g| 2^-24 of the result: EXACT puts that back.
template <bool EXACT> __device__ __forceinline__ float OneMinusLogistic(float g) {
  constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
#if defined(__AMDGCN__)
  const float p = g * kLog2e;
  float t = __builtin_amdgcn_exp2f(p);
  if (EXACT) {
    const float more = t * (fmaf(g, kLog2e, -p) * kLn2);
    t += t < __builtin_inff() ? more : 0.0f;
  }
  return __builtin_amdgcn_rcpf(1.0f + t);
#else
  return (float)(1.0 / (1.0 + exp((double)g)));
#endif
}

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_SEQUENCE_COMMON_H_
