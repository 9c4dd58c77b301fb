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
// Rows start wherever their elements may: the hardware takes 8 and 16 byte accesses at any address, and the types say so.
typedef uint32_t UnalignedWords __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t UnalignedPair __attribute__((ext_vector_type(2), aligned(2)));
template <typename T, int V> __device__ __forceinline__ void LoadWide(Group<T, V> &g, const T *p) {
  constexpr int kWords = Group<T, V>::kWords;
  if constexpr (kWords % 4 == 0) {
#pragma unroll
    for (int k = 0; k < kWords / 4; k++) {
      const UnalignedWords w = reinterpret_cast<const UnalignedWords *>(p)[k];
#pragma unroll
      for (int i = 0; i < 4; i++) g.word[4 * k + i] = w[i];
    }
  } else {
    const UnalignedPair w = *reinterpret_cast<const UnalignedPair *>(p);
    g.word[0] = w[0], g.word[1] = w[1];
  }
}
template <typename T, int V> __device__ __forceinline__ void StoreWide(T *p, const float *f) {
  constexpr int kWords = Group<T, V>::kWords;
  Group<T, V> g;
#pragma unroll
  for (int j = 0; j < V; j++) g.Set(j, FromFloat<T>(f[j]));
  if constexpr (kWords % 4 == 0) {
#pragma unroll
    for (int k = 0; k < kWords / 4; k++)
      reinterpret_cast<UnalignedWords *>(p)[k] = UnalignedWords{g.word[4 * k], g.word[4 * k + 1], g.word[4 * k + 2], g.word[4 * k + 3]};
  } else {
    *reinterpret_cast<UnalignedPair *>(p) = UnalignedPair{g.word[0], g.word[1]};
  }
}

// The V channels that a thread has of a row, the `first`-th on.  Where the row ends inside them, the thread takes the row's last V
// and leaves those out that are another thread's: every load is a whole one, and none is conditional (a load under a condition is
// waited for where the condition ends).  Rows of fewer than V channels: one by one.
// WHOLE: the row's channels are a multiple of V; a thread has V of them or none.  Then stores need no second path either, whose
// branches would make the compiler wait for all memory operations in front of them.
template <int V, bool WHOLE = false> struct Channels {
  int base, begin, end;   // elements [begin, end) of the V from channel `base` on are this thread's; none: begin >= end
  bool narrow;
  __device__ __forceinline__ Channels(int first, int channels) {
    narrow = !WHOLE && channels < V;
    base = max(0, min(first, channels - V));
    begin = first - base;
    end = min(V, channels);
  }
  // (32 bits of bytes: a row that is the same in all lanes stays in scalar registers)
  template <typename T> __device__ __forceinline__ T *At(T *row, uint32_t offset = 0) const {
    typedef typename std::conditional<std::is_const<T>::value, const char, char>::type Byte;
    return reinterpret_cast<T *>(reinterpret_cast<Byte *>(row) + ((uint32_t)base + offset) * (uint32_t)sizeof(T));
  }
  template <typename T> __device__ __forceinline__ void Load(Group<T, V> &g, const T *row) const {
    if (narrow) {
#pragma unroll
      for (int j = 0; j < V; j++) g.Set(j, row[min(j, end - 1)]);
    } else {
      LoadWide(g, At(row));
    }
  }
  // zeros in the places of others
  template <typename T> __device__ __forceinline__ void Mask(Group<T, V> &g) const {
#pragma unroll
    for (int k = 0; k < Group<T, V>::kWords; k++) {
      if constexpr (WHOLE) {
        g.word[k] = begin == 0 ? g.word[k] : 0u;
      } else if constexpr (sizeof(T) == 4) {
        g.word[k] = k >= begin && k < end ? g.word[k] : 0u;
      } else {
        const uint32_t low = 2 * k >= begin && 2 * k < end ? 0xffffu : 0u, high = 2 * k + 1 >= begin && 2 * k + 1 < end ? 0xffff0000u : 0u;
        g.word[k] &= low | high;
      }
    }
  }
  // offset: elements that lanes are apart by already
  template <typename T> __device__ __forceinline__ void Store(T *row, const float *f, uint32_t offset = 0) const {
    if constexpr (WHOLE) {
      if (begin == 0) StoreWide<T, V>(At(row, offset), f);
    } else if (begin == 0 && end == V) {
      StoreWide<T, V>(At(row, offset), f);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (j >= begin && j < end) At(row, offset)[j] = FromFloat<T>(f[j]);
    }
  }
};

__device__ __forceinline__ float LoadElement(const void *p, int64_t i, int dtype) {
  return dtype == DALIAMD_FLOAT ? static_cast<const float *>(p)[i]
       : dtype == DALIAMD_FLOAT16 ? ToFloat(static_cast<const F16 *>(p)[i]) : ToFloat(static_cast<const Bf16 *>(p)[i]);
}
__device__ __forceinline__ void StoreElement(void *p, int64_t i, int dtype, float v) {
  if (dtype == DALIAMD_FLOAT) static_cast<float *>(p)[i] = v;
  else if (dtype == DALIAMD_FLOAT16) static_cast<F16 *>(p)[i] = FromFloat<F16>(v);
  else static_cast<Bf16 *>(p)[i] = FromFloat<Bf16>(v);
}

// workgroups of `threads` that one launch may have: its threads are counted in 32 bits
inline int64_t MaxWorkgroups(int threads) { return (((int64_t)1 << 32) - 1) / threads; }

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

// dense: the sequence that `row` belongs to, or -1 if it is padding
__device__ __forceinline__ int FindDenseSequence(const daliamdSequenceRows &q, int row, int *begin, int *end) {
  const int s = (uint32_t)row / (uint32_t)q.steps;
  SequenceRange(q, s, begin, end);
  return row < *end ? s : -1;
}

// The logistic function f(g) = 1 / (1 + exp(-g)) in the instructions that the hardware has for it: 2^x and 1 / x, each good to the
// last bit or two.  The product with log2(e) is off by 2^-24 of itself, which is |g| 2^-24 of the power; EXACT puts that back
// where the power is neither 0 nor infinity: there g may be infinite, or its product with log2(e).
__device__ __forceinline__ float PowerOf2(float v) {
#if defined(__AMDGCN__)
  return __builtin_amdgcn_exp2f(v);
#else
  return exp2f(v);
#endif
}
template <bool EXACT> __device__ __forceinline__ float ExpOf(float g) {
  constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
  const float p = g * kLog2e;
  float t = PowerOf2(p);
  if (EXACT) {
    const float more = t * (fmaf(g, kLog2e, -p) * kLn2);
    t += t > 0.0f && t < __builtin_inff() ? more : 0.0f;
  }
  return t;
}
__device__ __forceinline__ float Reciprocal(float v) {
#if defined(__AMDGCN__)
  return __builtin_amdgcn_rcpf(v);
#else
  return 1.0f / v;
#endif
}
// f and 1 - f, both to their last bits
__device__ __forceinline__ void LogisticPair(float g, float *f, float *k) {
  const float t = ExpOf<true>(-fabsf(g)), big = Reciprocal(1.0f + t), small = t * big;
  *f = g < 0 ? small : big;
  *k = g < 0 ? big : small;
}
// The smaller one of f and 1 - f, negative where that is f: of the other, which is near 1, it is all that matters.  To its last bits if EXACT;
// without, it is off by |g| 2^-24 of itself, a 2^-16th (bf16; f16: 2^-13th) of what the half step that g was rounded by makes of it.
template <bool EXACT> __device__ __forceinline__ float SmallerOfLogistic(float g) {
  return copysignf(Reciprocal(1.0f + ExpOf<EXACT>(fabsf(g))), g);
}
// g f(g)
__device__ __forceinline__ float Silu(float g) { return g * Reciprocal(1.0f + ExpOf<true>(-g)); }

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_SEQUENCE_COMMON_H_
