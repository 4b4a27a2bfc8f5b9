// What the kernels of learned type vectors share: element types that are computed with in float,
// several elements at a time, row numbers out of type indices, and the counter-based generator.
#ifndef LIBMOLGRID_AMD_ELEMENT_TYPES_H_
#define LIBMOLGRID_AMD_ELEMENT_TYPES_H_

#include "device_common.h"
#include "type_vector_args.h"

namespace mg {

// Arrays of 16-bit types are read and written as their bits; everything is computed in float and
// rounded once, to the nearest, where it is stored.
struct Half {
  uint16_t bits;
};
struct Bfloat16 {
  uint16_t bits;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(Half v) { return half_bits_to_float(v.bits); }
__device__ __forceinline__ float widen(Bfloat16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ Half narrow<Half>(float v) {
  return Half{float_to_half_bits(v)};
}
template <>
__device__ __forceinline__ Bfloat16 narrow<Bfloat16>(float v) {
  return Bfloat16{float_to_bfloat16_bits(v)};
}

// VEC elements that are loaded and stored by one instruction (or two, above 16 bytes), kept in
// whole words: as 16-bit numbers they would take a register each.
template <typename T, int VEC>
struct __align__(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
  static constexpr int kWords = sizeof(T) * VEC / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ float operator[](int i) const;
  __device__ __forceinline__ void set(const float (&v)[VEC]);
  __device__ __forceinline__ void zero_unless(bool keep) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = keep ? w[i] : 0u;
  }
};
template <typename T>
struct __align__(sizeof(T)) Pack<T, 1> {
  T v;
  __device__ __forceinline__ float operator[](int) const { return widen(v); }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = narrow<T>(f[0]); }
  __device__ __forceinline__ void zero_unless(bool keep) { v = keep ? v : T(); }
};
__device__ __forceinline__ float widen_word(uint32_t w, int, float) { return __uint_as_float(w); }
__device__ __forceinline__ float widen_word(uint32_t w, int upper, Half) {
  return half_bits_to_float((uint16_t)(upper ? w >> 16 : w));
}
__device__ __forceinline__ float widen_word(uint32_t w, int upper, Bfloat16) {
  return __uint_as_float(upper ? w & 0xFFFF0000u : w << 16);
}
__device__ __forceinline__ uint32_t narrow_word(float a, float b, Half) { return floats_to_half_bits(a, b); }
__device__ __forceinline__ uint32_t narrow_word(float a, float b, Bfloat16) {
  return floats_to_bfloat16_bits(a, b);
}
template <typename T, int VEC>
__device__ __forceinline__ float Pack<T, VEC>::operator[](int i) const {
  constexpr int kEach = 4 / sizeof(T);
  return widen_word(w[i / kEach], i % kEach, T());
}
template <typename T, int VEC>
__device__ __forceinline__ void Pack<T, VEC>::set(const float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (sizeof(T) == 4)
      w[i] = __float_as_uint(v[i]);
    else
      w[i] = narrow_word(v[2 * i], v[2 * i + 1], T());
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void load_floats(const T* p, float (&out)[VEC]) {
  const Pack<T, VEC> pack = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = pack[i];
}
template <typename T, int VEC>
__device__ __forceinline__ void store_floats(T* p, const float (&in)[VEC]) {
  Pack<T, VEC> pack;
  pack.set(in);
  *reinterpret_cast<Pack<T, VEC>*>(p) = pack;
}

// Row of the table that a type index names, or -1 for one that names none.  A float index counts
// as the whole number below it, as in the forward splat; not-a-number names no row.
__device__ __forceinline__ int table_row(float index, int nrows) {
  if (!(index >= 0.f && index < 2147483648.f)) return -1;
  const int row = (int)index;
  return row < nrows ? row : -1;
}
__device__ __forceinline__ int table_row(int32_t index, int nrows) {
  return (uint32_t)index < (uint32_t)nrows ? index : -1;
}
__device__ __forceinline__ int table_row(int64_t index, int nrows) {
  return (uint64_t)index < (uint64_t)nrows ? (int)index : -1;
}

__device__ __forceinline__ int token_row(const TokenArg& t, size_t n) {
  switch (t.index_kind) {   // (the same in every lane)
    case MG_INDEX_FLOAT32: return table_row(static_cast<const float*>(t.index)[n], t.nrows);
    case MG_INDEX_INT32: return table_row(static_cast<const int32_t*>(t.index)[n], t.nrows);
    default: return table_row(static_cast<const int64_t*>(t.index)[n], t.nrows);
  }
}

// Sum over the lanes of a wave, in every lane.
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = kWave / 2; m > 0; m /= 2) v += __shfl_xor(v, m);
  return v;
}

// Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011): four 32-bit words out of a 128-bit counter and a 64-bit key.
struct Words4 {
  uint32_t w[4];
};
__device__ __forceinline__ Words4 philox(uint64_t low, uint64_t high, uint64_t key) {
  uint32_t c0 = (uint32_t)low, c1 = (uint32_t)(low >> 32);
  uint32_t c2 = (uint32_t)high, c3 = (uint32_t)(high >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    const uint32_t n0 = xor3((uint32_t)(b >> 32), c1, k0), n2 = xor3((uint32_t)(a >> 32), c3, k1);
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words4{{c0, c1, c2, c3}};
}

__device__ __forceinline__ void drop_key(const DropArg& a, uint64_t& seed, uint64_t& offset) {
  seed = a.seed + (a.state ? a.state[0] : 0);   // (modulo 2^64)
  offset = a.offset + (a.state ? a.state[1] : 0);
}
__device__ __forceinline__ uint32_t drop_half(const Words4& words, int i) {
  return i & 1 ? words.w[i >> 1] >> 16 : words.w[i >> 1] & 0xFFFFu;
}

}  // namespace mg

#endif
