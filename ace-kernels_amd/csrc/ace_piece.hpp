// 16 bytes of neighbouring elements, as a lane loads and stores them: kept packed in
// four registers, so that rows on the way take no more of them than their bytes.
// Addresses need the elements' alignment only.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace ace {

template <typename T>
struct Piece {
  static constexpr int V = 16 / (int)sizeof(T);
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  Words words;

  __device__ float operator[](int e) const {  // e: a constant once unrolled
    if constexpr (std::is_same_v<T, float>) {
      return __uint_as_float(words[e]);
    } else if constexpr (std::is_same_v<T, __bf16>) {
      return __uint_as_float(e & 1 ? words[e / 2] & 0xffff0000u : words[e / 2] << 16);
    } else {
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(words[e / 2] >> (e & 1) * 16));
    }
  }
  // Each value rounded once.
  __device__ void set(const float (&x)[V]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int e = 0; e < V; ++e) words[e] = __float_as_uint(x[e]);
    } else {
      typedef T Two __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int e = 0; e < V; e += 2)
        words[e / 2] = __builtin_bit_cast(uint32_t, Two{(T)x[e], (T)x[e + 1]});
    }
  }
  __device__ void fill(T x) {
    typedef T All __attribute__((ext_vector_type(V)));
    All all;
#pragma unroll
    for (int e = 0; e < V; ++e) all[e] = x;
    words = __builtin_bit_cast(Words, all);
  }
  __device__ void load(const T* at) { __builtin_memcpy(&words, at, 16); }
  // STREAM: past the caches, where what a launch reads and writes would not fit the
  // last-level one anyway and drives out what is read.
  template <bool STREAM>
  __device__ void store(T* at) const {
    typedef uint32_t Unaligned __attribute__((ext_vector_type(4), aligned(2)));
    if constexpr (STREAM)
      __builtin_nontemporal_store(words, reinterpret_cast<Unaligned*>(at));
    else
      *reinterpret_cast<Unaligned*>(at) = words;
  }
  // The first n elements; the others are `rest`, or not stored.
  __device__ void load_some(const T* at, int64_t n, T rest) {
    typedef T All __attribute__((ext_vector_type(V)));
    All all;
#pragma unroll
    for (int e = 0; e < V; ++e) all[e] = e < n ? at[e] : rest;
    words = __builtin_bit_cast(Words, all);
  }
  __device__ void store_some(T* at, int64_t n) const {
    typedef T All __attribute__((ext_vector_type(V)));
    const All all = __builtin_bit_cast(All, words);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) at[e] = all[e];
  }
};

}  // namespace ace
