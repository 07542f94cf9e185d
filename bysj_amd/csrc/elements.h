// Elements of float32, bfloat16 and float16 tensors in vectors, whole or ragged,
// at any element alignment (device code of the expert and block-norm operators).
#pragma once

#include "common.h"

namespace dpa4k {

// The host's element types (DPA4K_TYPE_*) as a type argument.
template <typename T>
struct type_of {
  typedef T type;
};

// Calls `use(type_of<T>{})` with the element type of `code`; `otherwise` for an
// unknown one.
template <typename F>
inline int with_type(int code, int otherwise, F&& use) {
  switch (code) {
    case DPA4K_TYPE_F32: return use(type_of<float>{});
    case DPA4K_TYPE_BF16: return use(type_of<__bf16>{});
    case DPA4K_TYPE_F16: return use(type_of<_Float16>{});
  }
  return otherwise;
}

inline bool known_type(int code) { return code == DPA4K_TYPE_F32 || code == DPA4K_TYPE_BF16 || code == DPA4K_TYPE_F16; }
inline int64_t size_of_type(int code) { return code == DPA4K_TYPE_F32 ? 4 : 2; }

// N elements at element alignment: one wide access (the memory unit takes any
// alignment; a row of an odd width starts anywhere).
template <typename T, int N>
struct pack_of {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
using Pack = typename pack_of<T, N>::type;

template <typename T, int N>
struct zero_pack_of {
  static __device__ __forceinline__ Pack<T, N> get() {
    Pack<T, N> out;
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = static_cast<T>(0.0f);
    return out;
  }
};

// The first `live` of N elements at p, zeros behind them; `room` elements may be
// read from p on (a ragged row's neighbour is read along with it and masked).
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* __restrict__ p, int live, int64_t room) {
  Pack<T, N> out = zero_pack_of<T, N>::get();
  if (live >= N) {
    out = *reinterpret_cast<const Pack<T, N>*>(p);
  } else if (live > 0) {
    if (room >= N) {
      out = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
      for (int j = 1; j < N; ++j) out[j] = j < live ? out[j] : static_cast<T>(0.0f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < live) out[j] = p[j];
    }
  }
  return out;
}

// N floats, of which the first `live` are stored.  STREAM: past the caches, for
// outputs that the same kernel's loads would otherwise be displaced by.
template <bool STREAM, typename T, int N>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float (&value)[N], int live) {
  Pack<T, N> out;
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = static_cast<T>(value[j]);
  if (live >= N) {
    if constexpr (STREAM) __builtin_nontemporal_store(out, reinterpret_cast<Pack<T, N>*>(p));
    else *reinterpret_cast<Pack<T, N>*>(p) = out;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < live) p[j] = out[j];
  }
}

// Row and piece of piece `at` of rows of `pieces`: divided in 32 bits where `short_`,
// the same for the launch, says that all numbers fit.
__device__ __forceinline__ void split_piece(int64_t at, int64_t pieces, bool short_, int64_t& row, int64_t& piece) {
  if (short_) {
    const uint32_t quotient = static_cast<uint32_t>(at) / static_cast<uint32_t>(pieces);
    row = quotient;
    piece = static_cast<uint32_t>(at) - quotient * static_cast<uint32_t>(pieces);
  } else {
    row = at / pieces;
    piece = at - row * pieces;
  }
}

// 1 / (1 + exp(-x)) to about two roundings, NaN for NaN.  The product x log2(e) is
// carried with its rounding error; past +-88 the result is 0 (6e-39) and 1;
// exp(90) would be infinite and its rounding error NaN.
// `other`: 1 minus it, with all its digits where the result is near 1.
__device__ __forceinline__ float logistic(float x, float& other) {
  constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147182f;
  x = x < -88.0f ? -88.0f : x;
  x = x > 88.0f ? 88.0f : x;
  const float t = -x * kLog2e;
  const float rest = fmaf(-x, kLog2eRest, fmaf(-x, kLog2e, -t));
  float e = __builtin_amdgcn_exp2f(t);
  e = fmaf(e, rest * kLn2, e);
  const float s = __builtin_amdgcn_rcpf(1.0f + e);
  other = x < -80.0f ? 1.0f : e * s;   // s may be 0 there
  return s;
}

__device__ __forceinline__ float logistic(float x) {
  float other;
  return logistic(x, other);
}

}  // namespace dpa4k
