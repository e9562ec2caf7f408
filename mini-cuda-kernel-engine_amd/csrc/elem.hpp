// elem.hpp -- row elements in fp32, fp16 or bf16: 16-byte vectors at any element
// alignment, widened to float on load and rounded to nearest even once on store.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace mcke_amd {

template <typename T> constexpr int kVecElems = 16 / static_cast<int>(sizeof(T));

// 16 bytes of T at T's own alignment (gfx950 loads and stores them at any such address).
template <typename T> struct VecOf;
template <> struct VecOf<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct VecOf<__bf16> {
  typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct VecOf<_Float16> {
  typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2)));
};
template <typename T> using VecT16 = typename VecOf<T>::type;

// The vector's first `n` elements (n < kVecElems), `fill` behind them: the end of a row.
template <typename T>
__device__ __forceinline__ VecT16<T> load_part(const T* __restrict__ p, int n, float fill) {
  VecT16<T> v;
#pragma unroll
  for (int e = 0; e < kVecElems<T>; ++e) v[e] = e < n ? p[e] : static_cast<T>(fill);
  return v;
}

template <typename T>
__device__ __forceinline__ void store_part(T* __restrict__ p, VecT16<T> v, int n) {
#pragma unroll
  for (int e = 0; e < kVecElems<T>; ++e)
    if (e < n) p[e] = v[e];
}

template <typename T> __device__ __forceinline__ VecT16<T> load_vec(const T* __restrict__ p) {
  return *reinterpret_cast<const VecT16<T>*>(p);
}

// The same, for data that is touched once (non-temporal).
template <typename T> __device__ __forceinline__ VecT16<T> load_stream(const T* __restrict__ p) {
  return __builtin_nontemporal_load(reinterpret_cast<const VecT16<T>*>(p));
}
template <typename T> __device__ __forceinline__ void store_stream(T* __restrict__ p, VecT16<T> v) {
  __builtin_nontemporal_store(v, reinterpret_cast<VecT16<T>*>(p));
}

// N floats from p[c ..] (at P's alignment), or `none` where there is no p.
template <typename P, int N>
__device__ __forceinline__ void load_params(float (&v)[N], const P* __restrict__ p, int64_t c,
                                            float none) {
  constexpr int VE = kVecElems<P>;
  if (!p) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = none;
  } else if constexpr (N >= VE) {
#pragma unroll
    for (int q = 0; q < N / VE; ++q) {
      const VecT16<P> w = load_vec<P>(p + c + q * VE);
#pragma unroll
      for (int e = 0; e < VE; ++e) v[q * VE + e] = static_cast<float>(w[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = static_cast<float>(p[c + e]);
  }
}

// One element by its dtype, for vectors that are read once per row or launch.
__device__ __forceinline__ float load_elem(const void* __restrict__ p, int dtype, int64_t i) {
  if (dtype == MCKE_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == MCKE_DTYPE_F16) return static_cast<float>(static_cast<const _Float16*>(p)[i]);
  return static_cast<float>(static_cast<const __bf16*>(p)[i]);
}

inline bool is_dtype(int d) {
  return d == MCKE_DTYPE_F32 || d == MCKE_DTYPE_F16 || d == MCKE_DTYPE_BF16;
}
inline std::size_t dtype_bytes(int d) { return d == MCKE_DTYPE_F32 ? 4 : 2; }

// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
  const auto x = reinterpret_cast<std::uintptr_t>(a), y = reinterpret_cast<std::uintptr_t>(b);
  return a && b && na && nb && x < y + nb && y < x + na;
}

}  // namespace mcke_amd
