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

// N values at the alignment of one.
template <typename T, int N> struct Pack {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N> using PackT = typename Pack<T, N>::type;

template <typename T, int N>
__device__ __forceinline__ void load_cols(float (&v)[N], const T* __restrict__ p) {
  const PackT<T, N> w = *reinterpret_cast<const PackT<T, N>*>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = static_cast<float>(w[e]);
}

// A lane's N columns of a row: columns j N .. j N + N - 1.  In rows that are not whole vectors
// (WHOLE false) the last one is moved back to end with the row, and its first `skip` columns are
// its neighbour's too; a row shorter than a vector is one vector cut at `n`.
template <int N, bool WHOLE> struct Cols {
  int c, skip, n;
  bool any;
  __device__ __forceinline__ Cols(int64_t j, int cols) {
    const int64_t first = j * N;
    any = first < cols;
    c = static_cast<int>(first);
    skip = 0;
    n = N;
    if constexpr (!WHOLE) {
      if (first + N > cols) {
        c = cols > N ? cols - N : 0;
        skip = static_cast<int>(first) - c;
        n = cols < N ? cols : N;
      }
    }
  }
  // Calls f(e) for the columns that are this lane's alone, or (ALL) all of its columns.  (The
  // bounds go through an empty asm: as masks kept over a kernel they fill the scalar file.)
  template <bool ALL, class F> __device__ __forceinline__ void each(F f) const {
    int from = ALL ? 0 : skip, to = n;
    asm("" : "+v"(from), "+v"(to));
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e >= from && e < to) f(e);
  }
  template <typename T> __device__ __forceinline__ PackT<T, N> load_raw(const T* row) const {
    if (WHOLE || n == N)
      return __builtin_nontemporal_load(reinterpret_cast<const PackT<T, N>*>(row + c));
    PackT<T, N> w{};
    each<true>([&](int e) { w[e] = row[c + e]; });
    return w;
  }
  template <typename T>
  __device__ __forceinline__ void load_stream(float (&v)[N], const T* row) const {
    const PackT<T, N> w = load_raw(row);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = static_cast<float>(w[e]);
  }
  template <typename T> __device__ __forceinline__ void load(float (&v)[N], const T* row) const {
    if (WHOLE || n == N) {
      load_cols<T, N>(v, row + c);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = 0.0f;
      each<true>([&](int e) { v[e] = static_cast<float>(row[c + e]); });
    }
  }
  // All of the lane's columns, those of its neighbour too, which has the same values for them.
  template <typename T>
  __device__ __forceinline__ void store_stream_again(T* row, const float (&v)[N]) const {
    PackT<T, N> w;
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = static_cast<T>(v[e]);
    if (WHOLE || n == N)
      __builtin_nontemporal_store(w, reinterpret_cast<PackT<T, N>*>(row + c));
    else
      each<true>([&](int e) { row[c + e] = w[e]; });
  }
  // The columns that are this lane's alone, so that each is written once.
  template <typename T> __device__ __forceinline__ void store(T* row, const float (&v)[N]) const {
    PackT<T, N> w;
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = static_cast<T>(v[e]);
    if (WHOLE || (skip == 0 && n == N))
      *reinterpret_cast<PackT<T, N>*>(row + c) = w;
    else
      each<false>([&](int e) { row[c + e] = w[e]; });
  }
};

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
