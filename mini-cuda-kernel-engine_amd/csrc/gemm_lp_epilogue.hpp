// gemm_lp_epilogue.hpp -- what a 16-bit-input product does with a tile of sums before its
// one store:
//
//   y = act(alpha acc + bias[col]) + residual
//
// in fp32, rounded once to the output's type.  alpha acc is rounded to fp32 before the bias is added,
// as the plain product that stores it and the fp32 product's epilogue do, and what is absent adds -0,
// which changes nothing: with the sums of the plain product (few rows and odd extents take other
// kernels) a fp32 output has the bits of that product and mcke_launch_bias_act_f32.  The kernels take
// it as a template argument: NoEpilogue is the plain product (C = alpha A B + beta C), Epilogue this.
//
// The sums leave the accumulation registers as fp32 through LDS, row-major, and a rolled loop
// reads them back a row at a time.  There the lane's columns do not change, so the bias is
// loaded once; the residual's loads and the stores are whole rows of 16 bytes a lane; and the
// activation's code is there once per activation and not once per accumulator (written over
// the registers, 256 accumulators times four activations are 60 KB of code that each
// workgroup runs through once).
#pragma once

#include <hip/hip_runtime.h>

#include "device_math.hpp"
#include "elem.hpp"

namespace mcke_amd {

struct NoEpilogue {
  static constexpr bool kFused = false;
};

struct Epilogue {
  static constexpr bool kFused = true;
  const void* bias;        // n values of bias_dtype, or null
  const void* residual;    // m x n values of the output type, or null; may be the output
  int bias_dtype;
  int act;
};

// act(v + bias) + residual for one output, v = alpha acc: a register's value behind the empty asm, so
// that the product does not go into one multiply-add with the bias.  (The activation's extra
// operation a value, bf16 with GELU_erf and residual, us: 4096^3 123.9 -> 124.5-125.4, 8192 x 4096 x
// 128 82.7 -> 84.1; a volatile asm, which orders them too, 125.2 and 85.3.)
constexpr float kAbsent = -0.0f;
template <int ACT> __device__ __forceinline__ float fused_value(float v, float b, float res) {
  asm("" : "+v"(v));
  return act_xb<ACT>(v, b) + res;
}

// Calls f with the activation as a constant.
template <class F> __device__ __forceinline__ void with_act(int act, F f) {
  if (act == kActNone) f(std::integral_constant<int, kActNone>{});
  else if (act == kActRelu) f(std::integral_constant<int, kActRelu>{});
  else if (act == kActGeluErf) f(std::integral_constant<int, kActGeluErf>{});
  else f(std::integral_constant<int, kActGeluTanh>{});
}

// A pass of TR rows by BN columns of fp32 sums in LDS.  16-byte quad q of row r is at
// q ^ (r % 16): writers put quads of 16 rows side by side, readers take whole rows, and
// neither meets a bank twice.
template <int BN> __device__ __forceinline__ int sum_at(int r, int q) {
  return r * BN + 4 * (q ^ (r & 15));
}

// The stores of a pass: LDS row r is tile row `row_of(r)`, columns n_first .. min(n0 + BN, N) - 1 of
// the tile at (m0, n0).  THREADS lanes; every lane of the workgroup makes one and calls both of its
// functions.
//
// The residual's loads go out U rows at a time, the first ones before the sums are in LDS (they
// wait for nothing but the K loop) and the others behind the rows at work.  4000 x 4004 x 1000 bf16
// with a residual 61.6 -> 52.0 us (its last tile column, whose vectors belong to two tiles in part,
// had loaded element by element), 1531 x 2053 x 1021 to fp32 43.1 -> 37.7.
template <typename OutT, int TR, int BN, int THREADS, class RowOf>
struct FusedStore {
  static constexpr int VE = kVecElems<OutT>;
  static constexpr int kLanes = BN / VE, kRows = THREADS / kLanes, kSteps = TR / kRows;
  static constexpr int U = kSteps < 8 ? kSteps : 8;
  static_assert(THREADS % kLanes == 0 && TR % kRows == 0 && kSteps % U == 0, "whole steps");

  const Epilogue& ep;
  RowOf row_of;
  int M, N, m0, n_first, lr, lc, col;
  bool inside, whole;                   // the vector lies in the row; all of it is this tile's
  VecT16<OutT> old[U];

  __device__ __forceinline__ FusedStore(const Epilogue& ep_, RowOf row_of_, int M_, int N_, int m0_,
                                        int n0, int n_first_)
      : ep(ep_), row_of(row_of_), M(M_), N(N_), m0(m0_), n_first(n_first_) {
    lr = threadIdx.x / kLanes;
    lc = VE * (threadIdx.x % kLanes);
    col = n0 + lc;
    inside = col + VE <= N;
    whole = inside && col >= n_first;
  }

  // The residual of steps s .. s + U - 1.  Rows past M and columns of the tile before are loaded
  // (row M - 1 in their place) and not used.
  __device__ __forceinline__ void load_residual(int s, VecT16<OutT> (&to)[U]) const {
    const OutT* res = static_cast<const OutT*>(ep.residual);
    if (!res || !inside) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = m0 + row_of(lr + (s + u) * kRows);
      to[u] = load_vec<OutT>(res + static_cast<int64_t>(row < M ? row : M - 1) * N + col);
    }
  }

  __device__ __forceinline__ void begin() { load_residual(0, old); }

  __device__ __forceinline__ void finish(const float* sums, OutT* C, float alpha) {
    const OutT* res = static_cast<const OutT*>(ep.residual);
    float b[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e)
      b[e] = ep.bias && col + e < N ? load_elem(ep.bias, ep.bias_dtype, col + e) : kAbsent;
    with_act(ep.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
#pragma unroll 1
      for (int s = 0; s < kSteps; s += U) {
        VecT16<OutT> next[U];
        if (s + U < kSteps) load_residual(s + U, next);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = lr + (s + u) * kRows, row = m0 + row_of(r);
          if (row >= M) continue;
          float v[VE];
#pragma unroll
          for (int q = 0; q < VE / 4; ++q) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(sums + sum_at<BN>(r, lc / 4 + q));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * q + e] = alpha * a[e];
          }
          OutT* p = C + static_cast<int64_t>(row) * N + col;
          VecT16<OutT> o;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            float old_e = kAbsent;
            if (res && inside) old_e = static_cast<float>(old[u][e]);
            else if (res && col + e < N)
              old_e = static_cast<float>(res[static_cast<int64_t>(row) * N + col + e]);
            o[e] = static_cast<OutT>(fused_value<ACT>(v[e], b[e], old_e));
          }
          if (whole) {
            *reinterpret_cast<VecT16<OutT>*>(p) = o;
          } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
              if (col + e >= n_first && col + e < N) p[e] = o[e];
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) old[u] = next[u];
      }
    });
  }
};

template <typename OutT, int TR, int BN, int THREADS, class RowOf>
__device__ __forceinline__ FusedStore<OutT, TR, BN, THREADS, RowOf> fused_store(
    const Epilogue& ep, RowOf row_of, int M, int N, int m0, int n0, int n_first) {
  return FusedStore<OutT, TR, BN, THREADS, RowOf>(ep, row_of, M, N, m0, n0, n_first);
}

}  // namespace mcke_amd
