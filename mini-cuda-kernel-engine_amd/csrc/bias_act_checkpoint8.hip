// bias_act_checkpoint8.hip -- bias + activation whose input is kept in 8 bits for the backward
// pass, and that backward pass.
//
//   u = x + bias (fp32),  y = act(u)
//   saved: for each block of 32 columns of a row the smallest E >= -126 with |u| <= 448 * 2^E over
//   the block's finite values, as the byte E + 127, and u 2^-E in e4m3 (4 significant bits,
//   to nearest, ties to even; 448 is its largest value, so nothing is clipped).  Infinities and
//   NaN are saved as NaN.
//
//   u~ = code 2^E,  dx = dy act'(u~),  dbias = sum over rows of dx,  y~ = act(u~)
//
// The powers of two make the scaling exact both ways, so a value's only error is its rounding to
// e4m3 (at most 2^-4 relative; 2^-10 2^E absolute for what is small in its block).  Arithmetic
// is fp32, each output is rounded once, and dbias is added up in a fixed order.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "common.hpp"
#include "device_math.hpp"
#include "elem.hpp"

namespace mcke_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 32;                        // columns that share an exponent
constexpr int64_t kMaxCols = int64_t{1} << 24;

int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }

// ---------------------------------------------------------------------------
// Slopes.  Beyond |u| = 10 both GELUs' are 1, or less than 1e-20 from 0, so the argument is held
// there, where no power of it and no exponential overflows; a NaN passes through.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float held10(float v) {
  return v > 10.0f ? 10.0f : v < -10.0f ? -10.0f : v;
}

// d/dv [0.5 v (1 + tanh z)] with q = 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z)), z = sqrt(2/pi)
// (v + 0.044715 v^3):  q + v q (1 - q) 2 z'.  1 - q is e q with e = exp(-2 z): no cancellation
// where q is near 1, and with v held e is below 2^127.
__device__ __forceinline__ float gelu_tanh_slope(float v) {
  constexpr float c1 = -2.30220818520f;     // -2 log2(e) sqrt(2/pi)
  constexpr float c2 = -0.102943241596f;    // 0.044715 c1
  constexpr float d1 = 1.5957691216057308f; // 2 sqrt(2/pi)
  constexpr float d2 = 0.21406444881780073f;// 3 * 0.044715 d1
  v = held10(v);
  const float v2 = v * v;
  const float e = __builtin_amdgcn_exp2f(v * __builtin_fmaf(c2, v2, c1));
  const float q = __builtin_amdgcn_rcpf(1.0f + e);
  return __builtin_fmaf(v * __builtin_fmaf(d2, v2, d1), (e * q) * q, q);
}

// Phi(v) + v phi(v), Phi through erfc of |v| (device_math.hpp).
__device__ __forceinline__ float gelu_erf_slope(float v) {
  constexpr float kLog2e = 1.4426950408889634f;
  v = held10(v);
  const float half = 0.5f * erfc_nonneg(__builtin_fabsf(v) * 0.70710678118654752440f);
  const float cdf = v >= 0.0f ? 1.0f - half : half;
  const float pdf = 0.3989422804014327f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * v * v);
  return __builtin_fmaf(v, pdf, cdf);
}

template <int ACT> __device__ __forceinline__ float act_slope(float v) {
  if constexpr (ACT == kActNone) return v != v ? v : 1.0f;    // (a lost value has no gradient)
  else if constexpr (ACT == kActRelu) return v > 0.0f ? 1.0f : 0.0f;
  else if constexpr (ACT == kActGeluErf) return gelu_erf_slope(v);
  else return gelu_tanh_slope(v);
}

// ---------------------------------------------------------------------------
// A lane's vector of a row: columns j VE on.  Rows that are not whole vectors end in one that is
// cut at `n` and goes element by element.
// ---------------------------------------------------------------------------
template <int VE> struct Bytes;
template <> struct Bytes<4> {
  typedef unsigned type __attribute__((aligned(1)));
};
template <> struct Bytes<8> {
  typedef unsigned type __attribute__((ext_vector_type(2), aligned(1)));
};

template <typename T>
__device__ __forceinline__ void load_row(float (&v)[kVecElems<T>], const T* __restrict__ p, int n) {
  constexpr int VE = kVecElems<T>;
  VecT16<T> w;
  if (n == VE) w = load_stream<T>(p);
  else w = load_part<T>(p, n, 0.0f);
#pragma unroll
  for (int e = 0; e < VE; ++e) v[e] = static_cast<float>(w[e]);
}

template <typename T>
__device__ __forceinline__ void store_row(T* __restrict__ p, const float (&v)[kVecElems<T>], int n) {
  constexpr int VE = kVecElems<T>;
  VecT16<T> w;
#pragma unroll
  for (int e = 0; e < VE; ++e) w[e] = static_cast<T>(v[e]);
  if (n == VE) store_stream<T>(p, w);
  else store_part<T>(p, w, n);
}

struct Layout {
  int64_t rows;
  int cols, blocks, tpr_log2;         // blocks of a row; 2^tpr_log2 lanes a row
  const void* bias;
  int bias_dtype;
};

template <int VE>
__device__ __forceinline__ void load_bias(float (&b)[VE], const Layout& l, int c, int n) {
#pragma unroll
  for (int e = 0; e < VE; ++e)
    b[e] = l.bias && e < n ? load_elem(l.bias, l.bias_dtype, c + e) : -0.0f;
}

// ---------------------------------------------------------------------------
// Forward.  32 columns are 4 (16-bit types) or 8 neighbouring lanes.
// ---------------------------------------------------------------------------
template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void checkpoint8_fwd_kernel(
    const T* __restrict__ x, T* __restrict__ y, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ exponents, Layout l) {
  constexpr int VE = kVecElems<T>, LB = kBlock / VE;
  const int t = threadIdx.x & ((1 << l.tpr_log2) - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads >> l.tpr_log2);
  const int64_t c64 = ((static_cast<int64_t>(blockIdx.y) << l.tpr_log2) + t) * VE;
  // Lanes behind the row hold zeros: their block's exponent wants them.
  const int c = c64 < l.cols ? static_cast<int>(c64) : l.cols;
  const int n = l.cols - c < VE ? l.cols - c : VE;
  float b[VE];
  load_bias<VE>(b, l, c, n);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads >> l.tpr_log2) +
                   (threadIdx.x >> l.tpr_log2);
       r < l.rows; r += step) {
    float v[VE], u[VE];
    load_row<T>(v, x + r * l.cols + c, n);
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      u[e] = v[e] + b[e];
      const float a = __builtin_fabsf(u[e]);
      most = fmaxf(most, a < __builtin_inff() && e < n ? a : 0.0f);
    }
    most = wave_max<LB>(most);
    const int bits = __builtin_bit_cast(int, most);
    int ex = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0);   // 1.75: 448 = 1.75 * 2^8
    ex = ex < 1 ? 1 : ex;
    const float inv = __builtin_bit_cast(float, (254 - ex) << 23);
    int packed[VE / 4];
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) {
      float s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = u[4 * q + e];
        s[e] = __builtin_fabsf(w) < __builtin_inff() ? w * inv : __builtin_nanf("");
      }
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
      packed[q] = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], p, true);
    }
    uint8_t* to = codes + r * l.cols + c;
    if (n == VE) {
      using B = typename Bytes<VE>::type;
      if constexpr (VE == 4) *reinterpret_cast<B*>(to) = static_cast<unsigned>(packed[0]);
      else *reinterpret_cast<B*>(to) = B{static_cast<unsigned>(packed[0]),
                                         static_cast<unsigned>(packed[VE / 4 - 1])};
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e < n) to[e] = static_cast<uint8_t>(packed[e / 4] >> (8 * (e % 4)));
    }
    if (t % LB == 0 && n > 0)
      exponents[r * l.blocks + c / kBlock] = static_cast<uint8_t>(ex);
    if (y) {
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = act_xb<ACT>(v[e], b[e]);
      store_row<T>(y + r * l.cols + c, v, n);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward.  Workgroup (p, columns) walks the rows p per, p per + 1, .. of its part; a lane
// keeps its columns' sums of dx, and the workgroup's are row p of the workspace.
// ---------------------------------------------------------------------------
template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void checkpoint8_bwd_kernel(
    const T* __restrict__ dy, const uint8_t* __restrict__ codes,
    const uint8_t* __restrict__ exponents, T* __restrict__ dx, T* __restrict__ y,
    float* __restrict__ partials, Layout l, int64_t per) {
  constexpr int VE = kVecElems<T>;
  __shared__ float fold[kThreads * VE];
  const int tpr = 1 << l.tpr_log2, groups = kThreads >> l.tpr_log2;
  const int t = threadIdx.x & (tpr - 1), g = threadIdx.x >> l.tpr_log2;
  const int64_t c64 = ((static_cast<int64_t>(blockIdx.y) << l.tpr_log2) + t) * VE;
  const int c = c64 < l.cols ? static_cast<int>(c64) : l.cols;
  const int n = l.cols - c < VE ? l.cols - c : VE;
  const int64_t r0 = blockIdx.x * per, r1 = r0 + per < l.rows ? r0 + per : l.rows;
  float sum[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[e] = 0.0f;
  if (n > 0) {
#pragma unroll 2
    for (int64_t r = r0 + g; r < r1; r += groups) {
      const uint8_t* from = codes + r * l.cols + c;
      int packed[VE / 4];
      if (n == VE) {
        using B = typename Bytes<VE>::type;
        const B w = *reinterpret_cast<const B*>(from);
        if constexpr (VE == 4) {
          packed[0] = static_cast<int>(w);
        } else {
          packed[0] = static_cast<int>(w[0]);
          packed[1] = static_cast<int>(w[1]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < VE / 4; ++q) packed[q] = 0;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (e < n) packed[e / 4] |= from[e] << (8 * (e % 4));
      }
      const int ex = exponents[r * l.blocks + c / kBlock];
      const float scale = __builtin_bit_cast(float, ex << 23);
      float d[VE];
      if (dy) load_row<T>(d, dy + r * l.cols + c, n);
      float u[VE];
#pragma unroll
      for (int q = 0; q < VE / 4; ++q) {
        u[4 * q + 0] = scale * __builtin_amdgcn_cvt_f32_fp8(packed[q], 0);
        u[4 * q + 1] = scale * __builtin_amdgcn_cvt_f32_fp8(packed[q], 1);
        u[4 * q + 2] = scale * __builtin_amdgcn_cvt_f32_fp8(packed[q], 2);
        u[4 * q + 3] = scale * __builtin_amdgcn_cvt_f32_fp8(packed[q], 3);
      }
      if (dy) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          d[e] *= act_slope<ACT>(u[e]);
          sum[e] += d[e];
        }
        if (dx) store_row<T>(dx + r * l.cols + c, d, n);
      }
      if (y) {
#pragma unroll
        for (int e = 0; e < VE; ++e) u[e] = act_xb<ACT>(u[e], -0.0f);
        store_row<T>(y + r * l.cols + c, u, n);
      }
    }
  }
  if (!partials) return;
  if (groups > 1) {
    // The row groups' sums, in their order.
#pragma unroll
    for (int e = 0; e < VE; ++e) fold[e * kThreads + threadIdx.x] = sum[e];
    __syncthreads();
    if (g > 0) return;
    for (int k = 1; k < groups; ++k)
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += fold[e * kThreads + k * tpr + t];
  }
  float* to = partials + static_cast<int64_t>(blockIdx.x) * l.cols + c;
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (e < n) to[e] = sum[e];
}

// dbias from the workgroups' sums: kWays lanes a column, each every kWays-th part, then a tree.
constexpr int kFoldCols = 32, kFoldWays = 8;

__global__ __launch_bounds__(kFoldCols * kFoldWays) void checkpoint8_fold_kernel(
    const float* __restrict__ partials, void* __restrict__ dbias, int dtype, int64_t cols,
    int parts) {
  __shared__ float lds[kFoldWays][kFoldCols];
  const int lc = threadIdx.x % kFoldCols, way = threadIdx.x / kFoldCols;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kFoldCols + lc;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int p = way; p < parts; p += kFoldWays) s += partials[static_cast<int64_t>(p) * cols + c];
  }
  lds[way][lc] = s;
  __syncthreads();
  if (way > 0 || c >= cols) return;
  for (int w = 1; w < kFoldWays; ++w) s += lds[w][lc];
  if (dtype == MCKE_DTYPE_F32) static_cast<float*>(dbias)[c] = s;
  else if (dtype == MCKE_DTYPE_F16) static_cast<_Float16*>(dbias)[c] = static_cast<_Float16>(s);
  else static_cast<__bf16*>(dbias)[c] = static_cast<__bf16>(s);
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// Lanes a row: a power of two that covers the row's vectors, 8 (a block of fp32) to 256.
int lanes_log2(int64_t cols, int ve) {
  int log2 = 3;
  while (log2 < 8 && (int64_t{ve} << log2) < cols) ++log2;
  return log2;
}

// Parts of the rows whose sums of dx are kept apart.  (Of rows and cols alone: the workspace is
// sized without the type.)
int64_t parts_of(int64_t rows, int64_t cols) {
  const int64_t tiles = ceil_div(cols, 2048);
  int64_t parts = ceil_div(1024, tiles);
  if (parts > 256) parts = 256;
  const int64_t some = ceil_div(rows, 4);
  return parts < some ? parts : some;
}

template <class F> int with_types(int dtype, int act, F f) {
  auto with_dtype = [&](auto a) {
    if (dtype == MCKE_DTYPE_F32) return f(float{}, a);
    if (dtype == MCKE_DTYPE_F16) return f(_Float16{}, a);
    return f(__bf16{}, a);
  };
  if (act == kActNone) return with_dtype(std::integral_constant<int, kActNone>{});
  if (act == kActRelu) return with_dtype(std::integral_constant<int, kActRelu>{});
  if (act == kActGeluErf) return with_dtype(std::integral_constant<int, kActGeluErf>{});
  return with_dtype(std::integral_constant<int, kActGeluTanh>{});
}

int check_args(const std::string& who, int dtype, int bias_dtype, int64_t rows, int64_t cols,
               int act) {
  if (!is_dtype(dtype)) return invalid(who + ": unknown dtype " + std::to_string(dtype));
  if (bias_dtype != MCKE_DTYPE_F32 && bias_dtype != dtype)
    return invalid(who + ": bias_dtype must be MCKE_DTYPE_F32 or dtype, got " +
                   std::to_string(bias_dtype));
  if (act < MCKE_ACT_NONE || act > MCKE_ACT_GELU_TANH) return invalid(who + ": unknown Activation");
  if (rows < 0 || cols < 0) return invalid(who + ": negative extent");
  if (cols > kMaxCols || rows > INT32_MAX)
    return invalid(who + ": too large: rows up to 2^31 - 1, cols up to 2^24");
  return ok();
}

Layout layout_of(int64_t rows, int64_t cols, int dtype, const void* bias, int bias_dtype) {
  return {rows, static_cast<int>(cols), static_cast<int>(ceil_div(cols, kBlock)),
          lanes_log2(cols, 16 / static_cast<int>(dtype_bytes(dtype))), bias, bias_dtype};
}

}  // namespace
}  // namespace mcke_amd

using namespace mcke_amd;

extern "C" {

int mcke_launch_bias_act_checkpoint8(const void* x, const void* bias, void* y, uint8_t* codes,
                                     uint8_t* exponents, int dtype, int bias_dtype, int64_t rows,
                                     int64_t cols, int activation, void* stream) {
  const std::string who = "launch_bias_act_checkpoint8";
  if (int rc = check_args(who, dtype, bias_dtype, rows, cols, activation)) return rc;
  if (rows == 0 || cols == 0) return ok();
  if (!x || !codes || !exponents) return invalid(who + ": null pointer");
  const uint64_t e = dtype_bytes(dtype), be = dtype_bytes(bias_dtype), c = cols;
  const uint64_t n = static_cast<uint64_t>(rows) * c;
  const uint64_t blocks = static_cast<uint64_t>(rows) * ceil_div(cols, kBlock);
  if (!aligned(x, e) || !aligned(y, e) || !aligned(bias, be))
    return invalid(who + ": a pointer is not aligned to its type");
  const void* outs[] = {y, codes, exponents};
  const uint64_t out_bytes[] = {n * e, n, blocks};
  for (int i = 0; i < 3; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], x, n * e) || overlap(outs[i], out_bytes[i], bias, c * be);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid(who + ": an output overlaps another operand, which violates the "
                           "__restrict__ contract");
  }
  const Layout l = layout_of(rows, cols, dtype, bias, bias_dtype);
  const int ve = 16 / static_cast<int>(e);
  const int64_t gy = ceil_div(ceil_div(cols, ve), int64_t{1} << l.tpr_log2);
  const int64_t groups = ceil_div(rows, kThreads >> l.tpr_log2);
  const int64_t most = ceil_div(4096, gy);       // then they walk the rows
  const dim3 grid(static_cast<unsigned>(groups < most ? groups : most), static_cast<unsigned>(gy));
  return with_types(dtype, activation, [&](auto t, auto act) {
    using T = decltype(t);
    checkpoint8_fwd_kernel<T, decltype(act)::value>
        <<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const T*>(x), static_cast<T*>(y), codes, exponents, l);
    MCKE_LAUNCH_CHECK("checkpoint8_fwd_kernel");
    return ok();
  });
}

size_t mcke_bias_act_checkpoint8_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || rows > INT32_MAX || cols <= 0 || cols > kMaxCols) return 0;
  return static_cast<size_t>(parts_of(rows, cols)) * static_cast<size_t>(cols) * 4;
}

int mcke_launch_bias_act_checkpoint8_backward(const void* dy, const uint8_t* codes,
                                              const uint8_t* exponents, void* dx, void* y,
                                              void* dbias, int dtype, int bias_dtype, int64_t rows,
                                              int64_t cols, int activation, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  const std::string who = "launch_bias_act_checkpoint8_backward";
  if (int rc = check_args(who, dtype, bias_dtype, rows, cols, activation)) return rc;
  if (cols == 0) return ok();
  if (!dx && !y && !dbias) return invalid(who + ": no output is asked for");
  if (rows > 0 && (!codes || !exponents)) return invalid(who + ": null pointer");
  if (rows > 0 && (dx || dbias) && !dy) return invalid(who + ": dx and dbias need dy");
  const uint64_t e = dtype_bytes(dtype), be = dtype_bytes(bias_dtype), c = cols;
  const uint64_t n = static_cast<uint64_t>(rows) * c;
  const uint64_t blocks = static_cast<uint64_t>(rows) * ceil_div(cols, kBlock);
  if (!aligned(dy, e) || !aligned(dx, e) || !aligned(y, e) || !aligned(dbias, be))
    return invalid(who + ": a pointer is not aligned to its type");
  const size_t need =
      dbias ? mcke_bias_act_checkpoint8_backward_workspace_bytes(rows, cols) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return invalid(who + ": dbias needs a 16-byte aligned workspace of " + std::to_string(need) +
                   " bytes, got " + std::to_string(workspace ? workspace_bytes : 0));
  const void* outs[] = {dx, y, dbias, need > 0 ? workspace : nullptr};
  const uint64_t out_bytes[] = {n * e, n * e, c * be, need};
  for (int i = 0; i < 4; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], dy, n * e) || overlap(outs[i], out_bytes[i], codes, n) ||
               overlap(outs[i], out_bytes[i], exponents, blocks);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid(who + ": an output or the workspace overlaps another operand, which violates "
                           "the __restrict__ contract");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t parts = rows > 0 ? parts_of(rows, cols) : 0;
  if (rows > 0) {
    const Layout l = layout_of(rows, cols, dtype, nullptr, bias_dtype);
    const int ve = 16 / static_cast<int>(e);
    const int64_t gy = ceil_div(ceil_div(cols, ve), int64_t{1} << l.tpr_log2);
    const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(gy));
    const int64_t per = ceil_div(rows, parts);
    // Without dx or dbias, dy is not looked at.
    const void* grad = dx || dbias ? dy : nullptr;
    const int rc = with_types(dtype, activation, [&](auto t, auto act) {
      using T = decltype(t);
      checkpoint8_bwd_kernel<T, decltype(act)::value><<<grid, kThreads, 0, s>>>(
          static_cast<const T*>(grad), codes, exponents, static_cast<T*>(dx), static_cast<T*>(y),
          dbias ? static_cast<float*>(workspace) : nullptr, l, per);
      MCKE_LAUNCH_CHECK("checkpoint8_bwd_kernel");
      return ok();
    });
    if (rc) return rc;
  }
  if (!dbias) return ok();
  checkpoint8_fold_kernel<<<static_cast<unsigned>(ceil_div(cols, kFoldCols)),
                            kFoldCols * kFoldWays, 0, s>>>(static_cast<const float*>(workspace),
                                                           dbias, bias_dtype, cols,
                                                           static_cast<int>(parts));
  MCKE_LAUNCH_CHECK("checkpoint8_fold_kernel");
  return ok();
}

}  // extern "C"
