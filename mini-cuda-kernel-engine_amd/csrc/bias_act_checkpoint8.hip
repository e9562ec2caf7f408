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
// Activations with their slopes.  Beyond |v| = 10 both GELUs' slopes are 1, or less than 1e-20 from
// 0, so the argument of what needs it is held there, where no power of it and no exponential
// overflows; a NaN passes through.  Far below 0 the value is 0, whatever v is (-infinity where a
// code stands for -2^128): what is left of q or of the erfc is multiplied by a v that is held too.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float held10(float v) {
  return v > 10.0f ? 10.0f : v < -10.0f ? -10.0f : v;
}

template <int ACT> __device__ __forceinline__ void act_and_slope(float v, float& y, float& slope) {
  if constexpr (ACT == kActNone) {
    y = v;
    slope = v != v ? v : 1.0f;          // (a lost value has no gradient)
  } else if constexpr (ACT == kActRelu) {
    y = v > 0.0f ? v : 0.0f;
    slope = v > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (ACT == kActGeluErf) {
    // Phi through erfc of |v| (device_math.hpp); slope = Phi(v) + v phi(v).
    constexpr float kLog2e = 1.4426950408889634f;
    const float half = 0.5f * erfc_nonneg(__builtin_fabsf(v) * 0.70710678118654752440f);
    const float h = held10(v);
    const float pdf = 0.3989422804014327f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * h * h);
    const float cdf = v >= 0.0f ? 1.0f - half : half;
    y = fmaxf(v, -30.0f) * cdf;               // (there cdf is 0, or NaN if v is)
    slope = __builtin_fmaf(h, pdf, cdf);
  } else {
    // q = 0.5 (1 + tanh z) = 1 / (1 + e), e = exp(-2 z), z = sqrt(2/pi) (v + 0.044715 v^3):
    // y = v q, slope = q + v q (1 - q) 2 z'.  1 - q is e q: no cancellation where q is near 1, and
    // with v held e is below 2^127.
    constexpr float c1 = -2.30220818520f;     // -2 log2(e) sqrt(2/pi)
    constexpr float c2 = -0.102943241596f;    // 0.044715 c1
    constexpr float d1 = 1.5957691216057308f; // 2 sqrt(2/pi)
    constexpr float d2 = 0.21406444881780073f;// 3 * 0.044715 d1
    const float h = held10(v), h2 = h * h;
    const float e = __builtin_amdgcn_exp2f(h * __builtin_fmaf(c2, h2, c1));
    const float q = __builtin_amdgcn_rcpf(1.0f + e);
    y = fmaxf(v, -10.0f) * q;                 // (there q is 2^-126, or NaN if v is)
    slope = __builtin_fmaf(h * __builtin_fmaf(d2, h2, d1), (e * q) * q, q);
  }
}

struct Layout {
  int64_t rows;
  int cols, blocks, tpr_log2;         // blocks of a row; 2^tpr_log2 lanes a row
  const void* bias;
  int bias_dtype;
};

// ---------------------------------------------------------------------------
// Forward.  32 columns are 4 (16-bit types) or 8 neighbouring lanes.  A row's last vector is
// moved back to end with it (WHOLE false): its first values are the lane's before it, and count
// and are saved there.
// ---------------------------------------------------------------------------
template <typename T, int ACT, bool WHOLE>
__global__ __launch_bounds__(kThreads) void checkpoint8_fwd_kernel(
    const T* __restrict__ x, T* __restrict__ y, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ exponents, Layout l) {
  constexpr int VE = kVecElems<T>, LB = kBlock / VE;
  const int t = threadIdx.x & ((1 << l.tpr_log2) - 1), group = threadIdx.x >> l.tpr_log2;
  const int groups = kThreads >> l.tpr_log2;
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  const int64_t j = (static_cast<int64_t>(blockIdx.y) << l.tpr_log2) + t;
  // Lanes behind the row hold zeros: their block's exponent wants them.
  const Cols<VE, WHOLE> at(j, l.cols);
  float b[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) b[e] = -0.0f;
  if (l.bias && at.any) {
    if (l.bias_dtype == MCKE_DTYPE_F32) at.load(b, static_cast<const float*>(l.bias));
    else at.load(b, static_cast<const T*>(l.bias));
  }

  for (int64_t r = static_cast<int64_t>(blockIdx.x) * groups + group; r < l.rows; r += step) {
    float xv[VE], u[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) xv[e] = 0.0f;
    if (at.any) at.load_stream(xv, x + r * l.cols);
    float most = 0.0f, any = 0.0f;                // `any`: not finite where a value is not
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      u[e] = xv[e] + b[e];
      any += u[e];
      if (WHOLE || (e >= at.skip && e < at.n)) most = fmaxf(most, __builtin_fabsf(u[e]));
    }
    if (__ballot(!(__builtin_fabsf(any) < __builtin_inff()))) {
      most = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float a = __builtin_fabsf(u[e]);
        if (!(a < __builtin_inff()))
          u[e] = __builtin_nanf("");
        else if (WHOLE || (e >= at.skip && e < at.n))
          most = fmaxf(most, a);
      }
    }
    most = wave_max<LB>(most);
    const int bits = __builtin_bit_cast(int, most);
    // 1.75: 448 = 1.75 * 2^8.
    int ex = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0);
    ex = ex < 1 ? 1 : ex;
    const float inv = __builtin_bit_cast(float, (254 - ex) << 23);
    typedef unsigned Packed __attribute__((ext_vector_type(VE / 4), aligned(1)));
    Packed packed;
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) {
      const int p = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * q] * inv, u[4 * q + 1] * inv, 0, false);
      packed[q] = static_cast<unsigned>(
          __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * q + 2] * inv, u[4 * q + 3] * inv, p, true));
    }
    if (!at.any) continue;
    uint8_t* to = codes + r * l.cols + at.c;
    if (WHOLE || (at.skip == 0 && at.n == VE)) {
      *reinterpret_cast<Packed*>(to) = packed;
    } else {
      at.template each<false>(
          [&](int e) { to[e] = static_cast<uint8_t>(packed[e / 4] >> (8 * (e % 4))); });
    }
    if (t % LB == 0) exponents[r * l.blocks + j / LB] = static_cast<uint8_t>(ex);
    if (y) {
#pragma unroll
      for (int e = 0; e < VE; ++e) u[e] = act_xb<ACT>(xv[e], b[e]);
      at.store_stream_again(y + r * l.cols, u);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward.  Workgroup (p, columns) walks the rows p per, p per + 1, .. of its part; a lane
// keeps its columns' sums of dx, and the workgroup's are row p of the workspace.
// ---------------------------------------------------------------------------
template <typename T, int ACT, bool WHOLE>
__global__ __launch_bounds__(kThreads) void checkpoint8_bwd_kernel(
    const T* __restrict__ dy, const uint8_t* __restrict__ codes,
    const uint8_t* __restrict__ exponents, T* __restrict__ dx, T* __restrict__ y,
    float* __restrict__ partials, Layout l, int64_t per) {
  constexpr int VE = kVecElems<T>;
  constexpr int U = 4;                            // rows whose loads are in flight
  __shared__ float fold[kThreads * VE];
  const int tpr = 1 << l.tpr_log2, groups = kThreads >> l.tpr_log2;
  const int t = threadIdx.x & (tpr - 1), g = threadIdx.x >> l.tpr_log2;
  const Cols<VE, WHOLE> at((static_cast<int64_t>(blockIdx.y) << l.tpr_log2) + t, l.cols);
  const int64_t r0 = blockIdx.x * per, r1 = r0 + per < l.rows ? r0 + per : l.rows;
  // A vector that is moved back may begin in the block before: its values from `turn` on are the
  // second block's.
  const int block = at.c / kBlock;
  [[maybe_unused]] const int turn = kBlock - at.c % kBlock;
  [[maybe_unused]] const int block2 = WHOLE ? block : (at.c + at.n - 1) / kBlock;
  float sum[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[e] = 0.0f;
  if (at.any) {
    for (int64_t rb = r0 + g; rb < r1; rb += U * groups) {
      typedef unsigned Packed __attribute__((ext_vector_type(VE / 4), aligned(1)));
      Packed packed[U];
      int ex[U], ex2[U];
      PackT<T, VE> d[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        // (Past the part its last row again, for nothing.)
        const int64_t r = rb + k * groups < r1 ? rb + k * groups : rb;
        const uint8_t* from = codes + r * l.cols + at.c;
        if (WHOLE || at.n == VE) {
          packed[k] = *reinterpret_cast<const Packed*>(from);
        } else {
          packed[k] = Packed{};
          at.template each<true>([&](int e) {
            packed[k][e / 4] |= static_cast<unsigned>(from[e]) << (8 * (e % 4));
          });
        }
        ex[k] = exponents[r * l.blocks + block];
        ex2[k] = WHOLE ? ex[k] : exponents[r * l.blocks + block2];
        if (dy) d[k] = at.load_raw(dy + r * l.cols);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t r = rb + k * groups;
        if (r >= r1) break;
        float u[VE], s[VE], v[VE];
#pragma unroll
        for (int q = 0; q < VE / 4; ++q) {
          const int p = static_cast<int>(packed[k][q]);
          u[4 * q + 0] = __builtin_amdgcn_cvt_f32_fp8(p, 0);
          u[4 * q + 1] = __builtin_amdgcn_cvt_f32_fp8(p, 1);
          u[4 * q + 2] = __builtin_amdgcn_cvt_f32_fp8(p, 2);
          u[4 * q + 3] = __builtin_amdgcn_cvt_f32_fp8(p, 3);
        }
        const float scale = __builtin_bit_cast(float, ex[k] << 23);
        const float scale2 = __builtin_bit_cast(float, ex2[k] << 23);
        int second = turn;
        if constexpr (!WHOLE) asm("" : "+v"(second));   // (kept as masks, these fill the scalar file)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          u[e] *= WHOLE || e < second ? scale : scale2;
          act_and_slope<ACT>(u[e], v[e], s[e]);
        }
        if (dy) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            s[e] *= static_cast<float>(d[k][e]);
            sum[e] += s[e];
          }
          if (dx) at.store_stream_again(dx + r * l.cols, s);
        }
        if (y) at.store_stream_again(y + r * l.cols, v);
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
  if (at.any) at.store(partials + static_cast<int64_t>(blockIdx.x) * l.cols, sum);
}

// dbias from the workgroups' sums: kFoldWays lanes a column, each every kFoldWays-th part, then a
// tree.
constexpr int kFoldCols = 32, kFoldWays = 32;

__global__ __launch_bounds__(kFoldCols * kFoldWays) void checkpoint8_fold_kernel(
    const float* __restrict__ partials, void* __restrict__ dbias, int dtype, int64_t cols,
    int parts) {
  __shared__ float lds[kFoldWays][kFoldCols + 1];
  const int lc = threadIdx.x % kFoldCols, way = threadIdx.x / kFoldCols;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kFoldCols;
  float s = 0.0f;
  if (c0 + lc < cols) {
#pragma unroll 8
    for (int p = way; p < parts; p += kFoldWays)
      s += partials[static_cast<int64_t>(p) * cols + c0 + lc];
  }
  lds[way][lc] = s;
  __syncthreads();
  // Column `way` of the workgroup's, its lanes' sums as a tree.
  s = wave_sum<kFoldWays>(lds[lc][way]);
  const int64_t c = c0 + way;
  if (lc > 0 || c >= cols) return;
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

constexpr int64_t kParts = 1024;

// Parts of the rows whose sums of dx are kept apart.  (Of rows and cols alone: the workspace is
// sized without the type.)
int64_t parts_of(int64_t rows, int64_t cols) {
  const int64_t tiles = ceil_div(cols, 2048), at_once = cols < 512 ? 2048 / cols : 4;
  const int64_t parts = ceil_div(kParts, tiles), some = ceil_div(rows, at_once);
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
    auto* fn = cols % kVecElems<T> == 0 ? &checkpoint8_fwd_kernel<T, decltype(act)::value, true>
                                        : &checkpoint8_fwd_kernel<T, decltype(act)::value, false>;
    fn<<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
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
      auto* fn = cols % kVecElems<T> == 0 ? &checkpoint8_bwd_kernel<T, decltype(act)::value, true>
                                          : &checkpoint8_bwd_kernel<T, decltype(act)::value, false>;
      fn<<<grid, kThreads, 0, s>>>(
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
