// layer_norm.hip -- layer norm over rows, forward and backward.
//
//   mean = sum(x) / cols,  rstd = 1 / sqrt(sum((x - mean)^2) / cols + eps)
//   xhat = (x - mean) rstd,  y = xhat weight + bias
//
//   g = dy weight
//   dx = rstd (g - sum(g) / cols - xhat sum(g xhat) / cols)
//   dweight = sum over rows of dy xhat,  dbias = sum over rows of dy
//
// x, y, dy and dx in fp32, fp16 or bf16; weight, bias and their gradients in that type or
// fp32; mean and rstd in fp32.  All arithmetic is fp32; each output is rounded once.  The
// variance is the sum of squared differences from the row's own mean (a sum of squares less
// a squared mean cancels where the mean is large).
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "common.hpp"
#include "device_math.hpp"
#include "elem.hpp"

namespace mcke_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// Sums of a pair over the workgroup, the same bits in every lane.  `lds` is free again
// after the caller's next barrier.
template <int WAVES>
__device__ __forceinline__ f32x2 block_sum2(f32x2 v, f32x2* lds) {
  v[0] = wave_sum(v[0]);
  v[1] = wave_sum(v[1]);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  f32x2 s = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    s[0] += lds[w][0];
    s[1] += lds[w][1];
  }
  return s;
}

// ---------------------------------------------------------------------------
// Rows of any width: one workgroup per row, three sweeps over it.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void ln_fwd_any_kernel(
    const T* __restrict__ x, const void* __restrict__ weight, const void* __restrict__ bias,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, int param_dtype,
    int64_t rows, int64_t cols, float eps) {
  __shared__ f32x2 lds[2][kWaves];
  const float n = static_cast<float>(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * cols;
    T* yr = y + r * cols;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) s += static_cast<float>(xr[c]);
    const float mean = block_sum2<kWaves>(f32x2{s, 0.0f}, lds[0])[0] / n;
    float q = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float d = static_cast<float>(xr[c]) - mean;
      q += d * d;
    }
    const float var = block_sum2<kWaves>(f32x2{q, 0.0f}, lds[1])[0] / n;
    const float rstd = 1.0f / sqrtf(var + eps);
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      float v = (static_cast<float>(xr[c]) - mean) * rstd;
      if (weight) v *= load_elem(weight, param_dtype, c);
      if (bias) v += load_elem(bias, param_dtype, c);
      yr[c] = static_cast<T>(v);
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_bwd_dx_any_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ weight,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
    int param_dtype, int64_t rows, int64_t cols) {
  __shared__ f32x2 lds[kWaves];
  const float n = static_cast<float>(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t at = r * cols;
    const float mean = mean_in[r], rstd = rstd_in[r];
    f32x2 s{0.0f, 0.0f};
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float w = weight ? load_elem(weight, param_dtype, c) : 1.0f;
      const float g = static_cast<float>(dy[at + c]) * w;
      s[0] += g;
      s[1] += g * ((static_cast<float>(x[at + c]) - mean) * rstd);
    }
    s = block_sum2<kWaves>(s, lds);
    const float a = s[0] / n, b = s[1] / n;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float w = weight ? load_elem(weight, param_dtype, c) : 1.0f;
      const float g = static_cast<float>(dy[at + c]) * w;
      const float xhat = (static_cast<float>(x[at + c]) - mean) * rstd;
      dx[at + c] = static_cast<T>((g - a - xhat * b) * rstd);
    }
    __syncthreads();   // lds is written again
  }
}

// Partial sums of dweight and dbias: workgroup (strip, part) sums rows part, part + parts, ..
// of one strip of columns, a column to a lane; part p's sums are rows 2 p (dweight) and
// 2 p + 1 (dbias) of the workspace.
template <typename T>
__global__ __launch_bounds__(kThreads) void ln_bwd_params_any_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, float* __restrict__ ws, int64_t rows, int64_t cols,
    int parts) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= cols) return;
  for (int p = blockIdx.y; p < parts; p += gridDim.y) {
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = p; r < rows; r += parts) {
      const float d = static_cast<float>(dy[r * cols + c]);
      dw += d * ((static_cast<float>(x[r * cols + c]) - mean_in[r]) * rstd_in[r]);
      db += d;
    }
    ws[(2 * static_cast<int64_t>(p)) * cols + c] = dw;
    ws[(2 * static_cast<int64_t>(p) + 1) * cols + c] = db;
  }
}

// Folds the parts in a fixed order: 64 columns a workgroup, its waves take parts in turn and
// their sums meet in LDS.  blockIdx.y 0 is dweight, 1 dbias.
template <typename P>
__global__ __launch_bounds__(kThreads) void ln_bwd_fold_kernel(const float* __restrict__ ws,
                                                               P* __restrict__ dweight,
                                                               P* __restrict__ dbias,
                                                               int64_t cols, int parts) {
  __shared__ float lds[kWaves][kWave];
  P* out = blockIdx.y == 0 ? dweight : dbias;
  if (!out) return;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kWave + lane;
  float s = 0.0f;
  if (c < cols)
    for (int p = wave; p < parts; p += kWaves)
      s += ws[(2 * static_cast<int64_t>(p) + blockIdx.y) * cols + c];
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < cols) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s += lds[w][lane];
    out[c] = static_cast<P>(s);
  }
}

// How many partial sums of dweight and dbias a launch keeps.
int ln_parts(int64_t rows, int64_t) { return static_cast<int>(rows < 512 ? rows : 512); }

// One workgroup per row up to the grid's 32-bit work size, which the kernels then walk.
unsigned row_grid(int64_t rows) {
  const int64_t most = int64_t{UINT32_MAX} / kThreads;
  return static_cast<unsigned>(rows < most ? rows : most);
}

template <typename T>
int ln_fwd(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
           int param_dtype, int64_t rows, int64_t cols, float eps, hipStream_t s) {
  ln_fwd_any_kernel<T><<<row_grid(rows), kThreads, 0, s>>>(
      static_cast<const T*>(x), weight, bias, static_cast<T*>(y), mean, rstd, param_dtype, rows,
      cols, eps);
  MCKE_LAUNCH_CHECK("ln_fwd_any_kernel");
  return ok();
}

struct LnBwdArgs {
  const void *dy, *x, *weight;
  const float *mean, *rstd;
  void *dx, *dweight, *dbias;
  int param_dtype;
  int64_t rows, cols;
  float* ws;
  hipStream_t s;
};

template <typename P> int ln_fold(const LnBwdArgs& a, int parts) {
  const dim3 grid(static_cast<unsigned>((a.cols + kWave - 1) / kWave), 2);
  ln_bwd_fold_kernel<P><<<grid, kThreads, 0, a.s>>>(a.ws, static_cast<P*>(a.dweight),
                                                    static_cast<P*>(a.dbias), a.cols, parts);
  MCKE_LAUNCH_CHECK("ln_bwd_fold_kernel");
  return ok();
}

int ln_fold_any(const LnBwdArgs& a, int parts) {
  if (a.param_dtype == MCKE_DTYPE_F32) return ln_fold<float>(a, parts);
  if (a.param_dtype == MCKE_DTYPE_F16) return ln_fold<_Float16>(a, parts);
  return ln_fold<__bf16>(a, parts);
}

template <typename T> int ln_bwd(const LnBwdArgs& a) {
  const T* dy = static_cast<const T*>(a.dy);
  const T* x = static_cast<const T*>(a.x);
  if (a.dx && a.rows > 0) {
    ln_bwd_dx_any_kernel<T><<<row_grid(a.rows), kThreads, 0, a.s>>>(
        dy, x, a.weight, a.mean, a.rstd, static_cast<T*>(a.dx), a.param_dtype, a.rows, a.cols);
    MCKE_LAUNCH_CHECK("ln_bwd_dx_any_kernel");
  }
  if (!a.dweight && !a.dbias) return ok();
  const int parts = ln_parts(a.rows, a.cols);
  if (parts > 0) {
    const dim3 grid(static_cast<unsigned>((a.cols + kThreads - 1) / kThreads),
                    static_cast<unsigned>(parts));
    ln_bwd_params_any_kernel<T><<<grid, kThreads, 0, a.s>>>(dy, x, a.mean, a.rstd, a.ws, a.rows,
                                                            a.cols, parts);
    MCKE_LAUNCH_CHECK("ln_bwd_params_any_kernel");
  }
  return ln_fold_any(a, parts);
}

// The widest row: column strips of 64 lanes stay within the grid's 32-bit work size.
constexpr int64_t kMaxCols = int64_t{1} << 30;

int check_types(const char* who, int dtype, int param_dtype) {
  if (!is_dtype(dtype))
    return invalid(std::string(who) + ": unknown dtype " + std::to_string(dtype));
  if (param_dtype != MCKE_DTYPE_F32 && param_dtype != dtype)
    return invalid(std::string(who) + ": param_dtype must be MCKE_DTYPE_F32 or dtype, got " +
                   std::to_string(param_dtype));
  return ok();
}

int check_extents(const char* who, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return invalid(std::string(who) + ": negative extent");
  if (cols > kMaxCols || (cols > 0 && rows > INT64_MAX / 16 / cols))
    return invalid(std::string(who) + ": extent too large");
  return ok();
}

}  // namespace
}  // namespace mcke_amd

using namespace mcke_amd;

extern "C" {

int mcke_launch_layer_norm(const void* x, const void* weight, const void* bias, void* y,
                           float* mean, float* rstd, int dtype, int param_dtype, int64_t rows,
                           int64_t cols, float eps, void* stream) {
  if (int rc = check_types("launch_layer_norm", dtype, param_dtype)) return rc;
  if (int rc = check_extents("launch_layer_norm", rows, cols)) return rc;
  if (!(eps >= 0.0f) || std::isinf(eps))
    return invalid("launch_layer_norm: eps must be finite and not negative");
  if (rows == 0 || cols == 0) return ok();
  if (!x || !y) return invalid("launch_layer_norm: null pointer");
  const uint64_t e = dtype_bytes(dtype), p = dtype_bytes(param_dtype), n = rows, c = cols;
  if (!aligned(x, e) || !aligned(y, e) || !aligned(weight, p) || !aligned(bias, p) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return invalid("launch_layer_norm: a pointer is not aligned to its type");
  const void* outs[] = {y, mean, rstd};
  const uint64_t out_bytes[] = {n * c * e, 4 * n, 4 * n};
  for (int i = 0; i < 3; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], x, n * c * e) ||
               overlap(outs[i], out_bytes[i], weight, c * p) ||
               overlap(outs[i], out_bytes[i], bias, c * p);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid("launch_layer_norm: an output overlaps another operand, which violates the "
                     "__restrict__ contract");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MCKE_DTYPE_F32)
    return ln_fwd<float>(x, weight, bias, y, mean, rstd, param_dtype, rows, cols, eps, s);
  if (dtype == MCKE_DTYPE_F16)
    return ln_fwd<_Float16>(x, weight, bias, y, mean, rstd, param_dtype, rows, cols, eps, s);
  return ln_fwd<__bf16>(x, weight, bias, y, mean, rstd, param_dtype, rows, cols, eps, s);
}

size_t mcke_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  return 2 * sizeof(float) * static_cast<size_t>(ln_parts(rows, cols)) * static_cast<size_t>(cols);
}

int mcke_launch_layer_norm_backward(const void* dy, const void* x, const void* weight,
                                    const float* mean, const float* rstd, void* dx, void* dweight,
                                    void* dbias, int dtype, int param_dtype, int64_t rows,
                                    int64_t cols, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  const char* who = "launch_layer_norm_backward";
  if (int rc = check_types(who, dtype, param_dtype)) return rc;
  if (int rc = check_extents(who, rows, cols)) return rc;
  if (cols == 0) return ok();
  const uint64_t e = dtype_bytes(dtype), p = dtype_bytes(param_dtype), n = rows, c = cols;
  if (rows > 0 && (!dy || !x || !mean || !rstd))
    return invalid("launch_layer_norm_backward: null pointer");
  if (!dx && !dweight && !dbias)
    return invalid("launch_layer_norm_backward: no gradient is asked for");
  if (!aligned(dy, e) || !aligned(x, e) || !aligned(dx, e) || !aligned(weight, p) ||
      !aligned(dweight, p) || !aligned(dbias, p) || !aligned(mean, 4) || !aligned(rstd, 4))
    return invalid("launch_layer_norm_backward: a pointer is not aligned to its type");
  const bool params = dweight || dbias;
  const size_t need = params ? mcke_layer_norm_backward_workspace_bytes(rows, cols) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return invalid("launch_layer_norm_backward: dweight and dbias need a 16-byte aligned "
                   "workspace of " + std::to_string(need) + " bytes, got " +
                   std::to_string(workspace ? workspace_bytes : 0));
  const void* outs[] = {dx, dweight, dbias, need > 0 ? workspace : nullptr};
  const uint64_t out_bytes[] = {n * c * e, c * p, c * p, need};
  for (int i = 0; i < 4; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], dy, n * c * e) ||
               overlap(outs[i], out_bytes[i], x, n * c * e) ||
               overlap(outs[i], out_bytes[i], weight, c * p) ||
               overlap(outs[i], out_bytes[i], mean, 4 * n) ||
               overlap(outs[i], out_bytes[i], rstd, 4 * n);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid("launch_layer_norm_backward: an output or the workspace overlaps another "
                     "operand, which violates the __restrict__ contract");
  }
  const LnBwdArgs a{dy, x, weight, mean, rstd, dx, dweight, dbias, param_dtype, rows, cols,
                    static_cast<float*>(workspace), static_cast<hipStream_t>(stream)};
  if (dtype == MCKE_DTYPE_F32) return ln_bwd<float>(a);
  if (dtype == MCKE_DTYPE_F16) return ln_bwd<_Float16>(a);
  return ln_bwd<__bf16>(a);
}

}  // extern "C"
