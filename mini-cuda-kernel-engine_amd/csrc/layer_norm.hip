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

// Sums over groups of TPR lanes (a row's), the same bits in every lane of a group.  Groups wider
// than a wave meet in `lds` (the workgroup's waves), which is free again after the caller's next
// barrier; every lane of the workgroup calls these.
template <int TPR, int N, int NW>
__device__ __forceinline__ void group_sums(float (&v)[N], float (&lds)[N][NW]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = wave_sum<(TPR < kWave ? TPR : kWave)>(v[k]);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    const int first = (threadIdx.x / TPR) * W;
    if ((threadIdx.x % kWave) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) lds[k][threadIdx.x / kWave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = wave_sum<W>(lds[k][first + threadIdx.x % W]);
  }
}

// ---------------------------------------------------------------------------
// Rows that fit in registers: NT-lane workgroups, TPR lanes a row, VPT 16-byte vectors a lane,
// ROWS rows a lane at once.  x is read once and y written once; a row stays in registers over
// both reductions.
// WHOLE: cols is a multiple of the vector.  Otherwise (cols >= one vector) the row's last vector
// is moved back to end with the row: what it repeats of the vector before it is taken out of
// the sums again and is stored twice, the same bits.  Loaded and stored element by element instead, the end of
// each row cost more instructions than the rest of it: 131072 x 500 bf16 69 us against 47.
// ---------------------------------------------------------------------------
template <typename T, bool WHOLE> struct RowVectors {
  static constexpr int VE = kVecElems<T>;
  int cols;
  // Whether vector j is the row's, and its first column.
  __device__ __forceinline__ bool has(int j) const { return j * VE < cols; }
  __device__ __forceinline__ int col(int j) const {
    return WHOLE || j * VE + VE <= cols ? j * VE : cols - VE;
  }
  // Calls f(e) for the elements of vector j that the one before it has too.
  template <class F> __device__ __forceinline__ void repeated(int j, F f) const {
    if constexpr (!WHOLE) {
      if (has(j) && j * VE + VE > cols) {
        const int n = (cols + VE - 1) / VE * VE - cols;
#pragma unroll
        for (int e = 0; e < VE - 1; ++e)
          if (e < n) f(e);
      }
    }
  }
};

template <typename T, typename P, int TPR, int VPT, int NT, int ROWS, bool WHOLE>
__global__ __launch_bounds__(NT) void ln_fwd_regs_kernel(
    const T* __restrict__ x, const P* __restrict__ weight, const P* __restrict__ bias,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows,
    int cols, float eps) {
  constexpr int VE = kVecElems<T>;
  __shared__ float lds[2][ROWS][NT / kWave];
  const int t = threadIdx.x % TPR;
  const int64_t r0 =
      (static_cast<int64_t>(blockIdx.x) * (NT / TPR) + threadIdx.x / TPR) * ROWS;
  const float n = static_cast<float>(cols);
  const RowVectors<T, WHOLE> rv{cols};

  // Rows past the end take part in the barriers and in nothing else.
  float v[ROWS][VPT][VE];
#pragma unroll
  for (int k = 0; k < ROWS; ++k)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = i * TPR + t;
      VecT16<T> w{};
      if (r0 + k < rows && rv.has(j)) w = load_stream<T>(x + (r0 + k) * cols + rv.col(j));
#pragma unroll
      for (int e = 0; e < VE; ++e) v[k][i][e] = static_cast<float>(w[e]);
    }
  float mean[ROWS], rstd[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) s += v[k][i][e];
#pragma unroll
    for (int i = 0; i < VPT; ++i) rv.repeated(i * TPR + t, [&](int e) { s -= v[k][i][e]; });
    mean[k] = s;
  }
  group_sums<TPR, ROWS>(mean, lds[0]);
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    mean[k] /= n;      // (times 1 / n would not be exact where the sum is)
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float qi = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        v[k][i][e] -= mean[k];
        qi += v[k][i][e] * v[k][i][e];
      }
      if (rv.has(i * TPR + t)) q += qi;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      rv.repeated(i * TPR + t, [&](int e) { q -= v[k][i][e] * v[k][i][e]; });
    rstd[k] = q;
  }
  group_sums<TPR, ROWS>(rstd, lds[1]);
#pragma unroll
  for (int k = 0; k < ROWS; ++k) rstd[k] = 1.0f / sqrtf(rstd[k] / n + eps);

#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = i * TPR + t, c = rv.col(j);
    if (!rv.has(j)) continue;
    float w[VE], b[VE];
    load_params<P, VE>(w, weight, c, 1.0f);
    load_params<P, VE>(b, bias, c, 0.0f);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (r0 + k >= rows) continue;
      VecT16<T> o;
#pragma unroll
      for (int e = 0; e < VE; ++e) o[e] = static_cast<T>(v[k][i][e] * rstd[k] * w[e] + b[e]);
      store_stream<T>(y + (r0 + k) * cols + c, o);
    }
  }
  if (t == 0) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (r0 + k >= rows) continue;
      if (mean_out) mean_out[r0 + k] = mean[k];
      if (rstd_out) rstd_out[r0 + k] = rstd[k];
    }
  }
}

// The backward pass over rows that fit in registers.  Workgroups walk rows NT / TPR at a time, a
// lane keeps its columns' sums of dy xhat and dy over all of its rows, and x and dy are read
// once, each row's behind the one before it.  At the end the groups of a workgroup add up
// their columns, and the workgroup's sums are rows 2 p and 2 p + 1 of the workspace.  What a
// row's moved-back last vector repeats is summed up twice to the same bits, and counts once in
// the row's own sums.
// PARAMS false: only dx, for rows whose column sums do not fit beside them.
template <typename T, typename P, int TPR, int VPT, int NT, bool WHOLE, bool PARAMS>
__global__ __launch_bounds__(NT) void ln_bwd_regs_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ weight,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
    float* __restrict__ ws, int64_t rows, int cols) {
  constexpr int VE = kVecElems<T>, G = NT / TPR, NW = NT / kWave;
  constexpr int kSums = 2 * VPT * VE;                   // of a lane
  // Groups of a wave add up by lane permutations, those of different waves through LDS.
  constexpr int L = TPR < kWave ? kWave : TPR;          // lanes that are left to a wave or row
  constexpr int GL = NT / L;
  __shared__ float lds[2][2][NW];
  __shared__ float fold[PARAMS && GL > 1 ? NT * kSums : 1];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const RowVectors<T, WHOLE> rv{cols};
  const float inv_n = 1.0f / static_cast<float>(cols);

  // Workgroups of 1024 lanes have 128 registers a lane: they load the weights for each row.
  constexpr bool KEEP = PARAMS && NT < 1024;
  float w[KEEP ? VPT : 1][VE], dw[PARAMS ? VPT : 1][VE], db[PARAMS ? VPT : 1][VE];
  if constexpr (PARAMS) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) dw[i][e] = db[i][e] = 0.0f;
  }
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = i * TPR + t;
#pragma unroll
      for (int e = 0; e < VE; ++e) w[i][e] = 0.0f;
      if (rv.has(j)) load_params<P, VE>(w[i], weight, rv.col(j), 1.0f);
    }
  }
  auto weights = [&](int i) -> const float(&)[VE] {
    if constexpr (KEEP) {
      return w[i];
    } else {
      const int j = i * TPR + t;
#pragma unroll
      for (int e = 0; e < VE; ++e) w[0][e] = 0.0f;
      if (rv.has(j)) load_params<P, VE>(w[0], weight, rv.col(j), 1.0f);
      return w[0];
    }
  };
  auto load = [&](int64_t r, VecT16<T> (&xv)[VPT], VecT16<T> (&dv)[VPT], float& m, float& rs) {
    m = rs = 0.0f;
    if (r < rows) {
      m = mean_in[r];
      rs = rstd_in[r];
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = i * TPR + t;
      xv[i] = VecT16<T>{};
      dv[i] = VecT16<T>{};
      if (r < rows && rv.has(j)) {
        xv[i] = load_stream<T>(x + r * cols + rv.col(j));
        dv[i] = load_stream<T>(dy + r * cols + rv.col(j));
      }
    }
  };

  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  VecT16<T> xv[VPT], dv[VPT];
  float mean, rstd;
  load(static_cast<int64_t>(blockIdx.x) * G + g, xv, dv, mean, rstd);
  int odd = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * G; r0 < rows; r0 += step) {
    const int64_t r = r0 + g;
    [[maybe_unused]] VecT16<T> xn[PARAMS ? VPT : 1], dn[PARAMS ? VPT : 1];
    [[maybe_unused]] float mean_n, rstd_n;
    if constexpr (PARAMS) load(r + step, xn, dn, mean_n, rstd_n);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const auto& wi = weights(i);
      float s1 = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = static_cast<float>(dv[i][e]);
        const float xhat = (static_cast<float>(xv[i][e]) - mean) * rstd;
        if constexpr (PARAMS) {
          dw[i][e] += d * xhat;
          db[i][e] += d;
        }
        s[0] += d * wi[e];
        s1 += d * wi[e] * xhat;
      }
      // A lane without vector i has zeros there: its (0 - mean) rstd is not a value of the row,
      // and may be past fp32's range.
      if (rv.has(i * TPR + t)) s[1] += s1;
      rv.repeated(i * TPR + t, [&](int e) {
        const float dg = static_cast<float>(dv[i][e]) * wi[e];
        s[0] -= dg;
        s[1] -= dg * ((static_cast<float>(xv[i][e]) - mean) * rstd);
      });
    }
    if (dx) {
      group_sums<TPR, 2>(s, lds[odd]);
      odd ^= 1;
      const float a = s[0] * inv_n, b = s[1] * inv_n;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = i * TPR + t;
        const auto& wi = weights(i);
        VecT16<T> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float xhat = (static_cast<float>(xv[i][e]) - mean) * rstd;
          o[e] = static_cast<T>((static_cast<float>(dv[i][e]) * wi[e] - a - xhat * b) * rstd);
        }
        if (r < rows && rv.has(j)) store_stream<T>(dx + r * cols + rv.col(j), o);
      }
    }
    if constexpr (PARAMS) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        xv[i] = xn[i];
        dv[i] = dn[i];
      }
      mean = mean_n;
      rstd = rstd_n;
    } else {
      load(r + step, xv, dv, mean, rstd);
    }
  }
  if constexpr (PARAMS) {
    if (!ws) return;

#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e)
#pragma unroll
        for (int k = TPR; k < kWave; k *= 2) {
          dw[i][e] += __shfl_xor(dw[i][e], k, 64);
          db[i][e] += __shfl_xor(db[i][e], k, 64);
        }
    if constexpr (GL > 1) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          fold[(2 * (i * VE + e)) * NT + threadIdx.x] = dw[i][e];
          fold[(2 * (i * VE + e) + 1) * NT + threadIdx.x] = db[i][e];
        }
      __syncthreads();
      if (threadIdx.x >= L) return;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int k = 1; k < GL; ++k) {
            dw[i][e] += fold[(2 * (i * VE + e)) * NT + threadIdx.x + k * L];
            db[i][e] += fold[(2 * (i * VE + e) + 1) * NT + threadIdx.x + k * L];
          }
    }
    if (threadIdx.x >= TPR) return;
    float* out = ws + 2 * static_cast<int64_t>(blockIdx.x) * cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = i * TPR + t;
      if (!rv.has(j)) continue;
#pragma unroll
      for (int q = 0; q < VE / 4; ++q) {
        float* p = out + rv.col(j) + 4 * q;
        *reinterpret_cast<f32x4_a4*>(p) =
            f32x4_a4{dw[i][4 * q], dw[i][4 * q + 1], dw[i][4 * q + 2], dw[i][4 * q + 3]};
        *reinterpret_cast<f32x4_a4*>(p + cols) =
            f32x4_a4{db[i][4 * q], db[i][4 * q + 1], db[i][4 * q + 2], db[i][4 * q + 3]};
      }
    }
  }
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

// dx of rows that do not fit in registers, at least a vector wide: a workgroup per row, two
// sweeps over it (the second one from the caches).
constexpr int kWideThreads = 1024;
template <typename T>
__global__ __launch_bounds__(kWideThreads) void ln_bwd_dx_wide_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ weight,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
    int param_dtype, int64_t rows, int64_t cols) {
  constexpr int VE = kVecElems<T>;
  __shared__ float lds[2][2][kWideThreads / kWave];
  const float n = static_cast<float>(cols);
  int odd = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, odd ^= 1) {
    const int64_t at = r * cols;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float s[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x * VE; c < cols; c += kWideThreads * VE) {
      const int64_t from = c + VE <= cols ? c : cols - VE;     // c - from elements are repeated
      const VecT16<T> dv = load_vec<T>(dy + at + from), xv = load_vec<T>(x + at + from);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float w = weight ? load_elem(weight, param_dtype, from + e) : 1.0f;
        const float g = from + e >= c ? static_cast<float>(dv[e]) * w : 0.0f;
        s[0] += g;
        s[1] += g * ((static_cast<float>(xv[e]) - mean) * rstd);
      }
    }
    group_sums<kWideThreads, 2>(s, lds[odd]);
    const float a = s[0] / n, b = s[1] / n;
    for (int64_t c = threadIdx.x * VE; c < cols; c += kWideThreads * VE) {
      const int64_t from = c + VE <= cols ? c : cols - VE;
      const VecT16<T> dv = load_vec<T>(dy + at + from), xv = load_vec<T>(x + at + from);
      VecT16<T> o;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float w = weight ? load_elem(weight, param_dtype, from + e) : 1.0f;
        const float xhat = (static_cast<float>(xv[e]) - mean) * rstd;
        o[e] = static_cast<T>((static_cast<float>(dv[e]) * w - a - xhat * b) * rstd);
      }
      store_stream<T>(dx + at + from, o);
    }
  }
}

// Partial sums of dweight and dbias, for rows that ln_bwd_regs_kernel does not hold: workgroup
// (strip, part) sums rows part, part + parts, ... of one strip of columns, a vector to a lane
// (moved back at the row's end, to the same bits twice), to rows 2 part and 2 part + 1 of the
// workspace.  Rows narrower than a vector: a column to a lane.
template <typename T, bool NARROW>
__global__ __launch_bounds__(kThreads) void ln_bwd_params_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, float* __restrict__ ws, int64_t rows, int64_t cols,
    int parts) {
  constexpr int VE = NARROW ? 1 : kVecElems<T>;
  int64_t c = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * VE;
  if (c >= cols) return;
  if (c + VE > cols) c = cols - VE;
  const int64_t p = blockIdx.y;
  float dw[VE], db[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) dw[e] = db[e] = 0.0f;
#pragma unroll 4
  for (int64_t r = p; r < rows; r += parts) {
    const float mean = mean_in[r], rstd = rstd_in[r];
    const T *dp = dy + r * cols + c, *xp = x + r * cols + c;
    float d[VE], v[VE];
    if constexpr (NARROW) {
      d[0] = static_cast<float>(*dp);
      v[0] = static_cast<float>(*xp);
    } else {
      const VecT16<T> dv = load_stream<T>(dp), xv = load_stream<T>(xp);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        d[e] = static_cast<float>(dv[e]);
        v[e] = static_cast<float>(xv[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      dw[e] += d[e] * ((v[e] - mean) * rstd);
      db[e] += d[e];
    }
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    ws[2 * p * cols + c + e] = dw[e];
    ws[(2 * p + 1) * cols + c + e] = db[e];
  }
}

// Folds the parts in a fixed order: kFoldCols columns a workgroup at a time, kFoldWays lanes a
// column take the parts in turn and meet in LDS.  blockIdx.y 0 is dweight, 1 dbias.  Workgroups walk
// the columns: 32 lanes a column are past the grid's 32-bit work size from 2^27 columns on.
constexpr int kFoldCols = 32, kFoldWays = 32;
template <typename P>
__global__ __launch_bounds__(kFoldCols * kFoldWays) void ln_bwd_fold_kernel(
    const float* __restrict__ ws, P* __restrict__ dweight, P* __restrict__ dbias, int64_t cols,
    int parts) {
  __shared__ float lds[kFoldWays][kFoldCols + 1];
  P* out = blockIdx.y == 0 ? dweight : dbias;
  if (!out) return;
  const int lc = threadIdx.x % kFoldCols, way = threadIdx.x / kFoldCols;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kFoldCols;
  for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * kFoldCols;;) {
    const int64_t c = c0 + lc;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 16
      for (int p = way; p < parts; p += kFoldWays)
        s += ws[(2 * static_cast<int64_t>(p) + blockIdx.y) * cols + c];
    }
    lds[way][lc] = s;
    __syncthreads();
    // Column `way` of the workgroup's, its lanes' sums as a tree.
    s = wave_sum<kFoldWays>(lds[lc][way]);
    const int64_t oc = c0 + way;
    if (lc == 0 && oc < cols) out[oc] = static_cast<P>(s);
    c0 += step;
    if (c0 >= cols) return;
    __syncthreads();   // lds is written again
  }
}

// ---------------------------------------------------------------------------
// Which kernel a row width takes.  `vecs` is the row's 16-byte vectors (the last one may be in
// part); widths under one vector and over the last entry take the sweeping kernels.
// ---------------------------------------------------------------------------
// Calls f with a shape of the forward kernel as constants.  Two rows a lane share the weight's
// and bias's loads.  bf16 and fp32, 134217728 bytes of x, us (the best of 44 shapes, by width in
// vectors): 8 44.3, 16 45.6, 32 44.9, 64 45.2, 128 44.5, 256 45.2, 512 45.1 (128 x 4 one row 45.6,
// 512 x 1 48.6; 16384 x 4095: 50.7 and 49.2), 1024 90.0 at twice the bytes (256 x 4 one row 92.2),
// 2048 92.5 (1024 lanes x 2 99.3), 4096 95.6, 8192 106; one row instead of two 1 to 6 us more up to
// 512 vectors.  Non-temporal loads and stores: 45.1; stores alone 46.2, loads alone 47.8,
// neither 48.4.
template <int TPR_, int VPT_, int NT_, int ROWS_> struct RowShape {
  static constexpr int TPR = TPR_, VPT = VPT_, NT = NT_, ROWS = ROWS_;
};
template <typename T, bool WHOLE, class F> int with_forward_shape(int64_t vecs, F f) {
  if (vecs <= 8) return f(RowShape<8, 1, 256, 2>{});
  if (vecs <= 16) return f(RowShape<16, 1, 256, 2>{});
  if (vecs <= 32) return f(RowShape<32, 1, 256, 2>{});
  if (vecs <= 64) return f(RowShape<64, 1, 256, 2>{});
  if (vecs <= 128) return f(RowShape<128, 1, 256, 2>{});
  if (vecs <= 256) return f(RowShape<128, 2, 256, 2>{});
  if (vecs <= 512) {
    if constexpr (WHOLE) return f(RowShape<256, 2, 256, 2>{});
    else return f(RowShape<512, 1, 512, 2>{});
  }
  if (vecs <= 1024) return f(RowShape<512, 2, 512, sizeof(T) == 2 ? 2 : 1>{});
  if (vecs <= 2048) return f(RowShape<512, 4, 512, 1>{});
  if (vecs <= 4096) return f(RowShape<1024, 4, 1024, 1>{});
  return f(RowShape<1024, 8, 1024, 1>{});
}
constexpr int64_t kMaxForwardVecs = 8192;

// The backward kernel with column sums in registers, and how many workgroups walk the rows
// (two or three to a CU, as its registers allow; each ends with its sums' store, so more of
// them cost more than they hide).  At 402653184 bytes of x, dy and dx, us: 8 vectors 68.5 (768
// workgroups; 512 75.0, 1024 70.1), 32 69.3, 64 69.6, 128 70.1, 256 70.6 (fp32 66.7), 512 73.7
// (512 x 1 75.8, 256 x 2 77.0), 1024 143 at twice the bytes (512 x 4 155), 2048 147 (256 workgroups;
// 512 159).  8192 rows of 640 and 768 vectors 55.5 and 61.5 (256 x 4 58.1 and 62.3).  4096 vectors
// in 16 bits would spill (965): dx and the column sums apart.
template <int TPR_, int VPT_, int NT_, int WGS_> struct BackShape {
  static constexpr int TPR = TPR_, VPT = VPT_, NT = NT_, kWorkgroups = WGS_;
};
template <int VE, bool WHOLE, class F> int with_backward_shape(int64_t vecs, F f) {
  if (vecs <= 8) return f(BackShape<8, 1, 256, 768>{});
  if (vecs <= 16) return f(BackShape<16, 1, 256, 768>{});
  if (vecs <= 32) return f(BackShape<32, 1, 256, 768>{});
  if (vecs <= 64) return f(BackShape<64, 1, 256, 768>{});
  if (vecs <= 128) return f(BackShape<128, 1, 512, 512>{});
  if (vecs <= 256) return f(BackShape<256, 1, 512, 512>{});
  // 16384 x 4095: 90.6 us, 128 x 4 over 102 (the end's selects cost registers).
  if (vecs <= 512) {
    if constexpr (WHOLE) return f(BackShape<128, 4, 256, 512>{});
    else return f(BackShape<256, 2, 256, 512>{});
  }
  if (vecs <= 768) return f(BackShape<256, 3, 256, 512>{});
  // A row's end takes 256 x 4 over 256 registers in 16 bits, one workgroup a CU: 8192 x 6143 110 us
  // (256 x 3 74.6), 8192 x 8191 129 (512 x 2 112, with 512 workgroups 120; 1024 x 1 115).  fp32 has
  // them: 8192 x 4095 79.1, 512 x 2 85.4.
  if (vecs <= 1024) {
    if constexpr (WHOLE || VE == 4) return f(BackShape<256, 4, 256, 512>{});
    else return f(BackShape<512, 2, 512, 256>{});
  }
  return f(BackShape<1024, 2, 1024, 256>{});
}
constexpr int64_t kMaxBackwardVecs = 2048;
constexpr int64_t kMaxDxVecs = 4096;      // dx alone, with the row in registers

// Workgroups of a launch over `rows`: each walks two rounds of rows at least (512 x 4096, us:
// 11.5 with 256 workgroups, 16.3 with 512).
template <class S> int backward_workgroups(int64_t rows) {
  const int64_t need = (rows + 2 * (S::NT / S::TPR) - 1) / (2 * (S::NT / S::TPR));
  return static_cast<int>(need < S::kWorkgroups ? need : S::kWorkgroups);
}

// Parts of the column sums taken apart: workgroups of one strip for 1024 in all.
int params_parts(int64_t rows, int64_t cols, int vec) {
  const int64_t strips = (cols + int64_t{kThreads} * vec - 1) / (int64_t{kThreads} * vec);
  int64_t parts = 1024 / strips < 1 ? 1 : 1024 / strips;
  if (parts > 256) parts = 256;
  return static_cast<int>(parts < rows ? parts : rows);
}

// How many partial sums of dweight and dbias a launch keeps, `vec` elements to a vector.
int ln_parts(int64_t rows, int64_t cols, int vec) {
  if (rows <= 0) return 0;
  if (cols < vec) return params_parts(rows, cols, 1);
  const int64_t vecs = (cols + vec - 1) / vec;
  if (vecs > kMaxBackwardVecs) return params_parts(rows, cols, vec);
  auto count = [&](auto shape) { return backward_workgroups<decltype(shape)>(rows); };
  const bool whole = cols % vec == 0;
  if (vec == 4)
    return whole ? with_backward_shape<4, true>(vecs, count)
                 : with_backward_shape<4, false>(vecs, count);
  return whole ? with_backward_shape<8, true>(vecs, count)
               : with_backward_shape<8, false>(vecs, count);
}

// A workgroup of up to 1024 lanes per row, or per strip of columns, up to the grid's 32-bit work
// size; the kernels walk what is left.
unsigned grid_of_1024(int64_t n) {
  const int64_t most = int64_t{UINT32_MAX} / 1024;
  return static_cast<unsigned>(n < most ? n : most);
}

struct LnFwdArgs {
  const void *x, *weight, *bias;
  void* y;
  float *mean, *rstd;
  int param_dtype;
  int64_t rows, cols;
  float eps;
  hipStream_t s;
};

template <typename T, typename P, bool WHOLE> int ln_fwd_regs(const LnFwdArgs& a) {
  constexpr int VE = kVecElems<T>;
  return with_forward_shape<T, WHOLE>((a.cols + VE - 1) / VE, [&](auto shape) {
    using S = decltype(shape);
    constexpr int64_t kRows = S::NT / S::TPR * S::ROWS;
    const int64_t groups = (a.rows + kRows - 1) / kRows;
    if (groups * S::NT > int64_t{UINT32_MAX})
      return invalid("launch_layer_norm: rows exceed the grid's 32-bit work size");
    ln_fwd_regs_kernel<T, P, S::TPR, S::VPT, S::NT, S::ROWS, WHOLE>
        <<<static_cast<unsigned>(groups), S::NT, 0, a.s>>>(
            static_cast<const T*>(a.x), static_cast<const P*>(a.weight),
            static_cast<const P*>(a.bias), static_cast<T*>(a.y), a.mean, a.rstd, a.rows,
            static_cast<int>(a.cols), a.eps);
    MCKE_LAUNCH_CHECK("ln_fwd_regs_kernel");
    return ok();
  });
}

template <typename T> int ln_fwd(const LnFwdArgs& a) {
  constexpr int VE = kVecElems<T>;
  const bool whole = a.cols % VE == 0;
  if (a.cols >= VE && a.cols <= kMaxForwardVecs * VE) {
    if (a.param_dtype == MCKE_DTYPE_F32)
      return whole ? ln_fwd_regs<T, float, true>(a) : ln_fwd_regs<T, float, false>(a);
    return whole ? ln_fwd_regs<T, T, true>(a) : ln_fwd_regs<T, T, false>(a);
  }
  ln_fwd_any_kernel<T><<<grid_of_1024(a.rows), kThreads, 0, a.s>>>(
      static_cast<const T*>(a.x), a.weight, a.bias, static_cast<T*>(a.y), a.mean, a.rstd,
      a.param_dtype, a.rows, a.cols, a.eps);
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
  const dim3 grid(grid_of_1024((a.cols + kFoldCols - 1) / kFoldCols), 2);
  ln_bwd_fold_kernel<P><<<grid, kFoldCols * kFoldWays, 0, a.s>>>(a.ws, static_cast<P*>(a.dweight),
                                                    static_cast<P*>(a.dbias), a.cols, parts);
  MCKE_LAUNCH_CHECK("ln_bwd_fold_kernel");
  return ok();
}

int ln_fold_any(const LnBwdArgs& a, int parts) {
  if (a.param_dtype == MCKE_DTYPE_F32) return ln_fold<float>(a, parts);
  if (a.param_dtype == MCKE_DTYPE_F16) return ln_fold<_Float16>(a, parts);
  return ln_fold<__bf16>(a, parts);
}

template <typename T, typename P, bool WHOLE, class S, bool PARAMS>
int ln_bwd_launch(const LnBwdArgs& a, unsigned grid, float* ws) {
  ln_bwd_regs_kernel<T, P, S::TPR, S::VPT, S::NT, WHOLE, PARAMS><<<grid, S::NT, 0, a.s>>>(
      static_cast<const T*>(a.dy), static_cast<const T*>(a.x), static_cast<const P*>(a.weight),
      a.mean, a.rstd, static_cast<T*>(a.dx), ws, a.rows, static_cast<int>(a.cols));
  MCKE_LAUNCH_CHECK("ln_bwd_regs_kernel");
  return ok();
}

// dx, with the column sums where they are asked for and fit; `summed`: they are in the
// workspace.
template <typename T, typename P, bool WHOLE>
int ln_bwd_rows(const LnBwdArgs& a, int parts, bool* summed) {
  constexpr int VE = kVecElems<T>;
  const int64_t vecs = (a.cols + VE - 1) / VE;
  const bool params = a.dweight || a.dbias;
  *summed = params && vecs <= kMaxBackwardVecs;
  if (vecs <= kMaxBackwardVecs)
    return with_backward_shape<VE, WHOLE>(vecs, [&](auto shape) {
      using S = decltype(shape);
      // The workspace and the fold count on it.
      if (backward_workgroups<S>(a.rows) != parts)
        return fail(MCKE_STATUS_INTERNAL, "launch_layer_norm_backward: workgroups and parts differ");
      return ln_bwd_launch<T, P, WHOLE, S, true>(a, parts, params ? a.ws : nullptr);
    });
  if (!a.dx) return ok();
  return ln_bwd_launch<T, P, WHOLE, BackShape<1024, 4, 1024, 0>, false>(a, grid_of_1024(a.rows),
                                                                        nullptr);
}

template <typename T> int ln_bwd(const LnBwdArgs& a) {
  constexpr int VE = kVecElems<T>;
  const T* dy = static_cast<const T*>(a.dy);
  const T* x = static_cast<const T*>(a.x);
  const bool params = a.dweight || a.dbias;
  const int parts = ln_parts(a.rows, a.cols, VE);
  bool summed = false;
  if (a.rows > 0) {
    const bool whole = a.cols % VE == 0;
    int rc = ok();
    if (a.cols >= VE && a.cols <= kMaxDxVecs * VE) {
      if (a.param_dtype == MCKE_DTYPE_F32)
        rc = whole ? ln_bwd_rows<T, float, true>(a, parts, &summed)
                   : ln_bwd_rows<T, float, false>(a, parts, &summed);
      else
        rc = whole ? ln_bwd_rows<T, T, true>(a, parts, &summed) : ln_bwd_rows<T, T, false>(a, parts, &summed);
    } else if (a.dx && a.cols >= VE) {
      ln_bwd_dx_wide_kernel<T><<<grid_of_1024(a.rows), kWideThreads, 0, a.s>>>(
          dy, x, a.weight, a.mean, a.rstd, static_cast<T*>(a.dx), a.param_dtype, a.rows, a.cols);
      MCKE_LAUNCH_CHECK("ln_bwd_dx_wide_kernel");
    } else if (a.dx) {
      ln_bwd_dx_any_kernel<T><<<grid_of_1024(a.rows), kThreads, 0, a.s>>>(
          dy, x, a.weight, a.mean, a.rstd, static_cast<T*>(a.dx), a.param_dtype, a.rows, a.cols);
      MCKE_LAUNCH_CHECK("ln_bwd_dx_any_kernel");
    }
    if (rc) return rc;
  }
  if (!params) return ok();
  if (parts > 0 && !summed) {
    const int vec = a.cols < VE ? 1 : VE;
    const dim3 grid(static_cast<unsigned>((a.cols + int64_t{kThreads} * vec - 1) /
                                          (int64_t{kThreads} * vec)),
                    static_cast<unsigned>(parts));
    auto* fn = a.cols < VE ? &ln_bwd_params_kernel<T, true> : &ln_bwd_params_kernel<T, false>;
    fn<<<grid, kThreads, 0, a.s>>>(dy, x, a.mean, a.rstd, a.ws, a.rows, a.cols, parts);
    MCKE_LAUNCH_CHECK("ln_bwd_params_kernel");
  }
  return ln_fold_any(a, parts);
}

// The widest row: a lane per column of it is within the grid's 32-bit work size.
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
  const LnFwdArgs a{x, weight, bias, y, mean, rstd, param_dtype, rows, cols, eps,
                    static_cast<hipStream_t>(stream)};
  if (dtype == MCKE_DTYPE_F32) return ln_fwd<float>(a);
  if (dtype == MCKE_DTYPE_F16) return ln_fwd<_Float16>(a);
  return ln_fwd<__bf16>(a);
}

size_t mcke_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  // The most that any type needs.
  const int p32 = ln_parts(rows, cols, 4), p16 = ln_parts(rows, cols, 8);
  return 2 * sizeof(float) * static_cast<size_t>(p32 > p16 ? p32 : p16) * static_cast<size_t>(cols);
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
