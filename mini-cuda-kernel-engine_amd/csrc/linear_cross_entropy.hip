// linear_cross_entropy.hip -- softmax cross entropy of hidden states and a vocabulary's weights,
// and its gradients, without the logits being kept.
//
//   z = scale H W^T (H: rows x dim, W: vocab x dim, as layers hold it)
//   lse = log sum exp z,  loss = lse - z[target]
//   dz = scale ((dloss + dlse) p - dloss [j == target]),  p = exp(z - lse)
//   dH = dz W,  dW = dz^T H
//
// Forward.  Each tile of logits stays in the accumulation registers: a wave reduces its rows to
// (largest logit, sum of exponentials against it) and stores those two numbers and the target's
// logit.  A second launch joins them.  What is written is 8 bytes for 128 (or 64) logits.
//
// Backward.  The vocabulary goes in pieces.  For each, the logits are computed once more (the
// third of three products: the alternative is to keep them), become dz in 16 bits, and two more
// products take dz: dH adds up over the pieces in fp32, dW's rows are the piece's own.  dz is
// rounded to the operands' type because the matrix cores take it so: at most half a step
// relative to each value, as the rounding of a stored logit's gradient would be.  (With the outputs'
// own rounding, 1.6e-3 of the gradients' size in bf16, they are off by 1.7e-3 at 4096 x 131072 x 4096 and
// 1.9e-3 where few terms add up, 7 x 5248 x 64; in fp16 by 2.3e-4 to 2.8e-4 for 2.1e-4.)  It is stored
// relative to the largest gradient m of a row, as 2^14 dz / m, and the fp32 sums are multiplied by m
// 2^-14.  With that, fp16 keeps all bits of p down to 4e-9 (dloss is often 1 / rows, and its
// own smallest full value is 6e-5); and where all rows have the same dloss, as under a mean, the
// target's - dloss is -2^14 with no rounding, in either type.  (It is the largest term of dH,
// and rounds to the same side in all rows: 2047 rows, 32001 tokens, fp16, off by 3.5e-4 of the
// gradients' size with a power of two for m, 2.4e-4 like this; 2.1e-4 is the outputs' own rounding.)
//
// Rows without a target (target < 0) are not read.  The rows that have one are copied side by
// side first, which skips the products of the others and ends rows and columns with zeros at
// whole stages of the products.  (4096 x 4096: 25 us of 9 ms.)  How many there are is known on the
// device alone: the launches cover all rows, and workgroups past the last one end.
//
// The weights are read as they are where dim is even: 16-byte loads that end behind a row meet the
// zeros of the hidden states.  The last rows, whose loads would leave the matrix, are a copy.  Odd
// rows are not at 4-byte addresses, as loads into LDS need them: they are copied a piece at a time
// into rows of whole stages.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "common.hpp"
#include "device_math.hpp"
#include "elem.hpp"
#include "gemm_lp_any.hpp"
#include "linear_cross_entropy_plan.hpp"

namespace mcke_amd {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kPrepThreads = 1024;
constexpr int kThreads = 256;

// Device-side facts that the launches of a call share.
struct Meta {
  int rows;            // that have a target
  float factor;        // what dz is stored times, and what takes it out again
  float unfactor;
  int pad;
};

// The rows that have a target, packed.
struct Rows {
  Meta* meta;
  int* from;           // packed row -> row
  int* rank;           // row -> packed row, or -1
  int* target;         // of packed rows; -2 where it is past the vocabulary (NaN results)
  float* lse2;         // lse log2 e                                   (backward)
  float* cp;           // what p and the target's 1 are multiplied by  (backward)
  float* ct;
};

// What dz is stored times, and its inverse, for the largest gradient m of a row.
__device__ __forceinline__ void factors(float m, float& factor, float& unfactor) {
  factor = unfactor = 1.0f;
  if (m > 0.0f) {
    m = fmaxf(m, 0x1p-100f);       // (2^14 / m stays finite)
    factor = 0x1p14f / m;
    unfactor = m * 0x1p-14f;
  }
}

struct RowsIn {
  const int64_t* targets;
  const float* lse;              // null forward
  const float* dloss;
  const float* dlse;
  int rows;
  int64_t vocab;
  float scale;
  // The largest gradient of row r, 0 where that is not finite or the row has no target.
  __device__ __forceinline__ float size(int r) const {
    if (targets[r] < 0) return 0.0f;
    const float a = dloss ? scale * dloss[r] : 0.0f, b = dlse ? scale * dlse[r] : 0.0f;
    const float big = __builtin_fabsf(a) + __builtin_fabsf(b);
    return big < __builtin_inff() ? big : 0.0f;
  }
};

// Row r, whose target is t >= 0, is packed row k.
template <bool BACKWARD>
__device__ __forceinline__ void put_row(const RowsIn& in, const Rows& out, int r, int64_t t, int k,
                                        float factor) {
  out.rank[r] = k;
  out.from[k] = r;
  out.target[k] = t < in.vocab ? static_cast<int>(t) : -2;
  if constexpr (BACKWARD) {
    const float a = in.dloss ? in.scale * in.dloss[r] * factor : 0.0f;
    const float b = in.dlse ? in.scale * in.dlse[r] * factor : 0.0f;
    out.lse2[k] = in.lse[r] * kLog2e;
    out.cp[k] = t < in.vocab ? a + b : __builtin_nanf("");
    out.ct[k] = a;
  }
}
// Row r has no target.
__device__ __forceinline__ void put_none(const Rows& out, int r, float* loss, float* lse) {
  out.rank[r] = -1;
  if (loss) loss[r] = 0.0f;
  if (lse) lse[r] = 0.0f;
}

// ---------------------------------------------------------------------------
// Rows that have a target, in order; one workgroup.
// ---------------------------------------------------------------------------
template <bool BACKWARD>
__global__ __launch_bounds__(kPrepThreads) void lce_rows_kernel(RowsIn in, Rows out,
                                                               float* __restrict__ loss,
                                                               float* __restrict__ lse) {
  constexpr int W = kPrepThreads / kWave;
  static_assert(W == 16, "a value of each wave to the lanes of a row of 16");
  __shared__ int waves[W];
  __shared__ float most[W];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  float factor = 1.0f, unfactor = 1.0f;
  if constexpr (BACKWARD) {
    float m = 0.0f;
    for (int r = threadIdx.x; r < in.rows; r += kPrepThreads) m = fmaxf(m, in.size(r));
    m = wave_max(m);
    if (lane == 0) most[wave] = m;
    __syncthreads();
    factors(wave_max<W>(most[threadIdx.x % W]), factor, unfactor);
  }
  int count = 0;
  for (int r0 = 0; r0 < in.rows; r0 += kPrepThreads) {
    const int r = r0 + threadIdx.x;
    const int64_t t = r < in.rows ? in.targets[r] : -1;
    const uint64_t set = __ballot(t >= 0);
    if (lane == 0) waves[wave] = __popcll(set);
    __syncthreads();
    int before = count + __popcll(set & ((uint64_t{1} << lane) - 1));
    for (int w = 0; w < W; ++w) {
      if (w < wave) before += waves[w];
      count += waves[w];
    }
    if (r < in.rows) {
      if (t >= 0) put_row<BACKWARD>(in, out, r, t, before, factor);
      else put_none(out, r, loss, lse);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *out.meta = Meta{count, factor, unfactor, 0};
}

// A copy of the last values of a matrix, zeros behind them.
struct Tail {
  const uint16_t* from;
  uint16_t* to;
  int64_t values, all;         // copied; written
};

typedef unsigned short u16x8 __attribute__((ext_vector_type(8), aligned(2)));

// `n` values from x (null: none) and zeros behind them, as eight.
__device__ __forceinline__ u16x8 load8(const uint16_t* __restrict__ x, int64_t n) {
  u16x8 v{};
  if (x && n >= 8) {
    v = *reinterpret_cast<const u16x8*>(x);
  } else if (x && n > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) v[e] = x[e];
  }
  return v;
}

// Workgroup `block` of `blocks` copies its part of the tail.
__device__ __forceinline__ void copy_tail(const Tail& tail, int64_t block, int64_t blocks) {
  for (int64_t i = 8 * (block * kThreads + threadIdx.x); i < tail.all; i += 8 * blocks * kThreads) {
    const u16x8 v = load8(tail.from + i, tail.values - i);
    if (i + 8 <= tail.all) {
      *reinterpret_cast<u16x8*>(tail.to + i) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < tail.all) tail.to[i + e] = v[e];
    }
  }
}

// A row of `cols` values (null: none) as one of `width`, zeros behind it.
__device__ __forceinline__ void copy_row(const uint16_t* __restrict__ row, uint16_t* __restrict__ to,
                                         int cols, int width) {
  for (int c = 8 * threadIdx.x; c < width; c += 8 * kThreads)
    *reinterpret_cast<u16x8*>(to + c) = load8(row ? row + c : nullptr, cols - c);
}

// Rows of zeros follow the packed ones up to here.
__device__ __forceinline__ int rows_up(int n) { return n > 0 ? (n + 63) / 64 * 64 : 64; }

// Packed rows: row k of `to` (`width` values, a multiple of 64) is row from[k] of x (`cols`
// values) with zeros behind it, and behind the last row are rows of zeros up to the next multiple
// of 64 (64 at least).  from null: the `given` rows as they are, and zeros up to `rows`.  A
// workgroup a row; those from `blocks` on copy the tail.
__global__ __launch_bounds__(kThreads) void lce_pack_kernel(
    const uint16_t* __restrict__ x, const int* __restrict__ from, const Meta* __restrict__ meta,
    uint16_t* __restrict__ to, int64_t given, int64_t rows, int cols, int width, int blocks,
    Tail tail) {
  if (static_cast<int>(blockIdx.x) >= blocks) {
    copy_tail(tail, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  for (int64_t k = blockIdx.x; k < rows; k += blocks) {
    const uint16_t* row = nullptr;
    if (!from) {
      if (k < given) row = x + k * cols;
    } else {
      const int n = meta->rows;
      if (k >= rows_up(n)) return;
      if (k < n) row = x + static_cast<int64_t>(from[k]) * cols;
    }
    copy_row(row, to + k * width, cols, width);
  }
}

// Both for up to kFewRows rows: each workgroup has a row, counts the targets before it, and copies
// its row there; those without a target make the zeros behind the packed rows.  (A launch less: 4
// us of 16 for two tokens over a small vocabulary.)
constexpr int kFewRows = 1024;

template <bool BACKWARD>
__global__ __launch_bounds__(kThreads) void lce_few_rows_kernel(
    RowsIn in, Rows out, float* __restrict__ loss, float* __restrict__ lse,
    const uint16_t* __restrict__ x, uint16_t* __restrict__ to, int cols, int width, int blocks,
    Tail tail) {
  constexpr int W = kThreads / kWave;
  __shared__ int counts[2][W];
  __shared__ float most[W];
  if (static_cast<int>(blockIdx.x) >= blocks) {
    copy_tail(tail, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const int mine = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int before = 0, n = 0;
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < kFewRows / kThreads; ++k) {
    const int r = k * kThreads + threadIdx.x;
    const bool has = r < in.rows && in.targets[r] >= 0;
    before += __popcll(__ballot(has && r < mine));
    n += __popcll(__ballot(has));
    if constexpr (BACKWARD)
      if (has) m = fmaxf(m, in.size(r));
  }
  if constexpr (BACKWARD) m = wave_max(m);
  if (lane == 0) {
    counts[0][wave] = before;
    counts[1][wave] = n;
    most[wave] = m;
  }
  __syncthreads();
  before = n = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    before += counts[0][w];
    n += counts[1][w];
    m = fmaxf(m, most[w]);
  }
  float factor, unfactor;
  factors(m, factor, unfactor);
  const int64_t t = mine < in.rows ? in.targets[mine] : -1;
  if (threadIdx.x == 0) {
    if (mine == 0) *out.meta = Meta{n, factor, unfactor, 0};
    if (t >= 0) put_row<BACKWARD>(in, out, mine, t, before, factor);
    else if (mine < in.rows) put_none(out, mine, loss, lse);
  }
  const int k = t >= 0 ? before : n + mine - before;
  if (k < rows_up(n))
    copy_row(t >= 0 ? x + static_cast<int64_t>(mine) * cols : nullptr,
             to + static_cast<int64_t>(k) * width, cols, width);
}

// ---------------------------------------------------------------------------
// Tiles
// ---------------------------------------------------------------------------
// The tile of this workgroup, or false where the rows that have a target end before it.
template <int BM>
__device__ __forceinline__ bool tile_of_rows(int n, int tiles_n, int& tm, int& tn) {
  const int tiles_m = n > 0 ? (n + BM - 1) / BM : 1;
  if (static_cast<int>(blockIdx.x) >= tiles_m * tiles_n) return false;
  mfma_tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
  return true;
}

// Over the lanes 16 and 32 apart, each step a swap of half the lanes of two copies.
template <class F> __device__ __forceinline__ float across_groups(float v, F f) {
  auto both = [&](auto pair) {
    const unsigned a = pair[0], b = pair[1];
    v = f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    return __builtin_bit_cast(unsigned, v);
  };
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const unsigned w = both(__builtin_amdgcn_permlane16_swap(u, u, false, false));
  both(__builtin_amdgcn_permlane32_swap(w, w, false, false));
  return v;
}

// x[row] of the rows row0, row0 + 16, .. that are below n, `none` for others.  Loaded before a
// tile's products, behind which nothing waits for them: a wave has its SIMD to itself.  (4096 x
// 65536 x 128 bf16 at 256 x 256 tiles: the forward pass takes 177 us with each row's loads where they
// are used, and with __shfl_xor across the groups; 152 like this.  It has 128 x 128 tiles now: 148.)
template <int MT, typename T>
__device__ __forceinline__ void of_rows(T (&v)[MT], const T* x, int64_t row0, int n, T none) {
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = row0 + 16 * i;
    v[i] = x[row < n ? row : 0];
    v[i] = row < n ? v[i] : none;
  }
}

struct Logits {
  const uint16_t* hidden;      // packed rows, `width` apart
  int width;                   // a multiple of 64
  Piece w;
  float scale;
};

template <int BM, int BN, int D, typename T>
__device__ __forceinline__ void logits_tile(f32x4 (&acc)[BM / 32][BN / 32], char* smem,
                                            const Logits& l, int n, int64_t m0, int64_t n0) {
  const LpOperand A{l.hidden, l.width, n > 0 ? n : 1};
  lp_any_loop<T, BM, BN, Along::kAlongK, Along::kAlongK, D>(acc, smem, A, l.w.of_logits(n0), m0, n0,
                                                            0, l.width / kStageK);
}

// (largest, sum) of each row's part in the tile: wave column wn of vocabulary tile `tile` is
// entry 2 tile + wn, `stride` values apart.
template <typename T, int BM, int BN, int D>
__global__ __launch_bounds__(kMfmaThreads, 1) void lce_stats_kernel(
    Logits l, const Meta* __restrict__ meta, const int* __restrict__ target,
    float* __restrict__ largest, float* __restrict__ sums, float* __restrict__ at_target,
    int64_t stride, int tile0, int tiles_n) {
  using S = LpAnyShape<BM, BN, Along::kAlongK, Along::kAlongK, D>;
  constexpr int MT = S::MT, NT = S::NT, WN = BN / 2;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLdsBytes];
  const int n = __builtin_amdgcn_readfirstlane(meta->rows);
  int tm, tn;
  if (!tile_of_rows<BM>(n, tiles_n, tm, tn)) return;
  const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int wm = wave / 2, wn = wave % 2, g = lane / 16, r16 = lane % 16;
  int t[MT];
  of_rows(t, target, m0 + wm * (BM / 2) + r16, n, -1);
  f32x4 acc[MT][NT];
  logits_tile<BM, BN, D, T>(acc, smem, l, n, m0, n0);

  const float c = l.scale * kLog2e;
  // Columns of the wave that are in the vocabulary, less this lane's 4 g.
  const bool cut = n0 + BN > l.w.rows;
  const int left = static_cast<int>(cut ? l.w.rows - n0 - wn * WN - 4 * g : BN);
  const int64_t at = 2 * static_cast<int64_t>(tile0 + tn) + wn;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = m0 + wm * (BM / 2) + 16 * i + r16;
    float v[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = acc_get(acc[i][j][e]);
    if (cut) {
      int past = left;
      asm("" : "+v"(past));        // (kept over the rows, the 4 NT comparisons fill the scalar file)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * j + e >= past) v[j][e] = -__builtin_inff();
    }
    float m = v[0][0];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, v[j][e]);
    m = across_groups(m, [](float a, float b) { return fmaxf(a, b); });
    // Exponentials of c v - fl(c m), one operation, and what fl() took off put back into their sum.
    const float ref = m == -__builtin_inff() ? 0.0f : m, cref = c * ref;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s += __builtin_amdgcn_exp2f(__builtin_fmaf(c, v[j][e], -cref));
    s = across_groups(s, [](float a, float b) { return a + b; });
    s *= __builtin_amdgcn_exp2f(-__builtin_fmaf(c, ref, -cref));
    if (g == 0 && row < n) {
      largest[at * stride + row] = m;
      sums[at * stride + row] = s;
    }
    // The target's column, where it is one of this wave's.
    const int tc = t[i] - static_cast<int>(l.w.first + n0 + wn * WN);
    if (__ballot(tc >= 0 && tc < WN)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tc == 16 * j + 4 * g + e) at_target[row] = v[j][e];
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// loss and lse of packed rows from their parts.  A workgroup has 2^rows_log2 rows, up to 16, and
// its other lanes the parts in turn: few loads are behind each other in a lane.  (64 rows a
// workgroup: 4 rows of 2048 parts 26 us, like this 5.)
constexpr int kJoinWaves = 16;

__global__ __launch_bounds__(kJoinWaves * kWave) void lce_join_kernel(
    const float* __restrict__ largest, const float* __restrict__ sums,
    const float* __restrict__ at_target, const int* __restrict__ from,
    const int* __restrict__ target, const Meta* __restrict__ meta, float* __restrict__ loss,
    float* __restrict__ lse_out, int64_t stride, int parts, int rows_log2, float scale) {
  __shared__ float lm[kJoinWaves][16], ls[kJoinWaves][16];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, rows = 1 << rows_log2;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) << rows_log2) + lane % rows;
  const int n = meta->rows;
  const float c = scale * kLog2e;
  if ((static_cast<int64_t>(blockIdx.x) << rows_log2) >= n) return;
  float m = -__builtin_inff(), s = 0.0f;
  auto add = [&](float m2, float s2) {
    // (An empty part has no largest logit; -inf against itself moves nothing.)
    const float most = fmaxf(m, m2);
    const float f = m == most ? 1.0f : __builtin_amdgcn_exp2f((m - most) * c);
    const float f2 = m2 == most ? 1.0f : __builtin_amdgcn_exp2f((m2 - most) * c);
    s = f * s + f2 * s2;
    m = most;
  };
  // What the result wants, on its way with the parts.
  const bool out = threadIdx.x < static_cast<unsigned>(rows) && row < n;
  const int to = out ? from[row] : 0, t = out ? target[row] : -1;
  const float z = out ? at_target[row] : 0.0f;
  const int step = kJoinWaves * kWave >> rows_log2;
  if (row < n) {
#pragma unroll 8
    for (int p = threadIdx.x >> rows_log2; p < parts; p += step)
      add(largest[p * stride + row], sums[p * stride + row]);
  }
  // The lanes of a row; then the waves, by the first one in the same way.
  auto over_lanes = [&] {
    for (int d = kWave / 2; d >= rows; d /= 2) {
      const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
      add(m2, s2);
    }
  };
  over_lanes();
  if (lane < rows) {
    lm[wave][lane] = m;
    ls[wave][lane] = s;
  }
  __syncthreads();
  if (wave > 0) return;
  m = -__builtin_inff();
  s = 0.0f;
  for (int w = lane >> rows_log2; w < kJoinWaves; w += kWave >> rows_log2)
    add(lm[w][lane % rows], ls[w][lane % rows]);
  over_lanes();
  if (!out) return;
  const float lse = __builtin_fmaf(kLn2, __builtin_amdgcn_logf(s), scale * m);
  if (lse_out) lse_out[to] = lse;
  if (loss) loss[to] = t < 0 ? __builtin_nanf("") : lse - scale * z;
}

// dz of a tile, row-major (`ld` values a row), zeros in rows and columns that pad it.
template <typename T, int BM, int BN, int D>
__global__ __launch_bounds__(kMfmaThreads, 1) void lce_dz_kernel(Logits l, Rows rows,
                                                                uint16_t* __restrict__ dz,
                                                                int64_t ld, int tiles_n) {
  using S = LpAnyShape<BM, BN, Along::kAlongK, Along::kAlongK, D>;
  using O = LpOut<T>;
  constexpr int MT = S::MT, NT = S::NT, WM = BM / 2, WN = BN / 2;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLdsBytes];
  const int n = __builtin_amdgcn_readfirstlane(rows.meta->rows);
  int tm, tn;
  if (!tile_of_rows<BM>(n, tiles_n, tm, tn)) return;
  const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int wm = wave / 2, wn = wave % 2, g = lane / 16, r16 = lane % 16;
  const int64_t row0 = m0 + wm * WM + r16;
  int target[MT];
  float lse2[MT], cps[MT];
  of_rows(target, rows.target, row0, n, -1);
  of_rows(lse2, rows.lse2, row0, n, 0.0f);
  of_rows(cps, rows.cp, row0, n, 0.0f);
  f32x4 acc[MT][NT];
  logits_tile<BM, BN, D, T>(acc, smem, l, n, m0, n0);

  const float c = l.scale * kLog2e;
  const bool cut = n0 + BN > l.w.rows;
  const int left = static_cast<int>(cut ? l.w.rows - n0 - wn * WN - 4 * g : BN);
  // Through LDS, so that the stores are whole rows: chunk q of tile row r at q ^ (r % kChunks).
  struct alignas(8) Quad { T v[4]; };
  constexpr int kRowBytes = BN * 2, kChunks = kRowBytes / 16, kSwz = kChunks < 32 ? kChunks : 32;
  static_assert(BM * kRowBytes <= S::kLdsBytes, "the tile must fit the stage buffers");
  __syncthreads();
  __builtin_amdgcn_sched_barrier(0);
  const bool whole = !cut && m0 + BM <= n;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int rt = wm * WM + 16 * i + r16;
    const int64_t row = m0 + rt;
    const bool have = row < n;
    const int t = target[i] - static_cast<int>(l.w.first + n0 + wn * WN);
    float v[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[j][e] = cps[i] * __builtin_amdgcn_exp2f(__builtin_fmaf(acc_get(acc[i][j][e]), c, -lse2[i]));
    // The target's column, where it is one of this wave's.
    if (__ballot(t >= 0 && t < WN)) {
      const float ct = have ? rows.ct[row] : 0.0f;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t == 16 * j + 4 * g + e) v[j][e] -= ct;
    }
    // Columns past the weights, and rows past the last, are zeros whatever their exponentials are.
    if (!whole) {
      int past = have ? left : 0;
      asm("" : "+v"(past));        // (as in the statistics)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * j + e >= past) v[j][e] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      Quad o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o.v[e] = O::from_f32(v[j][e]);
      const int col = wn * WN + 16 * j + 4 * g;
      *reinterpret_cast<Quad*>(smem + rt * kRowBytes + (((col / 8) ^ (rt % kSwz)) * 16) +
                               (col % 8) * 2) = o;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  constexpr int kRowsPerPass = kMfmaThreads / kChunks;
  const int q = threadIdx.x % kChunks;
  const int up = rows_up(n);
#pragma unroll 4
  for (int r0 = 0; r0 < BM; r0 += kRowsPerPass) {
    const int rt = r0 + threadIdx.x / kChunks;
    const u32x4 v =
        *reinterpret_cast<const u32x4*>(smem + rt * kRowBytes + ((q ^ (rt % kSwz)) * 16));
    if (m0 + rt < up) *reinterpret_cast<u32x4*>(dz + (m0 + rt) * ld + n0 + 8 * q) = v;
  }
}

// dH's sums over part blockIdx.y of a piece: acc = dz W, written or added to the part's sums.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(kMfmaThreads, 1) void lce_dh_kernel(
    const uint16_t* __restrict__ dz, int64_t ld, Piece w, int width,
    const Meta* __restrict__ meta, float* __restrict__ out, int64_t part_stride,
    int stages_per_part, bool add, int tiles_n) {
  using S = LpAnyShape<BM, BN, Along::kAlongK, Along::kAcrossK>;
  constexpr int MT = S::MT, NT = S::NT;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLdsBytes];
  const int n = __builtin_amdgcn_readfirstlane(meta->rows);
  int tm, tn;
  if (!tile_of_rows<BM>(n, tiles_n, tm, tn)) return;
  const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
  const int all = static_cast<int>((w.rows + 63) / 64);
  const int first = blockIdx.y * stages_per_part;
  const int stages = all - first < stages_per_part ? all - first : stages_per_part;
  if (stages <= 0) return;
  const LpOperand A{dz, ld, n > 0 ? n : 1};
  f32x4 acc[MT][NT];
  lp_any_loop<T, BM, BN, Along::kAlongK, Along::kAcrossK>(acc, smem, A, w.of_dh(), m0, n0, first,
                                                          stages);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int wm = wave / 2, wn = wave % 2, g = lane / 16, r16 = lane % 16;
  out += blockIdx.y * part_stride;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = m0 + wm * (BM / 2) + 16 * i + r16;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t col = n0 + wn * (BN / 2) + 16 * j + 4 * g;
      if (row < n && col < width) {
        f32x4* p = reinterpret_cast<f32x4*>(out + row * width + col);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc_get(acc[i][j][e]);
        if (add) v += *p;
        *p = v;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// dH from its parts' sums, the factor taken out; zeros for rows without a target.  2^lanes_log2
// lanes have eight columns of a row each, and a workgroup's other lanes the parts in turn.
template <typename T>
__global__ __launch_bounds__(kThreads) void lce_dh_store_kernel(
    const float* __restrict__ sums, int64_t part_stride, int parts, const int* __restrict__ rank,
    const Meta* __restrict__ meta, T* __restrict__ dhidden, int rows, int cols, int width,
    int lanes_log2) {
  __shared__ float fold[kThreads * 8];
  const float unfactor = meta->unfactor;
  const int lanes = 1 << lanes_log2, groups = kThreads >> lanes_log2;
  const int t = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log2;
  const int c = 8 * ((static_cast<int>(blockIdx.y) << lanes_log2) + t);
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int k = rank[r];
    float v[8] = {};
    if (k >= 0 && c < width) {
      const float* p = sums + static_cast<int64_t>(k) * width + c;
#pragma unroll 4
      for (int s = group; s < parts; s += groups) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p + s * part_stride);
        const f32x4 b = *reinterpret_cast<const f32x4*>(p + s * part_stride + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += a[e];
          v[4 + e] += b[e];
        }
      }
    }
    if (groups > 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) fold[e * kThreads + threadIdx.x] = v[e];
      __syncthreads();
      if (group == 0) {
        for (int g = 1; g < groups; ++g)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += fold[e * kThreads + g * lanes + t];
      }
      __syncthreads();         // fold is written again
    }
    if (group > 0 || c >= cols) continue;
    VecT16<T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(v[e] * unfactor);
    T* to = dhidden + static_cast<int64_t>(r) * cols + c;
    if (c + 8 <= cols) *reinterpret_cast<VecT16<T>*>(to) = o;
    else store_part<T>(to, o, cols - c);
  }
}

// dW's rows of a piece: dz^T H, the factor taken out.  ONE: for up to 64 rows, a single stage.
// `lines`: rows are whole 128-byte lines, and go past the caches, which the weights are read
// through again (4 x 131072 x 4096: the next call's logits 247 -> 178 us).  Cut lines do not: 13 x
// 27442 x 4918 took 124 us so, and 77 through the caches.
template <typename T, int BM, int BN, bool ONE>
__global__ __launch_bounds__(kMfmaThreads, ONE ? 3 : 1) void lce_dw_kernel(
    const uint16_t* __restrict__ dz, int64_t ld, const uint16_t* __restrict__ hidden, int width,
    const Meta* __restrict__ meta, T* __restrict__ dweight, int64_t piece, int cols, bool lines,
    int tiles_m, int tiles_n) {
  using S = LpAnyShape<BM, BN, Along::kAcrossK, Along::kAcrossK>;
  using O = LpOut<T>;
  constexpr int MT = S::MT, NT = S::NT, WM = BM / 2, WN = BN / 2;
  constexpr int kLds = ONE ? kLdsOne<BM, BN> : S::kLdsBytes;
  static_assert(BM * BN * 2 <= kLds, "the tile must fit the stage buffers");
  __shared__ __attribute__((aligned(1024))) char smem[kLds];
  int tm, tn;
  mfma_tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
  const int n = __builtin_amdgcn_readfirstlane(meta->rows), stages = n > 0 ? (n + 63) / 64 : 1;
  const LpOperand A{dz, ld, ld};
  const LpOperand B{hidden, width, width};
  f32x4 acc[MT][NT];
  if constexpr (ONE)
    lp_any_one<T, BM, BN, Along::kAcrossK, Along::kAcrossK>(acc, smem, A, B, m0, n0);
  else
    lp_any_loop<T, BM, BN, Along::kAcrossK, Along::kAcrossK>(acc, smem, A, B, m0, n0, 0, stages);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int wm = wave / 2, wn = wave % 2, g = lane / 16, r16 = lane % 16;
  const float unfactor = meta->unfactor;
  struct alignas(8) Quad { T v[4]; };
  constexpr int kRowBytes = BN * 2, kChunks = kRowBytes / 16, kSwz = kChunks < 32 ? kChunks : 32;
  __syncthreads();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int rt = wm * WM + 16 * i + r16;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      Quad o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o.v[e] = O::from_f32(unfactor * acc_get(acc[i][j][e]));
      const int col = wn * WN + 16 * j + 4 * g;
      *reinterpret_cast<Quad*>(smem + rt * kRowBytes + (((col / 8) ^ (rt % kSwz)) * 16) +
                               (col % 8) * 2) = o;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  constexpr int kRowsPerPass = kMfmaThreads / kChunks;
  const int q = threadIdx.x % kChunks;
  const int64_t col = n0 + 8 * q;
#pragma unroll 4
  for (int r0 = 0; r0 < BM; r0 += kRowsPerPass) {
    const int rt = r0 + threadIdx.x / kChunks;
    const u32x4 v =
        *reinterpret_cast<const u32x4*>(smem + rt * kRowBytes + ((q ^ (rt % kSwz)) * 16));
    if (m0 + rt >= piece) continue;
    T* to = dweight + (m0 + rt) * cols + col;
    if (col + 8 <= cols) {
      if (lines) __builtin_nontemporal_store(static_cast<u32x4_a2>(v), reinterpret_cast<u32x4_a2*>(to));
      else *reinterpret_cast<u32x4_a2*>(to) = v;
    } else {
      const VecT16<T> w = __builtin_bit_cast(VecT16<T>, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < cols) to[e] = w[e];
    }
  }
}

// No rows: the weights have no gradient.
__global__ __launch_bounds__(kThreads) void lce_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    p[i] = 0;
}

// ---------------------------------------------------------------------------
// Plans of either pass
// ---------------------------------------------------------------------------
struct RowsAt {
  int64_t meta, from, rank, target, lse2, cp, ct, hidden, weight;
  RowsAt(Plan& p, bool backward) {
    meta = p.take(sizeof(Meta));
    from = p.take(4 * p.up);
    rank = p.take(4 * p.up);
    target = p.take(4 * p.up);
    lse2 = cp = ct = 0;
    if (backward) {
      lse2 = p.take(4 * p.up);
      cp = p.take(4 * p.up);
      ct = p.take(4 * p.up);
    }
    hidden = p.take(2 * p.up * p.width);
    weight = p.take(p.pad ? 2 * p.piece * p.width : 2 * p.tail_values);
  }
  Rows rows(char* ws) const {
    return {reinterpret_cast<Meta*>(ws + meta),     reinterpret_cast<int*>(ws + from),
            reinterpret_cast<int*>(ws + rank),      reinterpret_cast<int*>(ws + target),
            reinterpret_cast<float*>(ws + lse2),    reinterpret_cast<float*>(ws + cp),
            reinterpret_cast<float*>(ws + ct)};
  }
};

struct FwdPlan : Plan {
  RowsAt r;
  int64_t stride, parts, largest, sums, at_target;
  FwdPlan(int64_t rows, int64_t vocab, int64_t dim) : Plan(rows, vocab, dim, false), r(*this, false) {
    stride = rows < 64 ? rows : up;      // (lines of 64 for 4 rows of 2048 parts: 8 us more)
    parts = 2 * ceil_div(vocab, tile_cols(tile));
    largest = take(4 * parts * stride);
    sums = take(4 * parts * stride);
    at_target = take(4 * up);
  }
};

struct BwdPlan : Plan {
  RowsAt r;
  Tile dh_tile, dw_tile;
  int64_t dz, ld, dh_tiles, parts, stages_per_part, dh, part_stride;   // (tiles and parts of dH)
  BwdPlan(int64_t rows, int64_t vocab, int64_t dim) : Plan(rows, vocab, dim, true), r(*this, true) {
    ld = piece;
    dz = take(2 * up * ld);
    // Few tiles of dH share a piece's stages: up to a workgroup a CU at 256 x 256 and two at smaller
    // tiles, at least 8 stages each, and up to 80 MB of sums.  256 x 256 from 192 workgroups on
    // (2047 x 32001 x 1024 fp16: 109 us with 8 parts, against 136 at 128 x 128 with 4).
    part_stride = up * width;
    const int64_t stages = ceil_div(at_once(), 64);
    auto share = [&](Tile t) {
      dh_tiles = ceil_div(rows, tile_rows(t)) * ceil_div(dim, tile_cols(t));
      parts = (t == Tile::k256 ? 256 : 512) / dh_tiles;
      if (parts > 20 * (int64_t{1} << 20) / part_stride) parts = 20 * (int64_t{1} << 20) / part_stride;
      if (parts > ceil_div(stages, 8)) parts = ceil_div(stages, 8);
      if (parts < 1) parts = 1;
      stages_per_part = ceil_div(stages, parts);
      parts = ceil_div(stages, stages_per_part);
    };
    dh_tile = Tile::k256;
    if (rows > 128 && dim > 128) share(dh_tile);
    if (rows <= 128 || dim <= 128 || dh_tiles * parts < 192) {
      dh_tile = rows <= 64 ? Tile::k64x128 : Tile::k128;
      share(dh_tile);
    }
    dh = take(4 * parts * part_stride);
    dw_tile = rows > 128 && ceil_div(piece, 256) * ceil_div(dim, 256) >= 192 ? Tile::k256 : Tile::k128;
  }
};

// f(BM, BN) as std::integral_constants, for a tile.
template <class F> int with_tile(Tile t, F f) {
  using I64 = std::integral_constant<int, 64>;
  using I128 = std::integral_constant<int, 128>;
  using I256 = std::integral_constant<int, 256>;
  if (t == Tile::k64x128) return f(I64{}, I128{});
  if (t == Tile::k128) return f(I128{}, I128{});
  return f(I256{}, I256{});
}

// f(BM, BN, D) for tiles of logits: with as many stages in flight as LDS holds where each has a CU
// for itself, with two elsewhere.
template <class F> int with_logits_tile(Tile t, int64_t tiles, F f) {
  return with_tile(t, [&](auto bm, auto bn) {
    constexpr int BM = decltype(bm)::value;
    constexpr int kDeep = BM == 64 ? 6 : BM == 128 ? 4 : 2;
    if (tiles <= 256) return f(bm, bn, std::integral_constant<int, kDeep>{});
    return f(bm, bn, std::integral_constant<int, 2>{});
  });
}

unsigned tail_blocks(const Tail& tail) {
  const int64_t blocks = ceil_div(tail.all, 8 * kThreads);
  return static_cast<unsigned>(blocks < 1024 ? blocks : 1024);
}

int launch_pack(const void* x, const int* from, const Meta* meta, void* to, int64_t given,
                int64_t rows, int64_t cols, int64_t width, const Tail& tail, hipStream_t s) {
  const int blocks = static_cast<int>(rows < 65536 ? rows : 65536);
  lce_pack_kernel<<<static_cast<unsigned>(blocks) + tail_blocks(tail), kThreads, 0, s>>>(
      static_cast<const uint16_t*>(x), from, meta, static_cast<uint16_t*>(to), given, rows,
      static_cast<int>(cols), static_cast<int>(width), blocks, tail);
  MCKE_LAUNCH_CHECK("lce_pack_kernel");
  return ok();
}

// The rows that have a target, their hidden states, and the tail of the weights.
template <bool BACKWARD>
int pack_rows(const Plan& p, const RowsAt& r, const RowsIn& in, float* loss, float* lse,
              const void* hidden, const void* weight, char* ws, hipStream_t s) {
  const Rows rows = r.rows(ws);
  const uint16_t* last = static_cast<const uint16_t*>(weight) + p.tail_first * p.dim;
  const Tail tail{last, reinterpret_cast<uint16_t*>(ws + r.weight),
                  p.tail_values ? (p.vocab - p.tail_first) * p.dim : 0, p.tail_values};
  if (p.rows <= kFewRows) {
    lce_few_rows_kernel<BACKWARD>
        <<<static_cast<unsigned>(p.up) + tail_blocks(tail), kThreads, 0, s>>>(
            in, rows, loss, lse, static_cast<const uint16_t*>(hidden),
            reinterpret_cast<uint16_t*>(ws + r.hidden), static_cast<int>(p.dim),
            static_cast<int>(p.width), static_cast<int>(p.up), tail);
    MCKE_LAUNCH_CHECK("lce_few_rows_kernel");
    return ok();
  }
  lce_rows_kernel<BACKWARD><<<1, kPrepThreads, 0, s>>>(in, rows, loss, lse);
  MCKE_LAUNCH_CHECK("lce_rows_kernel");
  return launch_pack(hidden, rows.from, rows.meta, ws + r.hidden, p.rows, p.up, p.dim, p.width,
                     tail, s);
}

// Calls f(piece) for each piece of the weights.
template <class F>
int for_pieces(const Plan& p, const RowsAt& r, const void* weight, char* ws, hipStream_t s, F f) {
  uint16_t* copy = reinterpret_cast<uint16_t*>(ws + r.weight);
  for (int64_t i = 0; i < p.pieces; ++i) {
    const Piece piece = p.piece_of(i, static_cast<const uint16_t*>(weight), copy);
    if (p.pad) {
      const uint16_t* w = static_cast<const uint16_t*>(weight) + piece.first * p.dim;
      if (int rc = launch_pack(w, nullptr, nullptr, copy, piece.rows, round_up(piece.rows, 64),
                               p.dim, p.width, Tail{nullptr, nullptr, 0, 0}, s))
        return rc;
    }
    if (int rc = f(piece)) return rc;
  }
  return ok();
}

template <typename T>
int lce_forward(const void* hidden, const void* weight, const int64_t* targets, float* loss,
                float* lse, const FwdPlan& p, float scale, char* ws, hipStream_t s) {
  const Rows rows = p.r.rows(ws);
  const RowsIn in{targets, nullptr, nullptr, nullptr, static_cast<int>(p.rows), p.vocab, scale};
  if (int rc = pack_rows<false>(p, p.r, in, loss, lse, hidden, weight, ws, s)) return rc;
  const uint16_t* packed = reinterpret_cast<const uint16_t*>(ws + p.r.hidden);
  float* largest = reinterpret_cast<float*>(ws + p.largest);
  float* sums = reinterpret_cast<float*>(ws + p.sums);
  float* at_target = reinterpret_cast<float*>(ws + p.at_target);
  const int rc = for_pieces(p, p.r, weight, ws, s, [&](const Piece& w) {
    return with_logits_tile(p.tile, p.logits_tiles(w.rows), [&](auto bm, auto bn, auto d) {
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, D = decltype(d)::value;
      const int64_t tiles_n = ceil_div(w.rows, BN), tiles = p.logits_tiles(w.rows);
      lce_stats_kernel<T, BM, BN, D><<<static_cast<unsigned>(tiles), kMfmaThreads, 0, s>>>(
          Logits{packed, static_cast<int>(p.width), w, scale}, rows.meta, rows.target, largest,
          sums, at_target, p.stride, static_cast<int>(w.first / BN), static_cast<int>(tiles_n));
      MCKE_LAUNCH_CHECK("lce_stats_kernel");
      return ok();
    });
  });
  if (rc) return rc;
  int rows_log2 = 0;
  while (rows_log2 < 4 && (int64_t{1} << rows_log2) < p.rows) ++rows_log2;
  lce_join_kernel<<<static_cast<unsigned>(ceil_div(p.rows, int64_t{1} << rows_log2)),
                    kJoinWaves * kWave, 0, s>>>(
      largest, sums, at_target, rows.from, rows.target, rows.meta, loss, lse, p.stride,
      static_cast<int>(p.parts), rows_log2, scale);
  MCKE_LAUNCH_CHECK("lce_join_kernel");
  return ok();
}

struct BwdArgs {
  const void* hidden;
  const void* weight;
  const int64_t* targets;
  const float* lse;
  const float* dloss;
  const float* dlse;
  void* dhidden;
  void* dweight;
  float scale;
  char* ws;
  hipStream_t s;
};

template <typename T> int lce_backward(const BwdArgs& a, const BwdPlan& p) {
  const Rows rows = p.r.rows(a.ws);
  const RowsIn in{a.targets, a.lse, a.dloss, a.dlse, static_cast<int>(p.rows), p.vocab, a.scale};
  if (int rc = pack_rows<true>(p, p.r, in, nullptr, nullptr, a.hidden, a.weight, a.ws, a.s))
    return rc;
  const uint16_t* packed = reinterpret_cast<const uint16_t*>(a.ws + p.r.hidden);
  const bool lines = p.dim % 64 == 0 && aligned(a.dweight, 128);
  uint16_t* dz = reinterpret_cast<uint16_t*>(a.ws + p.dz);
  float* dh = reinterpret_cast<float*>(a.ws + p.dh);
  const int width = static_cast<int>(p.width);
  const int rc =
      for_pieces(p, p.r, a.weight, a.ws, a.s, [&](const Piece& w) {
        int rc = with_logits_tile(p.tile, p.logits_tiles(w.rows), [&](auto bm, auto bn, auto d) {
          constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, D = decltype(d)::value;
          const int64_t tiles_n = ceil_div(w.rows, BN), tiles = p.logits_tiles(w.rows);
          lce_dz_kernel<T, BM, BN, D><<<static_cast<unsigned>(tiles), kMfmaThreads, 0, a.s>>>(
              Logits{packed, width, w, a.scale}, rows, dz, p.ld, static_cast<int>(tiles_n));
          MCKE_LAUNCH_CHECK("lce_dz_kernel");
          return ok();
        });
        if (rc) return rc;
        if (a.dhidden) {
          rc = with_tile(p.dh_tile, [&](auto bm, auto bn) {
            constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value;
            const int64_t tiles_n = ceil_div(p.dim, BN), tiles = ceil_div(p.rows, BM) * tiles_n;
            lce_dh_kernel<T, BM, BN>
                <<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(p.parts)),
                   kMfmaThreads, 0, a.s>>>(dz, p.ld, w, width, rows.meta, dh, p.part_stride,
                                           static_cast<int>(p.stages_per_part), w.first > 0,
                                           static_cast<int>(tiles_n));
            MCKE_LAUNCH_CHECK("lce_dh_kernel");
            return ok();
          });
          if (rc) return rc;
        }
        if (!a.dweight) return ok();
        auto dw = [&](auto bt, auto one) {
          constexpr int B = decltype(bt)::value;
          const int64_t tiles_m = ceil_div(w.rows, B), tiles_n = ceil_div(p.dim, B);
          lce_dw_kernel<T, B, B, decltype(one)::value>
              <<<static_cast<unsigned>(tiles_m * tiles_n), kMfmaThreads, 0, a.s>>>(
                  dz, p.ld, packed, width, rows.meta, static_cast<T*>(a.dweight) + w.first * p.dim,
                  w.rows, static_cast<int>(p.dim), lines, static_cast<int>(tiles_m),
                  static_cast<int>(tiles_n));
          MCKE_LAUNCH_CHECK("lce_dw_kernel");
          return ok();
        };
        using I128 = std::integral_constant<int, 128>;
        if (p.rows <= 64) return dw(I128{}, std::true_type{});
        if (p.dw_tile == Tile::k256)
          return dw(std::integral_constant<int, 256>{}, std::false_type{});
        return dw(I128{}, std::false_type{});
      });
  if (rc) return rc;
  if (!a.dhidden) return ok();
  // A wave a row and four groups of parts where there are parts, else as many lanes as columns.
  int lanes_log2 = 3;
  while (lanes_log2 < (p.parts > 4 ? 6 : 8) && (int64_t{8} << lanes_log2) < p.width) ++lanes_log2;
  const dim3 grid(static_cast<unsigned>(p.rows < 65536 ? p.rows : 65536),
                  static_cast<unsigned>(ceil_div(p.width, int64_t{8} << lanes_log2)));
  lce_dh_store_kernel<T><<<grid, kThreads, 0, a.s>>>(
      dh, p.part_stride, static_cast<int>(p.parts), rows.rank, rows.meta,
      static_cast<T*>(a.dhidden), static_cast<int>(p.rows), static_cast<int>(p.dim), width,
      lanes_log2);
  MCKE_LAUNCH_CHECK("lce_dh_store_kernel");
  return ok();
}

constexpr int64_t kMaxRows = int64_t{1} << 24, kMaxVocab = int64_t{1} << 24,
                  kMaxDim = int64_t{1} << 16;

bool extents_fit(int64_t rows, int64_t vocab, int64_t dim) {
  return rows <= kMaxRows && vocab <= kMaxVocab && dim <= kMaxDim;
}

int check_args(const std::string& who, int dtype, int64_t rows, int64_t vocab, int64_t dim,
               float scale) {
  if (dtype != MCKE_DTYPE_F16 && dtype != MCKE_DTYPE_BF16)
    return invalid(who + ": dtype must be MCKE_DTYPE_BF16 or MCKE_DTYPE_F16, got " +
                   std::to_string(dtype));
  if (rows < 0 || vocab < 0 || dim < 0) return invalid(who + ": negative extent");
  if (!extents_fit(rows, vocab, dim))
    return invalid(who + ": too large: rows and vocab up to 2^24, dim up to 2^16");
  if (!(scale > 0.0f) || !std::isfinite(scale) || !std::isfinite(scale * kLog2e))
    return invalid(who + ": scale must be finite and > 0");
  return ok();
}

int check_workspace(const std::string& who, const void* ws, size_t bytes, size_t need) {
  if (!ws || bytes < need || !aligned(ws, 16))
    return invalid(who + ": needs a 16-byte aligned workspace of " + std::to_string(need) +
                   " bytes, got " + std::to_string(ws ? bytes : 0));
  return ok();
}

int check_weight(const std::string& who, const void* weight, int64_t dim) {
  if (dim % 2 == 0 && !aligned(weight, 4))
    return invalid(who + ": weight must be 4-byte aligned where dim is even");
  return ok();
}

}  // namespace
}  // namespace mcke_amd

using namespace mcke_amd;

extern "C" {

size_t mcke_linear_cross_entropy_workspace_bytes(int64_t rows, int64_t vocab, int64_t dim) {
  if (rows <= 0 || vocab <= 0 || dim <= 0 || !extents_fit(rows, vocab, dim)) return 0;
  return static_cast<size_t>(FwdPlan(rows, vocab, dim).at);
}

size_t mcke_linear_cross_entropy_backward_workspace_bytes(int64_t rows, int64_t vocab,
                                                          int64_t dim) {
  if (rows <= 0 || vocab <= 0 || dim <= 0 || !extents_fit(rows, vocab, dim)) return 0;
  return static_cast<size_t>(BwdPlan(rows, vocab, dim).at);
}

int mcke_launch_linear_cross_entropy(const void* hidden, const void* weight, const int64_t* targets,
                                     float* loss, float* lse, int dtype, int64_t rows,
                                     int64_t vocab, int64_t dim, float scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const std::string who = "launch_linear_cross_entropy";
  if (int rc = check_args(who, dtype, rows, vocab, dim, scale)) return rc;
  if (rows == 0) return ok();
  if (vocab == 0 || dim == 0) return invalid(who + ": vocab and dim must be > 0");
  if (!hidden || !weight || !targets) return invalid(who + ": null pointer");
  if (!loss && !lse) return invalid(who + ": no output is asked for");
  if (!aligned(hidden, 2) || !aligned(weight, 2) || !aligned(targets, 8) || !aligned(loss, 4) ||
      !aligned(lse, 4))
    return invalid(who + ": a pointer is not aligned to its type");
  if (int rc = check_weight(who, weight, dim)) return rc;
  const FwdPlan p(rows, vocab, dim);
  if (!p.fits())
    return invalid(who + ": rows x vocab exceed the grid's 32-bit work size");
  const size_t need = static_cast<size_t>(p.at);
  if (int rc = check_workspace(who, workspace, workspace_bytes, need)) return rc;
  const uint64_t n = rows, h = 2 * n * dim, w = 2 * static_cast<uint64_t>(vocab) * dim;
  const void* outs[] = {loss, lse, workspace};
  const uint64_t out_bytes[] = {4 * n, 4 * n, need};
  for (int i = 0; i < 3; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], hidden, h) ||
               overlap(outs[i], out_bytes[i], weight, w) ||
               overlap(outs[i], out_bytes[i], targets, 8 * n);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid(who + ": an output or the workspace overlaps another operand, which violates "
                           "the __restrict__ contract");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  return dtype == MCKE_DTYPE_F16
             ? lce_forward<_Float16>(hidden, weight, targets, loss, lse, p, scale, ws, s)
             : lce_forward<__bf16>(hidden, weight, targets, loss, lse, p, scale, ws, s);
}

int mcke_launch_linear_cross_entropy_backward(const void* hidden, const void* weight,
                                              const int64_t* targets, const float* lse,
                                              const float* dloss, const float* dlse, void* dhidden,
                                              void* dweight, int dtype, int64_t rows, int64_t vocab,
                                              int64_t dim, float scale, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  const std::string who = "launch_linear_cross_entropy_backward";
  if (int rc = check_args(who, dtype, rows, vocab, dim, scale)) return rc;
  if (!dhidden && !dweight) return invalid(who + ": no gradient is asked for");
  if (vocab == 0 || dim == 0) {
    if (rows == 0) return ok();
    return invalid(who + ": vocab and dim must be > 0");
  }
  if (rows > 0 && (!hidden || !weight || !targets || !lse)) return invalid(who + ": null pointer");
  if (rows > 0 && !dloss && !dlse) return invalid(who + ": no gradient is given");
  if (!aligned(hidden, 2) || !aligned(weight, 2) || !aligned(dhidden, 2) || !aligned(dweight, 2) ||
      !aligned(targets, 8) || !aligned(lse, 4) || !aligned(dloss, 4) || !aligned(dlse, 4))
    return invalid(who + ": a pointer is not aligned to its type");
  if (rows == 0) {
    if (!dweight) return ok();
    lce_zero_kernel<<<1024, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<uint16_t*>(dweight), vocab * dim);
    MCKE_LAUNCH_CHECK("lce_zero_kernel");
    return ok();
  }
  if (int rc = check_weight(who, weight, dim)) return rc;
  const BwdPlan p(rows, vocab, dim);
  const size_t need = static_cast<size_t>(p.at);
  if (int rc = check_workspace(who, workspace, workspace_bytes, need)) return rc;
  const uint64_t n = rows, h = 2 * n * dim, w = 2 * static_cast<uint64_t>(vocab) * dim;
  const void* outs[] = {dhidden, dweight, workspace};
  const uint64_t out_bytes[] = {h, w, need};
  for (int i = 0; i < 3; ++i) {
    bool bad = overlap(outs[i], out_bytes[i], hidden, h) ||
               overlap(outs[i], out_bytes[i], weight, w) ||
               overlap(outs[i], out_bytes[i], targets, 8 * n) ||
               overlap(outs[i], out_bytes[i], lse, 4 * n) ||
               overlap(outs[i], out_bytes[i], dloss, 4 * n) ||
               overlap(outs[i], out_bytes[i], dlse, 4 * n);
    for (int j = 0; j < i; ++j) bad |= overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]);
    if (bad)
      return invalid(who + ": an output or the workspace overlaps another operand, which violates "
                           "the __restrict__ contract");
  }
  const BwdArgs a{hidden,  weight,  targets, lse,   dloss, dlse, dhidden,
                  dweight, scale,   static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
  return dtype == MCKE_DTYPE_F16 ? lce_backward<_Float16>(a, p) : lce_backward<__bf16>(a, p);
}

}  // extern "C"
