// gemm_lp_launch.hpp -- which kernel a 16-bit-input product runs, by shape and alignment, for
// the plain product and for the one with an epilogue (gemm_lp_epilogue.hpp).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "common.hpp"
#include "gemm_lp.hpp"
#include "gemm_lp_split.hpp"

namespace mcke_amd {

using LpKernel = const void*;

// Direct-to-LDS 16x16x32 kernel for a BM x BN tile: whole tiles with 16-byte aligned
// operands and K % 64 == 0, or the EDGE form.  Its per-lane source offsets are 32-bit: BM
// rows of A and 64 rows of B must span less than 4 GiB.
template <int BM, int BN>
bool dma_offsets32(int n, int k) {
  return static_cast<int64_t>(BM) * k * 2 + 4096 < (int64_t{1} << 32) &&
         static_cast<int64_t>(64) * n * 2 < (int64_t{1} << 32);
}

inline int64_t tile_count(int m, int n, int bm, int bn) {
  return static_cast<int64_t>(steps_along(m, bm)) * steps_along(n, bn);
}

template <class E>
struct LpArgs {
  const uint16_t* a;
  const uint16_t* b;
  void* c;
  int m, n, k;
  float alpha, beta;
  E ep;
  hipStream_t s;
};

template <class E>
int check_grid(int64_t tiles, int threads) {
  if (tiles * threads > int64_t{UINT32_MAX})
    return invalid(std::string(E::kFused ? "launch_gemm_lp_bias_act" : "launch_gemm_lp") +
                   ": tiles x lanes exceed the grid's 32-bit work size; use a larger tile");
  return ok();
}

template <typename T, typename OutT, int BM, int BN, bool EDGE, class E>
int launch_dma(const LpArgs<E>& x) {
  const int64_t tiles = tile_count(x.m, x.n, BM, BN);
  if (int rc = check_grid<E>(tiles, kMfmaThreads)) return rc;
  gemm_lp_dma16_kernel<T, OutT, BM, BN, EDGE, E>
      <<<static_cast<unsigned>(tiles), kMfmaThreads, 0, x.s>>>(
          x.a, x.b, static_cast<OutT*>(x.c), x.m, x.n, x.k, x.alpha, x.beta,
          steps_along(x.m, BM), steps_along(x.n, BN), x.ep);
  MCKE_LAUNCH_CHECK("gemm_lp_dma16_kernel");
  return ok();
}

template <typename T, typename OutT, int MT, int NW, int WV, int AHEAD = 1, class E>
int launch_split_as(const LpArgs<E>& x) {
  constexpr int TM = 16 * MT, TN = 16 * NW;
  const int64_t tiles = tile_count(x.m, x.n, TM, TN);
  if (int rc = check_grid<E>(tiles, WV * kWave)) return rc;
  gemm_lp_split_kernel<T, OutT, MT, NW, WV, E, AHEAD>
      <<<static_cast<unsigned>(tiles), WV * kWave, 0, x.s>>>(
          x.a, x.b, static_cast<OutT*>(x.c), x.m, x.n, x.k, x.alpha, x.beta,
          steps_along(x.m, TM), steps_along(x.n, TN), x.ep);
  MCKE_LAUNCH_CHECK("gemm_lp_split_kernel");
  return ok();
}

// The split-K kernel by shape.  Few rows over up to 8192 columns: 32 columns a workgroup
// and 8 waves, for as many workgroups as there are (16 x 4096 x 4096: 16 x 32 11.9 us,
// 32 x 64 14.8, 64 x 64 16.4; 16 x 16384 x 4096: 38.6, 25.8, 26.8).  Else 32 x 64 up to
// four tiles per CU (64 x 4096 x 4096: 15.6 us against 21.3 for 64 x 64; 1628 x 800 x 1109:
// 14.9 against 17.4), 64 x 64 past that (1531 x 4096 x 1024: 28.2 against 33.3;
// 4032 x 843 x 2744: 62.7 against 83.8).  Widths of 32 .. 63 take 32 columns.
template <typename T, typename OutT, class E>
int launch_split(const LpArgs<E>& x) {
  if (x.n < 64 || (x.m <= 32 && x.n <= 8192))
    return x.m <= 16 ? launch_split_as<T, OutT, 1, 2, 8>(x) : launch_split_as<T, OutT, 2, 2, 8>(x);
  if (tile_count(x.m, x.n, 32, 64) <= 1024) return launch_split_as<T, OutT, 2, 4, 4>(x);
  return launch_split_as<T, OutT, 4, 4, 4>(x);
}

// Few rows (tokens) with an epilogue: bound by reading B, of which these kernels' loads bring 8 to 9
// bytes a clock to a CU, more of it from whole 128-byte lines.  So as many workgroups as there are CUs
// where N allows it, then 64 columns each (with bias and GELU, bf16, us; MT x NW, waves,
// chunks ahead):
//   rows 1, K 4096:   N 16384  1x4 4w 25.2, 1x2 8w 41, 128 x 128 tiles 48   N 12288  1x4 4w two ahead
//     22.6, one 23.8   N 8192  1x2 8w 13.6, 1x4 13.6   N 4096  1x1 8w two ahead 11.4, 1x2 8w 11.8
//   rows 1, K 16384:  N 4096  1x1 53.8, 1x2 61      N 1000  1x1 28, 1x2 31
//   rows 32:          32 x 4096 x 16384  1x2 two ahead 62.6, one 66.8    32 x 8192 x 4096  1x4 8w
//     15.4, 2x2 8w 16.2      32 x 16384 x 4096  2x4 4w 29.0, 4x4 4w 29.9
//   rows 64:          64 x 4096 x 16384  2x2 8w two ahead 66.5, one 72.8, 1x4 8w 70.0
//     64 x 8192 x 4096  2x4 8w 17.3, 2x4 4w 19.8    64 x 16384 x 4096  4x4 8w 37.4, 4w 40.4
// Past 16384 columns each workgroup's A comes to a second round of workgroups: from 33 rows on, and
// from 17 on where N is odd, the other products' kernels (bf16 with bias, these and those, us):
//   K 4096:   64 x 16384  35.7  48.7   64 x 16400  51.7  48.9   64 x 24576  62.8  51.3   64 x 131072  306  236
//     33 x 16384  31.4  48.3   33 x 24576  52.5  50.9   33 x 131072  262  234   32 x 24576  53.7  50.7
//     32 x 50304  94.5  95.6   32 x 50257  118  101     16 x 50257  104  99     1 x 50257  92.4  99.5
//   K 1024:   64 x 16384  10.6  14.5   64 x 24576  17.9  14.8   33 x 24576  16.2  14.3
//     32 x 24576  13.0  14.0   32 x 50304  24.5  32.6   32 x 50257  29.8  28.7   17 x 50257  26.9  28.3
template <class E> bool few_rows(const LpArgs<E>& x) {
  return x.m <= 64 && x.n >= 64 && x.k >= 64 &&
         (x.n <= 16384 || x.m <= 16 || (x.m <= 32 && x.n % 2 == 0));
}
template <typename T, typename OutT, class E>
int launch_few_rows(const LpArgs<E>& x) {
  if (x.m <= 16) {
    if (x.n <= 4096) return launch_split_as<T, OutT, 1, 1, 8, 2>(x);
    if (x.n <= 8192) return launch_split_as<T, OutT, 1, 2, 8>(x);
    if (x.n < 16384) return launch_split_as<T, OutT, 1, 4, 4, 2>(x);
    return launch_split_as<T, OutT, 1, 4, 4>(x);
  }
  if (x.m <= 32) {
    if (x.n <= 4096) return launch_split_as<T, OutT, 1, 2, 8, 2>(x);
    if (x.n <= 8192) return launch_split_as<T, OutT, 1, 4, 8>(x);
    return launch_split_as<T, OutT, 2, 4, 4>(x);
  }
  if (x.n <= 4096) return launch_split_as<T, OutT, 2, 2, 8, 2>(x);
  if (x.n <= 8192) return launch_split_as<T, OutT, 2, 4, 8>(x);
  return launch_split_as<T, OutT, 4, 4, 8>(x);
}

// The register-staged kernel's checked forms at the requested tile: what is narrower than
// any other kernel's tile, or past their 32-bit offsets or grids.
template <typename T, typename OutT, int BM, int BN, class E>
int launch_staged(const LpArgs<E>& x, bool vec) {
  const int64_t tiles = tile_count(x.m, x.n, BM, BN);
  if (int rc = check_grid<E>(tiles, kMfmaThreads)) return rc;
  auto* fn = vec ? &gemm_lp_kernel<T, OutT, BM, BN, true, false, E>
                 : &gemm_lp_kernel<T, OutT, BM, BN, false, false, E>;
  fn<<<static_cast<unsigned>(tiles), kMfmaThreads, 0, x.s>>>(
      x.a, x.b, static_cast<OutT*>(x.c), x.m, x.n, x.k, x.alpha, x.beta,
      steps_along(x.m, BM), steps_along(x.n, BN), x.ep);
  MCKE_LAUNCH_CHECK("gemm_lp_kernel");
  return ok();
}

// Short K over many tiles: the product is its C store, and the register-staged kernel's four
// waves share a tile's one stage where the split-K kernel has one wave work and three add
// zeros.  16-byte operands up to 63 of K (fp16 to fp16, 2460 x 1608 x 40: 6.7 us at 64 x 64
// against 9.9 for split K; up to 1024 tiles they tie, fp32 C, 853 x 1880 x 64 5.5 against 5.4),
// others up to 7, as their loads are element by element (fp32 C, 2293 x 1737 x 7: 10.3 against
// 12.8; x 15: 11.6 against 11.7).  128 x 128 tiles where they fill two rounds of CUs or more to 80%
// (2166 x 3544 x 40: 10.9 us against 12.1 at 64 x 64; 2460 x 1608, 260 tiles: 10.3 against 7.6).
template <class E> bool short_k(const LpArgs<E>& x, bool vec) {
  return x.k < (vec ? 64 : 8) && tile_count(x.m, x.n, 32, 64) > 1024;
}

template <typename T, typename OutT, class E>
int launch_short_k(const LpArgs<E>& x, bool vec) {
  const int64_t tiles = tile_count(x.m, x.n, 128, 128), rounds = (tiles + 255) / 256;
  if (rounds >= 2 && 10 * tiles >= 8 * 256 * rounds)
    return launch_staged<T, OutT, 128, 128>(x, vec);
  return launch_staged<T, OutT, 64, 64>(x, vec);
}

// The WHOLE form.
template <typename T, typename OutT, int BM, int BN, int AHEAD = 1, class E>
int launch_whole(const LpArgs<E>& x) {
  const int64_t tiles = tile_count(x.m, x.n, BM, BN);
  if (int rc = check_grid<E>(tiles, kMfmaThreads)) return rc;
  gemm_lp_kernel<T, OutT, BM, BN, false, true, E, AHEAD>
      <<<static_cast<unsigned>(tiles), kMfmaThreads, 0, x.s>>>(
          x.a, x.b, static_cast<OutT*>(x.c), x.m, x.n, x.k, x.alpha, x.beta,
          steps_along(x.m, BM), steps_along(x.n, BN), x.ep);
  MCKE_LAUNCH_CHECK("gemm_lp_kernel");
  return ok();
}

template <typename T, typename OutT, int BM, int BN>
int launch_dma32(const LpArgs<NoEpilogue>& x) {
  constexpr int kStages = 4;
  const int64_t tiles = tile_count(x.m, x.n, BM, BN);
  if (int rc = check_grid<NoEpilogue>(tiles, kMfmaThreads)) return rc;
  gemm_lp_dma_kernel<T, OutT, BM, BN, kStages>
      <<<static_cast<unsigned>(tiles), kMfmaThreads, 0, x.s>>>(
          x.a, x.b, static_cast<OutT*>(x.c), x.m, x.n, x.k, x.alpha, x.beta, x.m / BM, x.n / BN);
  MCKE_LAUNCH_CHECK("gemm_lp_dma_kernel");
  return ok();
}

// The EDGE form at BM x BN, where the shape and the addresses allow it.
template <int BM, int BN, class E> bool edge_fits(const LpArgs<E>& x) {
  return x.n >= BN && x.k >= 64 && x.n % 2 == 0 && x.k % 2 == 0 && aligned(x.a, 4) &&
         aligned(x.b, 4) && aligned(x.c, 4) && dma_offsets32<BM, BN>(x.n, x.k);
}

// The register-staged kernel's WHOLE form at BM x BN, where the shape and the addresses
// allow it.
template <int BM, int BN, typename OutT, class E> bool whole_fits(const LpArgs<E>& x) {
  return x.n >= BN && x.k >= 64 && aligned(x.a, 2) && aligned(x.b, 2) &&
         aligned(x.c, sizeof(OutT));
}

// Odd extents with an epilogue: the register-staged kernel's WHOLE form, with two stages of loads
// in registers at 128 x 128 and 64 x 128.  By tiles of 128 x 128 (t), fp16 to fp32 with GELU and
// residual, us:
//                        t    256   128, 128 one ahead   64 x 128   64    split K 64 x 64
//   4001^3             1024   217   236     240            274     362      374
//   1635 x 12638 x 3991 1287  404   287     304            331     455      487
//   3216 x 3091 x 10672 650   462   350     415            426     568      694
//   2501 x 2501 x 1001  400          41                     48      52       66
//   613 x 5107 x 5864   200   271    78     106             92     114      138
//   1531 x 2053 x 1021  204    86    31      35             28      34       40
//   3001 x 1201 x 901   240    82    29      33             27      31       37
//   1300 x 1901 x 4095  165   208    73      85             73      70       81
//   1200 x 1701 x 513   140    62    20      22             19      15       22
//   900 x 1501 x 4001    96          65                     45      54       56
//   1000 x 1301 x 2001   88          41                     27      31       31
//   300 x 3001 x 2001    72          39                     27      30       24
// A tile of 256 takes as long as 3.7 rounds of 128.  64 x 128 is for one round of its tiles, one to a
// CU, and for up to two a CU (200 .. 256 tiles of 128) below 2048 of K, where 128 x 128 has one tile a
// CU and too few K steps to cover its ends (64 x 128, 128 x 128 and 64 x 64, fp16 to fp32 with GELU and
// residual; bf16 to bf16 within 1 us of it):
//   K                       1021             2047             2049             4095
//   1535 x 1931, t 192   27  29  26       42  43  41       41  40  39       72  69  70
//   1531 x 2053, t 204   28  30  33       42  43  56       41  41  54       73  69 101
//   2047 x 2047, t 256   29  30  33       44  44  55       43  41  53       75  70 101
//   2301 x 2047, t 288   36  40  45       59  61  74       57  59  70      103 104 132
//   the same to bf16     42  41  45       64  62  74       61  59  71      108 104 132
// `rc`: the launch's result, if there is one.
template <typename T, typename OutT, class E> bool launch_odd(const LpArgs<E>& x, int* rc) {
  const int64_t tiles = tile_count(x.m, x.n, 128, 128);
  if (whole_fits<128, 128, OutT>(x)) {
    if (tiles >= 200) {
      const int64_t t256 = tile_count(x.m, x.n, 256, 256);
      const int64_t rounds256 = (t256 + 255) / 256, rounds = (tiles + 255) / 256;
      if (whole_fits<256, 256, OutT>(x) && t256 >= 192 && 37 * rounds256 < 10 * rounds)
        *rc = launch_whole<T, OutT, 256, 256>(x);
      else if (tiles <= 256 && x.k < 2048)
        *rc = launch_whole<T, OutT, 64, 128, 2>(x);
      else
        *rc = launch_whole<T, OutT, 128, 128, 2>(x);
      return true;
    }
    const int64_t halves = tile_count(x.m, x.n, 64, 128);
    if (halves >= 170 && halves <= 256) {
      *rc = launch_whole<T, OutT, 64, 128, 2>(x);
      return true;
    }
  }
  if (whole_fits<64, 64, OutT>(x) && tile_count(x.m, x.n, 64, 64) >= 448) {
    *rc = launch_whole<T, OutT, 64, 64>(x);
    return true;
  }
  return false;
}

// Whether the split-K kernel's limits hold: 16-bit values at 2-byte addresses, per-lane offsets
// below 4 GiB, and a grid that holds 32 x 32 tiles of 512 lanes.
template <typename OutT, class E> bool split_fits(const LpArgs<E>& x) {
  return x.k > 0 && tile_count(x.m, x.n, 32, 32) <= int64_t{UINT32_MAX} / 512 &&
         aligned(x.a, 2) && aligned(x.b, 2) && aligned(x.c, sizeof(OutT)) &&
         static_cast<int64_t>(64) * x.k * 2 < (int64_t{1} << 32) &&
         static_cast<int64_t>(64) * x.n * 2 < (int64_t{1} << 32);
}

template <typename T, typename OutT, int BM, int BN>
struct LpTile {
  // Whole tiles run the requested tile's direct-to-LDS kernel (tiles of 128 and more).
  // Other shapes run its EDGE form, at 128 x 128 from 208 such tiles on, or from 80 on where
  // K is long enough to pay for a tile alone on its CU, and at 256 x 256 where they nearly
  // fill the CUs (fp16 to fp32: 2757 x 432 x 6080, 88 tiles of 128, 49.8 us against 56.9 for
  // split K; 1628 x 800 x 1110, 91 tiles, 15.9 against 15.2; 300 x 520 x 1032, 15 tiles, 14.4
  // against 7.6; 4524 x 344 x 96, 108 tiles, 7.5 against 5.8, to fp16 5.9 against 5.5;
  // 4095 x 4094 x 4090, 256 tiles of 256, 126 us against 206 at 128).  Odd extents run the
  // register-staged kernel's WHOLE form where its 128 x 128 tiles fill most of the CUs (a tile
  // alone on its CU takes 1.3 us per 64 of K, so fewer lose to split K: 1531 x 1021 x 2053, 96
  // tiles, 44.4 us against 29.9; 1700 x 1701 x 1024, 196 tiles, 24.0 against 20.8;
  // 4032 x 843 x 2744, 224 tiles, 54.5 against 63.9; 1901 x 2001 x 511, 240 tiles, 20.4 against
  // 22.1; 3001 x 2501 x 901, 480 tiles, 33.1 against 50.0), at 256 x 256 from 192 such tiles on
  // (4095^3 199 us against 229 at 128 and 406 for split K; 3500 x 3501 x 2001, 196 tiles, 99
  // against 105).  What is left takes the split-K kernel, as 64 x 64 launches do, but for
  // short K over many tiles (short_k).  The tile counts here and below are for 256 CUs.
  template <class E> static int launch(const LpArgs<E>& x, bool vec) {
    if constexpr (E::kFused)
      if (few_rows(x) && split_fits<OutT>(x)) return launch_few_rows<T, OutT>(x);
    if constexpr (BN >= 128) {
      if (vec && x.m % BM == 0 && x.n % BN == 0 && x.k % 64 == 0 && x.k > 0 &&
          dma_offsets32<BM, BN>(x.n, x.k))
        return launch_dma<T, OutT, BM, BN, false>(x);
      // (With an epilogue these take the EDGE form.)
      if constexpr (BM == 128 && !E::kFused)
        if (vec && x.m % BM == 0 && x.n % BN == 0 && x.k % 64 == 32 &&
            tile_count(x.m, x.n, BM, BN) >= 80 && dma_offsets32<BM, BN>(x.n, x.k))
          return launch_dma32<T, OutT, BM, BN>(x);
      if constexpr (BM == 256)
        if (edge_fits<256, 256>(x) && tile_count(x.m, x.n, 256, 256) >= 192)
          return launch_dma<T, OutT, 256, 256, true>(x);
      const int64_t tiles = tile_count(x.m, x.n, 128, 128);
      if (edge_fits<128, 128>(x) &&
          (tiles >= 208 || (tiles >= 80 && x.k >= (sizeof(OutT) == 4 ? 256 : 100))))
        return launch_dma<T, OutT, 128, 128, true>(x);
      if constexpr (E::kFused)
        if (int rc = 0; launch_odd<T, OutT>(x, &rc)) return rc;
      if constexpr (BM == 256 && !E::kFused)
        if (whole_fits<256, 256, OutT>(x) && tile_count(x.m, x.n, 256, 256) >= 192)
          return launch_whole<T, OutT, 256, 256>(x);
      if constexpr (!E::kFused)
        if (whole_fits<128, 128, OutT>(x) && tiles >= 208)
          return launch_whole<T, OutT, 128, 128>(x);
    }
    if (x.n >= 32 && split_fits<OutT>(x))
      return short_k(x, vec) ? launch_short_k<T, OutT>(x, vec) : launch_split<T, OutT>(x);
    // (With an epilogue at most 128 x 128: the checked 256 x 256 form spills as it is.)
    if constexpr (E::kFused && BM == 256) return launch_staged<T, OutT, 128, 128>(x, vec);
    else return launch_staged<T, OutT, BM, BN>(x, vec);
  }
  // The instantiation whole-tile shapes run, for attribute queries.
  static LpKernel kernel() {
    if constexpr (BN >= 128)
      return reinterpret_cast<LpKernel>(&gemm_lp_dma16_kernel<T, OutT, BM, BN, false>);
    else
      return reinterpret_cast<LpKernel>(&gemm_lp_split_kernel<T, OutT, 4, 4, 4>);
  }
};

// Instantiated tiles: (bm, bn) with bk = 64 and 256 lanes, so (tm, tn) = (bm/16, bn/16).
constexpr int kLpTiles[][2] = {{256, 256}, {128, 128}, {64, 64}};

inline int lp_tile_index(const mcke_gemm_tile* t) {
  if (!t) return -1;
  for (int i = 0; i < 3; ++i) {
    const int bm = kLpTiles[i][0], bn = kLpTiles[i][1];
    if (t->bm == bm && t->bn == bn && t->bk == kLpBK && t->tm == bm / 16 && t->tn == bn / 16)
      return i;
  }
  return -1;
}

template <typename T, typename OutT>
struct LpTable {
  template <class E> static int launch(int ti, const LpArgs<E>& x, bool vec) {
    switch (ti) {
      case 0: return LpTile<T, OutT, 256, 256>::launch(x, vec);
      case 1: return LpTile<T, OutT, 128, 128>::launch(x, vec);
      default: return LpTile<T, OutT, 64, 64>::launch(x, vec);
    }
  }
  static LpKernel kernel(int ti) {
    switch (ti) {
      case 0: return LpTile<T, OutT, 256, 256>::kernel();
      case 1: return LpTile<T, OutT, 128, 128>::kernel();
      default: return LpTile<T, OutT, 64, 64>::kernel();
    }
  }
};

// The products with an epilogue, each pair of types in a translation unit with its kernels.
int launch_fused_bf16_f32(int ti, const LpArgs<Epilogue>& x, bool vec);
int launch_fused_bf16_bf16(int ti, const LpArgs<Epilogue>& x, bool vec);
int launch_fused_f16_f32(int ti, const LpArgs<Epilogue>& x, bool vec);
int launch_fused_f16_f16(int ti, const LpArgs<Epilogue>& x, bool vec);

}  // namespace mcke_amd
