// gemm_lp_any.hpp -- the main loop of a 16-bit product whose operands lie either way:
//
//   acc[m][n] += sum over k of A(m, k) B(k, n),   bf16 or fp16, fp32 accumulation
//
// each operand with its k contiguous (kAlongK: rows of A[m][k], of B[n][k], as a layer's weights
// [out][in] and activations are) or with its other index contiguous (kAcrossK: A[k][m],
// B[k][n]).  The products of a layer and its gradients, y = x W^T, dx = dy W and dW = dy^T x, are one of
// these each, with no transposed copy: those of the cross entropy of hidden states are made so.
//
// A workgroup of four waves (2 x 2) owns BM x BN, a wave MT x NT blocks of 16 x 16
// (v_mfma_f32_16x16x32).  K goes in stages of 64 (two steps of 32), each operand's stage straight
// from memory into LDS (global_load_lds_dwordx4):
//   kAlongK   rows of 128 bytes, 16-byte chunk c of row r at c ^ (r % 8); a fragment is one
//             ds_read_b128;
//   kAcrossK  64 rows (one k each) of 2 BM or 2 BN bytes, chunk c of row k at
//             c ^ (4 (k % 4) + 2 ((k / 8) % 2)); a fragment is two ds_read_b64_tr_b16.
// Neither read meets a bank twice.  With D stages in flight A has D + 1 stage buffers and B has D:
// 160 KB at 256 x 256 and D = 2.
//
// Stage p is two steps; a step computes on fragments read in the step before it:
//   step 2 p      MFMAs of k half 0; reads of half 1; DMA of A stage p + D
//   step 2 p + 1  wait for A and B of stage p + 1, barrier; MFMAs of half 1; reads of
//                 half 0 of stage p + 1; DMA of B stage p + D into the buffer of stage p
// so a stage has D to D + 1 steps or more to land, and there is one barrier per 64 of K.  Each
// wave waits for its own reads before that barrier, which makes every buffer of stage p free
// behind it.  D is 2 where two workgroups share a CU or one fills it; small tiles that are alone on
// their CU take as many as fit, or every stage waits for memory.
// Past the end the DMA repeats the last stage into buffers that nobody reads, which keeps the
// count of loads in flight the same in every step.
//
// K is a multiple of 64 here.  Rows past an operand's end along M and N repeat its last row and are
// not to be stored.  16-byte loads may begin inside a row and end behind it, in the next one: what
// lies there has to be multiplied by zeros of the other operand (along K), or not stored (along N).
// Where that leaves the operand, or K ends inside a stage of a kAcrossK operand, the caller has a copy of
// the last rows with zeros behind them (`tail`, or the operand itself).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <utility>

#include "gemm_lp.hpp"
#include "lp_operand.hpp"

namespace mcke_amd {

enum class Along { kAlongK, kAcrossK };

template <int B, Along L> struct LpAnyOperand {
  static constexpr bool kAcross = L == Along::kAcrossK;
  static constexpr int kBuf = B * 128;               // one stage, either way: B x 64 values
  static constexpr int kDma = kBuf / 1024 / 4;       // DMA instructions per wave and stage
  static constexpr int kBlocks = B / 32;             // 16-wide blocks of a wave
  static constexpr int kRow = kAcross ? 2 * B : 128; // an LDS row
  static constexpr int kLanes = kRow / 16;           // lanes a row of a DMA instruction
  static constexpr int kReads = kBlocks * (kAcross ? 2 : 1);
  static_assert(kLanes <= 32 && (!kAcross || B >= 128), "the swizzle takes 16 chunks a row");
  static __host__ __device__ constexpr int swz(int r) {
    return kAcross ? 4 * (r % 4) + 2 * ((r / 8) % 2) : r % 8;
  }

  // A lane's sources, relative to the stage's uniform base.
  const char* base;                                  // of stage 0
  LpOperand operand;                                 // (kAcrossK)
  uint32_t src[kDma];
  uint32_t off[2];                                   // fragment addresses in a buffer

  // A DMA instruction's immediate offset (1 KB times its index, modulo four) moves its source too:
  // the offsets have it taken off, and are kept positive by 3 KB that the base gives back.
  static constexpr uint32_t kBias = 3 * 1024;

  // The workgroup's rows or columns begin at `first`, the wave's at `wave_first` of them.
  __device__ __forceinline__ void begin(const LpOperand& o, int64_t first, int wave_first,
                                        int wave) {
    const int lane = threadIdx.x % kWave, g = lane / 16, r16 = lane % 16;
    if constexpr (!kAcross) {
      base = reinterpret_cast<const char*>(o.p + first * o.row) - kBias;
      const int64_t last = o.extent - 1 - first;
#pragma unroll
      for (int q = 0; q < kDma; ++q) {
        const int rt = 8 * (wave * kDma + q) + lane / 8;
        const int c = (lane % 8) ^ swz(rt);
        src[q] = static_cast<uint32_t>(2 * lp_along_load(rt, c, o.row, last)) + kBias -
                 1024u * (q % 4);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
        off[s] = (wave_first + r16) * kRow + 16 * ((4 * s + g) ^ (r16 % 8));
    } else {
      operand = o;
#pragma unroll
      for (int q = 0; q < kDma; ++q) {
        const int rt = (64 / kLanes) * (wave * kDma + q) + lane / kLanes;
        const int64_t col = first + 8 * ((lane % kLanes) ^ swz(rt));
        src[q] = static_cast<uint32_t>(2 * lp_across_load(rt, col, o.row, o.extent)) + kBias -
                 1024u * (q % 4);
      }
      // Lane r16 = 4 jq + qa of group g reads row 8 g + 4 t + jq at columns 4 qa of its block and
      // receives column r16 of rows 8 g + 4 t .. + 3.
      // Block b's chunks differ from block 0's in bits that the wave's first chunk does not have,
      // and buffers begin at multiples of 1 KB: the blocks' addresses are one, xor 32 b.
      const int jq = r16 / 4, qa = r16 % 4, k = 8 * g + jq, col = wave_first + 4 * qa;
      off[0] = k * kRow + 16 * ((col / 8) ^ swz(k)) + (col % 8) * 2;
    }
  }

  // Instruction Q of stage p, whose uniform source is `from`, into the buffer at LDS `buf`.
  template <int Q>
  __device__ __forceinline__ void dma(const char* from, uint32_t buf, uint32_t wave) const {
    lds_dma16<(Q % 4) * 1024>(src[Q], from, buf + (wave * kDma + Q / 4 * 4) * 1024);
  }
  __device__ __forceinline__ const char* source(int64_t p) const {
    if constexpr (kAcross) return reinterpret_cast<const char*>(operand.stage(p)) - kBias;
    else return base + p * (2 * kStageK);
  }

  struct Frags {
    u32x4 whole[kAcross ? 1 : kBlocks];
    u32x2 half[kAcross ? kBlocks : 1][2];
  };
  // Read RR of half S of the stage at LDS `buf`.
  template <int S, int RR> __device__ __forceinline__ void read(uint32_t buf, Frags& f) const {
    if constexpr (kAcross)
      f.half[RR / 2][RR % 2] =
          lds_read_tr16<(32 * S + 4 * (RR % 2)) * kRow>((buf + off[0]) ^ (32 * (RR / 2)));
    else
      f.whole[RR] = lds_read128<RR * 16 * kRow>(buf + off[S]);
  }
  template <int I> static __device__ __forceinline__ void touch(Frags& f) {
    if constexpr (kAcross) {
      asm volatile("" : "+v"(f.half[I][0]));
      asm volatile("" : "+v"(f.half[I][1]));
    } else {
      asm volatile("" : "+v"(f.whole[I]));
    }
  }
  static __device__ __forceinline__ u32x4 get(const Frags& f, int i) {
    if constexpr (kAcross)
      return u32x4{f.half[i][0][0], f.half[i][0][1], f.half[i][1][0], f.half[i][1][1]};
    else
      return f.whole[i];
  }
};

template <int BM, int BN, Along LA, Along LB, int D = 2> struct LpAnyShape {
  using OA = LpAnyOperand<BM, LA>;
  using OB = LpAnyOperand<BN, LB>;
  static constexpr int kDepth = D, kABufs = D + 1, kBBufs = D;
  static_assert(D >= 2 && D * (OA::kDma + OB::kDma) + OA::kDma <= 63, "vmcnt counts to 63");
  static constexpr int kBBase = kABufs * OA::kBuf;
  static constexpr int kLdsBytes = kBBase + kBBufs * OB::kBuf;
  static constexpr int MT = BM / 32, NT = BN / 32;
  static constexpr int kMfmas = MT * NT;
  static constexpr int kReads = OB::kReads + OA::kReads;       // B's blocks first, then A's
  // Reads in the first three quarters of a step, so that those of step 2 p have come back at the
  // barrier behind it.
  static constexpr int read_slot(int rr) { return rr * (3 * kMfmas) / (4 * kReads); }
  static constexpr int dma_slot(int ii, int n) { return ii * kMfmas / n + (kMfmas / n) / 2; }
  static_assert(kLdsBytes <= 160 * 1024, "LDS holds 160 KiB");
  // Block row i of an even step waits for B's reads and A block i's, issued in the step before; A
  // reads behind them and this step's so far may be outstanding (lgkmcnt counts to 15).
  static constexpr int wait_before_row(int i) {
    int n = (OA::kReads / MT) * (MT - 1 - i);
    for (int rr = 0; rr < kReads; ++rr) n += read_slot(rr) < i * NT ? 1 : 0;
    return n < 15 ? n : 15;
  }
};

// What a step needs besides the fragments.
struct LpAnyStep {
  uint32_t a_read, b_read;       // LDS buffers that are read
  uint32_t dma_buf;              // LDS buffer that is filled
  const char* dma_from;
};

// MFMA IDX of a step, on the fragments cur, with the reads (of half RS, into next) and the DMA
// (of A or of B) that go out behind it.  The product is transposed: a lane holds four
// neighbouring columns of a row.
template <typename T, class S, int PARITY, int IDX>
__device__ __forceinline__ void lp_any_slot(
    f32x4 (&acc)[S::MT][S::NT], typename S::OA::Frags& ca, typename S::OB::Frags& cb,
    typename S::OA::Frags& na, typename S::OB::Frags& nb, const typename S::OA& oa,
    const typename S::OB& ob, const LpAnyStep& sp, uint32_t wave) {
  constexpr int NT = S::NT, RS = 1 - PARITY;
  constexpr int i = IDX / NT, jj = IDX % NT, j = mfma_snake_col(i, jj, NT);
  if constexpr (jj == 0) {
    if constexpr (PARITY == 0) lds_wait_n<S::wait_before_row(i)>();
    S::OA::template touch<i>(ca);
    if constexpr (i == 0) {
      [&]<int... J>(std::integer_sequence<int, J...>) {
        (S::OB::template touch<J>(cb), ...);
      }(std::make_integer_sequence<int, NT>{});
    }
  }
  acc[i][j] = LpMfma16<T>::run(S::OB::get(cb, j), S::OA::get(ca, i), acc[i][j]);
  __builtin_amdgcn_sched_barrier(0);
  [&]<int... RR>(std::integer_sequence<int, RR...>) {
    ([&] {
      if constexpr (S::read_slot(RR) == IDX) {
        if constexpr (RR < S::OB::kReads) ob.template read<RS, RR>(sp.b_read, nb);
        else oa.template read<RS, RR - S::OB::kReads>(sp.a_read, na);
      }
    }(), ...);
  }(std::make_integer_sequence<int, S::kReads>{});
  if constexpr (PARITY == 0) {
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      ([&] {
        if constexpr (S::dma_slot(Q, S::OA::kDma) == IDX)
          oa.template dma<Q>(sp.dma_from, sp.dma_buf, wave);
      }(), ...);
    }(std::make_integer_sequence<int, S::OA::kDma>{});
  } else {
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      ([&] {
        if constexpr (S::dma_slot(Q, S::OB::kDma) == IDX)
          ob.template dma<Q>(sp.dma_from, sp.dma_buf, wave);
      }(), ...);
    }(std::make_integer_sequence<int, S::OB::kDma>{});
  }
  __builtin_amdgcn_sched_barrier(0);
}

// The products of stages first .. first + stages - 1 (stages >= 1) of the tile at (m0, n0) into
// acc, from zero.  `smem`: S::kLdsBytes, 1024-byte aligned; free behind the caller's next barrier.
// Lane (g, r16), register e of block (i, j): row wm BM/2 + 16 i + r16, column
// wn BN/2 + 16 j + 4 g + e of the tile.
template <typename T, int BM, int BN, Along LA, Along LB, int D = 2>
__device__ __forceinline__ void lp_any_loop(f32x4 (&acc)[BM / 32][BN / 32], char* smem,
                                            const LpOperand& A, const LpOperand& B, int64_t m0,
                                            int64_t n0, int64_t first, int stages) {
  using S = LpAnyShape<BM, BN, LA, LB, D>;
  constexpr int MT = S::MT, NT = S::NT;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / 2, wn = wave % 2;
  typename S::OA oa;
  typename S::OB ob;
  oa.begin(A, m0, wm * (BM / 2), wave);
  ob.begin(B, n0, wn * (BN / 2), wave);
  const uint32_t lds0 = lds_addr(smem), ldsb = lds0 + S::kBBase;
  const uint32_t w = static_cast<uint32_t>(wave);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // The accumulators are in the accumulation registers from here on: left to itself the compiler
  // keeps some elsewhere and moves them back and forth in every stage.
  auto pin = [&] {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) asm volatile("" : "+a"(acc[i][j]));
  };
  pin();

  auto stage = [&](int p) { return first + (p < stages ? p : stages - 1); };
  auto dma_a = [&](int p, uint32_t buf) {
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      (oa.template dma<Q>(oa.source(stage(p)), buf, w), ...);
    }(std::make_integer_sequence<int, S::OA::kDma>{});
  };
  auto dma_b = [&](int p, uint32_t buf) {
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      (ob.template dma<Q>(ob.source(stage(p)), buf, w), ...);
    }(std::make_integer_sequence<int, S::OB::kDma>{});
  };
#pragma unroll
  for (int p = 0; p < D; ++p) {
    dma_a(p, lds0 + p * S::OA::kBuf);
    dma_b(p, ldsb + p * S::OB::kBuf);
  }
  // Stage 0 is there, the others may be on their way.
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"((D - 1) * (S::OA::kDma + S::OB::kDma)) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  typename S::OA::Frags fa[2];
  typename S::OB::Frags fb[2];
  [&]<int... RR>(std::integer_sequence<int, RR...>) {
    (ob.template read<0, RR>(ldsb, fb[0]), ...);
  }(std::make_integer_sequence<int, S::OB::kReads>{});
  [&]<int... RR>(std::integer_sequence<int, RR...>) {
    (oa.template read<0, RR>(lds0, fa[0]), ...);
  }(std::make_integer_sequence<int, S::OA::kReads>{});

  // Buffers of stage p, and A's of stage p + D.
  uint32_t abuf = 0, bbuf = 0, afill = D;
  for (int p = 0; p < stages; ++p) {
    const uint32_t a1 = abuf == D ? 0 : abuf + 1, b1 = bbuf == D - 1 ? 0 : bbuf + 1;
    const uint32_t bcur = ldsb + bbuf * S::OB::kBuf, bnext = ldsb + b1 * S::OB::kBuf;
    const LpAnyStep even{lds0 + abuf * S::OA::kBuf, bcur, lds0 + afill * S::OA::kBuf,
                         oa.source(stage(p + D))};
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (lp_any_slot<T, S, 0, I>(acc, fa[0], fb[0], fa[1], fb[1], oa, ob, even, w),
       ...);
    }(std::make_integer_sequence<int, S::kMfmas>{});
    // Of the loads in flight those of stages from p + 2 on may be outstanding, and none of this
    // wave's reads.  A bare s_barrier: __syncthreads() would wait for all loads.
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((D - 2) * (S::OA::kDma + S::OB::kDma) +
                                                       S::OA::kDma)
                 : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const LpAnyStep odd{lds0 + a1 * S::OA::kBuf, bnext, bcur, ob.source(stage(p + D))};
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (lp_any_slot<T, S, 1, I>(acc, fa[1], fb[1], fa[0], fb[0], oa, ob, odd, w),
       ...);
    }(std::make_integer_sequence<int, S::kMfmas>{});
    afill = abuf;              // free behind the barrier
    abuf = a1;
    bbuf = b1;
    pin();
  }
  // The last stage's reads of the next one go unused, but they land in these registers: named
  // behind the wait, those hold nothing else before it.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  [&]<int... I>(std::integer_sequence<int, I...>) {
    (S::OA::template touch<I>(fa[0]), ...);
  }(std::make_integer_sequence<int, MT>{});
  [&]<int... I>(std::integer_sequence<int, I...>) {
    (S::OB::template touch<I>(fb[0]), ...);
  }(std::make_integer_sequence<int, NT>{});
  // They are read by acc_get, inline asm that the hazard checks do not see into: 16 cycles for the
  // last MFMA's results.
  pin();
  asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");
}

// The same for one stage, which nothing overlaps with: a third of the LDS, so that more
// workgroups share a CU.  `smem`: kLdsOne bytes.
template <int BM, int BN> constexpr int kLdsOne = (BM + BN) * 128;

template <typename T, int BM, int BN, Along LA, Along LB>
__device__ __forceinline__ void lp_any_one(f32x4 (&acc)[BM / 32][BN / 32], char* smem,
                                           const LpOperand& A, const LpOperand& B, int64_t m0,
                                           int64_t n0) {
  using OA = LpAnyOperand<BM, LA>;
  using OB = LpAnyOperand<BN, LB>;
  constexpr int MT = BM / 32, NT = BN / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  OA oa;
  OB ob;
  oa.begin(A, m0, wave / 2 * (BM / 2), wave);
  ob.begin(B, n0, wave % 2 * (BN / 2), wave);
  const uint32_t lds_a = lds_addr(smem), lds_b = lds_a + OA::kBuf;
  [&]<int... Q>(std::integer_sequence<int, Q...>) {
    (oa.template dma<Q>(oa.source(0), lds_a, wave), ...);
  }(std::make_integer_sequence<int, OA::kDma>{});
  [&]<int... Q>(std::integer_sequence<int, Q...>) {
    (ob.template dma<Q>(ob.source(0), lds_b, wave), ...);
  }(std::make_integer_sequence<int, OB::kDma>{});
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      asm volatile("" : "+a"(acc[i][j]));
    }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  typename OA::Frags fa;
  typename OB::Frags fb;
  auto half = [&]<int H>() {
    [&]<int... RR>(std::integer_sequence<int, RR...>) {
      (ob.template read<H, RR>(lds_b, fb), ...);
    }(std::make_integer_sequence<int, OB::kReads>{});
    [&]<int... RR>(std::integer_sequence<int, RR...>) {
      (oa.template read<H, RR>(lds_a, fa), ...);
    }(std::make_integer_sequence<int, OA::kReads>{});
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (OA::template touch<I>(fa), ...);
    }(std::make_integer_sequence<int, MT>{});
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (OB::template touch<I>(fb), ...);
    }(std::make_integer_sequence<int, NT>{});
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        acc[i][j] = LpMfma16<T>::run(OB::get(fb, j), OA::get(fa, i), acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  half.template operator()<0>();
  half.template operator()<1>();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+a"(acc[i][j]));
  asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");
}

}  // namespace mcke_amd
