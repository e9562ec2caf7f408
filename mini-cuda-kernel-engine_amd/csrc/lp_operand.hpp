// lp_operand.hpp -- where the 16-byte loads of an operand of gemm_lp_any.hpp begin.  Plain
// arithmetic, the same for a kernel and for a host program that looks at every load's bounds.
#pragma once

#include <cstdint>

namespace mcke_amd {

constexpr int kStageK = 64;       // of K in a stage

// An operand's memory, 4-byte aligned, `row` elements (an even number) between neighbouring rows.
// `extent`: its rows (kAlongK), or how many elements a row has (kAcrossK).
struct LpOperand {
  const uint16_t* p;
  int64_t row;
  int64_t extent;
  // kAcrossK: stages from tail_stage on (it may be below 0) are at `tail`, which begins with that
  // stage, instead (null: none).
  const uint16_t* tail = nullptr;
  int64_t tail_stage = INT64_MAX;

  // kAcrossK: the first value of stage p.
  constexpr const uint16_t* stage(int64_t p) const {
    return tail && p >= tail_stage ? tail + (p - tail_stage) * kStageK * row
                                   : this->p + p * kStageK * row;
  }
};

// The load of eight values at row rt, column `col` of a kAcrossK stage, in values from the stage's
// first: columns past the row's end repeat its first.
constexpr int64_t lp_across_load(int64_t rt, int64_t col, int64_t row, int64_t extent) {
  return rt * row + (col < extent ? col : 0);
}
// The load at tile row rt, chunk c of a kAlongK stage, in values from the tile's first row at the
// stage's K: rows past `last` repeat it.
constexpr int64_t lp_along_load(int64_t rt, int c, int64_t row, int64_t last) {
  return (rt < last ? rt : last) * row + 8 * c;
}

}  // namespace mcke_amd
