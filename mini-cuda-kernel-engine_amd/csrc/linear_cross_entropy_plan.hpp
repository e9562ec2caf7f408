// linear_cross_entropy_plan.hpp -- tiles, pieces of the vocabulary and the workspace of the cross
// entropy of hidden states, by the extents alone, and which memory its products read the weights
// from.  Plain arithmetic: a host program checks every load's bounds with it.
#pragma once

#include <cstdint>

#include "lp_operand.hpp"

namespace mcke_amd {

constexpr int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }
constexpr int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

constexpr int64_t kPieceAlign = 256;
constexpr int64_t kPieceValues = int64_t{1} << 26;     // of dz, and of a padded piece of W

enum class Tile { k64x128, k128, k256 };

// 256 x 256 where such tiles are most of the CUs' or more; 64 rows at 64 x 128.  Not for products of
// up to 128 of K, most of which is the tile's epilogue: two workgroups a CU overlap theirs (gradients
// of 7424 x 33536 x 64 573 -> 529 us, 4096 x 32768 x 128 284 -> 276, x 192 321 -> 325).
constexpr Tile tile_of(int64_t rows, int64_t cols, int64_t dim) {
  if (rows <= 64) return Tile::k64x128;
  if (rows > 128 && dim > 128 && ceil_div(rows, 256) * ceil_div(cols, 256) >= 192) return Tile::k256;
  return Tile::k128;
}
constexpr int tile_rows(Tile t) { return t == Tile::k64x128 ? 64 : t == Tile::k128 ? 128 : 256; }
constexpr int tile_cols(Tile t) { return t == Tile::k256 ? 256 : 128; }

// Workgroups of a launch: 256 lanes each of the grid's 32-bit work size.
constexpr int64_t kMostTiles = INT32_MAX / 256;

// A piece of the weights: `rows` rows from `first` on, `row` values apart.  Rows from tail_first
// on (a multiple of 256) are at `tail` too, as far apart, with zeros behind the last up to a
// multiple of 64 rows and 64 values more (null: none are).
struct Piece {
  const uint16_t* p;
  int64_t row, rows, first;
  const uint16_t* tail;
  int64_t tail_first;

  // Of a tile of logits from column n0 on: the weights' rows along K.
  constexpr LpOperand of_logits(int64_t n0) const {
    return {tail && first + n0 >= tail_first ? tail - (tail_first - first) * row : p, row, rows};
  }
  // Of dH: the weights' rows are K.  The last stage ends behind the weights, which is not the
  // caller's to read (dz has zeros there), and 16-byte loads of narrow rows in the stage before it
  // may: stages of the tail are all its copy's.
  constexpr LpOperand of_dh() const {
    return {p, row, row, tail, tail ? (tail_first - first) / kStageK : INT64_MAX};
  }
};

struct Plan {
  int64_t rows, vocab, dim;
  int64_t width;             // dim, a multiple of 64
  int64_t up;                // rows, a multiple of 64
  bool pad;                  // the weights need a padded copy, a piece at a time
  int64_t tail_first, tail_values;   // or one of their last rows and zeros behind them (0: none)
  int64_t piece, pieces;     // rows of W at once
  Tile tile;                 // of the logits
  int64_t at;                // bytes of workspace so far

  Plan(int64_t r, int64_t v, int64_t d, bool backward) : rows(r), vocab(v), dim(d), at(0) {
    width = round_up(d, 64);
    up = round_up(r, 64);
    pad = d % 2 != 0;
    // Whole tiles before it read up to 63 values past their last row, which the matrix has to hold.
    tail_first = (v - 1) / kPieceAlign * kPieceAlign;
    if (tail_first > 0 && (v - tail_first) * d < 64) tail_first -= kPieceAlign;
    tail_values = pad || (d % 64 == 0 && (!backward || v % 64 == 0))
                      ? 0
                      : (round_up(v, 64) - tail_first) * d + 64;
    int64_t most = round_up(v, kPieceAlign);
    auto limit = [&](int64_t per_row) {
      int64_t m = kPieceValues / per_row / kPieceAlign * kPieceAlign;
      if (m < kPieceAlign) m = kPieceAlign;
      if (m < most) most = m;
    };
    if (backward) limit(up);
    if (pad) limit(width);
    piece = round_up(ceil_div(v, ceil_div(v, most)), kPieceAlign);
    pieces = ceil_div(v, piece);
    // Tiles that are too many for a launch are larger instead (the backward pass's pieces never are).
    tile = tile_of(r, backward ? at_once() : v, d);
    if (!fits()) tile = Tile::k256;
  }
  int64_t at_once() const { return piece < vocab ? piece : vocab; }
  bool fits() const { return logits_tiles(at_once()) <= kMostTiles; }
  // Piece i of `weight`, with `copy` where the tail's copy or the piece's padded one is.
  Piece piece_of(int64_t i, const uint16_t* weight, const uint16_t* copy) const {
    const int64_t first = i * piece, n = vocab - first < piece ? vocab - first : piece;
    if (pad) return {copy, width, n, first, nullptr, 0};
    return {weight + first * dim, dim, n, first, tail_values ? copy : nullptr, tail_first};
  }
  // Tiles of logits over `n` rows of the weights.
  int64_t logits_tiles(int64_t n) const {
    return ceil_div(rows, tile_rows(tile)) * ceil_div(n, tile_cols(tile));
  }
  int64_t take(int64_t bytes) {
    const int64_t from = at;
    at += round_up(bytes, 256);
    return from;
  }
};

}  // namespace mcke_amd
