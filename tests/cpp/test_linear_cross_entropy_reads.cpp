// Every 16-byte load of the weights that the products of the cross entropy of hidden states make,
// by the kernels' own arithmetic, against the matrix and the copy that it may read: no load begins
// before either or ends behind it, in either pass, at every width and vocabulary where the last
// rows are narrow.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "../../mini-cuda-kernel-engine_amd/csrc/linear_cross_entropy_plan.hpp"

using namespace mcke_amd;

namespace {

const std::uintptr_t kWeight = std::uintptr_t{1} << 40, kCopy = std::uintptr_t{1} << 44;
long g_loads = 0, g_failures = 0;

struct Memory {
  std::uintptr_t weight_end, copy_end;
  Memory(const Plan& p)
      : weight_end(kWeight + 2 * static_cast<std::uintptr_t>(p.vocab * p.dim)),
        copy_end(kCopy + 2 * static_cast<std::uintptr_t>(p.pad ? p.piece * p.width : p.tail_values)) {}
  void load(const uint16_t* from, int64_t values, const Plan& p, const char* what) const {
    const std::uintptr_t a = reinterpret_cast<std::uintptr_t>(from) + 2 * values, b = a + 16;
    ++g_loads;
    if ((a >= kWeight && b <= weight_end) || (a >= kCopy && b <= copy_end)) return;
    if (++g_failures <= 20)
      std::printf("FAIL %s: %lld x %lld x %lld reads %lld bytes past its end\n", what,
                  static_cast<long long>(p.rows), static_cast<long long>(p.vocab),
                  static_cast<long long>(p.dim),
                  static_cast<long long>(a < kCopy ? b - weight_end : b - copy_end));
  }
};

void scan(int64_t rows, int64_t vocab, int64_t dim, bool backward) {
  const Plan p(rows, vocab, dim, backward);
  const Memory mem(p);
  const auto* weight = reinterpret_cast<const uint16_t*>(kWeight);
  const auto* copy = reinterpret_cast<const uint16_t*>(kCopy);
  for (int64_t i = 0; i < p.pieces; ++i) {
    const Piece w = p.piece_of(i, weight, copy);
    // Logits: tiles of BN rows, all of the width along K.
    const int bn = tile_cols(p.tile);
    for (int64_t n0 = 0; n0 < w.rows; n0 += bn) {
      const LpOperand o = w.of_logits(n0);
      for (int64_t k = 0; k < p.width; k += kStageK)
        for (int rt = 0; rt < bn; ++rt)
          for (int c = 0; c < kStageK / 8; ++c)
            mem.load(o.p, n0 * o.row + k + lp_along_load(rt, c, o.row, o.extent - 1 - n0), p,
                     "logits");
    }
    if (!backward) continue;
    // dH: stages of 64 rows, all columns of whole tiles of the widest kind.
    const LpOperand o = w.of_dh();
    for (int64_t s = 0; s < ceil_div(w.rows, kStageK); ++s)
      for (int rt = 0; rt < kStageK; ++rt)
        for (int64_t col = 0; col < round_up(dim, 256); col += 8)
          mem.load(o.stage(s), lp_across_load(rt, col, o.row, o.extent), p, "dH");
  }
}

}  // namespace

int main() {
  for (int64_t dim = 1; dim <= 130; ++dim)
    for (int64_t vocab = 1; vocab <= 330; ++vocab) {
      scan(1, vocab, dim, false);
      scan(1, vocab, dim, true);
      if (vocab % 64 < 5) scan(300, vocab, dim, true);
    }
  // In pieces, the last one short.
  for (int64_t dim : {1, 2, 4, 6, 63, 66, 192, 1026})
    for (int64_t vocab : {5376, 5377, 7001, 10752, 10753, 10754, 10817, 10818})
      for (bool backward : {false, true}) scan(12300, vocab, dim, backward);
  // Pieces of 256, the last one of so few rows that the copy begins a piece before it.
  for (int64_t dim : {2, 4, 6, 8, 30, 62, 130})
    for (int64_t vocab = 510; vocab <= 580; ++vocab) scan(131100, vocab, dim, true);
  std::printf("%ld loads, %ld failures\n", g_loads, g_failures);
  return g_failures ? 1 : 0;
}
