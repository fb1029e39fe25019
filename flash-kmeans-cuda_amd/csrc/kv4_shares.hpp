// Weights by which the 4-bit cache's attention is cut into equal shares; plain
// arithmetic, the same on the device, for the launch's checks and in tests.
#pragma once

#include <cstdint>

namespace fkc {

// Granules that an item costs by itself (us with 2 / 3 / 5 / 8: 64 ragged requests
// 142 / 132 / 134 / 137, drafted tokens 38.9 / 38.5 / 40.4 / 44.1, prompts 399 /
// 397 / 408 / 430).
constexpr int kItem = 3;

// Granules of a tile that sees nothing, or hardly anything (us with 1 / 2 / 4: a
// prompt of 2048 in a step padded to 4096 rows 125 / 107 / 114, to 16384 171 / 147 /
// 186, one of 700 padded to 8192 54 / 60 / 80).
constexpr int kIdle = 2;

// Weight of the first j tiles of `cols` columns of a request with nq queries of
// G columns each over `end` tokens, in granules of gr tokens.
//
// Tile j of a causal request sees about A + (j + 1) cols / G tokens, A those in
// front of its queries; of one with more queries than tokens (rows of no request
// have none) the first `idle` tiles see nothing, or part of a tile's first tokens.
constexpr int kv4_weight(int cols, int gr, int G, bool causal, int nq, int end, int j) {
  const int own = (causal ? (end > nq ? end - nq : 0) : end) / gr + 1 + kItem;
  const uint32_t blind = nq > end ? (uint32_t)(nq - end) * (uint32_t)G : 0;  // columns
  const int idle = (int)((blind + (uint32_t)cols - 1) / (uint32_t)cols);
  const int k = end == 0 || (causal && j < idle) ? 0 : causal ? j - idle : j;
  const int sum = (j - k) * kIdle + k * own;
  if (!causal || k <= 1) return sum;
  return sum + (int)((int64_t)cols * k * (k + 1) / 2 / (G * gr));
}

// What j tiles of a request of up to max_seq tokens weigh at most, per tile: k of
// them see something, cols * k < G * min(nq, end) + 2 * cols, so
//   cols (k + 1) / (2 G gr) < min(nq, end) / (2 gr) + 3 cols / (2 G gr).
constexpr int64_t kv4_most_weight(int cols, int gr, int G, int64_t max_seq) {
  return max_seq / gr + 2 * cols / ((int64_t)G * gr) + 3 + kItem;
}

}  // namespace fkc
