// How the backward pass of a loss at the vocabulary head cuts the vocabulary into pieces, and a piece's sums for dbias into
// parts.  The numbers that the workspace is laid out by are the ones that the launches take.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace ixk {
namespace head {

constexpr size_t kPieceBytes = size_t(256) << 20;  // of the logits' gradient
// Columns that a piece of the gradient had best be a multiple of.
constexpr int kPieceUnit = 256;

// dbias: columns of a CTA; warps that take its rows in turn; parts at most.
constexpr int kBiasCols = 256, kBiasGroups = 32, kBiasParts = 32;

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Pieces {
  int64_t vocab, columns, count;   // count pieces of `columns` columns, the last one what is left
  int64_t bias_parts;              // CTAs along the rows for the sums of a piece's columns, of every piece
  int64_t columns_of(int64_t first) const { return std::min(columns, vocab - first); }
  // fp32 partial sums of dbias: [bias_parts][the piece's columns]
  int64_t bias_partials() const { return bias_parts * columns; }
};

// Pieces of equal size, as few as the bytes allow.  Sums of a piece's columns: as many parts as give the SMs one CTA each, with
// four rows a warp or more; the last piece, which may be shorter, takes no more of them than there is room for.
inline Pieces pieces_for(int64_t rows, int64_t vocab) {
  Pieces p{};
  const int64_t padded = round_up(rows, 256);
  const int64_t most = std::max<int64_t>(static_cast<int64_t>(kPieceBytes) / (2 * padded) / kPieceUnit * kPieceUnit, kPieceUnit);
  p.vocab = vocab;
  p.count = (vocab + most - 1) / most;
  p.columns = std::min(round_up((vocab + p.count - 1) / p.count, kPieceUnit), round_up(vocab, 8));
  p.count = (vocab + p.columns - 1) / p.columns;
  const int64_t blocks = (std::min(p.columns, vocab) + kBiasCols - 1) / kBiasCols;
  p.bias_parts = std::clamp<int64_t>(std::min<int64_t>(148 / blocks, rows / (4 * kBiasGroups)), 1, kBiasParts);
  return p;
}

}  // namespace head
}  // namespace ixk
