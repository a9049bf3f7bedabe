// Sizes and the workspace of the embedding's gradient, shared by the launchers and
// the host checks.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace mf {

constexpr int kEmbedMostTokens = 1 << 24;
constexpr int kEmbedMostVocabulary = 1 << 27;
constexpr int kEmbedMostDim = 1 << 16;
constexpr long long kEmbedMostValues = 1ll << 34;  // of the output: launches stay below 2^32 threads

constexpr int kSortDigit = 9;               // bits of a key in one pass
constexpr int kSortBins = 1 << kSortDigit;
constexpr int kSortTiles = 128;             // waves that share the tokens, at most
constexpr int kEmbedChunk = 32;             // sorted tokens that a wave adds

// A token and the row of the table that it adds to (the vocabulary: none).
struct SortedToken {
  uint32_t key, token;
};

struct EmbedLayout {
  int passes, bits;    // of the sort: digits and their bits
  int tiles, rounds;   // waves, and the 64 tokens each that they take in turn
  int chunks;
  size_t histogram, tokens[2], partials, total;  // offsets in bytes
};

inline EmbedLayout embed_layout(int tokens, int vocabulary, int dim) {
  EmbedLayout l;
  int bits = 1;
  while (bits < 31 && vocabulary >> bits) ++bits;  // of the key `vocabulary`
  l.passes = (bits + kSortDigit - 1) / kSortDigit;
  l.bits = (bits + l.passes - 1) / l.passes;
  const int waves = (tokens + 63) / 64;
  l.rounds = (waves + kSortTiles - 1) / kSortTiles;
  if (l.rounds < 4) l.rounds = 4;
  l.tiles = (waves + l.rounds - 1) / l.rounds;
  l.chunks = (tokens + kEmbedChunk - 1) / kEmbedChunk;
  auto align = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t at = 0;
  l.histogram = at;
  at += align(sizeof(int) * (size_t)l.tiles * kSortBins);
  for (int i = 0; i < 2; ++i) {
    l.tokens[i] = at;
    at += align(sizeof(SortedToken) * (size_t)tokens);
  }
  l.partials = at;
  at += align(sizeof(float) * 2 * (size_t)l.chunks * dim);
  l.total = at;
  return l;
}

}  // namespace mf
