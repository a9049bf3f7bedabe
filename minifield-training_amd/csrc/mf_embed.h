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
constexpr int kSortFewest = 5;              // (kernels are made for 5 to 9)
constexpr int kSortBins = 1 << kSortDigit;
constexpr int kSortTiles = 64;              // workgroups that share the tokens, at most
constexpr int kSortWaves = 8;               // of each
constexpr int kSortRuns = 2;                // runs of 64 tokens that a wave takes in a step
constexpr int kSortStep = kSortWaves * kSortRuns * 64;
static_assert(kSortBins == kSortWaves * 64, "a thread for each digit");
constexpr int kSortOne = 8192;              // tokens that one workgroup sorts
constexpr int kEmbedMinChunk = 8;           // sorted tokens that a wave adds, at least
constexpr int kEmbedMaxChunk = 64;          // (one for each lane)
constexpr int kEmbedWaves = 2048;           // waves that the chunks are made for

// A token and the row of the table that it adds to (the vocabulary: none).
struct SortedToken {
  uint32_t key, token;
};

struct EmbedLayout {
  int passes, bits;    // of the sort: digits and their bits
  int tiles, steps;    // workgroups, and how many kSortStep tokens each takes; 1, 0: all at once
  int chunk, chunks;   // sorted tokens that a wave adds, and how many such
  int width;           // of a piece of a row: a multiple of 4
  size_t histogram, tokens[2], partials, total;  // offsets in bytes
};

inline EmbedLayout embed_layout(int tokens, int vocabulary, int dim) {
  EmbedLayout l;
  int bits = 1;
  while (bits < 31 && vocabulary >> bits) ++bits;  // of the key `vocabulary`
  l.passes = (bits + kSortDigit - 1) / kSortDigit;
  l.bits = (bits + l.passes - 1) / l.passes;
  if (l.bits < kSortFewest) l.bits = kSortFewest;
  const int steps = (tokens + kSortStep - 1) / kSortStep;
  l.steps = (steps + kSortTiles - 1) / kSortTiles;
  l.tiles = (steps + l.steps - 1) / l.steps;
  if (tokens <= kSortOne) {
    l.tiles = 1;
    l.steps = 0;
  }
  // (512 columns a wave: chunks that leave the card idle are not worth their fewer pieces)
  l.chunk = kEmbedMinChunk;
  const long long slabs = (dim + 511) / 512;
  while (l.chunk < kEmbedMaxChunk && tokens * slabs > (long long)l.chunk * kEmbedWaves) l.chunk *= 2;
  l.chunks = (tokens + l.chunk - 1) / l.chunk;
  auto align = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t at = 0;
  l.histogram = at;
  at += align(sizeof(int) * (size_t)l.tiles * kSortBins);
  for (int i = 0; i < 2; ++i) {
    l.tokens[i] = at;
    at += align(sizeof(SortedToken) * (size_t)tokens);
  }
  l.partials = at;
  l.width = (dim + 3) / 4 * 4;
  at += align(sizeof(float) * 2 * (size_t)l.chunks * l.width);
  l.total = at;
  return l;
}

}  // namespace mf
