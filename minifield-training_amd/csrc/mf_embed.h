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
constexpr int kSortWaves = 8;               // of each
constexpr int kSortRuns = 2;                // runs of 64 tokens that a wave takes in a step
constexpr int kSortStep = kSortWaves * kSortRuns * 64;
static_assert(kSortBins == kSortWaves * 64, "a thread for each digit");
// Tokens that one workgroup sorts.  The whole gradient of a table of 512 bf16 columns, us, one
// workgroup -> tiles: 1025 tokens of 65536 rows 20.1 -> 25.9, of 300000 58.2 -> 60.9; 8192 of 65536
// 27.5 -> 29.7, of 300000 61.1 -> 63.6; 8192 of 1024 columns and 5000 rows 30.1 -> 31.1, of 500 rows
// (one digit) 26.0 -> 24.1.
constexpr int kSortOne = 8192;
constexpr int kEmbedMinChunk = 8;           // sorted tokens that a wave adds, at least
constexpr int kEmbedMaxChunk = 64;          // (one for each lane)
// Waves that the chunks are made for: with twice as many the sums of 32768 tokens of 1024 columns
// take the same 19 us and joining their pieces 6.9 instead of 4.5.
constexpr int kEmbedWaves = 2048;

// Few tokens, in one launch: a workgroup has every 2^shift-th row of the table over 16 vectors of 16
// bytes of its columns (a slab), and looks through all ids.
constexpr int kEmbedFewBits = 13, kEmbedFewTokens = 1 << kEmbedFewBits;
constexpr int kEmbedFewWaves = 16;
constexpr int kEmbedFewLanes = 16;    // of a row: a load of a wave takes four
constexpr int kEmbedFewGroups = 512;  // workgroups, at most: two a CU
inline int few_slabs(int dim, int vec) { return (dim + kEmbedFewLanes * vec - 1) / (kEmbedFewLanes * vec); }
inline int few_shift(int slabs) {
  int shift = 0;
  while ((2 << shift) * slabs <= kEmbedFewGroups) ++shift;
  return shift;
}
// Rows of one slab, and of up to four of a small table.  What it saves is two launches, 5 us of the
// host a pass (5001 tokens of 1003 x 129 fp32, forward and backward through autograd, 69 us -> 64).
// On the card, us, sorting, sums and joining in launches of their own -> one launch, with ids of
// frequency 1 / rank, and with one id half of the time:
//   bf16  64 wide:   64 tokens of   1003 rows 11.0 ->  7.9, 12.0 ->  8.5
//                  8192 tokens of   1003 rows 22.5 -> 14.9, 31.2 -> 22.3
//                  8192 tokens of 131072 rows 26.6 -> 19.9, 35.2 -> 27.4   (one token 7.2 -> 7.3)
//   fp32 129 wide:   64 tokens of   1003 rows 10.9 ->  8.4, 11.3 ->  9.3
//                  8192 tokens of   1003 rows 22.8 -> 23.2, 31.0 -> 31.2
//                  8192 tokens of   4000 rows 24.0 -> 25.6, 32.1 -> 35.5
//   bf16 512 wide: 8192 tokens of   4000 rows 24.5 -> 28.1, 34.5 -> 35.2: what the host saves still
// Wider rows' slabs look through the ids again, and write a large table's zeros in short pieces: 8192
// tokens of 16000 x 512 bf16 26.3 -> 33.2, of 65536 x 256 26.5 -> 33.0.
inline bool embed_few(int tokens, int vocabulary, int dim, bool f32) {
  const int slabs = few_slabs(dim, f32 ? 4 : 8);
  return tokens <= kEmbedFewTokens &&
         (slabs == 1 ? vocabulary <= 1 << 17 : slabs <= 4 && vocabulary <= 1 << 12);
}

// Workgroups that share the tokens, at most: every one reads the digit counts of all, and takes
// its share step by step.  The whole gradient of 65536 x 64 bf16, us, with 64, 128 and 256: 65536
// tokens 36.9, 38.3, 37.5; 131072 51.1, 52.8, 53.3; 180000 59.4, 57.7, 62.1; 524288 102.6, 91.8, 95.3;
// 700000 128, 113, 112; 2^20 171, 144, 139; 2^23 1153, 877, 759.
inline int sort_tiles(int tokens) { return tokens <= 1 << 17 ? 64 : tokens <= 1 << 19 ? 128 : 256; }

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
  l.steps = (steps + sort_tiles(tokens) - 1) / sort_tiles(tokens);
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
