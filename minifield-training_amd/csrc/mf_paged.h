// The plan of a paged serving step, shared by the kernels that build it
// (mf_paged_plan.hip) and those that read it (mf_rotary.hip's append,
// mf_paged_attn.hip).
//
// A step has `sequences` ragged sequences.  Sequence r brings the new tokens
// query_starts[r] .. query_starts[r + 1] - 1 of a [tokens, heads, 64] batch;
// its context (new tokens included) holds context_lengths[r] tokens, and token
// position p lives in page page_table[r][p / page_size], slot p % page_size.
// The attention of KV head h works on rows: row i * G + g of a sequence is
// query token i and head h * G + g (G query heads per KV head).  Rows are cut
// into tiles and a tile's visible keys into items.  There are two kinds: tiles
// of few rows (a sequence of up to 32, or in fp32 every 32 rows), whose items are
// bound by the keys they read, and tiles of many (up to 256), bound by their
// products.  Everything is derived on the device: the host never reads a length
// back.
#pragma once

#include "mf_common.h"

namespace mf {

constexpr int kFewRows = 32;
constexpr int kManyRows = 256;
constexpr int kMaxSequences = 4096;
constexpr int kKeyWaves = 4;                // waves of a workgroup, which share a few-rows item's keys
constexpr int kFewKeys = 32 * kKeyWaves;    // keys come in units of this many there
constexpr int kManyKeys = 64;               // and of this many here
// Shares times workgroups of a share: what is resident at once, two per CU.  Many
// rows with 256, 384, 640, 768 and 1024: three chunks 97, 93, 96, 96 and 94 us, with
// 512 83; a chunk over 28 K keys 355, 324 and 320 with 640 and more, with 512 309.
// Few rows with 1024: drafts 80 us, with 512 76.
constexpr int kFewGroups = 512;
constexpr int kManyGroups = 512;
// A tile of many rows writes up to 66 KB of partial results per item and KV head:
// its shares have at least this many units.  With 1, 2, 3, 4 and 8, us: 300 tokens
// behind 500 15.7, 15.9, 19.4, 21.1 and 26.4; 128 behind 2000 17.7, 15.5, 16.2, 16.4
// and 23.1.
constexpr int kManyUnits = 2;
// What the first item of a tile costs beside its keys, in units, where there is a unit for
// every share: a share of many short tiles is then as long as one of a long tile's
// middle.  Many rows with 0, 1, 2, 3 and 4, us: prompts of 491, 3814 and 699 tokens
// 112, 103, 97, 98 and 96; 14 chunks of up to 624 behind 1000 to 2300 129, 129, 121,
// 118 and 121.  Few rows with 0 and 1: drafts 76.5 and 75, 200 single tokens over up to
// 500 keys 31.2 and 29.1.  (Where there are fewer units than shares, none has several
// tiles: 300 tokens behind 500 16 without and 18 with.)
constexpr int kFewStart = 1, kManyStart = 2;
// Quarters of a later share of many rows that those of the first workgroup of each CU
// get: its waves, the older ones, are served first (with equal shares it ends a chunk
// after 229 us, the second after 290).  With 4, 5, 6 and 7, us: a chunk over 28 K keys
// 302, 297, 292 and 298, 16 K causal 621, 605, 616 and 634, a mixed step 126, 125, 128
// and 131, 8 x 200 tokens behind 300 26.0, 25.2, 25.4 and 26.4.
constexpr int kEarlyShare = 5;
// Rows of a split tile that one workgroup joins: 8, whose items it shares out to four
// groups of threads, or 32 of a tile of many rows with up to 8 items, which leaves a
// quarter of the records to the plan (of a mixed step 6.4 us against 6.9, of 20912
// prompt tokens 7.3 against 8.7; the join takes the same).  32 rows of fp32 tiles
// made their join 1 us longer.
constexpr int kJoinRows = 8;
constexpr int kJoinManyRows = 32, kJoinFewItems = 8;
__host__ __device__ inline int join_rows(int kind, int items) {
  return kind != 0 && items <= kJoinFewItems ? kJoinManyRows : kJoinRows;
}

// One new token: where it is and where its key and value go (page < 0: nowhere).
struct PagedToken {
  int position, page, slot, sequence;
};

// One item: keys [key0, key1) of `nrows` rows from row0 on.
struct PagedItem {
  int start;     // the sequence's first token
  int row0, nrows;
  int base;      // position of the sequence's first new token (negative: it has no keys yet)
  int key0, key1;
  int partial;   // first row of its partial results, or -1 when it writes the output
  int sequence;
};

// Up to join_rows() rows of a tile that was split, whose items' partial results are
// joined: item i's are rows partial + i * step.
struct PagedJoin {
  int start, row0, nrows, partial, splits, step, pad[2];
};

// Kinds of tiles.
constexpr int kFew = 0, kMany = 1;

struct PagedLayout {
  size_t zeros, tokens, shares[2], items[2], joins, total;
  int head_pair;       // KV heads a wave of a few-rows item takes (bf16: 2 where they are even)
  int target[2];       // shares of each kind at most
  int cap_tiles, cap_items[2], cap_joins;
  size_t cap_rows;     // rows of partial results
};

// header (ints): shares of each kind (0 and 1), join records, the first sequence's first
// token and the one behind the last sequence
constexpr int kHeadShares = 0, kHeadJoins = 2, kHeadEnd = 3, kHeadBegin = 4;

// Bounds: a sequence of M rows has one tile (M <= 32) or ceil(M / 256), so at
// most sequences + tokens G / 256 in all.  Every boundary between shares adds an
// item, so there are at most shares + tiles of each kind.  Only a tile that a boundary
// cuts has partial rows, an item's worth for each boundary and one more: fewer than
// rows of a tile * shares for the boundaries, and for the tiles not more than that again
// nor than there are rows.  And only such a tile has join records: four (32 rows by 8),
// or, of many rows, 8 with up to 8 items and 32 with more, which takes 8 boundaries.
// (Of 131072 tokens, 16/8 heads: 87 MB of partial results.  Bounded by the rows of all
// tiles it was 600.)
static_assert(kManyRows / kJoinRows <= kJoinFewItems * (kManyRows / kJoinManyRows),
              "a tile's records against the boundaries that cut it");
__host__ __device__ inline PagedLayout paged_layout(int sequences, int tokens, int G, int Hkv,
                                                    bool f32) {
  PagedLayout p;
  const long long rows = (long long)tokens * G;
  p.head_pair = !f32 && Hkv % 2 == 0 ? 2 : 1;
  const int pairs = Hkv / p.head_pair;
  const bool many = !f32 && rows > kFewRows;
  p.target[kFew] = kFewGroups / pairs < 1 ? 1 : kFewGroups / pairs;
  p.target[kMany] = !many ? 0 : kManyGroups / Hkv < 1 ? 1 : kManyGroups / Hkv;
  p.cap_tiles = (int)(sequences + rows / (f32 ? kFewRows : kManyRows));
  p.cap_items[kFew] = p.target[kFew] + (f32 ? p.cap_tiles : sequences);
  p.cap_items[kMany] = many ? p.target[kMany] + p.cap_tiles : 0;
  const long long joins = p.cap_tiles + rows / kJoinRows;
  const long long cut_joins = (long long)(kFewRows / kJoinRows) * p.target[kFew] +
                              (long long)(kManyRows / kJoinManyRows) * p.target[kMany];
  p.cap_joins = (int)(joins < cut_joins ? joins : cut_joins);
  const long long cut_rows = (long long)kFewRows * p.target[kFew] + (long long)kManyRows * p.target[kMany];
  p.cap_rows = (size_t)((rows < kFewRows ? rows : kFewRows) * p.target[kFew] +
                        (rows < kManyRows ? rows : kManyRows) * p.target[kMany] +
                        (rows < cut_rows ? rows : cut_rows));
  size_t off = 256;
  p.zeros = off;  off += 256;
  p.tokens = off; off = align256(off + sizeof(PagedToken) * (size_t)tokens);
  for (int k = 0; k < 2; ++k) {
    p.shares[k] = off;
    off = align256(off + sizeof(int) * (size_t)(p.target[k] + 1));
    p.items[k] = off;
    off = align256(off + sizeof(PagedItem) * (size_t)p.cap_items[k]);
  }
  p.joins = off;  off = align256(off + sizeof(PagedJoin) * (size_t)p.cap_joins);
  p.total = off;
  return p;
}

// Partial results: (max in log2 units, sum) and 64 unnormalised outputs per row
// and KV head, fp32.
inline size_t paged_workspace_bytes(const PagedLayout& p, int Hkv) {
  return align256(p.cap_rows * Hkv * (2 * sizeof(float))) + p.cap_rows * Hkv * (kD * sizeof(float));
}

// Strides of one page pool, in elements: [page][slot][head][64], the last dense.
struct PagedStrides {
  long long page, slot, head;
};

}  // namespace mf
