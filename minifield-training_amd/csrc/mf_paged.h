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
// into tiles, a tile's visible keys into items; one workgroup takes an item of
// one KV head.  Everything is derived on the device: the host never reads a
// length back.
#pragma once

#include "mf_common.h"

namespace mf {

constexpr int kFewRows = 32;     // rows up to which a sequence's waves split the keys
constexpr int kManyRows = 128;   // rows of a tile whose waves split the rows (bf16)
constexpr int kUnitKeys = 128;   // an item's keys come in units of this many
constexpr int kMaxSequences = 4096;
// Items per KV head times KV heads that the splitting aims at: the workgroups
// the chip holds at once (four per CU).
constexpr int kTargetItems = 1024;

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

// One tile that was split: its items' partial results are joined.
struct PagedTile {
  int start, row0, nrows, partial, splits, pad[3];
};

struct PagedLayout {
  size_t zeros, tokens, items, tiles, total;
  int tile_rows;      // rows of the largest tile
  int cap_items, cap_tiles;
  size_t cap_rows;    // rows of partial results
  int target;         // items per KV head aimed at
};

// header (ints): 0 items, 1 split tiles, 2 end of the last sequence's tokens
constexpr int kHeadItems = 0, kHeadTiles = 1, kHeadEnd = 2;

// Bounds: a sequence of M rows has one tile (M <= 32) or ceil(M / 128), so at
// most sequences + tokens G / 128 in all.  With W units of keys over all tiles
// and items of C = max(1, ceil(W / target)) units, the items are at most
// sum ceil(w / C) <= W / C + tiles <= target + tiles, and the partial rows
// sum n ceil(w / C) <= rows of a tile * target + sum n.
__host__ __device__ inline PagedLayout paged_layout(int sequences, int tokens, int G, int Hkv,
                                                    bool f32) {
  PagedLayout p;
  const long long rows = (long long)tokens * G;
  p.tile_rows = f32 ? kFewRows : kManyRows;
  p.target = kTargetItems / Hkv < 1 ? 1 : kTargetItems / Hkv;
  p.cap_tiles = (int)(sequences + rows / p.tile_rows);
  p.cap_items = p.target + p.cap_tiles;
  const long long most = rows < p.tile_rows ? rows : p.tile_rows;
  p.cap_rows = (size_t)(most * p.target + rows);
  size_t off = 256;
  p.zeros = off;  off += 256;
  p.tokens = off; off = align256(off + sizeof(PagedToken) * (size_t)tokens);
  p.items = off;  off = align256(off + sizeof(PagedItem) * (size_t)p.cap_items);
  p.tiles = off;  off = align256(off + sizeof(PagedTile) * (size_t)p.cap_tiles);
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
