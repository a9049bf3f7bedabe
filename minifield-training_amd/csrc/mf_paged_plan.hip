// The plan of a paged serving step: where every new token goes, and the work
// items of the attention (mf_paged.h has the terms).  One launch: workgroup 0
// cuts the sequences into tiles and items, the others find the tokens' pages.
//
// Bound: latency (a chain of a few dependent loads, prefix sums over at most a
// few thousand tiles); a step's layers share the plan.
//
// Lengths are taken as they come: starts are held to [0, tokens] and a context to
// the table's reach, so no length can make a later kernel leave its buffers.
#include "mf_paged.h"

namespace mf {

struct PlanArgs {
  const int32_t* starts;     // [R + 1]
  const int32_t* contexts;   // [R]
  const int32_t* table;      // [R][>= width]
  long long table_stride;
  int R, N, width, page_size, pages, G, Hkv, f32;
  FastDiv div_page, div_g;
  char* plan;
  PagedLayout lay;
};

constexpr int kPlanThreads = 256;
// A tile of many rows writes 33 KB of partial results per item and KV head:
// its items are at least this many units.
constexpr int kManyUnits = 4;

// Inclusive prefix sum over the workgroup; `sum` gets the total.
__device__ __forceinline__ int block_prefix(int x, int* lds, int& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();  // the previous round's readers are done
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += lds[w];
    sum += lds[w];
  }
  return x + before;
}

struct Span {
  int start, count, context;
};

__device__ __forceinline__ Span span_of(const PlanArgs& a, int r) {
  Span s;
  s.start = min(max(a.starts[r], 0), a.N);
  s.count = max(min(max(a.starts[r + 1], 0), a.N) - s.start, 0);
  const long long reach = (long long)a.width * a.page_size;
  s.context = (int)min((long long)max(a.contexts[r], 0), min(reach, (long long)INT32_MAX));
  return s;
}

__device__ __forceinline__ int tile_rows_of(const PlanArgs& a, long long rows) {
  return a.f32 || rows <= kFewRows ? kFewRows : kManyRows;
}

// Tile `t` of sequence r: its rows and the keys that its last row sees.
struct TileSpan {
  Span s;
  int r, row0, nrows, keys, units;
};

__device__ __forceinline__ TileSpan tile_of(const PlanArgs& a, const int* pre, int t) {
  TileSpan x;
  int lo = 0, hi = a.R - 1;  // last r with pre[r] <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= t) lo = mid; else hi = mid - 1;
  }
  x.r = lo;
  x.s = span_of(a, lo);
  const long long rows = (long long)x.s.count * a.G;
  const int tr = tile_rows_of(a, rows);
  x.row0 = (t - pre[lo]) * tr;
  x.nrows = (int)max(min((long long)tr, rows - x.row0), 0ll);
  const int last = fast_div(x.row0 + max(x.nrows, 1) - 1, a.div_g);  // token of the last row
  x.keys = max(min(x.s.context - x.s.count + last + 1, x.s.context), 0);
  x.units = (x.keys + kUnitKeys - 1) / kUnitKeys;
  return x;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  if (blockIdx.x > 0) {
    const int t = (blockIdx.x - 1) * kPlanThreads + threadIdx.x;
    if (t >= a.N) return;
    PagedToken rec = {0, -1, 0, -1};
    int lo = 0, hi = a.R - 1;  // last r with starts[r] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.starts[mid] <= t) lo = mid; else hi = mid - 1;
    }
    const Span s = span_of(a, lo);
    if (t >= s.start && t < s.start + s.count) {
      rec.position = s.context - s.count + (t - s.start);
      rec.sequence = lo;
      if (rec.position >= 0) {
        const int p = fast_div(rec.position, a.div_page);
        rec.slot = rec.position - p * a.page_size;
        const int page = a.table[(long long)lo * a.table_stride + p];
        rec.page = page >= 0 && page < a.pages ? page : -1;
      }
    }
    reinterpret_cast<PagedToken*>(a.plan + a.lay.tokens)[t] = rec;
    return;
  }
  __shared__ int pre[kMaxSequences + 1];
  __shared__ int sums[kPlanThreads / 64];
  __shared__ unsigned long long work;
  if (threadIdx.x < 64) reinterpret_cast<int*>(a.plan + a.lay.zeros)[threadIdx.x] = 0;
  if (threadIdx.x == 0) work = 0;
  // tiles before every sequence
  int carry = 0;
  for (int r0 = 0; r0 < a.R; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    int tiles = 0;
    if (r < a.R) {
      const long long rows = (long long)span_of(a, r).count * a.G;
      const int tr = tile_rows_of(a, rows);
      tiles = (int)((rows + tr - 1) / tr);
    }
    int sum;
    const int incl = block_prefix(tiles, sums, sum);
    if (r < a.R) pre[r] = carry + incl - tiles;
    carry += sum;
  }
  const int ntiles = min(carry, a.lay.cap_tiles);
  __syncthreads();
  // units of keys over all tiles
  unsigned long long mine = 0;
  for (int t = threadIdx.x; t < ntiles; t += kPlanThreads) mine += tile_of(a, pre, t).units;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mine += __shfl_xor(mine, off);
  if ((threadIdx.x & 63) == 0) atomicAdd(&work, mine);  // (integers: any order)
  __syncthreads();
  const int target = a.lay.target;
  const int chunk = (int)max((work + target - 1) / target, 1ull);
  int items = 0, split_tiles = 0, rows = 0;
  PagedItem* item = reinterpret_cast<PagedItem*>(a.plan + a.lay.items);
  PagedTile* tile = reinterpret_cast<PagedTile*>(a.plan + a.lay.tiles);
  for (int t0 = 0; t0 < ntiles; t0 += kPlanThreads) {
    const int t = t0 + threadIdx.x;
    TileSpan x = {};
    int splits = 0;
    if (t < ntiles) {
      x = tile_of(a, pre, t);
      const int c = !a.f32 && x.nrows > kFewRows ? max(chunk, kManyUnits) : chunk;
      splits = max((x.units + c - 1) / c, 1);
    }
    int sum_items, sum_tiles, sum_rows;
    const int at = items + block_prefix(splits, sums, sum_items) - splits;
    const int split = splits > 1;
    const int at_tile = split_tiles + block_prefix(split, sums, sum_tiles) - split;
    const int need = split ? splits * x.nrows : 0;
    // (overlapping sequences, which no caller should make, could need more rows
    // than there are: they share the first ones)
    int at_rows = rows + block_prefix(need, sums, sum_rows) - need;
    if ((size_t)at_rows + need > a.lay.cap_rows) at_rows = 0;
    for (int i = 0; i < splits; ++i) {
      if (at + i >= a.lay.cap_items) break;
      PagedItem it;
      it.start = x.s.start;
      it.row0 = x.row0;
      it.nrows = x.nrows;
      it.base = x.s.context - x.s.count;
      it.key0 = (int)((long long)x.units * i / splits) * kUnitKeys;
      it.key1 = min((int)((long long)x.units * (i + 1) / splits) * kUnitKeys, x.keys);
      it.partial = split ? at_rows + i * x.nrows : -1;
      it.sequence = x.r;
      item[at + i] = it;
    }
    if (split) tile[at_tile] = PagedTile{x.s.start, x.row0, x.nrows, at_rows, splits, {0, 0, 0}};
    items += sum_items;
    split_tiles += sum_tiles;
    rows += sum_rows;
  }
  if (threadIdx.x == 0) {
    int* head = reinterpret_cast<int*>(a.plan);
    head[kHeadItems] = min(items, a.lay.cap_items);
    head[kHeadTiles] = split_tiles;
    head[kHeadEnd] = min(max(a.starts[a.R], 0), a.N);
  }
}

hipError_t launch_paged_plan(const int32_t* query_starts, const int32_t* context_lengths,
                             const int32_t* page_table, long long table_stride, int sequences,
                             int tokens, int max_pages, int page_size, int pages, int Hq, int Hkv,
                             bool f32, void* plan, hipStream_t stream) {
  PlanArgs a = {};
  a.starts = query_starts;
  a.contexts = context_lengths;
  a.table = page_table;
  a.table_stride = table_stride;
  a.R = sequences;
  a.N = tokens;
  a.width = max_pages;
  a.page_size = page_size;
  a.pages = pages;
  a.G = Hq / Hkv;
  a.Hkv = Hkv;
  a.f32 = f32;
  a.div_page = make_fastdiv(page_size);
  a.div_g = make_fastdiv(a.G);
  a.plan = reinterpret_cast<char*>(plan);
  a.lay = paged_layout(sequences, tokens, a.G, Hkv, f32);
  const unsigned blocks = 1 + (tokens + kPlanThreads - 1) / kPlanThreads;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mf
