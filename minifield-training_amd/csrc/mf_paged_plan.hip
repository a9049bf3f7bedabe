// The plan of a paged serving step: where every new token goes, and the work
// items of the attention (mf_paged.h has the terms).  One launch: workgroup 0
// cuts the sequences into tiles and items, the others find the tokens' pages.
//
// Bound: latency (a chain of a few dependent loads, prefix sums over at most a
// few thousand tiles): one token of one sequence 5.4 us, 64 sequences 6.7, 20912
// prompt tokens 7.2, 4096 sequences 92.  A step's layers share the plan.
//
// Lengths are taken as they come: starts are held to [0, tokens], and keys end at the
// table's reach, so no length can make a later kernel leave its buffers.
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

// Two counters that are summed together.
struct Two {
  int a, b;
};

// Inclusive prefix sum over a wave, with DPP row shifts and broadcasts (a shuffle
// goes through LDS: six of them took 0.2 us).
__device__ __forceinline__ int wave_prefix_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2, 3
  return x;
}

// Exclusive prefix sums over the workgroup, in place; `sum` gets the totals.
template <int N>
__device__ __forceinline__ void block_prefix(int (&x)[N], int (*lds)[4], int (&sum)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = wave_prefix_sum(x[i]);
  __syncthreads();  // the previous call's readers are done
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) lds[wave][i] = y[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = y[i] - x[i];
    sum[i] = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      const int t = lds[w][i];
      x[i] += w < wave ? t : 0;
      sum[i] += t;
    }
  }
}
__device__ __forceinline__ Two block_prefix(Two x, int (*lds)[4], Two& sum) {
  int y[2] = {x.a, x.b}, s[2];
  block_prefix(y, lds, s);
  sum = {s[0], s[1]};
  return {y[0], y[1]};
}

struct Span {
  int start, count, context;
};

__device__ __forceinline__ Span span_of(const PlanArgs& a, int r) {
  Span s;
  const int start = a.starts[r], next = a.starts[r + 1], context = a.contexts[r];
  s.start = min(max(start, 0), a.N);
  s.count = max(min(max(next, 0), a.N) - s.start, 0);
  s.context = max(context, 0);
  return s;
}

// A tile: its rows, the keys that its last row sees and those in units; what it costs in
// all (its units and the start of an item); the cost of its kind's tiles before it; its
// items (the first one's place, their number) and its first partial row.
struct Tile {
  int sequence, start, row0, nrows, base, keys, units, kind;
  int cost, cost0, item0, items, row;
};


// Workgroup 0's sequences, so that each is read once, and a round's tiles.
struct PlanLds {
  int tiles[kMaxSequences];  // tiles before each sequence
  int start[kMaxSequences], count[kMaxSequences], context[kMaxSequences];
  int sums[kPlanThreads / 64][4];
  int item_at[kPlanThreads], join_at[kPlanThreads];  // before each tile of the round
  Tile tile[kPlanThreads];
};

// The last of `n` ascending entries that is at most x.
__device__ __forceinline__ int last_not_above(const int* at, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool is_few(const PlanArgs& a, long long rows) {
  return a.f32 || rows <= kFewRows;
}

__device__ __forceinline__ Tile tile_of(const PlanArgs& a, const PlanLds& l, int t) {
  Tile x = {};
  const int r = last_not_above(l.tiles, a.R, t);
  x.sequence = r;
  x.start = l.start[r];
  const int count = l.count[r], context = l.context[r];
  const long long rows = (long long)count * a.G;
  x.kind = is_few(a, rows) ? kFew : kMany;
  const int tr = x.kind == kFew ? kFewRows : kManyRows;
  x.row0 = (t - l.tiles[r]) * tr;
  x.nrows = (int)max(min((long long)tr, rows - x.row0), 0ll);
  const int last = fast_div(x.row0 + max(x.nrows, 1) - 1, a.div_g);  // token of the last row
  x.base = context - count;
  x.keys = max(min(x.base + last + 1, a.width * a.page_size), 0);  // (a reach of at most 2^30)
  const int unit = x.kind == kFew ? kFewKeys : kManyKeys;
  x.units = (x.keys + unit - 1) / unit;
  return x;
}

// The shares of a kind: what the first `early` cost, and the others.
struct Shares {
  int early, first, then;
  __device__ int of(int cost) const {
    const int x = cost - early * first;
    const bool is_early = x < 0;  // (one division)
    return (is_early ? cost : x) / (is_early ? first : then) + (is_early ? 0 : early);
  }
  __device__ int begin(int share) const {
    return share < early ? share * first : early * first + (share - early) * then;
  }
};

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ PlanLds l;
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    // (the search in LDS: in memory each of its steps is a round trip)
    for (int r = tid; r < a.R; r += kPlanThreads) l.start[r] = a.starts[r];
    __syncthreads();
    const int t = (blockIdx.x - 1) * kPlanThreads + tid;
    if (t >= a.N) return;
    PagedToken rec = {0, -1, 0, -1};
    const int r = last_not_above(l.start, a.R, t);
    const Span s = span_of(a, r);
    if (t >= s.start && t < s.start + s.count) {
      rec.position = s.context - s.count + (t - s.start);
      rec.sequence = r;
      if (rec.position >= 0 && rec.position < a.width * a.page_size) {
        const int p = fast_div(rec.position, a.div_page);
        rec.slot = rec.position - p * a.page_size;
        const int page = a.table[(long long)r * a.table_stride + p];
        rec.page = page >= 0 && page < a.pages ? page : -1;
      }
    }
    reinterpret_cast<PagedToken*>(a.plan + a.lay.tokens)[t] = rec;
    return;
  }
  if (tid < 64) reinterpret_cast<int*>(a.plan + a.lay.zeros)[tid] = 0;
  // tiles before every sequence
  int ntiles = 0;
  for (int r0 = 0; r0 < a.R; r0 += kPlanThreads) {
    const int r = r0 + tid;
    int tiles = 0;
    if (r < a.R) {
      const Span s = span_of(a, r);
      const long long rows = (long long)s.count * a.G;
      const int tr = is_few(a, rows) ? kFewRows : kManyRows;
      // (never more than the bound, unless sequences overlap)
      tiles = (int)min((rows + tr - 1) / tr, (long long)a.lay.cap_tiles);
      l.start[r] = s.start;
      l.count[r] = s.count;
      l.context[r] = s.context;
    }
    Two total;
    const Two ahead = block_prefix({tiles, 0}, l.sums, total);
    if (r < a.R) l.tiles[r] = ntiles + ahead.a;
    ntiles = min(ntiles + total.a, 1 << 30);
  }
  ntiles = min(ntiles, a.lay.cap_tiles);
  __syncthreads();
  // the cost of each kind's tiles (below 2^31: the entry point checks tiles times the
  // table's reach); the first round's is summed again in its turn
  Tile x = tid < ntiles ? tile_of(a, l, tid) : Tile{};
  int units[2] = {0, 0}, tiles[2] = {0, 0}, ahead[4] = {}, sum4[4];
  for (int t0 = 0; t0 < ntiles; t0 += kPlanThreads) {
    const Tile y = t0 == 0 ? x : t0 + tid < ntiles ? tile_of(a, l, t0 + tid) : Tile{};
    // (a tile without keys, which writes zeros, counts as one unit)
    const bool few = y.kind == kFew, some = y.units > 0;
    const int n = y.nrows > 0 ? max(y.units, 1) : 0;
    int z[4] = {few ? n : 0, few ? 0 : n, few && some, !few && some};
    block_prefix(z, l.sums, sum4);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      units[k] += sum4[k];
      tiles[k] += sum4[2 + k];
      if (t0 == 0) ahead[k] = z[k], ahead[2 + k] = z[2 + k];
    }
  }
  // What a start costs, where there is a unit for every share, and the cost of a share:
  // more than a start's, so that every share has keys.
  const int target[2] = {a.lay.target[0], max(a.lay.target[1], 1)};
  int begin[2], work[2];
  Shares share[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    begin[k] = units[k] < target[k] ? 0 : k == kFew ? kFewStart : kManyStart;
    work[k] = units[k] + begin[k] * tiles[k];
    const int least = max(begin[k] + 1, k == kFew ? 1 : kManyUnits);
    share[k].early = 0;
    share[k].then = max((work[k] + target[k] - 1) / target[k], least);
    share[k].first = share[k].then;
    if (k == kMany && begin[k] > 0) {
      const int early = 256 / a.Hkv, late = target[k] - early;
      const int parts = early * kEarlyShare + late * 4;  // quarters of a later share
      share[k].early = early;
      share[k].then = max((int)((4ll * work[k] + parts - 1) / parts), least);
      share[k].first = (share[k].then * kEarlyShare + 3) / 4;
    }
  }
  Two sum, before;
  x.cost0 = x.kind == kFew ? ahead[0] + begin[0] * ahead[2] : ahead[1] + begin[1] * ahead[3];
  int* shares[2] = {reinterpret_cast<int*>(a.plan + a.lay.shares[0]),
                    reinterpret_cast<int*>(a.plan + a.lay.shares[1])};
  PagedItem* items[2] = {reinterpret_cast<PagedItem*>(a.plan + a.lay.items[0]),
                         reinterpret_cast<PagedItem*>(a.plan + a.lay.items[1])};
  PagedJoin* joins = reinterpret_cast<PagedJoin*>(a.plan + a.lay.joins);
  Two cost = {0, 0}, nitems = {0, 0}, nrest = {0, 0};  // by kind; by kind; joins and partial rows
  for (int t0 = 0; t0 < ntiles; t0 += kPlanThreads) {
    const bool live = t0 + tid < ntiles;
    if (t0 > 0) x = live ? tile_of(a, l, t0 + tid) : Tile{};
    x.cost = x.units > 0 ? x.units + (x.kind == kFew ? begin[0] : begin[1]) : x.nrows > 0 ? 1 : 0;
    if (ntiles > kPlanThreads) {
      before = block_prefix({x.kind == kFew ? x.cost : 0, x.kind == kFew ? 0 : x.cost}, l.sums, sum);
      x.cost0 = x.kind == kFew ? cost.a + before.a : cost.b + before.b;
      cost.a += sum.a;
      cost.b += sum.b;
    } else {
      cost = {work[0], work[1]};
    }
    const bool few = x.kind == kFew;
    const Shares& c = few ? share[0] : share[1];
    // (from the share of its first unit on: its start goes with that)
    x.items = !live ? 0 : x.units == 0 ? 1
              : c.of(x.cost0 + x.cost - 1) - c.of(x.cost0 + (few ? begin[0] : begin[1])) + 1;
    before = block_prefix({few ? x.items : 0, few ? 0 : x.items}, l.sums, sum);
    const int round_items = sum.a + sum.b;
    l.item_at[tid] = before.a + before.b;
    x.item0 = few ? nitems.a + before.a : nitems.b + before.b;
    nitems.a += sum.a;
    nitems.b += sum.b;
    const bool split = x.items > 1;
    const int jr = join_rows(x.kind, x.items);
    before = block_prefix({split ? (x.nrows + jr - 1) / jr : 0,
                           split ? x.items * x.nrows : 0}, l.sums, sum);
    l.join_at[tid] = before.a;
    // (overlapping sequences, which no caller should make, could need more rows
    // than there are: they share the first ones)
    x.row = nrest.b + before.b;
    if ((size_t)x.row + (size_t)x.items * x.nrows > a.lay.cap_rows) x.row = 0;
    l.tile[tid] = x;
    __syncthreads();
    const int round = min(ntiles - t0, kPlanThreads);
    for (int i = tid; i < round_items; i += kPlanThreads) {
      const int j = last_not_above(l.item_at, round, i);
      const Tile y = l.tile[j];
      const int k = i - l.item_at[j];
      const Shares& per = y.kind == kFew ? share[0] : share[1];
      const int unit = y.kind == kFew ? kFewKeys : kManyKeys;
      const int unit0 = y.cost0 + (y.units == 0 ? 0 : y.kind == kFew ? begin[0] : begin[1]);
      const int s = per.of(unit0) + k;
      PagedItem it;
      it.start = y.start;
      it.row0 = y.row0;
      it.nrows = y.nrows;
      it.base = y.base;
      it.key0 = k == 0 ? 0 : (per.begin(s) - unit0) * unit;
      it.key1 = k == y.items - 1 ? y.keys : (per.begin(s + 1) - unit0) * unit;
      it.partial = y.items > 1 ? y.row + k * y.nrows : -1;
      it.sequence = y.sequence;
      const int at = y.item0 + k;
      if (at < a.lay.cap_items[y.kind]) items[y.kind][at] = it;
      // is it the first item of its share?
      if (k > 0 || at == 0 || (y.cost0 > 0 && per.of(y.cost0 - 1) != s))
        if (s < a.lay.target[y.kind]) shares[y.kind][s] = at;
    }
    // (eight threads a tile: a search for each record's tile cost 4 us at 160 tiles of
    // many rows)
    for (int j = tid >> 3; j < round; j += kPlanThreads / 8) {
      const Tile y = l.tile[j];
      if (y.items <= 1) continue;
      const int first = nrest.a + l.join_at[j];
      const int rows = join_rows(y.kind, y.items);
      for (int g = tid & 7; g * rows < y.nrows; g += 8)
        if (first + g < a.lay.cap_joins)
          joins[first + g] = PagedJoin{y.start, y.row0 + g * rows, min(y.nrows - g * rows, rows),
                                       y.row + g * rows, y.items, y.nrows, {0, 0}};
    }
    __syncthreads();
    nrest.a += sum.a;
    nrest.b += sum.b;
  }
  if (tid == 0) {
    int* head = reinterpret_cast<int*>(a.plan);
    const int all_cost[2] = {cost.a, cost.b}, all_items[2] = {nitems.a, nitems.b};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int used = min(all_cost[k] > 0 ? share[k].of(all_cost[k] - 1) + 1 : all_items[k] > 0,
                           a.lay.target[k]);
      head[kHeadShares + k] = used;
      shares[k][used] = min(all_items[k], a.lay.cap_items[k]);
    }
    head[kHeadJoins] = min(nrest.a, a.lay.cap_joins);
    head[kHeadEnd] = min(max(a.starts[a.R], 0), a.N);
    head[kHeadBegin] = l.start[0];
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
