// Embedding lookup with scaling, and its gradient by sorted tokens, on gfx950.
//
//   out[n] = scale table[ids[n]],   dtable[v] = scale * sum of dout[n] over ids[n] = v,
// products and sums in fp32, rounded once.  Ids outside the table and the padding
// id have rows of zeros and no part in the gradient.
//
// The lookup is a copy of rows and bound by memory.
//
// The gradient writes the whole table and reads every row of dout once.  Tokens are
// sorted by id (stably, so a row adds its tokens in their order: the same bits every
// time, which atomic adds would not give), and waves take equal chunks of the sorted
// order, so the tokens of a frequent id are read by as many waves as any others.  A wave
// holds its columns' sum in registers and writes a row when the id changes; what
// runs past its chunk's ends goes to a workspace in fp32, and a last launch adds
// those pieces in chunk order, a run's by one workgroup of every 256 columns: their number
// is what a frequent id costs.  The whole gradient of 65536 x 1024 bf16, us, with even ids and
// with an id that half of the tokens have: 8192 tokens 36 and 46, 32768 55 and 62; 2^20 tokens
// 560, 630 with an id of a third, 760 with one id alone; 2^24 tokens of one id, 64 wide, 6.0 ms.
// The rows of ids that no token has are zeros: the launches that sort, which are a few
// waves' work each, zero the whole table beside it, a share each.
//
// The sort goes by digits of up to 9 bits from the lowest, each in two launches: tiles of
// the tokens count their digits, and then place their tokens.  A wave takes runs of 64;
// lanes with one digit find each other by ballots over its bits, so that a lane's place is
// its digit's first place, what the tiles, steps and waves before have of that digit, and
// the lanes before it.  Few tokens are sorted by one workgroup in one launch; of narrow rows, and of
// small tables, their whole gradient is one launch (embed_few_kernel).
//
// Measured, 32768 tokens of 65536 x 1024 bf16, us: lookup 17 (64 MiB written, the table's
// rows from the cache); zeroing 128 MiB beside sorting 28 (4.7 TB/s; the four launches
// alone 18, the zeros alone 20), sums 18.6 (6 TB/s with the rows and pieces they write),
// joining 4.5.  5001 tokens of 1003 x 129 fp32: in one launch 18.5 (as three, sorting 11, sums
// 4.1 and joining 4.7).
#include <algorithm>

#include "mf_embed.h"
#include "mf_rows.h"

namespace mf {

struct EmbedArgs {
  const void* ids;
  const void* rows;  // the table, or the gradient of the output
  void* out;         // the output, or the table's gradient
  long long stride, padding;
  int tokens, vocabulary, dim;
  float scale;
  bool ids64;
};

// Token n's id, and the table's row of an id: `vocabulary` for none.
__device__ __forceinline__ long long id_of(const EmbedArgs& a, int n) {
  return a.ids64 ? reinterpret_cast<const long long*>(a.ids)[n]
                 : (long long)reinterpret_cast<const int32_t*>(a.ids)[n];
}
__device__ __forceinline__ uint32_t row_of(const EmbedArgs& a, long long id) {
  return id >= 0 && id < a.vocabulary && id != a.padding ? (uint32_t)id : (uint32_t)a.vocabulary;
}

// L lanes a token.  Plain stores: the next operator reads the rows from the last-level cache.
// Streamed ones take 17 us instead of 20 at 32768 x 1024 bf16 by themselves, but the norm
// behind them 37 instead of 22.  (Four tokens a group of lanes, for more loads in flight,
// measured 21 us against 21, and 3.3 against 2.7 at 64 tokens.)
template <typename T, int L, Edge E>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs a) {
  constexpr int N = kVec<T>, C = 2;
  const int n = blockIdx.x * (256 / L) + threadIdx.x / L, lane = threadIdx.x % L;
  if (n >= a.tokens) return;
  const uint32_t id = row_of(a, id_of(a, n));
  const bool met = id < (uint32_t)a.vocabulary;
  const T* from = reinterpret_cast<const T*>(a.rows) + (size_t)(met ? id : 0) * a.stride;
  T* to = reinterpret_cast<T*>(a.out) + (size_t)n * a.dim;
  for (int first = 0; first * N < a.dim; first += L * C) {
    RowPlace<T, E> at[C];
    Vec<T> v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      at[c] = RowPlace<T, E>(first + c * L + lane, a.dim);
      v[c] = at[c].load(from);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = met ? (float)v[c][i] * a.scale : 0.f;
      at[c].store(to, x);
    }
  }
}

// ---------------------------------------------------------------------------

struct SortArgs {
  EmbedArgs e;
  const SortedToken* from;  // null: the ids as they come
  SortedToken* to;
  int* histogram;           // [tiles][kSortBins]
  int tiles, steps, shift, bits, passes;
  // a share of the table's gradient to zero, in bytes, and what a workgroup takes of it
  size_t zero_first, zero_last, zero_block;
};

// COUNT entries in runs of 64 from `first` on, loaded without a condition: those beyond the
// last are the last again.
template <int COUNT>
__device__ __forceinline__ void sort_entries(const SortArgs& a, int first, int lane,
                                             SortedToken (&t)[COUNT]) {
  if (a.from) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) t[j] = a.from[min(first + 64 * j + lane, a.e.tokens - 1)];
  } else {
    long long id[COUNT];
#pragma unroll
    for (int j = 0; j < COUNT; ++j) id[j] = id_of(a.e, min(first + 64 * j + lane, a.e.tokens - 1));
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
      t[j] = SortedToken{row_of(a.e, id[j]), (uint32_t)(first + 64 * j + lane)};
  }
}

// (as streams: what reads the gradient next comes long after the launches that add to it)
__device__ __forceinline__ void zero_share(const SortArgs& a) {
  const size_t first = a.zero_first + (size_t)(blockIdx.x - a.tiles) * a.zero_block;
  const size_t last = min(a.zero_last, first + a.zero_block);
  char* out = reinterpret_cast<char*>(a.e.out);
  const size_t step = blockDim.x * 16;
  size_t at = first + threadIdx.x * 16;
  for (; at + 3 * step + 16 <= last; at += 4 * step) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4*>(out + at + j * step));
  }
  for (; at < last; at += step) {
    if (at + 16 <= last) {
      __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4*>(out + at));
    } else {
      for (size_t b = at; b < last; b += 2) *reinterpret_cast<uint16_t*>(out + b) = 0;
    }
  }
}

// Lanes of the wave that have this lane's digit, among those that take part: for every
// bit, the lanes whose bit is the lane's own (four instructions).
template <int BITS>
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool live) {
  const uint64_t all = __ballot(live);
  uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const uint32_t own = (uint32_t)((int32_t)(digit << (31 - b)) >> 31);
    const uint64_t set = __ballot(own != 0);
    lo &= ~((uint32_t)set ^ own);
    hi &= ~((uint32_t)(set >> 32) ^ own);
  }
  return (uint64_t)hi << 32 | lo;
}

// The lane's place among the tokens of its digit: behind those that `count` (a wave's own
// counters) holds and the lanes before it; the counters then hold these too.  A wave's LDS
// operations keep their order.
template <int BITS>
__device__ __forceinline__ int place_of(volatile int* count, uint32_t digits, bool live, int lane) {
  const uint32_t digit = digits & ((1u << BITS) - 1);
  const uint64_t same = same_digit<BITS>(digit, live);
  const int before = __popcll(same & ((1ull << lane) - 1));
  int to = 0;
  if (live) {
    to = count[digit] + before;
    if (before == 0) count[digit] = to + __popcll(same);
  }
  return to;
}

// How many of its tokens each tile has of every digit.
__global__ __launch_bounds__(512) void sort_count_kernel(SortArgs a) {
  constexpr int AHEAD = 4;  // runs of 64 tokens that a wave has in flight
  __shared__ int counts[kSortBins];
  if ((int)blockIdx.x >= a.tiles) return zero_share(a);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int runs = a.steps * kSortRuns;
  counts[threadIdx.x] = 0;
  __syncthreads();
  for (int r0 = 0; r0 < runs; r0 += AHEAD) {
    const int first = ((blockIdx.x * kSortWaves + wave) * runs + r0) * 64;
    SortedToken t[AHEAD];
    sort_entries(a, first, lane, t);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (r0 + j < runs && first + 64 * j + lane < a.e.tokens)
        atomicAdd(&counts[t[j].key >> a.shift & ((1 << a.bits) - 1)], 1);
  }
  __syncthreads();
  a.histogram[(size_t)blockIdx.x * kSortBins + threadIdx.x] = counts[threadIdx.x];
}

// Each tile's tokens to their places by one digit, kSortStep at a time.  Thread d keeps where
// the tile's next token of digit d goes.
template <int BITS>
__global__ __launch_bounds__(512) void sort_place_kernel(SortArgs a) {
  constexpr int ROWS = 32;  // of the histogram in flight
  __shared__ int place[kSortWaves][kSortBins];
  __shared__ int wave_sums[kSortWaves];
  if ((int)blockIdx.x >= a.tiles) return zero_share(a);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  int first = blockIdx.x * a.steps * kSortStep + wave * kSortRuns * 64;
  SortedToken t[kSortRuns];
  sort_entries(a, first, lane, t);
  // digit tid: what the tiles before have of it, and all of them
  int before = 0, whole = 0;
  for (int t0 = 0; t0 < a.tiles; t0 += ROWS) {
    int h[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      h[j] = a.histogram[(size_t)min(t0 + j, a.tiles - 1) * kSortBins + tid];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      whole += t0 + j < a.tiles ? h[j] : 0;
      before += t0 + j < (int)blockIdx.x ? h[j] : 0;
    }
  }
  int sum = whole;  // of the digits up to this in the wave
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(sum, m);
    if (lane >= m) sum += o;
  }
  if (lane == 63) wave_sums[wave] = sum;
  int next = sum - whole + before;
  for (int step = 0; step < a.steps; ++step, first += kSortStep) {
#pragma unroll
    for (int d = 0; d < kSortBins; d += 64) place[wave][d + lane] = 0;
    int to[kSortRuns];
    bool live[kSortRuns];
    SortedToken now[kSortRuns];
#pragma unroll
    for (int j = 0; j < kSortRuns; ++j) {  // among the wave's own of the digit
      now[j] = t[j];
      live[j] = first + 64 * j + lane < a.e.tokens;
      to[j] = place_of<BITS>(place[wave], now[j].key >> a.shift, live[j], lane);
    }
    if (step + 1 < a.steps) sort_entries(a, first + kSortStep, lane, t);
    __syncthreads();
    if (step == 0)
      for (int i = 0; i < wave; ++i) next += wave_sums[i];
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) {
      const int c = place[i][tid];
      place[i][tid] = next;
      next += c;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortRuns; ++j)
      if (live[j]) a.to[place[wave][now[j].key >> a.shift & ((1 << BITS) - 1)] + to[j]] = now[j];
  }
}

// Up to 1024 ITEMS tokens, all digits in one launch: 16 waves with ITEMS runs of 64 each, kept
// in registers and exchanged through LDS from digit to digit.
template <int BITS, int ITEMS>
__global__ __launch_bounds__(1024) void sort_one_kernel(SortArgs a) {
  constexpr int WAVES = 16;
  __shared__ int place[WAVES][kSortBins];
  __shared__ SortedToken list[1024 * ITEMS];
  __shared__ int wave_sums[kSortBins / 64];
  if (blockIdx.x >= 1) return zero_share(a);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int n0 = wave * 64 * ITEMS + lane;
  SortedToken t[ITEMS];
  sort_entries(a, n0 - lane, lane, t);
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * BITS;
    for (int d = lane; d < kSortBins; d += 64) place[wave][d] = 0;
    int to[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)  // among the wave's own of the digit
      to[j] = place_of<BITS>(place[wave], t[j].key >> shift, n0 + 64 * j < a.e.tokens, lane);
    __syncthreads();
    // first places: over the digits, then over a digit's waves
    int whole = 0, sum = 0;
    if (tid < kSortBins) {
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const int c = place[i][tid];
        place[i][tid] = whole;
        whole += c;
      }
      sum = whole;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(sum, m);
        if (lane >= m) sum += o;
      }
      if (lane == 63) wave_sums[wave] = sum;
    }
    __syncthreads();
    if (tid < kSortBins) {
      int start = sum - whole;
      for (int i = 0; i < wave; ++i) start += wave_sums[i];
#pragma unroll
      for (int i = 0; i < WAVES; ++i) place[i][tid] += start;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (n0 + 64 * j < a.e.tokens)
        list[place[wave][t[j].key >> shift & ((1 << BITS) - 1)] + to[j]] = t[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (n0 + 64 * j < a.e.tokens) t[j] = list[n0 + 64 * j];
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (n0 + 64 * j < a.e.tokens) a.to[n0 + 64 * j] = t[j];
}

// ---------------------------------------------------------------------------

struct SumArgs {
  const SortedToken* sorted;
  const void* dout;
  void* dtable;
  float* partials;  // [chunks][2][width]: what a chunk has of the run it begins in, and ends in
  long long stride;
  int tokens, vocabulary, dim, width, chunk, chunks, slabs;
  float scale;
};

// A wave adds the tokens of a chunk over 64 vectors of columns.
template <typename T, Edge E>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
  constexpr int N = kVec<T>, AHEAD = 8;
  const int lane = threadIdx.x & 63;
  const int item = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int chunk = item / a.slabs;
  const RowPlace<T, E> at((item % a.slabs) * 64 + lane, a.dim);
  if (chunk >= a.chunks) return;
  const int first = chunk * a.chunk, count = min(a.chunk, a.tokens - first);
  // lane i holds entry i; the keys on either side of the chunk beside them
  const SortedToken mine = a.sorted[first + min(lane, count - 1)];
  const uint32_t none = a.vocabulary;
  const uint32_t before = first > 0 ? a.sorted[first - 1].key : none;
  const uint32_t behind = first + count < a.tokens ? a.sorted[first + count].key : none;
  // tokens without a row come last
  const int live = __popcll(__ballot(lane < count && mine.key < none));
  if (live == 0) return;
  auto key_at = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane(mine.key, i); };
  const T* dout = reinterpret_cast<const T*>(a.dout);
  auto fetch = [&](int i) {
    const uint32_t token = __builtin_amdgcn_readlane(mine.token, min(i, live - 1));
    return at.template load<true>(dout + (size_t)token * a.stride);
  };
  float sum[N] = {};
  bool head = key_at(0) == before;
  Vec<T> ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) ahead[j] = fetch(j);
  for (int i0 = 0; i0 < live; i0 += AHEAD) {
    Vec<T> v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v[j] = ahead[j];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ahead[j] = fetch(i0 + AHEAD + j);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j;
      if (i >= live) break;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += (float)v[j][e];
      const uint32_t key = key_at(i), next = i + 1 < count ? key_at(i + 1) : behind;
      if (i + 1 < live && next == key) continue;
      // the run ends here, or with the chunk
      const bool open = next == key;
      if (head || open) {
        float* to = a.partials + ((size_t)chunk * 2 + (head ? 0 : 1)) * a.width;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (at.any() && at.mine(e)) to[at.at + e] = sum[e];
      } else {
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = sum[e] * a.scale;
        at.store(reinterpret_cast<T*>(a.dtable) + (size_t)key * a.dim, x);
      }
      head = false;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = 0.f;
    }
  }
}

// The runs that pass a chunk's end: the workgroup of the chunk that one begins in adds
// its pieces over 256 columns, each wave a quarter of the chunks, in order.
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a) {
  __shared__ f32x4 sums[4][64];
  const int chunk = blockIdx.x, first = chunk * a.chunk, next = first + a.chunk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the keys on both sides of the chunk's end and in front of its start
  const uint32_t none = a.vocabulary;
  const uint32_t key = a.sorted[next - 1].key, behind = a.sorted[next].key;
  const uint32_t before = first > 0 ? a.sorted[first - 1].key : none;
  // (a run that fills the chunk from an earlier one on is that one's)
  if (key >= none || behind != key || before == key) return;
  // the chunks that begin within the run: the next 64 at once, of the others every `step`th
  int count = 0, most = a.chunks - 1 - chunk;
  for (int step = 1; count < most; step = (most - count + 63) / 64) {
    const int c = count + (lane + 1) * step;
    const bool in = c <= most && a.sorted[(size_t)(chunk + min(c, most)) * a.chunk].key == key;
    const int more = __popcll(__ballot(in));  // (the keys are sorted: the first lanes)
    count += more * step;
    if (more < 64) most = min(most, count + step - 1);
  }
  const int col = (blockIdx.y * 64 + lane) * 4;
  const int per = (count + 4) / 4, from = wave * per, to = min(count + 1, from + per);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  // (rows of `width`, a multiple of 4; lanes beyond it read its start)
  const float* piece = a.partials + ((size_t)chunk * 2 + 1) * a.width + (col < a.width ? col : 0);
  // (64 at a time: added in a row, 2^20 equal tokens of one id would be off by 1e-5 and more)
  for (int c0 = from; c0 < to; c0 += 64) {
    const int c1 = min(to, c0 + 64);
    f32x4 some = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int c = c0; c < c1; ++c) {
      // the run's first piece is its chunk's second, the others their chunks' first
      some += *reinterpret_cast<const f32x4*>(piece + (c == 0 ? 0ll : (2ll * c - 1) * a.width));
    }
    s += some;
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) s += sums[i][lane];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < a.dim)
      reinterpret_cast<T*>(a.dtable)[(size_t)key * a.dim + col + i] = (T)(s[i] * a.scale);
}

// ---------------------------------------------------------------------------

struct FewArgs {
  EmbedArgs e;
  const void* dout;
  long long stride;
  int shift;  // groups of rows: 1 << shift
};

// The whole gradient of few tokens in one launch: a workgroup has every 2^shift-th row
// of the table over kEmbedFewLanes vectors of columns.  It looks through all ids, sorts the tokens
// of its rows by row in LDS (by one digit, stably), and its waves take equal shares of them, a
// run at a time, four tokens in a load.  What passes a share's end stays in LDS and is added there
// by the wave that a run begins in.
template <typename T, Edge E>
__global__ __launch_bounds__(1024) void embed_few_kernel(FewArgs a) {
  constexpr int N = kVec<T>, W = kEmbedFewWaves, RUNS = kEmbedFewTokens / (W * 64);
  constexpr int L = kEmbedFewLanes, R = 64 / L, AHEAD = 8;
  constexpr uint32_t kToken = (1 << kEmbedFewBits) - 1;
  __shared__ uint32_t list[kEmbedFewTokens];  // a token and, above it, its row
  // first the places of a wave's tokens by row, then the pieces of its share's two ends
  __shared__ union {
    int place[W][kSortBins];
    float piece[W][2][N][L];
  } lds;
  __shared__ int row_sums[kSortBins / 64];
  __shared__ uint64_t met[kSortBins / 64];  // rows that have tokens
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  // (workgroups go to the XCDs in turn: a frequent id's columns to different ones)
  const int group = (blockIdx.x + blockIdx.y) % gridDim.x, vec = lane % L, sub = lane / L;
  const RowPlace<T, E> at(blockIdx.y * L + vec, a.e.dim);
  T* out = reinterpret_cast<T*>(a.e.out);
  auto row_at = [&](int r) { return out + (((size_t)r << a.shift) + group) * a.e.dim; };
  const int n0 = wave * RUNS * 64 + lane;
  uint32_t row[RUNS];
  long long id[RUNS];
#pragma unroll
  for (int j = 0; j < RUNS; ++j) id[j] = id_of(a.e, min(n0 + 64 * j, a.e.tokens - 1));
  for (int d = lane; d < kSortBins; d += 64) lds.place[wave][d] = 0;
  int to[RUNS];
  uint32_t live = 0;
#pragma unroll
  for (int j = 0; j < RUNS; ++j) {
    const uint32_t r = row_of(a.e, id[j]);
    const bool in = n0 + 64 * j < a.e.tokens && r < (uint32_t)a.e.vocabulary &&
                    (int)(r & ((1u << a.shift) - 1)) == group;
    row[j] = r >> a.shift;
    live |= (uint32_t)in << j;
    to[j] = 0;
    if (__any(in)) to[j] = place_of<kSortDigit>(lds.place[wave], row[j], in, lane);
  }
  __syncthreads();
  // first places: over the rows, then over a row's waves
  int whole = 0, sum = 0;
  if (tid < kSortBins) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int c = lds.place[i][tid];
      lds.place[i][tid] = whole;
      whole += c;
    }
    sum = whole;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(sum, m);
      if (lane >= m) sum += o;
    }
    const uint64_t some = __ballot(whole > 0);
    if (lane == 63) row_sums[wave] = sum;
    if (lane == 0) met[wave] = some;
  }
  __syncthreads();
  if (tid < kSortBins) {
    int start = sum - whole;
    for (int i = 0; i < wave; ++i) start += row_sums[i];
#pragma unroll
    for (int i = 0; i < W; ++i) lds.place[i][tid] += start;
  }
  int tokens = 0;
  for (int i = 0; i < kSortBins / 64; ++i) tokens += row_sums[i];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < RUNS; ++j)
    if (live >> j & 1)
      list[lds.place[wave][row[j]] + to[j]] = row[j] << kEmbedFewBits | (uint32_t)(n0 + 64 * j);
  // rows without tokens
  const int rows = ((a.e.vocabulary - 1 - group) >> a.shift) + 1;
  const float zero[N] = {};
  for (int r = wave * R + sub; r < rows; r += W * R)
    if (!(met[r >> 6] >> (r & 63) & 1)) at.store(row_at(r), zero);
  __syncthreads();
  constexpr int none = kSortBins;  // (no row's number)
  const int per = (tokens + W - 1) / W;
  const int first = wave * per, last = min(tokens, first + per);
  auto key_of = [&](int i) {
    return i >= 0 && i < tokens ? uniform((int)(list[i] >> kEmbedFewBits)) : none;
  };
  const T* dout = reinterpret_cast<const T*>(a.dout);
  int open = none;  // the row whose run begins in the share and goes on behind it
  for (int i = first; i < last;) {
    const int key = key_of(i);
    const bool head = i == first && key_of(first - 1) == key;
    int end = i;  // of the run, or of the share
    for (int more = 64; more == 64 && end < last; end += more) {
      const int k = min(end + lane, last - 1);
      const uint64_t same = __ballot(end + lane < last && (int)(list[k] >> kEmbedFewBits) == key);
      more = same == ~0ull ? 64 : __ffsll((long long)~same) - 1;
    }
    float s[N] = {};
    auto add = [&](auto count, auto all) {  // loads at once; all: none of their tokens is behind the end
      constexpr int C = decltype(count)::value;
      Vec<T> x[C];
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const uint32_t token = list[min(i + R * j + sub, end - 1)] & kToken;
        x[j] = at.load(dout + (size_t)token * a.stride);
      }
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e)
          s[e] += decltype(all)::value || i + R * j + sub < end ? (float)x[j][e] : 0.f;
      i += R * C;
    };
    using std::integral_constant;
    while (i + R * AHEAD <= end) add(integral_constant<int, AHEAD>{}, std::true_type{});
    while (i + R < end) add(integral_constant<int, AHEAD / 2>{}, std::false_type{});
    if (i < end) add(integral_constant<int, 1>{}, std::false_type{});
    i = end;
    if constexpr (L == 16) {
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = halves_sum(rows16_sum(s[e]));
    }
    if (head || key_of(i) == key) {
      if (!head) open = key;
      if (sub == 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) lds.piece[wave][head ? 0 : 1][e][vec] = s[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] *= a.e.scale;
      if (sub == 0) at.store(row_at(key), s);
    }
  }
  __syncthreads();
  if (open == none) return;
  float s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = lds.piece[wave][1][e][vec];
  for (int i = wave + 1; i < W && key_of(i * per) == open; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += lds.piece[i][0][e][vec];
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] *= a.e.scale;
  if (sub == 0) at.store(row_at(open), s);
}

// ---------------------------------------------------------------------------

template <typename T, Edge E>
static void launch_embed_e(const EmbedArgs& a, hipStream_t stream) {
  const int vectors = (a.dim + kVec<T> - 1) / kVec<T>;
  auto go = [&](auto l) {
    constexpr int L = decltype(l)::value;
    hipLaunchKernelGGL((embed_kernel<T, L, E>), dim3((a.tokens + 256 / L - 1) / (256 / L)),
                       dim3(256), 0, stream, a);
  };
  // Rows that 16 lanes take at once.  (32768 tokens, bf16, 16 lanes a token against 64: 128
  // columns 5.8 us and 9.1, 256 7.5 and 10.4, in several turns 512 12.9 and 13.8, 1024 23.4
  // and 23.0; 5001 tokens of 129 fp32 3.4 and 3.1.)
  if (vectors <= 2 * 16)
    go(std::integral_constant<int, 16>{});
  else
    go(std::integral_constant<int, 64>{});
}

template <typename T>
static hipError_t launch_embed_t(const EmbedArgs& a, hipStream_t stream) {
  switch (edge_of<T>(a.dim)) {
    case EDGE_WHOLE: launch_embed_e<T, EDGE_WHOLE>(a, stream); break;
    case EDGE_CUT: launch_embed_e<T, EDGE_CUT>(a, stream); break;
    default: launch_embed_e<T, EDGE_SHORT>(a, stream);
  }
  return hipGetLastError();
}

hipError_t launch_embed(const void* ids, bool ids64, const void* table, long long stride, bool f32,
                        int tokens, int vocabulary, int dim, long long padding, float scale,
                        void* out, hipStream_t stream) {
  const EmbedArgs a{ids, table, out, stride, padding, tokens, vocabulary, dim, scale, ids64};
  return f32 ? launch_embed_t<float>(a, stream) : launch_embed_t<bf16>(a, stream);
}

template <typename T>
static hipError_t launch_sums(SumArgs a, hipStream_t stream) {
  a.slabs = (a.dim + 64 * kVec<T> - 1) / (64 * kVec<T>);
  const dim3 grid((unsigned)(((long long)a.chunks * a.slabs + 3) / 4));
  switch (edge_of<T>(a.dim)) {
    case EDGE_WHOLE:
      hipLaunchKernelGGL((embed_sum_kernel<T, EDGE_WHOLE>), grid, dim3(256), 0, stream, a);
      break;
    case EDGE_CUT:
      hipLaunchKernelGGL((embed_sum_kernel<T, EDGE_CUT>), grid, dim3(256), 0, stream, a);
      break;
    default:
      hipLaunchKernelGGL((embed_sum_kernel<T, EDGE_SHORT>), grid, dim3(256), 0, stream, a);
  }
  if (a.chunks > 1)
    hipLaunchKernelGGL((embed_join_kernel<T>), dim3(a.chunks - 1, (a.dim + 255) / 256), dim3(256), 0,
                       stream, a);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_few(const FewArgs& a, hipStream_t stream) {
  const int slabs = few_slabs(a.e.dim, kVec<T>);
  const dim3 grid(std::min(1 << a.shift, a.e.vocabulary), slabs);
  switch (edge_of<T>(a.e.dim)) {
    case EDGE_WHOLE:
      hipLaunchKernelGGL((embed_few_kernel<T, EDGE_WHOLE>), grid, dim3(64 * kEmbedFewWaves), 0, stream, a);
      break;
    case EDGE_CUT:
      hipLaunchKernelGGL((embed_few_kernel<T, EDGE_CUT>), grid, dim3(64 * kEmbedFewWaves), 0, stream, a);
      break;
    default:
      hipLaunchKernelGGL((embed_few_kernel<T, EDGE_SHORT>), grid, dim3(64 * kEmbedFewWaves), 0, stream, a);
  }
  return hipGetLastError();
}

template <typename F>
static void with_bits(int bits, F&& f) {
  using std::integral_constant;
  switch (bits) {
    case 5: return f(integral_constant<int, 5>{});
    case 6: return f(integral_constant<int, 6>{});
    case 7: return f(integral_constant<int, 7>{});
    case 8: return f(integral_constant<int, 8>{});
    default: return f(integral_constant<int, 9>{});
  }
}

hipError_t launch_embed_bwd(const void* ids, bool ids64, const void* dout, long long stride,
                            bool f32, int tokens, int vocabulary, int dim, long long padding,
                            float scale, void* dtable, void* workspace, hipStream_t stream) {
  if (embed_few(tokens, vocabulary, dim, f32)) {
    const FewArgs a{EmbedArgs{ids, nullptr, dtable, 0, padding, tokens, vocabulary, dim, scale, ids64},
                    dout, stride, few_shift(few_slabs(dim, f32 ? 4 : 8))};
    return f32 ? launch_few<float>(a, stream) : launch_few<bf16>(a, stream);
  }
  const EmbedLayout l = embed_layout(tokens, vocabulary, dim);
  char* ws = reinterpret_cast<char*>(workspace);
  SortedToken* lists[2] = {reinterpret_cast<SortedToken*>(ws + l.tokens[0]),
                           reinterpret_cast<SortedToken*>(ws + l.tokens[1])};
  SortArgs s{};
  s.e = EmbedArgs{ids, nullptr, dtable, stride, padding, tokens, vocabulary, dim, scale, ids64};
  s.histogram = reinterpret_cast<int*>(ws + l.histogram);
  s.tiles = l.tiles;
  s.steps = l.steps;
  s.bits = l.bits;
  s.passes = l.passes;
  const size_t bytes = (size_t)vocabulary * dim * (f32 ? 4 : 2);
  SortedToken* sorted = lists[0];
  if (l.steps == 0) {
    s.to = sorted;
    s.zero_last = bytes;
    s.zero_block = 256 << 10;
    const unsigned zero = (unsigned)((bytes + s.zero_block - 1) / s.zero_block);
    with_bits(l.bits, [&](auto b) {
      constexpr int B = decltype(b)::value;
      // (900 tokens of 1000 rows: 5.2 us, with room for 8192 9.2)
      if (tokens <= 1024)
        hipLaunchKernelGGL((sort_one_kernel<B, 1>), dim3(1 + zero), dim3(1024), 0, stream, s);
      else
        hipLaunchKernelGGL((sort_one_kernel<B, kSortOne / 1024>), dim3(1 + zero), dim3(1024), 0,
                           stream, s);
    });
  } else {
    s.zero_block = 64 << 10;
    // placing takes about twice what counting does (5.8 us and 3.3 at 32768 tokens, by
    // themselves): so are their shares
    const size_t share = (bytes / (3 * l.passes) / s.zero_block + 1) * s.zero_block;
    for (int step = 0; step < 2 * l.passes; ++step) {
      const int pass = step / 2;
      s.shift = pass * l.bits;
      s.from = pass ? lists[(pass + 1) & 1] : nullptr;
      s.to = sorted = lists[pass & 1];
      s.zero_first = s.zero_last;
      s.zero_last = std::min(bytes, (pass * 3 + (step % 2 ? 3 : 1)) * share);
      const unsigned zero =
          (unsigned)((s.zero_last - s.zero_first + s.zero_block - 1) / s.zero_block);
      const dim3 grid((unsigned)s.tiles + zero);
      if (step % 2 == 0)
        hipLaunchKernelGGL(sort_count_kernel, grid, dim3(512), 0, stream, s);
      else
        with_bits(l.bits, [&](auto b) {
          hipLaunchKernelGGL((sort_place_kernel<decltype(b)::value>), grid, dim3(512), 0, stream, s);
        });
    }
  }
  const SumArgs a{sorted, dout, dtable, reinterpret_cast<float*>(ws + l.partials), stride, tokens,
                  vocabulary, dim, l.width, l.chunk, l.chunks, 0, scale};
  return f32 ? launch_sums<float>(a, stream) : launch_sums<bf16>(a, stream);
}

}  // namespace mf
