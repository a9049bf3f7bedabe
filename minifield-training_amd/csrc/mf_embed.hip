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
// order, so a token that is half of the batch costs no more than any other.  A wave
// holds its columns' sum in registers and writes a row when the id changes; what
// runs past its chunk's ends goes to a workspace in fp32, and a last launch adds
// those pieces in chunk order.  The rows of ids that no token has are zeros: the
// launches that sort, which are a few waves' work each, zero the whole table beside
// it, a share each.
//
// The sort goes by digits of up to 9 bits from the lowest.  A wave takes a run of
// tokens, 64 at a time; lanes with one digit find each other by ballots over its
// bits, so that a lane's place is its digit's first place, what the waves and rounds
// before have of that digit, and the lanes before it.
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

// The table's row of token n, `vocabulary` for none.
__device__ __forceinline__ uint32_t row_of(const EmbedArgs& a, int n) {
  const long long id = a.ids64 ? reinterpret_cast<const long long*>(a.ids)[n]
                               : (long long)reinterpret_cast<const int32_t*>(a.ids)[n];
  return id >= 0 && id < a.vocabulary && id != a.padding ? (uint32_t)id : (uint32_t)a.vocabulary;
}

// L lanes a token.
template <typename T, int L, bool TAIL>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs a) {
  constexpr int N = kVec<T>, C = 4;
  const int n = blockIdx.x * (256 / L) + threadIdx.x / L, lane = threadIdx.x % L;
  if (n >= a.tokens) return;
  const uint32_t id = row_of(a, n);
  const bool met = id < (uint32_t)a.vocabulary;
  const T* from = reinterpret_cast<const T*>(a.rows) + (size_t)(met ? id : 0) * a.stride;
  T* to = reinterpret_cast<T*>(a.out) + (size_t)n * a.dim;
  for (int first = 0; first < a.dim; first += L * N * C) {
    Vec<T> v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = load_row<T, TAIL>(from, first + (c * L + lane) * N, a.dim);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = met ? (float)v[c][i] * a.scale : 0.f;
      store_row<T, TAIL>(to, first + (c * L + lane) * N, a.dim, x);
    }
  }
}

// ---------------------------------------------------------------------------

struct SortArgs {
  EmbedArgs e;
  const SortedToken* from;  // null: the ids as they come
  SortedToken* to;
  int* histogram;           // [tiles][kSortBins]
  int tiles, rounds, shift, bits, blocks;
  // a share of the table's gradient to zero, in bytes
  size_t zero_first, zero_last;
};

__device__ __forceinline__ SortedToken sort_entry(const SortArgs& a, int n) {
  return a.from ? a.from[n] : SortedToken{row_of(a.e, n), (uint32_t)n};
}

constexpr int kZeroBlock = 64 << 10;  // bytes that a workgroup zeroes

__device__ __forceinline__ void zero_share(const SortArgs& a) {
  const size_t first = a.zero_first + (size_t)(blockIdx.x - a.blocks) * kZeroBlock;
  const size_t last = min(a.zero_last, first + kZeroBlock);
  char* out = reinterpret_cast<char*>(a.e.out);
  for (size_t at = first + threadIdx.x * 16; at < last; at += 256 * 16) {
    if (at + 16 <= last) {
      *reinterpret_cast<u32x4*>(out + at) = u32x4{0, 0, 0, 0};
    } else {
      for (size_t b = at; b < last; b += 2) *reinterpret_cast<uint16_t*>(out + b) = 0;
    }
  }
}

// Lanes of the wave that have this lane's digit, among those that take part.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool live) {
  uint64_t same = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot(digit >> b & 1);
    same &= digit >> b & 1 ? set : ~set;
  }
  return same;
}

// How many of its tokens each wave has of every digit.
__global__ __launch_bounds__(256) void sort_count_kernel(SortArgs a) {
  __shared__ int counts[4][kSortBins];
  if ((int)blockIdx.x >= a.blocks) return zero_share(a);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int tile = blockIdx.x * 4 + wave;
  for (int d = lane; d < kSortBins; d += 64) counts[wave][d] = 0;
  __syncthreads();
  if (tile < a.tiles)
    for (int r = 0; r < a.rounds; ++r) {
      const int n = (tile * a.rounds + r) * 64 + lane;
      if (n < a.e.tokens)
        atomicAdd(&counts[wave][sort_entry(a, n).key >> a.shift & ((1 << a.bits) - 1)], 1);
    }
  __syncthreads();
  if (tile < a.tiles)
    for (int d = lane; d < kSortBins; d += 64)
      a.histogram[(size_t)tile * kSortBins + d] = counts[wave][d];
}

__global__ __launch_bounds__(256) void sort_place_kernel(SortArgs a) {
  __shared__ int place[4][kSortBins];
  __shared__ int wave_sums[4];
  if ((int)blockIdx.x >= a.blocks) return zero_share(a);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // digits 2 tid and 2 tid + 1: all of them, and those of the workgroup's waves' forerunners
  int whole[2] = {0, 0};
  for (int t = 0; t < a.tiles; ++t) {
    if ((t & 3) == 0 && t == (int)blockIdx.x * 4) place[0][2 * tid] = whole[0], place[0][2 * tid + 1] = whole[1];
    const int2 h = *reinterpret_cast<const int2*>(a.histogram + (size_t)t * kSortBins + 2 * tid);
    whole[0] += h.x;
    whole[1] += h.y;
  }
  // first place of the thread's two digits: an exclusive sum over the threads
  const int pair = whole[0] + whole[1];
  int sum = pair;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(sum, m);
    if (lane >= m) sum += o;
  }
  if (lane == 63) wave_sums[wave] = sum;
  __syncthreads();
  int start = sum - pair;
  for (int i = 0; i < wave; ++i) start += wave_sums[i];
  int at[2] = {start + place[0][2 * tid], start + whole[0] + place[0][2 * tid + 1]};
  for (int i = 0; i < 4; ++i) {
    place[i][2 * tid] = at[0];
    place[i][2 * tid + 1] = at[1];
    const int t = blockIdx.x * 4 + i;
    if (t < a.tiles) {
      const int2 h = *reinterpret_cast<const int2*>(a.histogram + (size_t)t * kSortBins + 2 * tid);
      at[0] += h.x;
      at[1] += h.y;
    }
  }
  __syncthreads();
  const int tile = blockIdx.x * 4 + wave;
  if (tile >= a.tiles) return;
  for (int r = 0; r < a.rounds; ++r) {
    const int n = (tile * a.rounds + r) * 64 + lane;
    const bool live = n < a.e.tokens;
    const SortedToken t = live ? sort_entry(a, n) : SortedToken{0, 0};
    const uint32_t digit = t.key >> a.shift & ((1 << a.bits) - 1);
    const uint64_t same = same_digit(digit, a.bits, live);
    const int before = __popcll(same & ((1ull << lane) - 1));
    // (the wave's own counters; its LDS operations keep their order)
    volatile int* counter = &place[wave][digit];
    int to = 0;
    if (live) {
      to = *counter + before;
      if (before == 0) *counter = to + __popcll(same);
      a.to[to] = t;
    }
  }
}

// ---------------------------------------------------------------------------

struct SumArgs {
  const SortedToken* sorted;
  const void* dout;
  void* dtable;
  float* partials;  // [chunks][2][dim]: what a chunk has of the run it begins in, and ends in
  long long stride;
  int tokens, vocabulary, dim, chunks, slabs;
  float scale;
};

// A wave adds the tokens of a chunk over 64 vectors of columns.
template <typename T, bool TAIL>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
  constexpr int N = kVec<T>, AHEAD = 8;
  const int lane = threadIdx.x & 63;
  const int item = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int chunk = item / a.slabs, col = ((item % a.slabs) * 64 + lane) * N;
  if (chunk >= a.chunks) return;
  const int first = chunk * kEmbedChunk, count = min(kEmbedChunk, a.tokens - first);
  // lane i < 32 holds entry i; the keys on either side of the chunk beside them
  const SortedToken mine = a.sorted[first + min(lane, count - 1)];
  const uint32_t none = a.vocabulary;
  const uint32_t before = first > 0 ? a.sorted[first - 1].key : none;
  const uint32_t behind = first + count < a.tokens ? a.sorted[first + count].key : none;
  // tokens without a row come last
  const int live = __popcll(__ballot(lane < count && mine.key < none));
  const T* dout = reinterpret_cast<const T*>(a.dout);
  auto key_at = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane(mine.key, i); };
  auto fetch = [&](int i) {
    const uint32_t token = __builtin_amdgcn_readlane(mine.token, min(i, count - 1));
    return load_row<T, TAIL, true>(dout + (size_t)token * a.stride, col, a.dim);
  };
  float sum[N] = {};
  bool head = live > 0 && key_at(0) == before;
  for (int i0 = 0; i0 < live; i0 += AHEAD) {
    Vec<T> v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i0 + j < live) v[j] = fetch(i0 + j);
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
        float* to = a.partials + ((size_t)chunk * 2 + (head ? 0 : 1)) * a.dim;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (col + e < a.dim) to[col + e] = sum[e];
      } else {
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = sum[e] * a.scale;
        store_row<T, TAIL>(reinterpret_cast<T*>(a.dtable) + (size_t)key * a.dim, col, a.dim, x);
      }
      head = false;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = 0.f;
    }
  }
}

// The runs that pass a chunk's end: the workgroup of the chunk that one begins in adds
// its pieces, each wave a quarter of the chunks, in order.
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a) {
  __shared__ float sums[4][64];
  const int chunk = blockIdx.x, first = chunk * kEmbedChunk;
  const int next = first + kEmbedChunk;
  if (next >= a.tokens) return;
  const uint32_t key = a.sorted[next - 1].key;
  if (key >= (uint32_t)a.vocabulary || a.sorted[next].key != key) return;
  // the run fills the chunk from an earlier one on: it is that one's
  if (first > 0 && a.sorted[first - 1].key == key) return;
  // the run's end, by bisection
  int lo = next, hi = a.tokens;  // sorted[lo] has the key; the first beyond it is in (lo, hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.sorted[mid].key == key)
      lo = mid;
    else
      hi = mid;
  }
  const int last = lo / kEmbedChunk;  // the last chunk with a piece
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.y * 64 + lane;
  const int per = (last - chunk + 4) / 4;
  const int from = chunk + wave * per, to = min(last + 1, from + per);
  float s = 0.f;
  if (col < a.dim) {
#pragma unroll 8
    for (int c = from; c < to; ++c)
      s += a.partials[((size_t)c * 2 + (c == chunk ? 1 : 0)) * a.dim + col];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || col >= a.dim) return;
  s += sums[1][lane];
  s += sums[2][lane];
  s += sums[3][lane];
  reinterpret_cast<T*>(a.dtable)[(size_t)key * a.dim + col] = (T)(s * a.scale);
}

// ---------------------------------------------------------------------------

template <typename T, bool TAIL>
static void launch_embed_t(const EmbedArgs& a, hipStream_t stream) {
  const int vectors = (a.dim + kVec<T> - 1) / kVec<T>;
  auto go = [&](auto l) {
    constexpr int L = decltype(l)::value;
    hipLaunchKernelGGL((embed_kernel<T, L, TAIL>), dim3((a.tokens + 256 / L - 1) / (256 / L)),
                       dim3(256), 0, stream, a);
  };
  if (vectors <= 16)
    go(std::integral_constant<int, 16>{});
  else
    go(std::integral_constant<int, 64>{});
}

hipError_t launch_embed(const void* ids, bool ids64, const void* table, long long stride, bool f32,
                        int tokens, int vocabulary, int dim, long long padding, float scale,
                        void* out, hipStream_t stream) {
  const EmbedArgs a{ids, table, out, stride, padding, tokens, vocabulary, dim, scale, ids64};
  const bool tail = dim % (f32 ? 4 : 8);
  if (f32)
    tail ? launch_embed_t<float, true>(a, stream) : launch_embed_t<float, false>(a, stream);
  else
    tail ? launch_embed_t<bf16, true>(a, stream) : launch_embed_t<bf16, false>(a, stream);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_sums(SumArgs a, hipStream_t stream) {
  a.slabs = (a.dim + 64 * kVec<T> - 1) / (64 * kVec<T>);
  const dim3 grid((unsigned)(((long long)a.chunks * a.slabs + 3) / 4));
  if (a.dim % kVec<T>)
    hipLaunchKernelGGL((embed_sum_kernel<T, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((embed_sum_kernel<T, false>), grid, dim3(256), 0, stream, a);
  if (a.chunks > 1)
    hipLaunchKernelGGL((embed_join_kernel<T>), dim3(a.chunks - 1, (a.dim + 63) / 64), dim3(256), 0,
                       stream, a);
  return hipGetLastError();
}

hipError_t launch_embed_bwd(const void* ids, bool ids64, const void* dout, long long stride,
                            bool f32, int tokens, int vocabulary, int dim, long long padding,
                            float scale, void* dtable, void* workspace, hipStream_t stream) {
  const EmbedLayout l = embed_layout(tokens, vocabulary, dim);
  char* ws = reinterpret_cast<char*>(workspace);
  SortedToken* lists[2] = {reinterpret_cast<SortedToken*>(ws + l.tokens[0]),
                           reinterpret_cast<SortedToken*>(ws + l.tokens[1])};
  SortArgs s{};
  s.e = EmbedArgs{ids, nullptr, dtable, stride, padding, tokens, vocabulary, dim, scale, ids64};
  s.histogram = reinterpret_cast<int*>(ws + l.histogram);
  s.tiles = l.tiles;
  s.rounds = l.rounds;
  s.blocks = (l.tiles + 3) / 4;
  const size_t bytes = (size_t)vocabulary * dim * (f32 ? 4 : 2);
  const int launches = 2 * l.passes;
  const size_t share = (bytes / launches / kZeroBlock + 1) * kZeroBlock;
  for (int pass = 0; pass < l.passes; ++pass) {
    s.shift = pass * l.bits;
    s.bits = l.bits;
    s.from = pass ? lists[(pass + 1) & 1] : nullptr;
    s.to = lists[pass & 1];
    for (int step = 0; step < 2; ++step) {
      const size_t k = 2 * pass + step;
      s.zero_first = std::min(bytes, k * share);
      s.zero_last = std::min(bytes, (k + 1) * share);
      const unsigned zero = (unsigned)((s.zero_last - s.zero_first + kZeroBlock - 1) / kZeroBlock);
      const dim3 grid((unsigned)s.blocks + zero);
      if (step == 0)
        hipLaunchKernelGGL(sort_count_kernel, grid, dim3(256), 0, stream, s);
      else
        hipLaunchKernelGGL(sort_place_kernel, grid, dim3(256), 0, stream, s);
    }
  }
  SumArgs a{lists[(l.passes + 1) & 1], dout, dtable, reinterpret_cast<float*>(ws + l.partials), stride,
            tokens, vocabulary, dim, l.chunks, 0, scale};
  return f32 ? launch_sums<float>(a, stream) : launch_sums<bf16>(a, stream);
}

}  // namespace mf
